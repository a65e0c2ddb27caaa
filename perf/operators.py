"""The training-step operators of smart_compress_amd and the cases they are measured on.

Three operators: group norm with an activation on channels-last tensors (``group_norm``), softmax
cross entropy of a linear head over a vocabulary (``cross_entropy``), and the Newton-Schulz
orthogonalisation of an update (``orthogonalize``). ``run`` computes them in elementary torch
operations, or, where ``own`` is true, through the package's entry points.
"""

import functools
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
NS_STEPS = 5
NS_EPS = 1e-7
GN_EPS = 1e-5
IGNORE = -100


def _gn(name, n, c, h, w, groups, dtype, act, train):
    return {"name": name, "op": "group_norm", "n": n, "c": c, "h": h, "w": w, "groups": groups,
            "dtype": dtype, "act": act, "train": train}


def _ce(name, tokens, dim, vocab, dtype, ignored, train):
    return {"name": name, "op": "cross_entropy", "tokens": tokens, "dim": dim, "vocab": vocab,
            "dtype": dtype, "ignored": ignored, "train": train}


def _ns(name, batch, m, n, dtype):
    return {"name": name, "op": "orthogonalize", "batch": batch, "m": m, "n": n, "dtype": dtype}


def listed():
    return [
        # one small feature map at inference: launch latency
        _gn("gn_small_f32", 2, 64, 8, 8, 32, "f32", "relu", False),
        # ResNet-34 on CIFAR at batch 128, first stage, in place of its batch norm + ReLU
        _gn("gn_resnet_f32_train", 128, 64, 32, 32, 32, "f32", "relu", True),
        # a mid-level feature map of an image network, forward, half precision
        _gn("gn_mid_f16", 8, 320, 64, 64, 32, "f16", "silu", False),
        # a ragged map: 7 channels a group, odd height and width
        _gn("gn_odd_bf16_train", 3, 84, 31, 17, 12, "bf16", "gelu", True),
        # a large feature map: far more than the caches hold
        _gn("gn_large_bf16_train", 4, 256, 256, 256, 32, "bf16", "silu", True),
        # scoring one token under a small model's vocabulary: the read of the weight
        _ce("ce_token_f32", 1, 768, 30000, "f32", 0.0, False),
        # a small model's training step in the framework's usual float32, some targets padding
        _ce("ce_small_f32_train", 2048, 768, 30000, "f32", 0.15, True),
        # a ragged step: odd tokens, width and vocabulary, a third of the targets ignored
        _ce("ce_odd_f16_train", 777, 1001, 50001, "f16", 0.33, True),
        # a language model's step: 8192 tokens over a vocabulary of 131072
        _ce("ce_large_bf16_train", 8192, 4096, 131072, "bf16", 0.0, True),
        # one small odd matrix: launch latency
        _ns("ns_small_f32", 1, 97, 161, "f32"),
        # a 3x3 convolution of ResNet-34's last stage (512 x 512 x 3 x 3) as a matrix
        _ns("ns_conv_f32", 1, 512, 4608, "f32"),
        # six equal projections of a transformer's update, stacked
        _ns("ns_stack_bf16", 6, 1024, 4096, "bf16"),
    ]


def _log_int(rng, lo, hi):
    v = int(round(lo * (hi / lo) ** rng.random()))
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["group_norm", "cross_entropy", "orthogonalize"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "group_norm":
        while True:
            groups = rng.choice([1, 2, 3, 4, 8, 12, 16, 32])
            c = groups * _log_int(rng, 1, 32)
            n, h, w = _log_int(rng, 1, 128), _log_int(rng, 1, 256), _log_int(rng, 1, 256)
            size = 4 if dtype == "f32" else 2
            if 128 <= n * c * h * w <= (1 << 27) // size and c // groups * h * w >= 8:
                break
        act = rng.choice(["none", "relu", "silu", "gelu"])
        case = _gn("", n, c, h, w, groups, dtype, act, rng.random() < 0.6)
    elif op == "cross_entropy":
        while True:
            tokens, dim, vocab = (_log_int(rng, 1, 8192), _log_int(rng, 64, 4096),
                                  _log_int(rng, 1000, 131072))
            if tokens * dim * vocab <= 1 << 40 and tokens * vocab <= 1 << 30:
                break
        case = _ce("", tokens, dim, vocab, dtype, rng.choice([0.0, 0.0, 0.1, 0.5]),
                   rng.random() < 0.7)
    else:
        while True:
            batch, m, n = _log_int(rng, 1, 16), _log_int(rng, 16, 4096), _log_int(rng, 16, 8192)
            if batch * min(m, n) ** 2 * max(m, n) <= 6 << 32 and batch * m * n <= 1 << 25:
                break
        case = _ns("", batch, m, n, dtype)
    del case["name"]
    return case


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    if case["op"] == "group_norm":
        n, c, h, w = case["n"], case["c"], case["h"], case["w"]
        # convolution outputs: every channel its own offset and spread
        spread = 0.5 + torch.rand(c, generator=g, device=dev)
        shift = randn(c)
        x = (randn(n, h, w, c) * spread + shift).to(dt).permute(0, 3, 1, 2)
        state = {"x": x, "weight": 1.0 + 0.2 * randn(c), "bias": 0.2 * randn(c)}
        if case["train"]:
            state["dy"] = randn(n, h, w, c).to(dt).permute(0, 3, 1, 2)
    elif case["op"] == "cross_entropy":
        tokens, dim, vocab = case["tokens"], case["dim"], case["vocab"]
        weight = randn(vocab, dim) * dim ** -0.5
        target = torch.randint(0, vocab, (tokens,), generator=g, device=dev)
        # hidden states of a model that has learned something: the target's logit stands out by up
        # to about 8
        lean = 8.0 * torch.rand(tokens, 1, generator=g, device=dev)
        hidden = randn(tokens, dim) + lean * weight[target]
        if case["ignored"]:
            skip = torch.rand(tokens, generator=g, device=dev) < case["ignored"]
            skip[0] = False
            target = torch.where(skip, torch.full_like(target, IGNORE), target)
        state = {"hidden": hidden.to(dt), "weight": weight.to(dt), "target": target}
    else:
        b, m, n = case["batch"], case["m"], case["n"]
        # a gradient: a few strong directions over noise
        k = max(1, min(m, n) // 16)
        x = torch.bmm(randn(b, m, k), randn(b, k, n)) * (k ** -0.5) + 0.5 * randn(b, m, n)
        state = {"update": (x if b > 1 else x[0]).mul_(1e-3).to(dt)}
    state["case"] = case
    return state


@functools.lru_cache(None)
def _package():
    """The package's entry points (its folder is not importable by name)."""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "smart-quantization_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from smart_compress_amd.util.pytorch.loss import linear_cross_entropy
    from smart_compress_amd.util.pytorch.muon import orthogonalize
    from smart_compress_amd.util.pytorch.norm import group_norm_act

    return group_norm_act, linear_cross_entropy, orthogonalize


def _act(z, name):
    """The activation and its derivative."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    phi = 0.5 * (1 + torch.erf(z * 0.7071067811865476))
    return z * phi, phi + z * torch.exp(-0.5 * z * z) * 0.3989422804014327


def _group_norm(s):
    case, x = s["case"], s["x"]
    n, c, h, w, k = case["n"], case["c"], case["h"], case["w"], case["groups"]
    xs = x.permute(0, 2, 3, 1).reshape(n, h * w, k, c // k).float()
    mean = xs.mean((1, 3), keepdim=True)
    var = ((xs - mean) ** 2).mean((1, 3), keepdim=True)
    rstd = (var + GN_EPS) ** -0.5
    xhat = (xs - mean) * rstd
    gamma, beta = s["weight"].view(k, c // k), s["bias"].view(k, c // k)
    y, slope = _act(xhat * gamma + beta, case["act"])

    def out(t):
        return t.reshape(n, h, w, c).to(x.dtype).permute(0, 3, 1, 2)

    if not case["train"]:
        return out(y)
    dz = s["dy"].permute(0, 2, 3, 1).reshape(n, h * w, k, c // k).float() * slope
    dgamma, dbeta = (dz * xhat).sum((0, 1)).view(c), dz.sum((0, 1)).view(c)
    dn = dz * gamma
    dx = rstd * (dn - dn.mean((1, 3), keepdim=True)
                 - xhat * (dn * xhat).mean((1, 3), keepdim=True))
    return out(y), out(dx), dgamma, dbeta


def _cross_entropy(s):
    hidden, weight, target = s["hidden"], s["weight"], s["target"]
    h, w = hidden.float(), weight.float()
    keep = target != IGNORE
    at = torch.where(keep, target, torch.zeros_like(target)).view(-1, 1)
    count = keep.sum().float()
    logits = h @ w.t()
    top = logits.amax(1, keepdim=True)
    picked = logits.gather(1, at) - top
    p = logits.sub_(top).exp_()
    total = p.sum(1, keepdim=True)
    loss = ((total.log() - picked).view(-1) * keep).sum() / count
    if not s["case"]["train"]:
        return loss
    dl = p.div_(total)
    dl.scatter_add_(1, at, -torch.ones_like(picked))
    dl.mul_((keep / count).view(-1, 1))
    return loss, (dl @ w).to(hidden.dtype), (dl.t() @ h).to(weight.dtype)


def _orthogonalize(s):
    update = s["update"]
    x = update.float()
    x = x if x.dim() == 3 else x.unsqueeze(0)
    turned = x.shape[1] > x.shape[2]
    if turned:
        x = x.transpose(1, 2).contiguous()
    norm = (x.double() ** 2).sum((1, 2), keepdim=True) ** 0.5
    x = x / (norm + NS_EPS).float()
    a, b, c = NS_COEFFICIENTS
    for _ in range(NS_STEPS):
        gram = torch.bmm(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.bmm(b * gram + c * torch.bmm(gram, gram), x)
    x = x.transpose(1, 2) if turned else x
    return x.reshape(update.shape).to(update.dtype)


def run(state):
    case = state["case"]
    if own:
        group_norm_act, linear_cross_entropy, orthogonalize = _package()
        if case["op"] == "group_norm":
            args = (case["groups"],)
            kw = {"eps": GN_EPS, "activation": case["act"]}
            if not case["train"]:
                return group_norm_act(state["x"], *args, state["weight"], state["bias"], **kw)
            leaves = [state[k].detach().requires_grad_() for k in ("x", "weight", "bias")]
            y = group_norm_act(leaves[0], *args, leaves[1], leaves[2], **kw)
            return (y.detach(), *torch.autograd.grad(y, leaves, state["dy"]))
        if case["op"] == "cross_entropy":
            if not case["train"]:
                return linear_cross_entropy(state["hidden"], state["weight"], state["target"],
                                            ignore_index=IGNORE)
            leaves = [state[k].detach().requires_grad_() for k in ("hidden", "weight")]
            loss = linear_cross_entropy(*leaves, state["target"], ignore_index=IGNORE)
            return (loss.detach(), *torch.autograd.grad(loss, leaves))
        return orthogonalize(state["update"], steps=NS_STEPS, coefficients=NS_COEFFICIENTS,
                             eps=NS_EPS)
    if case["op"] == "group_norm":
        return _group_norm(state)
    if case["op"] == "cross_entropy":
        return _cross_entropy(state)
    return _orthogonalize(state)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "group_norm":
        elems = case["n"] * case["c"] * case["h"] * case["w"]
        if not case["train"]:
            return {"bytes": 2 * elems * size + 8 * case["c"], "flops": 10 * elems}
        # forward: x in, y out; backward: x and dy in, dx out
        return {"bytes": 5 * elems * size + 24 * case["c"], "flops": 40 * elems}
    if case["op"] == "cross_entropy":
        t, d, v = case["tokens"], case["dim"], case["vocab"]
        once = (t + v) * d * size + 8 * t
        if not case["train"]:
            return {"bytes": once, "flops": 2 * t * d * v}
        return {"bytes": 2 * once, "flops": 6 * t * d * v}
    b, m, n = case["batch"], case["m"], case["n"]
    m, n = min(m, n), max(m, n)
    # A and A^2 are symmetric: half of each is enough
    return {"bytes": 2 * b * m * n * size, "flops": NS_STEPS * b * (3 * m * m * n + m * m * m)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "group_norm":
        x = s["x"].double().requires_grad_()
        gamma, beta = s["weight"].double().requires_grad_(), s["bias"].double().requires_grad_()
        n, c, k = case["n"], case["c"], case["groups"]
        v = x.reshape(n, k, -1)
        dev = v - v.mean(2, keepdim=True)
        norm = dev / torch.sqrt((dev * dev).mean(2, keepdim=True) + GN_EPS)
        z = norm.reshape(x.shape) * gamma.view(1, c, 1, 1) + beta.view(1, c, 1, 1)
        if case["act"] == "relu":
            z = torch.relu(z)
        elif case["act"] == "silu":
            z = z * torch.sigmoid(z)
        elif case["act"] == "gelu":
            z = z * torch.special.ndtr(z)
        if not case["train"]:
            return z.detach()
        return (z.detach(), *torch.autograd.grad(z, [x, gamma, beta], s["dy"].double()))
    if case["op"] == "cross_entropy":
        h, w, t = s["hidden"].double(), s["weight"].double(), s["target"]
        rows = torch.nonzero(t != IGNORE).view(-1)
        logits = h[rows] @ w.t()
        lse = torch.logsumexp(logits, 1)
        index = (torch.arange(rows.numel(), device=t.device), t[rows])
        loss = (lse - logits[index]).mean()
        if not case["train"]:
            return loss
        grad = logits.sub_(lse.view(-1, 1)).exp_()
        grad[index] -= 1.0
        grad /= rows.numel()
        dh = torch.zeros_like(h)
        dh[rows] = grad @ w
        return loss, dh, grad.t().contiguous() @ h[rows]
    x = s["update"].double()
    shape = x.shape
    x = x.reshape(-1, shape[-2], shape[-1])
    a, b, c = NS_COEFFICIENTS
    results = []
    for one in x:
        flip = one.shape[0] > one.shape[1]
        y = (one.t() if flip else one).contiguous()
        y = y / (torch.linalg.vector_norm(y) + NS_EPS)
        eye = torch.eye(y.shape[0], dtype=y.dtype, device=y.device)
        for _ in range(NS_STEPS):
            gram = y @ y.t().contiguous()
            y = (a * eye + gram @ (b * eye + c * gram)) @ y
        results.append(y.t() if flip else y)
    return torch.stack(results).reshape(shape)
