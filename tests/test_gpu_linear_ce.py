"""linear_cross_entropy / LinearCrossEntropy on the GPU against the formula in float64.

Tolerances. u = 2^-24, k = dim. A logit is a float32 sum of k products in runs of 16: off by at most
e = (k / 16 + 24) u max_v sum|h w| (float32 inputs: each factor also off by 2^-23, the dropped product
of the low planes by 2^-24: within the 24). The loss is off by 2 e + 8 u (|lse| + |logit|). dl = g (p - 1) is
off by g p (2 e + 8 u) and rounds to an operand: half a step is 2^-11 (fp16, 10 stored bits) relative,
or 2^-23 (two planes: what hi leaves is below 2^-11, of which lo's half step is 2^-12 at most), and
2^-38 of the largest g absolute; the gradient products add (n / 16 + 24) u of their sums of magnitudes
over n terms and round to the inputs' type by half a step."""

import pytest
import torch
import torch.nn.functional as F

from smart_compress_amd.util.pytorch.loss import LinearCrossEntropy, linear_cross_entropy

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def make(tokens, dim, vocab, dtype, bias, ignored, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn(tokens, dim, generator=g, device="cuda").to(dtype)
    w = (torch.randn(vocab, dim, generator=g, device="cuda") * 2 * dim ** -0.5).to(dtype)
    b = torch.randn(vocab, generator=g, device="cuda") if bias else None
    t = torch.randint(0, vocab, (tokens,), generator=g, device="cuda")
    if ignored:
        t[torch.rand(tokens, generator=g, device="cuda") < ignored] = -100
    return h, w, b, t


def reference(h, w, b, t, reduction, g, ignore=-100):
    """float64 loss and gradients, and the bounds of their errors (module docstring)."""
    H, W = h.double(), w.double()
    keep = t != ignore
    H = torch.where(keep[:, None], H, torch.zeros_like(H))
    at = torch.where(keep, t, torch.zeros_like(t))
    logits = H @ W.t()
    size = (H.abs() @ W.abs().t()).amax(1)
    if b is not None:
        logits = logits + b.double()
        size = size + b.double().abs().max()
    lse = torch.logsumexp(logits, 1)
    pick = logits.gather(1, at[:, None])[:, 0]
    rows = torch.where(keep, lse - pick, torch.zeros_like(lse))
    count = keep.sum().double()
    e = (h.shape[1] / 16 + 24) * U * size
    br = 2 * e + 8 * U * (lse.abs() + pick.abs())
    if reduction == "none":
        loss, bl = rows, br
        gr = g.double() * keep
    else:
        div = count if reduction == "mean" else torch.ones_like(count)
        loss, bl = rows.sum() / div, (br * keep).sum() / div
        gr = g.double() / div * keep
    p = torch.exp(logits - lse[:, None])
    dl = p.clone()
    dl[torch.arange(len(t)), at] -= 1
    dl = dl * gr[:, None]
    half = 2.0 ** -23 if h.dtype == torch.float32 else 2.0 ** -11
    bdl = (gr.abs()[:, None] * p * (2 * e[:, None] + 8 * U) + dl.abs() * half
           + gr.abs().max() * 2.0 ** -38)

    def product(a, ba, c):
        n = a.shape[1]
        extra = 2.0 ** -23 * (a.abs() @ c.abs())  # planes of c, the scale's rounding
        return a @ c, ba @ c.abs() + ((n / 16 + 24) * U) * (a.abs() @ c.abs()) + extra

    dh, bh = product(dl, bdl, W)
    dw, bw = product(dl.t().contiguous(), bdl.t().contiguous(), H)
    db, bb = dl.sum(0), bdl.sum(0) + (len(t) / 8 + 24) * U * dl.abs().sum(0)
    return loss, bl, (dh, dw, db), (bh, bw, bb)


def close(got, want, bound, dtype):
    step = torch.finfo(dtype).eps / 2 * want.abs() + torch.finfo(dtype).smallest_normal * \
        torch.finfo(dtype).eps / 2
    assert not torch.isnan(got).any()
    over = ((got.double() - want).abs() - bound - step).max().item()
    assert over <= 0, f"over the bound by {over:.3g}"


def check(h, w, b, t, reduction, piece=0, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    grad = (torch.randn(len(t), generator=g, device="cuda") if reduction == "none"
            else torch.tensor(-1.7, device="cuda"))
    leaves = [x.detach().requires_grad_() for x in (h, w, b) if x is not None]
    loss = linear_cross_entropy(leaves[0], leaves[1], t, leaves[2] if b is not None else None,
                                reduction=reduction, vocab_piece=piece)
    assert loss.dtype == torch.float32
    got = torch.autograd.grad(loss, leaves, grad)
    want, bl, grads, bounds = reference(h, w, b, t, reduction, grad)
    close(loss, want, bl, torch.float32)
    for x, e, bound, leaf in zip(got, grads, bounds, leaves):
        assert x.shape == leaf.shape and x.dtype == leaf.dtype
        close(x, e, bound, leaf.dtype)
    return loss, got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,dim,vocab,bias,reduction,ignored,piece", [
    (1, 64, 1000, True, "mean", 0, 0), (1, 1, 1, False, "sum", 0, 0), (2, 3, 5, True, "none", 0, 2),
    (7, 33, 517, True, "none", 0.3, 0), (9, 64, 200, False, "mean", 0, 0),
    (33, 64, 300, False, "sum", 0.3, 100), (130, 129, 2001, True, "none", 0.3, 500),
    (257, 128, 4097, False, "mean", 0.1, 0), (600, 256, 5003, True, "mean", 0.3, 2048),
    (1030, 72, 9000, True, "mean", 0.1, 9000)])
def test_loss_and_gradients(tokens, dim, vocab, bias, reduction, ignored, piece, dtype):
    check(*make(tokens, dim, vocab, dtype, bias, ignored, seed=tokens), reduction, piece)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,dim,vocab,ignored", [
    (1, 68, 1003, 0), (2, 66, 50, 0), (3, 77, 5001, 0.3), (5, 2048, 400, 0.3), (8, 4096, 133, 0),
    (11, 130, 3, 0.3), (16, 2048, 1001, 0.3), (16, 2049, 300, 0), (17, 64, 300, 0.3),
    (4, 8192, 90, 0), (4, 8200, 90, 0)])
def test_few_tokens(tokens, dim, vocab, ignored, dtype):
    """Up to 16 tokens go without matrix cores while hidden fits the LDS: every vector width, row count
    and both sides of the limits."""
    for reduction in ("mean", "none"):
        check(*make(tokens, dim, vocab, dtype, True, ignored, seed=dim), reduction)


def test_few_tokens_take_strided_weights():
    h, w, b, t = make(6, 48, 300, torch.float16, True, 0.2, seed=21)
    base = check(h, w, b, t, "mean")
    for pad in (1, 2, 4):
        wide = torch.randn(300, 48 + 2 * pad, device="cuda").half()
        wide[:, pad:pad + 48] = w
        other = check(h, wide[:, pad:pad + 48], b, t, "mean")
        assert abs(other[0].item() - base[0].item()) <= 64 * U * abs(base[0].item())


@pytest.mark.parametrize("tokens", [3, 40])
def test_gradients_that_are_not_finite(tokens):
    """A row's infinite gradient leaves the other rows of the hidden's gradient as they are."""
    h, w, _, t = make(tokens, 64, 200, torch.float32, False, 0, seed=22)
    g = torch.ones(tokens, device="cuda")
    leaf = h.detach().requires_grad_()
    want = torch.autograd.grad(linear_cross_entropy(leaf, w, t, reduction="none"), leaf, g)[0]
    g[1] = float("inf")
    got = torch.autograd.grad(linear_cross_entropy(leaf, w, t, reduction="none"), leaf, g)[0]
    assert not torch.isfinite(got[1]).any()
    got[1] = want[1]
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_tiles(dtype):
    check(*make(2100, 320, 20011, dtype, True, 0.2), "mean", 7001)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    h, w, b, t = make(40, 64, 333, dtype, True, 0.2, seed=4)
    wide = torch.randn(40, 200, device="cuda").to(dtype)
    wide[:, 3:67] = h
    turned = w.t().contiguous().t()
    tt = torch.stack([t, t], 1)[:, 0]
    a = check(h, w, b, t, "mean")
    c = check(wide[:, 3:67], turned, b, tt, "mean")
    assert torch.equal(a[0], c[0])
    check(h[:1].expand(40, 64), w, b, t, "sum")  # one row seen forty times


def test_batched_hidden_and_views():
    h, w, _, t = make(60, 32, 100, torch.float32, False, 0.1, seed=5)
    leaf = h.view(3, 20, 32).detach().requires_grad_()
    loss = linear_cross_entropy(leaf, w, t.view(3, 20), reduction="none")
    assert loss.shape == (3, 20)
    flat = linear_cross_entropy(h, w, t, reduction="none")
    assert torch.equal(loss.view(-1), flat)
    assert torch.autograd.grad(loss.sum(), leaf)[0].shape == leaf.shape


@pytest.mark.parametrize("dtype", DTYPES)
def test_ignored_rows_hold_anything(dtype):
    h, w, b, t = make(70, 64, 400, dtype, True, 0.4, seed=6)
    base = check(h, w, b, t, "mean")
    dirty = h.clone()
    rows = torch.nonzero(t == -100).view(-1)
    dirty[rows[0]], dirty[rows[1]], dirty[rows[2:]] = float("nan"), float("inf"), 0.0
    other = [x.detach().requires_grad_() for x in (dirty, w, b)]
    loss = linear_cross_entropy(other[0], other[1], t, other[2])
    grads = torch.autograd.grad(loss, other, torch.tensor(-1.7, device="cuda"))
    if dtype == torch.float32:  # its scale is taken over all rows, inf among them
        assert torch.isfinite(loss)
    else:
        assert torch.equal(loss, base[0])
    assert (grads[0][rows] == 0).all()
    for g in grads:
        assert torch.isfinite(g.float()).all()


def test_all_ignored():
    h, w, b, t = make(5, 32, 50, torch.float32, True, 0)
    t.fill_(-100)
    leaves = [x.requires_grad_() for x in (h, w, b)]
    loss = linear_cross_entropy(h, w, t, b)
    assert torch.isnan(loss)
    for g in torch.autograd.grad(loss, leaves):
        assert (g == 0).all()
    assert linear_cross_entropy(h, w, t, b, reduction="sum") == 0
    assert (linear_cross_entropy(h, w, t, b, reduction="none") == 0).all()


def test_target_out_of_range_is_nan_and_stays_in_its_row():
    h, w, _, t = make(6, 32, 50, torch.float32, False, 0, seed=7)
    t[2], t[4] = 50, -3
    leaf = h.detach().requires_grad_()
    rows = linear_cross_entropy(leaf, w, t, reduction="none")
    bad = torch.tensor([False, False, True, False, True, False], device="cuda")
    assert torch.equal(torch.isnan(rows), bad)
    g = torch.autograd.grad(rows.sum(), leaf)[0]
    assert torch.equal(torch.isnan(g).all(1), bad) and torch.equal(torch.isnan(g).any(1), bad)


def test_other_ignore_index_and_masked_vocabulary():
    h, w, b, t = make(50, 64, 300, torch.float32, True, 0, seed=8)
    b[200:] = float("-inf")  # entries that can not be
    t = t % 200
    t[::7] = 5
    want = F.cross_entropy((h.double() @ w.double().t() + b.double()), t, ignore_index=5)
    leaves = [x.detach().requires_grad_() for x in (h, w)]
    got = linear_cross_entropy(*leaves, t, b, ignore_index=5)
    assert abs(got.item() - want.item()) <= 64 * U * 20
    dw = torch.autograd.grad(got, leaves)[1]
    assert (dw[200:] == 0).all() and torch.isfinite(dw).all()
    low = b.clone()
    low[200:] = torch.finfo(torch.float32).min  # the type's lowest value masks as well
    assert torch.equal(linear_cross_entropy(h, w, t, low, ignore_index=5), got)


@pytest.mark.parametrize("scale", [2.0 ** -60, 1.0, 2.0 ** 40])
def test_float32_range(scale):
    """Float32 inputs of any size: the planes' exponents follow the largest magnitude."""
    h, w, _, t = make(40, 96, 500, torch.float32, False, 0, seed=9)
    a = check(h, w, None, t, "mean")
    leaves = [(h * scale).requires_grad_(), (w / scale).requires_grad_()]
    loss = linear_cross_entropy(*leaves, t)
    assert torch.equal(loss, a[0])
    dh = torch.autograd.grad(loss, leaves, torch.tensor(-1.7, device="cuda"))[0]
    assert torch.equal(dh * scale, a[1][0])


def test_selected_gradients():
    h, w, b, t = make(70, 64, 400, torch.bfloat16, True, 0.2, seed=10)
    _, full = check(h, w, b, t, "mean")
    for pick in range(3):
        leaves = [x.detach().requires_grad_(i == pick) for i, x in enumerate((h, w, b))]
        loss = linear_cross_entropy(leaves[0], leaves[1], t, leaves[2])
        got = torch.autograd.grad(loss, leaves[pick], torch.tensor(-1.7, device="cuda"))[0]
        assert torch.equal(got, full[pick])


def test_pieces_agree():
    h, w, b, t = make(300, 64, 3000, torch.bfloat16, True, 0.2, seed=11)
    _, one = check(h, w, b, t, "mean", 3000)
    for piece in (1, 255, 1024):
        if piece == 1:
            part = check(h, w[:9], b[:9], torch.where(t < 0, t, t % 9), "sum", 1)
            assert torch.isfinite(part[0])
            continue
        _, got = check(h, w, b, t, "mean", piece)
        assert torch.equal(got[1], one[1]) and torch.equal(got[2], one[2])


def test_half_bias_and_module():
    m = LinearCrossEntropy(64, 300, device="cuda", dtype=torch.bfloat16)
    lin = torch.nn.Linear(64, 300, device="cuda", dtype=torch.bfloat16)
    m.load_state_dict(lin.state_dict())
    h, _, _, t = make(20, 64, 300, torch.bfloat16, False, 0.1, seed=12)
    loss = m(h, t)
    want, bl, _, _ = reference(h, lin.weight.detach(), lin.bias.detach().float(), t, "mean",
                               torch.tensor(1.0, device="cuda"))
    close(loss, want, bl, torch.float32)
    loss.backward()
    assert m.bias.grad.dtype == torch.bfloat16 and m.weight.grad.shape == (300, 64)


def test_directional_difference():
    h, w, b, t = make(12, 24, 70, torch.float32, True, 0.2, seed=13)
    leaves = [x.detach().requires_grad_() for x in (h, w, b)]
    loss = linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], reduction="sum")
    grads = torch.autograd.grad(loss, leaves)
    for i, grad in enumerate(grads):
        d = torch.randn_like(leaves[i])
        d /= d.norm()
        s = 2.0 ** -6
        f = [linear_cross_entropy(*[x + (s * k * d if j == i else 0) for j, x in
                                    enumerate(leaves[:2])], t,
                                  leaves[2] + (s * k * d if i == 2 else 0), reduction="sum").item()
             for k in (1, -1)]
        # rounding of two losses of ~60 over 2 s, and s^2 / 6 of a third derivative below 12 * |h|^3
        assert abs((f[0] - f[1]) / (2 * s) - (grad * d).sum().item()) <= \
            64 * 60 * U / s + s * s / 6 * 12 * h.norm(dim=1).max().item() ** 3 * 0.1


def test_graph_replays():
    h, w, b, t = make(300, 128, 5000, torch.bfloat16, True, 0.2, seed=14)
    leaves = [x.detach().clone().requires_grad_() for x in (h, w, b)]

    def call():
        loss = linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], vocab_piece=2048)
        return (loss.detach(), *torch.autograd.grad(loss, leaves))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    for k in range(3):
        with torch.no_grad():
            leaves[0].copy_(h * (k + 1) / 2)
        t.copy_(t.roll(1))
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = call()
        for _, out in graphs:
            assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_results_repeat():
    runs = [check(*make(515, 192, 9001, torch.float32, True, 0.2, seed=15), "mean", 4000)
            for _ in range(3)]
    for loss, grads in runs[1:]:
        assert torch.equal(loss, runs[0][0])
        assert all(torch.equal(a, c) for a, c in zip(grads, runs[0][1]))


def test_empty():
    h = torch.empty(0, 16, device="cuda", requires_grad=True)
    w = torch.randn(30, 16, device="cuda", requires_grad=True)
    t = torch.empty(0, dtype=torch.int64, device="cuda")
    assert torch.isnan(linear_cross_entropy(h, w, t))
    total = linear_cross_entropy(h, w, t, reduction="sum")
    total.backward()
    assert total == 0 and (w.grad == 0).all()
    assert linear_cross_entropy(h, w, t, reduction="none").shape == (0,)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ignored_rows_do_not_set_the_scale(dtype):
    """Values far above the rest in rows that take no part: the others' results keep every bit."""
    h, w, b, t = make(300, 96, 700, dtype, True, 0.4, seed=23)
    zeroed = torch.where((t == -100)[:, None], torch.zeros_like(h), h)
    huge = torch.full_like(h, 6e4 if dtype == torch.float16 else 1e30)
    dirty = torch.where((t == -100)[:, None], huge, h)
    base, other = check(zeroed, w, b, t, "mean"), check(dirty, w, b, t, "mean")
    assert torch.equal(base[0], other[0])
    assert all(torch.equal(x, y) for x, y in zip(base[1], other[1]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [9, 60, 300])
def test_rows_that_are_not_finite_leave_the_others(tokens, dtype):
    h, w, _, t = make(tokens, 96, 700, dtype, False, 0, seed=24)
    h[1], h[4] = 0.0, 0.0
    g = torch.randn(tokens, device="cuda")
    got = []
    for value in (0.0, float("inf"), float("nan")):
        leaf = h.clone()
        leaf[1], leaf[4, 5] = value, value
        leaf.requires_grad_()
        loss = linear_cross_entropy(leaf, w, t, reduction="none")
        got.append((loss.detach(), torch.autograd.grad(loss, leaf, g)[0]))
    rest = torch.ones(tokens, dtype=torch.bool, device="cuda")
    rest[1] = rest[4] = False
    assert torch.isfinite(got[0][0]).all()
    for loss, grad in got[1:]:
        assert torch.isnan(loss[~rest]).all() and torch.isnan(grad[~rest]).all()
        assert torch.equal(loss[rest], got[0][0][rest]) and torch.equal(grad[rest], got[0][1][rest])


@pytest.mark.parametrize("tokens,dim,vocab,ignored,piece", [
    (17, 32, 33, 0, 0), (100, 96, 4097, 0.3, 1000), (128, 160, 700, 0.1, 0), (129, 160, 700, 0.1, 0),
    (64, 1024, 515, 0, 0), (90, 36, 517, 0, 0)])
def test_float32_around_the_raw_products(tokens, dim, vocab, ignored, piece):
    """Both sides of 128 tokens and of whole 128-byte rows."""
    h, w, b, t = make(tokens, dim, vocab, torch.float32, True, ignored, seed=vocab)
    check(h, w, b, t, "mean", piece)
    wide = torch.randn(vocab, dim + 8, device="cuda")
    for at in (4, 3):  # 16-byte rows, and not
        wide[:, at:at + dim] = w
        check(h, wide[:, at:at + dim], b, t, "none", piece)


@pytest.mark.parametrize("tokens,dim,vocab,dtype", [
    (1, 64, 300, torch.bfloat16), (16, 2048, 700, torch.float32), (64, 128, 5000, torch.float32),
    (200, 100, 900, torch.float32)])
def test_graph_replays_of_few_tokens(tokens, dim, vocab, dtype):
    """The forms for few tokens (128 KiB of LDS among them) under capture, two graphs, replayed in turn."""
    h, w, b, t = make(tokens, dim, vocab, dtype, True, 0, seed=25)
    leaves = [x.detach().clone().requires_grad_() for x in (h, w, b)]

    def call():
        loss = linear_cross_entropy(leaves[0], leaves[1], t, leaves[2])
        return (loss.detach(), *torch.autograd.grad(loss, leaves))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    for k in range(3):
        with torch.no_grad():
            leaves[0].copy_(h * (k + 1) / 2)
        t.copy_((t + 1) % vocab)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = call()
        for _, out in graphs:
            assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_backward_twice_and_two_calls_at_once():
    h, w, b, t = make(200, 64, 900, torch.float32, True, 0.2, seed=26)
    leaves = [x.detach().requires_grad_() for x in (h, w, b)]
    one = linear_cross_entropy(leaves[0], leaves[1], t, leaves[2])
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        two = linear_cross_entropy(leaves[0] * 2, leaves[1], t, leaves[2])
        late = torch.autograd.grad(two, leaves[1], retain_graph=True)[0]
    first = torch.autograd.grad(one, leaves, retain_graph=True)
    again = torch.autograd.grad(one, leaves)
    assert all(torch.equal(x, y) for x, y in zip(first, again))
    torch.cuda.current_stream().wait_stream(other)
    alone = linear_cross_entropy(leaves[0] * 2, leaves[1], t, leaves[2])
    assert torch.equal(late, torch.autograd.grad(alone, leaves[1])[0])


class HookError(Exception):
    pass


@pytest.mark.parametrize("binding", [True, False])
@pytest.mark.parametrize("tokens", [8, 60, 200])
def test_saved_tensor_hooks(tokens, binding, monkeypatch):
    """Saved tensors that come back elsewhere (other strides and alignment than the forward saw), and a
    hook's own error."""
    from smart_compress_amd import _native as N
    if not binding:
        monkeypatch.setattr(N, "train_fast", lambda: None)
    h, w, b, t = make(tokens, 64, 500, torch.float32, True, 0.2, seed=27)
    wide = torch.randn(500, 70, device="cuda")
    wide[:, 3:67] = w
    leaves = [x.detach().requires_grad_() for x in (h, wide[:, 3:67], b)]
    with torch.autograd.graph.save_on_cpu():
        loss = linear_cross_entropy(leaves[0], leaves[1], t, leaves[2])
    grad = torch.tensor(-1.7, device="cuda")
    got = torch.autograd.grad(loss, leaves, grad)
    want, bl, grads, bounds = reference(h, w, b, t, "mean", grad)
    close(loss, want, bl, torch.float32)
    for x, e, bound in zip(got, grads, bounds):
        close(x, e, bound, torch.float32)

    def refuse(_):
        raise HookError("no")

    with torch.autograd.graph.saved_tensors_hooks(refuse, lambda x: x), pytest.raises(HookError):
        linear_cross_entropy(leaves[0], leaves[1], t, leaves[2])


GATHERED = (520, 704, 100003)  # long enough for the rows that take part to be gathered


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ignored,reduction,piece", [(0.5, "mean", 0), (0.1, "none", 40000), (0, "sum", 0)])
def test_gathered_rows(ignored, reduction, piece, dtype):
    h, w, b, t = make(*GATHERED, dtype, True, ignored, seed=28)
    h = torch.where((t == -100)[:, None], torch.full_like(h, float("nan")), h)
    check(h, w, b, t, reduction, piece)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kept", [0, 1, 63, 64, 65, 257])
def test_few_gathered_rows(kept, dtype):
    h, w, b, t = make(*GATHERED, dtype, True, 0, seed=29)
    t[torch.randperm(len(t), device="cuda")[kept:]] = -100
    if kept:
        check(h, w, b, t, "sum")
    else:
        leaves = [x.requires_grad_() for x in (h, w, b)]
        loss = linear_cross_entropy(h, w, t, b, reduction="none")
        assert (loss == 0).all()
        for x in torch.autograd.grad(loss.sum(), leaves):
            assert (x == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_graph_replays_with_other_ignored_rows(dtype):
    h, w, b, t = make(*GATHERED, dtype, True, 0, seed=30)
    leaves = [x.detach().clone().requires_grad_() for x in (h, w, b)]

    def call():
        loss = linear_cross_entropy(leaves[0], leaves[1], t, leaves[2])
        return (loss.detach(), *torch.autograd.grad(loss, leaves))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for k in range(4):
        t[:: k + 2] = -100
        t[1:: k + 3] = k
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, call()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,dim", [(16, 2368), (16, 2369), (13, 2542), (9, 4209), (5, 7577), (3, 12629),
                                        (1, 37888), (1, 37889)])
def test_few_tokens_to_the_last_of_the_lds(tokens, dim, dtype):
    # (a single row takes part: the mean over none is NaN)
    check(*make(tokens, dim, 77, dtype, True, 0.2 if tokens > 1 else 0, seed=tokens), "mean")


@pytest.mark.parametrize("power", [16, 24, 40])
@pytest.mark.parametrize("tokens,dim,vocab,ignored", [(9, 64, 500, 0), (60, 36, 500, 0.2), (100, 64, 500, 0),
                                                      (200, 100, 900, 0), (*GATHERED, 0.5)])
def test_a_large_row_leaves_the_others_losses(tokens, dim, vocab, ignored, power):
    """One finite row of hidden, or of the weight (masked by its bias), far above the rest: float32 losses of
    the other rows keep every bit, at every number of tokens."""
    h, w, b, t = make(tokens, dim, vocab, torch.float32, True, ignored, seed=31)
    b[7], t[t == 7], t[3] = float("-inf"), 8, 5
    rest = torch.arange(tokens, device="cuda") != 3
    base = linear_cross_entropy(h, w, t, b, reduction="none")
    want, bl, _, _ = reference(h, w, b.clamp(min=-1e30), t, "none", torch.ones(tokens, device="cuda"))
    large_h, large_w = h.clone(), w.clone()
    large_h[3] *= 2.0 ** power
    large_w[7] *= 2.0 ** power
    assert torch.equal(linear_cross_entropy(large_h, w, t, b, reduction="none")[rest], base[rest])
    assert torch.equal(linear_cross_entropy(h, large_w, t, b, reduction="none"), base)
    assert torch.isfinite(base).all()


SPREAD = [(9, 64, 500, 0), (60, 36, 500, 0.2), (100, 64, 500, 0), (200, 100, 900, 0), (*GATHERED, 0.5)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,dim,vocab,ignored", SPREAD)
def test_a_large_gradient_leaves_the_others(tokens, dim, vocab, ignored, dtype):
    """One finite gradient of a loss, or one finite row of hidden, far above the rest: the other rows of
    hidden's gradient keep every bit."""
    h, w, b, t = make(tokens, dim, vocab, dtype, True, ignored, seed=32)
    t[3] = 5
    rest = torch.arange(tokens, device="cuda") != 3
    g = torch.randn(tokens, device="cuda")

    def run(h, g):
        leaf = h.detach().requires_grad_()
        return torch.autograd.grad(linear_cross_entropy(leaf, w, t, b, reduction="none"), leaf, g)[0]

    base = run(h, g)
    assert (base[rest & (t != -100)] != 0).any(1).all()
    large = g.clone()
    for power in (24, 40, -40):
        large[3] = 2.0 ** power
        assert torch.equal(run(h, large)[rest], base[rest])
    if dtype != torch.float16:
        for power in (24, 40):
            spread = h.clone()
            spread[3] *= 2.0 ** power
            assert torch.equal(run(spread, g)[rest], base[rest])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("power", [24, 40])
@pytest.mark.parametrize("tokens,dim,vocab,ignored", SPREAD)
def test_the_weights_gradient_beside_large_rows(tokens, dim, vocab, ignored, power, dtype):
    """Rows of hidden 2^k above the others, each sure of one entry: the weight's and the bias' gradients of
    the other entries are those of the small rows alone. The operands of such a sum share k, which leaves them
    2^(k / 2 - 38) of a row's largest product and more."""
    h, w, b, t = make(tokens, dim, vocab, dtype, True, ignored, seed=33)
    t[::50] = 5
    large = torch.zeros(tokens, dtype=torch.bool, device="cuda")
    large[::50] = True
    h[large] *= 2.0 ** power
    g = torch.randn(tokens, device="cuda")
    leaves = [x.detach().requires_grad_() for x in (h, w, b)]
    loss = linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], reduction="none")
    dw, db = torch.autograd.grad(loss, leaves[1:], g)
    others = torch.ones(vocab, dtype=torch.bool, device="cuda")
    others[5] = False
    others[(h[large].double() @ w.double().t() + b.double()).argmax(1)] = False
    small = ~large
    _, _, want, bounds = reference(h[small], w, b, t[small], "none", g[small])
    size = (g.abs() * h.abs().amax(1) * (t != -100))[small].double().sum() * 2.0 ** ((power + 4) / 2 - 37)
    close(dw[others], want[1][others], bounds[1][others] + size, dtype)
    close(db[others], want[2][others], bounds[2][others], torch.float32)


@pytest.mark.parametrize("power", [24, 40])
@pytest.mark.parametrize("tokens,dim,vocab,ignored", SPREAD)
def test_hiddens_gradient_beside_a_large_entry(tokens, dim, vocab, ignored, power):
    """An entry of the weight 2^k above the others, masked by its bias: float32 gradients of hidden are those of
    the other entries alone, whose factors in the sum share k: every term is off by 2^(k / 2 - 38) of its largest
    at most, and they add up as a random walk."""
    h, w, b, t = make(tokens, dim, vocab, torch.float32, True, ignored, seed=34)
    t = torch.where(t == -100, t, t % (vocab - 1))
    b[-1] = float("-inf")
    g = torch.randn(tokens, device="cuda")
    large = w.clone()
    large[-1] *= 2.0 ** power
    leaves = [h.requires_grad_(), b.requires_grad_()]
    loss = linear_cross_entropy(h, large, t, b, reduction="none")
    dh, db = torch.autograd.grad(loss, leaves, g)
    _, _, want, bounds = reference(h.detach(), w[:-1], b.detach()[:-1], t, "none", g)
    size = (g.abs() * (t != -100))[:, None].double() * w[:-1].abs().max() * 2.0 ** ((power + 4) / 2 - 37)
    close(dh, want[0], bounds[0] + size * min(vocab, 8 * vocab ** 0.5), torch.float32)
    close(db[:-1], want[2], bounds[2], torch.float32)
    assert db[-1] == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,dim,vocab,ignored", SPREAD)
def test_bad_targets_under_a_zero_gradient(tokens, dim, vocab, ignored, dtype):
    """A target outside the vocabulary makes its row's gradient NaN, and what sums over the rows, whatever the
    gradient of its loss: 0 times NaN."""
    h, w, b, t = make(tokens, dim, vocab, dtype, True, ignored, seed=35)
    t[3], t[5] = vocab, -7
    g = torch.ones(tokens, device="cuda")
    g[3] = 0.0
    leaves = [x.detach().requires_grad_() for x in (h, w, b)]
    loss = linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], reduction="none")
    dh, dw, db = torch.autograd.grad(loss, leaves, g)
    bad = torch.zeros(tokens, dtype=torch.bool, device="cuda")
    bad[3] = bad[5] = True
    assert torch.equal(torch.isnan(loss), bad)
    assert torch.isnan(dh[bad]).all() and torch.isfinite(dh[~bad]).all()
    assert torch.isnan(dw).all() and torch.isnan(db).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,dim,vocab", [(9, 64, 400), (70, 36, 400), (70, 64, 400), (200, 64, 400), GATHERED])
def test_ignored_rows_change_no_bit(tokens, dim, vocab, dtype):
    """NaN, infinities and zeros in ignored rows: the loss and all gradients are those of the clean call."""
    h, w, b, t = make(tokens, dim, vocab, dtype, True, 0.4, seed=36)
    rows = torch.nonzero(t == -100).view(-1)
    assert len(rows) > 2
    dirty = h.clone()
    dirty[rows[0]], dirty[rows[1]], dirty[rows[2:]] = float("nan"), float("inf"), 0.0
    got = []
    for x in (h, dirty):
        leaves = [y.detach().requires_grad_() for y in (x, w, b)]
        loss = linear_cross_entropy(leaves[0], leaves[1], t, leaves[2])
        got.append((loss, *torch.autograd.grad(loss, leaves, torch.tensor(-1.7, device="cuda"))))
    assert all(torch.equal(x, y) for x, y in zip(*got))
    assert (got[1][1][rows] == 0).all() and torch.isfinite(got[1][0])


@pytest.mark.parametrize("tokens,dim,vocab", [(100, 64, 500), (60, 36, 500), (200, 100, 900)])
def test_small_probabilities_of_small_rows(tokens, dim, vocab):
    """Rows of hidden some 2^-13 of a few large ones, which are sure of one entry, under a bias that makes most
    entries improbable (to 2^-23): the weight's gradient keeps 2^-38 of a probability in float32, as where all
    rows are of one size."""
    h, w, b, t = make(tokens, dim, vocab, torch.float32, True, 0, seed=37)
    b[:] = torch.linspace(0, -16, vocab, device="cuda")
    t %= 20
    t[::50] = 5
    large = torch.zeros(tokens, dtype=torch.bool, device="cuda")
    large[::50] = True
    h[~large] *= 2.0 ** -6
    h[large] = 400.0 * w[5] / w[5].norm() ** 2
    g = torch.randn(tokens, device="cuda")
    leaf = w.detach().requires_grad_()
    dw = torch.autograd.grad(linear_cross_entropy(h, leaf, t, b, reduction="none"), leaf, g)[0]
    _, _, want, bounds = reference(h[~large], w, b, t[~large], "none", g[~large])
    p = torch.softmax(h[large].double() @ w.double().t() + b.double(), 1)
    others = torch.arange(20, vocab, device="cuda")
    assert (p[:, others] < 2.0 ** -100).all()
    close(dw[others], want[1][others], bounds[1][others], torch.float32)
