"""The training-step operators together, as a training program uses them: a channels-last convolution
net with GroupNormAct, a LinearCrossEntropy head, Muon for the matrices under OptimLP, and the SmaQ
codec on activations, gradient maps, gradients, weights and momenta."""

from argparse import Namespace

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from helpers import smaq_hparams
from smart_compress_amd.util.pytorch.loss import LinearCrossEntropy
from smart_compress_amd.util.pytorch.muon import Muon
from smart_compress_amd.util.pytorch.norm import GroupNormAct
from smart_compress_amd.util.pytorch.optimizer import OptimLP, wrap_optimizer

pytestmark = pytest.mark.gpu


class Net(nn.Module):
    def __init__(self, classes=50):
        super().__init__()
        self.body = nn.Sequential(
            nn.Conv2d(3, 32, 3, padding=1, bias=False), GroupNormAct(8, 32),
            nn.Conv2d(32, 48, 3, padding=1, stride=2, bias=False), GroupNormAct(8, 48, activation="silu"),
            nn.Conv2d(48, 64, 3, padding=1, bias=False), GroupNormAct(16, 64, activation="gelu"),
            nn.AdaptiveAvgPool2d(1), nn.Flatten())
        self.head = LinearCrossEntropy(64, classes)

    def forward(self, x, target):
        return self.head(self.body(x), target)


def plain(net, x, target):
    """The same net in torch's own operators and float64, on the CPU; its gradients by name."""
    params = {k: p.detach().double().cpu().requires_grad_() for k, p in net.named_parameters()}
    h = x.double().cpu()
    for i, m in enumerate(net.body):
        if isinstance(m, nn.Conv2d):
            h = F.conv2d(h, params[f"body.{i}.weight"], stride=m.stride, padding=m.padding)
        elif isinstance(m, GroupNormAct):
            h = F.group_norm(h, m.num_groups, params[f"body.{i}.weight"], params[f"body.{i}.bias"])
            h = {"relu": F.relu, "silu": F.silu, "gelu": F.gelu}[m.activation](h)
        else:
            h = m(h)
    loss = F.cross_entropy(F.linear(h, params["head.weight"], params["head.bias"]), target.cpu())
    loss.backward()
    return loss.detach(), {k: p.grad for k, p in params.items()}


def batch(seed=0, n=32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, 3, 16, 16, generator=g, device="cuda")
    return (x.contiguous(memory_format=torch.channels_last),
            torch.randint(0, 50, (n,), generator=g, device="cuda"))


def test_gradients_of_the_net():
    torch.manual_seed(1)
    net = Net().cuda().to(memory_format=torch.channels_last)
    x, t = batch()
    loss = net(x, t)
    loss.backward()
    want, grads = plain(net, x, t)
    # float32 throughout: sums of up to 32 * 256 * 9 terms through three layers, 2^-24 a step; a
    # value on relu's kink may fall on the other side, 1 of 32 * 256 * 32 with a share of the sum
    assert abs(loss.item() - want.item()) <= 1e-5 * abs(want.item())
    for k, p in net.named_parameters():
        e = grads[k]
        assert (p.grad.double().cpu() - e).norm() <= 1e-3 * e.norm(), k


def compressed_steps(packed, steps=2):
    from smart_compress_amd.compress import SmartFP, SmartFPPacked
    from smart_compress_amd.util.pytorch.autograd import register_autograd_module
    from smart_compress_amd.util.pytorch.saved import PackedActivations

    torch.manual_seed(2)
    hp = smaq_hparams()
    hp.compress_weights = hp.compress_gradients = hp.compress_momentum_vectors = True
    net = Net().cuda().to(memory_format=torch.channels_last)
    codec = (SmartFPPacked if packed else SmartFP)(hp)
    codec.rng.seed, codec.rng.offset = 5, 0
    acts = PackedActivations(codec) if packed else None
    register_autograd_module(net.body, acts if packed else codec, Namespace(
        compress_forward=True, compress_backward=True, use_batch_norm=False))
    update = SmartFP(hp)  # the optimizer's own random stream
    update.rng.seed, update.rng.offset = 6, 0
    opt = wrap_optimizer(Muon([p for p in net.parameters() if p.dim() > 1], lr=0.02), update, hp)
    assert isinstance(opt, OptimLP)
    rest = torch.optim.SGD([p for p in net.parameters() if p.dim() < 2], lr=0.02)
    out = []
    for k in range(steps):
        x, t = batch(k)
        opt.zero_grad()
        rest.zero_grad()
        if packed:
            with acts:
                loss = net(x, t)
        else:
            loss = net(x, t)
        loss.backward()
        out.append((loss.detach(), [p.grad.clone() for p in net.parameters()]))
        opt.step()
        rest.step()
        out[-1][1].extend(p.detach().clone() for p in net.parameters())
    return out, acts


def test_compressed_training_steps():
    """Steps with every codec call site on; with the saved activations held as packed streams the
    losses, gradients and weights are the same bit for bit."""
    prev = torch.backends.cudnn.deterministic, torch.backends.cudnn.benchmark
    torch.backends.cudnn.deterministic, torch.backends.cudnn.benchmark = True, False
    try:
        a, _ = compressed_steps(False)
        b, acts = compressed_steps(True)
    finally:
        torch.backends.cudnn.deterministic, torch.backends.cudnn.benchmark = prev
    for (la, ta), (lb, tb) in zip(a, b):
        assert torch.isfinite(la) and torch.equal(la, lb)
        for p, q in zip(ta, tb):
            assert torch.isfinite(p).all() and torch.equal(p, q)
    assert acts.stats()["saved_packed"] > 0


def test_python_functions_equal_the_binding(monkeypatch):
    """Without the C binding the Python autograd Functions give the same bits."""
    from smart_compress_amd import _native as N
    from smart_compress_amd.util.pytorch.loss import linear_cross_entropy
    from smart_compress_amd.util.pytorch.muon import orthogonalize
    from smart_compress_amd.util.pytorch.norm import group_norm_act

    assert N.train_fast() is not None
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(2, 24, 9, 9, generator=g, device="cuda").to(torch.bfloat16)
    w, b = (torch.randn(24, generator=g, device="cuda").half() for _ in range(2))
    h = torch.randn(50, 40, generator=g, device="cuda")
    v = torch.randn(300, 40, generator=g, device="cuda")
    c = torch.randn(300, generator=g, device="cuda").to(torch.bfloat16)
    t = torch.randint(0, 300, (50,), generator=g, device="cuda")
    wide = torch.randn(3, 30, 70, generator=g, device="cuda")[:, :, 5:45]

    def run():
        out = []
        leaves = [p.detach().requires_grad_() for p in (x, w, b)]
        y = group_norm_act(leaves[0], 6, leaves[1], leaves[2], activation="gelu")
        out += [y, *torch.autograd.grad(y.float().square().sum(), leaves)]
        leaves = [p.detach().requires_grad_() for p in (h, v, c)]
        loss = linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], reduction="none")
        out += [loss, *torch.autograd.grad(loss.square().sum(), leaves)]
        return out + [orthogonalize(wide), orthogonalize(wide[0].t())]

    want = run()
    monkeypatch.setattr(N, "_train_fast", None)
    for a, e in zip(run(), want):
        assert a.dtype == e.dtype and a.stride() == e.stride() and torch.equal(a, e)


@pytest.mark.parametrize("binding", [True, False])
def test_no_second_derivative(binding, monkeypatch):
    from smart_compress_amd import _native as N
    from smart_compress_amd.util.pytorch.loss import linear_cross_entropy
    from smart_compress_amd.util.pytorch.norm import group_norm_act

    if not binding:
        N.train_fast()
        monkeypatch.setattr(N, "_train_fast", None)
    x = torch.randn(2, 8, 4, 4, device="cuda", requires_grad=True)
    h = torch.randn(5, 8, device="cuda", requires_grad=True)
    t = torch.zeros(5, dtype=torch.int64, device="cuda")
    for out, leaf in ((group_norm_act(x, 2).sum(), x),
                      (linear_cross_entropy(h, torch.randn(9, 8, device="cuda"), t), h)):
        with pytest.raises(RuntimeError):
            grad = torch.autograd.grad(out, leaf, create_graph=True)[0]
            torch.autograd.grad(grad.sum(), leaf)


def test_autograd_keeps_only_what_is_said():
    """The loss keeps a number a row, not the logits; the norm its input and two floats a group."""
    from smart_compress_amd.util.pytorch.loss import linear_cross_entropy
    from smart_compress_amd.util.pytorch.norm import group_norm_act

    h = torch.randn(512, 64, device="cuda", requires_grad=True)
    v = torch.randn(40000, 64, device="cuda", requires_grad=True)
    t = torch.randint(0, 40000, (512,), device="cuda")
    x = torch.randn(8, 64, 32, 32, device="cuda").contiguous(
        memory_format=torch.channels_last).requires_grad_()
    torch.cuda.synchronize()
    base = torch.cuda.memory_allocated()
    loss = linear_cross_entropy(h, v, t)
    assert torch.cuda.memory_allocated() - base <= 16 * 1024
    y = group_norm_act(x, 8, activation="silu")
    assert torch.cuda.memory_allocated() - base <= 32 * 1024 + y.numel() * 4
    del loss, y
