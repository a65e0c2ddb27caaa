"""group_norm_act / GroupNormAct on the GPU against the formula in float64.

Tolerances. u = 2^-24. z = (x - mean) rstd w + b: the float32 mean is off by up to u |mean|, the
differences and products by u each, so z is off by at most 16 u ((|x| + |mean|) rstd |w| + |b|); the
activations' slopes are below 1.13. Sums run over at most 64 values in one register before they
are joined, so a mean of terms t is off by at most 128 u mean|t|. Results round to their type by half
a step."""

import pytest
import torch

from smart_compress_amd.util.pytorch.norm import GroupNormAct, group_norm_act

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def act64(z, name):
    if name == "relu":
        return torch.relu(z)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    return z


def reference(x, groups, w, b, eps, name, dy=None):
    """float64 result, gradients, and the bounds of their errors apart from the final rounding."""
    x = x.double().requires_grad_()
    c = x.shape[1]
    w = torch.ones(c, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(c, dtype=torch.float64, device=x.device) if b is None else b.double()
    w, b = w.clone().requires_grad_(), b.clone().requires_grad_()
    shape = (1, c) + (1,) * (x.dim() - 2)
    v = x.reshape(x.shape[0], groups, -1)
    mean = v.mean(2, keepdim=True)
    rstd = ((v - mean) ** 2).mean(2, keepdim=True).add(eps).rsqrt()
    xhat = ((v - mean) * rstd).reshape(x.shape)
    z = xhat * w.view(shape) + b.view(shape)
    y = act64(z, name)
    size = ((v.abs() + mean.abs()) * rstd).reshape(x.shape) * w.abs().view(shape) + b.abs().view(shape)
    bound = 1.13 * 16 * U * size.detach()
    if dy is None:
        return y.detach(), bound, z.detach()
    slope = torch.autograd.grad(y.sum(), z, retain_graph=True)[0]
    grads = torch.autograd.grad(y, [x, w, b], dy.double())
    dz = dy.double() * slope
    per = (x.shape[0], groups, -1)
    curve = dy.double().abs() * size.detach() * 16 * U  # |act''| <= 1 away from the kink
    t1 = (dz * w.view(shape)).abs()
    t2 = t1 * xhat.abs()
    m1 = t1.reshape(per).mean(2, keepdim=True).expand(v.shape).reshape(x.shape)
    m2 = t2.reshape(per).mean(2, keepdim=True).expand(v.shape).reshape(x.shape)
    r = rstd.expand(v.shape).reshape(x.shape)
    ratio = 1 + (mean.abs() * rstd).expand(v.shape).reshape(x.shape)
    bx = (r * ratio * (t1 + m1 + xhat.abs() * m2) * 128 * U
          + r * (curve * w.abs().view(shape) * (2 + xhat.abs()))).detach()
    dims = [d for d in range(x.dim()) if d != 1]
    wide = 128 * U * ratio
    bw = ((dz * xhat).abs() * wide + dz.abs() * wide + curve * xhat.abs()).sum(dims).detach()
    bb = (dz.abs() * wide + curve).sum(dims).detach()
    return y.detach(), bound, z.detach(), [g.detach() for g in grads], [bx, bw, bb]


def close(got, want, bound, dtype):
    step = torch.finfo(dtype).eps / 2 * want.abs() + torch.finfo(dtype).smallest_normal * \
        torch.finfo(dtype).eps
    bad = (got.double() - want).abs() - (bound + step)
    assert not torch.isnan(got).any()
    assert bad.max().item() <= 0, f"over the bound by {bad.max().item():.3g}"


def make(shape, dtype, offset=1.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, c, *sp = shape
    x = torch.randn(n, *sp, c, generator=g, device="cuda") + offset
    dy = torch.randn(n, *sp, c, generator=g, device="cuda")
    w = 1 + 0.3 * torch.randn(c, generator=g, device="cuda")
    b = 0.3 * torch.randn(c, generator=g, device="cuda")
    return x.to(dtype).movedim(-1, 1), dy.to(dtype).movedim(-1, 1), w, b


SHAPES = [((2, 64, 8, 8), 32), ((1, 1, 1, 9), 1), ((3, 84, 31, 17), 12), ((2, 320, 64, 64), 32),
          ((1, 2100, 9, 3), 1), ((2, 5000, 70, 3), 2), ((5, 33, 24, 24), 11), ((4, 32), 4),
          ((2, 48, 100), 3), ((2, 16, 4, 6, 5), 16), ((64, 8, 1, 1), 1), ((1, 64, 200, 200), 32)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_forward_and_gradients(shape, groups, dtype):
    name = ["none", "relu", "silu", "gelu"][sum(shape) % 4]
    x, dy, w, b = make(shape, dtype)
    z = reference(x, groups, w, b, 1e-5, name)[2]
    dy = torch.where(z.abs() < 1e-4, torch.zeros_like(dy), dy)  # no element on relu's kink
    want, bound, _, grads, bounds = reference(x, groups, w, b, 1e-5, name, dy)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    y = group_norm_act(leaves[0], groups, leaves[1], leaves[2], 1e-5, name)
    assert y.dtype == dtype and y.shape == x.shape
    got = torch.autograd.grad(y, leaves, dy)
    close(y, want, bound, dtype)
    for g, e, t, d in zip(got, grads, bounds, (dtype, torch.float32, torch.float32)):
        assert g.dtype == d
        close(g, e, t, d)


@pytest.mark.parametrize("name", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("affine", [(True, True), (True, False), (False, True), (False, False)])
def test_activations_and_absent_parameters(name, affine):
    x, dy, w, b = make((2, 24, 10, 10), torch.float32, seed=3)
    w, b = w if affine[0] else None, b if affine[1] else None
    z = reference(x, 6, w, b, 1e-3, name)[2]
    dy = torch.where(z.abs() < 1e-4, torch.zeros_like(dy), dy)
    want, bound, _, grads, bounds = reference(x, 6, w, b, 1e-3, name, dy)
    leaf = x.detach().requires_grad_()
    y = group_norm_act(leaf, 6, w, b, 1e-3, name)
    close(y, want, bound, torch.float32)
    close(torch.autograd.grad(y, leaf, dy)[0], grads[0], bounds[0], torch.float32)


@pytest.mark.parametrize("offset", [0.0, 100.0, 3000.0])
@pytest.mark.parametrize("shape", [(2, 32, 12, 12), (1, 32, 256, 256)])
def test_large_mean(shape, offset):
    """No cancellation: the variance of values far from zero, in either form of the kernel."""
    x, _, w, b = make(shape, torch.float32, offset, seed=5)
    want, bound, _ = reference(x, 8, w, b, 1e-5, "none")
    close(group_norm_act(x, 8, w, b), want, bound, torch.float32)


def test_constant_group_and_single_values():
    x = torch.full((2, 8, 5, 5), 3.0, device="cuda")
    b = torch.arange(8.0, device="cuda")
    torch.testing.assert_close(group_norm_act(x, 2, None, b), b.view(1, 8, 1, 1).expand_as(x),
                               rtol=0, atol=0)
    one = torch.randn(3, 4, device="cuda", requires_grad=True)
    y = group_norm_act(one, 4)  # one value a group
    assert (y == 0).all()
    assert (torch.autograd.grad(y.sum(), one)[0] == 0).all()


def test_layouts_agree_bit_for_bit():
    x, dy, w, b = make((3, 40, 9, 7), torch.float32, seed=7)
    want = group_norm_act(x, 5, w, b, activation="silu")
    pad = torch.randn(3, 9, 7, 64, device="cuda")
    pad[..., 11:51] = x.movedim(1, -1)
    for other in (x.contiguous(), pad[..., 11:51].movedim(-1, 1),
                  x.transpose(2, 3).contiguous().transpose(2, 3)):
        leaf = other.detach().requires_grad_()
        y = group_norm_act(leaf, 5, w, b, activation="silu")
        assert torch.equal(y, want)
        assert y.movedim(1, -1).is_contiguous()
        g = torch.autograd.grad(y, leaf, dy.contiguous())[0]
        ref = x.detach().requires_grad_()
        assert torch.equal(g, torch.autograd.grad(
            group_norm_act(ref, 5, w, b, activation="silu"), ref, dy)[0])


def test_expanded_gradient_and_misaligned_input():
    x, _, w, b = make((2, 16, 6, 6), torch.float16, seed=8)
    flat = torch.empty(x.numel() + 1, dtype=torch.float16, device="cuda")
    off = flat[1:].view(2, 6, 6, 16).copy_(x.movedim(1, -1)).movedim(-1, 1)
    leaf, ref = off.detach().requires_grad_(), x.detach().requires_grad_()
    ya = group_norm_act(leaf, 4, w, b, activation="gelu")
    yb = group_norm_act(ref, 4, w, b, activation="gelu")
    z = reference(x, 4, w, b, 1e-5, "gelu", torch.ones_like(x))
    close(ya, z[0], z[1], torch.float16)
    close(yb, z[0], z[1], torch.float16)
    close(torch.autograd.grad(ya.sum(), leaf)[0], z[3][0], z[4][0], torch.float16)  # expanded dy


def test_nan_stays_in_its_group():
    x, _, w, b = make((2, 16, 6, 6), torch.float32, seed=9)
    want = group_norm_act(x, 4, w, b, activation="relu")
    x = x.clone()
    x[1, 5, 2, 3] = float("nan")
    y = group_norm_act(x, 4, w, b, activation="relu")
    assert torch.isnan(y[1, 4:8]).all()
    y[1, 4:8] = want[1, 4:8]
    assert torch.equal(y, want)


def test_directional_difference():
    x, dy, w, b = make((2, 12, 7, 5), torch.float32, seed=11)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(group_norm_act(leaves[0], 3, leaves[1], leaves[2],
                                               activation="gelu"), leaves, dy)
    for leaf, grad in zip(leaves, grads):
        d = torch.randn_like(leaf)
        h = 2.0 ** -7
        args = [[t if t is not leaf else t + s * h * d for t in leaves] for s in (1, -1)]
        hi, lo = (group_norm_act(a[0], 3, a[1], a[2], activation="gelu").detach().double()
                  for a in args)
        slope = ((hi - lo) * dy.double()).sum().item() / (2 * h)
        # rounding of y (half a step each) over 2h, and h^2 / 6 of a third derivative of size <= 30
        size = (dy.double().abs().sum() * (2 * U * 4 / h + h * h / 6 * 30)).item()
        assert abs(slope - (grad.double() * d.double()).sum().item()) <= size


def test_module_matches_group_norm_module():
    m = GroupNormAct(4, 24, activation="silu", device="cuda")
    ref = torch.nn.GroupNorm(4, 24, device="cuda")
    with torch.no_grad():
        ref.weight.uniform_(0.5, 1.5)
        ref.bias.uniform_(-1, 1)
    m.load_state_dict(ref.state_dict())
    x, _, _, _ = make((2, 24, 8, 8), torch.float32, seed=12)
    want, bound, _ = reference(x, 4, ref.weight.detach(), ref.bias.detach(), 1e-5, "silu")
    close(m(x), want, bound, torch.float32)
    assert "activation=silu" in repr(m)


def test_graph_replays_and_streams():
    x, dy, w, b = make((4, 64, 40, 40), torch.bfloat16, seed=13)
    leaf = x.detach().clone(memory_format=torch.preserve_format).requires_grad_()

    def call():
        y = group_norm_act(leaf, 16, w, b, activation="silu")
        return y.detach(), torch.autograd.grad(y, leaf, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = call()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs captured on one stream share nothing
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    for k in range(3):
        with torch.no_grad():
            leaf.copy_(x * (k + 1))
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = call()
        for _, out in graphs:
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    assert torch.isfinite(eager[0].float()).all()


def test_results_repeat():
    x, dy, w, b = make((2, 256, 96, 96), torch.float32, seed=14)
    runs = []
    for _ in range(3):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = group_norm_act(leaves[0], 32, leaves[1], leaves[2], activation="relu")
        runs.append((y, *torch.autograd.grad(y, leaves, dy)))
    for other in runs[1:]:
        assert all(torch.equal(a, c) for a, c in zip(runs[0], other))


def test_empty():
    x = torch.empty(0, 8, 4, 4, device="cuda", requires_grad=True)
    w = torch.ones(8, device="cuda", requires_grad=True)
    y = group_norm_act(x, 2, w)
    assert y.shape == x.shape
    y.sum().backward()
    assert (w.grad == 0).all()


@pytest.mark.parametrize("value", [-65504.0, 1e4])
@pytest.mark.parametrize("shape", [(2, 32, 12, 12), (1, 32, 256, 256), (1, 6, 300, 211)])
def test_outlier_in_the_first_place(shape, value):
    """One value far off, where a channel's sums begin. The variance is a sum of non-negative terms of at
    most 32 values a thread and 256 threads a chunk: off by 300 u relative at most and 50 u at these sizes
    (4 + 32 values; 9 + 128 in the odd shape, of which all but a few are small against the outlier's own
    term), rstd by half of it: 25 u |z| beside the 16 u of the bound."""
    x, _, w, b = make(shape, torch.float32, seed=31)
    x[:, :, 0, 0] = value
    y = group_norm_act(x, 2, w, b)
    want, bound, _ = reference(x, 2, w, b, 1e-5, "none")
    close(y, want, 3 * bound, torch.float32)


@pytest.mark.parametrize("binding", [True, False])
@pytest.mark.parametrize("shape", [(6, 32), (2, 24, 10), (2, 32, 9, 7), (2, 16, 4, 6, 5), (2, 8, 1, 1)])
def test_result_can_be_changed_in_place(shape, binding, monkeypatch):
    """As a residual block does (out += identity, an in-place relu): same values and gradients as out of
    place, and a result in channels-last memory that is no view."""
    from smart_compress_amd import _native as N
    if not binding:
        monkeypatch.setattr(N, "train_fast", lambda: None)
    x, dy, w, b = make(shape, torch.float32, seed=41)
    got = []
    for inplace in (True, False):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = group_norm_act(leaves[0], 4, leaves[1], leaves[2])
        assert not y._is_view() and y.movedim(1, -1).is_contiguous()
        if inplace:
            y += x
            y.mul_(2.0)
            torch.nn.ReLU(inplace=True)(y)
        else:
            y = torch.relu((y + x) * 2.0)
        got.append((y.detach(), *torch.autograd.grad(y, leaves, dy)))
    assert all(torch.equal(a, c) for a, c in zip(*got))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,groups", [((65535, 8), 2), ((65536, 8), 4), ((100001, 24), 6), ((66000, 3, 5), 1),
                                          ((70000, 4, 120), 2), ((65600, 1031), 1)])
def test_more_samples_than_a_grid_has(shape, groups, dtype):
    x, dy, w, b = make(shape, dtype, seed=51)
    want, bound, _, grads, bounds = reference(x, groups, w, b, 1e-5, "silu", dy)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    y = group_norm_act(leaves[0], groups, leaves[1], leaves[2], 1e-5, "silu")
    got = torch.autograd.grad(y, leaves, dy)
    close(y, want, bound, dtype)
    for g, e, t, d in zip(got, grads, bounds, (dtype, torch.float32, torch.float32)):
        close(g, e, t, d)
    half = group_norm_act(x[-7:], groups, w, b, 1e-5, "silu")
    assert torch.equal(half, y[-7:])
