"""orthogonalize, Muon and OptimLP(Muon) on the GPU against the recurrence in float64.

Tolerances, of the Frobenius norm. Two planes hold a value to 2^-23; a step rounds X, A and B once each
and its float32 sums add (k / 16 + 24) 2^-24, k the inner length. The relative error of a singular value
grows by at most 1.5 a step where all are of one size, and by their ratio more where they are not
(the polynomial raises small ones, and with them what the large ones left there). fp16 adds its
rounding, half a step of 2^-11 at most, bf16 its 2^-8 and, where the last two steps keep one plane of
2^-11, 16 of those."""

import copy
from argparse import Namespace

import pytest
import torch

from smart_compress_amd.util.pytorch.muon import COEFFICIENTS, Muon, orthogonalize
from smart_compress_amd.util.pytorch.optimizer import OptimLP, TaggedQuant, wrap_optimizer

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def reference(g, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    x = g.double().cpu()
    x = x.reshape(-1, *x.shape[-2:])
    turn = x.shape[1] > x.shape[2]
    x = (x.transpose(1, 2) if turn else x).contiguous()
    x = x / (x.flatten(1).norm(dim=1).view(-1, 1, 1) + eps)
    for _ in range(steps):
        gram = x @ x.transpose(1, 2)
        x = a * x + (b * gram + c * gram @ gram) @ x
    return (x.transpose(1, 2) if turn else x).reshape(g.shape)


def bound(dtype, length, ratio, steps=5):
    t = 2.0 ** -24 * steps * (6 + length / 16 + 24) * 1.5 ** (steps - 1) * ratio
    if dtype == torch.float16:
        t += 2.0 ** -11
    if dtype == torch.bfloat16:
        t += 2.0 ** -8 + 16 * 2.0 ** -11
    return t


def matrix(batch, m, n, ratio, seed=0):
    """Singular values between 1 and `ratio`, random directions."""
    g = torch.Generator().manual_seed(seed)
    k = min(m, n)
    out = []
    for _ in range(batch):
        u = torch.linalg.qr(torch.randn(m, k, generator=g, dtype=torch.float64))[0]
        v = torch.linalg.qr(torch.randn(n, k, generator=g, dtype=torch.float64))[0]
        s = ratio ** torch.rand(k, generator=g, dtype=torch.float64)
        out.append((u * s) @ v.t())
    return torch.stack(out)


def check(x, ratio, **kw):
    y = orthogonalize(x, **kw)
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
    want = reference(x, **kw)
    got = y.double().cpu()
    length = max(x.shape[-2:])
    for a, b in zip(got.reshape(-1, *x.shape[-2:]), want.reshape(-1, *x.shape[-2:])):
        err = ((a - b).norm() / b.norm()).item()
        assert err <= bound(x.dtype, length, ratio, kw.get("steps", 5)), err
    return y


SIZES = [(1, 1, 1), (1, 1, 7), (2, 5, 3), (3, 33, 64), (1, 97, 161), (2, 161, 97), (1, 64, 64),
         (1, 128, 1000), (4, 20, 700), (1, 700, 20), (1, 300, 300), (17, 31, 65), (1, 257, 513)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,m,n", SIZES)
def test_against_recurrence(batch, m, n, dtype):
    x = matrix(batch, m, n, 4.0, seed=m).to(dtype).cuda()
    check(x if batch > 1 else x[0], 4.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_spread_singular_values(dtype):
    check(matrix(2, 200, 320, 64.0, seed=3).to(dtype).cuda(), 64.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n", [(1024, 1536), (1536, 1024)])
def test_large_tiles(m, n, dtype):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(8, m, n, generator=g).to(dtype).cuda()  # ratio of a 2:3 Gaussian: about 10
    y = orthogonalize(x)
    for k in (0, 7):
        want = reference(x[k])
        err = ((y[k].double().cpu() - want).norm() / want.norm()).item()
        assert err <= bound(dtype, 1536, 10.0), err


@pytest.mark.parametrize("scale", [1e-20, 1e-3, 1e15])
def test_scale_does_not_matter(scale):
    x = matrix(1, 48, 80, 4.0, seed=7)[0].float().cuda()
    s = 2.0 ** round(torch.log2(torch.tensor(scale)).item())
    assert torch.equal(orthogonalize(x * s, eps=0.0), orthogonalize(x, eps=0.0))


def test_zero_matrix_and_eps():
    z = torch.zeros(2, 8, 12, device="cuda")
    z[1] = matrix(1, 8, 12, 2.0)[0].float().cuda()
    y = orthogonalize(z)
    assert (y[0] == 0).all() and torch.isfinite(y[1]).all()
    check(z[1], 2.0, eps=0.5)


def test_nan_stays_in_its_matrix():
    x = matrix(3, 40, 70, 2.0, seed=9).float().cuda()
    want = orthogonalize(x)
    x[1, 3, 4] = float("nan")
    y = orthogonalize(x)
    assert torch.isnan(y[1]).all()
    assert torch.equal(y[0], want[0]) and torch.equal(y[2], want[2])


def test_strides():
    x = matrix(3, 40, 70, 2.0, seed=10).float().cuda()
    want = orthogonalize(x)
    wide = torch.randn(3, 50, 90, device="cuda")
    wide[:, 5:45, 7:77] = x
    assert torch.equal(orthogonalize(wide[:, 5:45, 7:77]), want)
    assert torch.equal(orthogonalize(x.transpose(1, 2).contiguous().transpose(1, 2)), want)
    assert torch.equal(orthogonalize(x[:1].expand(3, 40, 70)), want[:1].expand(3, 40, 70))
    check(x.transpose(1, 2), 2.0)  # a transposed view


@pytest.mark.parametrize("steps,coefficients", [(1, COEFFICIENTS), (8, COEFFICIENTS),
                                                (12, (1.5, -0.5, 0.0)), (6, (1.875, -1.25, 0.375))])
def test_steps_and_coefficients(steps, coefficients):
    x = matrix(1, 40, 60, 2.0, seed=11)[0].float().cuda()
    y = check(x, 2.0, steps=steps, coefficients=coefficients)
    if steps == 12:  # this one converges to the orthogonal factor
        assert (y @ y.t() - torch.eye(40, device="cuda")).abs().max() < 1e-3


def test_graph_replays():
    x = matrix(2, 100, 300, 4.0, seed=12).to(torch.bfloat16).cuda()
    static = x.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        orthogonalize(static)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = orthogonalize(static)
        graphs.append((g, out))
    for k in range(3):
        static.copy_(x.roll(k, 2))
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = orthogonalize(static)
        assert all(torch.equal(out, want) for _, out in graphs)


def test_empty():
    assert orthogonalize(torch.empty(0, 5, device="cuda")).shape == (0, 5)
    assert orthogonalize(torch.empty(0, 4, 5, device="cuda")).shape == (0, 4, 5)


def muon_reference(ps, grads, bufs, lr, momentum, nesterov, decay):
    for p, g, m in zip(ps, grads, bufs):
        m.mul_(momentum).add_(g, alpha=1 - momentum)
        u = g * (1 - momentum) + m * momentum if nesterov else m
        flat = u.reshape(u.shape[0], -1)
        o = reference(flat.float()).reshape(p.shape)
        scale = max(1.0, flat.shape[0] / flat.shape[1]) ** 0.5
        p.mul_(1 - lr * decay).sub_(lr * scale * o)


@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_steps(nesterov):
    torch.manual_seed(0)
    shapes = [(40, 24), (40, 24), (24, 40), (16, 8, 3, 3), (16, 8, 3, 3)]
    ps = [torch.nn.Parameter(torch.randn(s, device="cuda")) for s in shapes]
    ref = [p.detach().double().cpu() for p in ps]
    bufs = [torch.zeros_like(p) for p in ref]
    opt = Muon(ps, lr=0.1, momentum=0.9, nesterov=nesterov, weight_decay=0.05)
    for _ in range(3):
        for p in ps:
            p.grad = torch.randn_like(p)
        muon_reference(ref, [p.grad.double().cpu() for p in ps], bufs, 0.1, 0.9, nesterov, 0.05)
        opt.step()
    for p, r in zip(ps, ref):
        # 3 updates of norm lr * sqrt(min) * scale each, their error as above; rounding of p
        t = 3 * 0.1 * 8 * bound(torch.float32, 72, 16.0) + 8 * 2.0 ** -24 * r.norm().item()
        assert (p.detach().double().cpu() - r).norm().item() <= t
    state = copy.deepcopy(opt.state_dict())
    again = Muon(ps, lr=0.1)
    again.load_state_dict(state)
    assert torch.equal(again.state[ps[0]]["momentum_buffer"], opt.state[ps[0]]["momentum_buffer"])


def test_muon_skips_missing_gradients_and_momentum_zero():
    a, b = (torch.nn.Parameter(torch.randn(6, 9, device="cuda")) for _ in range(2))
    keep = b.detach().clone()
    opt = Muon([a, b], lr=0.1, momentum=0.0)
    a.grad = torch.randn_like(a)
    before = a.detach().clone()
    opt.step()
    assert torch.equal(b, keep) and not opt.state[a]
    want = reference(a.grad.float())
    assert ((before - a).double().cpu() / 0.1 - want).norm() <= 1e-3


def test_optim_lp_wraps_muon():
    """OptimLP quantises weights, gradients and Muon's momentum_buffer as it does SGD's."""
    from helpers import smaq_hparams
    from smart_compress_amd.compress.smart import SmartFP

    hp = smaq_hparams()
    hp.compress_weights = hp.compress_gradients = hp.compress_momentum_vectors = True
    codec = SmartFP(hp)
    p = torch.nn.Parameter(torch.randn(32, 48, device="cuda"))
    opt = wrap_optimizer(Muon([p], lr=0.1), codec, hp)
    assert isinstance(opt, OptimLP)
    p.grad = torch.randn_like(p)
    opt.step()
    # SmaQ's 6 / 8 bits: few distinct values are left in each of the three
    for t in (p.detach(), p.grad, opt.optim.state[p]["momentum_buffer"]):
        assert t.unique().numel() < 400
    tags = []
    plain = OptimLP(Muon([p], lr=0.1), momentum_quant=lambda t, **kw: (tags.append(kw), t * 0)[1])
    plain.step()
    assert tags == [{}] and (plain.optim.state[p]["momentum_buffer"] == 0).all()
    none = OptimLP(Muon([p], lr=0.1, momentum=0.0), momentum_quant=lambda t, **kw: 1 / 0)
    none.step()


@pytest.mark.parametrize("shape", [(3, 20, 30), (2, 80, 100)])
def test_zero_matrix_with_a_tiny_eps(shape):
    """Zeros stay zeros for every eps above 0, beside matrices that are not."""
    x = torch.randn(shape, device="cuda")
    x[1] = 0.0
    y = orthogonalize(x, eps=1e-30)
    assert (y[1] == 0).all() and torch.isfinite(y).all()
    assert torch.equal(y[0], orthogonalize(x[:1], eps=1e-30)[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("steps", [5, 7, 8])
@pytest.mark.parametrize("m,n", [(32, 64), (48, 40), (64, 96)])
def test_deep_stacks_of_small_matrices(m, n, steps, dtype):
    """Far more matrices than the chip holds at once: each is what it is alone, bit for bit. The stages of a
    call change the format of the buffers that all its matrices share."""
    g = torch.Generator(device="cuda").manual_seed(steps)
    x = torch.randn(3000, m, n, generator=g, device="cuda").to(dtype)
    y = orthogonalize(x, steps=steps)
    assert torch.equal(y, orthogonalize(x.flip(0), steps=steps).flip(0))
    for k in (0, 1, 2, 255, 256, 1024, 1500, 2047, 2998, 2999):
        assert torch.equal(y[k], orthogonalize(x[k], steps=steps))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n", [(32, 512), (20, 1000), (1024, 17), (32, 480), (50, 513)])
def test_stacks_of_long_small_matrices(m, n, dtype):
    """At least 128 matrices, some with rows of whole 2 KiB as planes (which are padded)."""
    x = matrix(130, m, n, 4.0, seed=n).to(dtype).cuda()
    y = check(x, 4.0)
    assert torch.equal(y, orthogonalize(x.flip(0)).flip(0))


def tight(length):
    """Float32-class: per step six operands rounded to two planes (2^-23 each) and a sum of length / 16
    float32 roundings, all independent, each step's error growing by 1.5 in those behind it; twice that
    for the worst of a few. One fp16 plane in place of two is 1e-3 to 6e-3 off."""
    step = 2.0 ** -24 * (6 * 4 + length / 16) ** 0.5
    return 2 * step * ((1.5 ** 10 - 1) / (1.5 ** 2 - 1)) ** 0.5


def shapes():
    g = torch.Generator().manual_seed(5)
    yield "gauss", torch.randn(8, 1024, 1536, generator=g)
    yield "tall", torch.randn(1, 900, 300, generator=g)
    for ratio in (64.0, 1000.0):
        yield f"ratio{ratio:.0f}", matrix(2, 200, 320, ratio, seed=3)
    yield "small", matrix(3, 48, 80, 4.0, seed=7)
    yield "square", matrix(1, 64, 64, 64.0, seed=3)
    yield "long", matrix(2, 40, 900, 8.0, seed=8)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_16_bit_results_round_once(dtype):
    """What a result is off beyond half a step of its own type is float32-class: of a stage of three steps,
    whose powers of the Gram matrix keep less of its small singular values, four times tight(). (The
    last product in one plane of each operand, emulated: 6e-5 to 1.7e-4 of the norm beyond half a step.)"""
    for name, x in shapes():
        x = x.to(dtype)
        y = orthogonalize(x.cuda())
        for k in (0, len(x) - 1):
            want, got = reference(x[k]), y[k].double().cpu()
            bits = 11 if dtype == torch.float16 else 8
            lowest = -14 if dtype == torch.float16 else -126
            half = torch.ldexp(torch.ones_like(got), torch.frexp(got)[1].clamp(min=lowest + 1) - bits - 1)
            over = ((got - want).abs() - half).clamp(min=0).norm() / want.norm()
            print(name, k, over.item(), flush=True)
            assert over <= 4 * tight(max(x.shape[-2:])), (name, over)


def test_muon_in_several_calls(monkeypatch):
    """A stack over the workspace's budget steps as its parts do alone."""
    from smart_compress_amd.util.pytorch import muon

    g = torch.Generator(device="cuda").manual_seed(3)
    start = [torch.randn(96, 160, generator=g, device="cuda") for _ in range(7)]
    grads = [torch.randn(96, 160, generator=g, device="cuda") for _ in range(7)]
    got, real = [], orthogonalize
    for budget, whole in ((muon.STACK_BYTES, True), (3 << 20, False)):
        monkeypatch.setattr(muon, "STACK_BYTES", budget)
        ps = [torch.nn.Parameter(x.clone()) for x in start]
        opt = Muon(ps, lr=0.1, weight_decay=0.1)
        for p, x in zip(ps, grads):
            p.grad = x.clone()
        calls = []
        monkeypatch.setattr(muon, "orthogonalize", lambda x, *a: (calls.append(len(x)), real(x, *a))[1])
        opt.step()
        assert sum(calls) == 7 and (len(calls) > 1) != whole
        got.append([p.detach() for p in ps])
        if not whole:  # the same bits as the parts stepped by optimizers of their own
            at = 0
            for n in list(calls):
                qs = [torch.nn.Parameter(x.clone()) for x in start[at:at + n]]
                for q, x in zip(qs, grads[at:at + n]):
                    q.grad = x.clone()
                Muon(qs, lr=0.1, weight_decay=0.1).step()
                assert all(torch.equal(a, q.detach()) for a, q in zip(got[1][at:at + n], qs))
                at += n
    for a, c in zip(*got):
        assert (a - c).norm() <= 0.1 * 2 * tight(160) * 96 ** 0.5 + 2.0 ** -23 * c.norm()


def test_float32_is_float32_class():
    """Within tight(), twice that where singular values spread over 1000 (their small ones grow by more). One
    plane of 2^-11 in place of two would be 1e-3 to 6e-3 off, a lost cross term 1e-3 to 2e-3."""
    for name, x in shapes():
        y = orthogonalize(x.float().cuda())
        for k in (0, len(x) - 1):
            want = reference(x[k].float())
            off = ((y[k].double().cpu() - want).norm() / want.norm()).item()
            print(name, k, off, flush=True)
            assert off <= (2 if name == "ratio1000" else 1) * tight(max(x.shape[-2:])), (name, off)


def test_float32_of_a_convolution_and_an_odd_matrix():
    g = torch.Generator().manual_seed(6)
    for m, n in ((512, 4608), (97, 161)):
        low = torch.randn(m, m // 16, generator=g) @ torch.randn(m // 16, n, generator=g)
        x = (low * (m // 16) ** -0.5 + 0.5 * torch.randn(m, n, generator=g)) * 1e-3
        want = reference(x)
        off = ((orthogonalize(x.cuda()).double().cpu() - want).norm() / want.norm()).item()
        print(m, n, off, flush=True)
        assert off <= tight(n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 7, 8, 9, 13])
def test_every_number_of_steps(steps, dtype):
    """Stages of three steps end on each remainder, in the one-workgroup kernel (up to 8 steps) and in launches;
    each step past the fifth lets an error grow by 1.5 at most."""
    bits, lowest = {torch.float32: (24, -126), torch.float16: (11, -14), torch.bfloat16: (8, -126)}[dtype]
    for m, n in ((32, 64), (64, 48), (97, 161), (300, 320)):
        x = matrix(2, m, n, 4.0, seed=steps).to(dtype)
        y = orthogonalize(x.cuda(), steps=steps).double().cpu()
        want = reference(x, steps=steps)
        half = torch.ldexp(torch.ones_like(y), torch.frexp(y)[1].clamp(min=lowest + 1) - bits - 1)
        over = ((y - want).abs() - half).clamp(min=0).norm() / want.norm()
        print(m, n, over.item(), flush=True)
        assert over <= (1 if dtype == torch.float32 else 4) * tight(max(m, n)) * 1.5 ** max(0, steps - 5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,m,n", [(65535, 3, 5), (65536, 8, 6), (131075, 4, 4), (65600, 70, 66)])
def test_stacks_beyond_a_grid(batch, m, n, dtype):
    """More matrices than a grid's third dimension holds: each end of each part is what it is in a stack of its
    own part's kind."""
    g = torch.Generator(device="cuda").manual_seed(batch)
    x = torch.randn(batch, m, n, generator=g, device="cuda", dtype=torch.float32).to(dtype)
    y = orthogonalize(x)
    assert torch.isfinite(y.float()).all()
    for k in (0, 1, 65533, 65534, 65535, batch - 2, batch - 1):
        if k < batch:
            want, got = reference(x[k]), y[k].double().cpu()
            assert (got - want).norm() / want.norm() <= 8 * tight(n) + torch.finfo(dtype).eps / 2, k
