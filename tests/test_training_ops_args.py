"""What the training-step operators refuse, and the host logic of the C-ABI behind them (no GPU)."""

import ctypes

import pytest
import torch

from smart_compress_amd import _native as N
from smart_compress_amd.util.pytorch import loss as L
from smart_compress_amd.util.pytorch import norm as G
from smart_compress_amd.util.pytorch.layers import is_valid_layer_type
from smart_compress_amd.util.pytorch.muon import Muon, orthogonalize
from smart_compress_amd.util.pytorch.optimizer import OptimLP


def err():
    return N.lib().smq_last_error().decode()


def test_cpu_tensors_are_refused():
    x = torch.randn(2, 8, 3, 3)
    with pytest.raises(RuntimeError, match="ROCm device"):
        G.group_norm_act(x, 2)
    with pytest.raises(RuntimeError, match="ROCm device"):
        L.linear_cross_entropy(torch.randn(3, 4), torch.randn(5, 4), torch.zeros(3).long())
    with pytest.raises(RuntimeError, match="ROCm device"):
        orthogonalize(torch.randn(3, 4))


@pytest.fixture
def anywhere(monkeypatch):
    """Lets argument checks behind the device check be reached with CPU tensors."""
    monkeypatch.setattr(N, "require_device", lambda t, who: None)


@pytest.mark.parametrize("kw,error,match", [
    (dict(num_groups=3), ValueError, "do not divide"),
    (dict(num_groups=0), ValueError, "do not divide"),
    (dict(num_groups=2, weight=torch.ones(7)), ValueError, "parameter"),
    (dict(num_groups=2, bias=torch.ones(8, 1)), ValueError, "parameter"),
    (dict(num_groups=2, bias=torch.ones(8).double()), TypeError, "dtype"),
    (dict(num_groups=2, activation="tanh"), ValueError, "activation"),
    (dict(num_groups=2, eps=-1.0), ValueError, "eps"),
    (dict(num_groups=2, eps=float("nan")), ValueError, "eps"),
])
def test_group_norm_refusals(anywhere, kw, error, match):
    with pytest.raises(error, match=match):
        G.group_norm_act(torch.randn(2, 8, 3, 3), **kw)


def test_group_norm_refuses_types_and_shapes(anywhere):
    with pytest.raises(TypeError):
        G.group_norm_act(torch.randn(2, 8, 3, 3).double(), 2)
    with pytest.raises(ValueError):
        G.group_norm_act(torch.randn(8), 2)
    with pytest.raises(ValueError):
        G.GroupNormAct(2, 8, activation="tanh")


@pytest.mark.parametrize("args,kw,error", [
    ((torch.randn(3, 4), torch.randn(5, 6), torch.zeros(3).long()), {}, ValueError),
    ((torch.randn(3, 4), torch.randn(5, 4), torch.zeros(2).long()), {}, ValueError),
    ((torch.randn(3, 4), torch.randn(5, 4), torch.zeros(3).int()), {}, TypeError),
    ((torch.randn(3, 4), torch.randn(5, 4).half(), torch.zeros(3).long()), {}, TypeError),
    ((torch.randn(3, 4).double(), torch.randn(5, 4).double(), torch.zeros(3).long()), {}, TypeError),
    ((torch.randn(3, 4), torch.randn(0, 4), torch.zeros(3).long()), {}, ValueError),
    ((torch.randn(3, 4), torch.randn(5, 4), torch.zeros(3).long()), {"reduction": "max"}, ValueError),
    ((torch.randn(3, 4), torch.randn(5, 4), torch.zeros(3).long()), {"bias": torch.ones(4)}, ValueError),
    ((torch.randn(3, 4), torch.randn(5, 4), torch.zeros(3).long()),
     {"bias": torch.ones(5).double()}, TypeError),
    ((torch.randn(3, 4), torch.randn(5, 4), torch.zeros(3).long()), {"vocab_piece": -1}, ValueError),
])
def test_cross_entropy_refusals(anywhere, args, kw, error):
    with pytest.raises(error):
        L.linear_cross_entropy(*args, **kw)


def test_orthogonalize_refusals(anywhere):
    for bad, error in ((torch.randn(3), ValueError), (torch.randn(2, 2, 3, 3), ValueError),
                       (torch.randn(3, 3).double(), TypeError)):
        with pytest.raises(error):
            orthogonalize(bad)
    with pytest.raises(ValueError):
        orthogonalize(torch.randn(3, 3), coefficients=(1.0, 2.0))


def test_muon_refusals():
    w = torch.nn.Parameter(torch.randn(3, 4))
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            Muon([w], **kw)
    with pytest.raises(ValueError, match="not a matrix"):
        Muon([w, torch.nn.Parameter(torch.randn(3))])
    assert OptimLP(Muon([w])).momentum_keys == [("momentum_buffer", {})]


def test_modules_are_valid_layers():
    """The compression callers select them as the normalisation and the loss they are."""
    assert is_valid_layer_type(G.GroupNormAct(2, 4), ["normalization"])
    assert not is_valid_layer_type(G.GroupNormAct(2, 4), ["conv"])
    assert is_valid_layer_type(L.LinearCrossEntropy(4, 5), ["loss"])


def test_c_abi_refuses_bad_arguments():
    lib = N.lib()
    buf = (ctypes.c_char * 4096)()
    p = ctypes.addressof(buf)
    assert lib.smq_group_norm_workspace_bytes(9, 1, 1, 8, 2, 0) == 0 and "dtype" in err()
    assert lib.smq_group_norm_workspace_bytes(0, 1, 1, 8, 3, 0) == 0 and "divide" in err()
    assert lib.smq_group_norm_workspace_bytes(0, 0, 1, 8, 2, 0) == 0
    need = lib.smq_group_norm_workspace_bytes(0, 1, 4, 8, 2, 0)
    assert need > 0
    args = (p, 0, p, 1, 4, 8, 2, None, None, 1e-5)
    assert lib.smq_group_norm_act(*args, 7, p, p, p, need, None) == -1 and "activation" in err()
    assert lib.smq_group_norm_act(*args, 0, None, p, p, need, None) == -1
    assert lib.smq_group_norm_act(*args, 0, p, p, p, need - 1, None) == -2 and "workspace" in err()
    assert lib.smq_group_norm_act_backward(p, None, 0, p, 1, 4, 8, 2, None, None, 0, p, p, None,
                                           None, p, 1 << 20, None) == -1

    shape = (p, 8, p, 8, 0)
    assert lib.smq_linear_ce_workspace_bytes(*shape, 0, 8, 9, 0, 0) == 0 and "tokens" in err()
    assert lib.smq_linear_ce_workspace_bytes(p, 7, p, 8, 0, 4, 8, 9, 0, 0) == 0 and "pitch" in err()
    assert lib.smq_linear_ce_workspace_bytes(p, 8, p, 8, 5, 4, 8, 9, 0, 0) == 0
    need = lib.smq_linear_ce_workspace_bytes(*shape, 4, 8, 9, 0, 0)
    assert need > 0
    tail = (p, None, 4, 8, 9, -100)
    assert lib.smq_linear_ce_forward(*shape, *tail, 3, p, p, p, p, need, None) == -1
    assert lib.smq_linear_ce_forward(*shape, *tail, 1, None, p, p, p, need, None) == -1
    assert lib.smq_linear_ce_forward(*shape, *tail, 1, p, p, p, p, need - 1, None) == -2
    assert lib.smq_linear_ce_backward(*shape, *tail, 1, p, p, p, None, None, None, 0, p, 1 << 30,
                                      None) == -1
    assert lib.smq_linear_ce_backward(*shape, *tail, 1, p, p, p, p, None, None, -1, p, 1 << 30,
                                      None) == -1
    small = lib.smq_linear_ce_workspace_bytes(*shape, 4, 8, 9, 2, N.SMQ_CE_GRAD_HIDDEN)
    assert lib.smq_linear_ce_backward(*shape, *tail, 1, p, p, p, p, None, None, 2, p, small - 1,
                                      None) == -2

    c = (ctypes.c_double * 3)(3.4445, -4.7750, 2.0315)
    assert lib.smq_orthogonalize_workspace_bytes(0, 0, 4, 4) == 0
    assert lib.smq_orthogonalize_workspace_bytes(3, 1, 4, 4) == 0
    need = lib.smq_orthogonalize_workspace_bytes(0, 1, 4, 6)
    assert need > 0
    assert lib.smq_orthogonalize(p, 5, 24, 0, p, 1, 4, 6, 5, c, 1e-7, p, need, None) == -1
    assert lib.smq_orthogonalize(p, 6, 24, 0, p, 1, 4, 6, 0, c, 1e-7, p, need, None) == -1
    assert lib.smq_orthogonalize(p, 6, 24, 0, p, 1, 4, 6, 5, c, -1.0, p, need, None) == -1
    assert lib.smq_orthogonalize(p, 6, 24, 0, p, 1, 4, 6, 5, c, 1e-7, p, need - 1, None) == -2
    grows = (ctypes.c_double * 3)(9.0, 0.0, 0.0)
    assert lib.smq_orthogonalize(p, 6, 24, 0, p, 1, 4, 6, 5, grows, 1e-7, p, need, None) == -1
    assert "grow" in err()


def test_backward_workspace_follows_the_piece():
    lib = N.lib()
    buf = (ctypes.c_char * 64)()
    p = (ctypes.addressof(buf) + 15) & ~15
    sizes = [lib.smq_linear_ce_workspace_bytes(p, 1024, p, 1024, 2, 4096, 1024, 50000, piece, 3)
             for piece in (1024, 4096, 16384, 0)]
    assert sizes == sorted(sizes)
    full = 4096 * 50000 * 4  # one float32 copy of the logits
    assert sizes[0] < full / 8
    big = lib.smq_linear_ce_workspace_bytes(p, 4096, p, 4096, 2, 8192, 4096, 131072, 0, 3)
    assert big < 1.5 * 2 ** 30


def test_muon_keeps_no_refused_group():
    opt = Muon([torch.nn.Parameter(torch.zeros(3, 4))])
    with pytest.raises(ValueError, match="float32"):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(3, 4, dtype=torch.float64))]})
    assert len(opt.param_groups) == 1


def test_cross_entropy_limits_the_launch():
    lib = N.lib()
    one = ctypes.c_int(0)
    p = ctypes.addressof(one)
    for tokens, vocab, ok in ((1 << 18, 1 << 20, True), (1 << 19, 1 << 20, False), (1, 1 << 21, True)):
        need = lib.smq_linear_ce_workspace_bytes(p, 64, p, 64, N.SMQ_DTYPE_BF16, tokens, 64, vocab, 0, 0)
        assert (need > 0) == ok
    assert "2^38" in err()


def test_c_abi_refuses_bad_alignment():
    lib = N.lib()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 63) & ~63
    shape, tail = (p, 8, p, 8, 0), (p, None, 4, 8, 9, -100, 1)
    big = 1 << 30
    assert lib.smq_linear_ce_forward(*shape, *tail, p, p, p, p + 8, big, None) == -2 and "16-byte" in err()
    assert lib.smq_linear_ce_backward(*shape, *tail, p, p, p, p, None, None, 0, p + 4, big, None) == -2
    assert lib.smq_linear_ce_backward(*shape, *tail, p, p, p, p + 4, None, None, 0, p, big, None) == -1
    assert lib.smq_linear_ce_backward(*shape, *tail, p, p, p, None, p + 8, None, 0, p, big, None) == -1
    assert "boundaries" in err()
    gn = (p, 0, p, 1, 4, 8, 2, None, None, 1e-5, 0, p, p)
    assert lib.smq_group_norm_act(*gn, p + 4, big, None) == -2
    c = (ctypes.c_double * 3)(3.4445, -4.7750, 2.0315)
    assert lib.smq_orthogonalize(p, 6, 24, 0, p, 1, 4, 6, 5, c, 1e-7, p + 8, big, None) == -2


def test_orthogonalize_workspace_is_what_a_call_uses():
    """X and its transpose twice over as two 16-bit planes (16 bytes an element), squares of 4 bytes an element: two
    where steps are taken one by one (float32), seven in stages; and up to eight float32 shares of a product."""
    lib = N.lib()
    for code, m, n, squares in ((0, 4096, 4096, 2), (2, 4096, 4096, 7), (0, 1024, 4096, 2), (0, 64, 4096, 2)):
        shares = 0 if m == n else 8  # (a square of this size fills the chip)
        room = 16 * m * n + 4 * m * m * (squares + shares) + 64 * 16 * (m + n)  # (and the rows' padding)
        assert lib.smq_orthogonalize_workspace_bytes(code, 1, m, n) <= room


def test_muon_bounds_its_stacks(monkeypatch):
    """Parameters of one shape go in as many calls as 1 GiB of workspace each takes."""
    from smart_compress_amd.util.pytorch import muon

    calls = []
    monkeypatch.setattr(muon, "orthogonalize", lambda x, *a: (calls.append(tuple(x.shape)), x)[1])
    ps = [torch.nn.Parameter(torch.zeros(1024, 2048)) for _ in range(45)]
    ps += [torch.nn.Parameter(torch.zeros(3, 0, 5)), torch.nn.Parameter(torch.zeros(3, 4))]
    for k, p in enumerate(ps):
        p.grad = torch.full_like(p, k + 1.0)
    Muon(ps, lr=1.0, momentum=0.0).step()
    assert [c[1:] for c in calls] == [(1024, 2048)] * (len(calls) - 2) + [(3, 0), (3, 4)]
    assert sum(c[0] for c in calls[:-2]) == 45
    for batch, rows, cols in calls[:-2]:
        assert N.lib().smq_orthogonalize_workspace_bytes(0, batch, rows, cols) <= 1 << 30
    assert len(calls) - 2 <= 2
    for k, p in enumerate(ps[:45]):
        assert (p == -(k + 1.0)).all()
    big = muon._stack_of(torch.float32, 16384, 16384)
    assert big == 1


def test_cross_entropy_workspace_query_refuses_what_the_backward_does():
    lib = N.lib()
    one = ctypes.c_int(0)
    p = ctypes.addressof(one)
    for piece, flags, ok in ((0, 0, True), (0, 7, True), (1 << 20, 1, True), (-1, 1, False),
                             ((1 << 20) + 1, 1, False), (0, 8, False), (0, -1, False)):
        assert (lib.smq_linear_ce_workspace_bytes(p, 64, p, 64, 0, 4, 64, 9, piece, flags) > 0) == ok
    assert "piece" in err()
