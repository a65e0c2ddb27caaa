"""Group norm with an activation on channels-last tensors, forward and backward.

``group_norm_act(x, groups, weight, bias)`` is ``act(F.group_norm(x, groups, weight, bias))`` in one
operator (libsmq ``smq_group_norm_act`` / ``_backward``, csrc/group_norm.hip). Autograd keeps ``x``
and two floats per (sample, group): neither the normalised tensor nor the activation's input, which
the backward computes again; under ``PackedActivations`` an ``x`` that came out of a codec is held as
its packed stream. ``GroupNormAct`` takes the place of a batch norm (or ``nn.GroupNorm``) and the
activation behind it; the compression callers treat it as the normalisation layer it is.
"""

from typing import Optional

import torch
from torch import nn
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from ... import _native as N

__all__ = ["GroupNormAct", "group_norm_act"]

_ACTIVATIONS = {"none": N.SMQ_ACT_NONE, "relu": N.SMQ_ACT_RELU, "silu": N.SMQ_ACT_SILU,
                "gelu": N.SMQ_ACT_GELU}


def _channels_last(t: torch.Tensor) -> torch.Tensor:
    """The tensor as contiguous [n, *positions, channels] (a copy where its memory is not)."""
    return t.movedim(1, -1).contiguous()


def _channels_last_like(x: torch.Tensor) -> torch.Tensor:
    """A new tensor of x's shape in channels-last memory. No view: autograd refuses to change a view that
    a custom function returns in place, and what follows a normalisation often does (out += identity)."""
    strides, step = [0] * x.dim(), x.shape[1]
    strides[1] = 1
    for d in range(x.dim() - 1, 1, -1):
        strides[d] = step
        step *= x.shape[d]
    strides[0] = step
    return torch.empty_strided(x.shape, strides, dtype=x.dtype, device=x.device)


def _float_ptr(t: Optional[torch.Tensor]):
    """The parameter as contiguous fp32 and its address (the tensor has to outlive the launch)."""
    if t is None:
        return None, None
    t = t.detach().float().contiguous()
    return t, t.data_ptr()


class _GroupNormAct(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, activation):
        xl = _channels_last(x)
        n, c = xl.shape[0], xl.shape[-1]
        s = xl.numel() // (n * c)
        dev = x.device
        y = _channels_last_like(x)
        stats = torch.empty(2, n, groups, dtype=torch.float32, device=dev)
        with N.on_device(dev):
            lib = N.lib()
            code = N.DTYPE_CODES[x.dtype]
            need = lib.smq_group_norm_workspace_bytes(code, n, s, c, groups, 0)
            if need == 0:
                N.check(-1, "group_norm_act")
            ws = N.call_workspace(need, dev)
            w, wp = _float_ptr(weight)
            b, bp = _float_ptr(bias)
            N.check(lib.smq_group_norm_act(
                xl.data_ptr(), code, y.data_ptr(), n, s, c, groups, wp, bp, eps, activation,
                stats.data_ptr(), stats.data_ptr() + 4 * n * groups, ws.data_ptr(), need,
                N.stream_ptr(dev)), "group_norm_act")
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.args = (groups, activation)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        groups, activation = ctx.args
        xl, dl = _channels_last(x), _channels_last(dy)
        n, c = xl.shape[0], xl.shape[-1]
        s = xl.numel() // (n * c)
        dev = x.device
        dx = _channels_last_like(x)
        need_w, need_b = ctx.needs_input_grad[1:3]
        dw = torch.empty(c, dtype=torch.float32, device=dev) if need_w else None
        db = torch.empty(c, dtype=torch.float32, device=dev) if need_b else None
        with N.on_device(dev):
            lib = N.lib()
            code = N.DTYPE_CODES[x.dtype]
            need = lib.smq_group_norm_workspace_bytes(code, n, s, c, groups, 1)
            if need == 0:
                N.check(-1, "group_norm_act backward")
            ws = N.call_workspace(need, dev)
            w, wp = _float_ptr(weight)
            b, bp = _float_ptr(bias)
            N.check(lib.smq_group_norm_act_backward(
                xl.data_ptr(), dl.data_ptr(), code, dx.data_ptr(), n, s, c, groups, wp, bp,
                activation, stats.data_ptr(), stats.data_ptr() + 4 * n * groups,
                None if dw is None else dw.data_ptr(), None if db is None else db.data_ptr(),
                ws.data_ptr(), need, N.stream_ptr(dev)), "group_norm_act backward")
        return (dx if ctx.needs_input_grad[0] else None,
                None if dw is None else dw.to(weight.dtype),
                None if db is None else db.to(bias.dtype), None, None, None)


def group_norm_act(x: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None,
                   bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
                   activation: str = "none") -> torch.Tensor:
    """``activation(group_norm(x))`` of ``x`` [n, channels, ...] (float32, float16 or bfloat16, on a
    ROCm device), with ``weight`` / ``bias`` [channels] in any of these dtypes and ``activation`` one
    of "none", "relu", "silu", "gelu" (the exact one). Channels-last memory is used as it is, other
    layouts are copied into it first; the result, of ``x``'s dtype, and ``x``'s gradient are channels
    last. Statistics and the parameters' gradients are computed in float32 or wider; a group's single
    value normalises to 0. No second derivative."""
    who = "group_norm_act"
    params = [t for t in (weight, bias) if t is not None]
    device = x.device
    for t in (x, *params):
        N.require_device(t, who)
        if t.device != device:
            raise RuntimeError(f"{who}: tensors on {device} and {t.device}")
        if t.dtype not in N.DTYPE_CODES:
            raise TypeError(f"{who}: dtype {t.dtype} is not float32, float16 or bfloat16")
    if x.dim() < 2:
        raise ValueError(f"{who}: x [n, channels, ...] expected, got {tuple(x.shape)}")
    channels = x.shape[1]
    if num_groups < 1 or channels < 1 or channels % num_groups:
        raise ValueError(f"{who}: {num_groups} groups do not divide {channels} channels")
    for t in params:
        if t.shape != (channels,):
            raise ValueError(f"{who}: a parameter has shape {tuple(t.shape)}, expected "
                             f"({channels},)")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"{who}: activation {activation!r} is not one of {sorted(_ACTIVATIONS)}")
    if not eps >= 0.0:
        raise ValueError(f"{who}: eps {eps} is negative")
    if x.numel() == 0:  # nothing to launch: an empty result that still reaches every input
        out = x.clone()
        for t in params:
            out = out + 0.0 * t.sum().to(x.dtype)
        return out
    fast = N.train_fast()
    if fast is not None:
        return fast.group_norm(x, weight, bias, int(num_groups), float(eps),
                               _ACTIVATIONS[activation])
    return _GroupNormAct.apply(x, weight, bias, int(num_groups), float(eps),
                               _ACTIVATIONS[activation])


class GroupNormAct(nn.GroupNorm):
    """``nn.GroupNorm`` (same parameters and state dict) followed by ``activation``, on
    ``group_norm_act``."""

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-5, affine: bool = True,
                 activation: str = "relu", device=None, dtype=None):
        super().__init__(num_groups, num_channels, eps, affine, device=device, dtype=dtype)
        if activation not in _ACTIVATIONS:
            raise ValueError(f"GroupNormAct: activation {activation!r} is not one of "
                             f"{sorted(_ACTIVATIONS)}")
        self.activation = activation

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return group_norm_act(x, self.num_groups, self.weight, self.bias, self.eps,
                              self.activation)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, activation={self.activation}"
