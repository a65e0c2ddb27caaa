"""Orthogonalised updates: Newton-Schulz products and the Muon optimizer.

``orthogonalize(update)`` replaces a matrix by a nearly orthogonal one with the same singular vectors
(libsmq ``smq_orthogonalize``, csrc/orthogonalize.hip). ``Muon`` steps matrix parameters along the
orthogonalised momentum; it keeps one momentum per parameter (``momentum_buffer``, as SGD does), which
``OptimLP`` quantises like SGD's when it wraps this optimizer. Parameters that are not matrices
(biases, norms) belong in another optimizer.
"""

import ctypes
from typing import Dict, List, Sequence, Tuple

import torch
from torch.optim import Optimizer

from ... import _native as N

__all__ = ["Muon", "orthogonalize"]

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STACK_BYTES = 1 << 30  # workspace of one of Muon's calls: a few matrices of 4096 x 4096 fill the chip


def _stack_of(dtype: torch.dtype, rows: int, cols: int) -> int:
    """How many matrices of this shape go into one call."""
    if rows == 0 or cols == 0:
        return 1 << 30
    each = N.lib().smq_orthogonalize_workspace_bytes(N.DTYPE_CODES[dtype], 1, rows, cols)
    if each == 0:
        N.check(-1, "Muon")
    return max(1, STACK_BYTES // each)


def orthogonalize(update: torch.Tensor, steps: int = 5,
                  coefficients: Sequence[float] = COEFFICIENTS, eps: float = 1e-7) -> torch.Tensor:
    """``steps`` times ``A = X X^T; X = a X + (b A + c A A) X`` from ``X = update / (norm + eps)``,
    for a matrix [rows, cols] or a stack [batch, rows, cols] of them (float32, float16 or bfloat16,
    any strides, on a ROCm device); the result has the update's shape and dtype, contiguous. A matrix
    with more rows than columns is worked on transposed. Accuracy: float32-class in every type, then
    rounded to it. ``coefficients`` have to keep singular values that start at or below 1 bounded
    (below 256). Not differentiable."""
    who = "orthogonalize"
    N.require_device(update, who)
    if update.dtype not in N.DTYPE_CODES:
        raise TypeError(f"{who}: dtype {update.dtype} is not float32, float16 or bfloat16")
    if update.dim() not in (2, 3):
        raise ValueError(f"{who}: [rows, cols] or [batch, rows, cols] expected, got "
                         f"{tuple(update.shape)}")
    if len(coefficients) != 3:
        raise ValueError(f"{who}: three coefficients expected, got {len(coefficients)}")
    x = update.detach()
    if x.numel() == 0:
        return torch.empty(x.shape, dtype=x.dtype, device=x.device)
    fast = N.train_fast()
    if fast is not None:
        return fast.orthogonalize(x, steps, *map(float, coefficients), float(eps))
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    x = x if x.dim() == 3 else x.unsqueeze(0)
    batch, rows, cols = x.shape
    if (cols > 1 and x.stride(2) != 1) or (rows > 1 and x.stride(1) < cols):
        x = x.contiguous()
    ld = max(x.stride(1), cols) if rows > 1 else cols
    with N.on_device(x.device):
        lib = N.lib()
        code = N.DTYPE_CODES[x.dtype]
        need = lib.smq_orthogonalize_workspace_bytes(code, batch, rows, cols)
        if need == 0:
            N.check(-1, who)
        ws = N.call_workspace(need, x.device)
        N.check(lib.smq_orthogonalize(
            x.data_ptr(), ld, x.stride(0), code, out.data_ptr(), batch, rows, cols, steps,
            (ctypes.c_double * 3)(*coefficients), eps, ws.data_ptr(), need,
            N.stream_ptr(x.device)), who)
    return out


class Muon(Optimizer):
    """Momentum, orthogonalised: ``m <- momentum m + (1 - momentum) g``, the update is ``m`` or, with
    ``nesterov``, ``momentum m + (1 - momentum) g``, and ``p <- (1 - lr weight_decay) p
    - lr sqrt(max(1, rows / cols)) orthogonalize(update)``. A parameter of more than two dimensions (a
    convolution's weight) counts as the matrix [first, rest]. Parameters of one shape are
    orthogonalised in one call, as many as 1 GiB of workspace (or one matrix) allows."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True,
                 weight_decay: float = 0.0, steps: int = 5,
                 coefficients: Sequence[float] = COEFFICIENTS, eps: float = 1e-7):
        if lr < 0.0 or weight_decay < 0.0 or not 0.0 <= momentum < 1.0:
            raise ValueError(f"Muon: lr {lr}, momentum {momentum}, weight_decay {weight_decay}: "
                             "lr and weight_decay >= 0 and 0 <= momentum < 1 expected")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov,
                                      weight_decay=weight_decay, steps=steps,
                                      coefficients=tuple(coefficients), eps=eps))

    def add_param_group(self, group):
        super().add_param_group(group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() < 2 or p.dtype not in N.DTYPE_CODES:
                self.param_groups.pop()
                what = "not a matrix" if p.dim() < 2 else "not float32, float16 or bfloat16"
                raise ValueError(f"Muon: a parameter of shape {tuple(p.shape)} and dtype {p.dtype} is "
                                 f"{what}; give it to another optimizer")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            stacks: Dict[Tuple, List[torch.Tensor]] = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("Muon: sparse gradients are not supported")
                stacks.setdefault((p.shape, p.dtype, p.device), []).append(p)
            for (shape, dtype, _), ps in stacks.items():
                rows = shape[0]
                most = _stack_of(dtype, rows, shape.numel() // max(rows, 1))
                for k in range(0, len(ps), most):
                    self._step_stack(group, ps[k:k + most])
        return loss

    def _step_stack(self, group, ps: List[torch.Tensor]):
        momentum = group["momentum"]
        updates = [p.grad for p in ps]
        if momentum:
            for p in ps:
                if "momentum_buffer" not in self.state[p]:
                    self.state[p]["momentum_buffer"] = torch.zeros_like(p)
            buffers = [self.state[p]["momentum_buffer"] for p in ps]
            torch._foreach_lerp_(buffers, updates, 1.0 - momentum)
            updates = torch._foreach_lerp(updates, buffers, momentum) if group["nesterov"] else buffers
        rows = ps[0].shape[0]
        cols = ps[0].numel() // max(rows, 1)
        flat = [u.reshape(rows, cols) for u in updates]
        x = torch.stack(flat) if len(flat) > 1 else flat[0].unsqueeze(0)
        o = orthogonalize(x, group["steps"], group["coefficients"], group["eps"])
        scale = max(1.0, rows / max(cols, 1)) ** 0.5
        if group["weight_decay"]:
            torch._foreach_mul_(ps, 1.0 - group["lr"] * group["weight_decay"])
        torch._foreach_add_(ps, [o[i].view(p.shape) for i, p in enumerate(ps)],
                            alpha=-group["lr"] * scale)
