"""Softmax cross entropy of a linear head, without keeping the logits.

``linear_cross_entropy(hidden, weight, target, bias)`` is
``F.cross_entropy(F.linear(hidden, weight, bias), target)`` for a vocabulary whose logits would be
the largest activation of the step: the logits exist in registers only, the forward keeps one fp32
number a row, and the backward computes the logits again for a piece of the vocabulary at a time
(libsmq ``smq_linear_ce_forward`` / ``_backward``, csrc/linear_ce.hip). It stands next to
``PackedActivations``, which holds the activations that do have to be kept.

fp16 / bf16 inputs run on the matrix cores as they are, float32 inputs as pairs of fp16 planes with
float32-class results. Sums, the loss and the statistics are float32 or wider. The results do not
depend on timing.

Precision beyond 16 tokens (up to 16 all of it is float32). A row's loss and its gradient of ``hidden``
do not depend on how large other rows, or other rows' gradients, are. float32: an element of a row of
``hidden`` or ``weight`` is held to 2^-38 of the row's largest in the logits; in the gradients' sums
(over the entries for ``hidden``, over the rows for ``weight``) one whose row is 2^-k of the largest,
by |weight| or by |incoming gradient| |hidden|, to 2^-24 of its row's largest up to k = 30 and the
probability in front of it to 2^-38 (2^(k - 53) past k = 15); past k = 30 both to 2^(k / 2 - 38). fp16 and bf16: the logits'
gradients round to fp16 (2^-11 at most) before those sums, which are float32; bits are lost, for
``weight``, by rows of fp16 ``hidden`` whose incoming gradient is 2^-28 and less of the largest, and,
for ``hidden``, by entries of a bf16 ``weight`` 2^-30 and less of its largest element.
"""

from typing import Optional

import torch
from torch import nn
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from ... import _native as N

__all__ = ["LinearCrossEntropy", "linear_cross_entropy"]

_REDUCTIONS = {"none": N.SMQ_REDUCE_NONE, "mean": N.SMQ_REDUCE_MEAN, "sum": N.SMQ_REDUCE_SUM}


def _rows(t: torch.Tensor) -> torch.Tensor:
    """The matrix with unit column stride and rows that do not overlap (a copy where it has not)."""
    if (t.shape[1] == 1 or t.stride(1) == 1) and (t.shape[0] == 1 or t.stride(0) >= t.shape[1]):
        return t
    return t.contiguous()


def _pitch(t: torch.Tensor) -> int:
    return max(t.stride(0), t.shape[1]) if t.shape[0] > 1 else t.shape[1]


class _LinearCrossEntropy(Function):
    @staticmethod
    def forward(ctx, hidden, weight, bias, target, ignore_index, reduction, piece):
        h, w = _rows(hidden), _rows(weight)
        b = None if bias is None else bias.float().contiguous()
        target = target.contiguous()
        tokens, dim = h.shape
        vocab = w.shape[0]
        dev = h.device
        with N.on_device(dev):
            lib = N.lib()
            code = N.DTYPE_CODES[h.dtype]
            shape = (h.data_ptr(), _pitch(h), w.data_ptr(), _pitch(w), code)
            need = lib.smq_linear_ce_workspace_bytes(*shape, tokens, dim, vocab, 0, 0)
            if need == 0:
                N.check(-1, "linear_cross_entropy")
            loss = torch.empty(tokens if reduction == N.SMQ_REDUCE_NONE else (),
                               dtype=torch.float32, device=dev)
            lse = torch.empty(tokens, dtype=torch.float32, device=dev)
            head = torch.empty(N.SMQ_CE_HEAD_BYTES, dtype=torch.uint8, device=dev)
            ws = N.call_workspace(need, dev)
            N.check(lib.smq_linear_ce_forward(
                *shape, target.data_ptr(), None if b is None else b.data_ptr(), tokens, dim, vocab,
                ignore_index, reduction, loss.data_ptr(), lse.data_ptr(), head.data_ptr(),
                ws.data_ptr(), need, N.stream_ptr(dev)), "linear_cross_entropy")
        ctx.save_for_backward(hidden, weight, bias, target, lse, head)
        ctx.args = (ignore_index, reduction, piece)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        hidden, weight, bias, target, lse, head = ctx.saved_tensors
        ignore_index, reduction, piece = ctx.args
        need_h, need_w, need_b = ctx.needs_input_grad[:3]
        h, w = _rows(hidden), _rows(weight)
        b = None if bias is None else bias.float().contiguous()
        grad = grad.float().contiguous()
        tokens, dim = h.shape
        vocab = w.shape[0]
        dev = h.device
        with N.on_device(dev):
            lib = N.lib()
            shape = (h.data_ptr(), _pitch(h), w.data_ptr(), _pitch(w), N.DTYPE_CODES[h.dtype])
            flags = ((N.SMQ_CE_GRAD_HIDDEN if need_h else 0)
                     | (N.SMQ_CE_GRAD_WEIGHT if need_w else 0)
                     | (N.SMQ_CE_GRAD_BIAS if need_b else 0))
            need = lib.smq_linear_ce_workspace_bytes(*shape, tokens, dim, vocab, piece, flags)
            if need == 0:
                N.check(-1, "linear_cross_entropy backward")
            dh = torch.empty(tokens, dim, dtype=h.dtype, device=dev) if need_h else None
            dw = torch.empty(vocab, dim, dtype=w.dtype, device=dev) if need_w else None
            db = torch.empty(vocab, dtype=torch.float32, device=dev) if need_b else None
            ws = N.call_workspace(need, dev)
            ptr = [None if t is None else t.data_ptr() for t in (b, dh, dw, db)]
            N.check(lib.smq_linear_ce_backward(
                *shape, target.data_ptr(), ptr[0], tokens, dim, vocab, ignore_index, reduction,
                lse.data_ptr(), head.data_ptr(), grad.data_ptr(), *ptr[1:], piece, ws.data_ptr(),
                need, N.stream_ptr(dev)), "linear_cross_entropy backward")
        if db is not None:
            db = db.to(bias.dtype)
        return dh, dw, db, None, None, None, None


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor,
                         bias: Optional[torch.Tensor] = None, ignore_index: int = -100,
                         reduction: str = "mean", vocab_piece: int = 0) -> torch.Tensor:
    """Cross entropy of ``hidden @ weight.T + bias`` against ``target``, as float32.

    ``hidden`` [..., dim] and ``weight`` [vocab, dim] of one dtype (float32, float16 or bfloat16) on
    one ROCm device, any strides; ``target`` int64 of shape [...]; ``bias`` [vocab] of any of these
    dtypes. ``reduction``: "mean" over the targets that are not ``ignore_index`` (NaN if there are
    none, as torch), "sum", or "none" (the shape of ``target``). Ignored rows take no part, whatever
    they hold, NaN included; a target outside the vocabulary makes its loss, and what depends on it,
    NaN. Up to 2^20 tokens and 2^21 vocabulary entries, 2^38 of their products, and ``dim`` up to 2^20.
    Gradients reach ``hidden``, ``weight`` and ``bias``; there is no second derivative.
    ``vocab_piece``: vocabulary entries of one backward piece (0: what 1 GiB of buffers holds)."""
    who = "linear_cross_entropy"
    for t in (hidden, weight, target) + (() if bias is None else (bias,)):
        N.require_device(t, who)
        if t.device != hidden.device:
            raise RuntimeError(f"{who}: tensors on {hidden.device} and {t.device}")
    if hidden.dtype not in N.DTYPE_CODES or hidden.dtype != weight.dtype:
        raise TypeError(f"{who}: hidden and weight must share float32, float16 or bfloat16, got "
                        f"{hidden.dtype} and {weight.dtype}")
    if bias is not None and bias.dtype not in N.DTYPE_CODES:
        raise TypeError(f"{who}: bias dtype {bias.dtype} is not float32, float16 or bfloat16")
    if target.dtype != torch.int64:
        raise TypeError(f"{who}: target must be int64, got {target.dtype}")
    if (hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]
            or weight.numel() == 0):
        raise ValueError(f"{who}: hidden [..., dim] and weight [vocab, dim] expected, got "
                         f"{tuple(hidden.shape)} and {tuple(weight.shape)}")
    if target.shape != hidden.shape[:-1]:
        raise ValueError(f"{who}: target {tuple(target.shape)} does not match hidden "
                         f"{tuple(hidden.shape)}")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"{who}: bias {tuple(bias.shape)} does not match weight "
                         f"{tuple(weight.shape)}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"{who}: reduction {reduction!r} is not one of {sorted(_REDUCTIONS)}")
    if not 0 <= vocab_piece <= 1 << 20:
        raise ValueError(f"{who}: vocab_piece {vocab_piece} is not in [0, 2^20]")
    if target.numel() == 0:  # nothing to launch: the value and the (zero) gradients of an empty sum
        empty = hidden.float().sum(-1) + 0.0 * weight.float().sum()
        if bias is not None:
            empty = empty + 0.0 * bias.float().sum()
        return empty if reduction == "none" else getattr(empty, reduction)()
    fast = N.train_fast()
    call = _LinearCrossEntropy.apply if fast is None else fast.linear_ce
    loss = call(hidden.reshape(-1, hidden.shape[-1]), weight, bias, target.reshape(-1),
                int(ignore_index), _REDUCTIONS[reduction], int(vocab_piece))
    return loss.view(target.shape) if reduction == "none" else loss


class LinearCrossEntropy(nn.Module):
    """A linear head and its cross entropy in one module: ``forward(hidden, target)`` is the loss;
    ``weight`` [vocab, dim] and ``bias`` are those of an ``nn.Linear`` (same names, same
    initialisation), so a head's state dict loads as it is."""

    def __init__(self, dim: int, vocab: int, bias: bool = True, ignore_index: int = -100,
                 reduction: str = "mean", vocab_piece: int = 0, device=None, dtype=None):
        super().__init__()
        linear = nn.Linear(dim, vocab, bias=bias, device=device, dtype=dtype)
        self.weight, self.bias = linear.weight, linear.bias
        self.ignore_index, self.reduction, self.vocab_piece = ignore_index, reduction, vocab_piece

    def forward(self, hidden: torch.Tensor, target: torch.Tensor) -> torch.Tensor:
        return linear_cross_entropy(hidden, self.weight, target, self.bias, self.ignore_index,
                                    self.reduction, self.vocab_piece)

    def extra_repr(self) -> str:
        vocab, dim = self.weight.shape
        return f"dim={dim}, vocab={vocab}, bias={self.bias is not None}, reduction={self.reduction}"
