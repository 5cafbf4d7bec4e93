"""Cross entropy over an output head, in pieces of the vocabulary, without keeping logits (xq_lce_fwd / xq_lce_bwd).

The head stays in bf16 next to packed projections (`lm_head` is never quantized); its [tokens, vocabulary] logits would be the
largest tensor of a training step by far.  Counterpart of the reference's fused linear cross entropy (ops/loss).
"""

from __future__ import annotations

import ctypes
import math
from typing import Tuple

import torch
from torch import Tensor

from . import _C
from ._native import native
from .functional import _as_2d, _ld, refuse_tangents


def _rows_of(w: Tensor) -> Tensor:
    return w if w.stride(1) == 1 and w.stride(0) % 8 == 0 and w.stride(0) >= w.shape[1] and w.data_ptr() % 16 == 0 else w.contiguous()


def _problem(x2: Tensor, w2: Tensor, labels: Tensor, ignore_index: int, reduction: int, logit_scale: float) -> _C.XqLceProblem:
    q = _C.XqLceProblem()
    q.x, q.ldx, q.w, q.ldw = x2.data_ptr(), _ld(x2), w2.data_ptr(), w2.stride(0) if w2.shape[0] > 1 else w2.shape[1]
    q.labels, q.label_bytes = labels.data_ptr(), labels.element_size()
    q.M, q.V, q.H = x2.shape[0], w2.shape[0], w2.shape[1]
    q.ignore_index, q.reduction, q.logit_scale = ignore_index, reduction, logit_scale
    return q


def _fwd_impl(x: Tensor, weight: Tensor, labels: Tensor, ignore_index: int, reduction: int, logit_scale: float, keep: int) -> Tuple[Tensor, Tensor]:
    dev = x.device
    with torch.cuda.device(dev):
        x2, w2, l1 = _as_2d(x), _rows_of(weight), labels.reshape(-1).contiguous()
        q = _problem(x2, w2, l1, ignore_index, reduction, logit_scale)
        L = _C.lib()
        loss = torch.empty(labels.shape if reduction == 0 else (), dtype=torch.float32, device=dev)
        saved = torch.empty(L.xq_lce_saved_bytes(q.M, q.V, q.H, keep), dtype=torch.uint8, device=dev)
        ws_bytes = L.xq_lce_workspace_bytes(q.M, q.V, q.H, keep)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        _C.check(L.xq_lce_fwd(ctypes.byref(q), loss.data_ptr(), saved.data_ptr(), keep, ws.data_ptr(), ws_bytes, _C.stream_ptr(dev)))
    return loss, saved


def _bwd_impl(grad: Tensor, x: Tensor, weight: Tensor, labels: Tensor, saved: Tensor, ignore_index: int, reduction: int, logit_scale: float,
              keep: int, need_dx: bool, need_dw: bool) -> Tuple[Tensor, Tensor]:
    dev = x.device
    with torch.cuda.device(dev):
        x2, w2, l1 = _as_2d(x), _rows_of(weight), labels.reshape(-1).contiguous()
        q = _problem(x2, w2, l1, ignore_index, reduction, logit_scale)
        L = _C.lib()
        g = grad.to(torch.float32).contiguous()
        if x2.shape[1] != w2.shape[1] or saved.numel() != L.xq_lce_saved_bytes(q.M, q.V, q.H, keep) or g.numel() != (q.M if reduction == 0 else 1):
            raise _C.XqError("linear_cross_entropy: what the forward kept, or the gradient, is not that of this problem")
        dx = torch.empty(x.shape if need_dx else (0,), dtype=torch.bfloat16, device=dev)
        dw = torch.empty(weight.shape if need_dw else (0,), dtype=torch.bfloat16, device=dev)
        ws_bytes = L.xq_lce_workspace_bytes(q.M, q.V, q.H, _C.XQ_LCE_KEEP_HEAD_BWD) if need_dw else 0
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        _C.check(L.xq_lce_bwd(ctypes.byref(q), g.data_ptr(), saved.data_ptr(), keep, dx.data_ptr() if need_dx else None, q.H,
                              dw.data_ptr() if need_dw else None, q.H, ws.data_ptr() if need_dw else None, ws_bytes, _C.stream_ptr(dev)))
    return dx, dw


@torch.library.custom_op("xq::lce_fwd", mutates_args=(), device_types="cuda")
def _fwd_op(x: Tensor, weight: Tensor, labels: Tensor, ignore_index: int, reduction: int, logit_scale: float, keep: int) -> Tuple[Tensor, Tensor]:
    return _fwd_impl(x, weight, labels, ignore_index, reduction, logit_scale, keep)


@_fwd_op.register_fake
def _(x, weight, labels, ignore_index, reduction, logit_scale, keep):
    M = int(x.numel() // max(x.shape[-1], 1))
    saved = _C.lib().xq_lce_saved_bytes(M, int(weight.shape[0]), int(weight.shape[1]), keep)
    return (x.new_empty(labels.shape if reduction == 0 else (), dtype=torch.float32), x.new_empty(saved, dtype=torch.uint8))


@torch.library.custom_op("xq::lce_bwd", mutates_args=(), device_types="cuda")
def _bwd_op(grad: Tensor, x: Tensor, weight: Tensor, labels: Tensor, saved: Tensor, ignore_index: int, reduction: int, logit_scale: float,
            keep: int, need_dx: bool, need_dw: bool) -> Tuple[Tensor, Tensor]:
    return _bwd_impl(grad, x, weight, labels, saved, ignore_index, reduction, logit_scale, keep, need_dx, need_dw)


@_bwd_op.register_fake
def _(grad, x, weight, labels, saved, ignore_index, reduction, logit_scale, keep, need_dx, need_dw):
    return (x.new_empty(x.shape if need_dx else (0,)), weight.new_empty(weight.shape if need_dw else (0,)))


class LinearCrossEntropyFunction(torch.autograd.Function):
    """The forward leaves the input gradient but for the upstream factor (fp32), the backward scales and rounds it.  The head's
    gradient forms the logits again, a piece of the vocabulary at a time."""

    @staticmethod
    def forward(ctx, x, weight, labels, ignore_index: int, reduction: int, logit_scale: float):
        need_dx, need_dw = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        keep = _C.XQ_LCE_KEEP_DX if need_dx else _C.XQ_LCE_KEEP_HEAD if need_dw else _C.XQ_LCE_KEEP_NONE
        fwd = _fwd_op if torch.compiler.is_compiling() else _fwd_impl
        loss, saved = fwd(x, weight, labels, ignore_index, reduction, logit_scale, keep)
        ctx.save_for_backward(x, weight, labels, saved)
        ctx.args = (ignore_index, reduction, logit_scale, keep)
        ctx.shapes = (x.shape, weight.shape)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        if not torch.compiler.is_compiling() and torch.cuda.is_current_stream_capturing():
            # (torch may hand the gradients to another stream, which ends the process under capture; the native node looks at whose)
            raise RuntimeError("linear_cross_entropy: a captured backward takes plain tensors, no subclasses of them")
        x, weight, labels, saved = ctx.saved_tensors
        if (x.shape, weight.shape) != ctx.shapes:
            raise RuntimeError("linear_cross_entropy: x or weight was resized between forward and backward")
        need_dx, need_dw = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        bwd = _bwd_op if torch.compiler.is_compiling() else _bwd_impl
        dx, dw = bwd(grad, x, weight, labels, saved, *ctx.args, need_dx, need_dw)
        return (dx if need_dx else None), (dw if need_dw else None), None, None, None, None


def linear_cross_entropy(x: Tensor, weight: Tensor, labels: Tensor, *, ignore_index: int = -100, reduction: str = "mean",
                         logit_scale: float = 1.0) -> Tensor:
    """``cross_entropy(logit_scale * x @ weight.T, labels)`` without the logits: x [.., H] and weight [V, H] in bf16, labels [..] int64 or
    int32.  Returns fp32: the mean over the rows that count (NaN if none does), their sum, or with ``reduction="none"`` the loss of every row
    (minus the label's log-probability), 0 where the label is ``ignore_index``.  Such rows get zero gradients and cost nothing.  A label outside
    [0, V) gives its row NaN, in the loss and in the gradients, the weight's with it.

    Products accumulate in fp32, sums of exponentials in fp32 relative to the label's logit or the largest.  Gradients come in bf16. For x, the
    probabilities in them are rounded to bf16 once (half a step, 2^-8, each, of the difference between the column's row of the weight and the
    label's: what all rows have in common cancels), all but the label's; for the weight, probabilities and the label's
    1 - p times the row's upstream gradient are, unless at most 128 rows count (then 2^-16).  H must be a multiple of 64.  First derivatives
    only.  Under graph capture forward and backward go into the same graph, and no loss made outside it from the same x or weight may
    still be alive (refused; in a compiled call torch ends the process).  Rows of x and weight at multiples of 16 bytes are read in place; other layouts are copied, in both passes."""
    if isinstance(logit_scale, Tensor) and logit_scale.requires_grad and torch.is_grad_enabled():
        raise _C.XqError("linear_cross_entropy: logit_scale gets no gradient; scale x by one that is trained, or detach it")
    if not torch.compiler.is_compiling() and reduction in _C.LCE_REDUCTIONS:
        loss = native().cross_entropy(x, weight, labels, ignore_index, _C.LCE_REDUCTIONS[reduction], logit_scale)
        if loss is not None:
            return loss
    # what the native path leaves: traced calls, tensor subclasses, and the errors
    if x.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise _C.XqError(f"linear_cross_entropy: x and weight must be bf16, got {x.dtype} and {weight.dtype}")
    if labels.dtype not in (torch.int64, torch.int32):
        raise _C.XqError(f"linear_cross_entropy: labels must be int64 or int32, got {labels.dtype}")
    if reduction not in _C.LCE_REDUCTIONS:
        raise _C.XqError(f"linear_cross_entropy: reduction must be one of {sorted(_C.LCE_REDUCTIONS)}, got {reduction!r}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or x.shape[:-1] != labels.shape:
        raise _C.XqError(f"linear_cross_entropy: x [.., H], weight [V, H] and labels [..] do not go together: {tuple(x.shape)}, "
                         f"{tuple(weight.shape)}, {tuple(labels.shape)}")
    if weight.shape[1] % 64 or weight.shape[0] < 1 or weight.shape[1] < 64:
        raise _C.XqError(f"linear_cross_entropy: the hidden size must be a multiple of 64 and the vocabulary not empty, got {tuple(weight.shape)}")
    if not (logit_scale > 0.0 and math.isfinite(logit_scale)):
        raise _C.XqError(f"linear_cross_entropy: logit_scale must be positive and finite, got {logit_scale}")
    if not -2 ** 63 <= int(ignore_index) < 2 ** 63:
        raise _C.XqError(f"linear_cross_entropy: ignore_index must fit 64 bits, got {ignore_index}")
    if not torch.compiler.is_compiling():
        refuse_tangents(x, weight)
    _C.require_hip(x, weight, labels)
    if weight.device != x.device or labels.device != x.device:
        raise _C.XqError(f"linear_cross_entropy: x, weight and labels are on {x.device}, {weight.device} and {labels.device}")
    code = _C.LCE_REDUCTIONS[reduction]
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        return LinearCrossEntropyFunction.apply(x, weight, labels, int(ignore_index), code, float(logit_scale))
    fwd = _fwd_op if torch.compiler.is_compiling() else _fwd_impl
    return fwd(x.detach(), weight.detach(), labels, int(ignore_index), code, float(logit_scale), _C.XQ_LCE_KEEP_NONE)[0]
