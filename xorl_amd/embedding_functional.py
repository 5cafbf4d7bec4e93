"""Embedding rows of tokens, scaled, and the gradient of a trained embedding by sorted tokens (xq_embedding_fwd / xq_embedding_bwd).

The embedding stays in bf16 (or fp32) next to packed projections (`embed_tokens` is never quantized), often as the same tensor as the output head.
Counterpart of the embedding of the reference's models.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch
from torch import Tensor

from . import _C
from ._native import native
from .functional import refuse_tangents


def _rows(t: Tensor) -> Tensor:
    t2 = t.resolve_neg().reshape(-1, t.shape[-1])
    return t2 if t2.stride(1) == 1 and (t2.shape[0] <= 1 or t2.stride(0) >= t2.shape[1]) else t2.contiguous()


def _ld(t2: Tensor) -> int:
    return t2.stride(0) if t2.shape[0] > 1 else t2.shape[1]


def _problem(ids1: Tensor, V: int, H: int, dtype: torch.dtype, scale: float, padding_idx: int) -> _C.XqEmbedding:
    q = _C.XqEmbedding()
    q.ids, q.id_bytes, q.n_tokens = ids1.data_ptr(), ids1.element_size(), ids1.numel()
    q.V, q.H, q.padding_idx, q.scale = V, H, padding_idx, scale
    q.dtype = _C.XQ_DT_F32 if dtype == torch.float32 else _C.XQ_DT_BF16
    return q


def _check(ids: Tensor, weight: Tensor) -> None:
    if weight.dtype not in (torch.bfloat16, torch.float32) or weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise _C.XqError(f"embedding: the weight [V, H] must be bf16 or fp32 and not empty, got {weight.dtype} {tuple(weight.shape)}")
    if ids.dtype not in (torch.int64, torch.int32):
        raise _C.XqError(f"embedding: ids must be int64 or int32, got {ids.dtype}")


def _one_device(ids: Tensor, other: Tensor) -> None:
    _C.require_hip(ids, other)
    if ids.device != other.device:
        raise _C.XqError(f"embedding: the tensors are on {ids.device} and {other.device}")


# (the operators can be called by themselves: what they read is checked here too)
def _fwd_impl(ids: Tensor, weight: Tensor, scale: float) -> Tensor:
    _check(ids, weight)
    _one_device(ids, weight)
    _C.check_held("embedding", ids, weight)
    dev = weight.device
    with torch.cuda.device(dev):
        i1, w2 = ids.reshape(-1).contiguous().resolve_neg(), _rows(weight)
        q = _problem(i1, w2.shape[0], w2.shape[1], weight.dtype, scale, -1)
        q.weight, q.ldw = w2.data_ptr(), _ld(w2)
        out = torch.empty((*ids.shape, weight.shape[1]), dtype=weight.dtype, device=dev)
        _C.check(_C.lib().xq_embedding_fwd(ctypes.byref(q), out.data_ptr(), q.H, _C.stream_ptr(dev)))
    return out


def _bwd_impl(grad: Tensor, ids: Tensor, V: int, scale: float, padding_idx: int) -> Tensor:
    if grad.dtype not in (torch.bfloat16, torch.float32) or grad.dim() < 1 or grad.shape[-1] < 1 or ids.dtype not in (torch.int64, torch.int32) or V < 1:
        raise _C.XqError("embedding: what the forward kept, or the gradient, is not that of this problem")
    _one_device(ids, grad)
    _C.check_held("embedding", ids, grad)
    dev = grad.device
    with torch.cuda.device(dev):
        i1, g2 = ids.reshape(-1).contiguous().resolve_neg(), _rows(grad)
        if g2.shape[0] != i1.numel():
            raise _C.XqError("embedding: what the forward kept, or the gradient, is not that of this problem")
        q = _problem(i1, V, g2.shape[1], grad.dtype, scale, padding_idx)
        dw = torch.empty(V, g2.shape[1], dtype=grad.dtype, device=dev)
        L = _C.lib()
        ws_bytes = L.xq_embedding_workspace_bytes(q.n_tokens, q.V, q.H)
        ws = torch.empty(max(ws_bytes, 0), dtype=torch.uint8, device=dev)
        _C.check(L.xq_embedding_bwd(ctypes.byref(q), g2.data_ptr(), _ld(g2), dw.data_ptr(), q.H, ws.data_ptr(), ws_bytes, _C.stream_ptr(dev)))
    return dw


@torch.library.custom_op("xq::embedding_fwd", mutates_args=(), device_types="cuda")
def _fwd_op(ids: Tensor, weight: Tensor, scale: float) -> Tensor:
    return _fwd_impl(ids, weight, scale)


@_fwd_op.register_fake
def _(ids, weight, scale):
    return weight.new_empty((*ids.shape, weight.shape[1]))


@torch.library.custom_op("xq::embedding_bwd", mutates_args=(), device_types="cuda")
def _bwd_op(grad: Tensor, ids: Tensor, V: int, scale: float, padding_idx: int) -> Tensor:
    return _bwd_impl(grad, ids, V, scale, padding_idx)


@_bwd_op.register_fake
def _(grad, ids, V, scale, padding_idx):
    return grad.new_empty((V, grad.shape[-1]))


class EmbeddingFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale: float, padding_idx: int):
        ctx.save_for_backward(ids)
        ctx.args = (weight.shape[0], scale, padding_idx)
        ctx.dtype = weight.dtype
        return (_fwd_op if torch.compiler.is_compiling() else _fwd_impl)(ids, weight, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        if not torch.compiler.is_compiling() and torch.cuda.is_current_stream_capturing():
            # (torch may hand the gradients to another stream, which ends the process under capture; the native node looks at whose)
            raise RuntimeError("embedding: a captured backward takes plain tensors, no subclasses of them")
        ids, = ctx.saved_tensors
        return None, (_bwd_op if torch.compiler.is_compiling() else _bwd_impl)(grad.to(ctx.dtype), ids, *ctx.args), None, None


def embedding(ids: Tensor, weight: Tensor, *, scale: float = 1.0, padding_idx: Optional[int] = None) -> Tensor:
    """``scale * weight[ids]``: ids [..] int64 or int32, weight [V, H] bf16 or fp32, rounded once to the weight's type.  An id outside [0, V) gives a row of NaN
    (torch's ends the process) and no gradient.

    The weight's gradient comes whole, in the weight's type: tokens are sorted by their id and each row's gradients are added in fp32, in an order that the
    ids alone fix (the same bits on every call), then scaled and rounded once.  Row ``padding_idx`` (negative ones count from the end) gets none.  First derivatives
    only.  Under graph capture forward and backward go into the same graph, and no result made outside it from the same weight may still be alive
    (refused; in a compiled call torch ends the process)."""
    if not torch.compiler.is_compiling():
        out = native().embedding(ids, weight, scale, padding_idx)
        if out is not None:
            return out
    # what the native path leaves: traced calls, tensor subclasses, and the errors
    if isinstance(scale, Tensor):
        raise _C.XqError("embedding: scale is a number, not a tensor")
    _check(ids, weight)
    V = weight.shape[0]
    if padding_idx is not None and (not -V <= padding_idx < V or (isinstance(padding_idx, float) and not padding_idx.is_integer())):
        raise _C.XqError(f"embedding: padding_idx {padding_idx} is no row of a weight of {V}")
    if not math.isfinite(scale) or abs(scale) > 3.4e38:
        raise _C.XqError(f"embedding: scale must be finite in fp32, got {scale}")
    if not torch.compiler.is_compiling():
        refuse_tangents(weight)
    _one_device(ids, weight)
    pad = -1 if padding_idx is None else int(padding_idx) % V
    if torch.is_grad_enabled() and weight.requires_grad:
        return EmbeddingFunction.apply(ids, weight, float(scale), pad)
    return (_fwd_op if torch.compiler.is_compiling() else _fwd_impl)(ids, weight.detach(), float(scale))
