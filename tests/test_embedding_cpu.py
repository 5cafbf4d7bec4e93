"""Host side of the embedding: what embedding and the C entry points refuse before anything runs."""

import ctypes

import pytest
import torch

from xorl_amd import _C
from xorl_amd.embedding_functional import embedding


def _call(ids=None, w=None, **kw):
    return embedding(torch.zeros(3, dtype=torch.int64) if ids is None else ids, torch.zeros(10, 8) if w is None else w, **kw)


def test_cpu_tensors_raise():
    with pytest.raises(RuntimeError, match="HIP device only"):
        _call()


@pytest.mark.parametrize("kw,match", [
    (dict(ids=torch.zeros(3)), "int64 or int32"), (dict(w=torch.zeros(10, 8, dtype=torch.float16)), "bf16 or fp32"), (dict(w=torch.zeros(10)), "bf16 or fp32"),
    (dict(w=torch.zeros(0, 8)), "not empty"), (dict(w=torch.zeros(10, 0)), "not empty"), (dict(padding_idx=10), "padding_idx"), (dict(padding_idx=-11), "padding_idx"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=1e39), "scale"), (dict(scale=torch.ones(())), "scale"),
])
def test_argument_errors(kw, match):
    with pytest.raises(_C.XqError, match=match):
        _call(**kw)


def test_tangents_are_refused():
    import torch.autograd.forward_ad as fwAD

    with fwAD.dual_level(), pytest.raises(NotImplementedError, match="tangent"):
        _call(w=fwAD.make_dual(torch.zeros(10, 8), torch.ones(10, 8)))


def _problem(**over):
    # addresses that nothing reads: every call below is refused on the host
    f = dict(ids=4096, weight=4096, ldw=8, n_tokens=3, V=10, H=8, padding_idx=-1, scale=1.0, dtype=1, id_bytes=8)
    f.update(over)
    return _C.XqEmbedding(**f)


def _fwd(out=4096, ld_out=8, **over):
    return _C.lib().xq_embedding_fwd(ctypes.byref(_problem(**over)), out, ld_out, None)


def _bwd(grad=4096, ld_grad=8, dw=4096, ld_dw=8, ws=1 << 20, ws_bytes=1 << 30, **over):
    return _C.lib().xq_embedding_bwd(ctypes.byref(_problem(**over)), grad, ld_grad, dw, ld_dw, ws, ws_bytes, None)


BAD = [dict(ids=None), dict(ids=4100), dict(n_tokens=-1), dict(n_tokens=1 << 31), dict(V=0), dict(V=1 << 31), dict(H=0), dict(H=1 << 31), dict(padding_idx=10), dict(padding_idx=-2),
       dict(scale=float("inf")), dict(scale=float("nan")), dict(dtype=2), dict(id_bytes=2)]


@pytest.mark.parametrize("over", BAD + [dict(weight=None), dict(weight=4098), dict(ldw=7), dict(out=None), dict(out=4098), dict(ld_out=7)])
def test_forward_refuses(over):
    assert _fwd(**over) == -1
    assert b"xq_embedding_fwd" in _C.lib().xq_last_error()


@pytest.mark.parametrize("over", BAD + [dict(grad=None), dict(grad=4098), dict(ld_grad=7), dict(dw=None), dict(dw=4097), dict(ld_dw=7), dict(ws=None), dict(ws=8), dict(ws_bytes=0)])
def test_backward_refuses(over):
    assert _bwd(**over) == -1
    assert b"xq_embedding_bwd" in _C.lib().xq_last_error()


def test_sizes():
    L = _C.lib()
    assert ctypes.sizeof(_C.XqEmbedding) == 72
    assert L.xq_embedding_fwd(None, 4096, 8, None) == -1 and L.xq_embedding_bwd(None, 4096, 8, 4096, 8, 256, 1 << 20, None) == -1
    assert L.xq_embedding_workspace_bytes(-1, 10, 8) == -1 and L.xq_embedding_workspace_bytes(1, 0, 8) == -1 and L.xq_embedding_workspace_bytes(0, 1, 1) >= 0
    assert _fwd(n_tokens=0, ids=None, weight=None, out=None) == 0
