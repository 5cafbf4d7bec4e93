"""Host side of the cross entropy over an output head: what linear_cross_entropy and the C entry points refuse before anything runs."""

import ctypes

import pytest
import torch

from xorl_amd import _C
from xorl_amd.loss_functional import linear_cross_entropy

BF = torch.bfloat16


def _call(x=None, w=None, labels=None, **kw):
    x = torch.zeros(3, 64, dtype=BF) if x is None else x
    w = torch.zeros(10, 64, dtype=BF) if w is None else w
    labels = torch.zeros(3, dtype=torch.int64) if labels is None else labels
    return linear_cross_entropy(x, w, labels, **kw)


def test_cpu_tensors_raise():
    with pytest.raises(RuntimeError, match="HIP device only"):
        _call()


@pytest.mark.parametrize("kw,match", [
    (dict(x=torch.zeros(3, 64)), "must be bf16"), (dict(w=torch.zeros(10, 64)), "must be bf16"),
    (dict(labels=torch.zeros(3)), "int64 or int32"), (dict(labels=torch.zeros(4, dtype=torch.int64)), "do not go together"),
    (dict(x=torch.zeros(3, 128, dtype=BF)), "do not go together"), (dict(x=torch.zeros(1, 3, 64, dtype=BF)), "do not go together"),
    (dict(x=torch.zeros(3, 96, dtype=BF), w=torch.zeros(10, 96, dtype=BF)), "multiple of 64"),
    (dict(w=torch.zeros(0, 64, dtype=BF)), "not empty"), (dict(reduction="batchmean"), "reduction"),
    (dict(ignore_index=2 ** 63), "ignore_index"), (dict(logit_scale=0.0), "logit_scale"), (dict(logit_scale=float("inf")), "logit_scale"), (dict(logit_scale=float("nan")), "logit_scale"),
])
def test_argument_errors(kw, match):
    with pytest.raises(_C.XqError, match=match):
        _call(**kw)


def _problem(**over):
    # addresses that nothing reads: every call below is refused on the host
    f = dict(x=4096, ldx=64, w=8192, ldw=64, labels=12288, M=3, V=10, H=64, ignore_index=-100, logit_scale=1.0, label_bytes=8, reduction=1)
    f.update(over)
    return _C.XqLceProblem(**f)


def _fwd(loss=4096, saved=8192, keep=0, ws=1 << 20, ws_bytes=1 << 30, **over):
    return _C.lib().xq_lce_fwd(ctypes.byref(_problem(**over)), loss, saved, keep, ws, ws_bytes, None)


def _bwd(grad=4096, saved=8192, keep=2, dx=16384, lddx=64, dw=32768, lddw=64, ws=1 << 20, ws_bytes=1 << 30, **over):
    return _C.lib().xq_lce_bwd(ctypes.byref(_problem(**over)), grad, saved, keep, dx, lddx, dw, lddw, ws, ws_bytes, None)


BAD = [dict(x=None), dict(x=4098), dict(ldx=56), dict(ldx=68), dict(w=None), dict(w=8200), dict(ldw=60), dict(labels=None), dict(labels=12292),
       dict(M=-1), dict(M=1 << 30), dict(V=0), dict(H=0), dict(H=96), dict(reduction=3), dict(reduction=-1), dict(label_bytes=2), dict(logit_scale=-1.0),
       dict(logit_scale=float("nan")), dict(saved=None), dict(saved=8200), dict(ws=None), dict(ws=8), dict(ws_bytes=128)]


@pytest.mark.parametrize("over", BAD + [dict(loss=None), dict(loss=4097), dict(keep=3), dict(keep=-1)])
def test_forward_refuses(over):
    assert _fwd(**over) == -1
    assert b"xq_lce_fwd" in _C.lib().xq_last_error()


@pytest.mark.parametrize("over", BAD + [dict(grad=None), dict(keep=0), dict(keep=1), dict(dx=16392), dict(lddx=60), dict(dw=32776), dict(lddw=32)])
def test_backward_refuses(over):
    assert _bwd(**over) == -1


def test_sizes():
    L = _C.lib()
    assert ctypes.sizeof(_C.XqLceProblem) == 88
    assert L.xq_lce_saved_bytes(-1, 10, 64, 0) == -1 and L.xq_lce_workspace_bytes(1, 0, 64, 0) == -1
    for keep in (0, 1, 2):
        assert L.xq_lce_saved_bytes(0, 1, 64, keep) > 0
    # what a piece holds is bounded, whatever the sizes: 1 GiB of bf16, or 256 columns of all rows
    for M, V in ((1, 131072), (8192, 131072), (65536, 262144), (1 << 20, 131072)):
        rows = -(-M // 256) * 256
        for p in (2, 3):
            ws = L.xq_lce_workspace_bytes(M, V, 4096, p)
            assert ws <= max(1 << 30, rows * 512) + rows * 64 + rows * 8 * (V // 256 + 1) + (2 * M * 4096 if p == 3 else 0) + (1 << 20)


@pytest.mark.parametrize("M,V,H", [(1 << 24, 10, 64), (3, 1 << 28, 64), (3, 10, 1 << 24), (2 ** 63 - 1, 10, 64), (1, 2 ** 63 - 1, 64), (1 << 62, 1 << 62, 1 << 62)])
def test_sizes_out_of_range(M, V, H):
    """Launches that would have 2^32 threads and more, and sizes whose products pass 64 bits"""
    L = _C.lib()
    assert L.xq_lce_saved_bytes(M, V, H, 2) == -1 and L.xq_lce_workspace_bytes(M, V, H, 3) == -1
    assert _fwd(M=M, V=V, H=H, ldx=H, ldw=H) == -1 and _bwd(M=M, V=V, H=H, ldx=H, ldw=H) == -1


def test_largest_sizes():
    L = _C.lib()
    for M, V, H in (((1 << 24) - 1, 1000, 64), (1, (1 << 28) - 1, 64), (1, 1000, (1 << 24) - 64)):
        for p in (0, 1, 2, 3):
            assert L.xq_lce_workspace_bytes(M, V, H, p) > 0
