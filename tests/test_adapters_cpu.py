"""Host side of the adapters of many requests: what lora_adapters and xq_adapters_add refuse before anything runs."""

import ctypes

import pytest
import torch

from xorl_amd import _C
from xorl_amd.functional import lora_adapters

BF = torch.bfloat16


def _call(**over):
    a = dict(base=torch.zeros(3, 32, dtype=BF), x=torch.zeros(3, 64, dtype=BF), A=torch.zeros(5, 4, 64), B=torch.zeros(5, 32, 4), ids=torch.zeros(3, dtype=torch.int32),
             s=torch.ones(5), out=None)
    a.update(over)
    return lora_adapters(a["base"], a["x"], a["A"], a["B"], a["ids"], a["s"], out=a["out"])


def test_cpu_tensors_raise():
    with pytest.raises(RuntimeError, match="HIP device only"):
        _call()


@pytest.mark.parametrize("over,match", [
    (dict(base=torch.zeros(3, 32)), "must be bf16"), (dict(x=torch.zeros(3, 64)), "must be bf16"), (dict(A=torch.zeros(5, 4, 64, dtype=BF)), "both"),
    (dict(A=torch.zeros(5, 4, 64, dtype=torch.float16), B=torch.zeros(5, 32, 4, dtype=torch.float16)), "both"), (dict(s=torch.ones(5, dtype=BF)), "fp32"),
    (dict(ids=torch.zeros(3)), "int32 or int64"), (dict(ids=torch.zeros(4, dtype=torch.int32)), "do not go together"), (dict(s=torch.ones(4)), "do not go together"),
    (dict(A=torch.zeros(4, 4, 64)), "do not go together"), (dict(A=torch.zeros(5, 4, 128)), "do not go together"), (dict(B=torch.zeros(5, 16, 4)), "do not go together"),
    (dict(B=torch.zeros(5, 32, 3)), "do not go together"), (dict(x=torch.zeros(1, 3, 64, dtype=BF)), "do not go together"), (dict(A=torch.zeros(4, 64)), "do not go together"),
    (dict(x=torch.zeros(3, 96, dtype=BF), A=torch.zeros(5, 4, 96)), "multiple of 64"), (dict(base=torch.zeros(3, 24, dtype=BF), B=torch.zeros(5, 24, 4)), "multiple of 64"),
    (dict(A=torch.zeros(5, 65, 64), B=torch.zeros(5, 32, 65)), "rank"), (dict(A=torch.zeros(5, 0, 64), B=torch.zeros(5, 32, 0)), "rank"),
    (dict(A=torch.zeros(5, 4, 64, requires_grad=True)), "forward-only"), (dict(base=torch.zeros(3, 32, dtype=BF, requires_grad=True)), "forward-only"),
    (dict(out=torch.zeros(3, 32, dtype=BF, requires_grad=True)), "forward-only"),
])
def test_argument_errors(over, match):
    with pytest.raises(_C.XqError, match=match):
        _call(**over)


def test_tangents_are_refused():
    import torch.autograd.forward_ad as fwAD

    with fwAD.dual_level(), pytest.raises(NotImplementedError, match="tangent"):
        _call(x=fwAD.make_dual(torch.zeros(3, 64, dtype=BF), torch.ones(3, 64, dtype=BF)))


def _run(ws=1 << 20, ws_bytes=1 << 30, **over):
    # addresses that nothing reads: every call below is refused on the host
    f = dict(x=4096, ldx=64, base=8192, ld_base=32, out=8192, ld_out=32, A=4096, B=4096, scaling=4096, ids=4096, M=3, N=32, K=64, n_adapters=5, r=4, factor_dtype=1, id_bytes=4)
    f.update(over)
    return _C.lib().xq_adapters_add(ctypes.byref(_C.XqAdapters(**f)), ws, ws_bytes, None)


@pytest.mark.parametrize("over", [
    dict(x=None), dict(x=4104), dict(ldx=56), dict(ldx=68), dict(base=None), dict(base=8200), dict(ld_base=24), dict(ld_base=36), dict(out=None), dict(out=8194), dict(ld_out=16),
    dict(A=None), dict(A=4100), dict(B=None), dict(B=4104), dict(scaling=None), dict(scaling=4098), dict(ids=None), dict(ids=4098), dict(ids=4100, id_bytes=8), dict(id_bytes=2),
    dict(M=-1), dict(M=1 << 24), dict(N=0), dict(N=24), dict(N=1 << 24), dict(K=0), dict(K=96), dict(K=1 << 24), dict(n_adapters=-1), dict(r=0), dict(r=65), dict(factor_dtype=2),
    dict(ws=None), dict(ws=8), dict(ws_bytes=0), dict(M=2 ** 63 - 1), dict(N=2 ** 62), dict(K=2 ** 62)])
def test_refusals(over):
    assert _run(**over) == -1
    assert b"xq_adapters_add" in _C.lib().xq_last_error()


@pytest.mark.parametrize("over", [dict(K=1 << 23, ldx=1 << 23), dict(N=1 << 24, ld_base=1 << 24, ld_out=1 << 24), dict(M=1 << 24)])
def test_the_largest_sizes(over):
    """The first size that is too large is refused as a size, the one before only for the workspace that it does not have"""
    assert _run(**over) == -1 and b"must be a multiple of 64 below" in _C.lib().xq_last_error()
    step = {"K": 64, "N": 16, "M": 1}[next(iter(over))]
    below = {k: v - step if k in "MNK" else v for k, v in over.items()}
    assert _run(ws=None, **below) == -1 and b"workspace" in _C.lib().xq_last_error()


def test_sizes():
    L = _C.lib()
    assert ctypes.sizeof(_C.XqAdapters) == 120
    assert L.xq_adapters_add(None, 256, 1 << 20, None) == -1
    assert L.xq_adapters_workspace_bytes(0, 16, 64, 1) >= 0 and L.xq_adapters_workspace_bytes(-1, 16, 64, 1) == -1 and L.xq_adapters_workspace_bytes(1, 16, 64, 65) == -1
    assert _run(M=0, x=None, base=None, out=None, ids=None, ws=None) == 0
