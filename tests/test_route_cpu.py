"""Host side of the choice of experts: what moe_route and the C entry points refuse before anything runs."""

import ctypes

import pytest
import torch

from xorl_amd import _C
from xorl_amd.moe_functional import moe_route


def _call(z=None, top_k=2, **kw):
    return moe_route(torch.zeros(3, 16) if z is None else z, top_k, **kw)


def test_cpu_tensors_raise():
    with pytest.raises(RuntimeError, match="HIP device only"):
        _call()


@pytest.mark.parametrize("kw,match", [
    (dict(scoring="tanh"), "scoring"), (dict(group_score="mean"), "group_score"), (dict(z=torch.zeros(3, 16, dtype=torch.float16)), "bf16 or fp32"),
    (dict(z=torch.zeros(3, 16, dtype=torch.int64)), "bf16 or fp32"), (dict(z=torch.zeros(3, 0)), "experts"), (dict(z=torch.zeros(3, 1025)), "experts"),
    (dict(z=torch.tensor(1.0)), "bf16 or fp32"), (dict(bias=torch.zeros(15)), "bias"), (dict(bias=torch.zeros(16, dtype=torch.bfloat16)), "bias"),
    (dict(bias=torch.zeros(3, 16)), "bias"), (dict(num_groups=3), "groups"), (dict(num_groups=0), "groups"), (dict(num_groups=4, top_groups=5), "groups"),
    (dict(num_groups=4, top_groups=0), "groups"), (dict(top_k=0), "top_k"), (dict(top_k=17), "top_k"), (dict(z=torch.zeros(3, 64), top_k=33), "top_k"),
    (dict(top_k=5, num_groups=4, top_groups=1), "top_k"), (dict(z=torch.zeros(3, 130), num_groups=65), "groups"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=torch.ones(())), "numbers"),
])
def test_argument_errors(kw, match):
    with pytest.raises(_C.XqError, match=match):
        _call(**kw)


def _problem(**over):
    # addresses that nothing reads: every call below is refused on the host
    f = dict(logits=4096, ld=16, bias=8192, n_tokens=3, dtype=1, num_experts=16, top_k=2, scoring=0, num_groups=1, top_groups=1, group_score=0, renormalize=0, scale=1.0)
    f.update(over)
    return _C.XqMoeRoute(**f)


def _fwd(weights=4096, selected=8192, **over):
    return _C.lib().xq_moe_route_fwd(ctypes.byref(_problem(**over)), weights, selected, None)


def _bwd(weights=4096, selected=8192, grad=4096, dz=8192, ld_dz=16, **over):
    return _C.lib().xq_moe_route_bwd(ctypes.byref(_problem(**over)), weights, selected, grad, dz, ld_dz, None)


BAD = [dict(logits=None), dict(logits=4098), dict(ld=15), dict(bias=8194), dict(n_tokens=-1), dict(n_tokens=1 << 26), dict(dtype=2), dict(num_experts=0), dict(num_experts=1025),
       dict(top_k=0), dict(top_k=17), dict(num_experts=64, ld=64, top_k=33), dict(scoring=2), dict(scoring=-1), dict(num_groups=0), dict(num_groups=3),
       dict(num_experts=130, ld=130, num_groups=65), dict(num_groups=4, top_groups=0), dict(num_groups=4, top_groups=5), dict(num_groups=8, top_groups=1, top_k=3),
       dict(group_score=2), dict(scale=0.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(weights=None), dict(weights=4098), dict(selected=None), dict(selected=8196)]


@pytest.mark.parametrize("over", BAD)
def test_forward_refuses(over):
    assert _fwd(**over) == -1
    assert b"xq_moe_route_fwd" in _C.lib().xq_last_error()


@pytest.mark.parametrize("over", BAD + [dict(grad=None), dict(grad=4097), dict(dz=None), dict(dz=8194), dict(ld_dz=15)])
def test_backward_refuses(over):
    assert _bwd(**over) == -1
    assert b"xq_moe_route_bwd" in _C.lib().xq_last_error()


def test_null_problem_and_no_tokens():
    L = _C.lib()
    assert ctypes.sizeof(_C.XqMoeRoute) == 72
    assert L.xq_moe_route_fwd(None, 4096, 8192, None) == -1 and L.xq_moe_route_bwd(None, 4096, 8192, 4096, 8192, 16, None) == -1
    assert _fwd(n_tokens=0, logits=None, weights=None, selected=None) == 0
    assert _bwd(n_tokens=0, logits=None, weights=None, selected=None, grad=None, dz=None) == 0
