"""The forward-only calls of the packed modules refuse tangents of forward-mode differentiation, before anything else is looked at."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from xorl_amd import functional as F
from xorl_amd import moe_functional as MF

BF = torch.bfloat16


def _qw(rows, cols, experts=1):
    return F.QuantWeight("int4", "flat", torch.zeros(1), torch.zeros(1), torch.float32, rows, cols, 64, None, experts)


def _linear(x, A, B):
    return F.qlora_linear(x, _qw(128, 64), A, B, 4, 1.0)


def _swiglu(x, A, B):
    return F.qlora_linear_swiglu(x, _qw(128, 64), A, B, 4, 1.0)


def _multi(x, A, B):
    return F.qlora_linear_multi(x, [(_qw(128, 64), None, None, 0, 1.0, None), (_qw(128, 64), A, B, 4, 1.0, None)])


def _mlp(x, A, B):
    return F.qlora_mlp_infer(x, _qw(128, 64), _qw(128, 64), _qw(64, 128), None, None, A, B, None, None, 4, 1.0)


def _moe(x, A, B):
    rw, sel = torch.ones(3, 1), torch.zeros(3, 1, dtype=torch.int64)
    return MF.moe_experts_qlora_forward(1, rw, sel, x, _qw(64, 128), _qw(64, 128), _qw(128, 64), A, B, A, B, A, B, 1.0)


@pytest.mark.parametrize("call", [_linear, _swiglu, _multi, _mlp, _moe])
@pytest.mark.parametrize("which", ["x", "A", "B"])
def test_tangents_are_refused(call, which):
    t = {"x": torch.zeros(3, 64, dtype=BF), "A": torch.zeros(4, 64), "B": torch.zeros(128, 4)}
    with fwAD.dual_level():
        t[which] = fwAD.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(NotImplementedError, match="tangent"):
            call(t["x"], t["A"], t["B"])


def test_routing_weights_with_a_tangent_are_refused():
    with fwAD.dual_level():
        rw = fwAD.make_dual(torch.ones(3, 1), torch.ones(3, 1))
        f = [torch.zeros(1, 64, 4), torch.zeros(1, 4, 128)] * 2 + [torch.zeros(1, 128, 4), torch.zeros(1, 4, 64)]
        with pytest.raises(NotImplementedError, match="tangent"):
            MF.moe_experts_qlora_forward(1, rw, torch.zeros(3, 1, dtype=torch.int64), torch.zeros(3, 64, dtype=BF), _qw(64, 128), _qw(64, 128), _qw(128, 64), *f, 1.0)
