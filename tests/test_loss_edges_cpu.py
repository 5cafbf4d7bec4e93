"""Host side of linear_cross_entropy: what would be left out without a word is refused."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from xorl_amd import _C, loss_functional
from xorl_amd.loss_functional import linear_cross_entropy

BF = torch.bfloat16


def _stand_in(x, weight, labels, ignore_index, reduction, logit_scale, keep):
    loss = torch.nn.functional.cross_entropy(logit_scale * x.float() @ weight.float().t(), labels, reduction=("none", "mean", "sum")[reduction])
    return loss, torch.zeros(1, dtype=torch.uint8)


@pytest.mark.parametrize("head_grad", [False, True])
@pytest.mark.parametrize("which", ["x", "weight"])
def test_tangents_are_refused(monkeypatch, which, head_grad):
    """Not dropped: a loss without a tangent has the derivative zero.  (The kernel's place is taken, so that nothing else refuses the call.)"""
    monkeypatch.setattr(loss_functional, "_fwd_impl", _stand_in)
    monkeypatch.setattr(loss_functional._C, "require_hip", lambda *t: None)
    t = {"x": torch.randn(3, 64).to(BF), "weight": torch.randn(10, 64).to(BF).requires_grad_(head_grad)}
    labels = torch.tensor([1, 2, 3])
    with fwAD.dual_level():
        t[which] = fwAD.make_dual(t[which], torch.ones(t[which].shape, dtype=BF))
        with pytest.raises(NotImplementedError):
            linear_cross_entropy(t["x"], t["weight"], labels)
        with torch.no_grad(), pytest.raises(NotImplementedError):
            linear_cross_entropy(t["x"], t["weight"], labels)
    with fwAD.dual_level():                               # (a level without tangents refuses nothing)
        assert linear_cross_entropy(torch.zeros(3, 64, dtype=BF), torch.zeros(10, 64, dtype=BF), labels).shape == ()


def test_a_trained_scale_is_refused():
    """It is a number here: the gradient that a tensor waits for would never come"""
    scale = torch.tensor(2.0, requires_grad=True)
    x, w, labels = torch.zeros(3, 64, dtype=BF), torch.zeros(10, 64, dtype=BF), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(_C.XqError, match="logit_scale gets no gradient"):
        linear_cross_entropy(x, w, labels, logit_scale=scale)
    for call in (torch.no_grad(), torch.enable_grad()):
        with call, pytest.raises(RuntimeError, match="HIP device only"):
            linear_cross_entropy(x, w, labels, logit_scale=scale.detach())
