"""Host side of AdamW: what it takes of other optimizers' state dictionaries, and the states of sharded parameters."""

import pytest
import torch

from xorl_amd import _C
from xorl_amd.optim import AdamW


def _adam(weight_decay, **kw):
    p = torch.nn.Parameter(torch.ones(8))
    opt = torch.optim.Adam([p], lr=0.1, weight_decay=weight_decay, **kw)
    p.grad = torch.ones(8)
    opt.step()
    return opt.state_dict()


def test_decay_that_is_added_to_the_gradients_is_refused():
    p = torch.nn.Parameter(torch.ones(8))
    opt = AdamW([p], lr=1.0, weight_decay=0.5)
    with pytest.raises(_C.XqError, match="added to the gradients"):
        opt.load_state_dict(_adam(0.1))
    assert opt.param_groups[0]["lr"] == 1.0 and not opt.state
    for d in (_adam(0.0), _adam(0.1, decoupled_weight_decay=True)):
        opt.load_state_dict(d)
        assert opt.param_groups[0]["weight_decay"] == d["param_groups"][0]["weight_decay"] and float(opt.state[p]["step"]) == 1.0
        # what is saved here is this class's own update, whatever came in
        opt.param_groups[0]["weight_decay"] = 0.2
        again = AdamW([p])
        again.load_state_dict(opt.state_dict())
        assert again.param_groups[0]["weight_decay"] == 0.2
