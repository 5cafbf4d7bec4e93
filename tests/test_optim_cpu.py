"""Host side of the optimizer step: what adamw_step, grad_norm, AdamW and the C entry points refuse before anything runs."""

import copy
import ctypes

import pytest
import torch

from xorl_amd import _C
from xorl_amd.optim import AdamW, adamw_state_values, adamw_step, grad_norm


def _lists(n=3, shape=(4, 8)):
    make = lambda: [torch.zeros(shape) for _ in range(n)]  # noqa: E731
    return make(), make(), make(), make(), [torch.zeros(()) for _ in range(n)]


def test_cpu_tensors_raise():
    p, g, m, v, t = _lists()
    with pytest.raises(RuntimeError, match="HIP device only"):
        adamw_step(p, g, m, v, t, lr=1e-3)
    with pytest.raises(RuntimeError, match="HIP device only"):
        grad_norm(g)
    with pytest.raises(RuntimeError, match="HIP device only"):
        adamw_state_values(torch.zeros(4, dtype=torch.int8), torch.zeros(4, dtype=torch.uint8), torch.zeros(1), torch.zeros(1))
    q = torch.nn.Parameter(torch.zeros(4))
    q.grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="HIP device only"):
        AdamW([q]).step()


def test_argument_errors_on_the_host():
    p, g, m, v, t = _lists()
    with pytest.raises(_C.XqError, match="differ in length"):
        adamw_step(p[:2], g, m, v, t, lr=1e-3)
    with pytest.raises(_C.XqError, match="need exp_avg_scales and"):
        adamw_step(p, g, m, v, t, exp_avg_scales=[], lr=1e-3)
    with pytest.raises(_C.XqError, match="not a tensor"):
        adamw_step(p, [1.0, 2.0, 3.0], m, v, t, lr=1e-3)
    with pytest.raises(_C.XqError, match="no device"):
        grad_norm([])
    assert adamw_step([], [], [], [], [], lr=1e-3) is None
    with pytest.raises(_C.XqError, match="state_bits"):
        AdamW([torch.nn.Parameter(torch.zeros(1))], state_bits=4)
    with pytest.raises(_C.XqError, match="max_grad_norm"):
        AdamW([torch.nn.Parameter(torch.zeros(1))], max_grad_norm=0.0)


def _tensor(**over):
    # addresses that nothing reads: every call below is refused on the host
    a = dict(param=4096, grad=8192, exp_avg=12288, exp_avg_sq=16384, exp_avg_scale=20480, exp_avg_sq_scale=24576, step=28672, numel=16,
             param_dtype=_C.XQ_DT_F32, grad_dtype=_C.XQ_DT_F32)
    a.update(over)
    return _C.XqAdamwTensor(**a)


def _step(tensor, n=1, ws=1 << 20, ws_bytes=1 << 20, **over):
    o = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, max_norm=0.0, lr_device=None, norm=None, norm_given=0, state_bits=32)
    o.update(over)
    return _C.lib().xq_adamw_step(ctypes.byref(tensor), n, ctypes.byref(_C.XqAdamwOptions(**o)), ws, ws_bytes, None)


@pytest.mark.parametrize("over", [dict(numel=0), dict(numel=-1), dict(param=None), dict(grad=None), dict(exp_avg=None), dict(exp_avg_sq=None), dict(step=None),
                                  dict(param=4098), dict(grad=8193, grad_dtype=_C.XQ_DT_BF16), dict(exp_avg=12290), dict(param_dtype=7), dict(grad_dtype=-1)] + [{k: 1 << 48} for k in ("param", "grad", "exp_avg", "exp_avg_sq", "step")])
def test_step_refuses_tensor(over):
    assert _step(_tensor(**over)) == -1
    assert b"xq_adamw_step" in _C.lib().xq_last_error()


@pytest.mark.parametrize("over", [dict(lr=-1.0), dict(lr=float("nan")), dict(beta1=1.0), dict(beta2=-0.1), dict(eps=-1e-8), dict(weight_decay=-1.0),
                                  dict(state_bits=16), dict(norm=4096, max_norm=0.0), dict(norm=4097, max_norm=1.0), dict(norm_given=1),
                                  dict(lr_device=4097), dict(ws=None), dict(ws=1), dict(ws_bytes=64), dict(n=-1)])
def test_step_refuses_options(over):
    assert _step(_tensor(), **over) == -1


def test_step_refuses_8_bit_states_without_scales():
    assert _step(_tensor(exp_avg_scale=None), state_bits=8) == -1
    assert _step(_tensor(exp_avg_sq_scale=24578), state_bits=8) == -1


def test_norm_and_values_refuse():
    L = _C.lib()
    t = _tensor(grad=None)
    assert L.xq_grad_norm(ctypes.byref(t), 1, 4096, 1 << 20, 1 << 20, None) == -1
    t = _tensor()
    assert L.xq_grad_norm(ctypes.byref(t), 1, None, 1 << 20, 1 << 20, None) == -1
    assert L.xq_grad_norm(ctypes.byref(t), 1, 4096, 1 << 20, 16, None) == -1
    assert L.xq_adamw_values(4096, 4096, 4096, 4096, -1, 4096, 4096, _C.XQ_DT_F32, None) == -1
    assert L.xq_adamw_values(4096, 4096, 4096, 4096, 8, 4096, 4096, 5, None) == -1
    assert L.xq_adamw_values(4096, None, 4096, 4096, 8, 4096, 4096, _C.XQ_DT_F32, None) == -1
    assert L.xq_adamw_values(4096, 4096, 4098, 4096, 8, 4096, 4096, _C.XQ_DT_F32, None) == -1
    assert L.xq_adamw_values(None, None, None, None, 0, None, None, _C.XQ_DT_F32, None) == 0
    assert L.xq_adamw_workspace_bytes(-1) == -1 and L.xq_adamw_workspace_bytes(0) > 0


def test_struct_layout():
    assert ctypes.sizeof(_C.XqAdamwTensor) == 72 and ctypes.sizeof(_C.XqAdamwOptions) == 72


def test_states_of_torch_adamw_are_taken():
    """A dictionary of torch.optim.AdamW, with a bf16 parameter's bf16 moments and a step count that is a number, goes on in fp32 with 32 bits"""
    a, b = torch.nn.Parameter(torch.ones(8)), torch.nn.Parameter(torch.ones(8, dtype=torch.bfloat16))
    theirs = torch.optim.AdamW([a, b], lr=0.5, betas=(0.8, 0.9))
    a.grad, b.grad = torch.ones(8), torch.ones(8, dtype=torch.bfloat16)
    theirs.step()
    d = theirs.state_dict()
    d["state"][1]["step"] = 1
    opt = AdamW([a, b], state_bits=8)
    opt.load_state_dict(d)
    g = opt.param_groups[0]
    assert (g["lr"], g["betas"], g["state_bits"]) == (0.5, (0.8, 0.9), 32)
    for p in (a, b):
        s = opt.state[p]
        assert all(s[k].dtype == torch.float32 for k in ("step", "exp_avg", "exp_avg_sq")) and float(s["step"]) == 1.0
        assert torch.equal(s["exp_avg"], theirs.state[p]["exp_avg"].float())
    for variant in ("amsgrad", "maximize"):
        with pytest.raises(_C.XqError, match="amsgrad and maximize"):
            opt.load_state_dict(torch.optim.AdamW([a, b], **{variant: True}).state_dict())


def test_copies_and_groups_keep_the_options():
    q = torch.nn.Parameter(torch.zeros(4))
    opt = AdamW([q], state_bits=8, max_grad_norm=0.5)
    assert copy.deepcopy(opt).max_grad_norm == 0.5 and copy.deepcopy(opt).param_groups[0]["state_bits"] == 8
    for bits in (16, None):
        with pytest.raises(_C.XqError, match="state_bits"):
            opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(2))], "state_bits": bits})
