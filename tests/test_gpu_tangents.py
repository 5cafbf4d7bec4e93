"""GPU: frozen modules refuse tangents of forward-mode differentiation, as trained ones do."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from tests.test_gpu_moe import _make_experts
from tests.util_cases import gen, make_dense_module
from xorl_amd.qlora import linear as QL

pytestmark = pytest.mark.gpu


def test_frozen_modules_refuse_tangents(hip_device):
    up, gate = (make_dense_module("int4", 128, 256, 16, 32, s, hip_device)[0].requires_grad_(False) for s in (3, 4))
    down = make_dense_module("int4", 256, 128, 16, 32, 5, hip_device)[0].requires_grad_(False)
    x = gen((4, 256), 1.0, 4, torch.bfloat16).to(hip_device)
    with fwAD.dual_level():
        dual = fwAD.make_dual(x, torch.ones_like(x))
        for call in (lambda t: up(t), lambda t: QL.qlora_linears_forward([gate, up], t), lambda t: QL.qlora_gate_up_silu(up, t),
                     lambda t: QL.qlora_mlp_forward(gate, up, down, t)):
            call(x)
            with pytest.raises(NotImplementedError):
                call(dual)
            with torch.no_grad(), pytest.raises(NotImplementedError):
                call(dual)


def test_frozen_experts_refuse_tangents(hip_device):
    m = _make_experts("block_fp8", 4, 256, 256, 8, False, 7, hip_device)[0].requires_grad_(False)
    x = gen((3, 256), 1.0, 8, torch.bfloat16).to(hip_device)
    rw, sel = torch.full((3, 2), 0.5, device=hip_device), torch.tensor([[0, 1], [1, 2], [3, 0]], device=hip_device)
    m(x, rw, sel)
    with fwAD.dual_level():
        for args in ((fwAD.make_dual(x, torch.ones_like(x)), rw), (x, fwAD.make_dual(rw, torch.ones_like(rw)))):
            with pytest.raises(NotImplementedError):
                m(*args, sel)
