"""GPU: arguments whose memory is not what their shape says."""

import pytest
import torch

from tests.util_cases import make_dense_module
from xorl_amd import _C
from xorl_amd.moe_functional import moe_route

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def test_a_bias_whose_memory_was_freed_is_refused(hip_device):
    z, bias = torch.randn(6, 8, device=hip_device), torch.randn(8, device=hip_device)
    bias.untyped_storage().resize_(0)
    for t in (z, z.clone().requires_grad_(True)):
        with pytest.raises(_C.XqError, match="no memory"):
            moe_route(t, 2, bias=bias)


def test_a_linear_whose_bias_was_freed_is_refused(hip_device):
    m, _ = make_dense_module("int4", 64, 128, 8, 16, 3, hip_device, bias=True)
    m.bias = torch.nn.Parameter(m.bias.detach().to(BF))
    x = torch.randn(3, 128, device=hip_device).to(BF)
    with torch.no_grad():
        assert m(x).shape == (3, 64)
        m.bias.untyped_storage().resize_(0)
        with pytest.raises(_C.XqError, match="no memory"):
            m(x)
