"""GPU: arguments whose memory is not what they stand for: freed, or with the other sign."""

import numpy as np
import pytest
import torch

from tests.util_cases import make_dense_module
from xorl_amd import _C
from xorl_amd.embedding_functional import embedding
from xorl_amd.functional import lora_adapters
from xorl_amd.loss_functional import linear_cross_entropy
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


def _freed(t):
    """t behind eight others of a storage that is freed: its address is not 0"""
    flat = torch.cat([t.new_zeros(8), t.reshape(-1)])
    view = flat[8:].view(t.shape)
    flat.untyped_storage().resize_(0)
    return view


def test_views_into_freed_memory_are_refused(hip_device):
    z, bias = torch.randn(6, 8, device=hip_device), torch.randn(8, device=hip_device)
    w, ids = torch.randn(10, 16, device=hip_device), torch.tensor([3, 0, 9], device=hip_device)
    a = [torch.zeros(4, 16, dtype=BF, device=hip_device), torch.zeros(4, 64, dtype=BF, device=hip_device), torch.zeros(2, 4, 64, device=hip_device), torch.zeros(2, 16, 4, device=hip_device),
         torch.zeros(4, dtype=torch.int32, device=hip_device), torch.ones(2, device=hip_device)]
    calls = [lambda: moe_route(_freed(z), 2), lambda: moe_route(z, 2, bias=_freed(bias)), lambda: embedding(_freed(ids), w), lambda: embedding(ids, _freed(w)),
             lambda: embedding(ids, _freed(w).requires_grad_(True))]
    calls += [lambda i=i: lora_adapters(*a[:i], _freed(a[i]), *a[i + 1:]) for i in range(6)]
    # what the compiled host path leaves to Python
    calls += [lambda: moe_route(_freed(z), np.int64(2)), lambda: embedding(_freed(ids), w, scale=np.float32(1.0)), lambda: torch.ops.xq.embedding_fwd(ids, _freed(w), 1.0)]
    calls += [lambda i=i: lora_adapters(*a[:i], _freed(a[i]), *a[i + 1:], out=torch.empty_like(a[0])) for i in range(6)] + [lambda: lora_adapters(*a, out=_freed(a[0]))]
    for call in calls:
        with pytest.raises(_C.XqError, match="no memory"):
            call()


def _negated(t):
    """a view that stands for t: its memory holds the other sign"""
    return torch._neg_view(t.neg())


def test_negated_views_of_logits_and_biases(hip_device):
    g = torch.Generator(device=hip_device).manual_seed(1)
    z, bias, up = (torch.randn(n, device=hip_device, generator=g) for n in ((6, 16), (16,), (6, 4)))
    for options in (dict(renormalize=False), dict(scoring="sigmoid")):
        leaf = z.clone().requires_grad_(True)
        w, ids = moe_route(leaf, 4, bias=bias, **options)
        for zz, bb in ((_negated(z), bias), (z, _negated(bias)), (_negated(z), _negated(bias))):
            got = moe_route(zz, 4, bias=bb, **options)
            assert torch.equal(got[0], w) and torch.equal(got[1], ids)
            turned = zz.detach().requires_grad_(True)
            got = moe_route(turned, 4, bias=bb, **options)
            assert torch.equal(got[0], w) and torch.equal(got[1], ids)
            assert torch.equal(torch.autograd.grad(got[0], turned, _negated(up))[0], torch.autograd.grad(w, leaf, up, retain_graph=True)[0])
        assert torch.equal(torch.autograd.grad(w, leaf, _negated(up), retain_graph=True)[0], torch.autograd.grad(w, leaf, up)[0])


@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_negated_views_of_an_embedding(hip_device, dtype):
    g = torch.Generator(device=hip_device).manual_seed(2)
    w, up = torch.randn(10, 16, device=hip_device, generator=g).to(dtype), torch.randn(6, 16, device=hip_device, generator=g).to(dtype)
    ids = torch.tensor([3, 0, 9, 3, 1, 2], device=hip_device)
    leaf = w.clone().requires_grad_(True)
    out = embedding(ids, leaf, scale=2.0)
    dw, = torch.autograd.grad(out, leaf, up, retain_graph=True)
    assert torch.equal(embedding(ids, _negated(w), scale=2.0), out) and torch.equal(embedding(_negated(ids), w, scale=2.0), out)
    assert torch.equal(torch.autograd.grad(out, leaf, _negated(up))[0], dw)
    turned = _negated(w).detach().requires_grad_(True)
    out2 = embedding(_negated(ids), turned, scale=2.0)
    assert torch.equal(out2, out) and torch.equal(torch.autograd.grad(out2, turned, _negated(up))[0], dw)


def test_negated_views_of_adapters(hip_device):
    g = torch.Generator(device=hip_device).manual_seed(3)
    base, x = torch.randn(4, 16, device=hip_device, generator=g).to(BF), torch.randn(4, 64, device=hip_device, generator=g).to(BF)
    A, B = torch.randn(2, 4, 64, device=hip_device, generator=g), torch.randn(2, 16, 4, device=hip_device, generator=g)
    ids, s = torch.tensor([0, 1, -1, 1], dtype=torch.int32, device=hip_device), torch.rand(2, device=hip_device, generator=g)
    a = [base, x, A, B, ids, s]
    want = lora_adapters(*a)
    for i in range(6):
        assert torch.equal(lora_adapters(*a[:i], _negated(a[i]), *a[i + 1:]), want), i
    for out in (_negated(base), torch._neg_view(torch.empty_like(base))):
        with pytest.raises(_C.XqError, match="out must be"):
            lora_adapters(out, *a[1:], out=out)


def test_a_negated_gradient_of_the_loss(hip_device):
    g = torch.Generator(device=hip_device).manual_seed(4)
    x = torch.randn(5, 64, device=hip_device, generator=g).to(BF).requires_grad_(True)
    w = torch.randn(128, 64, device=hip_device, generator=g).to(BF).requires_grad_(True)
    loss = linear_cross_entropy(x, w, torch.tensor([1, 5, 0, 100, 127], device=hip_device))
    want = torch.autograd.grad(loss, (x, w), torch.tensor(-2.0, device=hip_device), retain_graph=True)
    got = torch.autograd.grad(loss, (x, w), torch._neg_view(torch.tensor(2.0, device=hip_device)))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
