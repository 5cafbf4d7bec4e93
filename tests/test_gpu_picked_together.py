"""GPU: embedding, adapters and the choice of experts as a model uses them: a training step and a serving step over the packed modules."""

import pytest
import torch

from tests.test_gpu_moe import _make_experts
from tests.util_cases import make_dense_module
from xorl_amd.embedding_functional import embedding
from xorl_amd.functional import lora_adapters
from xorl_amd.loss_functional import linear_cross_entropy
from xorl_amd.moe_functional import moe_route
from xorl_amd.optim import AdamW
from xorl_amd.qlora import qlora_adapters_forward

pytestmark = pytest.mark.gpu
B, BF = 2.0 ** -8, torch.bfloat16


def _model(device, fmt="block_fp8"):
    lin, _ = make_dense_module(fmt, 256, 256, 8, 16, seed=1, device=device)
    experts, _ = _make_experts(fmt, 16, 256, 256, 8, False, 5, device)
    g = torch.Generator(device=device).manual_seed(2)
    w = (torch.randn(1000, 256, device=device, generator=g) * 0.3).to(BF).requires_grad_(True)
    router = (torch.randn(16, 256, device=device, generator=g) * 0.05).requires_grad_(True)
    return lin, experts, w, router


def _plain_embedding(ids, w, scale):
    return (torch.nn.functional.embedding(ids, w).float() * scale).to(w.dtype)


def _plain_route(z, k):
    p, ids = torch.softmax(z, -1).topk(k, -1)
    return p / p.sum(-1, keepdim=True), ids


def _loss(model, ids, labels, own):
    lin, experts, w, router = model
    x = embedding(ids, w, scale=2.0) if own else _plain_embedding(ids, w, 2.0)
    x = x + lin(x)
    z = x.float() @ router.t()
    weights, chosen = moe_route(z, 4) if own else _plain_route(z, 4)
    x = x + experts(x, weights, chosen)
    return linear_cross_entropy(x, w, labels), chosen


def test_training_step(hip_device):
    model = _model(hip_device)
    lin, experts, w, router = model
    ids = torch.randint(0, 1000, (2, 150), device=hip_device)
    labels = torch.randint(0, 1000, (2, 150), device=hip_device)
    leaves = [w, router, lin.lora_A, lin.lora_B, experts.gate_proj_lora_A, experts.down_proj_lora_B]
    loss, chosen = _loss(model, ids, labels, True)
    grads = torch.autograd.grad(loss, leaves)
    loss2, chosen2 = _loss(model, ids, labels, False)
    grads2 = torch.autograd.grad(loss2, leaves)
    # the same formulas: weights differ by a step of fp32, which moves a few bf16 values by a step (2 B of them); two roundings of activations
    # and two of gradients lie on the way
    assert torch.equal(chosen, chosen2) and abs(float(loss) - float(loss2)) <= 8 * B * abs(float(loss2))
    for a, b in zip(grads, grads2):
        assert float((a.double() - b.double()).norm()) <= 8 * B * float(b.double().norm())
    for p, g in zip(leaves, grads):
        p.grad = g
    before = [p.detach().clone() for p in leaves]
    AdamW(leaves, lr=1e-2, weight_decay=0.0).step()
    assert all(not torch.equal(p, q) for p, q in zip(leaves, before))
    assert torch.isfinite(_loss(model, ids, labels, True)[0])


def _serve(model, ids, bank_A, bank_B, who, s):
    lin, experts, w, router = model
    x = embedding(ids, w, scale=2.0)
    x = x + qlora_adapters_forward(lin, x, bank_A, bank_B, who, s)
    weights, chosen = moe_route(x.float() @ router.t(), 4)
    return x + experts(x, weights, chosen)


@pytest.mark.parametrize("fmt", ["block_fp8", "nvfp4"])
@pytest.mark.parametrize("T", [1, 6, 40])
def test_serving_step(hip_device, fmt, T):
    model = _model(hip_device, fmt)
    g = torch.Generator(device=hip_device).manual_seed(3)
    bank_A = (torch.randn(5, 16, 256, device=hip_device, generator=g) / 16).to(BF)
    bank_B = (torch.randn(5, 256, 16, device=hip_device, generator=g) * 0.1).to(BF)
    s = torch.rand(5, device=hip_device, generator=g)
    ids, who = torch.zeros(T, dtype=torch.int64, device=hip_device), torch.zeros(T, dtype=torch.int32, device=hip_device)
    with torch.no_grad():
        for _ in range(2):
            _serve(model, ids, bank_A, bank_B, who, s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _serve(model, ids, bank_A, bank_B, who, s)
        for step in range(3):
            ids.copy_(torch.randint(0, 1000, (T,), device=hip_device, generator=g))
            who.copy_(torch.randint(-1, 5, (T,), device=hip_device, generator=g))
            graph.replay()
            torch.cuda.synchronize()
            want = _serve(model, ids, bank_A, bank_B, who, s)
            assert torch.equal(out, want) and out.isfinite().all()
            if T > 1:                                 # each request by itself: other kernels by size, the same formulas
                alone = torch.cat([_serve(model, ids[i:i + 1], bank_A, bank_B, who[i:i + 1], s) for i in range(T)])
                assert float((alone.double() - want.double()).norm()) <= 8 * B * float(want.double().norm())


def test_calls_on_two_streams_at_once(hip_device):
    """Each call has a workspace of its own: what two streams do side by side is what each does alone"""
    g = torch.Generator(device=hip_device).manual_seed(8)
    w = torch.randn(5000, 512, device=hip_device, generator=g).to(BF).requires_grad_(True)
    bank_A = (torch.randn(9, 16, 512, device=hip_device, generator=g) / 16).to(BF)
    bank_B = (torch.randn(9, 256, 16, device=hip_device, generator=g) * 0.1).to(BF)
    s, bias = torch.rand(9, device=hip_device, generator=g), 0.1 * torch.randn(256, device=hip_device, generator=g)

    def inputs(T):
        return (torch.randint(0, 5000, (T,), device=hip_device, generator=g), torch.randint(-1, 9, (T,), device=hip_device, generator=g),
                torch.randn(T, 256, device=hip_device, generator=g), torch.randn(T, 256, device=hip_device, generator=g).to(BF), torch.randn(T, 512, device=hip_device, generator=g).to(BF))

    def work(ids, who, z, base, up):
        out = embedding(ids, w, scale=2.0)
        dw, = torch.autograd.grad(out, w, up)
        with torch.no_grad():
            y = lora_adapters(base, out.detach(), bank_A, bank_B, who, s)
            weights, chosen = moe_route(z, 8, scoring="sigmoid", bias=bias, num_groups=8, top_groups=4)
        return out.detach(), dw, y, weights, chosen

    sets = [inputs(T) for T in (300, 3001)]
    want = [work(*a) for a in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(10):
        for st, a in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(work(*a))
    torch.cuda.synchronize()
    for i, results in enumerate(got):
        for a, b in zip(results, want[i % 2]):
            assert torch.equal(a, b)
