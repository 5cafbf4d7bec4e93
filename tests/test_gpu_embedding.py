"""GPU: the embedding and its gradient by sorted tokens, against 64 bits.  U = 2^-24, half a step of fp32; B = 2^-8, half a step of bf16."""

import math

import pytest
import torch

from xorl_amd import _C
from xorl_amd.embedding_functional import embedding

pytestmark = pytest.mark.gpu
U, B, BF = 2.0 ** -24, 2.0 ** -8, torch.bfloat16


def _gen(device, seed):
    return torch.Generator(device=device).manual_seed(seed)


def _check_grad(dw, ids, grad, V, scale, padding_idx=None):
    """Sums of n terms in fp32 lose at most n U of their magnitudes, the scale and the result's rounding come once"""
    ids, g = ids.reshape(-1).long(), grad.reshape(-1, grad.shape[-1]).double()
    ok = (ids >= 0) & (ids < V)
    if padding_idx is not None:
        ok &= ids != padding_idx % V
    want = torch.zeros(V, g.shape[1], dtype=torch.float64, device=g.device).index_put_((ids[ok],), g[ok], accumulate=True)
    mag = torch.zeros_like(want).index_put_((ids[ok],), g[ok].abs(), accumulate=True)
    n = torch.bincount(ids[ok], minlength=V).double()[:, None]
    c = float(torch.tensor(scale, dtype=torch.float32))
    half = B if dw.dtype == BF else U
    bound = abs(c) * ((n + 1) * U * mag) * (1 + half) + half * (c * want).abs() + 2.0 ** -133
    assert dw.shape == want.shape and ((dw.double() - c * want).abs() <= bound).all()
    assert (dw[n[:, 0] == 0] == 0).all()


CASES = [(1, 1, 1), (1, 7, 3), (5, 3, 8), (64, 10, 64), (63, 1000, 33), (300, 50, 130), (1000, 2, 256), (2049, 517, 100), (4097, 1, 72), (777, 32003, 1024), (5000, 70001, 24), (3, 5, 2056)]


@pytest.mark.parametrize("padding_idx", [None, 0, -1])
@pytest.mark.parametrize("scale", [1.0, 45.25, -0.3])
@pytest.mark.parametrize("dtype,id_dtype", [(BF, torch.int64), (torch.float32, torch.int32)])
@pytest.mark.parametrize("T,V,H", CASES)
def test_forward_and_gradient(hip_device, T, V, H, dtype, id_dtype, scale, padding_idx):
    g = _gen(hip_device, T + V)
    w = torch.randn(V, H, device=hip_device, generator=g).to(dtype)
    # half the tokens by a power of their rank, so that some come often
    ids = torch.exp(torch.rand(T, device=hip_device, generator=g) * math.log(V + 0.5)).long().clamp(1, V) - 1
    ids = ids.to(id_dtype)
    want = (w[ids.long()].float() * scale).to(dtype)
    assert torch.equal(embedding(ids, w, scale=scale, padding_idx=padding_idx), want)
    w.requires_grad_(True)
    out = embedding(ids, w, scale=scale, padding_idx=padding_idx)
    assert torch.equal(out, want)
    up = torch.randn(T, H, device=hip_device, generator=g).to(dtype)
    dw, = torch.autograd.grad(out, w, up, retain_graph=True)
    assert dw.dtype == dtype
    _check_grad(dw, ids, up, V, scale, padding_idx)
    assert torch.equal(dw, torch.autograd.grad(out, w, up)[0])


def test_gradient_against_differences(hip_device):
    """The result is linear in the weight: a difference is the gradient but for the roundings"""
    g = _gen(hip_device, 1)
    w = torch.randn(9, 5, device=hip_device, generator=g, requires_grad=True)
    ids = torch.tensor([3, 3, 0, 8, 3, 1], device=hip_device)
    up = torch.randn(6, 5, device=hip_device, generator=g)
    dw, = torch.autograd.grad(embedding(ids, w, scale=2.0), w, up)
    for v in range(9):
        for h in range(5):
            step = torch.zeros_like(w)
            step[v, h] = 1.0
            with torch.no_grad():
                num = ((embedding(ids, w + step, scale=2.0) - embedding(ids, w - step, scale=2.0)).double() * up).sum() / 2
            assert abs(num - dw[v, h].double()) <= 64 * U * float(up.abs().sum()) * 4


@pytest.mark.parametrize("T", [1, 31, 32, 33, 64, 100, 1023, 4096, 20011])
@pytest.mark.parametrize("kind", ["all the same", "one among others", "two in turn", "every one once", "sorted", "reversed"])
def test_how_often_a_token_comes(hip_device, T, kind):
    V, H = 20011, 40
    at = torch.arange(T, device=hip_device)
    ids = {"all the same": torch.full((T,), 7, device=hip_device), "one among others": torch.where(at % 3 == 0, at % V, 12345), "two in turn": 100 + at % 2,
           "every one once": torch.randperm(V, device=hip_device, generator=_gen(hip_device, 3))[:T], "sorted": at // 3, "reversed": V - 1 - at // 5}[kind]
    w = torch.zeros(V, H, device=hip_device, dtype=BF, requires_grad=True)
    up = torch.randn(T, H, device=hip_device, generator=_gen(hip_device, T)).to(BF)
    dw, = torch.autograd.grad(embedding(ids, w), w, up)
    _check_grad(dw, ids, up, V, 1.0)


def test_the_same_bits_on_every_call(hip_device):
    g = _gen(hip_device, 5)
    w = torch.zeros(3000, 512, device=hip_device, requires_grad=True)
    ids = torch.randint(0, 3000, (9000,), device=hip_device, generator=g) % torch.randint(1, 3000, (9000,), device=hip_device, generator=g)
    up = torch.randn(9000, 512, device=hip_device, generator=g)
    first, = torch.autograd.grad(embedding(ids, w), w, up)
    for _ in range(5):
        assert torch.equal(first, torch.autograd.grad(embedding(ids, w), w, up)[0])


@pytest.mark.parametrize("id_dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_ids_out_of_range(hip_device, dtype, id_dtype):
    g = _gen(hip_device, 6)
    w = torch.randn(50, 24, device=hip_device, generator=g).to(dtype).requires_grad_(True)
    ids = torch.tensor([3, -1, 50, 49, 2 ** 31 - 1, -2 ** 31, 0, 3], device=hip_device).to(id_dtype)
    if id_dtype == torch.int64:
        ids[2], ids[5] = 2 ** 32 + 3, -2 ** 63
    out = embedding(ids, w)
    bad = torch.tensor([False, True, True, False, True, True, False, False], device=hip_device)
    assert out[bad].isnan().all() and torch.equal(out[~bad], w[ids[~bad].long()])
    up = torch.randn(8, 24, device=hip_device, generator=g).to(dtype)
    up[bad] = math.nan
    dw, = torch.autograd.grad(out, w, up)
    _check_grad(dw, ids, up.nan_to_num(0.0), 50, 1.0)


def test_what_is_no_number_stays_in_its_row(hip_device):
    w = torch.ones(20, 16, device=hip_device, dtype=BF, requires_grad=True)
    ids = torch.arange(100, device=hip_device) % 20
    up = torch.ones(100, 16, device=hip_device, dtype=BF)
    up[25, 3], up[46, 4] = math.nan, math.inf
    dw, = torch.autograd.grad(embedding(ids, w), w, up)
    assert dw[5, 3].isnan() and dw[6, 4] == math.inf
    dw[5, 3], dw[6, 4] = 5.0, 5.0
    assert (dw == 5.0).all()


def test_no_tokens(hip_device):
    w = torch.randn(11, 24, device=hip_device, requires_grad=True)
    out = embedding(torch.zeros(2, 0, 3, dtype=torch.int64, device=hip_device), w)
    assert out.shape == (2, 0, 3, 24)
    dw, = torch.autograd.grad(out, w, torch.zeros_like(out))
    assert dw.shape == w.shape and (dw == 0).all()


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("H", [16, 30, 136])
def test_layouts(hip_device, H, dtype):
    g = _gen(hip_device, 8)
    w = torch.randn(40, H, device=hip_device, generator=g).to(dtype)
    ids = torch.randint(0, 40, (6, 5), device=hip_device, generator=g)
    up = torch.randn(6, 5, H, device=hip_device, generator=g).to(dtype)
    ref = w.clone().requires_grad_(True)
    want = embedding(ids, ref, scale=1.5)
    dwant, = torch.autograd.grad(want, ref, up)
    wide = torch.full((40, H + 3), math.nan, dtype=dtype, device=hip_device)
    wide[:, 2:2 + H] = w
    weights = {"slice": wide[:, 2:2 + H], "transposed": w.t().contiguous().t(), "off by one": torch.cat([w.new_zeros(1), w.reshape(-1)])[1:].view(40, H)}
    for name, v in weights.items():
        leaf = v.detach().requires_grad_(True)
        out = embedding(ids.t().contiguous().t(), leaf, scale=1.5)
        wide_up = torch.full((6, 5, H + 1), math.nan, dtype=dtype, device=hip_device)
        wide_up[..., 1:] = up
        assert torch.equal(out, want), name
        assert torch.equal(torch.autograd.grad(out, leaf, wide_up[..., 1:], retain_graph=True)[0], dwant), name
        assert torch.equal(torch.autograd.grad(out, leaf, up.transpose(0, 1).contiguous().transpose(0, 1))[0], dwant), name
    out = embedding(ids, ref, scale=1.5)
    ones, = torch.autograd.grad(out, ref, torch.ones_like(out), retain_graph=True)
    assert torch.equal(ones, torch.autograd.grad(out.sum(), ref, retain_graph=True)[0])
    assert torch.equal(torch.autograd.grad(out, ref, up[:1, :1].expand_as(out), retain_graph=True)[0],
                       torch.autograd.grad(out, ref, up[:1, :1].expand_as(out).contiguous())[0])
    one = embedding(ids[0, 0], w)
    assert one.shape == (H,) and torch.equal(one, w[ids[0, 0]])


def test_more_elements_than_32_bits_count(hip_device):
    V, H = 131072 + 5, 32776
    assert V * H > 1 << 32
    w = torch.zeros(V, H, dtype=BF, device=hip_device)
    w[-1] = torch.randn(H, device=hip_device, generator=_gen(hip_device, 9)).to(BF)
    w.requires_grad_(True)
    ids = torch.tensor([V - 1, 0, V - 1, V - 2], device=hip_device)
    out = embedding(ids, w)
    assert torch.equal(out[0], w[-1]) and torch.equal(out[2], w[-1]) and (out[1] == 0).all()
    up = torch.randn(4, H, device=hip_device, generator=_gen(hip_device, 10)).to(BF)
    dw, = torch.autograd.grad(out, w, up)
    assert torch.equal(dw[-1], (up[0].float() + up[2].float()).to(BF)) and torch.equal(dw[-2], up[3]) and torch.equal(dw[0], up[1])
    assert torch.count_nonzero(dw[1:-2]) == 0


def test_more_tokens_than_32_bits_of_elements(hip_device):
    T, H = 131072 + 3, 32776
    ids = torch.arange(T, device=hip_device) % 7
    w = torch.randn(7, H, device=hip_device, generator=_gen(hip_device, 11)).to(BF).requires_grad_(True)
    out = embedding(ids, w)
    assert out.numel() > 1 << 32 and torch.equal(out[-3:], w[ids[-3:]])
    up = torch.zeros(T, H, dtype=BF, device=hip_device)
    up[-1], up[-8] = 1.0, 2.0
    dw, = torch.autograd.grad(out, w, up)
    assert (dw[ids[-1]] == 3.0).all() and torch.count_nonzero(dw) == H


def test_another_stream(hip_device):
    w = torch.randn(500, 256, device=hip_device, requires_grad=True)
    ids = torch.randint(0, 500, (3000,), device=hip_device)
    up = torch.randn(3000, 256, device=hip_device)
    want = embedding(ids, w)
    dwant, = torch.autograd.grad(want, w, up)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        leaf = w.detach().clone().requires_grad_(True)
        out = embedding(ids.clone(), leaf)
        dw, = torch.autograd.grad(out, leaf, up)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, want) and torch.equal(dw, dwant)


def test_captured_forward_and_backward(hip_device):
    w = torch.randn(700, 128, device=hip_device, requires_grad=True)
    ids = torch.randint(0, 700, (900,), device=hip_device)
    up = torch.randn(900, 128, device=hip_device)
    graphs, got = [], []
    for k in range(2):                       # two graphs side by side: neither's scratch is the other's
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            out = embedding(ids, w, scale=1.0 + k, padding_idx=3)
            got.append((out.detach(), torch.autograd.grad(out, w, up)[0]))
    for seed in range(3):
        ids.copy_(torch.randint(0, 700 >> (4 * seed), (900,), device=hip_device))
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for k in range(2):
            leaf = w.detach().clone().requires_grad_(True)
            out = embedding(ids, leaf, scale=1.0 + k, padding_idx=3)
            assert torch.equal(got[k][0], out) and torch.equal(got[k][1], torch.autograd.grad(out, leaf, up)[0])


def test_capture_beside_a_living_result_is_refused(hip_device):
    w = torch.randn(70, 16, device=hip_device, requires_grad=True)
    ids = torch.randint(0, 70, (90,), device=hip_device)
    up = torch.randn(90, 16, device=hip_device)
    eager = embedding(ids, w)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="another stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(embedding(ids, w), w, up)
    torch.cuda.synchronize()
    _check_grad(torch.autograd.grad(eager, w, up)[0], ids, up, 70, 1.0)


class _Weight(torch.nn.Parameter):
    pass


def test_subclasses_take_the_python_path(hip_device):
    p = _Weight(torch.randn(70, 16, device=hip_device))
    w = p.detach().as_subclass(torch.Tensor).clone().requires_grad_(True)
    ids = torch.randint(0, 70, (90,), device=hip_device)
    up = torch.randn(90, 16, device=hip_device)
    a, b = embedding(ids, p, scale=3.0, padding_idx=-2), embedding(ids, w, scale=3.0, padding_idx=-2)
    assert torch.equal(a, b) and torch.equal(torch.autograd.grad(a, p, up)[0], torch.autograd.grad(b, w, up)[0])
    with pytest.raises(RuntimeError, match="no subclasses"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(embedding(ids, p), p, up)
    torch.cuda.synchronize()


def test_under_torch_compile(hip_device):
    w = torch.randn(70, 16, device=hip_device, requires_grad=True)
    ids = torch.randint(0, 70, (9, 10), device=hip_device)
    up = torch.randn(9, 10, 16, device=hip_device)
    a, b = torch.compile(lambda i, t: embedding(i, t, scale=3.0, padding_idx=5), backend="aot_eager", fullgraph=True)(ids, w), embedding(ids, w, scale=3.0, padding_idx=5)
    assert torch.equal(a, b) and torch.equal(torch.autograd.grad(a, w, up)[0], torch.autograd.grad(b, w, up)[0])


def test_changes_in_place_and_second_derivatives_are_refused(hip_device):
    w = torch.randn(70, 16, device=hip_device, requires_grad=True)
    ids = torch.randint(0, 70, (90,), device=hip_device)
    up = torch.randn(90, 16, device=hip_device, requires_grad=True)
    out = embedding(ids, w)
    dw, = torch.autograd.grad(out, w, up, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        dw.sum().backward()
    out = embedding(ids, w)
    ids.clamp_(max=3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, w, up.detach())
    out = embedding(ids, w)
    ids.data = torch.zeros(3, dtype=torch.int64, device=hip_device)
    with pytest.raises(RuntimeError, match="freed, resized or exchanged"):
        torch.autograd.grad(out, w, up.detach())


def test_tangents_transforms_and_devices_are_refused(hip_device):
    import torch.autograd.forward_ad as fwAD

    w = torch.randn(70, 16, device=hip_device)
    ids = torch.randint(0, 70, (90,), device=hip_device)
    for grad in (True, False):
        with fwAD.dual_level(), torch.set_grad_enabled(grad), pytest.raises(NotImplementedError):
            embedding(ids, fwAD.make_dual(w, torch.ones_like(w)))
    for f in (lambda: torch.func.jvp(lambda a: embedding(ids, a), (w,), (torch.ones_like(w),)), lambda: torch.func.grad(lambda a: embedding(ids, a).sum())(w),
              lambda: torch.vmap(lambda a: embedding(ids, a))(w[None])):
        with pytest.raises((RuntimeError, NotImplementedError)):
            f()
    with pytest.raises(RuntimeError, match="HIP device only"):
        embedding(ids.cpu(), w)
    with pytest.raises(_C.XqError, match="bf16 or fp32"):
        embedding(ids, w.half())
