"""GPU: adapters of many requests beside one projection (lora_adapters, qlora_adapters_forward) against 64 bits.

U = 2^-24, half a step of fp32; B = 2^-8, half a step of bf16."""

import math

import pytest
import torch

from tests.util_cases import make_dense_module
from xorl_amd import _C
from xorl_amd.functional import lora_adapters, qlora_linear
from xorl_amd.qlora import qlora_adapters_forward

pytestmark = pytest.mark.gpu
U, B, BF = 2.0 ** -24, 2.0 ** -8, torch.bfloat16


def _inputs(M, N, K, r, n, dtype, seed, device, order="mixed", without=0.2, id_dtype=torch.int32):
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(M, K, device=device, generator=g).to(BF)
    base = torch.randn(M, N, device=device, generator=g).to(BF)
    A = (torch.randn(n, r, K, device=device, generator=g) * K ** -0.5).to(dtype)
    Bm = (torch.randn(n, N, r, device=device, generator=g) * 0.3).to(dtype)
    ids = torch.randint(0, max(n, 1), (M,), device=device, generator=g)
    if order == "runs":
        ids = ids.sort().values
    elif order == "prompts":
        ids = ids[::max(1, M // 7)].repeat_interleave(max(1, M // 7))[:M]
    elif order == "one":
        ids[:] = max(n - 1, 0)
    ids[torch.rand(M, device=device, generator=g) < without] = -1
    return base, x, A, Bm, ids.to(id_dtype), 0.5 + torch.rand(n, device=device, generator=g)


def _check(out, base, x, A, Bm, ids, s):
    """x A^T sums K products in fp32 ((K / 8 + 80) U of the magnitudes, whatever the order) and enters the second product with 16 bits, as fp32 factors do in both
    (2^-16 each); the second product sums r terms and adds the base ((r + 8) U); the result is rounded once"""
    K, r, n = x.shape[-1], A.shape[1], A.shape[0]
    own = 2.0 ** -16 if A.dtype == torch.float32 else 0.0
    x2, o2, b2, i1 = x.reshape(-1, K).double(), out.reshape(-1, out.shape[-1]).double(), base.reshape(-1, base.shape[-1]), ids.reshape(-1).long()
    assert out.dtype == BF and out.shape == base.shape
    has = (i1 >= 0) & (i1 < n)
    assert torch.equal(out.reshape(b2.shape)[~has], b2[~has])
    for a in i1[has].unique().tolist():
        rows = torch.nonzero(i1 == a)[:, 0]
        Ad, Bd, c = A[a].double(), Bm[a].double(), float(s[a])
        t, S = x2[rows] @ Ad.t(), x2[rows].abs() @ Ad.abs().t()
        want = b2[rows].double() + c * (t @ Bd.t())
        err_t = ((K / 8 + 80) * U + own) * S
        bound = c * (err_t @ Bd.abs().t() + (2.0 ** -16 + 2 * own + (r + 8) * U) * (t.abs() @ Bd.abs().t())) + 2 * U * (b2[rows].double().abs() + want.abs())
        bound = bound * (1 + B) + B * want.abs()
        assert ((o2[rows] - want).abs() <= bound).all(), (a, float(((o2[rows] - want).abs() / bound).max()))


CASES = [  # M, N, K, r, n
    (1, 16, 64, 1, 1), (1, 4096, 4096, 16, 8), (2, 48, 128, 3, 2), (7, 1040, 320, 8, 3), (16, 512, 1024, 16, 1), (17, 256, 192, 24, 5), (48, 1024, 4096, 32, 64), (64, 272, 448, 64, 9),
    (100, 96, 576, 13, 4), (257, 2064, 256, 16, 6), (513, 144, 2112, 40, 3), (1023, 64, 64, 7, 20), (1025, 304, 704, 16, 5), (2049, 528, 832, 33, 4), (3001, 32, 128, 64, 11), (5000, 1008, 64, 16, 1)]


@pytest.mark.parametrize("order", ["mixed", "runs", "prompts", "one"])
@pytest.mark.parametrize("dtype,id_dtype", [(BF, torch.int32), (torch.float32, torch.int64)])
@pytest.mark.parametrize("M,N,K,r,n", CASES)
def test_adapters(hip_device, M, N, K, r, n, dtype, id_dtype, order):
    a = _inputs(M, N, K, r, n, dtype, M + r, hip_device, order, 0.0 if M == 1 else 0.2, id_dtype)
    out = lora_adapters(*a)
    _check(out, *a)
    assert torch.equal(out, lora_adapters(*a))                    # the same bits on every call
    base = a[0].clone()
    assert lora_adapters(base, *a[1:], out=base) is not None and torch.equal(base, out)


def test_more_adapters_than_a_launch_has_threads(hip_device):
    a = _inputs(1500, 32, 64, 4, 5000, BF, 1, hip_device)
    _check(lora_adapters(*a), *a)


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("M", [15, 16, 33, 64, 65, 255, 256, 511, 512, 513, 1024])
def test_where_rows_change_their_tiles(hip_device, M, dtype):
    """Each way that rows become tiles, up to its last row: every row its own adapter, all of one, in turn, 16 of each, 17 of each, none and one"""
    a = list(_inputs(M, 272, 128, 24, M, dtype, M, hip_device, without=0.0))
    i = torch.arange(M, device=hip_device)
    for ids in (i, i.flip(0), i * 0, i % 2, i % 5, i // 16, i // 17, i % 17 - 1, torch.where(i == M - 1, 3, -1), torch.where(i < M - 1, 3, -1)):
        a[4] = ids.to(torch.int64)
        out = lora_adapters(*a)
        _check(out, *a)
        assert torch.equal(lora_adapters(*a), out)


def test_no_adapters_and_no_rows(hip_device):
    a = _inputs(20, 32, 64, 4, 3, BF, 2, hip_device)
    none = lora_adapters(a[0], a[1], a[2][:0], a[3][:0], a[4], a[5][:0])
    assert torch.equal(none, a[0])
    all_off = lora_adapters(*a[:4], torch.full_like(a[4], -1), a[5])
    assert torch.equal(all_off, a[0])
    assert lora_adapters(a[0][:0], a[1][:0], *a[2:4], a[4][:0], a[5]).shape == (0, 32)


@pytest.mark.parametrize("M", [40, 1500])
def test_ids_that_are_no_adapters(hip_device, M):
    a = list(_inputs(M, 32, 64, 4, 3, BF, 3, hip_device, id_dtype=torch.int64))
    odd = torch.tensor([-1, 3, 2 ** 31, 2 ** 32, 2 ** 32 + 1, -2 ** 32, -2 ** 63, 2 ** 63 - 1, 0, 2], device=hip_device)
    a[4] = odd.repeat(M // 10)
    _check(lora_adapters(*a), *a)
    a[4] = a[4].clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32)
    _check(lora_adapters(*a), *a)


@pytest.mark.parametrize("M", [5, 60, 1200])
def test_what_is_no_number_stays_with_its_rows(hip_device, M):
    a = _inputs(M, 48, 128, 6, 4, BF, 4, hip_device, "mixed", 0.3)
    base, x, A, Bm, ids, s = (t.clone() for t in a)
    ids[0], ids[1], ids[2] = 0, 1, -1
    want = lora_adapters(base, x, A, Bm, ids, s)
    A[3, 2, 5] = math.nan
    Bm[2, 7, 1] = math.inf
    x[1, 3] = math.nan
    base[2, 4] = math.inf
    got = lora_adapters(base, x, A, Bm, ids, s)
    clean = (ids != 3) & (ids != 2)
    clean[1] = clean[2] = False
    assert torch.equal(got[clean], want[clean])
    assert got[1].isnan().all() and got[ids == 3].isnan().all() and got[2, 4] == math.inf and not got[ids == 2][:, 7].isfinite().any()
    rest = torch.arange(48, device=hip_device) != 7
    assert torch.equal(got[ids == 2][:, rest], want[ids == 2][:, rest])


def test_zeros_keep_their_sign_without_an_adapter(hip_device):
    a = list(_inputs(4, 16, 64, 4, 3, BF, 5, hip_device))
    a[0] = torch.full_like(a[0], -0.0)
    a[4] = torch.tensor([-1, -1, 7, 1], dtype=torch.int32, device=hip_device)
    assert torch.signbit(lora_adapters(*a)[:3]).all()


@pytest.mark.parametrize("M", [30, 1200])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_layouts(hip_device, M, dtype):
    base, x, A, Bm, ids, s = _inputs(M, 32, 64, 5, 4, dtype, 6, hip_device)
    want = lora_adapters(base, x, A, Bm, ids, s)

    def wide(t, left, right):
        w = torch.full((t.shape[0], t.shape[1] + left + right), math.nan, dtype=t.dtype, device=t.device)
        w[:, left:left + t.shape[1]] = t
        return w[:, left:left + t.shape[1]]

    for name, (b, y) in {"slices": (wide(base, 8, 16), wide(x, 16, 8)), "odd slices": (wide(base, 1, 0), wide(x, 3, 2)),
                         "transposed": (base.t().contiguous().t(), x.t().contiguous().t())}.items():
        assert torch.equal(lora_adapters(b, y, A, Bm, ids, s), want), name
    off = torch.cat([A.new_zeros(1), A.reshape(-1)])[1:].view(A.shape)
    assert torch.equal(lora_adapters(base, x, off, Bm.transpose(1, 2).contiguous().transpose(1, 2), torch.stack([ids, ids], 1)[:, 0], torch.stack([s, s], 1)[:, 1]), want)
    three = lora_adapters(base.view(2, -1, 32), x.view(2, -1, 64), A, Bm, ids.view(2, -1), s)
    assert torch.equal(three.view(-1, 32), want)
    one = lora_adapters(base[0], x[0], A, Bm, ids[0], s)
    assert one.shape == (32,) and torch.equal(one, lora_adapters(base[:1], x[:1], A, Bm, ids[:1], s)[0])
    same = lora_adapters(base[:1].expand(M, 32), x[:1].expand(M, 64), A, Bm, ids, s)
    assert torch.equal(same, lora_adapters(base[:1].repeat(M, 1), x[:1].repeat(M, 1), A, Bm, ids, s))


def test_results_in_place_and_elsewhere(hip_device):
    base, x, A, Bm, ids, s = _inputs(50, 32, 64, 5, 4, BF, 7, hip_device)
    want = lora_adapters(base, x, A, Bm, ids, s)
    out = torch.full((50, 40), 9.0, dtype=BF, device=hip_device)
    got = lora_adapters(base, x, A, Bm, ids, s, out=out[:, :32])
    assert torch.equal(got, want) and got.data_ptr() == out.data_ptr() and (out[:, 32:] == 9.0).all()
    strip = torch.full((50, 48), 9.0, dtype=BF, device=hip_device)
    strip[:, 8:40] = base
    view = strip[:, 8:40]
    version = view._version
    lora_adapters(view, x, A, Bm, ids, s, out=view)
    assert torch.equal(view, want) and view._version == version + 1 and (strip[:, :8] == 9.0).all() and (strip[:, 40:] == 9.0).all()
    for bad in (torch.empty(50, 33, dtype=BF, device=hip_device)[:, 1:], torch.empty(50, 32, device=hip_device), torch.empty(49, 32, dtype=BF, device=hip_device),
                torch.empty(32, 50, dtype=BF, device=hip_device).t()):
        with pytest.raises(_C.XqError, match="out must be"):
            lora_adapters(base, x, A, Bm, ids, s, out=bad)
    both = torch.empty(51, 32, dtype=BF, device=hip_device)
    with pytest.raises(_C.XqError, match="shares memory"):
        lora_adapters(both[:-1], x, A, Bm, ids, s, out=both[1:])
    wide = torch.empty(50, 96, dtype=BF, device=hip_device)
    with pytest.raises(_C.XqError, match="shares memory"):
        lora_adapters(wide[:, :32], wide[:, 32:], A, Bm, ids, s, out=wide[:, :32])
    with pytest.raises(_C.XqError, match="16 bytes"):
        odd = torch.empty(50, 33, dtype=BF, device=hip_device)[:, :32]
        lora_adapters(odd, x, A, Bm, ids, s, out=odd)


def test_more_elements_than_32_bits_count(hip_device):
    M, N = (1 << 18) + 5, 16400
    assert M * N > 1 << 32
    base = torch.zeros(M, N, dtype=BF, device=hip_device)
    x = torch.zeros(M, 64, dtype=BF, device=hip_device)
    _, xt, A, Bm, _, s = _inputs(6, N, 64, 4, 3, BF, 8, hip_device)
    ids = torch.full((M,), -1, dtype=torch.int32, device=hip_device)
    tail = torch.tensor([0, 2, 1, -1, 2, 2], dtype=torch.int32, device=hip_device)
    x[-6:], ids[-6:], base[0] = xt, tail, 1.0
    lora_adapters(base, x, A, Bm, ids, s, out=base)
    _check(base[-6:], torch.zeros_like(base[-6:]), xt, A, Bm, tail, s)
    assert (base[0] == 1.0).all() and torch.count_nonzero(base[1:200]) == 0


def test_a_bank_of_more_elements_than_32_bits_count(hip_device):
    n, r, K, N = 1100, 64, 65536, 64
    A = torch.zeros(n, r, K, dtype=BF, device=hip_device)
    assert A.numel() > 1 << 32
    base, x, At, Bm, ids, s = _inputs(20, N, K, r, 2, BF, 9, hip_device, without=0.0)
    A[-2:] = At
    full = torch.zeros(n, N, r, dtype=BF, device=hip_device)
    full[-2:] = Bm
    scale = torch.ones(n, device=hip_device)
    scale[-2:] = s
    assert torch.equal(lora_adapters(base, x, A, full, ids + (n - 2), scale), lora_adapters(base, x, At, Bm, ids, s))


@pytest.mark.parametrize("M", [40, 1300])
def test_another_stream_and_captured_graphs(hip_device, M):
    a = _inputs(M, 256, 256, 16, 6, BF, 10, hip_device)
    want = lora_adapters(*a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = lora_adapters(*(t.clone() for t in a))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for k, g in enumerate(graphs):                  # two graphs whose scratch is their own
        with torch.cuda.graph(g):
            outs.append(lora_adapters(a[0], a[1], a[2], a[3], a[4], a[5] * (k + 1)))
    for seed in range(3):
        b = _inputs(M, 256, 256, 16, 6, BF, 20 + seed, hip_device, ("mixed", "runs", "one")[seed])
        for t, v in zip(a, b):
            t.copy_(v)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for k, out in enumerate(outs):
            assert torch.equal(out, lora_adapters(*b[:5], b[5] * (k + 1)))


class _Factor(torch.nn.Parameter):
    pass


def test_subclasses_compiled_calls_and_gradients(hip_device):
    a = _inputs(30, 32, 64, 5, 4, torch.float32, 11, hip_device)
    want = lora_adapters(*a)
    assert torch.equal(lora_adapters(*a[:2], _Factor(a[2], requires_grad=False), *a[3:]), want)
    assert torch.equal(torch.compile(lora_adapters, backend="aot_eager", fullgraph=True)(*a), want)
    grads = [t.clone().requires_grad_(True) if t.is_floating_point() else t for t in a]
    with pytest.raises(_C.XqError, match="forward-only"):
        lora_adapters(*grads)
    with torch.no_grad():
        assert torch.equal(lora_adapters(*grads), want)
    with torch.inference_mode():
        base = a[0].clone()
        assert torch.equal(lora_adapters(base, *a[1:], out=base), want)


# ---------------------------------------------------------------- beside a packed projection
@pytest.mark.parametrize("fmt", ["block_fp8", "int4", "nvfp4", "nf4"])
@pytest.mark.parametrize("M", [1, 12, 200, 1500])
def test_beside_a_packed_projection(hip_device, fmt, M):
    m, _ = make_dense_module(fmt, 256, 512, 8, 16, seed=3, device=hip_device)
    _, x, A, Bm, ids, s = _inputs(M, 256, 512, 16, 5, BF, 12, hip_device)
    with torch.no_grad():
        base = qlora_linear(x, m._forward_quant_weight(), None, None, 0, 0.0, None)
        got = qlora_adapters_forward(m, x, A, Bm, ids, s)
    _check(got, base, x, A, Bm, ids, s)
    if M > 1:
        with pytest.raises(_C.XqError, match="forward-only"):
            qlora_adapters_forward(m, x.clone().requires_grad_(True), A, Bm, ids, s)


def test_a_bank_with_the_modules_own_factors(hip_device):
    """A request on the module's own adapter: the two forms of the low-rank term agree to its roundings (the module keeps x A^T and B in bf16: 3 B of the term)"""
    m, _ = make_dense_module("block_fp8", 256, 512, 8, 16, seed=4, device=hip_device)
    with torch.no_grad():
        m.lora_B.normal_(std=0.05)
        x = torch.randn(9, 512, device=hip_device).to(BF)
        bank_A, bank_B = m.lora_A.detach()[None, :8], m.lora_B.detach()[None, :, :8]
        got = qlora_adapters_forward(m, x, bank_A, bank_B, torch.zeros(9, dtype=torch.int32, device=hip_device), torch.full((1,), float(m.scaling), device=hip_device))
        term = (m.scaling * (x.double().abs() @ bank_A[0].double().t().abs()) @ bank_B[0].double().t().abs())
        want = m(x)
        assert ((got.double() - want.double()).abs() <= 2 * B * (got.double().abs() + want.double().abs()) + 4 * B * term).all()
