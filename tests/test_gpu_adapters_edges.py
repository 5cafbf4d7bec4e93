"""GPU: adapters of many requests (lora_adapters) where rows are taken 64 at a time, and with infinities."""

import math

import pytest
import torch

from tests.test_gpu_adapters import BF, _check, _inputs
from xorl_amd.functional import lora_adapters

pytestmark = pytest.mark.gpu


def _twice(a):
    out = lora_adapters(*a)
    _check(out, *a)
    assert torch.equal(lora_adapters(*a), out)                    # the same bits on every call
    return out


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("M,N,K,r", [(8191, 80, 320, 16), (8192, 64, 1088, 64), (8193, 48, 192, 33), (8193, 144, 1600, 8), (9001, 272, 704, 24), (9001, 64, 448, 48), (12345, 528, 64, 40),
                                     (8200, 1040, 576, 32)])
def test_many_rows(hip_device, M, N, K, r, dtype):
    for order, without in (("one", 0.0), ("runs", 0.1), ("mixed", 0.2)):
        _twice(_inputs(M, N, K, r, 3, dtype, M + r, hip_device, order, without))


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("r", [8, 24, 33, 64])
def test_pieces_of_a_window(hip_device, r, dtype):
    """An adapter in every choice of a window's four pieces, alone or beside another one or none, and in one row of a piece"""
    M = 8192 + 64 * 4 + 21
    a = list(_inputs(M, 96, 1088, r, 5, dtype, r, hip_device, without=0.0))
    piece = torch.arange(M, device=hip_device) // 16
    window, of = piece // 4, piece % 4
    inside = (window % 16) >> of & 1
    for rest in (-1, 2):
        a[4] = torch.where(inside == 1, 1 + 2 * (window % 2), rest).to(torch.int32)
        _twice(a)
    a[4] = torch.where((inside == 1) & (torch.arange(M, device=hip_device) % 16 == window % 16), 4, torch.where(of == 0, 0, -1)).to(torch.int32)
    _twice(a)


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("r", [6, 16, 24, 40, 64])
@pytest.mark.parametrize("M,K", [(1, 64), (5, 128), (60, 576), (300, 128), (1200, 704), (8200, 1088)])
def test_infinities_are_what_the_formula_makes_of_them(hip_device, M, K, r, dtype):
    base, x, A, Bm, ids, s = _inputs(M, 80, K, r, 8, dtype, M + r, hip_device, "mixed", 0.1, torch.int64)
    g = torch.Generator(device=hip_device).manual_seed(r)
    some = min(M, 3)
    if M > 1:
        ids[:min(M, 8)] = torch.arange(min(M, 8), device=hip_device)
    else:
        ids[0] = 3
    inf = math.inf
    x[some - 1, K // 3] = -inf                                    # (adapter 2, or 3 of one row)
    A[1, r - 1, K // 2] = inf
    A[6, 0, 1], A[6, r // 2, 2] = inf, -inf
    Bm[0, 5, r // 2] = -inf
    Bm[3, 17, 0] = inf
    Bm[3, 33] = torch.where(torch.rand(r, device=hip_device, generator=g) < 0.5, inf, -inf).to(dtype)
    Bm[7, 40:43, r - 1] = torch.tensor([inf, -inf, math.nan], device=hip_device).to(dtype)
    base[0, 7], base[0, 5] = inf, inf
    got = lora_adapters(base, x, A, Bm, ids, s)
    assert torch.equal(torch.nan_to_num(lora_adapters(base, x, A, Bm, ids, s), 77.0), torch.nan_to_num(got, 77.0))
    base, x, A, Bm, ids, s, got = (t.cpu() for t in (base, x, A, Bm, ids, s, got))
    rows = torch.cat([torch.nonzero(ids == a)[:20, 0] for a in range(8)]).tolist()
    for i in rows:
        a = int(ids[i])
        t = (A[a].double() * x[i].double()).sum(1) * s[a].double()
        want = base[i].double() + (Bm[a].double() * t).sum(1)
        y, known = got[i].double(), want.isfinite()
        assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y[want.isinf()], want[want.isinf()]), (i, a)
        if known.any() and bool(t.isfinite().all()):
            # as in _check: t to (K / 8 + 80) U and 2^-16 for fp32 factors, then r terms and one rounding to bf16
            U, own = 2.0 ** -24, 2.0 ** -16 if dtype == torch.float32 else 0.0
            S = (A[a].double() * x[i].double()).abs().sum(1) * s[a].double()
            Bk = Bm[a].double()[known].abs()
            bound = (Bk * (((K / 8 + 80) * U + own) * S)).sum(1) + (2.0 ** -16 + 2 * own + (r + 8) * U) * (Bk * t.abs()).sum(1) + 2 * U * (base[i].double().abs()[known] + want[known].abs())
            assert ((y - want)[known].abs() <= bound * (1 + 2.0 ** -8) + 2.0 ** -8 * want[known].abs()).all(), (i, a)
    none = ids < 0
    assert torch.equal(got[none], base[none])
