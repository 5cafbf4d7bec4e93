"""GPU: gradients of large embeddings, whose zeros are written before the rows that tokens have, and of more rows than 256 sorting blocks count."""

import math

import pytest
import torch

from tests.test_gpu_embedding import BF, _check_grad, _gen
from xorl_amd.embedding_functional import embedding

pytestmark = pytest.mark.gpu


def _runs(T, V, g, device):
    """tokens in any order that come 1 to 5, 16, 17, 33 or 400 times"""
    times = torch.tensor([1, 2, 3, 1, 4, 5, 1, 16, 2, 17, 3, 33, 1, 4, 400, 2, 5], device=device)
    ids = torch.randperm(V, device=device, generator=g)[:T].repeat_interleave(times.repeat(-(-T // times.numel()))[:T])[:T]
    return ids[torch.randperm(T, device=device, generator=g)]


def _gradient(w, ids, up, **kw):
    hole = torch.full_like(w, math.nan)                           # (what dW is likely to be made of: a row that is not written shows)
    del hole
    return torch.autograd.grad(embedding(ids, w, **kw), w, up)[0]


def _run(T, V, H, dtype, id_dtype, seed, device, scale, padding_idx, bad=True):
    g = _gen(device, seed)
    ids = _runs(T, V, g, device)
    if padding_idx is not None:
        ids[torch.rand(T, device=device, generator=g) < 0.1] = padding_idx % V
    if bad:
        at = torch.randperm(T, device=device, generator=g)
        ids[at[:T // 50 + 1]], ids[at[-1]] = -1, V
    w = torch.zeros(V, H, dtype=dtype, device=device, requires_grad=True)
    up = torch.randn(T, H, device=device, generator=g).to(dtype)
    ids = ids.to(id_dtype)
    dw = _gradient(w, ids, up, scale=scale, padding_idx=padding_idx)
    _check_grad(dw, ids, up, V, scale, padding_idx)
    assert torch.equal(dw, _gradient(w, ids, up, scale=scale, padding_idx=padding_idx))


# tokens, rows, columns: one and four tokens in a row of threads, 8 to 256 threads a token
LARGE = [(1, 131072, 1024), (777, 131072, 1024), (8191, 131072, 1024), (9001, 131072, 1024), (20011, 131072, 1032), (60001, 524288 + 3, 264), (140003, 2097152 + 7, 64), (5001, 66000, 2056)]


@pytest.mark.parametrize("scale,padding_idx", [(1.0, None), (-0.3, 0), (45.25, -1)])
@pytest.mark.parametrize("T,V,H", LARGE)
def test_zeros_first(hip_device, T, V, H, scale, padding_idx):
    assert V * H * 2 >= 256 << 20 and T < V // 2
    _run(T, V, H, BF, torch.int64, T + V, hip_device, scale, padding_idx)


@pytest.mark.parametrize("id_dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize("T,V,H", [(3, 70000, 1024), (4095, 70000, 1024), (4097, 70000, 1024), (30001, 131072, 516), (140003, 1048576 + 9, 68)])
def test_zeros_first_in_fp32(hip_device, T, V, H, id_dtype):
    assert V * H * 4 >= 256 << 20 and T < V // 2
    _run(T, V, H, torch.float32, id_dtype, T + V, hip_device, 1.5, 5)


@pytest.mark.parametrize("T", [1, 4097, 9000, 33003])
@pytest.mark.parametrize("V", [1 << 20, (1 << 20) + 1, (1 << 21) + 5])
def test_more_rows_than_256_blocks_count(hip_device, V, T):
    for dtype, H in ((BF, 8), (torch.float32, 5)):
        _run(T, V, H, dtype, torch.int32, T + V, hip_device, 1.0, None)


@pytest.mark.parametrize("V,H", [(131072, 1024), (70001, 2048)])
@pytest.mark.parametrize("T", [2999, 3000, 3001, 12000, 30000])
def test_one_token_in_a_large_vocabulary(hip_device, V, H, T):
    """More tokens of one sorting block than its list holds, at either end of the vocabulary and in the middle"""
    g = _gen(hip_device, T)
    up = torch.randn(T, H, device=hip_device, generator=g).to(BF)
    w = torch.zeros(V, H, dtype=BF, device=hip_device, requires_grad=True)
    for v in (0, V // 2, V - 1):
        ids = torch.full((T,), v, device=hip_device)
        _check_grad(_gradient(w, ids, up), ids, up, V, 1.0)
        ids[::3] = torch.randint(0, V, (len(ids[::3]),), device=hip_device, generator=g)
        _check_grad(_gradient(w, ids, up), ids, up, V, 1.0)
