"""GPU: choices of experts (moe_route) that single precision cannot tell, next to the last place and between groups."""

import math

import pytest
import torch

from xorl_amd.moe_functional import moe_route

pytestmark = pytest.mark.gpu
LOWEST = torch.finfo(torch.float32).min


def _order(z, k, scoring, bias):
    """ids in 64 bits: a stable sort leaves equal experts in the order of their index"""
    z = z.double().cpu()
    s = torch.sigmoid(z) if scoring == "sigmoid" else torch.softmax(z, 1)
    return (s + bias.double().cpu()).sort(dim=1, descending=True, stable=True)[1][:, :k]


# scoring, equal logits, a larger one whose score is the same in 32 bits, the rest, whether an expert with logit 0 goes first
NEAR = [("sigmoid", 18.0, 19.0, -3.0, False), ("sigmoid", 16.0, 16.125, -3.0, False), ("sigmoid", 20.0, 20.125, -3.0, False), ("sigmoid", 32.0, 33.0, 0.5, False),
        ("sigmoid", -100.0, -90.0, -110.0, False), ("softmax", -100.0, -90.0, -110.0, True)]
# rows and experts by how many lanes and values a lane a row has
SHAPES = [(5, 8), (33, 60), (7, 100), (2100, 200), (3, 200), (2, 400), (3, 1000)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,E", SHAPES)
@pytest.mark.parametrize("scoring,low,high,rest,front", NEAR)
def test_equal_experts_on_both_sides_of_the_last_place(hip_device, scoring, low, high, rest, front, T, E, dtype):
    """The last chosen and the first left out have the same logit and bias, and an expert behind them a larger one that 32 bits do not tell from theirs"""
    g = torch.Generator().manual_seed(T + E)
    for equal in (2, 3, 5, 14, 40, 70, 120):               # (so many that the lists of a row are short, long, or none)
        if equal + 2 > E:
            continue
        z = torch.full((T, E), rest)
        at = torch.rand(T, E, generator=g).argsort(1)[:, :equal + 1].sort(1)[0]
        z.scatter_(1, at, low)
        z.scatter_(1, at[:, -1:], high)
        if front:
            z.scatter_(1, (at[:, :1] + 1) % E, 0.0)        # (may take the place of one of the equal ones)
        z = z.to(dtype).to(hip_device)
        for bias in (torch.zeros(E), torch.full((E,), 0.25), -0.001 * torch.arange(E).remainder(2)):
            for k in sorted({1, 2, min(equal - 1, 15), min(equal, 16), min(equal, 32)}):
                _, ids = moe_route(z, k, scoring=scoring, bias=bias.to(hip_device))
                assert torch.equal(ids.cpu(), _order(z, k, scoring, bias)), (equal, k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,E", SHAPES)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_biases_as_small_as_scores_that_are_no_fp32_numbers(hip_device, scoring, T, E, dtype):
    g = torch.Generator().manual_seed(E)
    z = (-94 + 10 * torch.rand(T, E, generator=g)).to(dtype)
    if scoring == "softmax":
        z[:, 1] = 0.0
    bias = 1e-38 * torch.randn(E, generator=g)
    for k in (1, 2, 8):
        _, ids = moe_route(z.to(hip_device), k, scoring=scoring, bias=bias.to(hip_device))
        assert torch.equal(ids.cpu(), _order(z, k, scoring, bias)), k
    if E % 4 == 0:                                         # groups by the sum of their two best, the best two of four
        s = torch.sigmoid(z.double()) if scoring == "sigmoid" else torch.softmax(z.double(), 1)
        c = (s + bias.double()).view(T, 4, E // 4)
        best = c.sort(dim=2, descending=True)[0]
        kept = (best[..., 0] + (best[..., 1] if E > 4 else 0.0)).sort(dim=1, descending=True, stable=True)[1][:, :2]
        out = torch.ones(T, 4, dtype=torch.bool).scatter_(1, kept, False)
        want = c.masked_fill(out[:, :, None], -math.inf).view(T, E).sort(dim=1, descending=True, stable=True)[1][:, :4]
        _, ids = moe_route(z.to(hip_device), 4, scoring=scoring, bias=bias.to(hip_device), num_groups=4, top_groups=2, group_score="sum2")
        assert torch.equal(ids.cpu(), want)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E", [(4096, 256), (300, 128), (3, 1024)])
def test_a_router_that_starts_at_zero(hip_device, T, E, scoring):
    z, bias = torch.zeros(T, E, device=hip_device), torch.zeros(E, device=hip_device)
    _, ids = moe_route(z, 8, scoring=scoring, bias=bias)
    assert torch.equal(ids, torch.arange(8, device=hip_device).expand(T, 8))


@pytest.mark.parametrize("size", [2, 4, 6])
@pytest.mark.parametrize("T", [1, 70, 3000])
@pytest.mark.parametrize("groups", [4, 32])
def test_groups_of_biases_whose_sum_is_no_fp32_number(hip_device, groups, T, size):
    """Two scores with a bias near the type's lowest value make a strength below every fp32 number; a group without experts is weaker still"""
    E = groups * size
    z = torch.randn(T, E, generator=torch.Generator().manual_seed(T + E)).to(hip_device)
    bias = torch.full((groups, size), -math.inf)
    bias[1] = LOWEST
    bias[2] = 0.75 * LOWEST
    bias[3] = 0.0
    at = {g: list(range(g * size, (g + 1) * size)) for g in range(4)}
    b = bias.view(-1).to(hip_device)

    def rows(order, k):
        return torch.tensor((order + [-1] * k)[:k], device=hip_device).expand(T, k)

    first = z[:, at[3]].sort(dim=1, descending=True, stable=True)[1] + at[3][0]
    for top_groups, behind in ((1, []), (2, at[2]), (3, at[2] + at[1]), (4, at[2] + at[1])):
        k = min(32, top_groups * size)
        _, ids = moe_route(z, k, scoring="sigmoid", bias=b, num_groups=groups, top_groups=top_groups, group_score="sum2")
        assert torch.equal(ids, torch.cat([first, rows(behind, k - size)], 1)), top_groups
    b[at[3][0]:at[3][-1] + 1] = -math.inf
    _, ids = moe_route(z, size, scoring="sigmoid", bias=b, num_groups=groups, top_groups=1, group_score="sum2")
    assert torch.equal(ids, rows(at[2], size))
