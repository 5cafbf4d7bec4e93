"""GPU: the choice of experts (moe_route) against the definition in 64 bits, its gradient, its masks, ties and borders, its layouts and streams.

U = 2^-24, half a step of fp32; B = 2^-8, half a step of bf16."""

import math

import pytest
import torch

from xorl_amd import _C
from xorl_amd.moe_functional import moe_route

pytestmark = pytest.mark.gpu
U, B, BF = 2.0 ** -24, 2.0 ** -8, torch.bfloat16


def reference(z, k, scoring="softmax", bias=None, num_groups=1, top_groups=1, group_score="sum2", renormalize=True, scale=1.0):
    """(weights, ids, scores) in 64 bits on the CPU, a row and a comparison at a time; rows without NaN"""
    z = z.detach().double().cpu().reshape(-1, z.shape[-1])
    T, E = z.shape
    s = torch.sigmoid(z) if scoring == "sigmoid" else torch.softmax(z, 1).nan_to_num(0.0)
    b = None if bias is None else bias.double().cpu()
    c = z if b is None else s + b
    h = s if b is None and group_score == "sum2" else c
    ids, w = torch.full((T, k), -1), torch.zeros(T, k, dtype=torch.float64)
    for t in range(T):
        out = [z[t, e] == -math.inf or (b is not None and b[e] == -math.inf) for e in range(E)]
        allowed = range(E)
        if top_groups < num_groups:
            size = E // num_groups
            strength = []
            for g in range(num_groups):
                best = sorted((h[t, e].item() for e in range(g * size, (g + 1) * size) if not out[e]), reverse=True)
                strength.append(-math.inf if not best else best[0] + (best[1] if group_score == "sum2" and len(best) > 1 else 0.0))
            kept = set(sorted(range(num_groups), key=lambda g: (-strength[g], g))[:top_groups])
            allowed = [e for e in range(E) if e // size in kept]
        order = sorted((e for e in allowed if not out[e]), key=lambda e: (-c[t, e].item(), e))[:k]
        ids[t, :len(order)] = torch.tensor(order, dtype=torch.int64)
        picked = s[t, order]
        w[t, :len(order)] = scale * (picked / picked.sum() if renormalize and len(order) else picked)
    return w, ids, s


def gradient(z, up, w, ids, s, scoring, renormalize, scale):
    """dz, and the magnitudes that its terms have, by the formula in 64 bits"""
    up = up.double().cpu().reshape(ids.shape)
    is_ = ids >= 0
    at = ids.clamp(min=0)
    g, sel = scale * up * is_, s.gather(1, at) * is_
    u = w / scale
    if renormalize:
        d, m = u * (g - (g * u).sum(1, keepdim=True)), u * (g.abs() + (g * u).abs().sum(1, keepdim=True))
        if scoring == "sigmoid":
            d, m = d * (1 - sel), m * (1 - sel)
    elif scoring == "sigmoid":
        d = g * sel * (1 - sel)
        m = d.abs()
    else:
        d = g * sel
        m = d.abs()
    dz, mag = torch.zeros_like(s), torch.zeros_like(s)
    dz.scatter_add_(1, at, d * is_)
    mag.scatter_add_(1, at, m * is_)
    if scoring == "softmax" and not renormalize:
        dot = (g * sel).sum(1, keepdim=True)
        dz -= s * dot
        mag += s * (g * sel).abs().sum(1, keepdim=True)
    return dz, mag


def _inputs(T, E, dtype, seed, device, bias=False, off=0.0):
    g = torch.Generator(device=device).manual_seed(seed)
    z = (2.0 * torch.randn(T, E, device=device, generator=g)).to(dtype)
    if off:
        z[torch.rand(T, E, device=device, generator=g) < off] = -math.inf
    return z, 0.1 * torch.randn(E, device=device, generator=g) if bias else None


def _check(z, got, want):
    """Scores come from exponentials of differences (U |z - max| and 2 U each) and a sum of E terms (at most 16 a lane, then a tree of 6: 22 U); the quotients,
    the sum of the chosen and the scale add 8 U.  64-bit differences of at most 88 count, beyond that scores are denormal."""
    (w, ids), (want_w, want_ids, _) = got, want
    k = w.shape[-1]
    assert ids.dtype == torch.int64 and w.dtype == torch.float32 and w.shape == ids.shape == (*z.shape[:-1], k)
    assert torch.equal(ids.reshape(-1, k).cpu(), want_ids)
    zd = z.detach().double().cpu().reshape(-1, z.shape[-1])
    spread = (zd.amax(1) - zd.masked_fill(zd == -math.inf, math.inf).amin(1)).nan_to_num(0.0).clamp(0.0, 88.0)[:, None]
    bound = (2 * spread + 64) * U * want_w + 2.0 ** -126
    assert ((w.reshape(-1, k).double().cpu() - want_w).abs() <= bound).all()


CASES = [
    # T, E, k, groups, top_groups, group_score, scoring, bias, renormalize, scale
    (1, 1, 1, 1, 1, "sum2", "softmax", False, True, 1.0), (3, 5, 5, 1, 1, "sum2", "sigmoid", True, False, 2.5), (7, 8, 2, 1, 1, "sum2", "softmax", False, True, 1.0),
    (1, 128, 8, 1, 1, "sum2", "softmax", False, True, 1.0), (33, 60, 4, 1, 1, "sum2", "softmax", False, False, 1.0), (65, 64, 6, 8, 3, "max", "softmax", False, False, 16.0),
    (130, 127, 3, 1, 1, "sum2", "sigmoid", True, True, 1.0), (64, 160, 6, 8, 3, "max", "softmax", True, True, 1.0), (50, 256, 8, 8, 4, "sum2", "sigmoid", True, True, 2.5),
    (20, 256, 8, 8, 4, "sum2", "softmax", False, False, 2.5), (9, 257, 7, 1, 1, "sum2", "softmax", True, False, 1.0), (5, 384, 12, 1, 1, "sum2", "sigmoid", True, True, 2.5),
    (4, 512, 22, 16, 5, "sum2", "sigmoid", False, False, 1.0), (3, 1000, 10, 10, 2, "max", "sigmoid", True, True, 1.0), (2, 1024, 32, 64, 7, "sum2", "softmax", True, True, 1.0),
    (17, 12, 3, 12, 5, "sum2", "sigmoid", True, True, 1.0), (11, 96, 32, 3, 2, "sum2", "softmax", False, True, 0.5),
]


def _options(case):
    _, _, k, groups, top_groups, group_score, scoring, _, renormalize, scale = case
    return dict(top_k=k, num_groups=groups, top_groups=top_groups, group_score=group_score, scoring=scoring, renormalize=renormalize, scale=scale)


def _reference(z, o, bias):
    return reference(z, o["top_k"], o["scoring"], bias, o["num_groups"], o["top_groups"], o["group_score"], o["renormalize"], o["scale"])


@pytest.mark.parametrize("off", [0.0, 0.4])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"t{c[0]}e{c[1]}k{c[2]}")
def test_forward_and_gradient(hip_device, case, dtype, off):
    z, bias = _inputs(case[0], case[1], dtype, case[1] + case[0], hip_device, case[7], off)
    o = _options(case)
    want = _reference(z, o, bias)
    with torch.no_grad():
        _check(z, moe_route(z, bias=bias, **o), want)
    z.requires_grad_(True)
    w, ids = moe_route(z, bias=bias, **o)
    assert not ids.requires_grad
    _check(z, (w.detach(), ids), want)
    up = torch.randn(w.shape, device=hip_device, generator=torch.Generator(device=hip_device).manual_seed(3))
    dz, = torch.autograd.grad(w, z, up)
    assert dz.dtype == dtype and dz.shape == z.shape
    want_dz, mag = gradient(z, up, *want, o["scoring"], o["renormalize"], o["scale"])
    # weights as above (spread at most 20 here), each term's products and the sum over at most 32 of them: 40 U
    bound = (2 * 20 + 64 + 40 + 40) * U * mag + (B if dtype == BF else 0.0) * want_dz.abs() + 2.0 ** -120
    assert ((dz.double().cpu() - want_dz).abs() <= bound).all()


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_gradient_against_differences(hip_device, scoring, renormalize):
    """Central differences of the definition with the choice held: their error is h^2 / 6 of a third derivative of at most 8 times the magnitudes"""
    z, _ = _inputs(4, 24, torch.float32, 8, hip_device)
    up = torch.randn(4, 5, device=hip_device)
    z.requires_grad_(True)
    w, ids = moe_route(z, 5, scoring=scoring, renormalize=renormalize, scale=2.0)
    dz, = torch.autograd.grad(w, z, up)
    zd, h = z.detach().double().cpu(), 1e-4

    def value(q):
        s = torch.sigmoid(q) if scoring == "sigmoid" else torch.softmax(q, 1)
        p = s.gather(1, ids.cpu())
        return (2.0 * (p / p.sum(1, keepdim=True) if renormalize else p) * up.double().cpu()).sum(1)

    for e in range(24):
        step = torch.zeros(24, dtype=torch.float64)
        step[e] = h
        num = (value(zd + step) - value(zd - step)) / (2 * h)
        assert ((dz[:, e].double().cpu() - num).abs() <= 1e-6 * (1.0 + up.abs().sum(1).double().cpu())).all()


# ---------------------------------------------------------------- ties and borders
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [None, "zero", "steps"])
@pytest.mark.parametrize("groups", [1, 8])
def test_equal_experts_go_by_their_index(hip_device, scoring, bias, groups):
    g = torch.Generator(device=hip_device).manual_seed(5)
    z = torch.randint(-2, 3, (40, 64), device=hip_device, generator=g).to(BF)
    z[0] = 0.0
    z[1] = -0.0
    z[2, ::2] = -0.0
    z[2, 1::2] = 0.0
    b = None if bias is None else torch.zeros(64, device=hip_device)
    if bias == "steps":
        b += 0.25 * torch.randint(0, 3, (64,), device=hip_device, generator=g)
    o = dict(top_k=8, scoring=scoring, num_groups=groups, top_groups=max(1, groups // 2), group_score="sum2", renormalize=True, scale=1.0)
    _check(z, moe_route(z, bias=b, **o), _reference(z, o, b))


@pytest.mark.parametrize("E", [32, 256, 700])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_scores_nearer_than_fp32_tells_apart(hip_device, E, scoring):
    """Biases that bring every score to about the same sum: the order is that of 64 bits, far below a step of fp32"""
    z, _ = _inputs(6, E, torch.float32, E, hip_device)
    z = z[:1].repeat(6, 1)
    s = torch.sigmoid(z[0].double()) if scoring == "sigmoid" else torch.softmax(z[0].double(), 0)
    bias = (1.0 - s).float()                       # sums of 1 up to 2^-25: differences of about 1e-8
    sums = (s + bias.double()).sort().values
    assert sums[-1] - sums[0] < 1e-7 and (sums[1:] - sums[:-1]).min() > 4e-16
    for groups, top in ((1, 1), (4, 2)):
        if E % groups == 0:
            for score in ("max", "sum2"):
                o = dict(top_k=8, scoring=scoring, num_groups=groups, top_groups=top, group_score=score, renormalize=True, scale=1.0)
                _check(z, moe_route(z, bias=bias, **o), _reference(z, o, bias))


@pytest.mark.parametrize("lift", [0.0, -60.0, -200.0, 60.0])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_far_logits(hip_device, scoring, lift):
    """Scores that are nearly nothing keep their ratios (sigmoid of -200 is no fp32 number, its quotients are); those of 60 are all 1"""
    z, _ = _inputs(9, 64, torch.float32, 4, hip_device)
    z = z + lift
    o = dict(top_k=6, scoring=scoring, num_groups=1, top_groups=1, group_score="max", renormalize=True, scale=1.0)
    _check(z, moe_route(z, **o), _reference(z, o, None))


# ---------------------------------------------------------------- masks
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("groups", [1, 4])
def test_rows_with_few_experts_left_or_none(hip_device, scoring, renormalize, groups):
    z, _ = _inputs(6, 32, torch.float32, 9, hip_device)
    left = [0, 1, 2, 5, 8, 32]
    for t, n in enumerate(left):
        off = torch.randperm(32, device=hip_device, generator=torch.Generator(device=hip_device).manual_seed(t))[n:]
        z[t, off] = -math.inf
    z.requires_grad_(True)
    o = dict(top_k=8, scoring=scoring, num_groups=groups, top_groups=max(1, groups - 1), group_score="sum2", renormalize=renormalize, scale=1.0)
    for bias in (None, torch.zeros(32, device=hip_device)):
        want = _reference(z, o, bias)
        w, ids = moe_route(z, bias=bias, **o)
        _check(z, (w.detach(), ids), want)
        assert (ids[0] == -1).all() and (w[0] == 0).all() and (ids[1] >= 0).sum() == 1
        up = torch.randn(w.shape, device=hip_device)
        dz, = torch.autograd.grad(w, z, up)
        want_dz, mag = gradient(z, up, *want, scoring, renormalize, 1.0)
        assert ((dz.double().cpu() - want_dz).abs() <= 200 * U * mag + 2.0 ** -120).all()


def test_biases_without_end(hip_device):
    z, _ = _inputs(5, 24, BF, 11, hip_device)
    bias = torch.zeros(24, device=hip_device)
    bias[3], bias[7], bias[20] = math.inf, math.inf, -math.inf
    bias[torch.arange(8, 24, 5)] = -math.inf
    w, ids = moe_route(z, 4, bias=bias)
    assert (ids[:, 0] == 3).all() and (ids[:, 1] == 7).all() and not torch.isin(ids, torch.nonzero(bias == -math.inf)[:, 0]).any()
    o = dict(top_k=4, scoring="softmax", num_groups=1, top_groups=1, group_score="max", renormalize=True, scale=1.0)
    _check(z, (w, ids), _reference(z, o, bias))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_what_is_no_number_stays_in_its_row(hip_device, scoring, renormalize):
    z, _ = _inputs(6, 40, torch.float32, 12, hip_device)
    z[1, 39], z[3, 0], z[4, 5] = math.nan, math.inf, -math.nan
    z.requires_grad_(True)
    w, ids = moe_route(z, 5, scoring=scoring, renormalize=renormalize)
    dz, = torch.autograd.grad(w, z, torch.ones_like(w))
    bad = [1, 4] + ([3] if scoring == "softmax" else [])
    good = [t for t in range(6) if t not in bad]
    assert w[bad].isnan().all() and dz[bad].isnan().all() and (ids[bad] == torch.arange(5, device=hip_device)).all()
    assert w[good].isfinite().all() and dz[good].isfinite().all()
    zg = z.detach()[good]
    w2, ids2 = moe_route(zg, 5, scoring=scoring, renormalize=renormalize)
    assert torch.equal(w2, w[good]) and torch.equal(ids2, ids[good])
    b = torch.zeros(40, device=hip_device)
    b[8] = math.nan
    assert moe_route(zg, 5, scoring=scoring, renormalize=renormalize, bias=b)[0].isnan().all()


def _kinds(E, dtype, device):
    """Rows of every kind: ordinary, few left, none, all equal, two values, a run of equal ones, nearly equal, not numbers (the last two, by index)"""
    z, _ = _inputs(24, E, dtype, E, device, off=0.0)
    z[1, 3:] = -math.inf
    z[2] = -math.inf
    z[3] = 0.25
    z[4] = torch.where(torch.arange(E, device=device) % 3 == 0, 1.0, 0.5).to(dtype)
    z[5, E // 2:] = 3.0
    z[6, :-1] = -math.inf
    z[7, 20:E - 20] = -math.inf
    z[8] = torch.linspace(1.0, 1.00001, E, device=device).to(dtype)
    z[9, ::2] = -math.inf
    z[10, :90] = 2.0
    z[22, E - 1], z[23, 0] = math.nan, math.nan
    return z


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("E, k, groups, top_groups, score", [(100, 15, 1, 1, "sum2"), (128, 8, 8, 4, "max"), (160, 9, 10, 3, "sum2"), (203, 15, 1, 1, "max"), (256, 8, 8, 4, "sum2"),
                                                            (256, 8, 8, 1, "max"), (64, 15, 2, 1, "sum2"), (240, 12, 60, 7, "sum2")])
@pytest.mark.parametrize("scoring, with_bias", [("softmax", False), ("sigmoid", True), ("softmax", True)])
def test_many_rows_of_every_kind(hip_device, E, k, groups, top_groups, score, scoring, with_bias, dtype):
    """More rows than are done one a wave, in an order in which every kind is next to every other: each has what it has alone"""
    pool = _kinds(E, dtype, hip_device)
    bias = 0.1 * torch.randn(E, device=hip_device, generator=torch.Generator(device=hip_device).manual_seed(1)) if with_bias else None
    if with_bias:
        s = torch.sigmoid(pool[11].double()) if scoring == "sigmoid" else torch.softmax(pool[11].double(), 0)
        bias[:E // 2] = (0.75 - s[:E // 2]).float()            # half of this row's sums are nearly equal
    o = dict(top_k=k, scoring=scoring, num_groups=groups, top_groups=top_groups, group_score=score, renormalize=True, scale=2.5)
    w0, i0, s0 = _reference(pool[:22], o, bias)
    at = torch.randint(0, 24, (2 * 2048 + 3,), generator=torch.Generator().manual_seed(E))
    good, bad = (at < 22).nonzero()[:, 0], (at >= 22).nonzero()[:, 0]
    z = pool[at.to(hip_device)].requires_grad_(True)
    w, ids = moe_route(z, bias=bias, **o)
    up = torch.randn(w.shape, device=hip_device, generator=torch.Generator(device=hip_device).manual_seed(3))
    dz, = torch.autograd.grad(w, z, up)
    want = (w0[at[good]], i0[at[good]], s0[at[good]])
    _check(z.detach()[good.to(hip_device)], (w.detach()[good.to(hip_device)], ids[good.to(hip_device)]), want)
    want_dz, mag = gradient(z, up[good.to(hip_device)], *want, scoring, True, 2.5)
    bound = (2 * 20 + 64 + 40 + 40) * U * mag + (B if dtype == BF else 0.0) * want_dz.abs() + 2.0 ** -120
    assert ((dz[good.to(hip_device)].double().cpu() - want_dz).abs() <= bound).all()
    bad = bad.to(hip_device)
    assert w[bad].isnan().all() and dz[bad].isnan().all() and (ids[bad] == torch.arange(k, device=hip_device)).all()


@pytest.mark.parametrize("E, k, groups, top_groups, scoring, with_bias", [(300, 8, 1, 1, "softmax", False), (512, 17, 8, 3, "sigmoid", True), (1000, 20, 10, 4, "softmax", True),
                                                                         (120, 31, 1, 1, "sigmoid", True), (256, 16, 4, 2, "softmax", False)])
def test_more_rows_than_waves_of_one_row_each(hip_device, E, k, groups, top_groups, scoring, with_bias):
    """Many experts or many choices take a wave a row, and several rows one after the other"""
    pool = _kinds(E, torch.float32, hip_device)[:22]
    bias = 0.1 * torch.randn(E, device=hip_device, generator=torch.Generator(device=hip_device).manual_seed(1)) if with_bias else None
    o = dict(top_k=k, scoring=scoring, num_groups=groups, top_groups=top_groups, group_score="sum2", renormalize=True, scale=1.5)
    w0, i0, s0 = _reference(pool, o, bias)
    at = torch.randint(0, 22, (2 * 4096 + 5,), generator=torch.Generator().manual_seed(E))
    z = pool[at.to(hip_device)].requires_grad_(True)
    w, ids = moe_route(z, bias=bias, **o)
    up = torch.randn(w.shape, device=hip_device, generator=torch.Generator(device=hip_device).manual_seed(3))
    dz, = torch.autograd.grad(w, z, up)
    want = (w0[at], i0[at], s0[at])
    _check(z.detach(), (w.detach(), ids), want)
    want_dz, mag = gradient(z, up, *want, scoring, True, 1.5)
    assert ((dz.double().cpu() - want_dz).abs() <= (2 * 20 + 64 + 40 + 40) * U * mag + 2.0 ** -120).all()


@pytest.mark.parametrize("E", [15, 9, 32])
def test_all_experts_chosen_beside_rows_that_are_no_numbers(hip_device, E):
    z, bias = _inputs(7, E, torch.float32, E, hip_device, True)
    z[2, 1], z[6, E - 1] = math.nan, math.nan
    w, ids = moe_route(z, E, scoring="sigmoid", bias=bias)
    good = [0, 1, 3, 4, 5]
    o = dict(top_k=E, scoring="sigmoid", num_groups=1, top_groups=1, group_score="max", renormalize=True, scale=1.0)
    _check(z[good], (w[good], ids[good]), _reference(z[good], o, bias))
    assert w[[2, 6]].isnan().all() and (ids[[2, 6]] == torch.arange(E, device=hip_device)).all()


# ---------------------------------------------------------------- layouts, sizes, streams
def _layouts(z):
    T, E = z.shape
    wide = torch.full((T, E + 5), math.nan, dtype=z.dtype, device=z.device)
    wide[:, 3:3 + E] = z
    off = torch.cat([z.new_zeros(1), z.reshape(-1)])[1:].view(T, E)
    return {"slice": wide[:, 3:3 + E], "transposed": z.t().contiguous().t(), "off by one": off, "every other": torch.stack([z, z], 1)[:, 0],
            "three dimensions": z.view(2, T // 2, E), "one row for all": z[:1].expand(T, E)}


@pytest.mark.parametrize("E", [16, 30, 128, 520])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_layouts(hip_device, dtype, E):
    z, bias = _inputs(6, E, dtype, 13, hip_device, True)
    up = torch.randn(6, 3, device=hip_device)
    for name, v in _layouts(z).items():
        ref = v.contiguous().view(-1, E).requires_grad_(True)
        w0, i0 = moe_route(ref, 3, bias=bias, scoring="sigmoid")
        d0, = torch.autograd.grad(w0, ref, up)
        leaf = v.detach().requires_grad_(True)
        w, i = moe_route(leaf, 3, bias=torch.stack([bias, bias], 1)[:, 0], scoring="sigmoid")
        d, = torch.autograd.grad(w, leaf, up.view(w.shape).expand_as(w))
        assert torch.equal(w.view(-1, 3), w0) and torch.equal(i.view(-1, 3), i0) and torch.equal(d.reshape(-1, E), d0), name


def test_one_dimension_and_no_tokens(hip_device):
    z, _ = _inputs(1, 20, BF, 14, hip_device)
    w, i = moe_route(z[0], 3)
    w2, i2 = moe_route(z, 3)
    assert w.shape == (3,) and torch.equal(w, w2[0]) and torch.equal(i, i2[0])
    e = torch.zeros(0, 20, device=hip_device, requires_grad=True)
    w, i = moe_route(e, 3)
    assert w.shape == i.shape == (0, 3)
    assert torch.autograd.grad(w, e, torch.zeros_like(w))[0].shape == (0, 20)


def test_upstream_gradients_of_other_layouts(hip_device):
    z, _ = _inputs(8, 32, torch.float32, 15, hip_device)
    z.requires_grad_(True)
    w, _ = moe_route(z, 4, scoring="sigmoid", renormalize=False)
    ones, = torch.autograd.grad(w, z, torch.ones(8, 4, device=hip_device), retain_graph=True)
    summed, = torch.autograd.grad(w.sum(), z, retain_graph=True)
    assert torch.equal(ones, summed)
    turned = torch.randn(4, 8, device=hip_device).t()
    a, = torch.autograd.grad(w, z, turned, retain_graph=True)
    b, = torch.autograd.grad(w, z, turned.contiguous())
    assert torch.equal(a, b)


def test_more_elements_than_32_bits_count(hip_device):
    T, E = (1 << 22) + 3, 1024
    z = torch.zeros(T, E, dtype=BF, device=hip_device)
    assert z.numel() > 1 << 32
    tail, _ = _inputs(5, E, BF, 16, hip_device)
    z[-5:] = tail
    z.requires_grad_(True)
    w, i = moe_route(z, 4, scoring="sigmoid", renormalize=False)
    up = torch.ones_like(w)
    dz, = torch.autograd.grad(w, z, up)
    t2 = tail.clone().requires_grad_(True)
    w2, i2 = moe_route(t2, 4, scoring="sigmoid", renormalize=False)
    d2, = torch.autograd.grad(w2, t2, up[:5])
    assert torch.equal(w[-5:], w2) and torch.equal(i[-5:], i2) and torch.equal(dz[-5:], d2)
    assert (i[0] == torch.arange(4, device=hip_device)).all()


def test_another_stream(hip_device):
    z, bias = _inputs(700, 128, BF, 17, hip_device, True)
    want = moe_route(z, 8, bias=bias)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        zz = z.clone().requires_grad_(True)
        w, i = moe_route(zz, 8, bias=bias)
        dz, = torch.autograd.grad(w, zz, torch.ones_like(w))
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(w, want[0]) and torch.equal(i, want[1]) and dz.isfinite().all()


def _step(z, bias, up):
    w, i = moe_route(z, 8, bias=bias, scoring="sigmoid", num_groups=8, top_groups=4, scale=2.5)
    return w.detach(), i, torch.autograd.grad(w, z, up)[0]


def test_captured_forward_and_backward(hip_device):
    z, bias = _inputs(300, 256, torch.float32, 18, hip_device, True)
    z.requires_grad_(True)
    up = torch.randn(300, 8, device=hip_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _step(z, bias, up)
    for seed in range(3):
        with torch.no_grad():
            z.copy_(_inputs(300, 256, torch.float32, 30 + seed, hip_device)[0])
        graph.replay()
        torch.cuda.synchronize()
        other = z.detach().clone().requires_grad_(True)
        assert all(torch.equal(a, b) for a, b in zip(got, _step(other, bias, up)))


def test_capture_beside_living_weights_is_refused(hip_device):
    z, bias = _inputs(30, 64, torch.float32, 19, hip_device, True)
    z.requires_grad_(True)
    eager, _ = moe_route(z, 4, bias=bias)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="another stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(moe_route(z, 4, bias=bias)[0], z, torch.ones(30, 4, device=hip_device))
    torch.cuda.synchronize()
    assert torch.autograd.grad(eager, z, torch.ones_like(eager))[0].isfinite().all()


class _Logits(torch.nn.Parameter):
    pass


def test_subclasses_take_the_python_path(hip_device):
    z, bias = _inputs(30, 64, BF, 20, hip_device, True)
    up = torch.randn(30, 4, device=hip_device)
    for kw in (dict(), dict(scoring="sigmoid"), dict(renormalize=False)):
        p, q = _Logits(z.clone()), z.clone().requires_grad_(True)
        a, b = moe_route(p, 4, bias=bias, **kw), moe_route(q, 4, bias=bias, **kw)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        assert torch.equal(torch.autograd.grad(a[0], p, up)[0], torch.autograd.grad(b[0], q, up)[0])
    with pytest.raises(RuntimeError, match="no subclasses"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(moe_route(p, 4)[0], p, up)
    torch.cuda.synchronize()


def test_under_torch_compile(hip_device):
    z, bias = _inputs(30, 64, BF, 21, hip_device, True)
    up = torch.randn(30, 4, device=hip_device)
    for kw in (dict(), dict(scoring="sigmoid", num_groups=4, top_groups=2), dict(renormalize=False)):
        q = z.clone().requires_grad_(True)
        f = torch.compile(lambda t: moe_route(t, 4, bias=bias, **kw), backend="aot_eager", fullgraph=True)
        a, b = f(q), moe_route(q, 4, bias=bias, **kw)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        assert torch.equal(torch.autograd.grad(a[0], q, up)[0], torch.autograd.grad(b[0], q, up)[0])


# ---------------------------------------------------------------- what autograd is and is not told
def test_changes_in_place_and_second_derivatives_are_refused(hip_device):
    z, bias = _inputs(10, 32, torch.float32, 22, hip_device, True)
    z.requires_grad_(True)
    w, i = moe_route(z, 4, bias=bias)
    up = torch.ones_like(w)
    w.data.mul_(1.0)
    w.detach().mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(w, z, up)
    w, i = moe_route(z, 4, bias=bias)
    i.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(w, z, up)
    w, _ = moe_route(z, 4, bias=bias, scoring="sigmoid")
    dz, = torch.autograd.grad(w, z, up.requires_grad_(True), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        dz.sum().backward()
    w, _ = moe_route(z, 4, scoring="sigmoid")
    z.data = torch.zeros(3, 32, device=hip_device)
    with pytest.raises(RuntimeError, match="freed, resized or exchanged"):
        torch.autograd.grad(w, z, up.detach())


def test_tangents_and_transforms_are_refused(hip_device):
    import torch.autograd.forward_ad as fwAD

    z, bias = _inputs(10, 32, torch.float32, 23, hip_device, True)
    for grad in (True, False):
        with fwAD.dual_level(), torch.set_grad_enabled(grad), pytest.raises(NotImplementedError):
            moe_route(fwAD.make_dual(z, torch.ones_like(z)), 4)
    for f in (lambda: torch.func.jvp(lambda a: moe_route(a, 4)[0], (z,), (torch.ones_like(z),)), lambda: torch.func.grad(lambda a: moe_route(a, 4)[0].sum())(z),
              lambda: torch.vmap(lambda a: moe_route(a, 4)[0])(z[None])):
        with pytest.raises((RuntimeError, NotImplementedError)):
            f()


def test_a_bias_that_is_a_parameter_gets_no_gradient(hip_device):
    z, bias = _inputs(10, 32, torch.float32, 24, hip_device, True)
    z.requires_grad_(True)
    bias = torch.nn.Parameter(bias)
    moe_route(z, 4, bias=bias)[0].square().sum().backward()
    assert bias.grad is None and z.grad is not None


def test_devices_and_types_that_do_not_go_together(hip_device):
    z, bias = _inputs(10, 32, torch.float32, 25, hip_device, True)
    with pytest.raises(RuntimeError, match="HIP device only"):
        moe_route(z, 4, bias=bias.cpu())
    with pytest.raises(_C.XqError, match="bias"):
        moe_route(z, 4, bias=bias.double())
    with pytest.raises(_C.XqError, match="bf16 or fp32"):
        moe_route(z.half(), 4)
