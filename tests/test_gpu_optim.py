"""GPU: adamw_step, grad_norm, adamw_state_values and the AdamW optimizer against the update in 64 bits.

Bounds.  u = 2^-24 is half a step of fp32.  m' = b1 m + (1 - b1) g: the two constants are rounded (u each), two products and a sum: 3 u
of |b1 m| + |(1 - b1) g|, 4 with the gradient's scaling by the clip factor (its own two roundings come on top: 2 more).  v' the same with g
squared: 8 u of v'.  s = sqrt(v') half of that and a rounding: 5 u.  The update m' first / (s root + eps): m' (6 u), first, root and eps as
fp32 (3), two products, a sum, a quotient (4) and s (5): 18 u of the update with |b1 m| + |(1 - b1) g| in place of |m'|.  p: three more of
|p| (the decay's constant, its product, two differences of nearly |p|): 4 u.  A bf16 parameter is off by half a step of bf16 (2^-8) too."""

import pytest
import torch
from torch import nn

from tests.util_cases import make_dense_module
from xorl_amd import _C
from xorl_amd.optim import AdamW, adamw_state_values, adamw_step, grad_norm
from xorl_amd.qlora import maybe_merge_lora, reset_lora_optimizer_states

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
B1, B2, EPS = 0.9, 0.999, 1e-8
SIZES = [(1,), (3,), (255,), (256,), (257,), (1023,), (4095,), (4096,), (4097,), (16, 4096), (3, 7, 1153), (12289,)]


def _blocks(x):
    n = x.numel()
    pad = -n % 256
    return torch.nn.functional.pad(x.reshape(-1), (0, pad)).view(-1, 256)


def _decode(m, v, ms, vs):
    n = m.numel()
    c, d = _blocks(m.double()), _blocks(v.double())
    mm = c.sign() * (c / 127) ** 2 * ms.double()[:, None]
    vv = ((d / 255) ** 2 * vs.double()[:, None]) ** 2
    return mm.view(-1)[:n].view(m.shape), vv.view(-1)[:n].view(v.shape)


def _problem(shapes, bits, pdt, gdt, seed, device, offset=0, grad_std=1e-3):
    """Lists of a step, with the states that a run would have; `offset`: elements that every tensor starts behind an aligned address."""
    g = torch.Generator().manual_seed(seed)

    def put(x, dtype):
        n = x.numel()
        buf = torch.empty(n + offset + 64, dtype=dtype, device=device)
        view = buf[offset:offset + n].view(x.shape)
        view.copy_(x.to(dtype))
        return view

    p = [put(torch.randn(s, generator=g) * 0.05, pdt) for s in shapes]
    gr = [put(torch.randn(s, generator=g) * grad_std, gdt) for s in shapes]
    steps = [torch.tensor(float(3 + 7 * (i % 5)), device=device) for i in range(len(shapes))]
    if bits == 32:
        m = [put(torch.randn(s, generator=g) * 3e-4, torch.float32) for s in shapes]
        v = [put((torch.randn(s, generator=g) * 1e-3) ** 2, torch.float32) for s in shapes]
        return p, gr, m, v, steps, None, None
    m = [put(torch.randint(-127, 128, s, generator=g), torch.int8) for s in shapes]
    v = [put(torch.randint(0, 256, s, generator=g), torch.uint8) for s in shapes]
    n = [-(-x.numel() // 256) for x in p]
    ms = [(torch.rand(k, generator=g) * 1e-3).to(device) for k in n]
    vs = [(torch.rand(k, generator=g) * 1e-3 + 1e-5).to(device) for k in n]
    return p, gr, m, v, steps, ms, vs


def _expected(prob, bits, lr, wd, factor=1.0):
    """The step in 64 bits, with the sum of magnitudes that m's error counts by."""
    p, gr, m, v, steps, ms, vs = prob
    out = []
    for i in range(len(p)):
        if bits == 8:
            mi, vi = _decode(m[i], v[i], ms[i], vs[i])
        else:
            mi, vi = m[i].double(), v[i].double()
        g = gr[i].double() * factor
        t = float(steps[i]) + 1
        m1, mag = B1 * mi + (1 - B1) * g, B1 * mi.abs() + (1 - B1) * g.abs()
        v1 = B2 * vi + (1 - B2) * g * g
        den = v1.sqrt() / (1 - B2 ** t) ** 0.5 + EPS
        k = lr / (1 - B1 ** t)
        w = p[i].double()
        out.append((w - lr * wd * w - k * m1 / den, m1, v1, mag, k * mag / den, w))
    return out


def _check(prob, exp, bits, pdt, decoded_error=0.0):
    p, _, m, v, _, ms, vs = prob
    for i, (pe, me, ve, mag, upd, w) in enumerate(exp):
        bound = (4 * U * w.abs() + (18 + decoded_error) * U * upd) + (2.0 ** -8 * pe.abs() if pdt == torch.bfloat16 else 0)
        assert bool(((p[i].double() - pe).abs() <= bound + 1e-38).all()), f"p[{i}]"
        dm = (6 + decoded_error) * U * mag
        if bits == 32:
            assert bool(((m[i].double() - me).abs() <= dm + 1e-38).all()), f"m[{i}]"
            assert bool(((v[i].double() - ve).abs() <= 8 * U * ve + 1e-38).all()), f"v[{i}]"
            continue
        # scales: the largest magnitude of a block; codes: within half a code of where the value lies, and how far its error moves that
        for code, scale, val, dv, top in ((m[i].double().abs(), ms[i], me.abs(), dm, 127.0),
                                          (v[i].double(), vs[i], ve.sqrt(), (5 + decoded_error) * U * ve.sqrt(), 255.0)):
            amax = _blocks(val).amax(1)
            assert bool(((scale.double() - amax).abs() <= _blocks(dv).amax(1) + 1e-38).all()), f"scale {i}"
            a = amax.clamp(min=1e-300)[:, None]
            lo, hi = top * ((_blocks(val) - _blocks(dv)).clamp(min=0) / a).sqrt(), top * ((_blocks(val) + _blocks(dv)) / a).sqrt()
            # (the reciprocal of the scale, the scale's own error, two products and a root of one ulp: 12 u of the code)
            slack = 0.5 + 12 * U * top
            c = _blocks(code)
            low = c >= lo - slack
            high = c <= hi + slack
            if top == 255.0:
                high |= (c == 1) & (_blocks(val) > 0)         # a positive s is never rounded to zero
            assert bool(low.all()) and bool(high.all()), f"codes {i}"
        assert bool(((m[i].double().sign() == me.sign()) | (m[i] == 0) | (me.abs() <= dm)).all())


# decoding: the product of a code's square and the scale's share, three roundings (m) and, squared, seven (s)
DECODED = 8.0


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("pdt,gdt", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_step_by_type_and_alignment(hip_device, bits, pdt, gdt, offset):
    prob = _problem(SIZES, bits, pdt, gdt, 3, hip_device, offset)
    guard = [x.clone() for x in prob[1]]
    exp = _expected(prob, bits, 1e-3, 0.1)
    before = [float(t) for t in prob[4]]
    assert adamw_step(*prob[:5], exp_avg_scales=prob[5], exp_avg_sq_scales=prob[6], lr=1e-3, weight_decay=0.1) is None
    _check(prob, exp, bits, pdt, DECODED if bits == 8 else 0.0)
    assert [float(t) for t in prob[4]] == [b + 1 for b in before]
    assert all(torch.equal(a, b) for a, b in zip(guard, prob[1]))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [63, 64, 65, 84, 85, 200, 4200])
def test_step_over_many_tensors(hip_device, bits, count):
    shapes = [((i * 37) % 300 + 1,) if i % 50 else (9001,) for i in range(count)]
    prob = _problem(shapes, bits, torch.float32, torch.float32, 5, hip_device)
    exp = _expected(prob, bits, 2e-4, 0.0)
    adamw_step(*prob[:5], exp_avg_scales=prob[5], exp_avg_sq_scales=prob[6], lr=2e-4, weight_decay=0.0)
    if count > 1000:            # (the check looks at each tensor by itself: every 40th, and the ends)
        keep = sorted({*range(0, count, 40), *range(60), *range(count - 5, count)})
        prob = tuple(None if x is None else [x[i] for i in keep] for x in prob)
        exp = [exp[i] for i in keep]
    _check(prob, exp, bits, torch.float32, DECODED if bits == 8 else 0.0)


@pytest.mark.parametrize("bits,count", [(8, 83), (8, 168), (8, 169), (32, 111), (32, 112), (32, 113), (32, 225)])
@pytest.mark.parametrize("pdt,gdt", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
def test_step_where_a_table_launch_ends(hip_device, bits, count, pdt, gdt):
    prob = _problem([(300 * (i % 7) + i + 1,) for i in range(count)], bits, pdt, gdt, 6, hip_device)
    exp = _expected(prob, bits, 2e-4, 0.0)
    adamw_step(*prob[:5], exp_avg_scales=prob[5], exp_avg_sq_scales=prob[6], lr=2e-4, weight_decay=0.0)
    _check(prob, exp, bits, pdt, DECODED if bits == 8 else 0.0)


@pytest.mark.parametrize("count", [255, 256, 257, 512, 513])
def test_grad_norm_where_a_table_launch_ends(hip_device, count):
    grads = [torch.full((i + 1,), 0.5, device=hip_device, dtype=torch.bfloat16 if i % 2 else torch.float32) for i in range(count)]
    want = (0.25 * count * (count + 1) / 2) ** 0.5
    assert abs(float(grad_norm(grads)) - want) <= (U + 1e-10) * want


@pytest.mark.parametrize("clip", [None, 0.02])
@pytest.mark.parametrize("n", [256 * 4000, 256 * 33 + 77])
def test_codes_are_the_nearest_ones(hip_device, n, clip):
    """8-bit codes against the nearest ones of m' and s', both formed by the formula's operations in fp32: equal, whatever lies in the middle"""
    prob = _problem([(n,)], 8, torch.float32, torch.float32, 41, hip_device)
    m, v = _blocks(prob[2][0].float()), _blocks(prob[3][0].float())
    g = _blocks(prob[1][0])
    if clip is not None:
        norm = g.double().square().sum().sqrt().float()
        g = g * ((norm + 1e-6).reciprocal() * clip).clamp(max=1.0)
    m = m * m.abs() * (prob[5][0] * (1 / 16129))[:, None] * B1 + g * (1 - B1)
    old = v * v * (prob[6][0] * (1 / 65025))[:, None]
    s = (old * old * B2 + g * g * (1 - B2)).sqrt()
    adamw_step(*prob[:5], exp_avg_scales=prob[5], exp_avg_sq_scales=prob[6], lr=1e-3, max_norm=clip)
    ma, sa = m.abs().amax(1), s.amax(1)
    assert torch.equal(prob[5][0], ma) and torch.equal(prob[6][0], sa)
    c = (m.double().abs() / ma.double()[:, None]).sqrt().mul(127).round() * m.sign()
    d = (s.double() / sa.double()[:, None]).sqrt().mul(255).round().clamp(min=1) * (s > 0)
    assert torch.equal(c.view(-1)[:n].to(torch.int8), prob[2][0]) and torch.equal(d.view(-1)[:n].to(torch.uint8), prob[3][0])


def test_elements_outside_stay(hip_device):
    """What lies around a tensor's elements is left alone: the last pieces are stored one by one."""
    for bits in (32, 8):
        n, pad = 777, 300
        bufs = [torch.full((n + 2 * pad,), 3, dtype=dt, device=hip_device) for dt in
                (torch.float32, torch.float32 if bits == 32 else torch.int8, torch.float32 if bits == 32 else torch.uint8)]
        scales = [torch.full((4 + 8,), 0.5, device=hip_device) for _ in range(2)]
        p, m, v = (b[pad:pad + n] for b in bufs)
        adamw_step([p], [torch.ones(n, device=hip_device)], [m], [v], [torch.zeros((), device=hip_device)],
                   exp_avg_scales=[scales[0][4:8]] if bits == 8 else None, exp_avg_sq_scales=[scales[1][4:8]] if bits == 8 else None, lr=0.1)
        for b in bufs:
            assert bool((b[:pad] == 3).all()) and bool((b[pad + n:] == 3).all())
        for s in scales if bits == 8 else ():
            assert bool((s[:4] == 0.5).all()) and bool((s[8:] == 0.5).all()) and not bool((s[4:8] == 0.5).any())


@pytest.mark.parametrize("gdt", [torch.float32, torch.bfloat16])
def test_grad_norm(hip_device, gdt):
    prob = _problem(SIZES + [(300000,)], 32, torch.float32, gdt, 7, hip_device, offset=1)
    want = torch.cat([g.double().reshape(-1) for g in prob[1]]).norm()
    got = grad_norm(prob[1])
    # squares and sums in 64 bits: one rounding to fp32 (and 1e-10 for the sum)
    assert got.dtype == torch.float32 and got.dim() == 0
    assert abs(float(got) - float(want)) <= (U + 1e-10) * float(want)
    assert torch.equal(got, grad_norm(prob[1]))
    mixed = [g if i % 2 else g.float() for i, g in enumerate(prob[1])]
    assert abs(float(grad_norm(mixed)) - float(want)) <= (U + 1e-10) * float(want)
    big = [torch.full((5000,), 1e30, device=hip_device)]
    assert abs(float(grad_norm(big)) / (1e30 * 5000 ** 0.5) - 1) < 1e-6           # squares beyond fp32
    assert float(grad_norm([torch.zeros(0, device=hip_device)])) == 0.0


@pytest.mark.parametrize("count", [1, 251, 252, 253, 3000])
def test_grad_norm_over_many_tensors(hip_device, count):
    g = torch.Generator(device=hip_device).manual_seed(count)
    grads = [torch.randn((i * 53) % 9000 + 1, device=hip_device, generator=g).to(torch.bfloat16 if i % 3 == 0 else torch.float32) for i in range(count)]
    want = sum(float(x.double().square().sum()) for x in grads) ** 0.5
    assert abs(float(grad_norm(grads)) - want) <= (U + 1e-10) * want


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("max_norm", [0.01, 1e6])
def test_clipping(hip_device, bits, max_norm):
    prob = _problem(SIZES, bits, torch.float32, torch.float32, 11, hip_device)
    norm = float(torch.cat([g.double().reshape(-1) for g in prob[1]]).norm())
    exp = _expected(prob, bits, 1e-3, 0.0, min(1.0, max_norm / (norm + 1e-6)))
    got = adamw_step(*prob[:5], exp_avg_scales=prob[5], exp_avg_sq_scales=prob[6], lr=1e-3, weight_decay=0.0, max_norm=max_norm)
    assert abs(float(got) - norm) <= 2 * U * norm
    _check(prob, exp, bits, torch.float32, DECODED if bits == 8 else 0.0)


def test_norm_that_is_given(hip_device):
    prob = _problem(SIZES, 32, torch.float32, torch.float32, 12, hip_device)
    exp = _expected(prob, 32, 1e-3, 0.0, 0.25 / (1.0 + 1e-6))
    given = torch.tensor(1.0, device=hip_device)
    adamw_step(*prob[:5], lr=1e-3, weight_decay=0.0, max_norm=0.25, grad_norm=given)
    assert float(given) == 1.0
    _check(prob, exp, 32, torch.float32)


@pytest.mark.parametrize("bits", [32, 8])
def test_first_step_and_zero_gradients(hip_device, bits):
    """From zero states; where the gradient is zero nothing but the decay moves a parameter, and the states stay zero."""
    n = 1000
    g = torch.zeros(n, device=hip_device)
    g[600:] = torch.linspace(-1e-3, 1e-3, 400, device=hip_device)
    p = torch.ones(n, device=hip_device)
    dt = (torch.float32, torch.float32) if bits == 32 else (torch.int8, torch.uint8)
    m, v = torch.zeros(n, dtype=dt[0], device=hip_device), torch.zeros(n, dtype=dt[1], device=hip_device)
    sc = [torch.zeros(4, device=hip_device) for _ in range(2)]
    prob = ([p], [g], [m], [v], [torch.zeros((), device=hip_device)], [sc[0]], [sc[1]])
    exp = _expected(prob, bits, 1e-2, 0.5)
    adamw_step(*prob[:5], exp_avg_scales=[sc[0]] if bits == 8 else None, exp_avg_sq_scales=[sc[1]] if bits == 8 else None, lr=1e-2, weight_decay=0.5)
    _check(prob, exp, bits, torch.float32, DECODED if bits == 8 else 0.0)
    assert bool((m[:600] == 0).all()) and bool((v[:600] == 0).all()) and bool((p[:600] == p[0]).all())
    if bits == 8:
        assert bool((v[g != 0] > 0).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_non_finite_gradient_shows_in_its_block(hip_device, bad):
    prob = _problem([(2048,)], 8, torch.float32, torch.float32, 13, hip_device)
    prob[1][0][700] = bad
    adamw_step(*prob[:5], exp_avg_scales=prob[5], exp_avg_sq_scales=prob[6], lr=1e-3)
    m, v = adamw_state_values(prob[2][0], prob[3][0], prob[5][0], prob[6][0])
    block = torch.zeros(2048, dtype=torch.bool, device=hip_device)
    block[512:768] = True
    assert bool(torch.isfinite(m[~block]).all()) and bool(torch.isfinite(v[~block]).all()) and bool(torch.isfinite(prob[0][0][~block]).all())
    assert not bool(torch.isfinite(prob[6][0][2])) and not bool(torch.isfinite(prob[5][0][2]))
    assert not bool(torch.isfinite(v[block]).any())
    assert torch.isnan(prob[0][0][700])


def test_nan_norm_shows_everywhere(hip_device):
    prob = _problem([(300,), (5000,)], 32, torch.float32, torch.float32, 14, hip_device)
    prob[1][0][3] = float("nan")
    got = adamw_step(*prob[:5], lr=1e-3, max_norm=1.0)
    assert torch.isnan(got) and all(bool(torch.isnan(p).all()) for p in prob[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 255, 256, 1025, 70001])
def test_state_values(hip_device, dtype, n):
    prob = _problem([(n,)], 8, torch.float32, torch.float32, 17, hip_device, offset=n % 3)
    m, v = adamw_state_values(prob[2][0], prob[3][0], prob[5][0], prob[6][0], dtype)
    me, ve = _decode(prob[2][0], prob[3][0], prob[5][0], prob[6][0])
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    assert bool(((m.double() - me).abs() <= (4 * U + half) * me.abs()).all())
    assert bool(((v.double() - ve).abs() <= (8 * U + half) * ve + 1e-38).all())


def test_same_bits_twice_and_on_another_stream(hip_device):
    outs = []
    for stream in (None, None, torch.cuda.Stream()):
        prob = _problem(SIZES, 8, torch.float32, torch.float32, 19, hip_device)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            norm = adamw_step(*prob[:5], exp_avg_scales=prob[5], exp_avg_sq_scales=prob[6], lr=1e-3, max_norm=0.01)
        torch.cuda.synchronize()
        outs.append([norm, *prob[0], *prob[2], *prob[3], *prob[5], *prob[6]])
    for o in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], o))


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_follows_steps_and_lr(hip_device, bits):
    eager, graphed = (_problem(SIZES, bits, torch.float32, torch.float32, 23, hip_device) for _ in range(2))
    lr = torch.tensor(1e-3, device=hip_device)
    call = lambda q: adamw_step(*q[:5], exp_avg_scales=q[5], exp_avg_sq_scales=q[6], lr=lr, max_norm=0.05)  # noqa: E731
    warm = _problem(SIZES, bits, torch.float32, torch.float32, 24, hip_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(warm)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = call(graphed)
    for k in range(4):
        lr.fill_(1e-3 / (k + 1))
        for a, b in zip(eager[1], graphed[1]):
            a.normal_()
            b.copy_(a)
        want = call(eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want)
        for x, y in zip(eager, graphed):
            assert x is None or all(torch.equal(a, b) for a, b in zip(x, y)), k


def test_refusals(hip_device):
    def prob(bits=32):
        return list(_problem([(8, 8), (5,)], bits, torch.float32, torch.float32, 29, hip_device))

    def refused(q, match, error=_C.XqError, **kw):
        saved = [x.clone() for x in q[0] if isinstance(x, torch.Tensor)]
        with pytest.raises(error, match=match):
            adamw_step(*q[:5], exp_avg_scales=q[5], exp_avg_sq_scales=q[6], **{"lr": 1e-3, **kw})
        assert all(torch.equal(a, b) for a, b in zip(saved, q[0]))

    q = prob(); q[1][0] = q[1][0].reshape(-1); refused(q, "another shape")
    q = prob(); q[1][0] = q[1][0].half(); refused(q, "fp32 or bf16")
    q = prob(); q[0][0] = q[0][0].double(); refused(q, "fp32 or bf16")
    q = prob(); q[2][0] = q[2][0].bfloat16(); refused(q, "must be Float")
    q = prob(); q[3][1] = q[3][1][:4]; refused(q, "expected 5")
    q = prob(); q[0][0] = q[0][0].t(); refused(q, "contiguous")
    q = prob(); q[4][1] = q[4][0]; refused(q, "share")
    q = prob(); q[0][1] = q[0][0].view(-1)[:5]; refused(q, "share")
    q = prob(); q[2][1] = q[3][1]; refused(q, "share")
    q = prob(); both = torch.zeros(66, device=hip_device); q[2][0], q[3][0] = both[:64].view(8, 8), both[2:].view(8, 8); refused(q, "share")
    q = prob(8); q[5][0] = q[5][0].new_zeros(2); refused(q, r"1 element\(s\)")
    q = prob(8); q[2][0] = q[2][0].view(torch.uint8); refused(q, "must be Char")
    q = prob(8); q[5] = None; refused(q, "exp_avg_scales")
    q = prob(); q[4][0] = q[4][0].cpu(); refused(q, "HIP device only", RuntimeError)
    refused(prob(), "betas", betas=(0.9, 1.0))
    refused(prob(), "max_norm", max_norm=0.0)
    refused(prob(), "without max_norm", grad_norm=torch.ones((), device=hip_device))
    refused(prob(), "grad_norm must be", max_norm=1.0, grad_norm=torch.ones(2, device=hip_device))
    refused(prob(), "lr tensor", lr=torch.tensor(1e-3))
    m, v = torch.zeros(4, dtype=torch.int8, device=hip_device), torch.zeros(4, dtype=torch.uint8, device=hip_device)
    s = torch.zeros(1, device=hip_device)
    for bad in ((m, m, s, s), (m, v[:3], s, s), (m, v, s.double(), s), (m, v, s, s.expand(2))):
        with pytest.raises(_C.XqError):
            adamw_state_values(*bad)
    with pytest.raises(_C.XqError):
        adamw_state_values(m, v, s, s, torch.float16)


def test_gradient_of_another_layout(hip_device):
    prob = _problem([(40, 24)], 32, torch.float32, torch.float32, 31, hip_device)
    prob[1][0] = torch.randn(24, 40, device=hip_device).t()
    exp = _expected(prob, 32, 1e-3, 0.0)
    adamw_step(*prob[:5], lr=1e-3, weight_decay=0.0)
    _check(prob, exp, 32, torch.float32)


# ---------------------------------------------------------------- the optimizer class
def _params(device, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [nn.Parameter((torch.randn(s, generator=g) * 0.1).to(device)) for s in ((16, 512), (512, 16), (7,), (3, 5, 300))]


def test_class_matches_torch_over_steps(hip_device):
    ours, theirs = _params(hip_device), _params(hip_device)
    opts = [AdamW([{"params": ours[:2]}, {"params": ours[2:], "lr": 3e-3, "weight_decay": 0.0}], lr=1e-2, max_grad_norm=0.5),
            torch.optim.AdamW([{"params": theirs[:2]}, {"params": theirs[2:], "lr": 3e-3, "weight_decay": 0.0}], lr=1e-2)]
    g = torch.Generator(device=hip_device).manual_seed(1)
    for k in range(6):
        for a, b in zip(ours, theirs):
            a.grad = torch.randn(a.shape, device=hip_device, generator=g) if not (k == 2 and a is ours[2]) else None
            b.grad = None if a.grad is None else a.grad.clone()
        norm = torch.nn.utils.clip_grad_norm_(theirs, 0.5)
        for o in opts:
            o.step()
        assert abs(float(opts[0].grad_norm) - float(norm)) <= 1e-5 * float(norm)
    # six steps of at most lr each, every one with a relative error of 20 u and the clip factor's 1e-5 between the two norms
    for a, b, lr in zip(ours, theirs, (1e-2, 1e-2, 3e-3, 3e-3)):
        assert float((a - b).abs().max()) <= 6 * lr * 1.1 * 2e-5 + 6 * 4 * U * float(b.abs().max())


def test_gradients_that_share_memory(hip_device):
    """With each other they may; with what the step writes they may not: a block would read what another has written"""
    def prob():
        return list(_problem([(8, 8), (8, 8)], 32, torch.float32, torch.float32, 30, hip_device))

    q = prob()
    both = torch.randn(72, device=hip_device)
    q[1][0], q[1][1] = both[:64].view(8, 8), both[8:].view(8, 8)
    other = [[t.clone() for t in l] for l in q[:5]]
    adamw_step(*q[:5], lr=1e-2)
    adamw_step(*other, lr=1e-2)
    assert all(torch.equal(a, b) for a, b in zip(q[0], other[0]))
    for k in (0, 2, 3):
        q = prob()
        whole = torch.zeros(128, device=hip_device)
        q[k][1], q[1][0] = whole[:64].view(8, 8), whole[4:68].view(8, 8)
        with pytest.raises(_C.XqError, match="share"):
            adamw_step(*q[:5], lr=1e-2)
        q[1][0], q[1][1] = q[1][1], whole[60:124].view(8, 8)
        with pytest.raises(_C.XqError, match="share"):
            adamw_step(*q[:5], lr=1e-2)
        q[1][0], q[1][1], q[k][1] = q[1][0], whole[:64].view(8, 8), whole[4:68].view(8, 8)
        with pytest.raises(_C.XqError, match="share"):
            adamw_step(*q[:5], lr=1e-2)
        assert not whole.any()


def test_class_goes_on_from_torch(hip_device):
    """Two steps of torch.optim.AdamW, then two here, against four of it"""
    ours, theirs = _params(hip_device), _params(hip_device)
    first = torch.optim.AdamW(ours, lr=1e-2)
    all_theirs = torch.optim.AdamW(theirs, lr=1e-2)
    g = torch.Generator(device=hip_device).manual_seed(5)
    opt = first
    for k in range(4):
        if k == 2:
            opt = AdamW(ours)
            opt.load_state_dict(first.state_dict())
        for p, q in zip(ours, theirs):
            p.grad = torch.randn(p.shape, device=hip_device, generator=g)
            q.grad = p.grad.clone()
        opt.step()
        all_theirs.step()
    # two steps of either side: 2 roundings of the parameter each, and 16 of an update that is at most 1.1 lr after so few steps (the moments' own
    # roundings reach it enlarged by 1 / (1 - 0.9^3), hence twice the 8 operations)
    for p, q in zip(ours, theirs):
        assert (p - q).abs().max() <= 4 * 2.0 ** -24 * (2 * float(q.abs().max()) + 16 * 1.1e-2)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_class_state_dict_round_trip(hip_device, bits, dtype):
    runs = []
    for restored in (False, True):
        params = [nn.Parameter(p.detach().to(dtype)) for p in _params(hip_device)]
        opt = AdamW(params, lr=1e-2, state_bits=bits)
        g = torch.Generator(device=hip_device).manual_seed(2)
        for k in range(4):
            for p in params:
                p.grad = torch.randn(p.shape, device=hip_device, generator=g).to(dtype)
            opt.step()
            if restored and k == 1:
                saved = opt.state_dict()
                opt = AdamW(params, lr=5.0, state_bits=bits)
                opt.load_state_dict(saved)
                assert opt.param_groups[0]["lr"] == 1e-2
        runs.append((params, opt))
    for a, b in zip(*(r[0] for r in runs)):
        assert torch.equal(a, b)
    want = {"step", "exp_avg", "exp_avg_sq"} | ({"exp_avg_scale", "exp_avg_sq_scale"} if bits == 8 else set())
    for p, q in zip(*(r[0] for r in runs)):
        a, b = runs[0][1].state[p], runs[1][1].state[q]
        assert set(a) == want and all(a[k].dtype == b[k].dtype and torch.equal(a[k], b[k]) for k in want)
        assert a["exp_avg"].dtype == (torch.int8 if bits == 8 else torch.float32)


def test_class_under_the_merge_schedule(hip_device):
    m, _ = make_dense_module("block_fp8", 256, 384, 16, 32, seed=3, device=hip_device)
    model = nn.ModuleList([m])
    head = nn.Parameter(torch.randn(64, 256, device=hip_device))
    opt = AdamW([m.lora_A, m.lora_B, head], lr=1e-3, state_bits=8, max_grad_norm=1.0)
    for _ in range(2):
        for p in (m.lora_A, m.lora_B, head):
            p.grad = torch.randn_like(p)
        opt.step()
    assert reset_lora_optimizer_states(model, opt) == 2 and set(opt.state) == {head}
    opt.step()
    assert float(opt.state[m.lora_A]["step"]) == 1.0 and float(opt.state[head]["step"]) == 3.0
    maybe_merge_lora(model, enable_lora=False, enable_qlora=True, merge_interval=2, global_step=2, optimizer=opt, reset_optimizer=True)
    assert set(opt.state) == {head}
    m.lora_A.grad = torch.ones_like(m.lora_A)
    opt.step()
    assert float(opt.state[m.lora_A]["step"]) == 1.0


def test_class_in_a_graph(hip_device):
    """States are not made while a graph is captured; with states, replays are steps."""
    runs = []
    for graphed in (False, True):
        params = _params(hip_device)
        opt = AdamW(params, lr=torch.tensor(1e-2, device=hip_device), state_bits=8, max_grad_norm=1.0)
        grads = [torch.randn(p.shape, device=hip_device, generator=torch.Generator(device=hip_device).manual_seed(i)) for i, p in enumerate(params)]
        for p, g in zip(params, grads):
            p.grad = g.clone()
        graph = torch.cuda.CUDAGraph()
        if graphed:
            with pytest.raises(_C.XqError, match="before the capture"):
                with torch.cuda.graph(graph):
                    opt.step()
            graph = torch.cuda.CUDAGraph()
        opt.step()
        torch.cuda.synchronize()
        if graphed:
            with torch.cuda.graph(graph):
                opt.step()
        for k in range(3):
            for p, g in zip(params, grads):
                p.grad.copy_(g * (k + 1))
            opt.param_groups[0]["lr"].fill_(1e-2 / (k + 1))
            graph.replay() if graphed else opt.step()
            torch.cuda.synchronize()
        runs.append(params)
    for a, b in zip(*runs):
        assert torch.equal(a, b)


def test_step_is_seen_by_autograd(hip_device):
    p = nn.Parameter(torch.randn(64, device=hip_device))
    y = (p * p).sum()
    p.grad = torch.ones_like(p)
    AdamW([p], lr=1e-2).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
