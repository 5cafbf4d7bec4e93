"""GPU: linear_cross_entropy against the cross entropy and its gradients in 64 bits.

Bounds.  U = 2^-24, half a step of fp32; B = 2^-8, half a step of bf16.  A logit is a sum of H exact products in fp32, 32 in one
instruction and H / 32 of those one after the other, then scaled: off by at most d = (H / 32 + 36) U S, S = c max_v sum_k |x_k w_vk|, and 4 U
of its size.  The loss moves by (1 - p_t) times the error of the label's logit against the others', 2 d; the sum of exponentials (an
exponential within 4 U, chains of at most 64 + V / 4096 sums, 300 U in all) counts the same way, and rounding the loss 4 U of it.
dx = g c sum_v (p_v - [v = t]) w_v: every p is off by (2 d + 300 U) and rounded to bf16 (B), the sum over V adds (V / 32 + 64) U, the result is
rounded to bf16; all of it counts on the sum of magnitudes.  dw the same with the sum over the rows."""

import math

import pytest
import torch

from oracle import recipe as R
from tests.util_cases import make_dense_module
from xorl_amd import _C
from xorl_amd.loss_functional import linear_cross_entropy
from xorl_amd.optim import AdamW

pytestmark = pytest.mark.gpu
U, B = 2.0 ** -24, 2.0 ** -8
BF = torch.bfloat16


def _inputs(M, V, H, seed, device, std=0.02, lift=8.0, ignored=0.0, label_dtype=torch.int64):
    g = torch.Generator(device=device).manual_seed(seed)
    w = (torch.randn(V, H, device=device, generator=g) * std).to(BF)
    labels = torch.randint(0, V, (M,), device=device, generator=g)
    x = torch.randn(M, H, device=device, generator=g)
    x = (x + torch.rand(M, 1, device=device, generator=g) * lift * w[labels].float() / (std * std * H)).to(BF)
    labels[torch.rand(M, device=device, generator=g) < ignored] = -100
    return x, w, labels.to(label_dtype)


def _reference(x, w, labels, up, scale=1.0):
    """Loss by row, dx, dw in 64 bits for upstream gradients `up` by row, and their bounds."""
    M, H = x.shape
    V = w.shape[0]
    valid = labels != -100
    lab = labels.long().where(valid, 0)
    xd, wd = x.double(), w.double()
    l = scale * xd @ wd.t()
    logp = l - torch.logsumexp(l, 1, keepdim=True)
    p = logp.exp()
    onehot = torch.zeros_like(p).scatter_(1, lab[:, None], 1.0)
    # 1 - p_t without cancellation
    rest = (p * (1 - onehot)).sum(1)
    lt = l.gather(1, lab[:, None])[:, 0]
    loss = torch.where(rest < 0.5, -torch.log1p(-rest), -logp.gather(1, lab[:, None])[:, 0])
    S = scale * (xd.abs() @ wd.abs().t()).amax(1)
    top = l.abs().amax(1)
    logit = 2 * (H / 32 + 36) * U * S + 300 * U + 8 * U * (top + lt.abs())
    q = p * (1 - onehot) - rest[:, None] * onehot
    up = up.double().where(valid, 0) * scale
    dx = up[:, None] * (q @ wd)
    dx_b = (up.abs() * (B + 2 * logit + (V / 32 + 64) * U))[:, None] * (q.abs() @ wd.abs()) + B * dx.abs() + 1e-30
    dw = (up[:, None] * q).t().contiguous() @ xd
    dw_b = (up.abs()[:, None] * q.abs() * (B + 2 * logit + (M / 32 + 64) * U)[:, None]).t().contiguous() @ xd.abs() + B * dw.abs() + 1e-30
    zero = torch.zeros_like(loss)
    return (loss.where(valid, zero), (rest * logit + 4 * U * loss).where(valid, zero) + 1e-30), (dx, dx_b), (dw, dw_b), valid


def _within(got, pair, what):
    want, bound = pair
    off = (got.double() - want).abs() - bound
    assert bool(torch.isfinite(got).all()), what
    assert bool((off <= 0).all()), f"{what}: {int((off > 0).sum())} of {off.numel()} beyond their bound, by up to {float((off / bound).max())} of it"


def _case(x, w, labels, reduction="none", scale=1.0, head=True):
    """Loss, dx and dw of one call against the reference"""
    M = labels.numel()
    xl, wl = x.detach().requires_grad_(True), w.detach().requires_grad_(head)
    n = int((labels != -100).sum())
    g = torch.Generator(device=x.device).manual_seed(99)
    up = torch.randn(M, device=x.device, generator=g) if reduction == "none" else torch.full((M,), 1.0 / n if reduction == "mean" else 1.0, device=x.device)
    ref = _reference(x.reshape(-1, x.shape[-1]), w, labels.reshape(-1), up if reduction != "mean" else torch.full((M,), 1.0 / n, dtype=torch.float64, device=x.device), scale)
    with torch.no_grad():
        score = linear_cross_entropy(xl, wl, labels, reduction=reduction, logit_scale=scale)
    loss = linear_cross_entropy(xl, wl, labels, reduction=reduction, logit_scale=scale)
    assert loss.dtype == torch.float32
    want = ref[0]
    if reduction != "none":
        k = 1.0 / n if reduction == "mean" else 1.0
        want = (want[0].sum() * k, want[1].sum() * k + 2 * U * want[0].sum() * k)
    for name, got in (("score", score), ("loss", loss)):
        assert got.shape == (labels.shape if reduction == "none" else ())
        _within(got.detach().reshape(-1) if reduction == "none" else got.detach(), want, name)
    grads = torch.autograd.grad(loss, (xl, wl) if head else (xl,), up.view(labels.shape) if reduction == "none" else None)
    assert grads[0].dtype == BF and grads[0].shape == x.shape
    # (the upstream factor of a mean: a division more)
    _within(grads[0].reshape(ref[1][0].shape), (ref[1][0], ref[1][1] * (1 + 4 * U) + 4 * U * ref[1][0].abs()), "dx")
    if head:
        assert grads[1].dtype == BF and grads[1].shape == w.shape
        _within(grads[1], (ref[2][0], ref[2][1] * (1 + 4 * U) + 4 * U * ref[2][0].abs()), "dw")
    ignored = (labels == -100).reshape(-1)
    if reduction == "none":
        assert bool((loss.detach().reshape(-1)[ignored] == 0).all())
    assert bool((grads[0].reshape(M, -1)[ignored] == 0).all())


@pytest.mark.parametrize("M", [1, 2, 63, 64, 65, 127, 128, 129, 256, 257, 700])
@pytest.mark.parametrize("V,H", [(1000, 192), (4099, 128)])
def test_rows(hip_device, M, V, H):
    _case(*_inputs(M, V, H, M + V, hip_device))


@pytest.mark.parametrize("V", [1, 2, 31, 32, 33, 255, 256, 257, 511, 513, 32003])
@pytest.mark.parametrize("M", [5, 200, 300])
def test_vocabularies(hip_device, M, V):
    _case(*_inputs(M, V, 128, V, hip_device, std=0.1))


@pytest.mark.parametrize("H", [64, 128, 192, 256, 320, 448, 1024, 2048, 4096, 5120])
@pytest.mark.parametrize("M", [3, 130, 260])
def test_hidden_sizes(hip_device, M, H):
    _case(*_inputs(M, 777, H, H, hip_device))


@pytest.mark.parametrize("M,V,H", [(40, 70001, 128), (100, 70001, 128), (100, 70001, 64), (128, 40000, 192), (64, 140001, 64), (1, 66000, 320), (1100, 3000, 128),
                                   (300, 66000, 64), (513, 20000, 192), (90, 9000, 256), (33, 9000, 256)])
@pytest.mark.parametrize("far", [False, True])
def test_tiles_of_every_kind(hip_device, M, V, H, far):
    """Several tiles a block, narrow and wide ones, contractions shorter than the loads are ahead; and done again for logits far apart"""
    x, w, labels = _inputs(M, V, H, M + V + H, hip_device, std=0.05, ignored=0.1)
    if far:
        w[V // 2:V // 2 + 40] = (w[V // 2:V // 2 + 40].float() * 300).to(BF)
        w[V - 3:] = (w[V - 3:].float() * 500).to(BF)
    if M == 1:
        labels.clamp_(min=0)
    _case(x, w, labels, "none")


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("scale", [1.0, 0.3, 2.5])
@pytest.mark.parametrize("label_dtype", [torch.int64, torch.int32])
def test_reductions_scales_label_types(hip_device, reduction, scale, label_dtype):
    x, w, labels = _inputs(330, 2500, 256, 7, hip_device, ignored=0.3, label_dtype=label_dtype)
    _case(x.view(3, 110, 256), w, labels.view(3, 110), reduction, scale)


@pytest.mark.parametrize("M", [1, 40, 600])
@pytest.mark.parametrize("pattern", ["first", "last", "all but one", "every other"])
def test_ignored_rows(hip_device, M, pattern):
    x, w, labels = _inputs(M, 900, 128, 11, hip_device)
    keep = torch.arange(M, device=hip_device)
    drop = {"first": keep < M // 2, "last": keep >= (M + 1) // 2, "all but one": keep != M // 3, "every other": keep % 2 == 1}[pattern]
    labels[drop] = -100
    _case(x, w, labels, "sum")


def test_nothing_counts(hip_device):
    x, w, labels = _inputs(70, 500, 128, 13, hip_device)
    labels.fill_(-100)
    x.requires_grad_(True)
    w.requires_grad_(True)
    for reduction in ("none", "sum", "mean"):
        loss = linear_cross_entropy(x, w, labels, reduction=reduction)
        assert bool(torch.isnan(loss)) if reduction == "mean" else bool((loss == 0).all())
        dx, dw = torch.autograd.grad(loss.sum(), (x, w))
        assert bool((dx == 0).all()) and bool((dw == 0).all())
    other = linear_cross_entropy(x, w, torch.full_like(labels, 7), ignore_index=7, reduction="sum")
    assert float(other) == 0.0


def test_no_rows(hip_device):
    x, w = torch.zeros(0, 128, dtype=BF, device=hip_device, requires_grad=True), torch.ones(40, 128, dtype=BF, device=hip_device, requires_grad=True)
    labels = torch.zeros(0, dtype=torch.int64, device=hip_device)
    loss = linear_cross_entropy(x, w, labels, reduction="none")
    assert loss.shape == (0,)
    assert math.isnan(float(linear_cross_entropy(x, w, labels).detach()))
    total = linear_cross_entropy(x, w, labels, reduction="sum")
    dx, dw = torch.autograd.grad(total, (x, w))
    assert float(total.detach()) == 0.0 and dx.shape == x.shape and bool((dw == 0).all())


def test_labels_out_of_range_are_nan(hip_device):
    x, w, labels = _inputs(70, 500, 128, 17, hip_device)
    labels[3], labels[50] = 500, -1
    x.requires_grad_(True)
    bad = torch.zeros(70, dtype=torch.bool, device=hip_device)
    bad[[3, 50]] = True
    for grad in (False, True):
        with torch.set_grad_enabled(grad):
            loss = linear_cross_entropy(x, w, labels, reduction="none")
        assert bool((torch.isnan(loss) == bad).all())
    dx, = torch.autograd.grad(loss.sum(), x)
    assert bool((torch.isnan(dx).all(1) == bad).all()) and bool((torch.isfinite(dx).all(1) == ~bad).all())
    assert math.isnan(float(linear_cross_entropy(x, w, labels).detach()))


def test_nan_row_stays_its_own(hip_device):
    x, w, labels = _inputs(300, 1500, 128, 19, hip_device)
    x[299, 5] = float("nan")
    x[7, 5] = float("inf")
    x.requires_grad_(True)
    bad = torch.zeros(300, dtype=torch.bool, device=hip_device)
    bad[[7, 299]] = True
    with torch.no_grad():
        score = linear_cross_entropy(x, w, labels, reduction="none")
    loss = linear_cross_entropy(x, w, labels, reduction="none")
    dx, = torch.autograd.grad(loss.sum(), x)
    assert bool((torch.isfinite(score) == ~bad).all()) and bool((torch.isfinite(loss) == ~bad).all())
    assert bool((torch.isfinite(dx).all(1) == ~bad).all())


@pytest.mark.parametrize("where", ["all", "last tile", "label far below", "label far above"])
@pytest.mark.parametrize("M", [20, 300])
def test_logits_far_apart(hip_device, where, M):
    """Logits of some hundred: beyond the reference by more than an exponential in fp32 or bf16 can hold."""
    x, w, labels = _inputs(M, 3000, 256, 23, hip_device, lift=0.0)
    if where == "all":
        w = (w.float() * 30).to(BF)
    elif where == "last tile":
        w[2990:] = (w[2990:].float() * 60).to(BF)
    else:
        sign = -1.0 if where == "label far below" else 1.0
        x = (x.float() + sign * 100 * w[labels].float() / (0.02 * 0.02 * 256)).to(BF)
    _case(x, w, labels)


def test_confident_rows_keep_small_losses(hip_device):
    """A loss of 1e-9 and its gradient, where 1 - p_t has nothing left in fp32."""
    x, w, labels = _inputs(100, 1000, 256, 29, hip_device, lift=0.0)
    x = (0.1 * x.float() + 30 * w[labels].float() / (0.02 * 0.02 * 256)).to(BF)
    _case(x, w, labels)
    # (that the inputs are what this is about: by the reference, most of the losses are below what 1 - p_t resolves)
    losses = _reference(x, w, labels, torch.ones(100, device=hip_device))[0][0]
    assert float(losses.median()) < U and float(losses.min()) > 0.0


@pytest.mark.parametrize("far", [False, True])
def test_several_pieces(hip_device, far):
    """More of the vocabulary than one piece holds; the later ones with larger logits than their reference allows."""
    M, V, H = 4096, 140000, 64
    assert 2 * M * V > 1 << 30
    x, w, labels = _inputs(M, V, H, 31, hip_device, std=0.05, ignored=0.2)
    if far:
        w[100000:100200] = (w[100000:100200].float() * 300).to(BF)
        w[139000:] = (w[139000:].float() * 500).to(BF)
    _chunked(x, w, labels)


def _chunked(x, w, labels, rows=256):
    """_case by rows, for sizes whose logits in 64 bits are too many at a time"""
    xl, wl = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = linear_cross_entropy(xl, wl, labels, reduction="none")
    up = torch.linspace(-1, 1, labels.numel(), device=x.device)
    dx, dw = torch.autograd.grad(loss, (xl, wl), up)
    want, bound = 0.0, 0.0
    for a in range(0, labels.numel(), rows):
        s = slice(a, a + rows)
        ref = _reference(x[s], w, labels[s], up[s])
        _within(loss.detach()[s], ref[0], "loss")
        _within(dx[s], ref[1], "dx")
        want, bound = want + ref[2][0], bound + ref[2][1]
    # (the sum over all rows is one of M / 32 terms)
    _within(dw, (want, bound * (1 + labels.numel() * U) + B * want.abs()), "dw")


def test_strides(hip_device):
    M, V, H = 150, 700, 128
    x, w, labels = _inputs(M, V, H, 37, hip_device)
    wide, tall = torch.randn(M, 3 * H, device=hip_device).to(BF), torch.randn(V, 2 * H, device=hip_device).to(BF)
    wide[:, H:2 * H], tall[:, :H] = x, w
    up = torch.randn(M, device=hip_device)
    ref = _reference(x, w, labels, up)
    odd = torch.empty(M * (H + 3) + 1, dtype=BF, device=hip_device)[1:].view(M, H + 3)[:, :H]
    odd.copy_(x)
    for xv, wv in ((wide[:, H:2 * H], tall[:, :H]), (odd, w), (x.t().contiguous().t(), w.t().contiguous().t())):
        xl, wl = xv.detach().requires_grad_(True), wv.detach().requires_grad_(True)
        loss = linear_cross_entropy(xl, wl, labels.repeat_interleave(2)[::2], reduction="none")
        dx, dw = torch.autograd.grad(loss, (xl, wl), up)
        _within(loss.detach(), ref[0], "loss")
        _within(dx, ref[1], "dx")
        _within(dw, ref[2], "dw")


def test_rows_far_apart_in_memory(hip_device):
    """Rows whose offsets pass 2^32 bytes, in x and in the head"""
    M, V, H = 2300, 600, 64
    x, w, labels = _inputs(M, V, H, 41, hip_device)
    big = torch.empty(M, 1 << 20, dtype=BF, device=hip_device)
    big[:, 64:128] = x
    up = torch.ones(M, device=hip_device)
    ref = _reference(x, w, labels, up)
    xl = big[:, 64:128].requires_grad_(True)
    loss = linear_cross_entropy(xl, w.requires_grad_(True), labels, reduction="none")
    dx, dw = torch.autograd.grad(loss.sum(), (xl, w))
    _within(loss.detach(), ref[0], "loss")
    _within(dx, ref[1], "dx")
    _within(dw, ref[2], "dw")
    del big, xl, loss, dx, dw
    M, V, H = 70, 5000, 64
    x, w, labels = _inputs(M, V, H, 43, hip_device)
    big = torch.empty(V, 1 << 19, dtype=BF, device=hip_device)
    big[:, :64] = w
    ref = _reference(x, w, labels, torch.ones(M, device=hip_device))
    xl = x.requires_grad_(True)
    loss = linear_cross_entropy(xl, big[:, :64], labels, reduction="none")
    dx, = torch.autograd.grad(loss.sum(), xl)
    _within(loss.detach(), ref[0], "loss")
    _within(dx, ref[1], "dx")


def test_only_what_is_asked_for(hip_device):
    x, w, labels = _inputs(90, 600, 128, 47, hip_device, ignored=0.1)
    up = torch.randn(90, device=hip_device)
    ref = _reference(x, w, labels, up)
    for gx, gw in ((True, False), (False, True), (True, True)):
        xl, wl = x.detach().requires_grad_(gx), w.detach().requires_grad_(gw)
        loss = linear_cross_entropy(xl, wl, labels, reduction="none")
        loss.backward(up)
        if gx:
            _within(xl.grad, ref[1], "dx")
        if gw:
            _within(wl.grad, ref[2], "dw")
        assert (xl.grad is not None) == gx and (wl.grad is not None) == gw
    assert not linear_cross_entropy(x, w, labels).requires_grad


def test_gradients_against_differences(hip_device):
    """A directional derivative of the loss, by differences of the function in 64 bits at the kernel's own inputs"""
    x, w, labels = _inputs(40, 300, 64, 53, hip_device)
    xl, wl = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = linear_cross_entropy(xl, wl, labels, logit_scale=0.7)
    dx, dw = torch.autograd.grad(loss, (xl, wl))
    g = torch.Generator(device=hip_device).manual_seed(1)
    vx, vw = torch.randn(x.shape, device=hip_device, generator=g).double(), torch.randn(w.shape, device=hip_device, generator=g).double()

    def f(t):
        z = 0.7 * (x.double() + t * vx) @ (w.double() + t * vw).t()
        return float((torch.logsumexp(z, 1) - z.gather(1, labels[:, None])[:, 0]).mean())

    h = 1e-5
    slope = (f(h) - f(-h)) / (2 * h)
    got = float((dx.double() * vx).sum() + (dw.double() * vw).sum())
    bx, bw = (r[1] for r in _reference(x, w, labels, torch.full((40,), 1 / 40, device=hip_device, dtype=torch.float64), 0.7)[1:3])
    assert abs(got - slope) <= float((bx * vx.abs()).sum() + (bw * vw.abs()).sum()) + 1e-6 * abs(slope)


def _exact_head_gradient(x, w, labels, up):
    """The head's gradient in 64 bits, and the sum of its terms' magnitudes"""
    xd, wd = x.double(), w.double()
    p = torch.softmax(xd @ wd.t(), -1)
    p[torch.arange(len(labels), device=x.device), labels] -= 1
    p *= up.double()[:, None]
    return p.t() @ xd, p.abs().t() @ xd.abs()


@pytest.mark.parametrize("M", [1, 2, 31, 32, 33, 64, 65, 96, 97, 128])
def test_head_gradient_of_few_tokens_is_rounded_once(hip_device, M):
    """Half a step of the result (2^-8); G in two bf16 numbers (2^-16 of each term), products in fp32 (at most 256 sums of 2^-24 each), p to the
    logits' own error: 192 sums of 2^-24 of the magnitudes of a logit's terms, in numerator and denominator, and ten roundings of the exponential"""
    x, w, labels = _inputs(M, 1500, 192, 300 + M, hip_device, std=0.05)
    labels[M // 2] = labels[0]                                # (two tokens of one row)
    w.requires_grad_(True)
    up = torch.randn(M, device=hip_device, generator=torch.Generator(device=hip_device).manual_seed(M))
    dw, = torch.autograd.grad(linear_cross_entropy(x, w, labels, reduction="none"), w, up)
    want, terms = _exact_head_gradient(x, w.detach(), labels, up)
    logit_terms = float((x.double().abs() @ w.detach().double().abs().t()).max())
    near = 2.0 ** -16 + 256 * U + 2 * (192 * logit_terms + 10) * U
    assert bool(((dw.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1.01 * near * terms + 1e-37).all())


@pytest.mark.parametrize("reduction,M,grad", [("mean", 255, 1.0), ("mean", 100, 1.0), ("sum", 255, 257 / 256), ("sum", 300, 1.0)])
def test_what_all_rows_share_is_not_rounded(hip_device, reduction, M, grad):
    """1 / 255 and 257 / 256 lie in the middle between two bf16 numbers: rounded, the whole gradient would be off by 2^-8.  What may stay of that is the label's
    1 - p, off by the largest p where it rounds to 1 (upstream gradients by row are rounded with it)"""
    x, w, labels = _inputs(M, 4096, 128, 400 + M, hip_device, std=0.01, lift=0.0)
    w.requires_grad_(True)
    dw, = torch.autograd.grad(linear_cross_entropy(x, w, labels, reduction=reduction), w, torch.tensor(grad, device=hip_device))
    up = torch.full((M,), grad / (M if reduction == "mean" else 1), dtype=torch.float64, device=hip_device)
    want, _ = _exact_head_gradient(x, w.detach(), labels, up)
    p = float(torch.softmax(x.double() @ w.detach().double().t(), -1).max())
    assert p < 2.0 ** -10
    off = float((dw.double() * want).sum() / (want * want).sum()) - 1
    # the result's own roundings are of either sign: 2^-8 / sqrt of half a million elements
    assert abs(off) <= p + 2.0 ** -8 / 128


def test_backward_twice_and_expanded_upstream(hip_device):
    x, w, labels = _inputs(100, 800, 128, 59, hip_device)
    x.requires_grad_(True)
    w.requires_grad_(True)
    loss = linear_cross_entropy(x, w, labels, reduction="none")
    a = torch.autograd.grad(loss.sum(), (x, w), retain_graph=True)          # (the sum's gradient is one element, expanded)
    b = torch.autograd.grad(loss, (x, w), torch.ones(100, device=hip_device))
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_same_bits_twice_and_on_another_stream(hip_device):
    x, w, labels = _inputs(500, 5000, 256, 61, hip_device, ignored=0.2)
    x.requires_grad_(True)
    w.requires_grad_(True)
    outs = []
    for stream in (None, None, torch.cuda.Stream()):
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            loss = linear_cross_entropy(x, w, labels)
            outs.append((loss.detach(), *torch.autograd.grad(loss, (x, w))))
        torch.cuda.synchronize()
    for o in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], o))


@pytest.mark.parametrize("M", [8, 300])
def test_captured_step_with_changing_inputs(hip_device, M):
    x, w, labels = _inputs(M, 3000, 128, 67, hip_device)
    xs, ws, ls = x.clone().requires_grad_(True), w.clone().requires_grad_(True), labels.clone()

    def step():
        loss = linear_cross_entropy(xs, ws, ls)
        return (loss.detach(), *torch.autograd.grad(loss, (xs, ws)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        nx, nw, nl = _inputs(M, 3000, 128, 70 + k, hip_device, ignored=0.2 * k)
        with torch.no_grad():
            xs.copy_(nx)
            ws.copy_(nw * (1 if k != 2 else 40))                # (one replay whose logits lie far apart)
            ls.copy_(nl)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


def test_graph_captured_without_a_first_call(hip_device):
    """Shapes that no other call here has: nothing is left to be set up by a first call outside the graph"""
    x, w, labels = _inputs(77, 2345, 448, 71, hip_device)
    x.requires_grad_(True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = linear_cross_entropy(x, w, labels)
        dx, = torch.autograd.grad(loss, x)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        want = linear_cross_entropy(x, w, labels)
        assert torch.equal(loss.detach(), want.detach()) and torch.equal(dx, torch.autograd.grad(want, x)[0])


def test_capture_beside_a_living_loss_is_refused(hip_device):
    """Nothing is handed to the stream of the loss outside; what went before and comes after is as it was"""
    x, w, labels = _inputs(40, 1000, 128, 72, hip_device)
    x.requires_grad_(True)
    eager = linear_cross_entropy(x, w, labels)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="another stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(linear_cross_entropy(x, w, labels), x)
    torch.cuda.synchronize()
    want, = torch.autograd.grad(eager, x)
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dx, = torch.autograd.grad(linear_cross_entropy(x, w, labels), x)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dx, want)


def test_two_calls_at_once(hip_device):
    problems = [_inputs(M, 6000, 256, 80 + M, hip_device) for M in (400, 30)]
    want = []
    for x, w, labels in problems:
        x.requires_grad_(True)
        loss = linear_cross_entropy(x, w, labels)
        want.append((loss.detach(), *torch.autograd.grad(loss, x)))
    streams = [torch.cuda.Stream() for _ in problems]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for (x, w, labels), s in zip(problems, streams):
            with torch.cuda.stream(s):
                loss = linear_cross_entropy(x, w, labels)
                got.append((loss.detach(), *torch.autograd.grad(loss, x)))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, q in zip(got, want) for a, b in zip(g, q))


def test_under_compile(hip_device):
    x, w, labels = _inputs(60, 700, 128, 91, hip_device)
    x.requires_grad_(True)

    def f(x, w, labels):
        return linear_cross_entropy(x * 1.0, w, labels, reduction="sum")

    want = f(x, w, labels)
    dx, = torch.autograd.grad(want, x)
    torch._dynamo.reset()
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(x, w, labels)
    assert torch.equal(got, want) and torch.equal(torch.autograd.grad(got, x)[0], dx)
    with torch.no_grad():
        a = torch.compile(f, backend="aot_eager", fullgraph=True)(x, w, labels)
    assert torch.equal(a, f(x.detach(), w, labels))


def test_refusals_on_the_device(hip_device):
    x, w, labels = _inputs(10, 100, 64, 97, hip_device)
    with pytest.raises(RuntimeError, match="HIP device only"):
        linear_cross_entropy(x, w.cpu(), labels)
    with pytest.raises(RuntimeError, match="HIP device only"):
        linear_cross_entropy(x, w, labels.cpu())
    with pytest.raises(_C.XqError, match="must be bf16"):
        linear_cross_entropy(x.float(), w, labels)
    x.requires_grad_(True)
    loss = linear_cross_entropy(x, w, labels)
    g, = torch.autograd.grad(loss, x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_training_step_of_a_quantized_layer(hip_device):
    """What they are for, together: a packed projection, the head's loss, and the step of the factors; against the oracle's gradients of
    the projection and the update in 64 bits."""
    tokens, d_in, d_out, V, r = 200, 384, 256, 3001, 16
    m, w_ref = make_dense_module("block_fp8", d_out, d_in, r, 32, seed=3, device=hip_device)
    with torch.no_grad():
        m.lora_B.normal_(0, 0.02)
    x, head, labels = _inputs(tokens, V, d_out, 101, hip_device, std=0.05, ignored=0.25)
    inp = torch.randn(tokens, d_in, device=hip_device).to(BF)
    opt = AdamW([m.lora_A, m.lora_B], lr=1e-2, weight_decay=0.1, max_grad_norm=0.5)
    for k in range(3):
        before = [p.detach().double().clone() for p in (m.lora_A, m.lora_B)]
        states = [{n: s.clone() for n, s in opt.state[p].items()} for p in (m.lora_A, m.lora_B)]
        opt.zero_grad()
        y = m(inp)
        y.retain_grad()
        loss = linear_cross_entropy(y, head, labels)
        loss.backward()
        n = int((labels != -100).sum())
        ref = _reference(y.detach(), head, labels, torch.full((tokens,), 1.0 / n, dtype=torch.float64, device=hip_device))
        _within(loss.detach(), (ref[0][0].sum() / n, ref[0][1].sum() / n + 2 * U * ref[0][0].sum() / n), "loss")
        _within(y.grad, (ref[1][0], ref[1][1] * (1 + 4 * U)), "dy")
        ex = R.linear_fwd_bwd_exact(inp.cpu(), w_ref, m.lora_A.detach().cpu(), m.lora_B.detach().cpu(), m.scaling, y.grad.cpu())
        for name, p in (("dA", m.lora_A), ("dB", m.lora_B)):
            assert R.max_rel_err(p.grad.cpu(), ex[name]) <= 1e-2, name
        grads = [p.grad.double() for p in (m.lora_A, m.lora_B)]
        norm = torch.cat([g.reshape(-1) for g in grads]).norm()
        opt.step()
        assert abs(float(opt.grad_norm) - float(norm)) <= 2 * U * float(norm)
        f = min(1.0, 0.5 / (float(norm) + 1e-6))
        for p, w0, s, g in zip((m.lora_A, m.lora_B), before, states, grads):
            g = g * f
            m1 = 0.9 * (s["exp_avg"].double() if s else 0) + 0.1 * g
            v1 = 0.999 * (s["exp_avg_sq"].double() if s else 0) + 0.001 * g * g
            mag = 0.9 * (s["exp_avg"].double().abs() if s else 0) + 0.1 * g.abs()
            den = v1.sqrt() / (1 - 0.999 ** (k + 1)) ** 0.5 + 1e-8
            want = w0 - 1e-2 * 0.1 * w0 - 1e-2 / (1 - 0.9 ** (k + 1)) * m1 / den
            bound = 4 * U * w0.abs() + 18 * U * 1e-2 / (1 - 0.9 ** (k + 1)) * mag / den + 1e-30
            assert bool(((p.detach().double() - want).abs() <= bound).all())
