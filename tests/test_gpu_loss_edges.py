"""GPU: linear_cross_entropy where the plain bounds of its other tests let a mistake through, and the calls at the edge of what it takes.

U = 2^-24, half a step of fp32; B = 2^-8, half a step of bf16."""

import pytest
import torch

from tests.test_gpu_loss import B, BF, U, _inputs, _within
from xorl_amd import _C
from xorl_amd.loss_functional import linear_cross_entropy

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- the input gradient of a head whose rows have something in common
def _shared_head(M, V, H, seed, device, share, lift):
    """A head whose rows are a common vector of `share` times their own spread and rows of their own; every token leans to a wrong one"""
    g = torch.Generator(device=device).manual_seed(seed)
    own = torch.randn(V, H, device=device, generator=g) * 0.02
    w = (own + 0.02 * share * torch.randn(H, device=device, generator=g)).to(BF)
    labels, wrong = torch.randint(0, V // 2, (M,), device=device, generator=g), torch.randint(V // 2, V, (M,), device=device, generator=g)
    x = torch.randn(M, H, device=device, generator=g) + lift * own[wrong] / (0.0004 * H)
    return x.to(BF), w, labels


def _dx_of_differences(x, w, labels, up):
    """dx by row in 64 bits, and its bound where what the rows have in common cancels.  dx = g sum_v q_v (w_v - w_t), q = p without the label's: E is off by
    the logit's error and rounded to bf16 (B), in O = sum E w and Y = sum E alike, so that both count on |w_v - w_t|; the sums in fp32 count on
    the magnitudes ((V / 32 + 64) U for O, 300 U for Y, four roundings behind them), Z on the result, which is rounded to bf16 in the end."""
    V, H = w.shape
    xd, wd = x.double(), w.double()
    l = xd @ wd.t()
    q = torch.softmax(l, 1)
    rows = torch.arange(len(labels), device=x.device)
    S = (xd.abs() @ wd.abs().t()).amax(1)
    logit = 2 * (H / 32 + 36) * U * S + 300 * U + 8 * U * (l.abs().amax(1) + l[rows, labels].abs())
    q[rows, labels] = 0.0
    want, bound = torch.empty_like(xd), torch.empty_like(xd)
    for i in range(len(labels)):
        apart = wd - wd[labels[i]]
        dx = up[i].double() * (q[i] @ apart)
        own = (B + logit[i]) * (q[i] @ apart.abs()) + (V / 32 + 368) * U * (q[i] @ wd.abs() + q[i].sum() * wd[labels[i]].abs())
        want[i] = dx
        bound[i] = 1.01 * (up[i].double().abs() * own + logit[i] * dx.abs()) + B * dx.abs() + 1e-30
    return want, bound


@pytest.mark.parametrize("M", [3, 20, 100, 300])
@pytest.mark.parametrize("lift", [6.0, 80.0])                 # 80: beyond the label's logit as the reference, so that the tiles are done again
@pytest.mark.parametrize("share", [0.0, 16.0])
def test_what_the_heads_rows_share_cancels(hip_device, M, lift, share):
    x, w, labels = _shared_head(M, 2500, 128, M, hip_device, share, lift)
    x.requires_grad_(True)
    up = torch.randn(M, device=hip_device, generator=torch.Generator(device=hip_device).manual_seed(M))
    dx, = torch.autograd.grad(linear_cross_entropy(x, w, labels, reduction="none"), x, up)
    _within(dx, _dx_of_differences(x.detach(), w, labels, up), "dx")


@pytest.mark.parametrize("lift", [6.0, 80.0])
def test_what_the_heads_rows_share_cancels_over_pieces(hip_device, lift):
    M, V = 4096, 140000
    assert 2 * M * V > 1 << 30
    x, w, labels = _shared_head(M, V, 64, 5, hip_device, 16.0, lift)
    x.requires_grad_(True)
    up = torch.linspace(-1, 1, M, device=hip_device)
    dx, = torch.autograd.grad(linear_cross_entropy(x, w, labels, reduction="none"), x, up)
    some = torch.arange(7, M, 371, device=hip_device)
    _within(dx[some], _dx_of_differences(x.detach()[some], w, labels[some], up[some]), "dx")


# ---------------------------------------------------------------- heads that are laid out otherwise
def _laid_out(w, kind):
    """The head's values where its rows cannot be read in place"""
    V, H = w.shape
    if kind == "transposed":
        return w.t().contiguous().t()
    if kind == "odd pitch":
        return torch.zeros(V, H + 3, dtype=BF, device=w.device).index_copy_(1, torch.arange(H, device=w.device), w)[:, :H]
    return torch.cat([w.new_zeros(1), w.reshape(-1)])[1:].view(V, H)          # (contiguous, two bytes behind an aligned address)


@pytest.mark.parametrize("kind", ["transposed", "odd pitch", "off by one"])
def test_layouts_that_are_copied(hip_device, kind):
    x, w, labels = _inputs(150, 700, 128, 37, hip_device)
    up = torch.randn(150, device=hip_device)
    xl, wl = _laid_out(x, kind).requires_grad_(True), _laid_out(w, kind).requires_grad_(True)
    assert torch.equal(wl, w)
    loss = linear_cross_entropy(xl, wl, labels, reduction="none")
    grads = torch.autograd.grad(loss, (xl, wl), up)
    xp, wp = x.requires_grad_(True), w.requires_grad_(True)
    want = linear_cross_entropy(xp, wp, labels, reduction="none")
    assert torch.equal(loss, want) and all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(want, (xp, wp), up)))


@pytest.mark.parametrize("kind", ["transposed", "odd pitch", "off by one"])
def test_capture_beside_a_living_loss_over_a_copied_head_is_refused(hip_device, kind):
    x, w, labels = _inputs(40, 1000, 128, 72, hip_device)
    w = _laid_out(w, kind)
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


class _Head(torch.nn.Parameter):
    pass


def test_captured_backward_of_a_subclass_is_refused(hip_device):
    """A subclass goes by the Python function, which cannot see whom torch hands its gradients to; outside a capture it has the plain one's"""
    x, w, labels = _inputs(40, 1000, 128, 73, hip_device)
    x.requires_grad_(True)
    head = _Head(w, requires_grad=False)
    with pytest.raises(RuntimeError, match="no subclasses"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(linear_cross_entropy(x, head, labels), x)
    torch.cuda.synchronize()
    got, = torch.autograd.grad(linear_cross_entropy(x, head, labels), x)
    assert torch.equal(got, torch.autograd.grad(linear_cross_entropy(x, w, labels), x)[0])


@pytest.mark.parametrize("head_grad", [False, True])
@pytest.mark.parametrize("which", [0, 1])
def test_tangents_and_transforms_are_refused(hip_device, which, head_grad):
    import torch.autograd.forward_ad as fwAD

    x, w, labels = _inputs(20, 300, 64, 74, hip_device)
    t = [x, w.requires_grad_(head_grad)]
    for grad in (True, False):
        with fwAD.dual_level(), torch.set_grad_enabled(grad), pytest.raises(NotImplementedError):
            t[which] = fwAD.make_dual((x, w)[which], torch.ones_like((x, w)[which]))
            linear_cross_entropy(*t, labels)
        t = [x, w]
    for f in (lambda: torch.func.jvp(lambda a: linear_cross_entropy(a, w, labels), (x,), (torch.ones_like(x),)),
              lambda: torch.func.grad(lambda a: linear_cross_entropy(a, w, labels))(x),
              lambda: torch.vmap(lambda a: linear_cross_entropy(a, w, labels))(x[None])):
        with pytest.raises((RuntimeError, NotImplementedError)):
            f()


def test_captured_backward_over_two_streams_of_one_capture(hip_device):
    """What comes before the loss runs on a stream that the same capture has forked: its gradients may go there"""
    x, w, labels = _inputs(40, 1000, 128, 75, hip_device)
    x.requires_grad_(True)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):
            h = x * 2.0
        here.wait_stream(side)
        loss = linear_cross_entropy(h, w, labels)
        dx, = torch.autograd.grad(loss, x)
        here.wait_stream(side)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        want = linear_cross_entropy(x * 2.0, w, labels)
        assert torch.equal(loss.detach(), want.detach()) and torch.equal(dx, torch.autograd.grad(want, x)[0])
        torch.cuda.synchronize()


# ---------------------------------------------------------------- labels that name no column, and batches of which nothing counts, by every way to list the rows
ROWS = [1, 40, 64, 65, 70, 128, 129, 300, 1024, 1025, 1100]


@pytest.mark.parametrize("M", ROWS)
@pytest.mark.parametrize("label_dtype", [torch.int64, torch.int32])
def test_labels_out_of_range_are_nan_in_their_row(hip_device, M, label_dtype):
    x, w, labels = _inputs(M, 500, 128, M, hip_device, ignored=0.2 if M > 1 else 0.0, label_dtype=label_dtype)
    names_none = [500, -1, torch.iinfo(label_dtype).max, torch.iinfo(label_dtype).min, -101]
    bad = torch.zeros(M, dtype=torch.bool, device=hip_device)
    for k, name in enumerate(names_none[:M]):
        labels[k * 13 % M], bad[k * 13 % M] = name, True
    x.requires_grad_(True)
    w.requires_grad_(True)
    with torch.no_grad():
        assert torch.equal(torch.isnan(linear_cross_entropy(x, w, labels, reduction="none")), bad)
        assert all(bool(torch.isnan(linear_cross_entropy(x, w, labels, reduction=r))) for r in ("mean", "sum"))
    for leaves in ((x,), (w,), (x, w)):
        xl, wl = (t if any(t is l for l in leaves) else t.detach() for t in (x, w))
        loss = linear_cross_entropy(xl, wl, labels, reduction="none")
        assert torch.equal(torch.isnan(loss), bad)
        grads = torch.autograd.grad(loss, leaves, torch.ones(M, device=hip_device))
        if leaves[0] is x:
            assert torch.equal(torch.isnan(grads[0]).all(1), bad) and torch.equal(torch.isfinite(grads[0]).all(1), ~bad)
        if leaves[-1] is w:
            assert bool(torch.isnan(grads[-1]).all())


@pytest.mark.parametrize("M", ROWS)
def test_nothing_counts_in_any_batch(hip_device, M):
    x, w, labels = _inputs(M, 500, 128, M, hip_device)
    labels.fill_(-100)
    x[:] = float("nan")                                       # (nothing of rows that do not count is read)
    x.requires_grad_(True)
    w.requires_grad_(True)
    for reduction in ("none", "sum", "mean"):
        def right(loss):
            return bool(torch.isnan(loss)) if reduction == "mean" else bool((loss == 0).all())

        with torch.no_grad():
            assert right(linear_cross_entropy(x, w, labels, reduction=reduction))
        for leaves in ((x,), (w,), (x, w)):
            xl, wl = (t if any(t is l for l in leaves) else t.detach() for t in (x, w))
            loss = linear_cross_entropy(xl, wl, labels, reduction=reduction)
            assert right(loss.detach())
            assert all(bool((g == 0).all()) for g in torch.autograd.grad(loss.sum(), leaves))


# ---------------------------------------------------------------- tensors that another takes the place of between forward and backward
@pytest.mark.parametrize("head", [lambda w: w, _Head])
def test_tensors_exchanged_before_the_backward_are_refused(hip_device, head):
    """`.data` and the storage change without a word to autograd; what the forward kept is as long as what it saw"""
    x, w, labels = _inputs(300, 700, 128, 76, hip_device)
    wl = head(w.clone()).requires_grad_(True)
    for which, data in ((0, x[:260]), (0, x.repeat(2, 1)), (0, x[:, :64]), (1, w[:600]), (1, w[:, :64].contiguous())):
        xl = x.clone().requires_grad_(True)
        loss = linear_cross_entropy(xl, wl, labels)
        keep = (xl, wl)[which].data
        (xl, wl)[which].data = data
        with pytest.raises(RuntimeError, match="resized between"):
            torch.autograd.grad(loss, (xl, wl))
        (xl, wl)[which].data = keep
    xl = x.clone().requires_grad_(True)
    loss = linear_cross_entropy(xl, w, labels)
    xl.untyped_storage().resize_(0)
    with pytest.raises((RuntimeError, ValueError)):
        torch.autograd.grad(loss, xl)


def test_the_backward_op_checks_what_was_kept(hip_device):
    x, w, labels = _inputs(300, 700, 128, 77, hip_device)
    loss, saved = torch.ops.xq.lce_fwd(x, w, labels, -100, 1, 1.0, 1)
    up = torch.ones((), device=hip_device)
    args = (x, w, labels)
    for grad, kept, keep in ((up, saved, 2), (up, saved[:-256], 1), (up.expand(300), saved, 1)):
        with pytest.raises(ValueError, match="not that of this problem"):
            torch.ops.xq.lce_bwd(grad, *args, kept, -100, 1, 1.0, keep, keep == 2, True)
    dw = torch.ops.xq.lce_bwd(up, *args, saved, -100, 1, 1.0, 1, False, True)[1]
    w.requires_grad_(True)
    assert torch.equal(dw, torch.autograd.grad(linear_cross_entropy(x, w, labels), w)[0])


# ---------------------------------------------------------------- infinite logits
@pytest.mark.parametrize("M", [5, 100, 300, 1100])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), 3e38])
@pytest.mark.parametrize("column", ["label", "another", "last"])
def test_infinite_logits(hip_device, M, value, column):
    """A head row that has run away, under tokens that have a 0 there but for some: NaN where the definition has infinity less infinity or 0 times
    infinity, an infinite loss where the label's logit is minus infinity"""
    V = 600
    x, w, labels = _inputs(M, V, 128, M, hip_device, lift=0.0)
    labels.random_(0, V - 1, generator=torch.Generator(device=hip_device).manual_seed(M))
    hit = torch.arange(M, device=hip_device) % 3 == 1
    labels[hit], labels[~hit] = 17, labels[~hit] % 16
    x[:, 5] = torch.where(hit, 2.0, 0.0).to(BF)
    w[:, 5] = 0.0
    w[{"label": 17, "another": 400, "last": V - 1}[column], 5] = value
    l = x.double() @ w.double().t()
    # (in fp32 a product beyond its range is infinite)
    l = torch.where(l.abs() > 3.4028235e38, l.sign() * float("inf"), l)
    want = torch.nn.functional.cross_entropy(l, labels, reduction="none")
    x.requires_grad_(True)
    with torch.no_grad():
        score = linear_cross_entropy(x, w, labels, reduction="none")
    loss = linear_cross_entropy(x, w, labels, reduction="none")
    for got in (score, loss.detach()):
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isposinf(got), torch.isposinf(want))
        fine = torch.isfinite(want)
        assert bool(((got.double() - want)[fine].abs() <= 1e-4 * want[fine].abs()).all())
    dx, = torch.autograd.grad(loss.sum(), x)
    assert bool(torch.isnan(dx[torch.isnan(want)]).all(1).all())


def test_tensors_exchanged_by_a_number_are_looked_at_afterwards(hip_device):
    x, w, labels = _inputs(300, 700, 128, 78, hip_device)
    short = x[:, :64].clone()

    class Number:
        def __float__(self):
            x.data = short
            return 1.0

    with pytest.raises(_C.XqError, match="do not go together"):
        linear_cross_entropy(x, w, labels, logit_scale=Number())


# ---------------------------------------------------------------- what autograd offers around a node
def test_saved_tensor_hooks(hip_device):
    """Checkpointing and saving on the CPU give the same gradients; a hook that gives back something shorter is refused"""
    from torch.utils.checkpoint import checkpoint

    x, w, labels = _inputs(300, 700, 128, 79, hip_device, ignored=0.2)
    x.requires_grad_(True)
    w.requires_grad_(True)

    def f(x, w):
        return linear_cross_entropy(x * 2.0, w, labels)

    loss = f(x, w)
    want = torch.autograd.grad(loss, (x, w))
    again = checkpoint(f, x, w, use_reentrant=False)
    assert torch.equal(again, loss) and all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(again, (x, w)), want))
    with torch.autograd.graph.save_on_cpu():
        again = f(x, w)
    assert torch.equal(again, loss) and all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(again, (x, w)), want))
    for shorten in (lambda t: t[:-256], lambda t: t.cpu()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: shorten(t) if t.dtype == torch.uint8 else t):
            again = f(x, w)
        with pytest.raises(RuntimeError, match="hooks of saved tensors"):
            torch.autograd.grad(again, (x, w))


def test_batched_upstream_gradients_are_refused(hip_device):
    x, w, labels = _inputs(40, 300, 64, 80, hip_device)
    x.requires_grad_(True)
    for reduction, shape in (("sum", (2,)), ("none", (2, 40))):
        loss = linear_cross_entropy(x, w, labels, reduction=reduction)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(loss, x, torch.ones(shape, device=hip_device), is_grads_batched=True)


def test_fake_tensors_are_refused(hip_device):
    from torch._subclasses.fake_tensor import FakeTensorMode

    x, w, labels = _inputs(40, 300, 64, 81, hip_device)
    with FakeTensorMode() as mode, pytest.raises(Exception):
        linear_cross_entropy(*(mode.from_tensor(t) for t in (x, w, labels)))
