"""GPU: the optimizer step at the edge of what it takes."""

import threading

import pytest
import torch

from tests.test_gpu_fsdp2 import one_rank_group  # noqa: F401
from tests.test_gpu_optim import SIZES, U, _problem
from tests.util_cases import make_dense_module
from xorl_amd import _C
from xorl_amd.optim import AdamW, adamw_state_values, adamw_step, grad_norm

pytestmark = pytest.mark.gpu


def _step(prob, **kw):
    return adamw_step(*prob[:5], exp_avg_scales=prob[5], exp_avg_sq_scales=prob[6], **{"lr": 1e-3, **kw})


def _same(a, b):
    return all(x is None or all(torch.equal(s, t) for s, t in zip(x, y)) for x, y in zip(a, b))


# ---------------------------------------------------------------- lists that change
@pytest.mark.parametrize("bits", [32, 8])
def test_lists_that_a_callback_empties(hip_device, bits):
    """The clip's number is of a class whose conversion drops every tensor of the caller's lists (others stand for the same memory)"""
    prob, want = (_problem(SIZES, bits, torch.float32, torch.float32, 51, hip_device) for _ in range(2))
    shown = [None if l is None else [t.detach() for t in l] for l in prob]
    class Number:
        def __float__(self):
            for l in shown:
                if l is not None:
                    l[:] = []
            return 0.05

    norm = _step(shown, max_norm=Number())
    assert torch.equal(norm, _step(want, max_norm=0.05)) and _same(prob, want) and len(shown[0]) == 0


def test_lists_that_another_thread_changes(hip_device):
    prob = _problem([(300,)] * 200, 32, torch.float32, torch.float32, 52, hip_device)
    shown, done = [list(l) for l in prob[:5]], threading.Event()

    def change():
        while not done.is_set():
            for l, own in zip(shown, prob):
                for i in range(len(l)):
                    l[i] = own[i].detach()          # (another object over the same memory; the one before goes)

    thread = threading.Thread(target=change)
    thread.start()
    try:
        for _ in range(100):
            adamw_step(*shown, lr=1e-3)
    finally:
        done.set()
        thread.join()
    assert [float(t) for t in prob[4]] == [103.0 + 7 * (i % 5) for i in range(200)]


# ---------------------------------------------------------------- tensors without elements
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("shapes", [[(0,)], [(0, 3), (5,), (0,)], [(300,), (0,), (4097,), (7, 0)]])
@pytest.mark.parametrize("clip", [None, 0.01])
def test_tensors_without_elements_count_their_steps(hip_device, bits, shapes, clip):
    """like the others (a rank's share of a sharded parameter may be empty), and change nothing for them"""
    prob, want = (_problem(shapes, bits, torch.float32, torch.float32, 53, hip_device) for _ in range(2))
    before = [float(t) for t in prob[4]]
    versions = [t._version for t in prob[4]]
    norm = _step(prob, max_norm=clip)
    assert [float(t) for t in prob[4]] == [b + 1 for b in before] and all(t._version > v for t, v in zip(prob[4], versions))
    some = [i for i, s in enumerate(shapes) if 0 not in s]
    short, full = ([None if l is None else [l[i] for i in some] for l in q] for q in (prob, want))
    if some:
        assert clip is None or torch.equal(norm, grad_norm(full[1]))
        _step(full, max_norm=clip)
        assert _same(short, full)


def test_tensors_without_elements_in_a_graph(hip_device):
    prob = _problem([(0,), (9,), (0, 4)], 32, torch.float32, torch.float32, 54, hip_device)
    before = [float(t) for t in prob[4]]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _step(prob)
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert [float(t) for t in prob[4]] == [b + k + 1 for b in before]


# ---------------------------------------------------------------- modules under FSDP2, one rank
@pytest.mark.parametrize("bits", [32, 8])
def test_factors_under_fsdp2(hip_device, one_rank_group, bits):
    """The steps of a wrapped module's factors are the plain module's; a distributed checkpoint's state dictionary goes round"""
    from torch.distributed._composable.fsdp import fully_shard
    from torch.distributed.checkpoint.state_dict import get_optimizer_state_dict, set_optimizer_state_dict
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.tensor import DTensor

    plain, wrapped = (make_dense_module("block_fp8", 256, 384, 16, 32, 3, hip_device)[0] for _ in range(2))
    fully_shard(wrapped, mesh=init_device_mesh("cuda", (1,)), reshard_after_forward=True)
    runs = [(m, AdamW([m.lora_A, m.lora_B], lr=1e-2, state_bits=bits, max_grad_norm=0.5)) for m in (plain, wrapped)]
    assert isinstance(wrapped.lora_A, DTensor)
    for k in range(4):
        x = torch.randn(70, 384, device=hip_device, generator=torch.Generator(device=hip_device).manual_seed(k)).to(torch.bfloat16)
        if k == 2 and bits == 32:
            m, opt = runs[1]
            saved = get_optimizer_state_dict(m, opt)
            opt = AdamW([m.lora_A, m.lora_B], lr=5.0, max_grad_norm=0.5)
            set_optimizer_state_dict(m, opt, saved)
            assert opt.param_groups[0]["lr"] == 1e-2
            runs[1] = (m, opt)
        for m, opt in runs:
            opt.zero_grad()
            m(x).float().square().mean().backward()
            opt.step()
        assert torch.equal(runs[0][1].grad_norm, runs[1][1].grad_norm)
    for name in ("lora_A", "lora_B"):
        a, b = getattr(plain, name), getattr(wrapped, name)
        assert torch.equal(a, b.to_local())
        s, t = runs[0][1].state[a], runs[1][1].state[b]
        assert set(s) == set(t) and float(s["step"]) == 4.0
        for key, value in t.items():
            sharded = bits == 32 and key in ("exp_avg", "exp_avg_sq")
            assert isinstance(value, DTensor) == sharded and torch.equal(s[key], value.to_local() if sharded else value)


# ---------------------------------------------------------------- memory that arguments share
@pytest.mark.parametrize("bits", [32, 8])
def test_a_rate_or_norm_that_the_step_writes_is_refused(hip_device, bits):
    """Every block reads them while others write: a rate that is itself a parameter, a norm that is a step count or one of the scales"""
    prob = _problem([(1,), (700,)], bits, torch.float32, torch.float32, 55, hip_device)
    before = [None if l is None else [t.clone() for t in l] for l in prob]
    written = [prob[0][0], prob[0][1][300:301], prob[4][1]]
    written += [prob[5][1][2:3], prob[6][0]] if bits == 8 else [prob[2][0], prob[3][1][699:]]
    for t in written:
        for kw in (dict(lr=t), dict(max_norm=1.0, grad_norm=t), dict(lr=t, max_norm=1.0, grad_norm=t)):
            with pytest.raises(_C.XqError, match="share"):
                _step(prob, **kw)
    assert _same(prob, before)
    both = torch.tensor(1e-3, device=hip_device)               # (read by both, and a gradient at that: nothing is written)
    prob[1][0] = both.view(1)
    _step(prob, lr=both, max_norm=1.0, grad_norm=both)
    assert float(both) == torch.tensor(1e-3).item()


# ---------------------------------------------------------------- more elements than 32 bits count
def test_tensors_beyond_32_bits(hip_device):
    """Gradients that are zero but behind element 2^32: norm, parameters, codes and scales there are those of the end alone, and nothing else moved"""
    n, tail = (1 << 32) + 4661, 4661 + 512
    end = torch.randn(tail, device=hip_device).to(torch.bfloat16)

    def made(count):
        g = torch.zeros(count, dtype=torch.bfloat16, device=hip_device)
        g[count - tail:] = end
        return [[torch.zeros_like(g)], [g], [torch.zeros(count, dtype=torch.int8, device=hip_device)], [torch.zeros(count, dtype=torch.uint8, device=hip_device)],
                [torch.zeros((), device=hip_device)], *([torch.zeros(-(-count // 256), device=hip_device)] for _ in range(2))]

    big, small = made(n), made(tail)                         # (the end begins at a multiple of 256)
    norm, want = _step(big, lr=1e-2, max_norm=0.5), _step(small, lr=1e-2, max_norm=0.5)
    assert abs(float(norm) - float(end.double().norm())) <= 2 * U * float(norm) and abs(float(norm) - float(want)) <= 2 * U * float(norm)
    assert abs(float(grad_norm(big[1])) - float(norm)) == 0.0
    for a, b in zip(big, small):
        a, b = a[0].view(-1), b[0].view(-1)
        k = min(b.numel(), a.numel())
        assert torch.equal(a[a.numel() - k:], b)
        assert not bool(a[:a.numel() - k].any())
    m, v = adamw_state_values(big[2][0], big[3][0], big[5][0], big[6][0], torch.bfloat16)
    mw, vw = adamw_state_values(small[2][0], small[3][0], small[5][0], small[6][0], torch.bfloat16)
    assert torch.equal(m[n - tail:], mw) and torch.equal(v[n - tail:], vw) and not bool(m[:n - tail].any()) and not bool(v[:n - tail].any())
