"""GPU: the optimizer step at the edge of what it takes."""

import threading

import pytest
import torch

from tests.test_gpu_optim import SIZES, U, _problem
from xorl_amd import _C
from xorl_amd.optim import AdamW, adamw_step, grad_norm

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
