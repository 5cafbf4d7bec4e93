"""Host side of experts, adapters and embedding rows: calls that are traced and never run here."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from xorl_amd import _C
from xorl_amd.embedding_functional import _bwd_impl, _fwd_impl, embedding
from xorl_amd.functional import _adapters_impl, lora_adapters
from xorl_amd.moe_functional import _route_bwd_impl, _route_fwd_impl, _route_problem, moe_route

BF = torch.bfloat16


def _traced(monkeypatch, on="cuda", out=None, **elsewhere):
    """lora_adapters as a compiled program traces it, over tensors without memory"""
    shapes = {"base": (3, 32), "x": (3, 64), "A": (5, 4, 64), "B": (5, 32, 4), "ids": (3,), "s": (5,)}
    types = {"base": BF, "x": BF, "A": BF, "B": BF, "ids": torch.int32, "s": torch.float32}
    monkeypatch.setattr(torch.compiler, "is_compiling", lambda: True)
    with FakeTensorMode():
        a = {n: torch.empty(shapes[n], dtype=types[n], device=elsewhere.get(n, on)) for n in shapes}
        o = None if out is None else torch.empty(out[0], dtype=out[1], device=out[2])
        return lora_adapters(*a.values(), out=o)


def test_a_traced_call_gives_what_an_eager_one_does(monkeypatch):
    y = _traced(monkeypatch)
    assert y.shape == (3, 32) and y.dtype == BF and y.device.type == "cuda"
    assert _traced(monkeypatch, out=((3, 32), BF, "cuda")).dtype == BF


@pytest.mark.parametrize("which", ["base", "x", "A", "B", "ids", "s"])
def test_a_traced_call_refuses_host_memory(monkeypatch, which):
    with pytest.raises(RuntimeError, match="HIP device only"):
        _traced(monkeypatch, **{which: "cpu"})
    with pytest.raises(_C.XqError, match="different devices"):
        _traced(monkeypatch, **{which: "cuda:1"})


@pytest.mark.parametrize("out,match", [(((3, 32), torch.float32, "cuda"), "out must be"), (((2, 3, 32), BF, "cuda"), "out must be"), (((3, 16), BF, "cuda"), "out must be"),
                                       (((3, 32), BF, "cpu"), "HIP device only"), (((3, 32), BF, "cuda:1"), "different devices")])
def test_a_traced_call_refuses_an_out_of_another_kind(monkeypatch, out, match):
    with pytest.raises((_C.XqError, RuntimeError), match=match):
        _traced(monkeypatch, out=out)


@pytest.mark.parametrize("which", range(6))
def test_the_operator_itself_refuses_host_memory(which):
    """What a traced call leaves in a program is dispatched by any one of its tensors: without a device that is all of them, and the rest is refused here"""
    with FakeTensorMode():
        shapes = ((3, 32, BF), (3, 64, BF), (5, 4, 64, BF), (5, 32, 4, BF), (3, torch.int32), (5, torch.float32))
        a = [torch.empty(s[:-1], dtype=s[-1], device="cpu" if i == which else "cuda") for i, s in enumerate(shapes)]
        with pytest.raises(RuntimeError, match="HIP device only"):
            _adapters_impl(*a)


class _Wrapped(torch.Tensor):
    """a tensor whose values another one holds, as a distributed tensor's are"""

    @staticmethod
    def __new__(cls, inner):
        t = torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device)
        t.inner = inner
        return t

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise NotImplementedError


def test_a_bias_without_memory_of_its_own_is_refused():
    options = (2, 1, 1, 1, 1, True, 1.0)
    z, bias = torch.zeros(3, 8), torch.zeros(8)
    assert _route_problem(z, 3, 8, z.dtype, bias, options).bias == bias.data_ptr()
    assert _route_problem(z, 3, 8, z.dtype, None, options).bias is None
    with pytest.raises(_C.XqError, match="no memory"):
        _route_problem(z, 3, 8, z.dtype, _Wrapped(bias), options)
    assert _C.ptr(torch.empty(0)) == 0


def test_a_distributed_bias_is_refused(tmp_path):
    import torch.distributed as dist
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.tensor import Replicate, distribute_tensor

    dist.init_process_group("gloo", init_method=f"file://{tmp_path / 'store'}", rank=0, world_size=1)
    try:
        bias = distribute_tensor(torch.zeros(8), init_device_mesh("cpu", (1,)), [Replicate()])
        with pytest.raises(_C.XqError, match="no memory"):
            _route_problem(torch.zeros(3, 8), 3, 8, torch.float32, bias, (2, 1, 1, 1, 1, True, 1.0))
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("kw", [dict(top_k=2.5), dict(num_groups=2.5, top_groups=2), dict(num_groups=4, top_groups=2.5), dict(top_k=float("inf")), dict(top_k=float("nan"))])
def test_numbers_that_are_not_whole_are_refused(kw):
    with pytest.raises(_C.XqError, match="moe_route"):
        moe_route(torch.zeros(3, 20), **{"top_k": 2, **kw})


@pytest.mark.parametrize("padding_idx", [0.5, -1.5, float("nan")])
def test_a_padding_index_that_is_not_whole_is_refused(padding_idx):
    with pytest.raises(_C.XqError, match="padding_idx"):
        embedding(torch.zeros(3, dtype=torch.int64), torch.zeros(5, 4), padding_idx=padding_idx)


def test_the_workspace_holds_tiles_only_where_they_are_kept():
    """[rows][ranks, padded to 16] in fp32, of one part of K; from 65 rows on each row's tile beside it"""
    need = _C.lib().xq_adapters_workspace_bytes
    assert [need(M, 32, 64, 5) for M in (4, 64, 65, 512, 513)] == [256, 64 * 64, 65 * 128, 512 * 128, 513 * 64]


# ---- the custom operators by themselves: what a kernel would read or write out of bounds, or as another type, is refused before anything runs
def _z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


OPTIONS = (2, 1, 1, 1, 1, True, 1.0)


@pytest.mark.parametrize("z,bias", [(_z(3, 8, dtype=torch.float16), None), (_z(3, 8), _z(7)), (_z(3, 8), _z(8, dtype=torch.float64)), (_z(3, 8), _z(8, dtype=BF)), (_z(3, 0), None),
                                    (torch.tensor(1.0), None)])
def test_the_router_operator_refuses(z, bias):
    with pytest.raises(_C.XqError, match="moe_route"):
        _route_fwd_impl(z, bias, OPTIONS)


def test_the_routers_gradient_operator_refuses():
    def call(grad=_z(3, 2), w=_z(3, 2), ids=_z(3, 2, dtype=torch.int64), options=OPTIONS):
        _route_bwd_impl(grad, w, ids, _z(3, 8), 8, torch.float32, options)

    for kw in (dict(w=_z(3, 2, dtype=torch.float64)), dict(ids=_z(3, 2, dtype=torch.int32)), dict(w=_z(3, 4)), dict(ids=_z(2, 2, dtype=torch.int64)), dict(grad=_z(3, 1)), dict(grad=_z(6)),
               dict(grad=_z(3, 4), w=_z(3, 4), ids=_z(3, 4, dtype=torch.int64)), dict(options=(0, *OPTIONS[1:])), dict(w=_z(6), ids=_z(6, dtype=torch.int64), grad=_z(6))):
        with pytest.raises(_C.XqError, match="not that of this problem"):
            call(**kw)
    with pytest.raises(RuntimeError, match="HIP device only"):
        call()


@pytest.mark.parametrize("i", range(6))
def test_the_adapters_operator_refuses(i):
    good = (_z(3, 32, dtype=BF), _z(3, 64, dtype=BF), _z(5, 4, 64), _z(5, 32, 4), _z(3, dtype=torch.int32), _z(5))
    bad = ((_z(3, 16, dtype=BF), _z(2, 32, dtype=BF), _z(3, 32)), (_z(3, 128, dtype=BF), _z(3, 64)), (_z(5, 4, 32), _z(4, 4, 64), _z(5, 4, 64, dtype=torch.float16)),
           (_z(5, 32, 3), _z(5, 31, 4), _z(5, 32, 4, dtype=BF)), (_z(2, dtype=torch.int32), _z(3, dtype=torch.int16), _z(3)), (_z(4), _z(5, dtype=torch.float64)))
    for t in bad[i]:
        with pytest.raises(_C.XqError, match="lora_adapters"):
            _adapters_impl(*good[:i], t, *good[i + 1:])


def test_the_embedding_operators_refuse():
    ids = _z(3, dtype=torch.int64)
    for i, w in ((ids, _z(5, 4, dtype=torch.float16)), (ids, _z(5)), (ids, _z(0, 4)), (ids, _z(5, 0)), (_z(3), _z(5, 4)), (_z(3, dtype=torch.int16), _z(5, 4))):
        with pytest.raises(_C.XqError, match="embedding"):
            _fwd_impl(i, w, 1.0)
    for g, i, V in ((_z(3, 4, dtype=torch.float16), ids, 5), (torch.tensor(1.0), ids, 5), (_z(3, 0), ids, 5), (_z(3, 4), _z(3), 5), (_z(3, 4), ids, 0)):
        with pytest.raises(_C.XqError, match="not that of this problem"):
            _bwd_impl(g, i, V, 1.0, -1)
    for call in (lambda: _fwd_impl(ids, _z(5, 4), 1.0), lambda: _bwd_impl(_z(3, 4), ids, 5, 1.0, -1), lambda: _route_fwd_impl(_z(3, 8), _z(8), OPTIONS)):
        with pytest.raises(RuntimeError, match="HIP device only"):
            call()


def test_memory_that_was_freed_or_cut_is_found():
    flat = torch.zeros(24)
    view, rest = flat[8:].view(4, 4), flat[8:].view(4, 4).t()[:, 1:]
    inside, first, none = view[:, :3], view[:1], view[:0]          # (views of freed memory cannot be made)
    _C.check_held("x", flat, view, rest, None, flat[:0])
    flat.untyped_storage().resize_(23 * 4)
    for t in (flat, view, rest):
        with pytest.raises(_C.XqError, match="x: .*no memory"):
            _C.check_held("x", t)
    _C.check_held("x", inside, first)
    flat.untyped_storage().resize_(0)
    with pytest.raises(_C.XqError, match="no memory"):
        _C.check_held("x", first)
    _C.check_held("x", none)
