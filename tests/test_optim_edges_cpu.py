"""Host side of AdamW: what it takes of other optimizers' state dictionaries, and the states of sharded parameters."""

import pytest
import torch

from xorl_amd import _C
from xorl_amd.optim import AdamW


def _adam(weight_decay, **kw):
    p = torch.nn.Parameter(torch.ones(8))
    opt = torch.optim.Adam([p], lr=0.1, weight_decay=weight_decay, **kw)
    p.grad = torch.ones(8)
    opt.step()
    return opt.state_dict()


def test_decay_that_is_added_to_the_gradients_is_refused():
    p = torch.nn.Parameter(torch.ones(8))
    opt = AdamW([p], lr=1.0, weight_decay=0.5)
    with pytest.raises(_C.XqError, match="added to the gradients"):
        opt.load_state_dict(_adam(0.1))
    assert opt.param_groups[0]["lr"] == 1.0 and not opt.state
    for d in (_adam(0.0), _adam(0.1, decoupled_weight_decay=True)):
        opt.load_state_dict(d)
        assert opt.param_groups[0]["weight_decay"] == d["param_groups"][0]["weight_decay"] and float(opt.state[p]["step"]) == 1.0
        # what is saved here is this class's own update, whatever came in
        opt.param_groups[0]["weight_decay"] = 0.2
        again = AdamW([p])
        again.load_state_dict(opt.state_dict())
        assert again.param_groups[0]["weight_decay"] == 0.2


@pytest.mark.parametrize("step", [3, 3.0, torch.tensor(3), torch.tensor(3, dtype=torch.int32), torch.tensor(3.0, dtype=torch.float64)])
@pytest.mark.parametrize("default", [torch.float32, torch.bfloat16])
def test_step_counts_are_taken_in_fp32(step, default):
    """whatever the dictionary holds, and whatever numbers become tensors of by default"""
    p = torch.nn.Parameter(torch.ones(8))
    d = _adam(0.0)
    d["state"][0]["step"] = step
    torch.set_default_dtype(default)
    try:
        opt = AdamW([p])
        opt.load_state_dict(d)
    finally:
        torch.set_default_dtype(torch.float32)
    s = opt.state[p]
    assert s["step"].dtype == torch.float32 and s["step"].shape == () and float(s["step"]) == 3.0 and s["exp_avg"].dtype == torch.float32


def test_codes_are_taken_as_they_are():
    p = torch.nn.Parameter(torch.ones(300))
    opt = AdamW([p], state_bits=8)
    codes = {"step": torch.tensor(2.0), "exp_avg": torch.arange(300).to(torch.int8), "exp_avg_sq": torch.arange(300).to(torch.uint8),
             "exp_avg_scale": torch.rand(2), "exp_avg_sq_scale": torch.rand(2)}
    d = opt.state_dict()
    d["state"][0] = codes
    opt.load_state_dict(d)
    assert all(opt.state[p][k].dtype == v.dtype and torch.equal(opt.state[p][k], v) and opt.state[p][k] is not v for k, v in codes.items())


# ---------------------------------------------------------------- sharded parameters, two ranks over gloo
def _two_ranks(rank, path):
    import torch.distributed as dist
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.tensor import DTensor, Partial, Replicate, Shard, distribute_tensor

    dist.init_process_group("gloo", init_method=f"file://{path}", rank=rank, world_size=2)
    mesh = init_device_mesh("cpu", (2,))
    whole = torch.arange(21.0).view(7, 3)

    def made(placement, grad=None):
        p = torch.nn.Parameter(distribute_tensor(whole, mesh, [placement]))
        p.grad = distribute_tensor(torch.ones(7, 3), mesh, [grad or placement])
        return p

    def refused(match, p, error=_C.XqError, **kw):
        opt = AdamW([p], **kw)
        with pytest.raises(error, match=match):
            opt.step()
        return opt

    refused("norm over all ranks", made(Shard(0)), max_grad_norm=1.0)
    p = made(Shard(0))
    opt = refused("could not be resharded", p, state_bits=8)
    assert not opt.state
    # (and where a dictionary has them)
    opt.load_state_dict({**opt.state_dict(), "state": {0: {"step": 1.0, "exp_avg": torch.zeros(4 - rank, 3, dtype=torch.int8)}}})
    with pytest.raises(_C.XqError, match="could not be resharded"):
        opt.step()
    # (where the norm of what a rank has is that of all, and blocks are of the whole, nothing is refused but the CPU)
    refused("HIP device only", made(Replicate()), RuntimeError, max_grad_norm=1.0, state_bits=8)
    refused("distributed otherwise", made(Shard(0), Replicate()))
    p = made(Replicate())
    p.grad = DTensor.from_local(torch.ones(7, 3), mesh, [Partial()])            # (of the local shape that it should have, and a share of the sum)
    refused("distributed otherwise", p)
    # moments like the parameter, so that a checkpoint knows whose they are; a share of 4 and one of 3 rows
    p = made(Shard(0))
    opt = refused("HIP device only", p, RuntimeError)
    state = opt.state[p]
    for k in ("exp_avg", "exp_avg_sq"):
        assert isinstance(state[k], DTensor) and state[k].placements == p.placements and state[k].shape == (7, 3) and state[k].dtype == torch.float32
        assert state[k].to_local().shape == (4 - rank, 3) and not state[k].requires_grad
    assert type(state["step"]) is torch.Tensor
    with torch.no_grad():
        state["exp_avg"].copy_(p)
    again = AdamW([p], lr=7.0)
    again.load_state_dict(opt.state_dict())
    got = again.state[p]["exp_avg"]
    assert isinstance(got, DTensor) and got.placements == p.placements and torch.equal(got.full_tensor(), whole)
    dist.destroy_process_group()


def test_sharded_parameters(tmp_path):
    torch.multiprocessing.spawn(_two_ranks, args=(str(tmp_path / "store"),), nprocs=2)


def test_hooks_of_a_load_are_followed():
    """what a pre-hook puts in the place of the dictionary is loaded, what a post-hook changes stays"""
    p, q = torch.nn.Parameter(torch.ones(8)), torch.nn.Parameter(torch.ones(8))
    opt = AdamW([p])
    d = _adam(0.0)
    other = {"state": {0: {**d["state"][0], "exp_avg": torch.full((8,), 5.0), "step": 9}}, "param_groups": d["param_groups"]}
    a = opt.register_load_state_dict_pre_hook(lambda o, s: other)
    b = opt.register_load_state_dict_post_hook(lambda o: o.state[p].update(exp_avg_sq=torch.full((8,), 6.0)))
    opt.load_state_dict(d)
    s = opt.state[p]
    assert float(s["step"]) == 9.0 and bool((s["exp_avg"] == 5).all()) and bool((s["exp_avg_sq"] == 6).all())
    a.remove()
    b.remove()
    opt.load_state_dict(d)
    assert float(opt.state[p]["step"]) == 1.0 and torch.equal(opt.state[p]["exp_avg"], d["state"][0]["exp_avg"])
    assert not opt._optimizer_load_state_dict_pre_hooks and not opt._optimizer_load_state_dict_post_hooks
    with pytest.raises(ValueError):
        AdamW([p, q]).load_state_dict(d)
