"""AdamW over the parameters this package's modules are trained by: all of them in one call, with 32- or 8-bit states.

A QLoRA model trains some hundreds of factors of 10^4 to 10^6 elements.  ``adamw_step`` takes them as lists, in a handful of
launches and without a word of the device read by the host; ``AdamW`` is the ``torch.optim.Optimizer`` around it, whose state
``reset_lora_optimizer_states`` and ``maybe_merge_lora`` reset like any other's.  The update is that of ``torch.optim.AdamW``; the
reference builds its optimizers in optim/optimizer.py.
"""

from __future__ import annotations

from typing import Iterable, Optional, Sequence, Tuple, Union

import torch
from torch import Tensor

from . import _C
from ._native import native


STATE_BLOCK = 256       # consecutive elements of an 8-bit state that share a scale


def _scale_count(numel: int) -> int:
    return -(-numel // STATE_BLOCK)


def grad_norm(grads: Iterable[Tensor]) -> Tensor:
    """The 2-norm over all of ``grads`` (fp32 or bf16, any mixture) as a 0-dim fp32 tensor on their device, summed in 64 bits in
    an order that depends on the sizes alone."""
    return native().adamw(None, list(grads), None, None, None, None, None, None, None, None, None)


def adamw_step(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avgs: Sequence[Tensor], exp_avg_sqs: Sequence[Tensor],
               steps: Sequence[Tensor], *, exp_avg_scales: Optional[Sequence[Tensor]] = None,
               exp_avg_sq_scales: Optional[Sequence[Tensor]] = None, lr: Union[float, Tensor], betas: Tuple[float, float] = (0.9, 0.999),
               eps: float = 1e-8, weight_decay: float = 0.01, max_norm: Optional[float] = None,
               grad_norm: Optional[Tensor] = None) -> Optional[Tensor]:
    """One AdamW step over all ``params``, in place, with the states they come with.

    Parameters and gradients are fp32 or bf16, tensor by tensor; parameters, states and step counts are contiguous and share no
    memory, with gradients, ``lr`` and ``grad_norm`` neither (refused otherwise; a gradient that is not contiguous is copied).  States are fp32, or, with both lists of scales
    given, 8-bit codes: int8 ``exp_avgs`` and uint8 ``exp_avg_sqs`` with fp32 scales for every 256 elements (``adamw_state_values``
    says what they stand for).  ``steps`` are fp32 tensors of one element each, advanced here (of tensors without elements too).  ``lr`` may be a 0-dim fp32 tensor on
    the device: a captured step then follows it.

    ``max_norm`` scales the gradients by min(1, max_norm / (norm + 1e-6)) on the way, ``norm`` being the 2-norm over all of them
    (or ``grad_norm``, where that is given: of a larger set, or summed over ranks); ``grads`` themselves stay as they are.  A norm that
    is NaN makes every parameter NaN, an infinite one leaves the gradients zero where they are finite.  Returns the norm, or None."""
    lr_tensor = lr if isinstance(lr, Tensor) else None
    hyper = (0.0 if lr_tensor is not None else float(lr), float(betas[0]), float(betas[1]), float(eps), float(weight_decay))
    return native().adamw(params, grads, exp_avgs, exp_avg_sqs, steps, exp_avg_scales, exp_avg_sq_scales, hyper, lr_tensor, max_norm, grad_norm)


def adamw_state_values(exp_avg: Tensor, exp_avg_sq: Tensor, exp_avg_scale: Tensor, exp_avg_sq_scale: Tensor,
                       dtype: torch.dtype = torch.float32) -> Tuple[Tensor, Tensor]:
    """What 8-bit states stand for, as (exp_avg, exp_avg_sq) of ``dtype`` (fp32 or bf16) in the codes' shape."""
    _C.require_hip(exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale)
    if exp_avg.dtype != torch.int8 or exp_avg_sq.dtype != torch.uint8 or exp_avg.shape != exp_avg_sq.shape:
        raise _C.XqError(f"8-bit states are int8 and uint8 codes of one shape, got {exp_avg.dtype} {tuple(exp_avg.shape)} and "
                         f"{exp_avg_sq.dtype} {tuple(exp_avg_sq.shape)}")
    if dtype not in (torch.float32, torch.bfloat16):
        raise _C.XqError(f"state values are fp32 or bf16, got {dtype}")
    n = exp_avg.numel()
    for s in (exp_avg_scale, exp_avg_sq_scale):
        if s.dtype != torch.float32 or s.numel() != _scale_count(n) or not s.is_contiguous() or s.device != exp_avg.device:
            raise _C.XqError(f"scales of {n} elements are {_scale_count(n)} contiguous fp32 on {exp_avg.device}, got {s.dtype} "
                             f"{tuple(s.shape)} on {s.device}")
    if exp_avg_sq.device != exp_avg.device or not exp_avg.is_contiguous() or not exp_avg_sq.is_contiguous():
        raise _C.XqError("8-bit states must be contiguous and on one device")
    m, v = torch.empty(exp_avg.shape, dtype=dtype, device=exp_avg.device), torch.empty(exp_avg.shape, dtype=dtype, device=exp_avg.device)
    with torch.cuda.device(exp_avg.device):
        _C.check(_C.lib().xq_adamw_values(exp_avg.data_ptr(), exp_avg_sq.data_ptr(), exp_avg_scale.data_ptr(), exp_avg_sq_scale.data_ptr(), n,
                                          m.data_ptr(), v.data_ptr(), _C.XQ_DT_BF16 if dtype == torch.bfloat16 else _C.XQ_DT_F32,
                                          _C.stream_ptr(exp_avg.device)))
    return m, v


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` as one ``adamw_step`` over all parameters of a group.

    ``state_bits=8`` keeps the two moments as 8-bit codes (2.03 bytes an element in place of 8).  ``max_grad_norm`` clips by the norm
    over the parameters of all groups inside the step; the norm of the last step is ``self.grad_norm`` (a device tensor).  States are
    made at a parameter's first step and whenever its state has been dropped, but not while a graph is captured (refused: they would be made
    anew in every replay).  In a captured step ``lr`` follows a tensor, a number stays what it was.  State names: ``step``, ``exp_avg``, ``exp_avg_sq``, with
    8 bits ``exp_avg_scale`` and ``exp_avg_sq_scale`` too.  All parameters lie on one device.

    Distributed parameters (DTensor, as FSDP2 makes them): every rank steps its own share, gradients are to be distributed like their
    parameters, and 32-bit moments are distributed tensors like them, so that a distributed checkpoint can carry them.  Over several ranks
    ``max_grad_norm`` and 8-bit states of sharded parameters are refused: the norm would be a share's, and the blocks of codes that share a scale are
    blocks of a share, which no other number of ranks can take up."""

    def __init__(self, params, lr: Union[float, Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01, *, state_bits: int = 32, max_grad_norm: Optional[float] = None):
        if state_bits not in (8, 32):
            raise _C.XqError(f"state_bits must be 8 or 32, got {state_bits}")
        if max_grad_norm is not None and not max_grad_norm > 0.0:
            raise _C.XqError(f"max_grad_norm must be positive, got {max_grad_norm}")
        self.max_grad_norm = max_grad_norm
        self.grad_norm: Optional[Tensor] = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits))

    def __getstate__(self) -> dict:
        return {**super().__getstate__(), "max_grad_norm": self.max_grad_norm, "grad_norm": None}

    def add_param_group(self, param_group: dict) -> None:
        bits = param_group.get("state_bits", self.defaults["state_bits"])
        if bits not in (8, 32):
            raise _C.XqError(f"state_bits must be 8 or 32, got {bits}")
        super().add_param_group(param_group)

    def _init_state(self, p: Tensor, state_bits: int) -> dict:
        state = self.state[p]
        if not state:
            local = _local(p)
            if local.is_cuda and torch.cuda.is_current_stream_capturing():
                raise _C.XqError("AdamW: a captured step would make its states anew in every replay; take one step before the capture")
            state["step"] = torch.zeros((), dtype=torch.float32, device=local.device)
            if state_bits == 8:
                n = _scale_count(local.numel())
                state["exp_avg"] = torch.zeros(local.shape, dtype=torch.int8, device=local.device)
                state["exp_avg_sq"] = torch.zeros(local.shape, dtype=torch.uint8, device=local.device)
                state["exp_avg_scale"] = torch.zeros(n, dtype=torch.float32, device=local.device)
                state["exp_avg_sq_scale"] = torch.zeros(n, dtype=torch.float32, device=local.device)
            else:
                state["exp_avg"] = _zeros_fp32(p)
                state["exp_avg_sq"] = _zeros_fp32(p)
        return state

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        groups = [(g, [p for p in g["params"] if p.grad is not None]) for g in self.param_groups]
        groups = [(g, ps) for g, ps in groups if ps]
        distributed = [(g, p) for g, ps in groups for p in ps if hasattr(p, "to_local")]
        for g, p in distributed:
            if g["state_bits"] == 8 and _sharded(p):
                raise _C.XqError("AdamW: 8-bit states of a parameter that is sharded over ranks could not be resharded; take 32 bits")
            if _layout(p) != _layout(p.grad):
                raise _C.XqError(f"AdamW: a gradient is distributed otherwise than its parameter: {_layout(p.grad)}, {_layout(p)}")
        local = (lambda ts: [_local(t) for t in ts]) if distributed else (lambda ts: ts)
        norm = None
        if self.max_grad_norm is not None and groups:
            if any(_sharded(p) for _, p in distributed):
                raise _C.XqError("max_grad_norm over sharded parameters: clip them with a norm over all ranks, and leave it out here")
            if len(groups) > 1:
                norm = grad_norm(local([p.grad for _, ps in groups for p in ps]))
        for g, ps in groups:
            states = [self._init_state(p, g["state_bits"]) for p in ps]

            def of(name):
                return local([s[name] for s in states])

            eight = g["state_bits"] == 8
            out = adamw_step(local(ps), local([p.grad for p in ps]), of("exp_avg"), of("exp_avg_sq"), of("step"),
                             exp_avg_scales=of("exp_avg_scale") if eight else None, exp_avg_sq_scales=of("exp_avg_sq_scale") if eight else None,
                             lr=g["lr"], betas=g["betas"], eps=g["eps"], weight_decay=g["weight_decay"], max_norm=self.max_grad_norm,
                             grad_norm=norm)
            norm = norm if norm is not None else out
        self.grad_norm = norm
        return loss

    def load_state_dict(self, state_dict) -> None:
        """States of this class or of ``torch.optim.AdamW`` (a group of the latter goes on with 32 bits; its variants are refused)."""
        # around what the base class loads, so that hooks of the user's see, and may change, what is loaded and what has been
        taken: dict = {}

        def check(_, d):
            for g in d["param_groups"]:
                if g.get("amsgrad") or g.get("maximize"):
                    raise _C.XqError("AdamW: amsgrad and maximize have no counterpart here")
                if g.get("weight_decay") and not g.get("decoupled_weight_decay", True):
                    raise _C.XqError("AdamW: a weight decay that is added to the gradients has no counterpart here")
            taken.update(d)

        def finish(_):
            for g in self.param_groups:
                g.setdefault("state_bits", 32)
                if "decoupled_weight_decay" in g:           # (without a decay it may have come as False)
                    g["decoupled_weight_decay"] = True
            # (the base class has cast floating-point state, and codes with it, to the parameter's type)
            saved = [i for g in taken["param_groups"] for i in g["params"]]
            own = [p for g in self.param_groups for p in g["params"]]
            for i, p in zip(saved, own):
                if i in taken["state"]:
                    self.state[p] = {k: _state(v, _local(p).device) for k, v in taken["state"][i].items()}

        hooks = (self.register_load_state_dict_pre_hook(check), self.register_load_state_dict_post_hook(finish, prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for h in hooks:
                h.remove()


def _state(v, device):
    """A copy of a loaded state on ``device``: codes as they are, all else (moments in bf16, a step count that is a number or an integer) in fp32"""
    if isinstance(v, Tensor):
        return v.detach().to(device, v.dtype if v.dtype in (torch.int8, torch.uint8) else torch.float32, copy=True)
    return torch.tensor(float(v), dtype=torch.float32, device=device) if isinstance(v, (int, float)) else v


def _local(t: Tensor) -> Tensor:
    """The rank's own share of a distributed tensor (the update is elementwise); other tensors as they are."""
    return t.to_local() if hasattr(t, "to_local") else t


def _zeros_fp32(p: Tensor) -> Tensor:
    return torch.zeros_like(p, dtype=torch.float32, requires_grad=False) if hasattr(p, "to_local") else torch.zeros(p.shape, dtype=torch.float32, device=p.device)


def _layout(t: Tensor):
    return (t.device_mesh, tuple(t.placements)) if hasattr(t, "to_local") else None


def _sharded(p: Tensor) -> bool:
    return hasattr(p, "to_local") and any(p.device_mesh.size(i) > 1 and not q.is_replicate() for i, q in enumerate(p.placements))
