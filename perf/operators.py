"""Performance cases of what closes a QLoRA training step: the loss over the output head and the optimizer step of the factors.

`listed()` names the cases that are followed from version to version, `draw(rng)` gives further ones of the same ranges,
`prepare(case, seed)` builds what a program holds before the call, `run(state)` is one pass: where `own` is true through the
public entry points, else in elementary torch operations.  Everything is synthetic and made from the seed.

  op      what it stands for                                                        public entry point
  score   log-probabilities of given tokens, without gradients (rollouts, evaluation)   linear_cross_entropy
  loss    loss and gradient of the hidden states, the head frozen (QLoRA training)      linear_cross_entropy, autograd
  head    the same with the head trained: its gradient too                              linear_cross_entropy, autograd
  adamw   one optimizer step over all factors (or a trained head), 32- or 8-bit states  adamw_step, adamw_state_values
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
IGNORE = -100
BLOCK = 256                       # elements of an 8-bit state that share a scale
LR, BETA1, BETA2, EPS, DECAY = 2e-4, 0.9, 0.999, 1e-8, 0.01


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # the log-probability of one token under a large head: one read of 1 GiB of weights
        {"name": "score_t1", "op": "score", "tokens": 1, "hidden": 4096, "vocab": 131072, "ignored": 0.0, "reduction": "none", "scale": 1.0},
        # a decode batch of 48 sequences at a sampling temperature of 0.8, a vocabulary of an odd size
        {"name": "score_t48", "op": "score", "tokens": 48, "hidden": 2048, "vocab": 100003, "ignored": 0.0, "reduction": "none", "scale": 1.25},
        # the perplexity of one prompt of an uneven length
        {"name": "score_t1357", "op": "score", "tokens": 1357, "hidden": 4096, "vocab": 131072, "ignored": 0.0, "reduction": "mean", "scale": 1.0},
        # a small head and few tokens, each with a weight of its own (policy gradients)
        {"name": "loss_t96_v32003", "op": "loss", "tokens": 96, "hidden": 2048, "vocab": 32003, "ignored": 0.1, "reduction": "none", "scale": 1.0},
        # a small micro-batch
        {"name": "loss_t512", "op": "loss", "tokens": 512, "hidden": 4096, "vocab": 131072, "ignored": 0.0, "reduction": "mean", "scale": 1.0},
        # a full micro-batch, prompts masked: the workload of a fine-tuning step
        {"name": "loss_t8192", "op": "loss", "tokens": 8192, "hidden": 4096, "vocab": 131072, "ignored": 0.3, "reduction": "mean", "scale": 1.0},
        # a trained head
        {"name": "head_t4096", "op": "head", "tokens": 4096, "hidden": 2048, "vocab": 65536, "ignored": 0.0, "reduction": "sum", "scale": 1.0},
        # the factors of one layer: launch and host latency
        {"name": "adamw32_layer", "op": "adamw", "bits": 32, "set": "dense", "hidden": 4096, "kv": 1024, "inter": 12288, "layers": 1, "r": 8,
         "params": "float32", "grads": "float32", "clip": False},
        # all factors of an 8B model, gradients clipped
        {"name": "adamw32_dense_r32", "op": "adamw", "bits": 32, "set": "dense", "hidden": 4096, "kv": 1024, "inter": 12288, "layers": 36, "r": 32,
         "params": "float32", "grads": "float32", "clip": True},
        # the same with 8-bit states
        {"name": "adamw8_dense_r32", "op": "adamw", "bits": 8, "set": "dense", "hidden": 4096, "kv": 1024, "inter": 12288, "layers": 36, "r": 32,
         "params": "float32", "grads": "float32", "clip": True},
        # the factors of 128 routed experts, bf16 gradients
        {"name": "adamw8_experts", "op": "adamw", "bits": 8, "set": "experts", "hidden": 2048, "inter": 768, "experts": 128, "layers": 12, "r": 16,
         "params": "float32", "grads": "bfloat16", "clip": False},
        # a trained bf16 head
        {"name": "adamw8_head", "op": "adamw", "bits": 8, "set": "head", "hidden": 4096, "vocab": 65536, "layers": 1,
         "params": "bfloat16", "grads": "bfloat16", "clip": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(("score", "loss", "loss", "head", "adamw", "adamw"))
    if op != "adamw":
        hidden = 64 * _log_int(rng, 4, 80)
        vocab = _log_int(rng, 2000, 131072)
        most = {"score": 8192 * 4096 * 131072, "loss": 8192 * 4096 * 131072, "head": 4096 * 2048 * 65536}[op]
        tokens = _log_int(rng, 1, max(1, min(8192, most // (hidden * vocab))))
        return {"op": op, "tokens": tokens, "hidden": hidden, "vocab": vocab, "ignored": rng.choice((0.0, 0.0, 0.2, 0.5, 0.9)),
                "reduction": rng.choice(("none", "mean", "sum")), "scale": rng.choice((1.0, 1.0, 1.25, 0.5))}
    kind = rng.choice(("dense", "dense", "experts", "head"))
    c = {"op": op, "bits": rng.choice((8, 32)), "set": kind, "params": rng.choice(("float32", "float32", "bfloat16")),
         "grads": rng.choice(("float32", "bfloat16")), "clip": rng.choice((True, False))}
    if kind == "dense":
        hidden = 64 * _log_int(rng, 8, 80)
        return {**c, "hidden": hidden, "kv": 64 * _log_int(rng, 2, 16), "inter": 3 * hidden - 64 * rng.randrange(4),
                "layers": _log_int(rng, 1, 36), "r": _log_int(rng, 3, 32)}
    if kind == "experts":
        return {**c, "hidden": 64 * _log_int(rng, 8, 32), "inter": 64 * _log_int(rng, 4, 12), "experts": _log_int(rng, 4, 128),
                "layers": _log_int(rng, 1, 8), "r": _log_int(rng, 3, 16)}
    return {**c, "hidden": 64 * _log_int(rng, 4, 64), "vocab": _log_int(rng, 1000, 65536), "layers": 1}


def _shapes(case):
    """The factors' shapes, in the order of the modules."""
    if case["set"] == "head":
        return [(case["vocab"], case["hidden"])]
    h, i, r = case["hidden"], case["inter"], case["r"]
    if case["set"] == "experts":
        e = case["experts"]
        layer = [(e, h, r), (e, r, i), (e, h, r), (e, r, i), (e, i, r), (e, r, h)]
    else:
        kv = case["kv"]
        layer = [s for k, n in ((h, h), (h, kv), (h, kv), (h, h), (h, i), (h, i), (i, h)) for s in ((r, k), (n, r))]
    return layer * case["layers"]


def _valid_tokens(case):
    return case["tokens"] - min(case["tokens"] - 1, int(case["tokens"] * case["ignored"]))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, device=DEVICE, generator=g, dtype=torch.float32) * std).to(dtype)

    if case["op"] == "adamw":
        shapes = _shapes(case)
        sizes = [math.prod(s) for s in shapes]
        starts, total = [], 0
        for n in sizes:               # the tensors of a kind lie in one buffer, each from a multiple of a block on
            starts.append(total)
            total += -(-n // BLOCK) * BLOCK
        pd, gd = getattr(torch, case["params"]), getattr(torch, case["grads"])
        real = torch.zeros(total, dtype=torch.bool, device=DEVICE)
        for a, n in zip(starts, sizes):
            real[a:a + n] = True
        p = normal(total, std=0.02, dtype=pd).mul_(real)
        spread = torch.exp2(torch.randint(-6, 3, (total // BLOCK, 1), device=DEVICE, generator=g).float()).expand(-1, BLOCK).reshape(-1)
        grad = (normal(total, std=1e-4) * spread).mul_(real).to(gd)
        st = {"case": case, "p": p, "g": grad, "steps": torch.randint(20, 2000, (len(sizes),), device=DEVICE, generator=g).float(),
              "starts": starts, "sizes": sizes, "shapes": shapes, "tensor_of_block": None}
        sd = torch.cat([torch.full((-(-n // BLOCK),), k, dtype=torch.int64) for k, n in enumerate(sizes)])
        st["tensor_of_block"] = sd.to(DEVICE)
        if case["bits"] == 32:
            st["m"] = (normal(total, std=3e-5) * spread).mul_(real)
            st["v"] = (normal(total, std=1e-4) * spread).square_().mul_(real) + 1e-12 * real
        else:
            # codes as a run of steps leaves them: values about normally distributed below the largest of a block
            m = normal(total // BLOCK, BLOCK)
            m /= m.abs().amax(1, keepdim=True)
            st["m"] = (m.sign() * m.abs().sqrt().mul_(127).round_()).to(torch.int8).reshape(-1).mul_(real)
            s = normal(total // BLOCK, BLOCK).abs_() + 0.05
            s /= s.amax(1, keepdim=True)
            st["v"] = s.sqrt_().mul_(255).round_().clamp_(min=1).to(torch.uint8).reshape(-1).mul_(real)
            st["m_scale"] = spread.view(-1, BLOCK)[:, 0] * 1e-4
            st["v_scale"] = spread.view(-1, BLOCK)[:, 0] * 3e-4

        def views(flat):
            return [flat[a:a + n].view(s) for a, n, s in zip(starts, sizes, shapes)]

        st["lists"] = [views(st[k]) for k in ("p", "g", "m", "v")] + [list(st["steps"].unbind())]
        if case["bits"] == 8:
            st["scales"] = [[st[k][a // BLOCK:a // BLOCK + -(-n // BLOCK)] for a, n in zip(starts, sizes)] for k in ("m_scale", "v_scale")]
        return st

    t, h, v = case["tokens"], case["hidden"], case["vocab"]
    w = torch.empty(v, h, dtype=torch.bfloat16, device=DEVICE)
    for a in range(0, v, 16384):
        w[a:a + 16384] = normal(min(16384, v - a), h, std=0.02, dtype=torch.bfloat16)
    labels = torch.randint(0, v, (t,), device=DEVICE, generator=g)
    # hidden states that a trained model would have: most targets lie some way above the other logits
    lift = torch.rand(t, 1, device=DEVICE, generator=g) * 12.0
    x = normal(t, h) + lift * w[labels].float() / (0.0004 * h)
    masked = t - _valid_tokens(case)
    if masked:                        # prompts in front of answers, in sequences of up to 512 tokens
        order = torch.arange(t, device=DEVICE)
        rank = ((order % 512) * 100003 + order).argsort()
        labels[rank[:masked]] = IGNORE
    st = {"case": case, "x": x.to(torch.bfloat16), "w": w, "labels": labels, "weights": None}
    if case["reduction"] == "none" and case["op"] != "score":
        st["weights"] = normal(t, std=1.0 / t)
    if case["op"] != "score":
        st["x"].requires_grad_(True)
    if case["op"] == "head":
        st["w"].requires_grad_(True)
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if case["op"] == "adamw":
        return _adamw_own(state) if own else _adamw_plain(state)
    return _loss_own(state) if own else _loss_plain(state)


def _loss_own(state):
    from xorl_amd.loss_functional import linear_cross_entropy

    case = state["case"]
    if case["op"] == "score":
        with torch.no_grad():
            return linear_cross_entropy(state["x"], state["w"], state["labels"], ignore_index=IGNORE, reduction=case["reduction"],
                                        logit_scale=case["scale"])
    loss = linear_cross_entropy(state["x"], state["w"], state["labels"], ignore_index=IGNORE, reduction=case["reduction"],
                                logit_scale=case["scale"])
    leaves = (state["x"], state["w"]) if case["op"] == "head" else (state["x"],)
    return [loss.detach(), *torch.autograd.grad(loss, leaves, state["weights"])]


def _loss_plain(state):
    case = state["case"]
    x, w, labels = state["x"].detach().float(), state["w"].detach().float(), state["labels"]
    valid = labels != IGNORE
    target = labels.where(valid, 0)[:, None]
    logits = (x @ w.t()).mul_(case["scale"])
    top = logits.amax(1, keepdim=True)
    at_target = logits.gather(1, target)
    p = logits.sub_(top).exp_()
    total = p.sum(1, keepdim=True)
    loss = ((total.log() + (top - at_target))[:, 0]).where(valid, 0.0)
    count = valid.sum()
    if case["reduction"] == "mean":
        out = (loss.double().sum() / count).float()
    elif case["reduction"] == "sum":
        out = loss.double().sum().float()
    else:
        out = loss
    if case["op"] == "score":
        return out
    if case["reduction"] == "none":
        up = state["weights"]
    else:
        up = (1.0 / count if case["reduction"] == "mean" else torch.ones_like(count)).float().expand(labels.shape[0])
    up = up.where(valid, 0.0)[:, None] * case["scale"]
    p.div_(total)
    p.scatter_add_(1, target, torch.full_like(total, -1.0))
    p.mul_(up)
    dx = (p @ w).to(torch.bfloat16)
    if case["op"] == "head":
        return [out, dx, (p.t() @ x).to(torch.bfloat16)]
    return [out, dx]


def _adamw_own(state):
    from xorl_amd.optim import adamw_state_values, adamw_step

    case = state["case"]
    p, g, m, v, steps = state["lists"]
    ms, vs = state["scales"] if case["bits"] == 8 else (None, None)
    norm = adamw_step(p, g, m, v, steps, exp_avg_scales=ms, exp_avg_sq_scales=vs, lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY,
                      max_norm=_max_norm(case))
    out = [state["p"], state["steps"]]
    if case["bits"] == 32:
        out += [state["m"], state["v"]]
    else:
        out += list(adamw_state_values(state["m"], state["v"], state["m_scale"], state["v_scale"], dtype=torch.bfloat16))
    return out + ([norm] if case["clip"] else [])


def _max_norm(case):
    return 0.05 if case["clip"] else None


def _adamw_plain(state):
    case = state["case"]
    p, g, steps = state["p"], state["g"].float(), state["steps"]
    steps.add_(1.0)
    out = []
    if case["clip"]:
        norm = g.double().square().sum().sqrt().float()
        g = g * (_max_norm(case) / (norm + 1e-6)).clamp(max=1.0)
        out = [norm]
    each = steps.double()
    first = (LR / (1.0 - BETA1 ** each)).float()[state["tensor_of_block"]][:, None]
    root = (1.0 / (1.0 - BETA2 ** each).sqrt()).float()[state["tensor_of_block"]][:, None]
    if case["bits"] == 32:
        m = state["m"].mul_(BETA1).add_(g * (1.0 - BETA1))
        v = state["v"].mul_(BETA2).add_(g.square() * (1.0 - BETA2))
        s = v.sqrt()
    else:
        c, d = state["m"].view(-1, BLOCK).float(), state["v"].view(-1, BLOCK).float()
        m = (c * c.abs() * (state["m_scale"] / 16129.0)[:, None]).reshape(-1).mul_(BETA1).add_(g * (1.0 - BETA1))
        s = (d * d * (state["v_scale"] / 65025.0)[:, None]).reshape(-1)
        s = (s.square() * BETA2 + g.square() * (1.0 - BETA2)).sqrt()
    update = (m.view(-1, BLOCK) * first / (s.view(-1, BLOCK) * root + EPS)).view(-1)
    w = p.float()
    p.copy_(w - w * (LR * DECAY) - update)
    if case["bits"] == 32:
        return [p, steps, m, v] + out
    # codes next to a border: in 64 bits
    mb, sb = m.view(-1, BLOCK).double(), s.view(-1, BLOCK).double()
    ma, sa = mb.abs().amax(1, keepdim=True), sb.amax(1, keepdim=True)
    c = mb.sign() * (mb.abs() / ma.clamp(min=1e-300)).sqrt().mul(127).round()
    d = (sb / sa.clamp(min=1e-300)).sqrt().mul(255).round().clamp(min=1) * (sb > 0)
    state["m"].copy_(c.view(-1))
    state["v"].copy_(d.view(-1))
    state["m_scale"].copy_(ma[:, 0])
    state["v_scale"].copy_(sa[:, 0])
    return [p, steps, (c * c.abs() * (ma / 16129.0)).view(-1).to(torch.bfloat16), ((d * d * (sa / 65025.0)).square()).view(-1).to(torch.bfloat16)] + out


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its result in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "adamw":
        n = sum(math.prod(s) for s in _shapes(case))
        size = {"float32": 4, "bfloat16": 2}
        each = 2 * size[case["params"]] + size[case["grads"]]
        # 8-bit states: codes read and written, two scales a block, and the values that are returned
        each += 16 if case["bits"] == 32 else 4 + 16 / BLOCK + 4
        return {"bytes": n * each, "flops": 0}
    t, h, v = _valid_tokens(case), case["hidden"], case["vocab"]
    rows = case["tokens"]
    moved = 2 * v * h + 2 * t * h + 8 * rows + (4 * rows if case["reduction"] == "none" else 4)
    products = {"score": 1, "loss": 2, "head": 3}[case["op"]]
    if products > 1:
        moved += 2 * rows * h + (4 * rows if case["reduction"] == "none" else 4)
    if products > 2:
        moved += 2 * v * h
    return {"bytes": moved, "flops": 2 * products * t * v * h}


def exact(case, seed):
    state = prepare(case, seed)
    return _adamw_exact(state, case) if case["op"] == "adamw" else _loss_exact(state, case)


def _loss_exact(state, case):
    x, w, labels = state["x"].detach(), state["w"].detach().double(), state["labels"]
    t = x.shape[0]
    kept = torch.nonzero(labels != IGNORE)[:, 0]
    share = 1.0 / kept.numel() if case["reduction"] == "mean" else 1.0
    losses = torch.zeros(t, dtype=torch.float64, device=x.device)
    dx = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    dw = torch.zeros_like(w) if case["op"] == "head" else None
    for rows in kept.split(1024):
        xr, lr = x[rows].double(), labels[rows]
        z = case["scale"] * torch.mm(xr, w.transpose(0, 1))
        logp = torch.log_softmax(z, dim=1)
        losses[rows] = -logp[torch.arange(len(rows), device=x.device), lr]
        if case["op"] == "score":
            continue
        up = state["weights"][rows].double() if case["reduction"] == "none" else torch.full((len(rows),), share, dtype=torch.float64, device=x.device)
        e = torch.exp(logp)
        e[torch.arange(len(rows), device=x.device), lr] -= 1.0
        e *= (case["scale"] * up).unsqueeze(1)
        dx[rows] = torch.mm(e, w)
        if dw is not None:
            dw += torch.mm(e.transpose(0, 1).contiguous(), xr)
    out = losses if case["reduction"] == "none" else losses.sum() * share
    if case["op"] == "score":
        return out
    return [out, dx, dw] if dw is not None else [out, dx]


def _adamw_exact(state, case):
    eight = case["bits"] == 8
    g_all = state["g"].double()
    norm = torch.sqrt(torch.dot(g_all, g_all))
    factor = min(1.0, 0.05 / (float(norm) + 1e-6)) if case["clip"] else 1.0
    p_out, m_out, v_out = torch.zeros_like(g_all), torch.zeros_like(g_all), torch.zeros_like(g_all)
    steps = state["steps"].double() + 1.0
    for k, (a, n) in enumerate(zip(state["starts"], state["sizes"])):
        b = a + -(-n // BLOCK) * BLOCK
        g = g_all[a:b] * factor
        k1, k2 = 1.0 - BETA1 ** float(steps[k]), 1.0 - BETA2 ** float(steps[k])
        m, v = state["m"][a:b].double(), state["v"][a:b].double()
        if eight:
            ms, vs = (state[q][a // BLOCK:b // BLOCK].double().repeat_interleave(BLOCK) for q in ("m_scale", "v_scale"))
            m, v = torch.sign(m) * (m / 127.0) ** 2 * ms, ((v / 255.0) ** 2 * vs) ** 2
        m, v = BETA1 * m + (1.0 - BETA1) * g, BETA2 * v + (1.0 - BETA2) * g * g
        w = state["p"][a:b].double()
        p_out[a:b] = w * (1.0 - LR * DECAY) - LR * (m / k1) / (torch.sqrt(v / k2) + EPS)
        if eight:
            mb, sb = m.reshape(-1, BLOCK), torch.sqrt(v).reshape(-1, BLOCK)
            mt, st = mb.abs().max(dim=1, keepdim=True).values, sb.max(dim=1, keepdim=True).values
            mc = torch.round(127.0 * torch.sqrt(torch.nan_to_num(mb.abs() / mt)))
            sc = torch.round(255.0 * torch.sqrt(torch.nan_to_num(sb / st)))
            sc = torch.where(sb > 0, torch.maximum(sc, torch.ones_like(sc)), torch.zeros_like(sc))
            m, v = (torch.sign(mb) * (mc / 127.0) ** 2 * mt).reshape(-1), (((sc / 255.0) ** 2 * st) ** 2).reshape(-1)
        m_out[a:b], v_out[a:b] = m, v
    out = [p_out, steps, m_out, v_out]
    return out + [norm] if case["clip"] else out
