"""Performance cases of the work that a QLoRA program picks by an index per token: experts, adapters and embedding rows.

`listed()` names the cases that are followed from version to version, `draw(rng)` gives further ones of the same ranges,
`prepare(case, seed)` builds what a program holds before the call, `run(state)` is one pass: where `own` is true through the
public entry points, else in elementary torch operations.  Everything is synthetic and made from the seed.

  op        what it stands for                                                            public entry point
  route     the choice of experts without gradients (decode, rollout)                     moe_route
  gate      the same and the gradient of the router's logits (a trained router)           moe_route, autograd
  adapters  the low-rank updates of many requests added to one shared projection          lora_adapters
  lookup    rows of the embedding for given tokens, scaled, without gradients             embedding
  embed     the same and the gradient of a trained embedding                              embedding, autograd
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one token in front of 128 experts: launch and host latency
        {"name": "route_t1_e128", "op": "route", "tokens": 1, "experts": 128, "top_k": 8, "scoring": "softmax", "bias": False, "groups": 1,
         "top_groups": 1, "group_score": "max", "renormalize": True, "scale": 1.0, "dtype": "bfloat16", "masked": 0.0},
        # a rollout batch of an odd size over groups of experts, sigmoid scores and a bias for balance, fp32 logits
        {"name": "route_t333_e256_groups", "op": "route", "tokens": 333, "experts": 256, "top_k": 8, "scoring": "sigmoid", "bias": True, "groups": 8,
         "top_groups": 4, "group_score": "sum2", "renormalize": True, "scale": 2.5, "dtype": "float32", "masked": 0.0},
        # the router of a routed fine-tuning step, trained
        {"name": "gate_t16384_e128", "op": "gate", "tokens": 16384, "experts": 128, "top_k": 8, "scoring": "softmax", "bias": False, "groups": 1,
         "top_groups": 1, "group_score": "max", "renormalize": True, "scale": 1.0, "dtype": "bfloat16", "masked": 0.0},
        # a large batch over many experts in groups, a few of them switched off
        {"name": "gate_t65536_e256_groups", "op": "gate", "tokens": 65536, "experts": 256, "top_k": 8, "scoring": "sigmoid", "bias": True, "groups": 8,
         "top_groups": 4, "group_score": "sum2", "renormalize": True, "scale": 2.5, "dtype": "float32", "masked": 0.02},
        # one token of one request through one adapter of 64: launch and host latency
        {"name": "adapters_t1", "op": "adapters", "tokens": 1, "k": 4096, "n": 4096, "r": 16, "adapters": 64, "without": 0.0, "run": 1, "factors": "bfloat16"},
        # a decode batch of 48 requests, some of them on the base alone, down to a narrow projection
        {"name": "adapters_t48", "op": "adapters", "tokens": 48, "k": 4096, "n": 1024, "r": 32, "adapters": 128, "without": 0.2, "run": 1, "factors": "bfloat16"},
        # prompts of 257 tokens of eight requests, the last one cut, trained factors as they are in fp32
        {"name": "adapters_t2049", "op": "adapters", "tokens": 2049, "k": 4096, "n": 12288, "r": 16, "adapters": 16, "without": 0.1, "run": 257, "factors": "float32"},
        # a full prefill through the widest contraction
        {"name": "adapters_t16384", "op": "adapters", "tokens": 16384, "k": 12288, "n": 4096, "r": 64, "adapters": 8, "without": 0.0, "run": 2048,
         "factors": "bfloat16"},
        # the tokens of a decode batch
        {"name": "lookup_t64", "op": "lookup", "tokens": 64, "vocab": 131072, "hidden": 4096, "scale": 1.0, "padded": 0.0, "dtype": "bfloat16"},
        # a prefill, rows scaled by the root of their length
        {"name": "lookup_t16385_scaled", "op": "lookup", "tokens": 16385, "vocab": 100003, "hidden": 2048, "scale": 45.25, "padded": 0.0, "dtype": "bfloat16"},
        # a small trained fp32 embedding, a third of the tokens padding
        {"name": "embed_t4001_fp32", "op": "embed", "tokens": 4001, "vocab": 32003, "hidden": 2048, "scale": 1.0, "padded": 0.33, "dtype": "float32"},
        # a full micro-batch under the large vocabulary
        {"name": "embed_t8192_v131072", "op": "embed", "tokens": 8192, "vocab": 131072, "hidden": 4096, "scale": 1.0, "padded": 0.0, "dtype": "bfloat16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(("route", "gate", "adapters", "adapters", "lookup", "embed"))
    if op in ("route", "gate"):
        groups = rng.choice((1, 1, 2, 4, 8))
        experts = groups * max(2, _log_int(rng, 8, 384) // groups)
        top_groups = rng.randint((groups + 1) // 2, groups)
        top_k = rng.randint(1, min(12, experts // groups * top_groups))
        return {"op": op, "tokens": _log_int(rng, 1, 65536 * 256 // max(256, experts)), "experts": experts, "top_k": top_k,
                "scoring": rng.choice(("softmax", "sigmoid")), "bias": rng.choice((False, True)), "groups": groups, "top_groups": top_groups,
                "group_score": rng.choice(("max", "sum2")), "renormalize": rng.choice((True, False)), "scale": rng.choice((1.0, 2.5)),
                "dtype": rng.choice(("bfloat16", "float32")), "masked": rng.choice((0.0, 0.0, 0.05))}
    if op == "adapters":
        k, n = 64 * _log_int(rng, 8, 192), 16 * _log_int(rng, 16, 768)
        r = rng.choice((8, 16, 16, 24, 32, 64))
        tokens = _log_int(rng, 1, min(16384, 16384 * 20480 // (k + 2 * n)))
        adapters = _log_int(rng, 2, 64)
        return {"op": op, "tokens": tokens, "k": k, "n": n, "r": r, "adapters": adapters, "without": rng.choice((0.0, 0.0, 0.2)),
                "run": 1 if tokens <= 64 else _log_int(rng, 32, tokens), "factors": rng.choice(("bfloat16", "bfloat16", "float32"))}
    hidden = rng.choice((8, 64)) * _log_int(rng, 8, 64)
    dtype = rng.choice(("bfloat16", "bfloat16", "float32"))
    vocab = _log_int(rng, 1000, min(131072, 131072 * 8192 // (hidden * (4 if dtype == "float32" else 2))))
    return {"op": op, "tokens": _log_int(rng, 1, 8192 if op == "embed" else 16384), "vocab": vocab, "hidden": hidden, "scale": rng.choice((1.0, hidden ** 0.5)),
            "padded": rng.choice((0.0, 0.0, 0.3)), "dtype": dtype}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, device=DEVICE, generator=g, dtype=torch.float32) * std).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, device=DEVICE, generator=g)

    if case["op"] in ("route", "gate"):
        t, e = case["tokens"], case["experts"]
        # experts in demand by a power of their rank, and what the token adds
        popular = -1.1 * torch.log(1.0 + torch.randperm(e, device=DEVICE, generator=g).float())
        z = popular + normal(t, e) - torch.log(-torch.log(uniform(t, e).clamp(1e-6, 1.0 - 1e-6)))
        off = uniform(e) < case["masked"]
        off[torch.randperm(e, device=DEVICE, generator=g)[:(3 * e) // 4]] = False
        z[:, off] = -math.inf
        bias = normal(e, std=0.05) if case["bias"] else None
        st = {"case": case, "z": z.to(getattr(torch, case["dtype"])), "bias": bias}
        if case["op"] == "gate":
            st["z"].requires_grad_(True)
            st["up"] = normal(t, case["top_k"], std=1e-3)
        return st

    if case["op"] == "adapters":
        t, k, n, r, a = (case[q] for q in ("tokens", "k", "n", "r", "adapters"))
        dt = getattr(torch, case["factors"])
        runs = -(-t // case["run"])
        ids = torch.randint(0, a, (runs,), device=DEVICE, generator=g)
        ids[uniform(runs) < case["without"]] = -1
        return {"case": case, "x": normal(t, k, dtype=torch.bfloat16), "base": normal(t, n, dtype=torch.bfloat16),
                "A": normal(a, r, k, std=k ** -0.5, dtype=dt), "B": normal(a, n, r, std=0.1, dtype=dt),
                "ids": ids.repeat_interleave(case["run"])[:t].to(torch.int32), "scalings": 0.5 + 1.5 * uniform(a)}

    t, v, h = case["tokens"], case["vocab"], case["hidden"]
    dt = getattr(torch, case["dtype"])
    w = torch.empty(v, h, dtype=dt, device=DEVICE)
    for a in range(0, v, 16384):
        w[a:a + 16384] = normal(min(16384, v - a), h, std=0.02, dtype=dt)
    # words come by a power of their rank; the ranks lie anywhere in the vocabulary
    rank = torch.exp(uniform(t) * math.log(v)).long().clamp_(1, v) - 1
    ids = torch.randperm(v, device=DEVICE, generator=g)[rank]
    if case["padded"]:                # sequences of up to 512 tokens, padded behind
        ids[(torch.arange(t, device=DEVICE) % 512) >= 512 - int(512 * case["padded"])] = 0
    st = {"case": case, "w": w, "ids": ids, "padding_idx": 0 if case["padded"] else None}
    if case["op"] == "embed":
        st["w"].requires_grad_(True)
        st["up"] = normal(t, h, std=1e-3, dtype=dt)
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if op in ("route", "gate"):
        return _route_own(state) if own else _route_plain(state)
    if op == "adapters":
        return _adapters_own(state) if own else _adapters_plain(state)
    return _embed_own(state) if own else _embed_plain(state)


def _route_own(state):
    from xorl_amd.moe_functional import moe_route

    c = state["case"]
    weights, ids = moe_route(state["z"], c["top_k"], scoring=c["scoring"], bias=state["bias"], num_groups=c["groups"], top_groups=c["top_groups"],
                             group_score=c["group_score"], renormalize=c["renormalize"], scale=c["scale"])
    if c["op"] == "route":
        return [weights, ids]
    return [weights.detach(), ids, *torch.autograd.grad(weights, (state["z"],), state["up"])]


def _adapters_own(state):
    from xorl_amd.functional import lora_adapters

    return lora_adapters(state["base"], state["x"], state["A"], state["B"], state["ids"], state["scalings"])


def _embed_own(state):
    from xorl_amd.embedding_functional import embedding

    c = state["case"]
    out = embedding(state["ids"], state["w"], scale=c["scale"], padding_idx=state["padding_idx"])
    if c["op"] == "lookup":
        return out
    return [out.detach(), *torch.autograd.grad(out, (state["w"],), state["up"])]


def _route_plain(state):
    c = state["case"]
    z = state["z"].detach().float()
    t, e = z.shape
    sigmoid = c["scoring"] == "sigmoid"
    # the choice next to a border: in 64 bits; without a bias scores rise with the logits
    z64 = z.double()
    if c["bias"] or c["group_score"] == "sum2":
        if sigmoid:
            s64 = 1.0 / (1.0 + (-z64).exp())
        else:
            s64 = (z64 - z64.amax(1, keepdim=True)).exp()
            s64 = s64 / s64.sum(1, keepdim=True)
        choice = s64 + state["bias"].double() if c["bias"] else s64
        choice = choice.masked_fill(z64 == -math.inf, -math.inf)
    else:
        choice = z64
    if c["top_groups"] < c["groups"]:
        each = choice.view(t, c["groups"], e // c["groups"])
        best = each.amax(2)
        if c["group_score"] == "sum2" and each.shape[2] > 1:
            second = each.scatter(2, each.argmax(2, keepdim=True), -math.inf).amax(2)
            best = best + second.masked_fill(second == -math.inf, 0.0)
        order = best.sort(dim=1, descending=True, stable=True)[1][:, :c["top_groups"]]
        kept = torch.zeros_like(best, dtype=torch.bool).scatter_(1, order, True)
        choice = each.masked_fill(~kept[:, :, None], -math.inf).view(t, e)
    if not c["bias"]:
        choice = z64.masked_fill(choice == -math.inf, -math.inf)
    value, at = choice.sort(dim=1, descending=True, stable=True)
    ids = at[:, :c["top_k"]]
    none = value[:, :c["top_k"]] == -math.inf
    zs = z.gather(1, ids)
    if sigmoid:
        s = 1.0 / (1.0 + (-zs).exp())
    else:
        p = (z - z.amax(1, keepdim=True)).exp()
        p = p / p.sum(1, keepdim=True)
        s = p.gather(1, ids)
    s = s.masked_fill(none, 0.0)
    u = s / s.sum(1, keepdim=True) if c["renormalize"] else s
    weights = u * c["scale"]
    out = [weights, ids.masked_fill(none, -1)]
    if c["op"] == "route":
        return out
    g = state["up"] * c["scale"]
    if c["renormalize"]:
        d = u * (g - (g * u).sum(1, keepdim=True))
        if sigmoid:
            d = d * (1.0 - s)
    elif sigmoid:
        d = g * s * (1.0 - s)
    else:
        d = g * s
    dz = torch.zeros_like(z).scatter_(1, ids, d.masked_fill(none, 0.0))
    if not sigmoid and not c["renormalize"]:
        dz -= p * (g * s).sum(1, keepdim=True)
    return out + [dz.to(state["z"].dtype)]


def _adapters_plain(state):
    c = state["case"]
    x, ids = state["x"].float(), state["ids"].long()
    has = ids >= 0
    at = ids.clamp(min=0)
    if c["tokens"] <= c["adapters"]:      # few rows: each with the factors of its adapter
        u = (state["A"][at].float() * x[:, None, :]).sum(2)
        u = u * (state["scalings"][at] * has)[:, None]
        delta = (state["B"][at].float() * u[:, None, :]).sum(2)
    else:                                 # many rows: all adapters at once, each row's own kept
        a, r = c["adapters"], c["r"]
        u = (x @ state["A"].float().view(a * r, c["k"]).t()).view(-1, a, r)
        mine = (torch.arange(a, device=x.device) == ids[:, None])
        u = (u * (mine * state["scalings"])[:, :, None]).view(-1, a * r)
        delta = u @ state["B"].float().transpose(1, 2).reshape(a * r, c["n"])
    return (state["base"].float() + delta).to(torch.bfloat16)


def _embed_plain(state):
    c = state["case"]
    w, ids = state["w"].detach(), state["ids"]
    out = (w[ids].float() * c["scale"]).to(w.dtype)
    if c["op"] == "lookup":
        return out
    # long sums of an fp32 gradient: in 64 bits
    wide = torch.float64 if w.dtype == torch.float32 else torch.float32
    dw = torch.zeros(w.shape, dtype=wide, device=w.device).index_add_(0, ids, state["up"].to(wide))
    if state["padding_idx"] is not None:
        dw[state["padding_idx"]] = 0.0
    return [out, dw.mul_(c["scale"]).to(w.dtype)]


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its result in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    size = {"float32": 4, "bfloat16": 2}
    if case["op"] in ("route", "gate"):
        t, e, k, b = case["tokens"], case["experts"], case["top_k"], size[case["dtype"]]
        moved = t * e * b + t * k * 12 + (4 * e if case["bias"] else 0)
        if case["op"] == "gate":
            moved += t * e * b + t * k * 4
        return {"bytes": moved, "flops": 0}
    if case["op"] == "adapters":
        t, k, n, r = (case[q] for q in ("tokens", "k", "n", "r"))
        rows = t * (1.0 - case["without"])
        runs = -(-t // case["run"]) * (1.0 - case["without"])
        touched = case["adapters"] * (1.0 - (1.0 - 1.0 / case["adapters"]) ** runs)      # of so many draws, on average
        return {"bytes": rows * k * 2 + t * n * 4 + t * 4 + touched * (r * (k + n) * size[case["factors"]] + 4), "flops": 2 * rows * r * (k + n)}
    t, v, h, b = case["tokens"], case["vocab"], case["hidden"], size[case["dtype"]]
    distinct = min(t, v)
    moved = distinct * h * b + t * h * b + t * 8
    if case["op"] == "embed":
        moved += t * h * b + v * h * b
    return {"bytes": moved, "flops": 0}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] in ("route", "gate"):
        return _route_exact(state, case)
    return _adapters_exact(state, case) if case["op"] == "adapters" else _embed_exact(state, case)


def _route_exact(state, case):
    z = state["z"].detach().double()
    t, e, k, many = z.shape[0], case["experts"], case["top_k"], case["groups"]
    s = torch.sigmoid(z) if case["scoring"] == "sigmoid" else torch.softmax(z, dim=1)
    order = s + state["bias"].double()[None, :] if case["bias"] else s.clone()
    order[torch.isinf(z)] = -math.inf
    if case["top_groups"] < many:
        strength = torch.empty(t, many, dtype=torch.float64, device=z.device)
        span = e // many
        for j in range(many):
            best = torch.topk(order[:, j * span:(j + 1) * span], min(2, span) if case["group_score"] == "sum2" else 1, dim=1).values
            strength[:, j] = torch.where(torch.isinf(best), 0.0, best).sum(1)
            strength[torch.isinf(best[:, 0]), j] = -math.inf
        for _ in range(many - case["top_groups"]):          # the weakest out, of equals the last
            out = many - 1 - strength.flip(1).argmin(1)
            rows = torch.arange(t, device=z.device)
            strength[rows, out] = math.inf
            for j in range(span):
                order[rows, out * span + j] = -math.inf
    ids = torch.full((t, k), -1, dtype=torch.int64, device=z.device)
    picked = torch.zeros(t, k, dtype=torch.float64, device=z.device)
    rows = torch.arange(t, device=z.device)
    for j in range(k):
        top, at = order.max(dim=1)
        real = ~torch.isinf(top)
        ids[:, j] = torch.where(real, at, -1)
        picked[:, j] = torch.where(real, s[rows, at], 0.0)
        order[rows, at] = -math.inf
    total = picked.sum(1, keepdim=True) if case["renormalize"] else torch.ones_like(picked[:, :1])
    weights = case["scale"] * picked / total
    if case["op"] == "route":
        return [weights, ids]
    # the gradient by the chain: weights -> chosen scores -> logits
    up = state["up"].double()
    ds = case["scale"] * up / total
    if case["renormalize"]:
        ds = ds - (ds * picked).sum(1, keepdim=True) / total
    full = torch.zeros_like(s)
    for j in range(k):
        at = ids[:, j].clamp(min=0)
        full[rows, at] += torch.where(ids[:, j] >= 0, ds[:, j], 0.0)
    if case["scoring"] == "sigmoid":
        dz = full * s * (1.0 - s)
    else:
        dz = s * (full - (full * s).sum(1, keepdim=True))
    return [weights, ids, dz]


def _adapters_exact(state, case):
    out = state["base"].double()
    ids = state["ids"].long()
    for a in torch.unique(ids).tolist():
        if a < 0:
            continue
        rows = torch.nonzero(ids == a)[:, 0]
        u = torch.mm(state["x"][rows].double(), state["A"][a].double().transpose(0, 1).contiguous())
        out[rows] += state["scalings"][a].double() * torch.mm(u, state["B"][a].double().transpose(0, 1).contiguous())
    return out


def _embed_exact(state, case):
    w, ids = state["w"].detach(), state["ids"]
    out = torch.index_select(w, 0, ids).double() * case["scale"]
    if case["op"] == "lookup":
        return out
    # runs of equal tokens: differences of running sums would lose bits, so each run is added by itself
    used, place = torch.unique(ids, return_inverse=True)
    sums = torch.zeros(len(used), w.shape[1], dtype=torch.float64, device=w.device)
    sums.index_put_((place,), state["up"].double(), accumulate=True)
    if state["padding_idx"] is not None:
        sums[used == state["padding_idx"]] = 0.0
    dw = torch.zeros(w.shape, dtype=torch.float64, device=w.device)
    dw[used] = sums * case["scale"]
    return [out, dw]
