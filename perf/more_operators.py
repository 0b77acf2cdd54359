"""The operators around the experts' NF4 products of a sparse decoder layer, as measurable cases.

* ``norm``: the root-mean-square norm, with the residual's addition before it or without;
* ``route``: the router's choice of experts and their weights, from its logits;
* ``dispatch``: the rows of a batch in the experts' order (the order, and the rows in it);
* ``combine``: the experts' rows back to their tokens, weighted, with the residual's addition.

Each alone (``forward``) or with its gradients (``step``). ``listed()`` holds the named cases, ``draw(rng)`` gives
others of the same ranges, ``prepare`` makes what a program holds before the call, ``run`` makes the call (in plain
torch, or through the package where ``own`` is true), and ``exact`` computes the same outputs in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6


def listed():
    return [
        # One token of a small model: launches and host work.
        {"name": "norm fwd 1 row of 2048", "kind": "norm", "way": "forward", "rows": 1, "hidden": 2048, "dtype": "bf16",
         "residual": "bf16", "weight": "bf16", "weight_grad": False},
        # Every query head of a small model's training batch, normalised over its 128 columns; no residual.
        {"name": "norm step 131072 heads of 128", "kind": "norm", "way": "step", "rows": 131072, "hidden": 128,
         "dtype": "bf16", "residual": "", "weight": "bf16", "weight_grad": True},
        # A ragged batch with a residual stream in 32 bits and a width that is no multiple of anything.
        {"name": "norm step 1021 rows of 2050, fp32 stream", "kind": "norm", "way": "step", "rows": 1021,
         "hidden": 2050, "dtype": "fp16", "residual": "fp32", "weight": "fp32", "weight_grad": True},
        # A training batch of an 8B model with frozen norms.
        {"name": "norm step 8192 rows of 4096", "kind": "norm", "way": "step", "rows": 8192, "hidden": 4096,
         "dtype": "bf16", "residual": "bf16", "weight": "bf16", "weight_grad": False},
        # One token's choice among 128 experts.
        {"name": "route fwd 1 token of 128", "kind": "route", "way": "forward", "tokens": 1, "experts": 128, "top_k": 8,
         "dtype": "bf16", "score": "softmax", "bias": False, "groups": 1, "top_groups": 1, "group_score": "max",
         "renormalize": True, "scale": 1.0, "padded": 0.0},
        # A padded training batch over the same experts.
        {"name": "route step 8192 tokens of 128", "kind": "route", "way": "step", "tokens": 8192, "experts": 128,
         "top_k": 8, "dtype": "bf16", "score": "softmax", "bias": False, "groups": 1, "top_groups": 1,
         "group_score": "max", "renormalize": True, "scale": 1.0, "padded": 0.1},
        # A large ragged batch with sigmoid scores, a balancing bias and groups.
        {"name": "route step 16383 tokens of 256 in 8 groups", "kind": "route", "way": "step", "tokens": 16383,
         "experts": 256, "top_k": 8, "dtype": "fp32", "score": "sigmoid", "bias": True, "groups": 8, "top_groups": 4,
         "group_score": "top2", "renormalize": True, "scale": 2.5, "padded": 0.0},
        # A batch of sequences decoding, one token each.
        {"name": "dispatch fwd 16 tokens to 128", "kind": "dispatch", "way": "forward", "tokens": 16, "experts": 128,
         "top_k": 8, "hidden": 2048, "dtype": "bf16", "padded": 0.0},
        # The training batch of the benchmark's expert layer.
        {"name": "dispatch step 8192 tokens to 128", "kind": "dispatch", "way": "step", "tokens": 8192, "experts": 128,
         "top_k": 8, "hidden": 2048, "dtype": "bf16", "padded": 0.0},
        # One token of the same layer, back from its eight experts.
        {"name": "combine fwd 1 token", "kind": "combine", "way": "forward", "tokens": 1, "experts": 128, "top_k": 8,
         "hidden": 2048, "dtype": "bf16", "residual": True, "padded": 0.0},
        # A ragged, padded batch in the other type, few experts, an odd width.
        {"name": "combine step 2777 tokens of 1001", "kind": "combine", "way": "step", "tokens": 2777, "experts": 60,
         "top_k": 4, "hidden": 1001, "dtype": "fp16", "residual": False, "padded": 0.2},
        # The training batch again.
        {"name": "combine step 8192 tokens of 2048", "kind": "combine", "way": "step", "tokens": 8192, "experts": 128,
         "top_k": 8, "hidden": 2048, "dtype": "bf16", "residual": True, "padded": 0.0},
    ]


# ------------------------------------------------------------------ drawn cases

_MOST_NORM = 8192 * 4096         # elements of the largest listed norm
_MOST_ROUTE = 16383 * 256        # logits of the largest listed choice
_MOST_ROWS = 8192 * 8 * 2048     # elements of the experts' rows in the largest listed dispatch and combination


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _width(rng, low, high):
    """A width: a multiple of 64, as most models have, or any."""
    w = _log_int(rng, low, high)
    return max(low, w // 64 * 64) if rng.random() < 0.6 else w


def draw(rng):
    kind = rng.choice(["norm", "route", "dispatch", "combine"])
    way = rng.choice(["forward", "step"])
    if kind == "norm":
        hidden = _width(rng, 64, 8192)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        return {"kind": kind, "way": way, "rows": _log_int(rng, 1, min(262144, _MOST_NORM // hidden)), "hidden": hidden,
                "dtype": dtype, "residual": rng.choice(["", dtype, dtype, "fp32"]),
                "weight": rng.choice([dtype, dtype, "fp32"]), "weight_grad": rng.random() < 0.5}
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    padded = rng.choice([0.0, 0.0, 0.05, 0.5])
    if kind == "route":
        groups = rng.choice([1, 1, 4, 8])
        experts = groups * _log_int(rng, 8 if groups == 1 else 4, 512 // groups)
        top_groups = rng.randint(1, groups)
        score = rng.choice(["softmax", "sigmoid"])
        bias = rng.random() < 0.5
        return {"kind": kind, "way": way, "tokens": _log_int(rng, 1, min(32768, _MOST_ROUTE // experts)),
                "experts": experts, "top_k": rng.randint(1, min(10, experts // groups * top_groups)), "dtype": dtype,
                "score": score, "bias": bias, "groups": groups, "top_groups": top_groups,
                "group_score": rng.choice(["max", "top2"]), "renormalize": rng.random() < 0.7,
                "scale": rng.choice([1.0, 1.0, 2.5]), "padded": padded}
    experts = _log_int(rng, 4, 384)
    top_k = rng.randint(1, min(10, experts))
    hidden = _width(rng, 256, 7168)
    most = _MOST_ROWS // (top_k * hidden * (2 if dtype == "fp32" else 1))
    case = {"kind": kind, "way": way, "tokens": _log_int(rng, 1, min(32768, most)), "experts": experts, "top_k": top_k,
            "hidden": hidden, "dtype": dtype, "padded": padded}
    return case if kind == "dispatch" else {**case, "residual": rng.random() < 0.5}


# ------------------------------------------------------------------ inputs, from the seed alone

def _generator(seed, place):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 64 + place)


def _normal(seed, place, shape, std, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=_generator(seed, place))


def _present(case, seed):
    """Which tokens are real: those of the padded share, here and there in the batch, are not."""
    if not case["padded"]:
        return None
    return torch.rand(case["tokens"], device="cuda", generator=_generator(seed, 5)) >= case["padded"]


def _logits(case, seed, dtype):
    """A router's logits: some experts are liked more than others by all tokens."""
    liked = _normal(seed, 11, (1, case["experts"]), 0.5)
    return (_normal(seed, 10, (case["tokens"], case["experts"]), 1.5) + liked).to(dtype)


def _chosen(case, seed):
    """The experts of every token, int32 [tokens, top_k], -1 for the padding's."""
    chosen = _logits(case, seed, torch.float32).topk(case["top_k"], dim=1).indices.to(torch.int32)
    present = _present(case, seed)
    return chosen if present is None else torch.where(present.unsqueeze(1), chosen, -1)


def prepare(case, seed):
    kind, step = case["kind"], case["way"] == "step"
    dtype = DTYPES[case["dtype"]]
    state = {"kind": kind, "way": case["way"]}
    if kind == "norm":
        rows, h = case["rows"], case["hidden"]
        state["x"] = _normal(seed, 1, (rows, h), 1.0, dtype)
        state["weight"] = (1.0 + _normal(seed, 2, (h,), 0.2)).to(DTYPES[case["weight"]])
        state["residual"] = None
        if case["residual"]:
            state["residual"] = _normal(seed, 3, (rows, h), 2.0, DTYPES[case["residual"]])
        if step:
            state["dy"] = _normal(seed, 4, (rows, h), 1.0, dtype)
            state["x"].requires_grad_(True)
            if case["residual"]:
                state["dh"] = _normal(seed, 6, (rows, h), 1.0, DTYPES[case["residual"]])
                state["residual"].requires_grad_(True)
            state["weight"].requires_grad_(case["weight_grad"])
        return state
    if kind == "route":
        for name in ("top_k", "score", "groups", "top_groups", "group_score", "renormalize", "scale"):
            state[name] = case[name]
        state["logits"] = _logits(case, seed, dtype)
        state["mask"] = _present(case, seed)
        state["bias"] = _normal(seed, 12, (case["experts"],), 0.1) if case["bias"] else None
        if step:
            state["logits"].requires_grad_(True)
            state["dweights"] = _normal(seed, 13, (case["tokens"], case["top_k"]), 1.0)
        return state
    tokens, k, h = case["tokens"], case["top_k"], case["hidden"]
    chosen = _chosen(case, seed)
    if kind == "dispatch":
        state.update(num_experts=case["experts"], experts=chosen, x=_normal(seed, 20, (tokens, h), 1.0, dtype))
        if step:
            state["x"].requires_grad_(True)
            state["drows"] = _normal(seed, 21, (tokens * k, h), 1.0, dtype)
        return state
    state["order"] = _order(chosen, case["experts"])
    state["y"] = _normal(seed, 22, (tokens * k, h), 1.0, dtype)
    weights = torch.softmax(_normal(seed, 23, (tokens, k), 1.0), dim=1)
    state["weights"] = torch.where(chosen >= 0, weights, 0.0)
    state["residual"] = _normal(seed, 24, (tokens, h), 1.0, dtype) if case["residual"] else None
    if step:
        state["y"].requires_grad_(True)
        state["weights"].requires_grad_(True)
        state["dout"] = _normal(seed, 25, (tokens, h), 1.0, dtype)
    return state


# ------------------------------------------------------------------ one pass

def run(state):
    return (_own if own else _plain)(state)


def _own(state):
    kind, step = state["kind"], state["way"] == "step"
    with torch.set_grad_enabled(step):
        return _OWN[kind](state, step)


def _own_norm(state, step):
    from stratum_amd import rms_norm
    x, weight, residual = state["x"], state["weight"], state["residual"]
    y = rms_norm(x, weight, EPS, residual)
    out, grads = ({"y": y}, (state["dy"],)) if step or residual is None else ({"y": y[0], "h": y[1]}, None)
    if residual is not None and step:
        out, grads = {"y": y[0], "h": y[1]}, (state["dy"], state["dh"])
    if not step:
        return out
    wanted = {"dx": x, "dresidual": residual, "dweight": weight if weight.requires_grad else None}
    wanted = {name: t for name, t in wanted.items() if t is not None}
    got = torch.autograd.grad(tuple(out.values()), tuple(wanted.values()), grads)
    return {**{name: t.detach() for name, t in out.items()}, **dict(zip(wanted, got))}


def _own_route(state, step):
    from stratum_amd import moe_route
    weights, experts = moe_route(state["logits"], state["top_k"], score=state["score"], bias=state["bias"],
                                 groups=state["groups"], top_groups=state["top_groups"],
                                 group_score=state["group_score"], renormalize=state["renormalize"],
                                 scale=state["scale"], mask=state["mask"])
    out = {"weights": weights.detach(), "experts": experts}
    if step:
        out["dlogits"], = torch.autograd.grad(weights, state["logits"], state["dweights"])
    return out


def _own_dispatch(state, step):
    from stratum_amd import moe_gather, moe_sort
    order = moe_sort(state["experts"], state["num_experts"])
    rows = moe_gather(state["x"], order)
    out = {"offsets": order.offsets, "slots": order.slots, "positions": order.positions, "rows": rows.detach()}
    if step:
        out["dx"], = torch.autograd.grad(rows, state["x"], state["drows"])
    return out


def _own_combine(state, step):
    from stratum_amd import MoEOrder, moe_combine
    out = moe_combine(state["y"], state["weights"], MoEOrder(*state["order"]), state["residual"])
    if not step:
        return {"out": out}
    dy, dweights = torch.autograd.grad(out, (state["y"], state["weights"]), state["dout"])
    return {"out": out.detach(), "dy": dy, "dweights": dweights}


_OWN = {"norm": _own_norm, "route": _own_route, "dispatch": _own_dispatch, "combine": _own_combine}


def _plain(state):
    with torch.no_grad():
        return _PLAIN[state["kind"]](state, state["way"] == "step")


def _plain_norm(state, step):
    x, w, residual = state["x"], state["weight"].float(), state["residual"]
    s = x.float() if residual is None else x.float() + residual.float()
    r = 1.0 / torch.sqrt((s * s).mean(1, keepdim=True) + EPS)
    n = s * r
    out = {"y": (n * w).to(x.dtype)}
    if residual is not None:
        out["h"] = s.to(residual.dtype)
    if not step:
        return out
    dy = state["dy"].float()
    t = dy * w
    ds = r * (t - n * (t * n).mean(1, keepdim=True))
    if residual is not None:
        ds = ds + state["dh"].float()
        out["dresidual"] = ds.to(residual.dtype)
    out["dx"] = ds.to(x.dtype)
    if state["weight"].requires_grad:
        out["dweight"] = (dy * n).sum(0, dtype=torch.float64).to(state["weight"].dtype)
    return out


def _plain_route(state, step):
    logits, k, bias = state["logits"], state["top_k"], state["bias"]
    tokens, e = logits.shape
    # which keys are larger is decided next to equal keys: 64 bits
    l64 = logits.double()
    top = l64.amax(1, keepdim=True)
    if state["score"] == "softmax":
        s = torch.exp(l64 - top)
        s = s / s.sum(1, keepdim=True)
    else:
        s = 1.0 / (1.0 + torch.exp(-l64))
    # the scores are ordered as the logits are; only sums of scores need them
    keys = l64
    if bias is not None:
        keys = s + bias.double()
    elif state["group_score"] == "top2" and state["groups"] > 1:
        keys = s
    if state["groups"] > 1:
        g = state["groups"]
        best = keys.view(tokens, g, e // g).sort(dim=2, descending=True).values
        if state["group_score"] == "top2":
            best = best[:, :, :2].sum(2)
        else:
            best = best[:, :, 0]
        kept = best.sort(dim=1, descending=True, stable=True).indices[:, :state["top_groups"]]
        live = torch.zeros(tokens, g, dtype=torch.bool, device="cuda").scatter_(1, kept, True)
        keys = torch.where(live.repeat_interleave(e // g, dim=1), keys, -math.inf)
    chosen = keys.sort(dim=1, descending=True, stable=True).indices[:, :k]
    s = s.float()
    picked = s.gather(1, chosen)
    total = 1.0
    if state["renormalize"]:
        total = picked.sum(1, keepdim=True)
    p = picked / total
    weights, experts = p * state["scale"], chosen.to(torch.int32)
    mask = None if state["mask"] is None else state["mask"].unsqueeze(1)
    if mask is not None:
        weights, experts = torch.where(mask, weights, 0.0), torch.where(mask, experts, -1)
    out = {"weights": weights, "experts": experts}
    if step:
        dp = state["dweights"] * state["scale"]
        if state["renormalize"]:
            dp = (dp - (dp * p).sum(1, keepdim=True)) / total
        ds = torch.zeros_like(s).scatter_(1, chosen, dp)
        if state["score"] == "softmax":
            dl = s * (ds - (ds * s).sum(1, keepdim=True))
        else:
            dl = ds * s * (1.0 - s)
        if mask is not None:
            dl = torch.where(mask, dl, 0.0)
        out["dlogits"] = dl.to(logits.dtype)
    return out


def _order(chosen, num_experts):
    """(offsets, slots, positions) of int32 *chosen* [tokens, top_k]: the slots in their experts' order."""
    n = chosen.numel()
    key = torch.where(chosen >= 0, chosen, num_experts).view(-1).long()
    by_expert = torch.sort(key, stable=True).indices
    counts = torch.zeros(num_experts + 1, dtype=torch.long, device="cuda").scatter_add_(0, key, torch.ones_like(key))
    offsets = torch.zeros(num_experts + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = counts[:num_experts].cumsum(0)
    at = torch.arange(n, device="cuda")
    positions = torch.empty(n, dtype=torch.long, device="cuda").scatter_(0, by_expert, at)
    positions = torch.where(key < num_experts, positions, -1).to(torch.int32).view(chosen.shape)
    slots = torch.where(at < offsets[-1], by_expert, -1).to(torch.int32)
    return offsets, slots, positions


def _plain_dispatch(state, step):
    x, chosen = state["x"].detach(), state["experts"]
    offsets, slots, positions = _order(chosen, state["num_experts"])
    token = slots.clamp(min=0) // chosen.shape[1]
    rows = torch.where((slots >= 0).unsqueeze(1), x[token], 0.0)
    out = {"offsets": offsets, "slots": slots, "positions": positions, "rows": rows}
    if step:
        by_token = state["drows"][positions.clamp(min=0)].float()
        out["dx"] = torch.where((positions >= 0).unsqueeze(2), by_token, 0.0).sum(1).to(x.dtype)
    return out


def _plain_combine(state, step):
    y, weights, residual = state["y"].detach(), state["weights"].detach().unsqueeze(2), state["residual"]
    positions = state["order"][2]
    live = positions >= 0
    by_token = torch.where(live.unsqueeze(2), y[positions.clamp(min=0)].float(), 0.0)  # [tokens, top_k, hidden]
    total = (by_token * weights).sum(1)
    if residual is not None:
        total = total + residual.float()
    out = {"out": total.to(y.dtype)}
    if step:
        dout = state["dout"].float().unsqueeze(1)
        dy = y.new_zeros(y.shape[0] + 1, y.shape[1])  # (the last row: of no expert)
        dy[torch.where(live, positions, y.shape[0])] = (dout * weights).to(y.dtype)
        out["dy"], out["dweights"] = dy[:-1], (dout * by_token).sum(2)
    return out


_PLAIN = {"norm": _plain_norm, "route": _plain_route, "dispatch": _plain_dispatch, "combine": _plain_combine}


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    step = case["way"] == "step"
    size = SIZES[case["dtype"]]
    if case["kind"] == "norm":
        n = case["rows"] * case["hidden"]
        residual = SIZES.get(case["residual"], 0)
        each = 2 * size + 2 * residual  # x, y, residual, h
        if step:
            each += 2 * size + residual + (residual if residual != size else 0)  # dy, dx, dh, dresidual
        weight = SIZES[case["weight"]] * case["hidden"] * (2 if step and case["weight_grad"] else 1)
        return {"bytes": n * each + weight, "flops": n * (14 if step else 5)}
    if case["kind"] == "route":
        n, picked = case["tokens"] * case["experts"], case["tokens"] * case["top_k"]
        return {"bytes": n * size * (2 if step else 1) + picked * (12 if step else 8) +
                (case["tokens"] if case["padded"] else 0) + (4 * case["experts"] if case["bias"] else 0),
                "flops": n * (12 if step else 8)}
    rows, tokens = case["tokens"] * case["top_k"], case["tokens"]
    line = case["hidden"] * size
    if case["kind"] == "dispatch":  # the choice in; offsets, slots and positions out; x in, the rows out
        return {"bytes": (12 * rows + 4 * case["experts"] + (tokens + rows) * line) +
                ((tokens + rows) * line if step else 0),
                "flops": rows * case["hidden"] if step else rows}
    total = 8 * rows + (rows + tokens * (2 if case["residual"] else 1)) * line
    if step:
        total += 4 * rows + (rows + tokens) * line
    return {"bytes": total, "flops": rows * case["hidden"] * (5 if step else 2)}


# ------------------------------------------------------------------ the same in 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return _EXACT[case["kind"]](case, state, case["way"] == "step")


def _exact_norm(case, state, step):
    h = state["x"].double()
    if state["residual"] is not None:
        h = h + state["residual"].double()
    width = h.shape[1]
    w = state["weight"].double()
    power = torch.linalg.vector_norm(h, dim=1, keepdim=True).square() / width + EPS
    out = {"y": h * w / power.sqrt()}
    if state["residual"] is not None:
        out["h"] = h
    if step:
        g = state["dy"].double()
        along = torch.linalg.vecdot(g * w, h, dim=1).unsqueeze(1)
        grad = g * w * power.pow(-0.5) - h * along * power.pow(-1.5) / width
        if state["weight"].requires_grad:
            out["dweight"] = torch.linalg.vecdot(g, h / power.sqrt(), dim=0)
        if state["residual"] is not None:
            grad = grad + state["dh"].double()
            out["dresidual"] = grad
        out["dx"] = grad
    return out


def _exact_route(case, state, step):
    logits = state["logits"].detach().double()
    tokens, e = logits.shape
    k, scale = case["top_k"], case["scale"]
    softmax = case["score"] == "softmax"
    score = torch.softmax(logits, 1) if softmax else torch.sigmoid(logits)
    tops = case["group_score"] == "top2" and case["groups"] > 1
    key = score if tops or case["bias"] else logits
    if case["bias"]:
        key = key + state["bias"].double()
    gone = torch.zeros_like(key, dtype=torch.bool)
    if case["groups"] > 1:
        group = key.unflatten(1, (case["groups"], -1))
        value = group.topk(min(2, group.shape[2]), dim=2).values.sum(2) if tops else group.amax(2)
        out_of = torch.ones_like(value, dtype=torch.bool)
        for _ in range(case["top_groups"]):
            best = torch.where(out_of, value, -math.inf).amax(1, keepdim=True)
            first = ((value == best) & out_of).to(torch.int8).argmax(1)
            out_of[torch.arange(tokens, device="cuda"), first] = False
        gone |= out_of.repeat_interleave(e // case["groups"], 1)
    chosen = torch.empty(tokens, k, dtype=torch.long, device="cuda")
    lowest = torch.arange(e, device="cuda")
    for j in range(k):  # the largest key left, the lowest index among equal ones
        best = torch.where(gone, -math.inf, key).amax(1, keepdim=True)
        chosen[:, j] = torch.where((key == best) & ~gone, lowest, e).amin(1)
        gone[torch.arange(tokens, device="cuda"), chosen[:, j]] = True
    absent = torch.zeros(tokens, 1, dtype=torch.bool, device="cuda") if state["mask"] is None else \
        ~state["mask"].unsqueeze(1)
    picked = score.gather(1, chosen)
    weights = scale * (picked / picked.sum(1, keepdim=True) if case["renormalize"] else picked)
    out = {"weights": weights.masked_fill(absent, 0.0), "experts": chosen.to(torch.int32).masked_fill(absent, -1)}
    if step:
        leaf = logits.clone().requires_grad_(True)
        with torch.enable_grad():
            s = torch.softmax(leaf, 1) if softmax else torch.sigmoid(leaf)
            s = s.gather(1, chosen)
            w = scale * (s / s.sum(1, keepdim=True) if case["renormalize"] else s)
            w.masked_fill(absent, 0.0).backward(state["dweights"].double())
        out["dlogits"] = leaf.grad
    return out


def _exact_dispatch(case, state, step):
    chosen, x = state["experts"].long().view(-1), state["x"].detach().double()
    n, e, k = chosen.numel(), case["experts"], case["top_k"]
    ends = [0]
    order = []
    for expert in range(e):
        mine = (chosen == expert).nonzero().view(-1)
        order.append(mine)
        ends.append(ends[-1] + mine.numel())
    order = torch.cat(order)
    slots = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    slots[:order.numel()] = order.to(torch.int32)
    positions = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    positions[order] = torch.arange(order.numel(), dtype=torch.int32, device="cuda")
    rows = torch.zeros(n, x.shape[1], dtype=torch.float64, device="cuda")
    rows[:order.numel()] = x[torch.div(order, k, rounding_mode="floor")]
    out = {"offsets": torch.tensor(ends, dtype=torch.int32, device="cuda"), "slots": slots,
           "positions": positions.view(-1, k), "rows": rows}
    if step:
        by_slot = torch.zeros(n, x.shape[1], dtype=torch.float64, device="cuda")
        by_slot[order] = state["drows"][:order.numel()].double()
        out["dx"] = by_slot.view(-1, k, x.shape[1]).sum(1)
    return out


def _exact_combine(case, state, step):
    _, slots, positions = state["order"]
    tokens, k = positions.shape
    live = int((slots >= 0).sum())
    slot = slots[:live].long()
    by_slot = torch.zeros(tokens * k, case["hidden"], dtype=torch.float64, device="cuda")
    by_slot[slot] = state["y"].detach()[:live].double()
    by_slot = by_slot.view(tokens, k, -1)
    weights = state["weights"].detach().double()
    out = {"out": torch.bmm(weights.unsqueeze(1), by_slot).squeeze(1)}
    if state["residual"] is not None:
        out["out"] += state["residual"].double()
    if step:
        dout = state["dout"].double()
        dy = torch.zeros(tokens * k, case["hidden"], dtype=torch.float64, device="cuda")
        dy[:live] = dout[torch.div(slot, k, rounding_mode="floor")] * weights.view(-1)[slot].unsqueeze(1)
        out["dy"] = dy
        out["dweights"] = (by_slot * dout.unsqueeze(1)).sum(2)
    return out


_EXACT = {"norm": _exact_norm, "route": _exact_route, "dispatch": _exact_dispatch, "combine": _exact_combine}
