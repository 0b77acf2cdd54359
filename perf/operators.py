"""The operators of a fine-tuning step around the frozen NF4 products, as measurable cases.

* ``gated``: the gated feed-forward block on NF4 weights, ``silu(x Wg^T) * (x Wu^T)``, alone (``forward``)
  or with the gradient of its input (``step``);
* ``adamw``: one AdamW step over many tensors, with its states in 32 bits or in 8;
* ``norm``: the gradient norm over many tensors, and the factor that clips them.

``listed()`` holds the named cases, ``draw(rng)`` gives others of the same ranges, ``prepare`` makes what a program
holds before the call, ``run`` makes the call (in plain torch, or through the package where ``own`` is true), and
``exact`` computes the same outputs in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

# Hidden size, intermediate size and key/value width of the models that the tests and the benchmark use.
MODELS = {"1.1B": (2048, 5632, 256), "8B": (4096, 14336, 1024)}

BLOCK = 256  # elements that share one scale of an 8-bit state; every tensor starts on a multiple of it
LR, BETAS, EPS, DECAY = 2e-4, (0.9, 0.999), 1e-8, 0.01


def listed():
    return [
        # One token through a small model's block: launches and host work.
        {"name": "gated fwd 1 row (1.1B)", "kind": "gated", "way": "forward", "rows": 1, "hidden": 2048,
         "inter": 5632, "dtype": "bf16"},
        # An odd batch of sequences decoding through an 8B block: the packed weight is the traffic.
        {"name": "gated fwd 13 rows (8B)", "kind": "gated", "way": "forward", "rows": 13, "hidden": 4096,
         "inter": 14336, "dtype": "fp16"},
        # A short ragged prompt.
        {"name": "gated fwd 333 rows (8B)", "kind": "gated", "way": "forward", "rows": 333, "hidden": 4096,
         "inter": 14336, "dtype": "bf16"},
        # A training batch, forward only (the pass that a recomputing pipeline runs first).
        {"name": "gated fwd 8192 rows (8B)", "kind": "gated", "way": "forward", "rows": 8192, "hidden": 4096,
         "inter": 14336, "dtype": "bf16"},
        # A short fine-tuning sample on a small model: forward and the input's gradient.
        {"name": "gated step 509 rows (1.1B)", "kind": "gated", "way": "step", "rows": 509, "hidden": 2048,
         "inter": 5632, "dtype": "fp16"},
        # A training batch through an 8B block.
        {"name": "gated step 4096 rows (8B)", "kind": "gated", "way": "step", "rows": 4096, "hidden": 4096,
         "inter": 14336, "dtype": "bf16"},
        # Rank-16 adapters of one layer: the smallest set that is trained, launches and host work.
        {"name": "adamw32 1.1B layer adapters", "kind": "adamw", "bits": 32, "tensors": "adapters",
         "hidden": 2048, "inter": 5632, "kv": 256, "layers": 1, "rank": 16, "param": "bf16", "master": False},
        # Rank-16 adapters on every projection of an 8B model, with 32-bit masters of the 16-bit parameters.
        {"name": "adamw32 8B adapters masters", "kind": "adamw", "bits": 32, "tensors": "adapters",
         "hidden": 4096, "inter": 14336, "kv": 1024, "layers": 32, "rank": 16, "param": "bf16", "master": True},
        # The same adapters in 32 bits, with 8-bit states.
        {"name": "adamw8 8B adapters", "kind": "adamw", "bits": 8, "tensors": "adapters", "hidden": 4096,
         "inter": 14336, "kv": 1024, "layers": 32, "rank": 16, "param": "fp32", "master": False},
        # Every projection of four small layers trained in full, with 8-bit states.
        {"name": "adamw8 four 1.1B layers", "kind": "adamw", "bits": 8, "tensors": "dense", "hidden": 2048,
         "inter": 5632, "kv": 256, "layers": 4, "rank": 0, "param": "bf16", "master": False},
        # The norm over one layer's adapter gradients, and over those of a whole 8B model.
        {"name": "norm 1.1B layer adapters", "kind": "norm", "tensors": "adapters", "hidden": 2048,
         "inter": 5632, "kv": 256, "layers": 1, "rank": 16, "grad": "bf16"},
        {"name": "norm 8B adapters", "kind": "norm", "tensors": "adapters", "hidden": 4096, "inter": 14336,
         "kv": 1024, "layers": 32, "rank": 32, "grad": "bf16"},
    ]


# ------------------------------------------------------------------ drawn cases

_MOST_GATED = 8192 * 4096 * 14336  # rows x hidden x intermediate of the largest listed forward
_MOST_TENSORS = 180_000_000        # elements of the largest listed set of tensors


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _multiple(rng, low, high, step):
    return max(low, min(high, _log_int(rng, low, high) // step * step))


def draw(rng):
    kind = rng.choice(["gated", "gated", "gated", "gated", "adamw", "adamw", "adamw", "norm"])
    if kind == "gated":
        way = rng.choice(["forward", "forward", "step"])
        if rng.random() < 0.5:
            hidden, inter, _ = rng.choice(list(MODELS.values()))
        else:
            hidden, inter = _multiple(rng, 512, 5120, 64), _multiple(rng, 384, 14336, 32)
        most = _MOST_GATED // (2 if way == "step" else 1)
        rows = min(_log_int(rng, 1, 8192), most // (hidden * inter))
        return {"kind": kind, "way": way, "rows": rows, "hidden": hidden, "inter": inter,
                "dtype": rng.choice(["bf16", "fp16"])}
    tensors = rng.choice(["adapters", "adapters", "dense", "ragged"])
    if rng.random() < 0.5:
        hidden, inter, kv = rng.choice(list(MODELS.values()))
    else:  # widths that are no multiples of anything
        hidden = _log_int(rng, 500, 5000)
        inter, kv = round(hidden * rng.uniform(2.0, 4.0)), round(hidden * rng.uniform(0.1, 1.0))
    case = {"kind": kind, "tensors": tensors, "hidden": hidden, "inter": inter, "kv": kv,
            "layers": 1 if tensors == "dense" else _log_int(rng, 1, 32),
            "rank": 0 if tensors == "dense" else rng.choice([8, 16, 32]) if tensors == "adapters" else
            _log_int(rng, 3, 60)}
    while sum(_sizes(case)) > _MOST_TENSORS:
        case["hidden"], case["inter"], case["kv"] = (case[w] * 3 // 4 for w in ("hidden", "inter", "kv"))
    if kind == "norm":
        return {**case, "grad": rng.choice(["bf16", "fp16", "fp32"])}
    param = rng.choice(["bf16", "fp16", "fp32"])
    return {**case, "bits": rng.choice([32, 8]), "param": param, "master": param != "fp32" and rng.random() < 0.5}


def _sizes(case):
    """Elements of every tensor of a set."""
    h, i, kv, r = case["hidden"], case["inter"], case["kv"], case["rank"]
    shapes = [(h, h), (kv, h), (kv, h), (h, h), (i, h), (i, h), (h, i)]  # q, k, v, o, gate, up, down [out, in]
    if case["tensors"] == "dense":
        one = [n * k for n, k in shapes]
    elif case["tensors"] == "adapters":
        one = [size for n, k in shapes for size in (r * k, n * r)]
    else:  # norms and biases beside a few matrices: `rank` columns here
        one = [1, h, h, 37, r * h, i, kv, r * r * 7, h * r + 3]
    return one * case["layers"]


# ------------------------------------------------------------------ inputs, from the seed alone

_LEVELS = (  # the 16 NF4 levels (QLoRA, arXiv 2305.14314, appendix E)
    -1.0, -0.6961928009986877, -0.5250730514526367, -0.39491748809814453, -0.28444138169288635,
    -0.18477343022823334, -0.09105003625154495, 0.0, 0.07958029955625534, 0.16093020141124725,
    0.24611230194568634, 0.33791524171829224, 0.44070982933044434, 0.5626170039176941, 0.7229568362236023, 1.0)


def _normal(seed, place, shape, std, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 64 + place)
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)


def _weight(seed, rows, cols):
    """An N(0, 0.02) weight as NF4 holds it: (packed [rows cols / 2], absmax [rows cols / 64])."""
    w = _normal(seed, 1, (rows * cols // 64, 64), 0.02)
    top = w.abs().amax(1)
    levels = torch.tensor(_LEVELS, device="cuda")
    codes = torch.bucketize(w.div_(top.unsqueeze(1)), (levels[1:] + levels[:-1]) / 2).to(torch.uint8).view(-1, 2)
    return (codes[:, 0] << 4) | codes[:, 1], top


def _starts(case):
    """First element of every tensor in the flat buffers, and their length."""
    starts, at = [], 0
    for n in _sizes(case):
        starts.append(at)
        at += -(-n // BLOCK) * BLOCK
    return starts, at


def _inside(case, flat):
    """*flat* with zeros in the gaps between the tensors."""
    at = 0
    for n in _sizes(case):
        end = at + -(-n // BLOCK) * BLOCK
        flat[at + n:end].zero_()
        at = end
    return flat


def _views(case, flat):
    return [flat[s:s + n] for s, n in zip(_starts(case)[0], _sizes(case))]


def _grad_dtype(case):
    return DTYPES[case["param"]] if case["kind"] == "adamw" else DTYPES[case["grad"]]


def _gradient(case, seed, place=20):
    """Gradients whose size varies from tensor to tensor and from row to row, as they do in training."""
    total = _starts(case)[1]
    size = torch.exp(_normal(seed, place + 1, (total // BLOCK, 1), 1.0))
    g = _normal(seed, place, (total // BLOCK, BLOCK), 1e-3).mul_(size)
    return _inside(case, g.to(_grad_dtype(case)).view(-1))


def _codes_of(x, signed):
    """8-bit codes and block scales of fp32 values *x* (whole blocks): the nearest level, fp32 arithmetic."""
    rows = x.view(-1, BLOCK)
    top = rows.abs().amax(1, keepdim=True)
    s = rows.abs() * torch.where(top >= 2.0 ** -126, 1.0 / top, 0.0)
    last = 6 if signed else 7
    # segment z: 8^-(z + 1) <= s < 8^-z, the last one down to zero
    z = torch.zeros_like(s, dtype=torch.int32)
    for k in range(1, last + 1):
        z += (s < 8.0 ** -k).to(torch.int32)
    n = torch.bitwise_left_shift(torch.ones_like(z), last - z)
    y = s * torch.bitwise_left_shift(torch.ones_like(z), 3 * z).float()
    step = torch.where(z == last, y, (y - 0.125) * (n.float() * (8.0 / 7.0)))
    q = (n - 1 + torch.round(step).to(torch.int32)).clamp_(max=2 ** (last + 1) - 1)
    if signed:
        q += (rows < 0).to(torch.int32) * 128
    else:
        q = torch.where((q == 0) & (rows > 0), 1, q)  # a second moment that is not zero does not become it
    return q.to(torch.uint8).view(-1), top.view(-1)


def _table(signed, dtype=torch.float32):
    """The value of every code, relative to its block's scale."""
    last, values = (6, 128) if signed else (7, 256)
    half = [0.0]
    for q in range(1, values):
        k = q.bit_length() - 1
        half.append(math.ldexp(7 * q + 7 - 6 * 2 ** k, 2 * k - 3 - 3 * last))
    return torch.tensor(half + [-v for v in half] if signed else half, dtype=dtype, device="cuda")


def _values_of(codes, scales, signed, dtype=torch.float32):
    return (_table(signed, dtype)[codes.long()].view(-1, BLOCK) * scales.to(dtype).unsqueeze(1)).view(-1)


def _moments(case, seed, total):
    """Both moments after a while of training, in fp32."""
    size = torch.exp(_normal(seed, 31, (total // BLOCK, 1), 1.0))
    m = _inside(case, _normal(seed, 30, (total // BLOCK, BLOCK), 3e-4).mul_(size).view(-1))
    v = _normal(seed, 32, (total // BLOCK, BLOCK), 1e-3).mul_(size).square_()
    v += 1e-7 * size.square() * torch.exp(_normal(seed, 33, (total // BLOCK, BLOCK), 2.0))
    return m, _inside(case, v.view(-1))


def prepare(case, seed):
    if case["kind"] == "gated":
        dtype, h, i = DTYPES[case["dtype"]], case["hidden"], case["inter"]
        packed, absmax = _weight(seed, 2 * i, h)
        state = {"kind": "gated", "way": case["way"], "packed": packed, "absmax": absmax, "shape": (2 * i, h),
                 "x": _normal(seed, 2, (case["rows"], h), 1.0, dtype)}
        if case["way"] == "step":
            state["dh"] = _normal(seed, 3, (case["rows"], i), 1.0, dtype)
            state["x"].requires_grad_(True)
        return state
    state = {"kind": case["kind"], "flat_grad": _gradient(case, seed)}
    state["grads"] = _views(case, state["flat_grad"])
    if case["kind"] == "norm":
        state["max_norm"] = 1.0
        return state
    total = state["flat_grad"].numel()
    m, v = _moments(case, seed, total)
    master = _inside(case, _normal(seed, 34, (total,), 0.02))
    state["flat_param"] = master.to(DTYPES[case["param"]])
    state["params"] = _views(case, state["flat_param"])
    if case["master"]:
        state["flat_master"] = master
        state["masters"] = _views(case, master)
    state["step"] = 100 + int(seed) % 100
    state["scale"] = torch.rand((), device="cuda", generator=torch.Generator(device="cuda").manual_seed(int(seed)))
    state["bits"] = case["bits"]
    if case["bits"] == 32:
        for name, flat in (("m", m), ("v", v)):
            state["flat_" + name] = flat
            state[name] = _views(case, flat)
        return state
    starts, sizes = _starts(case)[0], _sizes(case)
    for name, flat, signed in (("m", m, True), ("v", v, False)):
        codes, scales = _codes_of(flat, signed)
        state["flat_" + name], state["flat_" + name + "_scale"] = codes, scales
        state[name] = _views(case, codes)
        state[name + "_scale"] = [scales[s // BLOCK:s // BLOCK + -(-n // BLOCK)] for s, n in zip(starts, sizes)]
    return state


# ------------------------------------------------------------------ one pass

def run(state):
    return (_own if own else _plain)(state)


def _own(state):
    if state["kind"] == "gated":
        from stratum_amd import nf4_gated
        x = state["x"]
        if state["way"] == "forward":
            with torch.no_grad():
                return nf4_gated(x, state["packed"], state["absmax"], state["shape"])
        x.grad = None
        h = nf4_gated(x, state["packed"], state["absmax"], state["shape"])
        h.backward(state["dh"])
        return {"h": h.detach(), "dx": x.grad}
    if state["kind"] == "norm":
        from stratum_amd.optim import grad_norm
        return grad_norm(state["grads"], state["max_norm"])
    from stratum_amd.optim import AdamWTensors, state_values
    tensors = state.get("tensors")
    if tensors is None:  # as an optimizer makes it once for its parameters
        tensors = state["tensors"] = AdamWTensors(
            state["params"], state["m"], state["v"], masters=state.get("masters"),
            scales=(state["m_scale"], state["v_scale"]) if state["bits"] == 8 else None)
    tensors.step(state["grads"], step=state["step"], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY,
                 grad_scale=state["scale"])
    out = {"param": state["flat_param"]}
    if "flat_master" in state:
        out["master"] = state["flat_master"]
    if state["bits"] == 32:
        return {**out, "m": state["flat_m"], "v": state["flat_v"]}
    return {**out, "m": state_values(state["flat_m"], state["flat_m_scale"], signed=True),
            "v": state_values(state["flat_v"], state["flat_v_scale"], signed=False)}


def _plain_weight(state, dtype):
    """The dequantized weight: fp32 level times absmax, rounded to the type (the value that a weight has)."""
    levels = torch.tensor(_LEVELS, device="cuda")
    packed = state["packed"]
    w = torch.stack([levels[(packed >> 4).long()], levels[(packed & 15).long()]], 1).view(-1, 64)
    return (w * state["absmax"].unsqueeze(1)).to(dtype).float().view(state["shape"])


def _plain(state):
    if state["kind"] == "gated":
        dtype, inter = state["x"].dtype, state["shape"][0] // 2
        x, w = state["x"].detach().float(), _plain_weight(state, state["x"].dtype)
        gu = x @ w.t()
        g, u = gu[:, :inter], gu[:, inter:]
        s = 1.0 / (1.0 + torch.exp(-g))
        h = (g * s * u).to(dtype)
        if state["way"] == "forward":
            return h
        dh = state["dh"].float()
        dgu = torch.cat([dh * u * s * (1.0 + g * (1.0 - s)), dh * g * s], 1)
        return {"h": h, "dx": (dgu @ w).to(dtype)}
    if state["kind"] == "norm":
        norm = state["flat_grad"].float().square().sum().sqrt()
        factor = torch.clamp(state["max_norm"] / (norm + 1e-6), max=1.0)
        return torch.stack([norm, factor])
    m, v = state["flat_m"], state["flat_v"]
    if state["bits"] == 8:
        m = _values_of(m, state["flat_m_scale"], True)
        v = _values_of(v, state["flat_v_scale"], False)
    g = state["flat_grad"].float() * state["scale"]
    b1, b2 = BETAS
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * (1 - b2) * g
    p = state.get("flat_master", state["flat_param"]).float()
    t = state["step"]
    denominator = v.sqrt() / math.sqrt(1 - b2 ** t) + EPS
    p = p * (1 - LR * DECAY) - (LR / (1 - b1 ** t)) * m / denominator
    out = {"param": state["flat_param"].copy_(p)}
    if "flat_master" in state:
        out["master"] = state["flat_master"].copy_(p)
    if state["bits"] == 32:
        return {**out, "m": state["flat_m"].copy_(m), "v": state["flat_v"].copy_(v)}
    for name, value, signed in (("m", m, True), ("v", v, False)):
        codes, scales = _codes_of(value, signed)
        state["flat_" + name].copy_(codes)
        state["flat_" + name + "_scale"].copy_(scales)
        out[name] = _values_of(codes, scales, signed)
    return out


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    if case["kind"] == "gated":
        m, h, i = case["rows"], case["hidden"], case["inter"]
        weight, product = 2 * i * h * 0.5625, 4 * m * i * h
        if case["way"] == "forward":
            return {"bytes": weight + 2 * m * (h + i), "flops": product + 6 * m * i}
        # x, dh, h, dx and the weight once; the products of the forward and of the input's gradient
        return {"bytes": weight + 4 * m * (h + i), "flops": 2 * product + 20 * m * i}
    n = sum(_sizes(case))
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if case["kind"] == "norm":
        return {"bytes": n * size[case["grad"]], "flops": 2 * n}
    param = size[case["param"]]
    each = 2 * param + param + (8 if case["master"] else 0)  # parameter, gradient, master
    if case["master"]:
        each -= param  # the 16-bit copy is only written
    # the states read and written; those of 8 bits are also given back as the fp32 values they stand for
    each += 16 if case["bits"] == 32 else 4 + 16 / BLOCK + 8
    return {"bytes": each * n, "flops": 20 * n}


# ------------------------------------------------------------------ the same in 64 bits

def _exact_codes(x, signed):
    """The values that *x* takes when it is held in 8 bits: the nearest level of each block's scale."""
    rows = x.view(-1, BLOCK)
    top = rows.abs().amax(1, keepdim=True)
    ratio = torch.where(top > 0, rows.abs() / top, 0.0)
    levels = _table(signed, torch.float64)[:128 if signed else 256]
    at = torch.bucketize(ratio, (levels[1:] + levels[:-1]) / 2)
    if not signed:
        at = torch.where((at == 0) & (rows > 0), 1, at)
    return (levels[at] * torch.sign(rows) * top).view(-1)


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "gated":
        dtype, inter, x = DTYPES[case["dtype"]], case["inter"], state["x"].detach().double()
        halves = torch.empty(state["packed"].numel(), 2, dtype=torch.long, device="cuda")
        halves[:, 0], halves[:, 1] = state["packed"].long() // 16, state["packed"].long() % 16
        scale = state["absmax"].repeat_interleave(64)
        w = (torch.tensor(_LEVELS, device="cuda")[halves.view(-1)] * scale).to(dtype).double().view(state["shape"])
        del halves, scale
        gate, up = x @ w[:inter].t(), x @ w[inter:].t()
        half = 0.5 * torch.tanh(0.5 * gate) + 0.5
        h = gate * half * up
        if case["way"] == "forward":
            return h
        dh = state["dh"].double()
        dgate = dh * up * (half + gate * half * (1 - half))
        return {"h": h, "dx": dgate @ w[:inter] + (dh * gate * half) @ w[inter:]}
    grad = state["flat_grad"].double()
    if case["kind"] == "norm":
        norm = torch.linalg.vector_norm(grad)
        return torch.stack([norm, torch.clamp(state["max_norm"] / (norm + 1e-6), max=1.0)])
    grad *= state["scale"].double()
    if case["bits"] == 32:
        m, v = state["flat_m"].double(), state["flat_v"].double()
    else:
        m = _values_of(state["flat_m"], state["flat_m_scale"], True, torch.float64)
        v = _values_of(state["flat_v"], state["flat_v_scale"], False, torch.float64)
    (b1, b2), t = BETAS, state["step"]
    m = b1 * m + (1 - b1) * grad
    v = b2 * v + (1 - b2) * grad.square()
    p = state.get("flat_master", state["flat_param"]).double()
    p = p - LR * DECAY * p - LR * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + EPS)
    out = {"param": p, "master": p} if case["master"] else {"param": p}
    if case["bits"] == 8:
        m, v = _exact_codes(m, True), _exact_codes(v, False)
    return {**out, "m": m, "v": v}
