"""GPU tests of the gradient norm and the AdamW step over many tensors, against the
formulas in 64 bits, with states in 32 bits and in 8.

Bounds. u = 2^-24 is the relative rounding of fp32. m: the scaled gradient, the factor
1 - b1, their product and the sum round once each, 5 u of |b1 m| + |(1 - b1) g| with the
second order; v: 8 u (the gradient twice). The update lr m^ / (sqrt(v^) + eps): m's 5, half
of v's, the root, two products, two rounded factors, the sum and the division, 20 u of its
magnitude with |m| replaced by its terms' magnitudes. p: those, 3 u of |p|, and half a step
of the parameter's type. An 8-bit state is within half a step of its code, at most (7/8) / 2^K / 2 of
the scale, of the fp32 value, or within half the lowest level (a full one for v) below that."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)


def levels(signed):
    """The values of all codes, from the format's definition (float64)."""
    K = 6 if signed else 7
    out = [0.0]
    for q in range(1, 1 << (K + 1)):
        k = int(math.floor(math.log2(q)))
        out.append((7 * q + 7 - 6 * 2 ** k) * 2.0 ** (2 * k - 3 - 3 * K))
    return torch.tensor(out + [-v for v in out] if signed else out, dtype=torch.float64)


def normal(shape, seed, std=1.0, dtype=torch.float32, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).to(device)


def reference(p, g, m, v, t, lr, betas, eps, weight_decay, scale=1.0):
    """New (p, m, v) in 64 bits, the magnitude of m's terms, and of the update with it."""
    b1, b2 = betas
    g = g.double() * scale
    m_terms = b1 * m.abs() + (1 - b1) * g.abs()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    denominator = torch.sqrt(v / (1 - b2 ** t)) + eps
    update = lr / (1 - b1 ** t) * m / denominator
    size = lr / (1 - b1 ** t) * m_terms / denominator
    return p.double() * (1 - lr * weight_decay) - update, m, v, m_terms, size


def check_state8(codes, scales, exact, slack, signed):
    """Each value within half a step of its code from the exact one, block by block."""
    from stratum_amd.optim import state_values
    K = 6 if signed else 7
    value = state_values(codes, scales, signed=signed).double()
    scale = scales.double().repeat_interleave(256)[:value.numel()]
    ratio = (exact.abs() / scale.clamp_min(1e-300)).clamp(8.0 ** -K, 1.0)
    segment = torch.floor(-torch.log2(ratio) / 3).clamp(0, K)  # 0: [1/8, 1]
    step = 8.0 ** -segment * 0.875 / 2 ** (K - segment)
    lowest = 8.0 ** -K * (0.5 if signed else 1.0)
    bound = torch.where(exact.abs() < scale * 8.0 ** -K, torch.full_like(step, lowest), step * 0.5) * scale
    assert (((value - exact).abs()) <= bound * (1 + 1e-5) + slack + 1e-45).all()
    top = torch.nn.functional.pad(exact.abs(), (0, -exact.numel() % 256)).view(-1, 256).amax(1)
    assert ((scales.double() - top).abs() <= 8 * U * top + 1e-40).all()


@pytest.mark.parametrize("signed", [True, False])
def test_state_codes_stand_for_the_levels_of_the_format(cuda, signed):
    from stratum_amd.optim import state_codes, state_values
    codes = torch.arange(256, dtype=torch.uint8, device=cuda)
    scale = torch.tensor([0.75], device=cuda)
    want = levels(signed).float() * 0.75  # exact: dyadic levels of at most 11 bits
    assert torch.equal(state_values(codes, scale, signed=signed).cpu(), want)
    # every level is kept: value -> code -> value
    again, top = state_codes(want.to(cuda), signed=signed)
    assert top.item() == 0.75
    assert torch.equal(state_values(again, top, signed=signed).cpu(), want)


@pytest.mark.parametrize("n", [1, 8, 255, 256, 257, 2048, 5001])
@pytest.mark.parametrize("signed", [True, False])
@pytest.mark.parametrize("offset", [0, 1])
def test_state_codes_take_the_nearest_level(cuda, n, signed, offset):
    from stratum_amd.optim import state_codes, state_values
    x = normal(n + offset, n, dtype=torch.float32)[offset:] * torch.exp(3 * normal(n, n + 1))
    x = x if signed else x.abs()
    codes, scales = state_codes(x, signed=signed)
    scale = scales.repeat_interleave(256)[:n].double()
    lev = levels(signed).to(cuda)
    d = (x.double().unsqueeze(1) - lev * scale.unsqueeze(1)).abs()
    if not signed:
        d[:, 0] = torch.where(x > 0, float("inf"), d[:, 0])
    got = (state_values(codes, scales, signed=signed).double() - x.double()).abs()
    # the fp32 ratio is off by two roundings, which a step's width turns into a few ulps of the scale
    assert (got <= d.amin(1) + 4 * U * scale).all()


def test_state_codes_of_blocks_that_have_no_scale(cuda):
    from stratum_amd.optim import state_codes, state_values
    x = torch.zeros(5 * 256, device=cuda)
    x[256 + 7] = 1e-41      # a subnormal scale: nothing but zeros
    x[2 * 256 + 9] = math.inf
    x[3 * 256 + 1] = math.nan
    x[4 * 256] = 1e-30
    codes, scales = state_codes(x, signed=True)
    back = state_values(codes, scales, signed=True).view(5, 256)
    assert (back[0] == 0).all() and (back[1] == 0).all()
    assert back[2, 9] == math.inf and back[3].isnan().all()
    assert back[4, 0] == x[4 * 256] and (back[4, 1:] == 0).all()
    codes, _ = state_codes(torch.cat([torch.full((256,), 1e-38, device=cuda), torch.ones(1, device=cuda)])[1:],
                           signed=False)
    assert (codes > 0).all()  # a second moment that is not zero never becomes zero


SIZES = [1, 7, 255, 256, 257, 2047, 2049, 40_000]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("param", DTYPES)
@pytest.mark.parametrize("grad", DTYPES)
@pytest.mark.parametrize("master", [False, True])
def test_step_matches_the_formula(cuda, bits, param, grad, master):
    from stratum_amd.optim import AdamWTensors, state_codes, state_values
    t, scale = 7, torch.tensor(0.37, device=cuda)
    p32 = [normal(n, n, 0.1) for n in SIZES]
    ps = [p.to(param) for p in p32]
    gs = [normal(n, n + 1, 0.01, grad) for n in SIZES]
    ms, vs = [normal(n, n + 2, 0.01) for n in SIZES], [normal(n, n + 3, 0.01).square() for n in SIZES]
    scales = None
    if bits == 8:
        cm, cv = [state_codes(m, signed=True) for m in ms], [state_codes(v, signed=False) for v in vs]
        ms, vs = [state_values(*c, signed=True) for c in cm], [state_values(*c, signed=False) for c in cv]
        scales = ([c[1] for c in cm], [c[1] for c in cv])
        held = ([c[0] for c in cm], [c[0] for c in cv])
    else:
        held = ([m.clone() for m in ms], [v.clone() for v in vs])
    masters = [p.clone() for p in p32] if master else None
    old = [(q if master else p).double() for p, q in zip(ps, p32)]
    AdamWTensors(ps, *held, masters=masters, scales=scales).step(gs, step=t, grad_scale=scale, **HYPER)
    for i in range(len(SIZES)):
        p, m, v, terms, size = reference(old[i], gs[i], ms[i].double(), vs[i].double(), t, scale=scale.double(), **HYPER)
        fp32 = 3 * U * old[i].abs() + 20 * U * size + 1e-40
        if master:
            assert ((masters[i].double() - p).abs() <= fp32).all()
            assert torch.equal(ps[i], masters[i].to(param))
        else:
            assert ((ps[i].double() - p).abs() <= fp32 + (HALF_STEP[param] + U) * p.abs() + 2.0 ** -25).all()
        if bits == 32:
            assert ((held[0][i].double() - m).abs() <= 5 * U * terms).all()
            assert ((held[1][i].double() - v).abs() <= 8 * U * v + 1e-45).all()
        else:
            check_state8(held[0][i], scales[0][i], m, 5 * U * terms, True)
            check_state8(held[1][i], scales[1][i], v, 8 * U * v, False)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [55, 56, 57, 130])
def test_every_tensor_of_a_long_list_is_stepped_wherever_it_starts(cuda, bits, count):
    """More tensors than one launch takes, empty ones among them, at odd addresses; equal
    bit for bit to the same tensors one by one and aligned."""
    from stratum_amd.optim import AdamWTensors, state_codes
    sizes = [(37 * i) % 700 if i % 9 else 0 for i in range(count)]

    def make(odd):
        def place(x):
            if not odd:
                return x.clone()
            box = torch.empty(x.numel() + 3, dtype=x.dtype, device=x.device)
            box[3:] = x
            return box[3:]
        ps = [place(normal(n, i, 0.1, torch.bfloat16)) for i, n in enumerate(sizes)]
        gs = [place(normal(n, i + 500, 0.01, torch.bfloat16)) for i, n in enumerate(sizes)]
        m, v = [normal(n, i + 900, 0.01) for i, n in enumerate(sizes)], [normal(n, i, 0.1).square() for i, n in enumerate(sizes)]
        if bits == 32:
            return ps, gs, [place(x) for x in m], [place(x) for x in v], None
        m, v = [state_codes(x, signed=True) for x in m], [state_codes(x, signed=False) for x in v]
        return ps, gs, [place(c) for c, _ in m], [place(c) for c, _ in v], ([s for _, s in m], [s for _, s in v])

    ps, gs, m, v, scales = make(True)
    AdamWTensors(ps, m, v, scales=scales).step(gs, step=3, **HYPER)
    qs, gs, m2, v2, scales2 = make(False)
    for i in range(count):
        one = ([scales2[0][i]], [scales2[1][i]]) if scales2 else None
        AdamWTensors([qs[i]], [m2[i]], [v2[i]], scales=one).step([gs[i]], step=3, **HYPER)
    for a, b in ((ps, qs), (m, m2), (v, v2), *(zip(scales, scales2) if scales else ())):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_factor_that_is_not_finite_leaves_everything_as_it_was(cuda, bits, bad):
    from stratum_amd.optim import AdamW
    ps = [torch.nn.Parameter(normal(n, n, dtype=torch.bfloat16)) for n in (300, 5)]
    opt = AdamW(ps, state_bits=bits, master_weights=True)
    for p in ps:
        p.grad = normal(p.shape, 9, dtype=torch.bfloat16)
    opt.step()
    before = [p.detach().clone() for p in ps] + [t.clone() for p in ps for k, t in opt.state[p].items() if k != "step"]
    opt.step(grad_scale=torch.tensor(bad, device=cuda))
    after = [p.detach() for p in ps] + [t for p in ps for k, t in opt.state[p].items() if k != "step"]
    assert all(torch.equal(a, b) for a, b in zip(before, after))


def test_a_gradient_that_is_not_finite_shows_in_its_own_elements(cuda):
    from stratum_amd.optim import AdamWTensors
    p, g = normal(1000, 1), normal(1000, 2)
    g[5], g[700] = math.nan, math.inf
    want = torch.ones(1000, dtype=torch.bool, device=cuda)
    want[5] = want[700] = False
    AdamWTensors([p], [torch.zeros_like(p)], [torch.zeros_like(p)]).step([g], step=1, **HYPER)
    assert torch.equal(p.isfinite(), want)


def test_a_missing_gradient_and_an_empty_tensor(cuda):
    from stratum_amd.optim import AdamWTensors
    ps = [normal(n, n) for n in (10, 0, 300)]
    m, v = [torch.zeros_like(p) for p in ps], [torch.zeros_like(p) for p in ps]
    old = [p.clone() for p in ps]
    versions = [p._version for p in ps]
    tensors = AdamWTensors(ps, m, v)
    tensors.step([None, None, None], step=1, **HYPER)
    tensors.step([None, normal(0, 1), normal(300, 1)], step=1, **HYPER)
    assert torch.equal(ps[0], old[0]) and not torch.equal(ps[2], old[2]) and (m[0] == 0).all()
    assert [p._version for p in ps] == [versions[0], versions[1] + 1, versions[2] + 1]


def test_gradients_of_another_layout_are_read_in_the_parameters_order(cuda):
    from stratum_amd.optim import AdamWTensors
    p, g = normal((40, 70), 1), normal((70, 40), 2).t()
    q = p.clone()
    for x, y in ((p, g), (q, g.contiguous())):
        AdamWTensors([x], [torch.zeros_like(x)], [torch.zeros_like(x)]).step([y], step=1, **HYPER)
    assert torch.equal(p, q)


@pytest.mark.parametrize("bits", [32, 8])
def test_sizes_past_32_bit_offsets(cuda, bits):
    """2^31 + 1000 elements (bf16 parameters and gradients; 8-bit states, or 32-bit ones of
    8.6 GB): the elements at the start, around 2^31 and at the end."""
    from stratum_amd.optim import AdamWTensors
    n = (1 << 31) + 1000
    p = torch.full((n,), 0.5, dtype=torch.bfloat16, device=cuda)
    g = torch.zeros(n, dtype=torch.bfloat16, device=cuda)
    spots = torch.tensor([0, 1, (1 << 30) + 5, (1 << 31) - 1, 1 << 31, n - 1], device=cuda)
    g[spots] = torch.tensor([1., -2., 3., -4., 5., -6.], dtype=torch.bfloat16, device=cuda)
    kind = torch.uint8 if bits == 8 else torch.float32
    m, v = (torch.zeros(n, dtype=kind, device=cuda) for _ in range(2))
    scales = tuple([torch.zeros(-(-n // 256), device=cuda)] for _ in range(2)) if bits == 8 else None
    AdamWTensors([p], [m], [v], scales=scales).step([g], step=1, lr=0.125, weight_decay=0.0)
    want = torch.tensor([0.375, 0.625] * 3, dtype=torch.bfloat16, device=cuda)  # the first step is lr sign(g)
    assert torch.equal(p[spots], want)
    assert int((p != 0.5).sum()) == 6
    assert int((m != 0).sum()) == 6
    if bits == 32:
        assert torch.allclose(m[spots], 0.1 * g[spots].float(), rtol=1e-6, atol=0)


# ------------------------------------------------------------------ the norm

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", [[1], [7], [16383, 16385, 0, 3], [100_001] * 3, [50] * 161, [0]])
@pytest.mark.parametrize("offset", [0, 1])
def test_norm_matches_64_bits(cuda, dtype, sizes, offset):
    from stratum_amd.optim import grad_norm
    gs = [normal(n + offset, i, 0.3, dtype)[offset:] for i, n in enumerate(sizes)]
    want = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
    norm, factor = grad_norm(gs, 2.5, loss_scale=4.0).tolist()
    # fp64 sums: one rounding to fp32 each
    assert abs(norm - want / 4) <= 2 * U * want
    assert abs(factor - min(1.0, 2.5 / (want / 4 + 1e-6)) / 4) <= 2 * U * 0.25
    assert grad_norm(gs).tolist()[1] == 1.0


@pytest.mark.parametrize("value,dtype", [(1e30, torch.float32), (1e-30, torch.float32), (6e4, torch.float16),
                                         (3e38, torch.bfloat16)])
def test_norm_of_the_types_ends(cuda, value, dtype):
    from stratum_amd.optim import grad_norm
    g = torch.full((4096,), value, dtype=dtype, device=cuda)
    want = float(g[0]) * 64
    got = grad_norm([g])[0].item()
    assert got == pytest.approx(want, rel=4 * U) if want < 3.4e38 else got == math.inf


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_norm_of_gradients_that_are_not_finite(cuda, bad):
    from stratum_amd.optim import grad_norm
    gs = [normal(100_000, 1), normal(33, 2)]
    gs[1][32] = bad
    norm, factor = grad_norm(gs, 1.0).tolist()
    assert not math.isfinite(norm) and math.isnan(factor)


def test_norm_is_the_same_every_time_and_reads_other_layouts(cuda):
    from stratum_amd.optim import grad_norm
    g = normal((3000, 501), 4, dtype=torch.bfloat16)
    first = grad_norm([g, g[:77]], 1.0)
    assert all(torch.equal(grad_norm([g, g[:77]], 1.0), first) for _ in range(5))
    assert torch.allclose(grad_norm([g.t(), None, g[:77, ::2]], 1.0)[0],
                          torch.sqrt(g.double().square().sum() + g[:77, ::2].double().square().sum()).float())


# ------------------------------------------------------------------ the optimizer

def test_optimizer_follows_torchs_over_many_steps(cuda):
    """20 steps on fp32 parameters, clipped, two groups, against torch's AdamW in 64 bits."""
    from stratum_amd.optim import AdamW
    start = [normal(s, i, 0.1) for i, s in enumerate([(64, 48), (1000,), (3, 5, 7)])]
    mine = [torch.nn.Parameter(p.clone()) for p in start]
    theirs = [torch.nn.Parameter(p.double()) for p in start]

    def groups(ps):
        return [{"params": ps[:1], "lr": 1e-2}, {"params": ps[1:], "weight_decay": 0.2}]
    a = AdamW(groups(mine), lr=3e-3, max_grad_norm=0.5)
    b = torch.optim.AdamW(groups(theirs), lr=3e-3)
    for step in range(20):
        for i, (p, q) in enumerate(zip(mine, theirs)):
            p.grad = normal(p.shape, 100 * step + i, 0.05)
            q.grad = p.grad.double()
        norm = torch.nn.utils.clip_grad_norm_(theirs, 0.5)
        a.step()
        b.step()
        assert a.grad_norm[0].item() == pytest.approx(norm.item(), rel=1e-6)
    for p, q in zip(mine, theirs):
        # 20 updates of at most 3.2 lr (a moment of 0.1 g over the root of 0.001 g^2); m's errors add up to
        # 5 u / (1 - b1), v's to 8 u a step, half of which reach the root; 20 roundings of p
        assert ((p.double() - q).abs() <= 20 * ((50 + 80 + 20) * U * 3.2e-2 + 3 * U * q.abs())).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_keeps_the_states_types(cuda, bits):
    from stratum_amd.optim import AdamW

    def make():
        p = torch.nn.Parameter(normal((30, 30), 1, 0.1, torch.bfloat16))
        return p, AdamW([p], lr=1e-2, state_bits=bits, master_weights=True)

    def go(p, opt, steps):
        for s in steps:
            p.grad = normal(p.shape, s, 0.1, torch.bfloat16)
            opt.step()
    p, opt = make()
    go(p, opt, range(6))
    q, first = make()
    go(q, first, range(3))
    r, second = make()
    r.data.copy_(q.data)
    second.load_state_dict(first.state_dict())
    go(r, second, range(3, 6))
    assert torch.equal(p, r) and torch.equal(opt.state[p]["master"], second.state[r]["master"])
    assert second.state[r]["exp_avg"].dtype == (torch.uint8 if bits == 8 else torch.float32)
    assert first.state[q]["exp_avg"].data_ptr() != second.state[r]["exp_avg"].data_ptr()


def test_masters_take_what_16_bits_would_round_away(cuda):
    from stratum_amd.optim import AdamW
    p = torch.nn.Parameter(torch.ones(64, dtype=torch.bfloat16, device=cuda))
    opt = AdamW([p], lr=1e-4, weight_decay=0.0, master_weights=True)
    for _ in range(100):
        p.grad = torch.ones_like(p)
        opt.step()
    assert torch.allclose(opt.state[p]["master"], torch.full((64,), 0.99, device=cuda), rtol=1e-5, atol=0)
    assert (p < 1).all()
    with torch.no_grad():
        p.fill_(3.0)  # written from outside: the master follows
    p.grad = torch.ones_like(p)
    opt.step()
    assert (opt.state[p]["master"] > 2.99).all()


def test_a_parameter_whose_memory_was_replaced_is_found_again(cuda):
    from stratum_amd.optim import AdamW
    p = torch.nn.Parameter(normal(500, 1))
    opt = AdamW([p], lr=0.1)
    p.grad = torch.ones_like(p)
    opt.step()
    old = p.data
    kept = old.clone()
    p.data = p.data.clone()
    opt.step()
    assert torch.equal(old, kept) and not torch.equal(p.data, kept)


def test_step_and_norm_run_on_the_current_stream(cuda):
    from stratum_amd.optim import AdamW
    p = torch.nn.Parameter(normal(1 << 20, 1))
    opt = AdamW([p], lr=0.1, max_grad_norm=1e6)
    grad = normal(1 << 20, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        p.grad = torch.zeros_like(p)
        for _ in range(20):
            p.grad += grad  # queued before the step on the same stream
        opt.step()
        result = p.detach().clone()
    side.synchronize()
    assert torch.allclose((result - normal(1 << 20, 1) * (1 - 0.1 * 1e-2)).abs(), torch.full_like(result, 0.1), atol=1e-3)


def test_mixed_gradient_types_share_one_norm(cuda):
    from stratum_amd.optim import AdamW
    ps = [torch.nn.Parameter(normal(100, 1)), torch.nn.Parameter(normal(100, 2, dtype=torch.bfloat16))]
    for p in ps:
        p.grad = torch.full_like(p, 3.0)
    opt = AdamW(ps, max_grad_norm=1.0)
    opt.step()
    assert opt.grad_norm[0].item() == pytest.approx(math.sqrt(200 * 9.0), rel=1e-6)
    want = 0.1 * 3.0 / math.sqrt(200 * 9.0)
    for p in ps:
        assert torch.allclose(opt.state[p]["exp_avg"], torch.full((100,), want, device=cuda), rtol=1e-5)
