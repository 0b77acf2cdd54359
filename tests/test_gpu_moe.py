"""GPU tests of routing, sorting, gathering and combining against plain 64-bit (and integer) forms on the CPU.

Bounds, u = 2^-24: a score's exponential errs by 2 u and by u times its argument, whose size is at most the
logits' range; sums of positive terms over at most 16 values a lane and 6 steps over lanes by 22 u; a handful of products
and quotients by 8 u. A combination's sum of k products and a residual errs by (k + 1) u of its terms' sizes; a dot
product over `hidden` columns by (8 ceil(hidden / 2048) + 10) u of them. One rounding to the type is half a step."""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF, FP, F4 = torch.bfloat16, torch.float16, torch.float32
HALF = {BF: 2.0 ** -8, FP: 2.0 ** -11, F4: 2.0 ** -24}
TINY = {BF: 0.0, FP: 2.0 ** -25, F4: 0.0}
INF = float("inf")


def seeded(shape, seed, std=1.0, dtype=F4):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype)


def assert_within(got, ref, err, what):
    got = got.cpu()
    assert got.shape == ref.shape, what
    dtype = got.dtype
    off = (got.double() - ref).abs() - (HALF[dtype] * ref.abs() + TINY[dtype] + err * (1 + HALF[dtype]))
    if off.numel():
        assert not off.isnan().any(), f"{what}: NaN"
        worst = int(off.argmax())
        assert off.max() <= 0, f"{what} [{worst}]: {got.reshape(-1)[worst]} for {ref.reshape(-1)[worst]}"


# ------------------------------------------------------------------ route
def choose(logits, k, score="softmax", bias=None, groups=1, top_groups=1, group_score="max", mask=None):
    """The experts of every token, one after the other in 64 bits."""
    tokens, E = logits.shape
    l64 = logits.double()
    s = torch.softmax(l64, 1) if score == "softmax" else torch.sigmoid(l64)
    sums = group_score == "top2" and groups > 1
    key = l64 if bias is None and not sums else s + (bias.double() if bias is not None else 0.0)
    key = torch.where(l64 == -INF, -INF, key)
    out = torch.full((tokens, k), -1, dtype=torch.int32)
    order = lambda v, i: (-INF if v != v else -v, i)  # noqa: E731  (NaN first)
    for t in range(tokens):
        if mask is not None and not mask[t]:
            continue
        keys = key[t].tolist()
        live = [e for e in range(E) if keys[e] != -INF]
        if groups > 1:
            size, value = E // groups, {}
            for g in range(groups):
                best = sorted((order(keys[e], e) for e in live if e // size == g))[:2]
                if best:
                    first = [keys[i] for _, i in best]
                    value[g] = first[0] + first[1] if sums and len(first) == 2 else first[0]
            kept = [g for _, g in sorted(order(v, g) for g, v in value.items())[:top_groups]]
            live = [e for e in live if e // size in kept]
        for j, (_, e) in enumerate(sorted(order(keys[e], e) for e in live)[:k]):
            out[t, j] = e
    return out


def weigh(logits, experts, score, renormalize, scale):
    """Weights in 64 bits, differentiable."""
    l64 = logits.double()
    s = torch.softmax(l64, 1) if score == "softmax" else torch.sigmoid(l64)
    live = experts >= 0
    s = torch.where(live, s.gather(1, experts.long().clamp(min=0)), 0.0)
    if renormalize:
        s = s / s.sum(1, keepdim=True).masked_fill(~live.any(1, keepdim=True), 1.0)
    return s * scale


def check_route(logits, k, mask=None, renormalize=True, scale=1.0, seed=5, **kw):
    from stratum_amd import moe_route
    on_gpu = {n: v.cuda() if torch.is_tensor(v) else v for n, v in kw.items()}
    leaf = logits.cuda().requires_grad_(True)
    call = lambda x: moe_route(x, k, mask=mask.cuda() if mask is not None else None, renormalize=renormalize,  # noqa: E731
                               scale=scale, **on_gpu)
    weights, experts = call(leaf.detach())
    assert weights.dtype == F4 and experts.dtype == torch.int32
    want = choose(logits, k, mask=mask, **kw)
    assert torch.equal(experts.cpu(), want)
    score = kw.get("score", "softmax")
    plain = logits if mask is None else logits.masked_fill(~mask.unsqueeze(1), 0.0)  # padding may hold anything
    wide = plain.double().requires_grad_(True)
    ref = weigh(wide, want, score, renormalize, scale)
    finite = plain.double().masked_fill(plain == -INF, 0.0)
    reach = float(finite.abs().max()) * 2 if finite.numel() else 0.0  # how far two logits are apart
    rel = (2 * (2 + min(reach, 200.0) + 22 + 8)) * U
    # (a score below the smallest normal number has its own steps)
    assert_within(weights, ref.detach(), rel * ref.detach().abs() + 2.0 ** -126, "weights")
    dw = seeded(want.shape, seed)
    again, same = call(leaf)
    assert torch.equal(again, weights) and torch.equal(same, experts) and not same.requires_grad
    got, = torch.autograd.grad(again, leaf, dw.cuda())
    ref.backward(dw.double())
    assert got.dtype == logits.dtype
    d = (dw * scale).abs().double()
    if not want.numel():
        assert got.shape == logits.shape
        return
    most = (d * (want >= 0)).amax(1, keepdim=True)
    size = torch.softmax(plain.double(), 1) if score == "softmax" else torch.sigmoid(finite)
    size = size.masked_fill(~(want >= 0).any(1, keepdim=True), 0.0)
    if renormalize:  # the chosen scores' share of each other, at most one
        size = (size / size.gather(1, want.long().clamp(min=0)).masked_fill(want < 0, 0.0).sum(1, keepdim=True)
                .clamp_min(1e-300)).clamp(max=1.0)
    assert_within(got, wide.grad.masked_fill(plain == -INF, 0.0), (4 * rel * size * most).nan_to_num(0.0) + 2.0 ** -126,
                  "dlogits")


@pytest.mark.parametrize("E", [1, 2, 7, 8, 9, 16, 17, 32, 33, 60, 64, 65, 100, 128, 200, 256, 300, 512, 513, 1024])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_experts_and_scores(cuda, E, renormalize, score):
    dtype = [BF, FP, F4][E % 3]
    for k in {1, min(E, 3), min(E, 8)}:
        check_route(seeded((37, E), E + k, 2.0, dtype), k, renormalize=renormalize, score=score, scale=1.0 + E % 2)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,top_groups,k", [(8, 4, 2, 3), (16, 8, 3, 6), (12, 3, 1, 4), (60, 6, 2, 5), (64, 64, 9, 9),
                                                   (128, 8, 4, 8), (256, 8, 4, 8), (260, 13, 5, 7), (512, 16, 4, 10),
                                                   (1024, 32, 6, 16), (30, 5, 5, 30)])
@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("with_bias", [True, False])
def test_groups_and_bias(cuda, E, groups, top_groups, k, score, group_score, with_bias):
    dtype = [BF, F4, FP][(E + groups) % 3]
    bias = seeded((E,), E, 0.2) if with_bias else None
    check_route(seeded((21, E), E + k, 1.5, dtype), k, score=score, bias=bias, groups=groups, top_groups=top_groups,
                group_score=group_score, scale=2.5)


@pytest.mark.parametrize("k,E", [(32, 40), (64, 64), (64, 300), (33, 128)])
def test_many_of_them(cuda, k, E):
    check_route(seeded((9, E), k, 1.5, BF), k)
    check_route(seeded((9, E), k, 1.5, F4), k, score="sigmoid", bias=seeded((E,), 1, 0.1), renormalize=False)


@pytest.mark.parametrize("tokens", [0, 1, 2, 3, 4, 5, 31, 32, 33, 1000])
def test_tokens(cuda, tokens):
    check_route(seeded((tokens, 10), tokens, 1.5, BF), 2)
    check_route(seeded((tokens, 70), tokens, 1.5, FP), 6, score="sigmoid")


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_equal_keys_take_the_lowest_index(cuda, score, bias):
    for E, groups in ((9, 3), (128, 8), (300, 1)):
        few = (seeded((50, E), E) * 1.5).round()  # a handful of values
        few[0] = 0.0
        few[1] = torch.where(few[1] < 0, -0.0, 0.0)  # both zeros are one value
        check_route(few, 5, score=score, bias=torch.zeros(E) if bias else None, groups=groups, top_groups=min(2, groups))
        check_route(few, 5, score=score, bias=(seeded((E,), 1).round() / 4) if bias else None, groups=groups,
                    top_groups=min(2, groups), group_score="top2")


def test_keys_a_rounding_apart(cuda):
    """Scores plus bias that are equal in 32 bits and not in 64."""
    E = 130
    logits = seeded((40, E), 3) * 1e-4
    bias = torch.full((E,), 64.0)
    check_route(logits, 8, score="sigmoid", bias=bias, renormalize=False)
    check_route(logits, 8, score="softmax", bias=bias, groups=10, top_groups=3, group_score="top2")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("dtype", [BF, FP, F4])
def test_masks_and_masked_logits(cuda, score, renormalize, dtype):
    E, k = 40, 6
    logits = seeded((30, E), 1, 1.5, dtype)
    mask = torch.rand(30, generator=torch.Generator().manual_seed(2)) < 0.6
    mask[:2] = False
    logits[0], logits[1, 3] = float("nan"), INF  # of tokens that take no part
    logits[2] = -INF                             # a token without any expert
    logits[3, 4:] = -INF                         # with fewer than it takes
    logits[4, ::2] = -INF
    mask[2:5] = True
    for bias in (None, seeded((E,), 3, 0.1)):
        for groups, top in ((1, 1), (5, 2)):
            check_route(logits, k, mask=mask, renormalize=renormalize, score=score, bias=bias, groups=groups,
                        top_groups=top, group_score="top2")
    check_route(logits, k, mask=torch.zeros(30, dtype=torch.bool), renormalize=renormalize, score=score)


def test_the_lowest_values_of_a_type_are_ordinary_logits(cuda):
    for dtype in (BF, FP, F4):
        logits = seeded((20, 24), 1, 1.0, dtype)
        logits[:, 3:] = torch.finfo(dtype).min  # three of eight are real, the rest come by index with weight 0
        check_route(logits, 8)
        check_route(logits, 8, renormalize=False)
        check_route(logits, 8, score="sigmoid")


def test_scores_far_below_one_are_renormalised(cuda):
    from stratum_amd import moe_route
    logits = torch.tensor([[-200.0, -201.0, -300.0], [-1e4, -1e4, -2e4]])
    w, e = moe_route(logits.cuda(), 2, score="sigmoid")
    ref = torch.softmax(logits.double(), 1)[:, :2]  # far below zero a sigmoid is an exponential
    ref = ref / ref.sum(1, keepdim=True)
    assert torch.equal(e.cpu(), torch.tensor([[0, 1], [0, 1]], dtype=torch.int32))
    assert_within(w, ref, 40 * U * ref, "weights")


def test_nan_and_inf_show_in_their_token_only(cuda):
    from stratum_amd import moe_route
    logits = seeded((6, 50), 1)
    clean = moe_route(logits.cuda(), 4)
    for score in ("softmax", "sigmoid"):
        for bias in (None, torch.zeros(50)):
            bad = logits.clone()
            bad[2, 30] = float("nan")
            w, e = moe_route(bad.cuda(), 4, score=score, bias=bias.cuda() if bias is not None else None)
            assert w[2].isnan().all() and (0 <= e[2]).all() and (e[2] < 50).all()
            if bias is None:
                assert e[2, 0] == 30
            if score == "softmax":
                rows = torch.tensor([0, 1, 3, 4, 5], device=cuda)
                assert torch.equal(e[rows], clean[1][rows]) and torch.equal(w[rows], clean[0][rows])
    bad = logits.clone()
    bad[2, 30] = INF
    w, e = moe_route(bad.cuda(), 4, score="sigmoid", renormalize=False)
    assert e[2, 0] == 30 and w[2, 0] == 1.0


def test_route_layouts(cuda):
    from stratum_amd import moe_route
    big = seeded((2, 5, 96), 1, 1.5, BF).cuda()
    x = big[:, :, 10:70]
    w, e = moe_route(x, 3, mask=torch.ones(2, 5, dtype=torch.bool, device=cuda))
    assert w.shape == e.shape == (2, 5, 3)
    w2, e2 = moe_route(x.contiguous().view(10, 60), 3)
    assert torch.equal(w.view(10, 3), w2) and torch.equal(e.view(10, 3), e2)
    leaf = x.detach().requires_grad_(True)
    w, _ = moe_route(leaf, 3)
    g, = torch.autograd.grad(w.sum(-1).sum(), leaf)  # an expanded gradient; the weights' sum is constant
    assert g.shape == leaf.shape and g.abs().max() < 1e-6


def test_the_routers_gradient_against_differences(cuda):
    from stratum_amd import moe_route
    for kw in ({}, {"renormalize": False}, {"score": "sigmoid"}, {"score": "sigmoid", "renormalize": False}):
        x, way, dw = seeded((5, 20), 1), seeded((5, 20), 2), seeded((5, 4), 3).cuda()
        bias = torch.zeros(20)  # the same experts at every step
        first = choose(x, 4, kw.get("score", "softmax"))
        bias = torch.full((5, 20), 0.0)
        for t in range(5):
            bias[t, first[t].long()] = 100.0

        def value(e):
            total = 0.0
            for t in range(5):  # one token at a time, so that each has its own bias
                w, c = moe_route((x[t:t + 1] + e * way[t:t + 1]).cuda(), 4, bias=bias[t].cuda(), **kw)
                order = c.long().argsort(1)
                at = first[t:t + 1].long().argsort(1)
                total += (w.gather(1, order).double() * dw[t:t + 1].gather(1, at.cuda())).sum().item()
            return total

        leaf = x.cuda().requires_grad_(True)
        w, c = moe_route(leaf, 4, **kw)
        assert torch.equal(c.cpu(), first)
        g, = torch.autograd.grad(w, leaf, dw)
        slope = (g.double().cpu() * way).sum().item()
        e = 2.0 ** -6
        short, long = ((value(s) - value(-s)) / (2 * s) for s in (e, 2 * e))
        noise = 64 * U * (w.abs() * dw.abs()).sum().item() / e
        assert abs(slope - short) <= abs(long - short) + noise


# ------------------------------------------------------------------ sort
def order_of(experts, E):
    flat = experts.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    by = torch.sort(key, stable=True).indices
    counts = torch.bincount(key, minlength=E + 1)[:E]
    offsets = torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)])
    live = int(offsets[-1])
    slots = torch.full_like(flat, -1)
    slots[:live] = by[:live]
    positions = torch.full_like(flat, -1)
    positions[by[:live]] = torch.arange(live)
    return [t.to(torch.int32) for t in (offsets, slots, positions.view(experts.shape))]


def check_sort(experts, E):
    from stratum_amd import moe_sort
    got = moe_sort(experts.cuda(), E)
    for name, a, b in zip(got._fields, got, order_of(experts, E)):
        assert a.shape == b.shape and torch.equal(a.cpu(), b), name


def drawn(n, E, seed, low=0):
    return torch.randint(low, E, (n,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)


@pytest.mark.parametrize("n", [0, 1, 2, 63, 64, 65, 127, 511, 512, 513, 1000, 2047, 2048, 2049, 3000, 4096, 5001, 65535,
                               65536, 65537, 100000])
@pytest.mark.parametrize("E", [1, 2, 3, 60, 128, 1000])
def test_sort(cuda, n, E):
    check_sort(drawn(n, E, n + E), E)


def test_sort_of_skewed_and_missing_slots(cuda):
    for n in (100, 2048, 2500, 70000):
        check_sort(torch.zeros(n, dtype=torch.int32), 7)
        check_sort(torch.full((n,), 6, dtype=torch.int32), 7)
        check_sort(torch.full((n,), -1, dtype=torch.int32), 7)
        check_sort(drawn(n, 9, n, low=-4), 7)  # -4 .. 8: both sides of the range are no expert
        wild = drawn(n, 5, n)
        wild[::3], wild[1::7] = 2 ** 31 - 1, -2 ** 31
        check_sort(wild, 5)
        check_sort((drawn(n, 1 << 20, n).double() ** 0.25).to(torch.int32), 32)


def test_sort_of_a_large_batch(cuda):
    check_sort(drawn(3_000_001, 384, 1, low=-20), 384)
    check_sort(drawn(1 << 20, 1024, 1).view(-1, 8), 1024)


def test_sort_shapes(cuda):
    check_sort(drawn(2 * 3 * 4, 5, 1).view(2, 3, 4), 5)
    check_sort(torch.empty(0, 8, dtype=torch.int32), 5)
    check_sort(torch.empty(4, 0, dtype=torch.int32), 5)
    check_sort(drawn(40, 5, 1).view(8, 5).t(), 5)


# ------------------------------------------------------------------ gather, combine
def batch(tokens, k, E, padded, seed):
    """(experts, order on the GPU, the rows by slot: -1 without)."""
    from stratum_amd import moe_sort
    g = torch.Generator().manual_seed(seed)
    experts = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(tokens)]).to(torch.int32) if tokens else \
        torch.empty(0, k, dtype=torch.int32)
    if padded:
        experts[torch.rand(tokens, generator=g) < padded] = -1
        experts[torch.rand(experts.shape, generator=g) < 0.1] = -1
    order = moe_sort(experts.cuda(), E)
    return order, order.positions.cpu().long()


def check_gather(tokens, k, hidden, dtype, padded=0.0, E=None, seed=1):
    from stratum_amd import moe_gather
    order, at = batch(tokens, k, E or max(2 * k, 4), padded, seed)
    x = seeded((tokens, hidden), seed, 1.0, dtype)
    leaf = x.cuda().requires_grad_(True)
    rows = moe_gather(leaf.detach(), order)
    want = torch.zeros(tokens * k, hidden, dtype=dtype)
    for j in range(k):
        live = at[:, j] >= 0
        want[at[live, j]] = x[live]
    assert torch.equal(rows.cpu(), want)
    g = seeded((tokens * k, hidden), seed + 1, 1.0, dtype)
    again = moe_gather(leaf, order)
    assert torch.equal(again, rows)
    dx, = torch.autograd.grad(again, leaf, g.cuda())
    picked = torch.where((at >= 0).unsqueeze(2), g.double()[at.clamp(min=0)], 0.0)
    assert_within(dx, picked.sum(1), picked.abs().sum(1) * (k + 1) * U, "dx")


def check_combine(tokens, k, hidden, dtype, padded=0.0, E=None, residual=None, seed=1, short=False):
    from stratum_amd import moe_combine
    order, at = batch(tokens, k, E or max(2 * k, 4), padded, seed)
    live = int(order.offsets[-1]) if short else tokens * k
    y = seeded((live, hidden), seed, 1.0, dtype)
    w = seeded((tokens, k), seed + 1)
    w[at < 0] = float("nan")  # the weight of a slot without a row does not matter
    r = seeded((tokens, hidden), seed + 2, 1.0, residual) if residual else None
    leaves = [t.cuda().requires_grad_(True) for t in (y, w, r) if t is not None]
    args = [leaves[0], leaves[1], order] + leaves[2:]
    out = moe_combine(*[t.detach() if torch.is_tensor(t) else t for t in args])
    assert out.dtype == (residual or dtype)
    there = at >= 0
    whole = torch.cat([y, y.new_zeros(1, hidden)]).double()
    picked = torch.where(there.unsqueeze(2), whole[at.clamp(min=0)], 0.0)
    terms = picked * torch.where(there, w.double(), 0.0).unsqueeze(2)
    ref, size = terms.sum(1), terms.abs().sum(1)
    if r is not None:
        ref, size = ref + r.double(), size + r.double().abs()
    assert_within(out, ref, size * (k + 2) * U, "out")
    again = moe_combine(*args)
    assert torch.equal(again, out)
    d = seeded((tokens, hidden), seed + 3, 1.0, out.dtype)
    grads = torch.autograd.grad(again, leaves, d.cuda())
    dy = torch.zeros(live, hidden, dtype=torch.float64)
    dy[at[there]] = (d.double().unsqueeze(1) * torch.where(there, w.double(), 0.0).unsqueeze(2))[there]
    assert grads[0].dtype == dtype and grads[1].dtype == F4
    assert_within(grads[0], dy, dy.abs() * U, "dy")
    prod = picked * d.double().unsqueeze(1)
    assert_within(grads[1], prod.sum(2), prod.abs().sum(2) * (8 * -(-hidden // 2048) + 10) * U, "dweights")
    if r is not None:
        assert torch.equal(grads[2].cpu(), d)


@pytest.mark.parametrize("dtype", [BF, FP, F4])
@pytest.mark.parametrize("hidden", [1, 7, 8, 9, 64, 255, 512, 520, 1001, 2048, 2056, 4100])
@pytest.mark.parametrize("k", [1, 2, 3, 8])
def test_gather_and_combine_widths(cuda, hidden, k, dtype):
    check_gather(19, k, hidden, dtype, seed=hidden)
    check_combine(19, k, hidden, dtype, residual=dtype if hidden % 2 else None, seed=hidden)


@pytest.mark.parametrize("k", [4, 5, 6, 7, 9, 10, 16, 17, 33, 64])
def test_gather_and_combine_slots_a_token(cuda, k):
    check_gather(11, k, 72, BF, seed=k)
    check_combine(11, k, 72, FP, residual=F4, seed=k)


@pytest.mark.parametrize("tokens", [0, 1, 2, 3, 4, 5, 700])
@pytest.mark.parametrize("padded", [0.3, 1.0])
def test_gather_and_combine_padded_batches(cuda, tokens, padded):
    for dtype, residual in ((BF, F4), (FP, FP), (F4, None)):
        check_gather(tokens, 4, 520, dtype, padded, seed=tokens)
        check_combine(tokens, 4, 520, dtype, padded, residual=residual, seed=tokens)
        check_combine(tokens, 4, 520, dtype, padded, residual=residual, seed=tokens, short=True)


def test_gather_and_combine_many_tokens(cuda):
    check_gather(3001, 8, 136, BF, 0.1, E=128)
    check_combine(3001, 8, 136, BF, 0.1, E=128, residual=BF)


def test_layouts_and_some_gradients(cuda):
    from stratum_amd import moe_combine, moe_gather
    order, at = batch(12, 3, 8, 0.0, 1)
    big = seeded((12, 200), 1, 1.0, BF).cuda()
    x = big[:, 5:105]
    assert torch.equal(moe_gather(x, order), moe_gather(x.contiguous(), order))
    assert torch.equal(moe_gather(x.contiguous().view(3, 4, 100), order), moe_gather(x.contiguous(), order))
    y, w = seeded((36, 100), 2, 1.0, BF).cuda(), seeded((12, 3), 3).cuda()
    wide = torch.zeros(36, 130, dtype=BF, device=cuda)
    wide[:, 7:107] = y
    want = moe_combine(y, w, order)
    assert torch.equal(moe_combine(wide[:, 7:107], w, order), want)
    assert torch.equal(moe_combine(y, w.t().contiguous().t(), order), want)
    both = [t.clone().requires_grad_(True) for t in (y, w)]
    d = seeded((12, 1), 4, 1.0, BF).cuda().expand(12, 100)
    dy, dw = torch.autograd.grad(moe_combine(*both, order), both, d)
    only, = torch.autograd.grad(moe_combine(both[0], w, order), both[0], d)
    assert torch.equal(only, dy)
    only, = torch.autograd.grad(moe_combine(y, both[1], order), both[1], d)
    assert torch.equal(only, dw)
    r = x.clone().requires_grad_(True)
    only, = torch.autograd.grad(moe_combine(y, w, order, r), r, d)
    assert torch.equal(only, d)
    # the result has the residual's sizes, or those of the order's slots
    assert moe_combine(y, w, order, x.contiguous().view(2, 6, 100)).shape == (2, 6, 100)


def test_rows_beyond_2_to_the_31_elements(cuda):
    from stratum_amd import moe_combine, moe_gather, moe_sort
    tokens, k, hidden = 1 << 17, 8, 2112
    experts = drawn(tokens * k, 64, 1).view(tokens, k).cuda()
    order = moe_sort(experts, 64)
    x = torch.empty(tokens, hidden, dtype=BF, device=cuda).normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    rows = moe_gather(x, order)
    for p in (0, 1 << 19, tokens * k - 5):
        assert torch.equal(rows[p:p + 5], x[(order.slots[p:p + 5] // k).long()])
    w = torch.full((tokens, k), 0.125, device=cuda)
    assert torch.equal(moe_combine(rows, w, order), x)  # eight equal parts of a row are the row
    rows.requires_grad_(True)
    dy, = torch.autograd.grad(moe_combine(rows, w, order), rows, x)
    assert torch.equal(dy[-5:], x[(order.slots[-5:] // k).long()] * 0.125)


# ------------------------------------------------------------------ a run of them
def test_streams_and_a_captured_step(cuda):
    """Norm, routing, sorting, gathering and combining with their gradients, captured once and replayed on new
    inputs between eager work; every replay equals the eager result."""
    from stratum_amd import moe_combine, moe_gather, moe_route, moe_sort, rms_norm
    tokens, hidden, E, k = 300, 264, 24, 4
    x0, r0 = seeded((tokens, hidden), 1, 1.0, BF).cuda(), seeded((tokens, hidden), 2, 1.0, BF).cuda()
    w0, router = seeded((hidden,), 3, 1.0, BF).cuda(), seeded((E, hidden), 4, 0.1, BF).cuda()
    d0 = seeded((tokens, hidden), 5, 1.0, BF).cuda()
    mask0 = torch.ones(tokens, dtype=torch.bool, device=cuda)
    statics = [t.clone() for t in (x0, r0, w0, d0, mask0)]

    def step(x, r, w, d, mask):
        leaves = [t.detach().requires_grad_(True) for t in (x, r, w)]
        y, h = rms_norm(leaves[0], leaves[2], 1e-6, leaves[1])
        weights, experts = moe_route((y @ router.t()), k, mask=mask)
        order = moe_sort(experts, E)
        out = moe_combine(moe_gather(y, order), weights, order, h)
        return [out.detach(), experts, *order, *torch.autograd.grad(out, leaves, d)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = step(*statics)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(warm, step(*statics)))
    del warm
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(*statics)
    for i in range(4):
        fresh = [seeded(t.shape, 10 + i, 1.0, t.dtype).cuda() if t.dtype == BF else
                 torch.rand(tokens, generator=torch.Generator().manual_seed(i)).cuda() < 0.2 + 0.2 * i for t in statics]
        for s, f in zip(statics, fresh):
            s.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step(*fresh)):
            assert torch.equal(a, b)
