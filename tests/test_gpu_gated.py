"""GPU tests of the gated block on NF4 weights, forward and backward, against the
formulas in 64 bits on the oracle-dequantized weight.

Bounds, per element: the fp32 sums of K products of 16-bit values err by at most
K u sum|x w| (u = 2^-24; in practice far less), which is taken as the error of g and u; the
gate passes it on with its slope (|silu'| <= 1.1, |silu''| <= 0.5) and adds a few fp32
roundings (8 u of the result's terms, the exponential's argument another u |g| of them); one
rounding to the type is half a step of the result."""

import numpy as np
import pytest
import torch

from oracle import c_oracle as C
from oracle import nf4_oracle as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
TAG = {torch.bfloat16: O.DT_BF16, torch.float16: O.DT_F16}


def seeded(shape, seed, std, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype)


def weight(inter, K, dtype, seed=1, blocksize=64, std=0.05):
    """(packed, absmax on the GPU, the dequantized [2 I, K] weight in fp64)."""
    w = seeded((2 * inter, K), seed, std, torch.float16)
    q, a = C.quantize(w.view(torch.int16).numpy().view(np.uint16), O.DT_F16, blocksize, "argmin")
    d = C.dequantize(q, a, w.numel(), blocksize, TAG[dtype]).view(np.int16).reshape(2 * inter, K)
    return (torch.from_numpy(q).cuda(), torch.from_numpy(a).cuda(),
            torch.from_numpy(d).view(dtype).cuda().double())


def reference(x, w, dh=None):
    """h and its bound's terms, or [dg | du] and theirs, in 64 bits."""
    inter, x = w.shape[0] // 2, x.double()
    K = x.shape[1]
    g, u = x @ w[:inter].t().contiguous(), x @ w[inter:].t().contiguous()
    size = x.abs() @ w.abs().t().contiguous()
    eg, eu = K * U * size[:, :inter] + 1e-30, K * U * size[:, inter:] + 1e-30
    s = torch.sigmoid(g)
    silu, slope = g * s, s * (1 + g * (1 - s))
    rounds = (8 + g.abs()) * U
    if dh is None:
        return silu * u, 1.1 * eg * u.abs() + silu.abs() * eu + rounds * (silu * u).abs() + 1.1 * eg * eu
    dh = dh.double()
    dg, du = dh * u * slope, dh * silu
    terms = s + (silu * (1 - s)).abs()
    eg_dg = dh.abs() * (u.abs() * 0.5 * eg + slope.abs() * eu + 0.5 * eg * eu) + rounds * (dh * u).abs() * terms
    eg_du = dh.abs() * 1.1 * eg + rounds * du.abs()
    return torch.cat([dg, du], 1), torch.cat([eg_dg, eg_du], 1)


def assert_within(y, ref, err, dtype):
    assert y.shape == ref.shape and y.dtype == dtype
    off = (y.double() - ref).abs() - (HALF[dtype] * ref.abs() * (1 + 1e-6) + TINY[dtype] + err * (1 + HALF[dtype]))
    worst = off.argmax().item() if off.numel() else 0
    assert not off.numel() or off.max() <= 0, (f"row {worst // ref.shape[1]}, column {worst % ref.shape[1]}: "
                                               f"{y.reshape(-1)[worst]} for {ref.reshape(-1)[worst]}")


def check(M, inter, K, dtype, blocksize=64, seed=3):
    from stratum_amd import nf4_gated_bwd, nf4_gated_fwd
    q, a, w = weight(inter, K, dtype, seed, blocksize)
    x, dh = seeded((M, K), seed + 1, 1.0, dtype).cuda(), seeded((M, inter), seed + 2, 1.0, dtype).cuda()
    assert_within(nf4_gated_fwd(x, q, a, (2 * inter, K), blocksize), *reference(x, w), dtype)
    assert_within(nf4_gated_bwd(dh, x, q, a, (2 * inter, K), blocksize), *reference(x, w, dh), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [1, 2, 4, 5, 8, 9, 13, 16, 17, 31, 32, 33, 48, 49, 64, 65, 127, 129, 300])
def test_rows_on_a_small_weight(cuda, M, dtype):
    check(M, 1000, 320, dtype)  # ragged columns, a reduction that is no multiple of 128 or 256


@pytest.mark.parametrize("M", [1, 3, 7, 16, 33, 70, 260, 700])
@pytest.mark.parametrize("inter,K,blocksize", [(8, 64, 64), (24, 1024, 256), (128, 128, 128), (2816, 1024, 64),
                                               (5632, 2048, 64), (768, 4096, 512), (40, 4096, 4096)])
def test_widths_and_blocksizes(cuda, M, inter, K, blocksize):
    check(M, inter, K, torch.bfloat16, blocksize, seed=M)


@pytest.mark.parametrize("M", [1, 13, 333, 509, 2047, 4100])
def test_a_large_weight(cuda, M):
    check(M, 14336, 4096, torch.bfloat16 if M % 2 else torch.float16)


@pytest.mark.parametrize("M,inter,K", [(6200, 5640, 2112), (8150, 3080, 1600), (8200, 2824, 2112)])
def test_many_rows_ragged(cuda, M, inter, K):
    """Rows, columns and reductions that fill no tile of the many-rows kernel."""
    check(M, inter, K, torch.float16)


@pytest.mark.parametrize("kind", [0, 1, 2, 3])
@pytest.mark.parametrize("M", [5, 100, 257, 520])
def test_every_tile_kind(cuda, kind, M):
    from stratum_amd import _lib
    before = _lib.lib().stm_nf4_gemm_set_tile(kind)
    try:
        check(M, 712, 1088, torch.float16, 64, seed=M + kind)
    finally:
        _lib.lib().stm_nf4_gemm_set_tile(before)


def test_no_rows_and_no_columns(cuda):
    from stratum_amd import nf4_gated_bwd, nf4_gated_fwd
    q, a, _ = weight(16, 64, torch.bfloat16)
    x = torch.empty(0, 64, dtype=torch.bfloat16, device=cuda)
    assert nf4_gated_fwd(x, q, a, (32, 64)).shape == (0, 16)
    assert nf4_gated_bwd(x[:, :16], x, q, a, (32, 64)).shape == (0, 32)
    assert nf4_gated_fwd(x.reshape(0, 3, 64), q, a, (32, 64)).shape == (0, 3, 16)
    assert nf4_gated_fwd(torch.zeros(5, 64, dtype=torch.bfloat16, device=cuda), q[:0], a[:0], (0, 64)).shape == (5, 0)


def test_gates_far_from_zero_and_values_that_are_not_finite(cuda):
    """Large gates of either sign saturate; a NaN or infinite activation reaches its own row alone."""
    from stratum_amd import nf4_gated_bwd, nf4_gated_fwd
    for M in (3, 40, 300):
        q, a, w = weight(64, 128, torch.bfloat16)
        x = seeded((M, 128), 5, 40.0, torch.bfloat16).cuda()  # |g| up to a hundred
        dh = seeded((M, 64), 6, 1.0, torch.bfloat16).cuda()
        assert_within(nf4_gated_fwd(x, q, a, (128, 128)), *reference(x, w), torch.bfloat16)
        assert_within(nf4_gated_bwd(dh, x, q, a, (128, 128)), *reference(x, w, dh), torch.bfloat16)
        clean = nf4_gated_fwd(x, q, a, (128, 128)), nf4_gated_bwd(dh, x, q, a, (128, 128))
        x[1, 7], x[2, 9] = float("nan"), float("inf")
        h, dgu = nf4_gated_fwd(x, q, a, (128, 128)), nf4_gated_bwd(dh, x, q, a, (128, 128))
        others = [r for r in range(M) if r not in (1, 2)]
        assert h[1].isnan().all() and dgu[1].isnan().all() and not h[2].isfinite().all()
        assert torch.equal(h[others], clean[0][others]) and torch.equal(dgu[others], clean[1][others])


@pytest.mark.parametrize("M", [2, 20, 90, 600])
def test_gradient_of_the_input(cuda, M):
    """Autograd against the formula in 64 bits and against central differences of the
    64-bit function along a direction."""
    from stratum_amd import nf4_gated
    inter, K, dtype = 224, 192, torch.bfloat16
    q, a, w = weight(inter, K, dtype)
    x = seeded((M, K), 8, 1.0, dtype).cuda().requires_grad_(True)
    dh = seeded((M, inter), 9, 1.0, dtype).cuda()
    h = nf4_gated(x, q, a, (2 * inter, K))
    h.backward(dh)
    dgu, err = reference(x.detach(), w, dh)
    want = dgu @ w
    # dgu is rounded to the type for the product: half a step of every term, then one rounding of dx
    bound = (HALF[dtype] * dgu.abs() + err) @ w.abs() * (1 + 2 * inter * U) + 2 * inter * U * (dgu.abs() @ w.abs())
    assert ((x.grad.double() - want).abs() <= bound + HALF[dtype] * (want.abs() + bound)).all()

    def value(y):
        g, u = y @ w[:inter].t().contiguous(), y @ w[inter:].t().contiguous()
        return (g * torch.sigmoid(g) * u * dh.double()).sum()
    v = seeded((M, K), 10, 1.0).cuda().double()
    y, e = x.detach().double(), 1e-4
    slope = ((value(y + e * v) - value(y - e * v)) / (2 * e)).item()
    got = (x.grad.double() * v).sum().item()
    assert abs(got - slope) <= (bound + HALF[dtype] * want.abs()).mul(v.abs()).sum().item()


def test_other_layouts_shapes_and_outputs(cuda):
    from stratum_amd import nf4_gated, nf4_gated_bwd, nf4_gated_fwd
    q, a, _ = weight(96, 128, torch.bfloat16)
    base = seeded((2, 11, 256), 3, 1.0, torch.bfloat16).cuda()
    x, dense = base[:, :, ::2], base[:, :, ::2].contiguous()
    want = nf4_gated_fwd(dense.view(22, 128), q, a, (192, 128))
    assert torch.equal(nf4_gated_fwd(x, q, a, (192, 128)), want.view(2, 11, 96))
    shifted = torch.empty(22 * 128 + 1, dtype=torch.bfloat16, device=cuda)[1:].view(22, 128)  # 2-byte aligned
    shifted.copy_(dense.view(22, 128))
    assert torch.equal(nf4_gated_fwd(shifted, q, a, (192, 128)), want)
    out = torch.empty(22, 96, dtype=torch.bfloat16, device=cuda)
    assert nf4_gated_fwd(dense.view(22, 128), q, a, (192, 128), out=out).data_ptr() == out.data_ptr()
    assert torch.equal(out, want)
    dh = seeded((96, 22), 4, 1.0, torch.bfloat16).cuda().t()
    one = nf4_gated_bwd(dh, dense.view(22, 128), q, a, (192, 128))
    assert torch.equal(one, nf4_gated_bwd(dh.contiguous(), dense.view(22, 128), q, a, (192, 128)))
    t = dense.clone().requires_grad_(True)
    nf4_gated(t, q, a, (192, 128)).sum().backward()  # a gradient that is an expanded scalar
    u = dense.clone().requires_grad_(True)
    nf4_gated(u, q, a, (192, 128)).backward(torch.ones(2, 11, 96, dtype=torch.bfloat16, device=cuda))
    assert torch.equal(t.grad, u.grad)


def test_refusals(cuda):
    from stratum_amd import nf4_gated, nf4_gated_bwd, nf4_gated_fwd
    q, a, _ = weight(40, 128, torch.bfloat16)
    x = torch.zeros(4, 128, dtype=torch.bfloat16, device=cuda)
    dh = torch.zeros(4, 40, dtype=torch.bfloat16, device=cuda)
    for bad in (lambda: nf4_gated_fwd(x.float(), q, a, (80, 128)), lambda: nf4_gated_fwd(x[:, :64], q, a, (80, 128)),
                lambda: nf4_gated_fwd(x, q, a, (81, 128)), lambda: nf4_gated_fwd(x, q, a, (82, 128)),
                lambda: nf4_gated_fwd(x, q, a, (80, 128), blocksize=256),
                lambda: nf4_gated_fwd(x, q[:100], a, (80, 128)), lambda: nf4_gated_fwd(x, q, a[:10], (80, 128)),
                lambda: nf4_gated_fwd(x, q.cpu(), a, (80, 128)),
                lambda: nf4_gated_fwd(x, q, a, (80, 128), out=torch.empty(4, 39, dtype=x.dtype, device=cuda)),
                lambda: nf4_gated_bwd(dh[:3], x, q, a, (80, 128)), lambda: nf4_gated_bwd(dh[:, :32], x, q, a, (80, 128)),
                lambda: nf4_gated_bwd(dh.half(), x, q, a, (80, 128)), lambda: nf4_gated_bwd(dh.cpu(), x, q, a, (80, 128)),
                lambda: nf4_gated(x.clone().requires_grad_(True), q, a, (80, 128))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        nf4_gated_fwd(x.cpu(), q.cpu(), a.cpu(), (80, 128))


@pytest.mark.parametrize("M", [1, 24, 80, 300])
def test_replayed_graph_and_repeated_calls_give_the_same_bits(cuda, M):
    from stratum_amd import nf4_gated_bwd, nf4_gated_fwd
    q, a, _ = weight(320, 512, torch.bfloat16)
    x, dh = (seeded((M, n), n, 1.0, torch.bfloat16).cuda() for n in (512, 320))
    h, dgu = nf4_gated_fwd(x, q, a, (640, 512)), nf4_gated_bwd(dh, x, q, a, (640, 512))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        nf4_gated_fwd(x, q, a, (640, 512))
        nf4_gated_bwd(dh, x, q, a, (640, 512))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h2, dgu2 = nf4_gated_fwd(x, q, a, (640, 512)), nf4_gated_bwd(dh, x, q, a, (640, 512))
    for _ in range(3):
        h2.zero_()
        dgu2.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(h, h2) and torch.equal(dgu, dgu2)
        assert torch.equal(nf4_gated_fwd(x, q, a, (640, 512)), h)


def test_outputs_past_32_bit_offsets(cuda):
    """300 001 rows of 2 x 4096 columns: a backward output of 4.9 GB, whose kernel runs in
    stretches of rows; rows at the start, at each stretch's seam and at the end."""
    from stratum_amd import nf4_gated_bwd, nf4_gated_fwd
    M, inter, K, dtype = 300_001, 4096, 64, torch.bfloat16
    q, a, w = weight(inter, K, dtype)
    x = torch.randn(M, K, device=cuda, dtype=torch.float32, generator=torch.Generator("cuda").manual_seed(1)).to(dtype)
    dh = torch.ones(M, inter, device=cuda, dtype=dtype)
    rows = torch.tensor([0, 1, 255, 131_071, 262_143, 262_144, 261_887, 261_888, 300_000], device=cuda)
    h, dgu = nf4_gated_fwd(x, q, a, (2 * inter, K)), nf4_gated_bwd(dh, x, q, a, (2 * inter, K))
    assert_within(h[rows], *reference(x[rows], w), dtype)
    assert_within(dgu[rows], *reference(x[rows], w, dh[rows]), dtype)
