"""GPU tests of the gated block's forward that keeps its sums and of the backward from them,
against the formulas in 64 bits on the oracle-dequantized weight.

Bounds: the sums of K products of 16-bit values err by at most K u sum|x w| (u = 2^-24); the
backward from kept sums is held to the bound of the one that computes them again."""

import pytest
import torch

from test_gpu_gated import U, assert_within, reference, seeded, weight

pytestmark = pytest.mark.gpu


def check(M, inter, K, dtype):
    from stratum_amd import nf4_gated_bwd_kept, nf4_gated_fwd, nf4_gated_fwd_keep
    q, a, w = weight(inter, K, dtype)
    x, dh = (seeded((M, n), M + n, 1.0, dtype).cuda() for n in (K, inter))
    h, sums = nf4_gated_fwd_keep(x, q, a, (2 * inter, K))
    assert torch.equal(h, nf4_gated_fwd(x, q, a, (2 * inter, K)))
    if M <= 64:
        assert sums is None
        return
    exact, size = x.double() @ w.t().contiguous(), x.double().abs() @ w.abs().t().contiguous()
    assert sums.shape == (M, 2 * inter) and sums.dtype == torch.float32
    assert ((sums.double() - exact).abs() <= K * U * size + 1e-30).all()
    assert_within(nf4_gated_bwd_kept(dh, sums), *reference(x, w, dh), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,inter,K", [(1, 96, 128), (64, 96, 128), (65, 96, 128), (130, 40, 192), (333, 200, 1024),
                                       (509, 1416, 64), (1000, 264, 576)])
def test_kept_sums(cuda, M, inter, K, dtype):
    check(M, inter, K, dtype)


@pytest.mark.parametrize("kind", [0, 1, 2, 3])
def test_every_tile_kind(cuda, kind):
    from stratum_amd import _lib
    try:
        _lib.lib().stm_nf4_gemm_set_tile(kind)
        check(300, 328, 1024, torch.bfloat16)
    finally:
        _lib.lib().stm_nf4_gemm_set_tile(-1)


def test_many_rows_from_the_dense_weight(cuda):
    check(2500, 5640, 1024, torch.bfloat16)


def test_both_ways_give_the_gradient(cuda):
    """dx = dgu W in 64 bits of the returned dgu's inputs: each way within 3 roundings of the type."""
    from stratum_amd import nf4_gated
    q, a, w = weight(320, 512, torch.bfloat16)
    x = seeded((200, 512), 1, 1.0, torch.bfloat16).cuda()
    dh = seeded((200, 320), 2, 1.0, torch.bfloat16).cuda()
    dgu, _ = reference(x, w, dh)
    exact = dgu @ w
    for recompute in (False, True):
        t = x.clone().requires_grad_(True)
        nf4_gated(t, q, a, (640, 512), recompute=recompute).backward(dh)
        assert ((t.grad.double() - exact).norm() / exact.norm()).item() <= 3 * 2.0 ** -9


def test_what_is_kept(cuda):
    from stratum_amd import nf4_gated
    q, a, _ = weight(320, 512, torch.bfloat16)
    x = seeded((200, 512), 1, 1.0, torch.bfloat16).cuda().requires_grad_(True)
    sizes = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: sizes.append((t.dtype, tuple(t.shape))) or t, lambda t: t):
        nf4_gated(x, q, a, (640, 512))
        assert (torch.float32, (200, 640)) in sizes and (torch.bfloat16, (200, 512)) not in sizes
        sizes.clear()
        nf4_gated(x, q, a, (640, 512), recompute=True)
        assert (torch.float32, (200, 640)) not in sizes and (torch.bfloat16, (200, 512)) in sizes


def test_refusals(cuda):
    from stratum_amd import nf4_gated_bwd_kept, nf4_gated_fwd_keep
    q, a, _ = weight(40, 128, torch.bfloat16)
    x, dh = (seeded((70, n), n, 1.0, torch.bfloat16).cuda() for n in (128, 40))
    _, sums = nf4_gated_fwd_keep(x, q, a, (80, 128))
    for bad in (lambda: nf4_gated_fwd_keep(x.float(), q, a, (80, 128)), lambda: nf4_gated_fwd_keep(x, q, a, (82, 128)),
                lambda: nf4_gated_fwd_keep(x, q[:64], a, (80, 128)), lambda: nf4_gated_bwd_kept(dh[:69], sums),
                lambda: nf4_gated_bwd_kept(dh, sums.double()), lambda: nf4_gated_bwd_kept(dh, sums.t()),
                lambda: nf4_gated_bwd_kept(dh.float(), sums), lambda: nf4_gated_bwd_kept(dh.cpu(), sums),
                lambda: nf4_gated_bwd_kept(dh, sums[:, :72].contiguous())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        nf4_gated_bwd_kept(dh.cpu(), sums.cpu())


def test_replayed_graph(cuda):
    from stratum_amd import nf4_gated_bwd_kept, nf4_gated_fwd_keep
    q, a, _ = weight(320, 512, torch.bfloat16)
    x, dh = (seeded((300, n), n, 1.0, torch.bfloat16).cuda() for n in (512, 320))

    def run():
        h, sums = nf4_gated_fwd_keep(x, q, a, (640, 512))
        return h, nf4_gated_bwd_kept(dh, sums)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, dgu = run()
    for _ in range(3):
        expected = run()
        h.zero_()
        dgu.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(h, expected[0]) and torch.equal(dgu, expected[1])
        x.mul_(-0.9)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,inter,K", [(65, 8200, 128), (128, 8200, 256), (150, 8200, 256), (192, 8200, 384), (257, 1000, 1024),
                                       (380, 4104, 2048)])
def test_reductions_that_two_pairs_of_waves_share(cuda, M, inter, K, dtype):
    from stratum_amd import nf4_gated_bwd
    check(M, inter, K, dtype)
    q, a, w = weight(inter, K, dtype)
    x, dh = (seeded((M, n), M + n, 1.0, dtype).cuda() for n in (K, inter))
    assert_within(nf4_gated_bwd(dh, x, q, a, (2 * inter, K)), *reference(x, w, dh), dtype)


@pytest.mark.parametrize("recompute", [False, True])
def test_gradients_of_other_layouts(cuda, recompute):
    """An expanded, a transposed and a sliced gradient, and x with leading sizes, as their copies."""
    from stratum_amd import nf4_gated
    q, a, _ = weight(96, 128, torch.bfloat16)
    x = seeded((5, 20, 128), 3, 1.0, torch.bfloat16).cuda()
    wide = seeded((5, 20, 192), 4, 1.0, torch.bfloat16).cuda()
    for grad in (torch.ones(1, 1, 1, dtype=x.dtype, device=cuda).expand(5, 20, 96), wide[..., 1:97],
                 wide.permute(2, 0, 1)[:96].permute(1, 2, 0)):
        got = []
        for g in (grad, grad.clone(memory_format=torch.contiguous_format)):
            t = x.clone().requires_grad_(True)
            nf4_gated(t, q, a, (192, 128), recompute=recompute).backward(g)
            got.append(t.grad)
        assert got[0].shape == x.shape and torch.equal(got[0], got[1])


def test_kept_sums_on_another_stream(cuda):
    """Forward and backward on a side stream while the default stream is busy."""
    from stratum_amd import nf4_gated
    q, a, _ = weight(320, 512, torch.bfloat16)
    x = seeded((300, 512), 5, 1.0, torch.bfloat16).cuda()
    dh = seeded((300, 320), 6, 1.0, torch.bfloat16).cuda()

    def step():
        t = x.clone().requires_grad_(True)
        nf4_gated(t, q, a, (640, 512)).backward(dh)
        return t.grad
    expected = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    busy = torch.randn(4096, 4096, device=cuda)
    for _ in range(4):
        busy = busy @ busy * 1e-4
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert torch.equal(got, expected)
