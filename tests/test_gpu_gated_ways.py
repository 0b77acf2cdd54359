"""GPU tests of kept sums where the keeping forward goes another way than the plain one, in
stretches of rows, and past 32-bit offsets; against the formulas in 64 bits, with the bounds of the
other tests of the block."""

import ctypes

import pytest
import torch

from test_gpu_gated import U, assert_within, reference, seeded, weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_keeping_forward_takes_no_workspace(cuda, dtype):
    """At the C entry, where the plain forward asks for the dequantized weight: NULL, and the output all the same."""
    from stratum_amd import _lib
    L = _lib.lib()
    M, inter, K = 6200, 5640, 2112
    assert L.stm_nf4_gated_workspace_bytes(M, inter, K) == -(-inter // 128) * 256 * K * 2  # the plain way is the dense one
    assert L.stm_nf4_gated_keep_workspace_bytes(M, inter, K) == 0
    q, a, w = weight(inter, K, dtype)
    x = seeded((M, K), 4, 1.0, dtype).cuda()
    h, sums = torch.empty(M, inter, dtype=dtype, device=cuda), torch.empty(M, 2 * inter, device=cuda)
    rc = L.stm_nf4_gated_fwd_keep(x.data_ptr(), q.data_ptr(), a.data_ptr(), h.data_ptr(), sums.data_ptr(), M, inter, K,
                                  64, _lib.dtype_tag(dtype), None, 0, ctypes.c_void_p(_lib.stream_handle(cuda)))
    assert rc == 0, L.stm_last_error()
    assert_within(h, *reference(x, w), dtype)


def test_the_keeping_forwards_space(cuda):
    """Nothing but h and the sums is allocated for a batch whose plain forward is dense."""
    from stratum_amd import nf4_gated_fwd_keep
    M, inter, K = 6200, 5640, 2112
    q, a, _ = weight(inter, K, torch.bfloat16)
    x = seeded((M, K), 4, 1.0, torch.bfloat16).cuda()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    h, sums = nf4_gated_fwd_keep(x, q, a, (2 * inter, K))
    assert torch.cuda.max_memory_allocated() - before <= h.numel() * 2 + sums.numel() * 4 + (4 << 20)


@pytest.mark.parametrize("M,inter,K", [(6200, 5640, 2112), (8192, 2824, 1344)])
def test_kept_sums_where_the_plain_forward_is_dense(cuda, M, inter, K):
    from stratum_amd import _lib, nf4_gated_bwd_kept, nf4_gated_fwd, nf4_gated_fwd_keep
    dtype = torch.bfloat16
    assert _lib.lib().stm_nf4_gated_workspace_bytes(M, inter, K) == -(-inter // 128) * 256 * K * 2
    q, a, w = weight(inter, K, dtype)
    x, dh = (seeded((M, n), M + n, 1.0, dtype).cuda() for n in (K, inter))
    h, sums = nf4_gated_fwd_keep(x, q, a, (2 * inter, K))
    exact, size = x.double() @ w.t().contiguous(), x.double().abs() @ w.abs().t().contiguous()
    assert ((sums.double() - exact).abs() <= K * U * size + 1e-30).all()
    del exact, size
    assert_within(h, *reference(x, w), dtype)
    assert_within(nf4_gated_fwd(x, q, a, (2 * inter, K)), *reference(x, w), dtype)
    assert_within(nf4_gated_bwd_kept(dh, sums), *reference(x, w, dh), dtype)


def test_kept_sums_past_32_bit_offsets_and_in_stretches_of_rows(cuda):
    """262 444 rows of 2 x 4096 sums (8.6 GB): the kernels run in stretches of 261 888 rows, and row
    262 144 starts at element 2^31."""
    from stratum_amd import nf4_gated_bwd_kept, nf4_gated_fwd_keep
    M, inter, K, dtype = 262_444, 4096, 1280, torch.bfloat16
    q, a, w = weight(inter, K, dtype)
    x = torch.randn(M, K, device=cuda, dtype=torch.float32, generator=torch.Generator("cuda").manual_seed(1)).to(dtype)
    dh = torch.ones(M, inter, device=cuda, dtype=dtype)
    h, sums = nf4_gated_fwd_keep(x, q, a, (2 * inter, K))
    dgu = nf4_gated_bwd_kept(dh, sums)
    rows = torch.tensor([0, 1, 255, 131_071, 261_887, 261_888, 262_143, 262_144, M - 1], device=cuda)
    exact, size = x[rows].double() @ w.t().contiguous(), x[rows].double().abs() @ w.abs().t().contiguous()
    assert ((sums[rows].double() - exact).abs() <= K * U * size + 1e-30).all()
    assert_within(h[rows], *reference(x[rows], w), dtype)
    assert_within(dgu[rows], *reference(x[rows], w, dh[rows]), dtype)


@pytest.mark.parametrize("M", [6, 300])
def test_a_backward_has_the_leading_sizes_of_x(cuda, M):
    """Whatever the gradient's are, and whether an operand has to be copied or not."""
    from stratum_amd import nf4_gated_bwd
    q, a, _ = weight(96, 128, torch.bfloat16)
    x, dh = seeded((M, 128), 1, 1.0, torch.bfloat16).cuda(), seeded((M, 96), 2, 1.0, torch.bfloat16).cuda()
    want = nf4_gated_bwd(dh, x, q, a, (192, 128))
    folded, spread = x.view(2, M // 2, 128), torch.stack([x, x], 2)[..., 0].view(2, M // 2, 128)
    assert not spread.is_contiguous()
    for y in (folded, spread):
        assert torch.equal(nf4_gated_bwd(dh, y, q, a, (192, 128)), want.view(2, M // 2, 192))
    for y in (x, spread.reshape(M, 128)):
        assert torch.equal(nf4_gated_bwd(dh.view(2, M // 2, 96), y, q, a, (192, 128)), want)
