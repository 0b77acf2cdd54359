"""GPU tests of kept sums where the keeping forward goes another way than the plain one, in
stretches of rows, and past 32-bit offsets; against the formulas in 64 bits, with the bounds of the
other tests of the block."""

import ctypes

import pytest
import torch

from test_gpu_gated import assert_within, reference, seeded, weight

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
