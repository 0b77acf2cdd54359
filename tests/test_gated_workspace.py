"""CPU tests of the space that the gated block's directions ask for."""

import pytest

from stratum_amd import _lib

WEIGHTS = [(14336, 4096), (5632, 2048), (8192, 4096), (5640, 2112), (2816, 1024), (512, 4096)]


@pytest.mark.parametrize("M", [100, 509, 2000, 4096, 8192])
@pytest.mark.parametrize("I,K", WEIGHTS)
def test_a_forward_that_keeps_its_sums_asks_for_no_dequantized_weight(M, I, K):  # noqa: E741
    """It never takes the way over a dequantized weight: fp32 parts of the sums, or nothing."""
    L = _lib.lib()
    keep, every = L.stm_nf4_gated_keep_workspace_bytes(M, I, K), L.stm_nf4_gated_workspace_bytes(M, I, K)
    assert 0 <= keep <= every
    assert keep % (M * 2 * I * 4) == 0


def test_a_training_batch_takes_no_workspace():
    L = _lib.lib()
    for M in (4096, 8192):
        assert L.stm_nf4_gated_keep_workspace_bytes(M, 14336, 4096) == 0
        assert L.stm_nf4_gated_workspace_bytes(M, 14336, 4096) == 2 * 14336 * 4096 * 2
    assert L.stm_nf4_gated_keep_workspace_bytes(-1, 64, 64) < 0 and L.stm_nf4_gated_keep_workspace_bytes(0, 64, 64) == 0
