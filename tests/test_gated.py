"""CPU tests of the gated block's refusals: what the C ABI, the Python layer and the MLP
module turn down before any launch."""

import ctypes

import pytest
import torch
import torch.nn as nn

from stratum_amd import NF4Linear, QuantState, nf4_gated, nf4_gated_bwd, nf4_gated_fwd
from stratum_amd.mlp import NF4GatedMLP


@pytest.fixture(scope="module")
def L():
    from stratum_amd import _lib
    return _lib.lib()


BUF = ctypes.create_string_buffer(256)
BASE = (ctypes.addressof(BUF) + 15) & ~15


def fwd(L, *, x=BASE, q=BASE, a=BASE, h=BASE, M=1, I=64, K=128, bs=64, dtype=1, ws=BASE, bytes=None):  # noqa: E741
    bytes = L.stm_nf4_gated_workspace_bytes(M, I, K) if bytes is None else bytes
    return L.stm_nf4_gated_fwd(x, q, a, h, M, I, K, bs, dtype, ws, bytes, None)


def bwd(L, dh=BASE, x=BASE, M=1, I=64, K=128, bytes=1 << 20):  # noqa: E741
    return L.stm_nf4_gated_bwd(dh, x, BASE, BASE, BASE, M, I, K, 64, 1, BASE, bytes, None)


def test_c_abi_refuses_what_the_kernels_cannot_take(L):
    err = lambda: L.stm_last_error().decode()  # noqa: E731
    for name in ("x", "q", "a", "h"):
        assert fwd(L, **{name: None}) < 0 and err()
    for name in ("x", "q", "h"):
        assert fwd(L, **{name: BASE + 2}) < 0 and "aligned" in err()
    for sizes in (dict(M=-1, bytes=0), dict(I=-8, bytes=0), dict(K=-64, bytes=0), dict(I=68), dict(K=96), dict(K=0),
                  dict(K=64, bs=128), dict(bs=96), dict(bs=32), dict(dtype=2), dict(dtype=7),
                  dict(I=1 << 21, K=1 << 22, bytes=0), dict(I=1 << 22, bytes=0), dict(K=1 << 23, bytes=0),
                  dict(I=1 << 60, K=1 << 60, bytes=0)):
        assert fwd(L, **sizes) < 0 and err(), sizes
    assert bwd(L, dh=None) < 0 and "gradient" in err()
    assert bwd(L, dh=BASE + 8) < 0 and "gradient" in err()
    # nothing to do: no launch, no error, whatever the pointers
    assert fwd(L, x=None, q=None, a=None, h=None, M=0) == 0 and fwd(L, q=None, a=None, h=None, I=0) == 0
    assert bwd(L, dh=None, x=None, M=0) == 0


def test_c_abi_refuses_a_workspace_that_is_too_small(L):
    M, I, K = 8192, 5632, 2048  # noqa: E741
    need = L.stm_nf4_gated_workspace_bytes(M, I, K)
    assert need > 0
    assert fwd(L, M=M, I=I, K=K, bytes=need - 1) < 0 and "workspace" in L.stm_last_error().decode()
    assert fwd(L, M=M, I=I, K=K, ws=None) < 0 and "workspace" in L.stm_last_error().decode()
    assert L.stm_nf4_gated_workspace_bytes(-1, I, K) < 0
    assert L.stm_nf4_gated_workspace_bytes(0, I, K) == 0


@pytest.mark.parametrize("M", [1, 2, 16, 17, 64, 65, 300, 1000, 5000, 70000, 1 << 20])
@pytest.mark.parametrize("I,K", [(8, 64), (768, 2048), (5632, 2048), (14336, 4096)])
def test_workspace_stays_within_a_bound(L, M, I, K):  # noqa: E741
    """At most fp32 partial sums of 32 parts for up to 4096 rows, or the 16-bit weight in
    256-row tiles."""
    most = max(32 * min(M, 4096) * 2 * I * 4, (I + 127) // 128 * 256 * K * 2)
    assert 0 <= L.stm_nf4_gated_workspace_bytes(M, I, K) <= most


def test_the_python_layer_refuses_cpu_tensors():
    q, a = torch.zeros(64 * 128, dtype=torch.uint8), torch.ones(256)
    x, dh = torch.zeros(3, 128, dtype=torch.bfloat16), torch.zeros(3, 64, dtype=torch.bfloat16)
    for call in (lambda: nf4_gated_fwd(x, q, a, (128, 128)), lambda: nf4_gated_bwd(dh, x, q, a, (128, 128)),
                 lambda: nf4_gated(x, q, a, (128, 128))):
        with pytest.raises(RuntimeError):
            call()


def projection(out_features, in_features, bias=None, blocksize=64):
    n = out_features * in_features
    state = QuantState(absmax=torch.ones(n // blocksize), shape=(out_features, in_features), blocksize=blocksize,
                       dtype=torch.bfloat16)
    return NF4Linear(torch.zeros(n // 2, 1, dtype=torch.uint8), state, bias)


class MLP(nn.Module):
    def __init__(self, gate, up, down, act=None):
        super().__init__()
        self.gate_proj, self.up_proj, self.down_proj, self.act_fn = gate, up, down, act or nn.SiLU()


def test_module_refuses_what_the_block_does_not_compute():
    down = nn.Linear(64, 128, bias=False)
    good = NF4GatedMLP(MLP(projection(64, 128), projection(64, 128), down))
    assert good.shape == (128, 128) and good.down is down
    with pytest.raises(TypeError):
        NF4GatedMLP(MLP(nn.Linear(128, 64, bias=False), projection(64, 128), down))
    with pytest.raises(TypeError):
        NF4GatedMLP(MLP(projection(64, 128), projection(64, 128, torch.zeros(64)), down))
    with pytest.raises(TypeError):
        NF4GatedMLP(MLP(projection(64, 128), projection(64, 128), down, nn.GELU()))
    with pytest.raises(ValueError):
        NF4GatedMLP(MLP(projection(64, 128), projection(96, 128), down))
    with pytest.raises(ValueError):
        NF4GatedMLP(MLP(projection(64, 128), projection(64, 128, blocksize=128), down))
    with pytest.raises(ValueError):  # the input gradient takes 32 columns at a time
        NF4GatedMLP(MLP(projection(40, 128), projection(40, 128), down))


def test_module_takes_adjacent_payloads_as_they_are_and_keeps_fp32_scales():
    both, scales = torch.zeros(2 * 64 * 64, 1, dtype=torch.uint8), torch.rand(2 * 128)
    halves = [QuantState(absmax=scales[i * 128:(i + 1) * 128], shape=(64, 128), blocksize=64, dtype=torch.bfloat16)
              for i in range(2)]
    gate, up = (NF4Linear(both[i * 4096:(i + 1) * 4096], s) for i, s in enumerate(halves))
    mlp = NF4GatedMLP(MLP(gate, up, nn.Linear(64, 128, bias=False)))
    assert mlp.gate_up_packed.data_ptr() == both.data_ptr() and mlp.gate_up_absmax.data_ptr() == scales.data_ptr()
    mlp.half()
    assert mlp.gate_up_absmax.dtype == torch.float32 and torch.equal(mlp.gate_up_absmax, scales)
    apart = NF4GatedMLP(MLP(projection(64, 128), projection(64, 128), nn.Linear(64, 128, bias=False)))
    assert apart.gate_up_packed.numel() == 64 * 128 and apart.gate_up_absmax.numel() == 256


def test_c_abi_of_the_kept_sums(L):
    err = lambda: L.stm_last_error().decode()  # noqa: E731

    def keep(sums=BASE, M=100, I=64, K=128):  # noqa: E741
        return L.stm_nf4_gated_fwd_keep(BASE, BASE, BASE, BASE, sums, M, I, K, 64, 1, BASE, 1 << 30, None)

    def kept(dh=BASE, sums=BASE, out=BASE, M=100, I=64, dtype=1):  # noqa: E741
        return L.stm_gated_bwd_kept(dh, sums, out, M, I, dtype, None)
    assert keep(sums=None) < 0 and "sums" in err()
    assert keep(sums=BASE + 4) < 0 and "sums" in err()
    assert keep(M=64) < 0 and "rows" in err()
    assert keep(M=0) == 0
    for bad in (dict(dh=None), dict(sums=None), dict(out=None), dict(dh=BASE + 2), dict(sums=BASE + 4),
                dict(out=BASE + 8), dict(I=12), dict(M=-1), dict(I=-8), dict(dtype=2)):
        assert kept(**bad) < 0 and err(), bad
    assert kept(M=0, dh=None, sums=None, out=None) == 0 and kept(I=0, dh=None) == 0
    assert L.stm_nf4_gated_sums_bytes(64, 64, 128) == 0 and L.stm_nf4_gated_sums_bytes(-1, 64, 128) < 0
    assert L.stm_nf4_gated_sums_bytes(100, 64, 128) == 100 * 2 * 64 * 4
    # a short reduction whose sums outgrow the cache is computed again
    assert L.stm_nf4_gated_sums_bytes(8192, 5632, 512) == 0 and L.stm_nf4_gated_sums_bytes(8192, 5632, 2048) > 0
