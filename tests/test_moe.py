"""CPU tests of the norm's and the sparse layer's operators: what the C ABI and the Python layer turn down
before any launch, and the sizes of their workspaces."""

import ctypes

import pytest
import torch

from stratum_amd import MoEOrder, NF4MoE, QuantState, RMSNorm, moe_combine, moe_gather, moe_route, moe_sort, rms_norm


@pytest.fixture(scope="module")
def L():
    from stratum_amd import _lib
    return _lib.lib()


BUF = ctypes.create_string_buffer(256)
BASE = (ctypes.addressof(BUF) + 15) & ~15


def norm_fwd(L, x=BASE, r=None, rt=1, w=BASE, wt=1, y=BASE, h=None, rstd=None, rows=1, cols=64, eps=1e-6, dtype=1):
    return L.stm_rms_norm_fwd(x, r, rt, w, wt, y, h, rstd, rows, cols, eps, dtype, None)


def norm_bwd(L, dy=BASE, dh=None, h=BASE, ht=1, rstd=BASE, w=BASE, wt=1, dx=BASE, dr=None, dw=None, rows=1, cols=64, dtype=1,
             ws=None, bytes=0, r=None):
    return L.stm_rms_norm_bwd(dy, dh, h, r, ht, rstd, w, wt, dx, dr, dw, rows, cols, dtype, ws, bytes, None)


def test_the_norms_c_abi_refuses(L):
    err = lambda: L.stm_last_error().decode()  # noqa: E731
    for bad in (dict(x=None), dict(w=None), dict(y=None), dict(r=BASE), dict(h=BASE), dict(rows=-1), dict(cols=-1),
                dict(dtype=3), dict(dtype=-1), dict(wt=0), dict(dtype=2, wt=1), dict(r=BASE, h=BASE, rt=0),
                dict(eps=-1.0), dict(eps=float("nan")), dict(x=BASE + 1), dict(rstd=BASE + 2), dict(wt=2, w=BASE + 2),
                dict(rows=1 << 31), dict(cols=1 << 30), dict(r=BASE, h=BASE + 2, rt=2)):
        assert norm_fwd(L, **bad) < 0 and "rms_norm" in err(), bad
    for bad in (dict(dy=None), dict(h=None), dict(rstd=None), dict(w=None), dict(ht=0), dict(wt=0), dict(rows=-1),
                dict(dtype=9), dict(dw=BASE), dict(dw=BASE, ws=BASE, bytes=255), dict(r=BASE, ht=2), dict(r=BASE + 1), dict(dh=BASE + 1), dict(dw=BASE + 1)):
        assert norm_bwd(L, **bad) < 0 and "rms_norm" in err(), bad
    # nothing to do
    assert norm_fwd(L, x=None, w=None, y=None, rows=0) == 0 and norm_fwd(L, x=None, w=None, y=None, cols=0) == 0
    assert norm_bwd(L, dy=None, h=None, rstd=None, w=None, dx=None, rows=0) == 0
    assert norm_bwd(L, dx=None) == 0


@pytest.mark.parametrize("rows", [0, 1, 3, 511, 513, 2047, 2048, 8192, 1 << 20])
@pytest.mark.parametrize("cols", [1, 64, 65, 512, 513, 4096, 4097, 8192, 32768, 32769, 100000])
def test_the_norms_workspace_stays_within_a_bound(L, rows, cols):
    """One row of fp32 sums a work-group, of which there are at most 1024, and at most one a row."""
    assert 0 <= L.stm_rms_norm_workspace_bytes(rows, cols) <= min(rows, 1024) * cols * 4
    assert L.stm_rms_norm_workspace_bytes(-1, cols) < 0


def route(L, logits=BASE, bias=None, mask=None, w=BASE, e=BASE, T=1, E=16, k=2, score=0, groups=1, top=1, sums=0, dtype=1):
    return L.stm_moe_route(logits, bias, mask, w, e, T, E, k, score, groups, top, sums, 1, 1.0, dtype, None)


def test_the_routers_c_abi_refuses(L):
    err = lambda: L.stm_last_error().decode()  # noqa: E731
    for bad in (dict(logits=None), dict(w=None), dict(e=None), dict(T=-1), dict(E=0), dict(E=1025), dict(k=0), dict(k=17),
                dict(E=128, k=65), dict(score=2), dict(score=-1), dict(groups=0), dict(groups=3), dict(E=130, groups=65),
                dict(groups=4, top=0), dict(groups=4, top=5), dict(groups=8, top=1, k=3), dict(dtype=4), dict(T=1 << 31),
                dict(logits=BASE + 1), dict(bias=BASE + 2), dict(w=BASE + 1), dict(e=BASE + 3)):
        assert route(L, **bad) < 0 and "moe_route" in err(), bad
    assert route(L, logits=None, w=None, e=None, T=0) == 0
    bwd = lambda dw=BASE, x=BASE, e=BASE, dx=BASE, T=1, E=16, k=2, score=0, dtype=1: \
        L.stm_moe_route_bwd(dw, x, e, dx, T, E, k, score, 1, 1.0, dtype, None)  # noqa: E731
    for bad in (dict(dw=None), dict(x=None), dict(e=None), dict(dx=None), dict(T=-1), dict(k=0), dict(E=2000), dict(score=5),
                dict(dtype=7), dict(dx=BASE + 1)):
        assert bwd(**bad) < 0 and "moe_route" in err(), bad
    assert bwd(dw=None, T=0) == 0


def test_the_sorts_c_abi_refuses(L):
    call = lambda e=BASE, n=4, E=8, o=BASE, s=BASE, p=BASE, ws=None, bytes=0: \
        L.stm_moe_sort(e, n, E, o, s, p, ws, bytes, None)  # noqa: E731
    for bad in (dict(e=None), dict(o=None), dict(s=None), dict(p=None), dict(n=-1), dict(n=1 << 31), dict(E=0), dict(E=1025),
                dict(o=BASE + 2), dict(n=1 << 20)):
        assert call(**bad) < 0 and "moe_sort" in L.stm_last_error().decode(), bad
    assert call(n=1 << 20, ws=BASE, bytes=L.stm_moe_sort_workspace_bytes(1 << 20, 8) - 1) < 0


@pytest.mark.parametrize("n", [0, 1, 64, 2048, 2049, 65536, 65537, 1 << 20, (1 << 31) - 1])
def test_the_sorts_workspace_stays_within_a_bound(L, n):
    for E in (1, 8, 128, 1024):
        assert 0 <= L.stm_moe_sort_workspace_bytes(n, E) <= 64 * E * 4
    assert L.stm_moe_sort_workspace_bytes(64, 8) == 0
    assert L.stm_moe_sort_workspace_bytes(-1, 8) < 0 and L.stm_moe_sort_workspace_bytes(n, 0) < 0


def test_the_rows_c_abi_refuses(L):
    err = lambda: L.stm_last_error().decode()  # noqa: E731
    gather = lambda x=BASE, p=BASE, o=BASE, E=4, out=BASE, T=1, k=2, H=8, dtype=1: \
        L.stm_moe_gather(x, p, o, E, out, T, k, H, dtype, None)  # noqa: E731
    for bad in (dict(x=None), dict(p=None), dict(o=None), dict(out=None), dict(E=0), dict(T=-1), dict(k=-1), dict(H=-1),
                dict(dtype=5), dict(T=1 << 30), dict(H=1 << 28), dict(x=BASE + 1), dict(out=BASE + 1)):
        assert gather(**bad) < 0 and "moe_gather" in err(), bad
    assert gather(x=None, p=None, o=None, out=None, T=0) == 0 and gather(x=None, H=0) == 0
    combine = lambda y=BASE, rows=2, w=BASE, p=BASE, r=None, out=BASE, ot=1, T=1, k=2, H=8, dtype=1: \
        L.stm_moe_combine(y, rows, w, p, r, out, ot, T, k, H, dtype, None)  # noqa: E731
    for bad in (dict(y=None), dict(rows=3), dict(rows=-1), dict(p=None), dict(out=None), dict(T=-1), dict(H=-1), dict(ot=0),
                dict(dtype=5), dict(out=BASE + 1), dict(r=BASE + 1), dict(ot=2, out=BASE + 2)):
        assert combine(**bad) < 0 and "moe_combine" in err(), bad
    assert combine(y=None, out=None, T=0, rows=0) == 0
    bwd = lambda d=BASE, dt=1, y=BASE, rows=2, w=BASE, p=BASE, o=BASE, E=4, dy=BASE, dw=BASE, T=1, k=2, H=8, dtype=1: \
        L.stm_moe_combine_bwd(d, dt, y, rows, w, p, o, E, dy, dw, T, k, H, dtype, None)  # noqa: E731
    for bad in (dict(d=None), dict(y=None), dict(w=None), dict(p=None), dict(o=None), dict(E=0), dict(rows=3), dict(dt=0),
                dict(dtype=8), dict(dw=BASE + 2), dict(d=BASE + 1)):
        assert bwd(**bad) < 0 and "moe_combine" in err(), bad
    assert bwd(dy=None, dw=None, d=None) == 0 and bwd(T=0, d=None, rows=0) == 0
    assert bwd(H=0, dw=None, d=None, y=None, w=None, o=None) == 0 and bwd(rows=0, dw=None, d=BASE, y=None, w=None, o=None) == 0


def order(tokens=4, k=2, E=8):
    return MoEOrder(torch.zeros(E + 1, dtype=torch.int32), torch.zeros(tokens * k, dtype=torch.int32),
                    torch.zeros(tokens, k, dtype=torch.int32))


def test_the_python_layer_refuses_cpu_tensors():
    x, w = torch.zeros(4, 16, dtype=torch.bfloat16), torch.ones(16)
    for call in (lambda: rms_norm(x, w), lambda: rms_norm(x, w, 1e-6, x), lambda: RMSNorm(16)(x),
                 lambda: rms_norm(x.clone().requires_grad_(True), w),
                 lambda: moe_route(x, 2), lambda: moe_route(x.float().requires_grad_(True), 2),
                 lambda: moe_sort(torch.zeros(4, 2, dtype=torch.int32), 8), lambda: moe_gather(x, order()),
                 lambda: moe_combine(torch.zeros(8, 16), torch.zeros(4, 2), order())):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_route_refuses_unknown_names():
    x = torch.zeros(4, 16)
    for kw in ({"score": "relu"}, {"group_score": "mean"}):
        with pytest.raises(ValueError, match="must be one of"):
            moe_route(x, 2, **kw)


def bank(*shape, blocksize=64):
    n = 1
    for d in shape:
        n *= d
    state = QuantState(absmax=torch.ones(n // blocksize), shape=shape, blocksize=blocksize, dtype=torch.bfloat16)
    return torch.zeros(n // 2, 1, dtype=torch.uint8), state


def test_the_layer_refuses_banks_that_do_not_fit():
    router = torch.nn.Linear(128, 4, bias=False)
    layer = NF4MoE(router, bank(4, 128, 128), bank(4, 128, 64), 2)
    assert (layer.num_experts, layer.hidden, layer.inter) == (4, 128, 64) and "top 2" in repr(layer)
    for gate_up, down in ((bank(512, 128), bank(4, 128, 64)), (bank(4, 128, 128), bank(4, 64, 128)),
                          (bank(4, 128, 128), bank(2, 128, 64)), (bank(4, 128, 128), bank(4, 128, 64, blocksize=128)),
                          (bank(4, 96, 128), bank(4, 128, 48))):
        with pytest.raises(ValueError):
            NF4MoE(router, gate_up, down, 2)
