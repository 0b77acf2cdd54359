"""CPU tests of the optimizer's refusals: what the C ABI and the Python layer turn down
before any launch."""

import ctypes

import numpy as np
import pytest
import torch


@pytest.fixture(scope="module")
def L():
    from stratum_amd import _lib
    return _lib.lib()


def table(n=16, **at):
    row = np.zeros(8, np.int64)
    buf = ctypes.create_string_buffer(256)
    base = (ctypes.addressof(buf) + 15) & ~15
    names = ("param", "grad", "master", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")
    for i, name in enumerate(names):
        row[i] = at.get(name, 0 if name == "master" else base)
    row[7] = n
    return row, base, buf


def step(L, row, *, count=1, param=2, grad=2, bits=32, betas=(0.9, 0.999), t=1):
    return L.stm_adamw_step(count, row.ctypes.data if row is not None else None, param, grad, bits, 1e-3, *betas, 1e-8,
                            0.0, t, None, None)


def test_adamw_step_refuses_what_it_cannot_run(L):
    row, base, _buf = table()
    err = lambda: L.stm_last_error().decode()  # noqa: E731
    assert step(L, None, count=1) == -1 and step(L, row, count=-1) == -1
    assert step(L, row, param=7) == -1 and step(L, row, grad=3) == -1 and "dtype" in err()
    assert step(L, row, bits=16) == -1 and "8 or 32" in err()
    assert step(L, row, t=0) == -1 and "step 1" in err()
    assert step(L, row, betas=(1.0, 0.999)) == -1 and step(L, row, betas=(0.9, float("nan"))) == -1
    assert step(L, table(-1)[0]) == -1 and "negative" in err()
    for name in ("param", "grad", "exp_avg", "exp_avg_sq"):
        assert step(L, table(**{name: 0})[0]) == -1 and "null" in err()
    for name in ("exp_avg_scale", "exp_avg_sq_scale"):
        assert step(L, table(**{name: 0})[0], bits=8) == -1 and "null" in err()
    for name in ("param", "grad", "master", "exp_avg"):
        assert step(L, table(**{name: base + 2})[0]) == -1 and "aligned" in err()
    assert step(L, table(**{"param": base + 1})[0], param=1) == -1
    # nothing to do: no launch, no error
    assert step(L, row, count=0) == 0 and step(L, table(0)[0]) == 0


def test_grad_norm_refuses_what_it_cannot_run(L):
    buf = ctypes.create_string_buffer(256)
    p = (ctypes.addressof(buf) + 15) & ~15
    one, n = np.array([p], np.int64), np.array([100], np.int64)
    assert L.stm_grad_norm_workspace_bytes(1, n.ctypes.data) == 8
    assert L.stm_grad_norm_workspace_bytes(3, np.array([0, 16384, 16385], np.int64).ctypes.data) == 24
    assert L.stm_grad_norm_workspace_bytes(1, np.array([-1], np.int64).ctypes.data) == -1

    def norm(grads=one, sizes=n, dtype=2, max_norm=1.0, loss_scale=1.0, out=p, ws=p, nbytes=8):
        return L.stm_grad_norm(len(sizes), grads.ctypes.data, sizes.ctypes.data, dtype, max_norm, loss_scale, out, ws,
                               nbytes, None)
    assert norm(dtype=5) == -1 and norm(out=None) == -1 and norm(out=p + 2) == -1
    assert norm(max_norm=-1.0) == -1 and norm(max_norm=float("nan")) == -1
    assert norm(loss_scale=0.0) == -1 and norm(loss_scale=float("inf")) == -1
    assert norm(ws=None) == -1 and norm(nbytes=7) == -1 and norm(ws=p + 4) == -1
    assert norm(grads=np.array([0], np.int64)) == -1 and norm(grads=np.array([p + 2], np.int64)) == -1


def test_state8_refuses_what_it_cannot_run(L):
    buf = ctypes.create_string_buffer(256)
    p = (ctypes.addressof(buf) + 15) & ~15
    for fn in (L.stm_state8_codes, L.stm_state8_values):
        args = (p, 16, 1, p, p) if fn is L.stm_state8_codes else (p, p, 16, 1, p)
        negative = (p, -1, 1, p, p) if fn is L.stm_state8_codes else (p, p, -1, 1, p)
        empty = (None, 0, 1, None, None) if fn is L.stm_state8_codes else (None, None, 0, 1, None)
        assert fn(*negative, None) == -1 and fn(*empty, None) == 0
        for i, a in enumerate(args):
            if a == p:
                assert fn(*args[:i], None, *args[i + 1:], None) == -1
        assert fn(*args[:-1], p + 2, None) == -1


def test_the_python_layer_refuses_cpu_tensors_and_bad_arguments():
    from stratum_amd.optim import AdamW, AdamWTensors, grad_norm, state_codes, state_values
    x = torch.zeros(8)
    for call in (lambda: grad_norm([x]), lambda: state_codes(x, signed=True), lambda: AdamWTensors([x], [x], [x]),
                 lambda: state_values(x.to(torch.uint8), x[:1], signed=True)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
    with pytest.raises(ValueError):
        grad_norm([])
    with pytest.raises(ValueError):
        grad_norm([None])
    with pytest.raises(ValueError):
        AdamWTensors([], [], [])
    p = torch.nn.Parameter(x)
    for bad in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1e-8), dict(weight_decay=-0.1),
                dict(max_grad_norm=-1.0), dict(max_grad_norm=float("nan"))):
        with pytest.raises(ValueError):
            AdamW([p], **bad)
