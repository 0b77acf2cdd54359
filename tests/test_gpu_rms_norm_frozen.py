"""GPU tests of the norm's gradients where the weight does not train: they are the same, bit for bit, as where it does,
and as exact (the bounds of test_gpu_rms_norm.py for a sum that is not rounded before its gradient)."""

import pytest
import torch

from test_gpu_rms_norm import BF, F4, FP, assert_within, reference, seeded

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(1, 96), (101, 384), (2000, 64), (300, 1000), (257, 4100), (70, 9000), (3, 40000)])
@pytest.mark.parametrize("dtype,residual,weight", [(BF, BF, BF), (BF, BF, F4), (FP, FP, FP), (BF, F4, BF), (FP, None, FP),
                                                   (F4, F4, F4)])
def test_a_frozen_weight_changes_no_gradient(cuda, shape, dtype, residual, weight):
    from stratum_amd import rms_norm
    x, w = seeded(shape, 1, 1.0, dtype), (1 + seeded(shape[-1:], 3, 0.3)).to(weight)
    r = seeded(shape, 2, 2.0, residual) if residual else None
    dy = seeded(shape, 4, 1.0, dtype)
    dh = seeded(shape, 5, 1.0, residual) if residual else None
    ref = reference(x, w, 1e-6, r, dy, dh, F4)
    grads = {}
    for train in (True, False):
        leaves = [t.clone().requires_grad_(True) for t in (x, r) if t is not None]
        out = rms_norm(leaves[0], w.clone().requires_grad_(train), 1e-6, leaves[1] if residual else None)
        grads[train] = torch.autograd.grad(out, leaves, (dy, dh) if residual else dy)
    for name, trained, frozen in zip(("dx", "dr"), grads[True], grads[False]):
        assert_within(frozen, *ref[name], name)
        assert torch.equal(trained, frozen), name
