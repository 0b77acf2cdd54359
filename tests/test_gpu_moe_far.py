"""GPU tests of the experts' rows where they pass the caches by (from 96 MiB, from 256 MiB in whole lines) and just before: all
values and gradients of gathering and combining against torch on the GPU, in 64 bits where there is a sum. Bounds
as in test_gpu_moe.py."""

import pytest
import torch

from test_gpu_moe import BF, F4, FP, HALF, TINY, U

pytestmark = pytest.mark.gpu

MIB = 1 << 20
BYTES = {BF: 2, FP: 2, F4: 4}


def drawn(shape, seed, dtype=F4):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(seed))


def assert_within(got, ref, err, what):
    """In place: ref and err are used up."""
    off = (got.double() - ref).abs_()
    off -= ref.abs_().mul_(HALF[got.dtype]).add_(TINY[got.dtype])
    off -= err.mul_(1 + HALF[got.dtype])
    assert got.shape == ref.shape and bool((off <= 0).all()), f"{what}: {float(off.nan_to_num(nan=1e30).max())}"


CASES = [(BF, 1024, 8, 96), (BF, 1024, 8, 256), (FP, 1001, 8, 96), (FP, 1001, 4, 256), (F4, 512, 4, 96), (F4, 1001, 8, 256),
         (BF, 4160, 2, 256), (F4, 130, 1, 96), (BF, 328, 10, 256)]


@pytest.mark.parametrize("side", [-1, 1])
@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("dtype,hidden,k,limit", CASES)
def test_rows_next_to_a_limit(cuda, dtype, hidden, k, limit, padded, side):
    from stratum_amd import moe_combine, moe_gather, moe_sort
    tokens = limit * MIB // (BYTES[dtype] * hidden * k) + side
    tokens += tokens * k * hidden * BYTES[dtype] < limit * MIB if side > 0 else 0
    assert (tokens * k * hidden * BYTES[dtype] >= limit * MIB) == (side > 0)
    g = torch.Generator(device="cuda").manual_seed(tokens)
    experts = torch.rand(tokens, 24, device=cuda, generator=g).topk(k, 1).indices.to(torch.int32)
    if padded:
        experts[torch.rand(tokens, device=cuda, generator=g) < 0.2] = -1
        experts[torch.rand(experts.shape, device=cuda, generator=g) < 0.05] = -1
    order = moe_sort(experts, 24)
    at = order.positions.long()
    live = at >= 0
    assert bool(live.all()) != padded

    x = drawn((tokens, hidden), 1, dtype).requires_grad_(True)
    rows = moe_gather(x, order)
    there = order.slots >= 0
    token = order.slots.long().clamp(min=0) // k
    assert torch.equal(rows.detach(), torch.where(there.unsqueeze(1), x.detach()[token], 0.0))
    y = drawn((tokens * k, hidden), 2, dtype)
    dx, = torch.autograd.grad(rows, x, y)
    del rows
    ref, size = (torch.zeros(tokens, hidden, dtype=torch.float64, device=cuda) for _ in range(2))
    for j in range(k):
        part = torch.where(live[:, j:j + 1], y[at[:, j].clamp(min=0)], 0.0).double()
        ref += part
        size += part.abs_()
    assert_within(dx, ref, size.mul_((k + 1) * U), "dx")
    del dx, ref, size

    residual = drawn((tokens, hidden), 3, F4 if padded else dtype)
    w = drawn((tokens, k), 4)
    w = torch.where(live, w, float("nan")).requires_grad_(True)
    y.requires_grad_(True)
    out = moe_combine(y, w, order, residual)
    d = drawn((tokens, hidden), 5, out.dtype)
    dy, dw = torch.autograd.grad(out, (y, w), d)
    values, weights = y.detach(), torch.where(live, w.detach(), 0.0).double()
    ref = residual.double()
    size = ref.abs()
    dot, dots = torch.empty(tokens, k, dtype=torch.float64, device=cuda), torch.empty(tokens, k, dtype=torch.float64, device=cuda)
    for j in range(k):
        part = torch.where(live[:, j:j + 1], values[at[:, j].clamp(min=0)], 0.0).double()
        dot[:, j], dots[:, j] = (part * d).sum(1), (part * d).abs_().sum(1)
        part *= weights[:, j:j + 1]
        ref += part
        size += part.abs_()
    assert_within(out.detach(), ref, size.mul_((k + 2) * U), "out")
    assert_within(dw, dot, dots.mul_((8 * -(-hidden // 2048) + 10) * U), "dweights")
    del ref, size, out
    want = d.double()[token] * torch.where(there, weights.view(-1)[order.slots.long().clamp(min=0)], 0.0).unsqueeze(1)
    assert_within(dy, want, want.abs().mul_(U), "dy")
