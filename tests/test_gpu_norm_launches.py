"""GPU tests of the gradient norm over more tensors than a launch takes (254), and over more partial
sums (one per 16384 elements) than one pass of the final sum takes (8 x 1024).

Every tensor has a magnitude of its own, so that one lost, doubled or read from its neighbour's place
changes the norm by more than the bound: each holds at least 1/2400 of the sum of squares, 2e-4 of the norm, against two
roundings to fp32, 1.2e-7."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def check(gs):
    from stratum_amd.optim import grad_norm
    want = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
    norm, factor = grad_norm(gs, 0.5).tolist()
    assert abs(norm - want) <= 2 * U * want
    assert abs(factor - 0.5 / (want + 1e-6)) <= 4 * U * factor
    assert grad_norm(gs, 0.5).tolist() == [norm, factor]


def tensors(sizes, dtype):
    """Tensors of those sizes whose sums of squares lie between 1 and 2, each another one."""
    g = torch.Generator().manual_seed(len(sizes))
    out = []
    for i, n in enumerate(sizes):
        x = torch.randn(n, generator=g)
        x *= math.sqrt(1 + (37 * i % 101) / 101) / max(x.norm().item(), 1e-30)
        out.append(x.to("cuda", dtype))
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("count", [254, 255, 508, 509, 600])
def test_more_tensors_than_one_launch(cuda, dtype, count):
    sizes = [(i * 731) % 900 + 1 for i in range(count)]
    for i in (0, 100, 252, 253, 254, 300, count - 1):
        if i < count:
            sizes[i] = 16384 * (1 + i % 3) + i % 2  # several tiles, whole and not, at the seams of the launches
    check(tensors(sizes, dtype))


@pytest.mark.parametrize("count", [254, 255, 600])
def test_empty_tensors_and_missing_ones_at_the_seam(cuda, count):
    sizes = [(i * 731) % 900 + 1 for i in range(count)]
    gs = tensors(sizes, torch.bfloat16)
    for i in (0, 252, 253, 254, 255, 507, 508, count - 1):
        if i < count:
            gs[i] = gs[i][:0]
    check(gs)
    from stratum_amd.optim import grad_norm
    some = [None if g.numel() == 0 else g for g in gs]
    assert torch.equal(grad_norm(some, 0.5), grad_norm(gs, 0.5))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("groups", [1023, 1024, 1025, 8191, 8192, 8193, 9300])
def test_more_partial_sums_than_one_pass(cuda, dtype, groups):
    """Two tensors of that many tiles together. One partial sum in 61, and those at the passes' ends, are 64
    times as large as the others: at least 3e-5 of the sum of squares each."""
    n = groups * 16384 - 5
    flat = torch.randn(n, device=cuda, generator=torch.Generator("cuda").manual_seed(groups)).to(dtype)
    tiles = sorted({*range(0, groups, 61), *(t for t in (1023, 1024, 8191, 8192, groups - 1) if t < groups)})
    for t in tiles:
        flat[t * 16384:(t + 1) * 16384] *= 8
    first = 700 * 16384
    check([flat[:first], flat[first:]])


def test_the_optimizers_norm_over_many_tensors(cuda):
    """Clipping through the optimizer, 300 parameters of several sizes."""
    from stratum_amd.optim import AdamW
    gs = tensors([(i * 731) % 900 + 1 for i in range(300)], torch.float32)
    ps = [torch.nn.Parameter(torch.zeros_like(g)) for g in gs]
    for p, g in zip(ps, gs):
        p.grad = g
    opt = AdamW(ps, max_grad_norm=0.5)
    opt.step()
    want = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
    assert abs(opt.grad_norm[0].item() - want) <= 2 * U * want
    for p, g in zip(ps, gs):
        m = 0.1 * g.double() * (0.5 / (want + 1e-6))
        assert ((opt.state[p]["exp_avg"].double() - m).abs() <= 8 * U * m.abs() + 1e-45).all()


@pytest.mark.parametrize("kinds", [(torch.bfloat16,), (torch.bfloat16, torch.float32)])
def test_a_norm_past_fp32_is_not_finite_for_the_factor_either(cuda, kinds):
    """64 gradients of 3e38: 2.4e39, infinite in fp32, so the factor is NaN and a step changes nothing, with
    one gradient type and with two."""
    from stratum_amd.optim import AdamW, grad_norm
    gs = [torch.full((64,), 3e38, dtype=kinds[0], device=cuda)] + [torch.ones(3, dtype=k, device=cuda) for k in kinds[1:]]
    norm, factor = grad_norm(gs[:1], 1.0).tolist()
    assert norm == math.inf and math.isnan(factor)
    ps = [torch.nn.Parameter(torch.ones_like(g)) for g in gs]
    for p, g in zip(ps, gs):
        p.grad = g
    opt = AdamW(ps, lr=0.1, max_grad_norm=1.0)
    opt.step()
    assert opt.grad_norm[0].item() == math.inf and all((p == 1).all() for p in ps)
    # one that fp32 still holds is clipped
    g = torch.full((64,), 2.0 ** 121, device=cuda)
    norm, factor = grad_norm([g], 1.0).tolist()
    assert norm == 2.0 ** 124 and factor == pytest.approx(2.0 ** -124, rel=1e-6)
