"""GPU tests of copied optimizers and of checkpoints between optimizers of other settings."""

import copy
import io

import pytest
import torch

pytestmark = pytest.mark.gpu


def run(opt, ps, steps):
    for t in steps:
        g = torch.Generator().manual_seed(t)
        for p in ps:
            p.grad = torch.randn(p.shape, generator=g).to(p)
        opt.step()


def params(seed=0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(n, generator=g).to("cuda", dtype)) for n in (700, 256, 3)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("way", ["deepcopy", "torch.save"])
def test_a_copied_optimizer_goes_on_with_the_same_bits(cuda, bits, way):
    from stratum_amd.optim import AdamW
    ps = params()
    opt = AdamW(ps, lr=1e-2, state_bits=bits, master_weights=True, max_grad_norm=1.0)
    run(opt, ps, range(3))
    if way == "deepcopy":
        other = copy.deepcopy(opt)
    else:
        box = io.BytesIO()
        torch.save(opt, box)
        box.seek(0)
        other = torch.load(box, weights_only=False)  # this test's own file
    qs = other.param_groups[0]["params"]
    run(opt, ps, range(3, 6))
    run(other, qs, range(3, 6))
    assert all(p.data_ptr() != q.data_ptr() and torch.equal(p, q) for p, q in zip(ps, qs))
    assert all(torch.equal(opt.state[p]["master"], other.state[q]["master"]) for p, q in zip(ps, qs))


@pytest.mark.parametrize("masters", [(False, True), (True, False), (True, True)])
@pytest.mark.parametrize("bits", [(32, 8), (8, 32)])
def test_a_checkpoint_of_the_other_width(cuda, bits, masters):
    """The moments become the nearest codes, or the values that the codes stand for, and training goes on."""
    from stratum_amd.optim import AdamW, state_codes, state_values
    ps, qs = params(1), params(1)
    first = AdamW(ps, lr=1e-2, state_bits=bits[0], master_weights=masters[0])
    second = AdamW(qs, lr=1e-2, state_bits=bits[1], master_weights=masters[1])
    run(first, ps, range(3))
    with torch.no_grad():
        for p, q in zip(ps, qs):
            q.copy_(p)
    second.load_state_dict(first.state_dict())
    for p, q in zip(ps, qs):
        a, b = first.state[p], second.state[q]
        for name, signed in (("exp_avg", True), ("exp_avg_sq", False)):
            if bits[1] == 8:
                codes, scales = state_codes(a[name], signed=signed)
                assert torch.equal(b[name], codes) and torch.equal(b[name + "_scale"], scales)
            else:
                want = state_values(a[name], a[name + "_scale"], signed=signed)
                assert torch.equal(b[name], want) and name + "_scale" not in b
        assert ("master" in b) == masters[1]
        if masters == (True, True):
            assert torch.equal(a["master"], b["master"])
    run(second, qs, range(3, 5))
    assert all(second.state[q]["step"] == 5 and torch.isfinite(q).all() for q in qs)
    assert all(not torch.equal(p, q) for p, q in zip(ps, qs))


@pytest.mark.parametrize("masters", [True, False])
def test_a_checkpoint_of_torchs_adamw_goes_on(cuda, masters):
    """Three steps of torch's AdamW in fp32, then one here: within fp32 rounding of its fourth."""
    from stratum_amd.optim import AdamW
    ps, qs = params(2, torch.float32), params(2, torch.float32)
    first, second = torch.optim.AdamW(ps, lr=1e-2), AdamW(qs, lr=0.5, master_weights=masters)
    run(first, ps, range(3))
    with torch.no_grad():
        for p, q in zip(ps, qs):
            q.copy_(p)
    second.load_state_dict(first.state_dict())
    run(first, ps, [3])
    run(second, qs, [3])
    # an update of at most 3.2 lr with 20 roundings here and as many there, 3 of the parameter each
    u = 2.0 ** -24
    assert all(((p - q).abs() <= 40 * u * 3.2e-2 + 6 * u * p.abs()).all() for p, q in zip(ps, qs))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_repeats_its_numbers(cuda, bits):
    """Replays of the optimizer's third step against eager steps of the number three; it counts once."""
    from stratum_amd.optim import AdamW, AdamWTensors
    ps = params(3, torch.float32)
    opt = AdamW(ps, lr=1e-2, state_bits=bits)
    run(opt, ps, range(2))
    mine = [p.detach().clone() for p in ps]
    names = ("exp_avg", "exp_avg_sq") + (("exp_avg_scale", "exp_avg_sq_scale") if bits == 8 else ())
    m, v, *scales = ([opt.state[p][name].clone() for p in ps] for name in names)
    tensors = AdamWTensors(mine, m, v, scales=tuple(scales) or None)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        for p in ps:
            p.grad.mul_(-0.7)
        graph.replay()
        tensors.step([p.grad for p in ps], step=3, lr=1e-2, grad_scale=torch.ones((), device=cuda))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ps, mine))
    assert all(opt.state[p]["step"] == 3 for p in ps)


def test_a_tensor_of_more_threads_than_one_launch_takes(cuda):
    """2^24 tiles of 1024 elements and some more: two launches. The elements around their seam."""
    from stratum_amd.optim import AdamWTensors
    seam, n = ((1 << 24) - 1) * 1024, (1 << 24) * 1024 + 5001
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 13 * n:  # 2 + 2 + 4 + 4 bytes an element
        pytest.skip("takes 206 GB")
    p, g = (torch.zeros(n, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    m, v = (torch.zeros(n, device=cuda) for _ in range(2))
    spots = torch.tensor([0, 1 << 32, seam - 1, seam, seam + 1, seam + 1024, n - 1], device=cuda)
    g[spots] = torch.tensor([1., -2., 3., -4., 5., -6., 7.], dtype=torch.bfloat16, device=cuda)
    AdamWTensors([p], [m], [v]).step([g], step=1, lr=0.125, weight_decay=0.0)
    want = torch.tensor([-0.125, 0.125] * 3 + [-0.125], dtype=torch.bfloat16, device=cuda)  # lr sign(g)
    assert torch.equal(p[spots], want)
    around = seam - (1 << 20)
    assert int((p[:1 << 20] != 0).sum()) == 1
    for t in (p, m, v):  # the five spots of the last stretch, and nothing else there
        assert int((t[around:] != 0).sum()) == 5
    del p, g, m, v, t
    torch.cuda.empty_cache()
