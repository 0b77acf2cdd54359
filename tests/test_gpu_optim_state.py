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
