"""GPU tests of gradients that are not finite in an optimizer: the step leaves parameters and
states as they were, with clipping and without, and the next one goes on from there."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def tensors(opt, ps):
    return [p.detach().clone() for p in ps] + [t.clone() for p in ps for k, t in opt.state[p].items() if k != "step"]


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("clip", [None, 1.0])
@pytest.mark.parametrize("kinds", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                   (torch.float32, torch.bfloat16)])
def test_such_a_step_changes_nothing(cuda, bad, bits, clip, kinds):
    from stratum_amd.optim import AdamW
    torch.manual_seed(1)
    ps = [torch.nn.Parameter(torch.randn(n, device=cuda).to(kind)) for n, kind in zip((1000, 300), kinds)]
    clean = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt, other = (AdamW(x, state_bits=bits, master_weights=True, max_grad_norm=clip) for x in (ps, clean))
    grads = [[torch.randn_like(p.detach()) for p in ps] for _ in range(2)]

    def go(x, o, g):
        for p, q in zip(x, g):
            p.grad = q.clone()
        o.step()
    go(ps, opt, grads[0])
    before = tensors(opt, ps)
    spoiled = [g.clone() for g in grads[1]]
    spoiled[1][299] = bad
    go(ps, opt, spoiled)
    assert all(torch.equal(a, b) for a, b in zip(before, tensors(opt, ps)))
    assert not math.isfinite(opt.grad_norm[0].item()) and opt.state[ps[0]]["step"] == 2
    go(clean, other, grads[0])
    for p in clean:
        other.state[p]["step"] = 2
    go(ps, opt, grads[1])
    go(clean, other, grads[1])
    assert all(torch.equal(a, b) for a, b in zip(tensors(opt, ps), tensors(other, clean)))


def test_an_unclipped_step_is_the_one_with_the_factor_one(cuda):
    from stratum_amd.optim import AdamW
    torch.manual_seed(2)
    a, b = (torch.nn.Parameter(x) for x in torch.randn(1, 5000, device=cuda).repeat(2, 1).unbind(0))
    first, second = AdamW([a]), AdamW([b])
    for _ in range(3):
        a.grad = torch.randn_like(a)
        b.grad = a.grad.clone()
        first.step()
        second.step(grad_scale=torch.ones((), device=cuda))
        assert torch.equal(a, b)
    assert first.grad_norm[0].item() == pytest.approx(a.grad.norm().item(), rel=1e-5) and second.grad_norm == []
