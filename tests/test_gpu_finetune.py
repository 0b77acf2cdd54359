"""GPU tests of the gated MLP module, of the fine-tuning example and of the norm and the
step recorded into a graph.

Bounds of the module, as relative norms in bfloat16: the forward rounds h and the output
(2 x 2^-8 at most, held to 1e-2); the input gradient rounds dh, [dg | du] and itself
(3 x 2^-8, held to 1.5e-2)."""

import os
import sys

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


class DenseMLP(nn.Module):
    def __init__(self, hidden, inter):
        super().__init__()
        self.gate_proj, self.up_proj = (nn.Linear(hidden, inter, bias=False) for _ in range(2))
        self.down_proj = nn.Linear(inter, hidden, bias=False)
        self.act_fn = nn.SiLU()


def rel(y, ref):
    return ((y.double() - ref).norm() / ref.norm()).item()


@pytest.mark.parametrize("rows", [1, 70, 400])
def test_gated_mlp_matches_64_bits(cuda, rows):
    from stratum_amd.mlp import NF4GatedMLP, quantize_mlp_
    torch.manual_seed(rows)
    mlp = quantize_mlp_(DenseMLP(256, 640).to(cuda, torch.bfloat16).requires_grad_(False))
    wg, wu, wd = (getattr(mlp, n).weight.double() for n in ("gate_proj", "up_proj", "down_proj"))
    gated = NF4GatedMLP(mlp)
    assert gated.gate_up_packed.data_ptr() == mlp.gate_proj.quantized.data_ptr()
    x = torch.randn(rows, 256, device=cuda, dtype=torch.bfloat16, requires_grad=True)
    dy = torch.randn(rows, 256, device=cuda, dtype=torch.bfloat16)
    y = gated(x)
    y.backward(dy)
    xd = x.detach().double().requires_grad_(True)
    yd = (nn.functional.silu(xd @ wg.t()) * (xd @ wu.t())) @ wd.t()
    yd.backward(dy.double())
    assert rel(y.detach(), yd.detach()) <= 1e-2 and rel(x.grad, xd.grad) <= 1.5e-2


@pytest.mark.parametrize("bits", [32, 8])
def test_example_learns_its_tokens(cuda, bits):
    from finetune_adapters import train
    losses, norms = train(steps=12, bits=bits, hidden=256, inter=768, vocab=512, batch=4, length=64)
    assert losses.shape == norms.shape == (12,)
    assert torch.isfinite(losses).all() and torch.isfinite(norms).all() and (norms > 0).all()
    assert losses[-1] < losses[0]
    assert (train(steps=3, bits=bits, hidden=256, inter=768, vocab=512, batch=4, length=64)[0][0] == losses[0])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [3, 130])
def test_norm_and_step_in_a_graph(cuda, bits, count):
    """Replayed with eager work between: every replay gives the eager call's bits."""
    from stratum_amd.optim import AdamWTensors, grad_norm
    torch.manual_seed(count)
    start = [torch.randn(900 + 37 * i, device=cuda) for i in range(count)]
    grads = [torch.randn_like(p) for p in start]

    def states(ps):
        if bits == 32:
            return [torch.zeros_like(p) for p in ps], [torch.zeros_like(p) for p in ps], None
        codes = lambda: [torch.zeros(p.shape, dtype=torch.uint8, device=cuda) for p in ps]  # noqa: E731
        scales = lambda: [torch.zeros((p.numel() + 255) // 256, device=cuda) for p in ps]  # noqa: E731
        return codes(), codes(), (scales(), scales())

    def run(t):
        norm = grad_norm(grads, 0.5)
        t.step(grads, step=1, lr=1e-2, weight_decay=0.01, grad_scale=norm[1:])
        return norm
    captured, eager = ([p.clone() for p in start] for _ in range(2))
    (mc, vc, sc), (me, ve, se) = states(captured), states(eager)
    tc, te = AdamWTensors(captured, mc, vc, scales=sc), AdamWTensors(eager, me, ve, scales=se)
    warm = [p.clone() for p in start]
    mw, vw, sw = states(warm)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(AdamWTensors(warm, mw, vw, scales=sw))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = run(tc)
    for _ in range(4):
        expected = run(te)
        norm.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, expected)
        for a, b in zip(captured + mc + vc, eager + me + ve):
            assert torch.equal(a, b)
        for g in grads:
            g.mul_(-0.7)
