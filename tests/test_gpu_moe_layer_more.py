"""GPU tests of the sparse layer as a module: its bias under conversions, the gradients of its parameters by value, and
recomputation."""

import copy

import pytest
import torch

from test_gpu_moe_layer import BF, F4, FP, close, dense, layer, seeded

pytestmark = pytest.mark.gpu


def test_the_bias_stays_in_32_bits(cuda):
    """A balancing bias tells keys apart that a 16-bit one does not."""
    bias = 1.0 + torch.arange(16, device=cuda) * 2.0 ** -12  # all of them 1 in bf16, and 2^-10 apart in fp16
    kw = dict(E=16, k=4, score="sigmoid")
    moe = layer(bias=bias, **kw)
    with torch.no_grad():
        moe.router.weight.zero_()  # the bias alone decides
    x, r = seeded((5, 128), 1, 1.0, BF), seeded((5, 128), 2, 1.0, BF)
    want = moe(x, r)
    for change in (lambda m: m.to(BF), lambda m: m.half().bfloat16(), lambda m: torch.nn.Sequential(m).to(BF)[0],
                   lambda m: m.to("cpu", BF).to(cuda), lambda m: copy.deepcopy(m).bfloat16(), lambda m: m.float().to(BF)):
        again = change(copy.deepcopy(moe))
        assert again.bias.dtype == F4 and torch.equal(again.bias, bias) and again.bias.device == bias.device
        assert "bias" in again.state_dict() and not again.bias.requires_grad
        assert torch.equal(again(x, r), want)
    moe.load_state_dict({n: t.to(BF) for n, t in moe.state_dict().items()})
    assert moe.bias.dtype == F4
