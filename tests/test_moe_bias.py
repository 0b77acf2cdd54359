"""CPU test of the sparse layer's balancing bias under conversions of the module."""

import torch

from test_moe import bank
from stratum_amd import NF4MoE


def test_the_bias_stays_in_32_bits():
    bias = 1.0 + torch.arange(4) * 2.0 ** -20
    layer = NF4MoE(torch.nn.Linear(128, 4, bias=False), bank(4, 128, 128), bank(4, 128, 64), 2, bias=bias)
    for change in (lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.double(), lambda m: m.float()):
        assert change(layer) is layer
        assert layer.bias.dtype == torch.float32 and torch.equal(layer.bias, bias)
    torch.nn.Sequential(torch.nn.Sequential(layer)).half()
    assert torch.equal(layer.bias, bias) and layer.router.weight.dtype == torch.float16
    assert torch.equal(layer.state_dict()["bias"], bias)
    assert layer.to("meta", torch.float16).bias.dtype == torch.float32 and layer.bias.is_meta
    plain = NF4MoE(torch.nn.Linear(128, 4, bias=False), bank(4, 128, 128), bank(4, 128, 64), 2)
    assert plain.half().bias is None
