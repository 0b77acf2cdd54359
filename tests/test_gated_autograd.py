"""CPU tests of how the gated block meets autograd, with a stand-in for its kernel."""

import importlib

import pytest
import torch
from torch.autograd import forward_ad

layers = importlib.import_module("stratum_amd.nf4_linear")


@pytest.fixture
def stand_in(monkeypatch):
    """The forward's kernel replaced by torch operations on plain values, as a kernel reads them."""
    def forward(x, packed, absmax, shape, blocksize=64):
        with torch.no_grad():
            plain = torch.from_numpy(x.detach().numpy().copy())
            return plain[..., :shape[0] // 2] * 2.0
    monkeypatch.setattr(layers, "nf4_gated_fwd", forward)


PACKED, ABSMAX = torch.zeros(64 * 128, dtype=torch.uint8), torch.ones(256)


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("requires_grad", [True, False])
def test_a_forward_mode_dual_is_refused_and_does_not_lose_its_tangent(stand_in, grad_mode, requires_grad):
    x, t = torch.randn(3, 128, requires_grad=requires_grad), torch.randn(3, 128)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        dual = forward_ad.make_dual(x, t)
        with pytest.raises((NotImplementedError, RuntimeError)):
            layers.nf4_gated(dual, PACKED, ABSMAX, (128, 128), recompute=True)


def test_plain_inputs_inside_and_outside_a_dual_level_run(stand_in):
    x = torch.randn(3, 128)
    want = x[:, :64] * 2.0
    assert torch.equal(layers.nf4_gated(x, PACKED, ABSMAX, (128, 128)), want)
    with forward_ad.dual_level():
        assert torch.equal(layers.nf4_gated(x, PACKED, ABSMAX, (128, 128)), want)
    with torch.inference_mode():
        assert torch.equal(layers.nf4_gated(x, PACKED, ABSMAX, (128, 128)), want)
