"""CPU tests of the optimizer's own bookkeeping: copies, checkpoints and the plans of its steps, with a
stand-in for the GPU's step where one is taken."""

import copy
import importlib
import pickle

import pytest
import torch

optim = importlib.import_module("stratum_amd.optim")


class Tensors:
    """Stands for AdamWTensors: counts what is built and stepped, and moves the parameters by lr."""
    built = 0

    def __init__(self, params, exp_avgs, exp_avg_sqs, *, masters=None, scales=None, follow=False):
        type(self).built += 1
        self.params, self.masters, self.scales = params, masters, scales

    def at(self):
        return [p.data_ptr() for p in self.params]

    def step(self, grads, *, step, lr, **rest):
        for p in self.params:
            p.sub_(lr)


@pytest.fixture
def on_cpu(monkeypatch):
    monkeypatch.setattr(optim, "AdamWTensors", Tensors)
    monkeypatch.setattr(optim, "grad_norm", lambda grads, most: torch.tensor([1.0, 1.0]))
    Tensors.built = 0


def parameter(n=10, dtype=torch.float32):
    p = torch.nn.Parameter(torch.ones(n, dtype=dtype))
    p.grad = torch.ones_like(p)
    return p


def copies(opt):
    return copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))


@pytest.mark.parametrize("bits,masters,clip", [(32, False, None), (8, True, 0.5)])
@pytest.mark.parametrize("steps", [0, 2])
def test_a_copied_optimizer_keeps_its_settings_and_steps(on_cpu, bits, masters, clip, steps):
    p = parameter(300, torch.bfloat16)
    opt = optim.AdamW([p], lr=0.25, state_bits=bits, master_weights=masters, max_grad_norm=clip)
    for _ in range(steps):
        opt.step()
    for other in copies(opt):
        assert (other.state_bits, other.master_weights, other.max_grad_norm) == (bits, masters, clip)
        q = other.param_groups[0]["params"][0]
        assert q is not p and torch.equal(q, p)
        q.grad = torch.ones_like(q)
        other.step()
        assert (q == 1.0 - 0.25 * (steps + 1)).all() and (p == 1.0 - 0.25 * steps).all()
        assert other.state[q]["step"] == steps + 1 and set(other.state[q]) >= {"exp_avg", "exp_avg_sq"}
        assert ("master" in other.state[q]) == masters and ("exp_avg_scale" in other.state[q]) == (bits == 8)
