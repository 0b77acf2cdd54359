"""CPU tests of the optimizer's own bookkeeping: copies, checkpoints and the plans of its steps, with a
stand-in for the GPU's step where one is taken."""

import copy
import ctypes
import importlib
import pickle

import numpy as np
import pytest
import torch

from stratum_amd import _lib

optim = importlib.import_module("stratum_amd.optim")


class Tensors:
    """Stands for AdamWTensors: counts what is built and stepped, and moves the parameters by lr."""
    built, newest = 0, []

    def __init__(self, params, exp_avgs, exp_avg_sqs, *, masters=None, scales=None, follow=False):
        type(self).built += 1
        assert masters is None or len(masters) == len(params)
        self.kept = None if masters is None else [m.data_ptr() for m in masters]
        type(self).newest.append(self)
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
    Tensors.newest.clear()


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


def test_a_checkpoint_without_masters_gets_them(on_cpu):
    p, q = parameter(300, torch.bfloat16), parameter(300, torch.bfloat16)
    opt, other = optim.AdamW([p], lr=0.25), optim.AdamW([q], lr=0.25, master_weights=True)
    opt.step()
    with torch.no_grad():
        q.copy_(p)
    other.load_state_dict(opt.state_dict())
    master = other.state[q]["master"]
    assert master.dtype == torch.float32 and torch.equal(master, p.detach().float())
    master.zero_()
    assert (q == 0.75).all()
    # a parameter that joins later has one too, in the same set of tensors
    late = parameter(5, torch.bfloat16)
    other.add_param_group({"params": [late]})
    other.step()
    assert "master" in other.state[late]


def test_a_checkpoint_with_masters_loses_them_where_none_are_kept(on_cpu):
    p, q = parameter(300, torch.bfloat16), parameter(300, torch.bfloat16)
    opt, other = optim.AdamW([p], master_weights=True), optim.AdamW([q])
    opt.step()
    other.load_state_dict(opt.state_dict())
    assert "master" not in other.state[q]
    other.step()


def test_a_checkpoint_of_torchs_adamw(on_cpu):
    p, q = parameter(300, torch.bfloat16), parameter(300, torch.bfloat16)
    opt, other = torch.optim.AdamW([p], lr=0.125), optim.AdamW([q], master_weights=True)
    for _ in range(3):
        opt.step()
    other.load_state_dict(opt.state_dict())
    state = other.state[q]
    assert state["step"] == 3 and type(state["step"]) is int
    for name in ("exp_avg", "exp_avg_sq"):
        assert state[name].dtype == torch.float32 and torch.equal(state[name], opt.state[p][name].float())
    assert other.param_groups[0]["lr"] == 0.125
    other.step()
    assert other.state[q]["step"] == 4


def test_what_is_no_state_of_an_adamw_is_refused(on_cpu):
    p, q = parameter(), parameter()
    sgd = torch.optim.SGD([p], lr=0.1, momentum=0.9)
    sgd.step()
    with pytest.raises(ValueError, match="exp_avg"):
        optim.AdamW([q]).load_state_dict(sgd.state_dict())
    good = optim.AdamW([p])
    good.step()
    with pytest.raises(ValueError, match="elements"):
        optim.AdamW([parameter(11)]).load_state_dict(good.state_dict())


def test_loaded_states_are_copies(on_cpu):
    p, q = parameter(300, torch.bfloat16), parameter(300, torch.bfloat16)
    opt, other = (optim.AdamW([x], state_bits=8, master_weights=True) for x in (p, q))
    opt.step()
    other.load_state_dict(opt.state_dict())
    for name, t in opt.state[p].items():
        if name != "step":
            assert t.data_ptr() != other.state[q][name].data_ptr() and torch.equal(t, other.state[q][name])
            assert t.dtype == other.state[q][name].dtype


def test_a_hook_before_loading_changes_what_is_loaded(on_cpu):
    p, q = parameter(), parameter()
    opt, other = optim.AdamW([p]), optim.AdamW([q])
    opt.step()

    def hook(_, given):
        return {**given, "state": {i: {**s, "exp_avg": torch.full_like(s["exp_avg"], 7.0)} for i, s in given["state"].items()}}
    other.register_load_state_dict_pre_hook(hook)
    for _ in range(2):
        other.load_state_dict(opt.state_dict())
        assert (other.state[q]["exp_avg"] == 7.0).all()
    assert len(other._optimizer_load_state_dict_pre_hooks) == 1


def test_sets_that_differ_in_their_step_count_keep_their_plans(on_cpu):
    early, late = parameter(), parameter()
    opt = optim.AdamW([early, late], lr=0.25)
    late.grad = None
    opt.step()
    late.grad = torch.ones_like(late)
    opt.step()
    before = Tensors.built
    for _ in range(5):
        opt.step()
    assert Tensors.built == before
    assert (opt.state[early]["step"], opt.state[late]["step"]) == (7, 6)
    assert (early == 1 - 7 * 0.25).all() and (late == 1 - 6 * 0.25).all()


def test_masters_switched_on_later_stand_apart_from_states_without(on_cpu):
    p, q = (parameter(4, torch.bfloat16) for _ in range(2))
    opt = optim.AdamW([p], lr=0.25)
    opt.step()
    opt.master_weights = True
    opt.add_param_group({"params": [q]})
    opt.param_groups[0]["params"].append(opt.param_groups.pop()["params"][0])
    opt.state[p]["step"] = 0
    opt.step()
    assert "master" in opt.state[q] and "master" not in opt.state[p]
    assert (p == 0.5).all() and (q == 0.75).all()
    assert [opt.state[q]["master"].data_ptr()] in [t.kept for t in Tensors.newest]  # the step writes it


# ------------------------------------------------------------------ launches of 2^32 threads and more

def row(n, where):
    return np.array([[where] * 2 + [0] + [where] * 4 + [n]], np.int64)


@pytest.mark.parametrize("bits,tile", [(32, 1024), (8, 2048)])
def test_a_table_holds_no_more_work_groups_than_a_launch_takes(bits, tile):
    L = _lib.lib()
    where = ctypes.addressof(ctypes.create_string_buffer(64)) // 16 * 16 + 16  # never read: the table is only filled
    table = ctypes.create_string_buffer(2 * 128)
    most = (1 << 24) - 1  # groups of 256 threads below 2^32 threads

    def fill(*sizes):
        rows = np.concatenate([row(n, where) for n in sizes])
        return L.stm_adamw_fill_table(len(sizes), rows.ctypes.data, 1, 1, bits, ctypes.addressof(table) + 15 & ~15)
    assert fill(most * tile) == most
    assert fill(most * tile + 1) == _lib.STM_ERR_UNSUPPORTED
    assert fill((most - 1) * tile, tile) == most
    assert fill((most - 1) * tile, tile + 1) == _lib.STM_ERR_UNSUPPORTED

    def step(groups):
        return L.stm_adamw_step_table(1, where, groups, 1, 1, bits, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, None, None)
    assert step(most + 1) == _lib.STM_ERR_INVALID and step(0) == 0


def test_a_norm_refuses_a_tensor_of_more_work_groups_than_a_launch_takes():
    L = _lib.lib()
    where = ctypes.addressof(ctypes.create_string_buffer(64)) // 16 * 16 + 16
    most = (1 << 23) - 1  # groups of 512 threads
    one, n = np.array([where], np.int64), np.array([most * 16384 + 1], np.int64)
    assert L.stm_grad_norm(1, one.ctypes.data, n.ctypes.data, 1, 1.0, 1.0, where, where, 1 << 40,
                           None) == _lib.STM_ERR_UNSUPPORTED


def test_a_parameter_that_was_looked_at_and_never_stepped_loads(on_cpu):
    ps, qs = ([parameter(), parameter()] for _ in range(2))
    opt, other = optim.AdamW(ps), optim.AdamW(qs, lr=0.25)
    ps[1].grad = None
    opt.step()
    assert len(opt.state[ps[1]]) == 0  # which leaves an empty entry
    other.load_state_dict(opt.state_dict())
    other.step()
    assert (other.state[qs[0]]["step"], other.state[qs[1]]["step"]) == (2, 1)


@pytest.mark.parametrize("other,kw", [(torch.optim.AdamW, dict(amsgrad=True)), (torch.optim.AdamW, dict(maximize=True)),
                                      (torch.optim.Adam, dict(weight_decay=0.1))])
def test_a_state_of_another_update_is_refused_and_nothing_changes(on_cpu, other, kw):
    p, q = parameter(), parameter()
    theirs, mine = other([p], lr=0.5, **kw), optim.AdamW([q], lr=0.25)
    theirs.step()
    mine.step()
    with pytest.raises(ValueError):
        mine.load_state_dict(theirs.state_dict())
    assert mine.param_groups[0]["lr"] == 0.25 and mine.state[q]["step"] == 1
    assert not mine._optimizer_load_state_dict_pre_hooks


def test_a_state_of_adam_without_weight_decay_loads(on_cpu):
    p, q = parameter(), parameter()
    theirs, mine = torch.optim.Adam([p], lr=0.5), optim.AdamW([q], lr=0.25)
    theirs.step()
    mine.load_state_dict(theirs.state_dict())
    assert mine.param_groups[0]["weight_decay"] == 0 and mine.state[q]["step"] == 1
    mine.step()
