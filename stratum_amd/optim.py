"""The end of a training step on the GPU: the norm of all gradients and AdamW over
many tensors, each in a few launches of hand-written kernels.

The reference steps its LoRA parameters with torch's AdamW, one tensor after another on
the host (``stratum/optim.py:72``), and unscales and clips their gradients there
(``stratum/grad_scaler.py``). Here nothing leaves the GPU: :func:`grad_norm` leaves the
norm and the factor that clips (and unscales) the gradients in device memory, the step
reads the factor there, and a step whose gradients are not finite changes nothing.

* :class:`AdamW` is a ``torch.optim.Optimizer`` with states in 32 bits or in 8, and
  optional fp32 masters of 16-bit parameters;
* :class:`AdamWTensors` is the step over lists of tensors that the caller holds;
* :func:`state_codes` and :func:`state_values` convert fp32 values to 8-bit states and back.

An 8-bit state holds one code per element and one fp32 scale per 256 elements (the largest
magnitude among them); the levels are dense near the scale and reach down to 8^-6 (first
moment, which has a sign) or 8^-7 (second moment) of it. A step reads and writes 4 bytes
of states per element instead of 16.
"""

from __future__ import annotations

import math
from typing import Iterable, Optional, Sequence

import numpy as np
import torch

from . import _lib

__all__ = ["AdamW", "AdamWTensors", "STATE_BLOCK", "grad_norm", "state_codes", "state_values"]

STATE_BLOCK = 256  # elements per scale of an 8-bit state

# Lists up to this length go as kernel arguments (one launch); longer ones as a table that is copied to
# the GPU, which costs 10 us and saves the drain between launches of 56 tensors (448 adapters of an
# 8B model: 257 us in 8 launches, where one launch over as many elements takes 219).
_ARGUMENT_TENSORS = 56

_FOLLOW = 0x100  # STM_ADAMW_FOLLOW

# columns of a row of the tensor table (stm_adamw_tensor)
_PARAM, _GRAD, _MASTER, _M, _V, _M_SCALE, _V_SCALE, _N = range(8)


def _blocks(n: int) -> int:
    return -(-n // STATE_BLOCK)


def _gpu(t: torch.Tensor, what: str) -> torch.device:
    if not t.is_cuda:
        raise RuntimeError(f"{what} runs on the GPU kernels; got a tensor on {t.device}")
    return t.device


def _held(name: str, t: torch.Tensor, like: torch.Tensor, dtype: torch.dtype, numel: int) -> None:
    """*t* can stand beside the parameter *like* in the tensor table."""
    if t.dtype != dtype or t.numel() != numel or t.device != like.device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of {numel} elements on {like.device}, got "
                         f"{t.dtype}, {t.numel()} elements on {t.device}, "
                         f"{'' if t.is_contiguous() else 'not '}contiguous")


def _laid_out(i: int, g: torch.Tensor, first: torch.Tensor) -> torch.Tensor:
    if g.is_contiguous():
        raise ValueError(f"gradient {i} is on {g.device}, the first one on {first.device}")
    return g.contiguous()


class AdamWTensors:
    """One AdamW step over lists of tensors: ``params`` of one dtype (fp32, bf16 or fp16),
    their moments, and optionally fp32 ``masters`` of which the parameters are rounded
    copies. ``scales`` = (first moments' scales, second moments' scales) makes the moments
    8-bit codes (uint8, with ``ceil(numel / 256)`` fp32 scales each); without it they are
    fp32. All contiguous, on one GPU. The tensors are checked once, here, and written in
    place by :meth:`step`. A step takes the masters as they are and does not read the
    parameters beside them; with ``follow`` it does, and an element of a parameter that is not its
    master rounded (something else has written it) replaces the master first.
    """

    def __init__(self, params: Sequence[torch.Tensor], exp_avgs: Sequence[torch.Tensor],
                 exp_avg_sqs: Sequence[torch.Tensor], *, masters: Optional[Sequence[torch.Tensor]] = None,
                 scales: Optional[tuple] = None, follow: bool = False):
        params, exp_avgs, exp_avg_sqs = list(params), list(exp_avgs), list(exp_avg_sqs)
        if not params:
            raise ValueError("AdamWTensors needs at least one tensor")
        first = params[0]
        self.device, self.dtype = _gpu(first, "AdamW"), first.dtype
        self.param_tag = _lib.dtype_tag(first.dtype)
        self.state_bits = 8 if scales is not None else 32
        self.follow = bool(follow) and masters is not None
        state_dtype = torch.uint8 if scales is not None else torch.float32
        columns = {"exp_avg": exp_avgs, "exp_avg_sq": exp_avg_sqs}
        if masters is not None:
            columns["master"] = masters = list(masters)
        if scales is not None:
            columns["exp_avg scale"], columns["exp_avg_sq scale"] = (list(s) for s in scales)
        for name, column in columns.items():
            if len(column) != len(params):
                raise ValueError(f"{len(params)} parameters, but {len(column)} of {name}")
        sizes = np.array([p.numel() for p in params], dtype=np.int64)
        blocks = -(-sizes // STATE_BLOCK)
        table = np.zeros((len(params), 8), dtype=np.int64)
        for name, at, column, dtype in (("parameter", _PARAM, params, first.dtype),
                                        ("exp_avg", _M, exp_avgs, state_dtype),
                                        ("exp_avg_sq", _V, exp_avg_sqs, state_dtype),
                                        ("master", _MASTER, columns.get("master"), torch.float32),
                                        ("exp_avg scale", _M_SCALE, columns.get("exp_avg scale"), torch.float32),
                                        ("exp_avg_sq scale", _V_SCALE, columns.get("exp_avg_sq scale"), torch.float32)):
            if column is None:
                continue
            want = blocks if name.endswith("scale") else sizes
            _, index, _, bad = _lib.fast().collect(column, table.ctypes.data + 8 * at, 8, want.ctypes.data, 0)
            if bad >= 0 or index != self.device.index or column[0].dtype != dtype:
                for i, t in enumerate(column):
                    _held(f"{name} {i}", t, first, dtype, int(want[i]))
        table[:, _N] = self._sizes = sizes
        self._table = table
        self._addresses = table.ctypes.data, sizes.ctypes.data  # (a microsecond each to ask numpy for)
        # everything a step writes: held here (the table has bare addresses), and its versions counted up
        self._written = [t for column in (params, *columns.values()) for t in column]

    def at(self) -> list:
        """The parameters' addresses."""
        return self._table[:, _PARAM].tolist()

    def _plain(self, i: int, grads: list) -> torch.Tensor:
        """Gradient *i* in the parameter's order of elements; raises if that is not what is wrong with it."""
        g, n = grads[i], int(self._sizes[i])
        first = next(x for x in grads if x is not None)
        if not isinstance(g, torch.Tensor) or g.layout != torch.strided:
            raise ValueError(f"gradient {i} must be a dense tensor")
        _lib.dtype_tag(first.dtype)
        if g.dtype != first.dtype or g.numel() != n or g.device != self.device:
            raise ValueError(f"gradient {i} must hold {n} {first.dtype} elements on {self.device}, got {g.numel()} "
                             f"{g.dtype} on {g.device}")
        return _laid_out(i, g, first)  # held by the list until the launch, on the stream it was made on

    def step(self, grads: Sequence[Optional[torch.Tensor]], *, step: int, lr: float, betas: tuple = (0.9, 0.999),
             eps: float = 1e-8, weight_decay: float = 0.01, grad_scale: Optional[torch.Tensor] = None) -> None:
        """Step number ``step`` (from 1) with one gradient per parameter, of one dtype; a
        tensor whose gradient is None stays as it is. ``grad_scale``, an fp32 scalar on the GPU, multiplies the
        gradients first (``grad_norm(...)[1]``); where it is not finite the step writes nothing.
        Runs on the current stream, without synchronising. Captured into a graph, a replay repeats
        these numbers: the rate, the step number and its bias corrections are part of the launch,
        and only what lies on the GPU (gradients, ``grad_scale``) is read anew."""
        if len(grads) != len(self._sizes):
            raise ValueError(f"{len(self._sizes)} parameters, but {len(grads)} gradients")
        if grad_scale is not None and (grad_scale.numel() != 1 or grad_scale.dtype != torch.float32
                                       or grad_scale.device != self.device):
            raise ValueError(f"grad_scale must be one fp32 value on {self.device}")
        grads, written = list(grads), self._written
        rows, sizes = self._addresses
        while True:
            tag, index, count, bad = _lib.fast().collect(grads, rows + 8 * _GRAD, 8, sizes, 0)
            if bad < 0:
                break
            grads[bad] = self._plain(bad, grads)
        if count == 0:
            return
        if tag < 0:
            raise ValueError("gradients must be float16, bfloat16 or float32")
        if index != self.device.index:
            raise ValueError(f"the gradients are on GPU {index}, the parameters on {self.device}")
        if count < len(grads):
            some = [i for i, g in enumerate(grads) if g is not None]
            per = len(grads)
            table = np.ascontiguousarray(self._table[some])
            rows = table.ctypes.data
            written = [written[c * per + i] for c in range(len(written) // per) for i in some]
        numbers = (lr, betas[0], betas[1], eps, weight_decay, step,
                   grad_scale.data_ptr() if grad_scale is not None else None)
        types = (self.param_tag, tag, self.state_bits | (_FOLLOW if self.follow else 0))
        lib, n = _lib.lib(), count
        with _lib.device_guard(self.device):
            stream = _lib.stream_handle(self.device)
            if n <= _ARGUMENT_TENSORS or torch.cuda.is_current_stream_capturing():
                rc = lib.stm_adamw_step(n, rows, *types, *numbers, stream)
            else:
                host = torch.empty(lib.stm_adamw_table_bytes(n), dtype=torch.uint8, pin_memory=True)
                rc = lib.stm_adamw_fill_table(n, rows, *types, host.data_ptr())
                if rc == _lib.STM_ERR_UNSUPPORTED:  # more elements than one launch takes
                    rc = lib.stm_adamw_step(n, rows, *types, *numbers, stream)
                elif rc >= 0:  # the caching host allocator keeps the pinned block until the copy has run
                    held = host.to(self.device, non_blocking=True)
                    rc = lib.stm_adamw_step_table(n, held.data_ptr(), rc, *types, *numbers, stream)
        _lib.check(rc, "stm_adamw_step")
        _lib.fast().bump(written)


def _plain_gradient(i: int, grads: list) -> torch.Tensor:
    """Gradient *i* as a contiguous tensor; raises if that is not what is wrong with it."""
    g, first = grads[i], next(x for x in grads if x is not None)
    if not isinstance(g, torch.Tensor) or g.layout != torch.strided:
        raise ValueError(f"gradient {i} must be a dense tensor")
    _gpu(first, "grad_norm")
    _lib.dtype_tag(first.dtype)
    if g.dtype != first.dtype or g.device != first.device:
        raise ValueError(f"gradient {i} must be {first.dtype} on {first.device}, got {g.dtype} on {g.device}")
    return _laid_out(i, g, first)


def grad_norm(grads: Iterable[Optional[torch.Tensor]], max_norm: float = math.inf, *,
              loss_scale: float = 1.0) -> torch.Tensor:
    """``[norm, factor]`` (fp32, on the GPU) over all elements of all gradients: the 2-norm
    divided by ``loss_scale``, and ``min(1, max_norm / (norm + 1e-6)) / loss_scale``, the
    factor to multiply the gradients with; NaN where the norm is not finite, which makes
    the step that reads it change nothing. fp64 sums in a fixed order; no synchronisation."""
    grads = list(grads)
    out = _lib.fast().grad_norm(_lib.address("stm_grad_norm"), _lib.address("stm_grad_norm_workspace_bytes"), grads,
                                max_norm, loss_scale, torch._C._cuda_getCurrentRawStream)
    if isinstance(out, torch.Tensor):
        return out
    if out is not None:
        _lib.check(out, "stm_grad_norm")
    table = np.empty((2, len(grads)), dtype=np.int64)
    addresses, sizes = table[0], table[1]
    while True:
        tag, index, count, bad = _lib.fast().collect(grads, addresses.ctypes.data, 1, 0, sizes.ctypes.data)
        if bad < 0:
            break
        grads[bad] = _plain_gradient(bad, grads)
    if count == 0:
        raise ValueError("grad_norm needs at least one gradient")
    if tag < 0:
        raise ValueError("gradients must be float16, bfloat16 or float32")
    dev = torch.device("cuda", index)
    out = torch.empty(2, dtype=torch.float32, device=dev)
    lib = _lib.lib()
    nbytes = lib.stm_grad_norm_workspace_bytes(len(grads), sizes.ctypes.data)
    ws = torch.empty(nbytes // 8, dtype=torch.float64, device=dev)
    with _lib.device_guard(dev):
        rc = lib.stm_grad_norm(len(grads), addresses.ctypes.data, sizes.ctypes.data, tag, max_norm, loss_scale,
                               out.data_ptr(), ws.data_ptr(), nbytes, _lib.stream_handle(dev))
    _lib.check(rc, "stm_grad_norm")
    return out


def state_codes(values: torch.Tensor, *, signed: bool) -> tuple:
    """(codes uint8 like ``values``, scales fp32 [ceil(numel / 256)]) of an 8-bit state."""
    dev = _gpu(values, "state_codes")
    x = values.detach().to(torch.float32).contiguous()
    codes = torch.empty(x.shape, dtype=torch.uint8, device=dev)
    scales = torch.empty(_blocks(x.numel()), dtype=torch.float32, device=dev)
    with _lib.device_guard(dev):
        rc = _lib.lib().stm_state8_codes(x.data_ptr(), x.numel(), int(signed), codes.data_ptr(), scales.data_ptr(),
                                         _lib.stream_handle(dev))
    _lib.check(rc, "stm_state8_codes")
    return codes, scales


def state_values(codes: torch.Tensor, scales: torch.Tensor, *, signed: bool) -> torch.Tensor:
    """The fp32 values that an 8-bit state stands for, in the shape of ``codes``."""
    dev = _gpu(codes, "state_values")
    n = codes.numel()
    if codes.dtype != torch.uint8:
        raise ValueError(f"codes must be uint8, got {codes.dtype}")
    if scales.dtype != torch.float32 or scales.numel() != _blocks(n) or scales.device != dev:
        raise ValueError(f"scales must hold {_blocks(n)} fp32 values on {dev}")
    c, s = codes.contiguous(), scales.contiguous()
    out = torch.empty(codes.shape, dtype=torch.float32, device=dev)
    with _lib.device_guard(dev):
        rc = _lib.lib().stm_state8_values(c.data_ptr(), s.data_ptr(), n, int(signed), out.data_ptr(),
                                          _lib.stream_handle(dev))
    _lib.check(rc, "stm_state8_values")
    return out


class AdamW(torch.optim.Optimizer):
    """AdamW over parameters on one or several GPUs, a few launches per step.

    ``state_bits`` = 32 or 8; ``master_weights`` keeps an fp32 master of every 16-bit
    parameter, which takes the updates that bf16 or fp16 would round away; an element of a
    parameter that something else wrote between two steps, in place, through ``.data`` or by loading,
    is taken over into its master (the step sees that it is not the master rounded).
    ``max_grad_norm`` clips by the norm over all parameters (of one GPU each). ``grad_norm``
    holds the last norms, one tensor per GPU, still on the device; they are taken without clipping
    too, since a gradient that is not finite makes the step change nothing on its GPU (it still counts as
    a step). With a ``grad_scale`` no norm is taken and that factor alone decides."""

    def __init__(self, params, lr: float = 1e-3, betas: tuple = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, master_weights: bool = False,
                 max_grad_norm: Optional[float] = None):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if lr < 0.0 or eps < 0.0 or weight_decay < 0.0:
            raise ValueError("lr, eps and weight_decay must not be negative")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"betas must lie in [0, 1), got {betas}")
        if max_grad_norm is not None and not max_grad_norm >= 0.0:
            raise ValueError(f"max_grad_norm must not be negative, got {max_grad_norm}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self.state_bits, self.master_weights, self.max_grad_norm = state_bits, master_weights, max_grad_norm
        self.grad_norm: list = []
        self._plans: dict = {}

    def __getstate__(self) -> dict:
        return {**super().__getstate__(), "state_bits": self.state_bits, "master_weights": self.master_weights,
                "max_grad_norm": self.max_grad_norm}

    def __setstate__(self, state: dict) -> None:
        super().__setstate__(state)
        self._plans = {}
        self.__dict__.setdefault("grad_norm", [])

    def _state(self, p: torch.Tensor) -> dict:
        state = self.state[p]
        if "step" not in state:
            state["step"] = 0
            dtype = torch.uint8 if self.state_bits == 8 else torch.float32
            for name in ("exp_avg", "exp_avg_sq"):
                state[name] = torch.zeros(p.shape, dtype=dtype, device=p.device)
                if self.state_bits == 8:
                    state[name + "_scale"] = torch.zeros(_blocks(p.numel()), dtype=torch.float32, device=p.device)
            if self._mastered(p):
                state["master"] = p.detach().to(torch.float32).contiguous()
        return state

    def _mastered(self, p: torch.Tensor) -> bool:
        return self.master_weights and p.dtype != torch.float32

    def _plan(self, key: tuple, params: list) -> AdamWTensors:
        """The checked tensor table of one set of a step's tensors; made again when
        one of them is no longer the same tensor or has moved."""
        states = [self.state[p] for p in params]
        held = [id(t) for s in states for name, t in s.items() if name != "step"]
        plan = self._plans.get(key)
        if plan is None or plan[0] != held or plan[1].at() != [p.data_ptr() for p in params]:
            eight = self.state_bits == 8
            tensors = AdamWTensors(
                [p.detach() for p in params], [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states],
                masters=[s["master"] for s in states] if "master" in states[0] else None,
                scales=([s["exp_avg_scale"] for s in states], [s["exp_avg_sq_scale"] for s in states]) if eight else None,
                follow=True)
            plan = self._plans[key] = (held, tensors)  # which keeps the tensors, so their ids stay theirs
        return plan[1]

    @torch.no_grad()
    def step(self, closure=None, *, grad_scale: Optional[torch.Tensor] = None):
        """One step. ``grad_scale`` (an fp32 scalar on the GPU, as :func:`grad_norm` leaves
        it) multiplies the gradients, in place of ``max_grad_norm``; a step whose factor is
        not finite changes nothing. A captured step repeats its own rate and step number on every
        replay (:meth:`AdamWTensors.step`) and counts once."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # the tensors of one launch: one group, device, types, with masters or without, and step number
        sets: dict = {}
        for gi, group in enumerate(self.param_groups):
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise ValueError("AdamW does not take sparse gradients")
                state = self._state(p)
                key = (gi, p.device, p.dtype, p.grad.dtype, "master" in state, state["step"])
                sets.setdefault(key, []).append(p)
        factors: dict = {}
        if grad_scale is None:
            factors = self._clip(sets)
        alike: dict = {}  # sets that differ in their step number alone, so far
        for (*kind, count), params in sets.items():
            gi, device, kind = kind[0], kind[1], tuple(kind)
            group, place = self.param_groups[gi], alike.setdefault(kind, 0)
            alike[kind] = place + 1
            self._plan((kind, place), params).step(
                [p.grad for p in params], step=count + 1, lr=float(group["lr"]), betas=group["betas"],
                eps=group["eps"], weight_decay=group["weight_decay"],
                grad_scale=grad_scale if grad_scale is not None else factors.get(device))
            for p in params:
                self.state[p]["step"] = count + 1
        return loss

    def _clip(self, sets: dict) -> dict:
        """The clip factor of each GPU, from the norm over all its gradients; 1 without clipping, and
        NaN where the norm is not finite."""
        most = math.inf if self.max_grad_norm is None else self.max_grad_norm
        grads: dict = {}
        for (_, device, _, grad_dtype, _, _), params in sets.items():
            grads.setdefault(device, {}).setdefault(grad_dtype, []).extend(p.grad for p in params)
        self.grad_norm, factors = [], {}
        for device, by_dtype in grads.items():
            norms = [grad_norm(gs, most) for gs in by_dtype.values()]
            if len(norms) == 1:
                norm = norms[0]
            else:  # several gradient types: the norm of their norms
                norm = grad_norm([torch.stack([n[0] for n in norms])], most)
            self.grad_norm.append(norm[0])
            factors[device] = norm[1]
        return factors

    def load_state_dict(self, state_dict: dict) -> None:
        """As torch's, but states keep fp32 or their codes (torch casts them to the parameter's type). A
        checkpoint of other settings, torch's own AdamW among them, is made one of these: its moments
        take ``state_bits``, and masters are made from the parameters, or dropped, as ``master_weights``
        says. Groups that ask for another update (amsgrad, maximize, weight decay in the gradient) are
        refused."""
        loaded: dict = {}  # what the hooks before loading leave of it

        def look(_, given: dict) -> None:
            for group in given["param_groups"]:
                for name in ("amsgrad", "maximize"):
                    if group.get(name):
                        raise ValueError(f"AdamW has no {name}, the state to load asks for it")
                if group.get("weight_decay") and not group.get("decoupled_weight_decay", True):
                    raise ValueError("AdamW's weight decay is decoupled, that of the state to load is not")
            loaded.update(given)
        last = self.register_load_state_dict_pre_hook(look)
        try:
            super().load_state_dict(state_dict)
        finally:
            last.remove()
        state_dict = loaded
        self._plans = {}
        saved = [i for group in state_dict["param_groups"] for i in group["params"]]
        params = [p for group in self.param_groups for p in group["params"]]
        for i, p in zip(saved, params):
            if state_dict["state"].get(i):  # empty: looked at, but never stepped
                self.state[p] = self._taken(p, state_dict["state"][i])

    def _taken(self, p: torch.Tensor, saved: dict) -> dict:
        """The state of *p* from a saved one of any width, with or without a master."""
        missing = [name for name in ("step", "exp_avg", "exp_avg_sq") if name not in saved]
        if missing:
            raise ValueError(f"not the state of an AdamW: {', '.join(missing)} missing")
        state = {"step": int(saved["step"])}
        for name, signed in (("exp_avg", True), ("exp_avg_sq", False)):
            value, scale = saved[name].detach(), saved.get(name + "_scale")
            if value.numel() != p.numel():
                raise ValueError(f"{name} has {value.numel()} elements, its parameter {p.numel()}")
            if self.state_bits == 8 and scale is not None:
                state[name] = value.to(p.device, copy=True).contiguous()
                state[name + "_scale"] = scale.detach().to(p.device, copy=True).contiguous()
            elif self.state_bits == 8:
                state[name], state[name + "_scale"] = state_codes(value.to(p.device), signed=signed)
            elif scale is not None:
                state[name] = state_values(value.to(p.device), scale.detach().to(p.device), signed=signed)
            else:
                state[name] = value.to(p.device, torch.float32, copy=True).contiguous()
        if self._mastered(p):
            master = saved["master"].detach() if "master" in saved else p.detach()
            state["master"] = master.to(p.device, torch.float32, copy=True).contiguous()
        return state
