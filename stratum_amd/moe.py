"""The operators around the experts' products of a sparse layer, and the layer's feed-forward half.

``nf4_grouped_gemm`` computes the experts' products on a bank of NF4 weights from rows that lie in the experts'
order. Here is what comes before and after it:

* :func:`moe_route`: every token's experts and their weights, from the router's logits;
* :func:`moe_sort`: the order of the rows by expert (:class:`MoEOrder`);
* :func:`moe_gather`: the tokens' rows in that order;
* :func:`moe_combine`: the experts' rows back to their tokens, weighted, plus the residual.

:class:`NF4MoE` runs them around an NF4 expert bank, with the norm and the residual's addition before.
The reference runs transformers' ``Qwen3MoeExperts`` and router there (``stratum/model/qwen3_moe.py``,
``stratum/moe.py``). None of the four reads anything back to the host; all can be captured into a graph, with their
gradients too, on as many streams as take part in the capture. A captured gradient that would go on from one of them to a
leaf that an eager graph on the default stream holds is refused (capture on leaves of its own:
``t.detach().requires_grad_()``).
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch
import torch.nn as nn

from . import _lib
from .functional import (_on_device, _rows, fused_supported, nf4_grouped_gemm, quantize_4bit, swiglu_bwd,
                         swiglu_fwd)
from .norm import _plain

__all__ = ["MoEOrder", "NF4MoE", "moe_combine", "moe_gather", "moe_route", "moe_sort"]

SCORES = {"softmax": 0, "sigmoid": 1}
GROUP_SCORES = {"max": 0, "top2": 1}
MAX_EXPERTS, MAX_TOP_K, MAX_GROUPS = 1024, 64, 64


class MoEOrder(NamedTuple):
    """The slots (token t, its j-th expert) of a batch in the order of their experts; int32 on the GPU."""

    offsets: torch.Tensor    # [experts + 1]: rows offsets[e] .. offsets[e + 1] are expert e's
    slots: torch.Tensor      # [n]: the slot t * top_k + j of a row; -1 from offsets[-1] on
    positions: torch.Tensor  # [..., top_k]: the row of a slot; -1 for a slot without an expert


def _gpu(t: torch.Tensor, what: str) -> torch.device:
    if not t.is_cuda:
        raise RuntimeError(f"{what} runs on the GPU kernels; its operands must be on the GPU")
    return t.device


def _slots(what: str, n: int) -> None:
    if n >= 1 << 31:
        raise ValueError(f"{what}: {n} slots are too many (2^31 - 1)")


# ------------------------------------------------------------ route
def _check_route(logits, bias, mask, top_k, groups, top_groups) -> None:
    dev = _gpu(logits, "moe_route")
    _lib.dtype_tag(logits.dtype)
    if logits.dim() < 1:
        raise ValueError("logits must be [..., experts]")
    E, lead = int(logits.shape[-1]), tuple(logits.shape[:-1])
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"1 to {MAX_EXPERTS} experts, got {E}")
    if not 1 <= top_k <= min(E, MAX_TOP_K):
        raise ValueError(f"top_k must be from 1 to min(experts, {MAX_TOP_K}), got {top_k} of {E} experts")
    if not 1 <= groups <= MAX_GROUPS or E % groups:
        raise ValueError(f"{E} experts do not make {groups} groups (1 to {MAX_GROUPS})")
    if not 1 <= top_groups <= groups:
        raise ValueError(f"top_groups must be from 1 to {groups}, got {top_groups}")
    if top_k > E // groups * top_groups:
        raise ValueError(f"{top_groups} groups of {E // groups} hold fewer than {top_k} experts")
    _on_device(dev, bias=bias, mask=mask)
    if bias is not None and (tuple(bias.shape) != (E,) or bias.dtype != torch.float32):
        raise ValueError(f"bias must be float32 [{E}], got {bias.dtype} {tuple(bias.shape)}")
    if mask is not None and (tuple(mask.shape) != lead or mask.dtype != torch.bool):
        raise ValueError(f"mask must be bool {lead}, got {mask.dtype} {tuple(mask.shape)}")
    _slots("moe_route", logits.numel() // E * top_k)


def moe_route(logits: torch.Tensor, top_k: int, *, score: str = "softmax", bias: Optional[torch.Tensor] = None,
              groups: int = 1, top_groups: int = 1, group_score: str = "max", renormalize: bool = True,
              scale: float = 1.0, mask: Optional[torch.Tensor] = None) -> tuple:
    """``(weights float32 [..., top_k], experts int32 [..., top_k])`` of the tokens whose router logits are
    ``logits`` [..., experts] (bf16, fp16 or fp32; at most 1024 experts, ``top_k`` at most 64).

    The scores are the logits' softmax or sigmoid. A token's experts are those of the ``top_k`` largest keys, in
    descending order, the lowest index first among equal ones. The key is the logit itself (the scores are in its
    order), or with ``bias`` (float32 [experts], for balance; it chooses and does not weigh) or sums over groups score
    + bias, computed in 64 bits. With ``groups`` > 1 (equal stretches of the experts, at most 64) only experts of
    the ``top_groups`` best ones are eligible, by their largest key (``group_score="max"``) or the sum of their two
    largest (``"top2"``). A weight is the expert's score, divided by the sum of the token's chosen scores
    (``renormalize``), times ``scale``.

    ``mask`` (bool [...]) is False for tokens that take no part: their experts are -1, their weights 0 and
    nothing of their logits matters. An expert whose logit (or key) is -inf is never chosen; slots left over hold
    -1 and 0 too. Differentiable in the logits through the weights (reverse mode, once), not in the bias."""
    if score not in SCORES:
        raise ValueError(f"score must be one of {sorted(SCORES)}, got {score!r}")
    if group_score not in GROUP_SCORES:
        raise ValueError(f"group_score must be one of {sorted(GROUP_SCORES)}, got {group_score!r}")
    rest = (top_k, SCORES[score], groups, top_groups, GROUP_SCORES[group_score], bool(renormalize), scale)
    out = _lib.sparse().route(logits, bias, mask, *rest)
    if out is None:  # an operand to refuse or to convert, or another device than the current one
        _check_route(logits, bias, mask, top_k, groups, top_groups)
        logits, bias, mask = _plain("moe_route", logits, bias, mask)
        with _lib.device_guard(logits.device):
            out = _lib.taken("moe_route", _lib.sparse().route(logits, bias, mask, *rest))
    return out


# ------------------------------------------------------------ rows by expert
def moe_sort(experts: torch.Tensor, num_experts: int) -> MoEOrder:
    """The order by expert of the slots ``experts`` (int32 [..., top_k], as :func:`moe_route` gives them): rows of one
    expert keep the slots' order. A slot whose value is not in 0 .. num_experts - 1 (-1) gets no row; as many rows at the
    end stay without a slot. At most 1024 experts."""
    out = _lib.sparse().sort(experts, num_experts)
    if out is None:
        dev = _gpu(experts, "moe_sort")
        if experts.dtype != torch.int32 or experts.dim() < 1:
            raise ValueError(f"experts must be int32 [..., top_k], got {experts.dtype} {tuple(experts.shape)}")
        if not 1 <= num_experts <= MAX_EXPERTS:
            raise ValueError(f"1 to {MAX_EXPERTS} experts, got {num_experts}")
        _slots("moe_sort", experts.numel())
        (experts,) = _plain("moe_sort", experts)
        with _lib.device_guard(dev):
            out = _lib.taken("moe_sort", _lib.sparse().sort(experts, num_experts))
    return MoEOrder(*out)


def _check_order(order: MoEOrder, dev: torch.device) -> tuple:
    """(tokens, top_k) of an order on *dev*."""
    offsets, slots, positions = order
    for name, t in (("offsets", offsets), ("slots", slots), ("positions", positions)):
        if t.dtype != torch.int32 or t.device != dev or not t.is_contiguous():
            raise ValueError(f"order.{name} must be contiguous int32 on {dev}, got {t.dtype} on {t.device}")
    if positions.dim() < 1 or positions.shape[-1] < 1 or slots.numel() != positions.numel() or offsets.numel() < 2:
        raise ValueError("order must be that of moe_sort, of at least one slot a token")
    top_k = int(positions.shape[-1])
    return positions.numel() // top_k, top_k


def moe_gather(x: torch.Tensor, order: MoEOrder) -> torch.Tensor:
    """The rows of ``x`` [..., hidden] in the order ``order`` of its slots: [tokens * top_k, hidden], row p the row of
    slot ``order.slots[p]``'s token, zeros where there is no slot. Differentiable in x (reverse mode, once): the
    gradient of a token is the sum, in 32 bits, over its slots."""
    out = _lib.sparse().gather(x, order)
    if out is None:
        dev = _gpu(x, "moe_gather")
        _lib.dtype_tag(x.dtype)
        tokens, _ = _check_order(order, dev)
        if x.dim() < 2 or x.numel() != tokens * x.shape[-1]:
            raise ValueError(f"x must hold [{tokens}, hidden], got {tuple(x.shape)}")
        x, *order = _plain("moe_gather", x, *order)
        with _lib.device_guard(dev):
            out = _lib.taken("moe_gather", _lib.sparse().gather(x, tuple(order)))
    return out


def _check_combine(y, weights, order, residual) -> None:
    dev = _gpu(y, "moe_combine")
    _lib.dtype_tag(y.dtype)
    tokens, top_k = _check_order(order, dev)
    _on_device(dev, weights=weights, residual=residual)
    if y.dim() != 2 or y.shape[0] > tokens * top_k:
        raise ValueError(f"y must be [rows, hidden] of at most {tokens * top_k} rows, got {tuple(y.shape)}")
    if weights.shape != order.positions.shape or weights.dtype != torch.float32:
        raise ValueError(f"weights must be float32 {tuple(order.positions.shape)}, got {weights.dtype} "
                         f"{tuple(weights.shape)}")
    hidden = int(y.shape[1])
    if residual is not None and (residual.dtype not in (y.dtype, torch.float32) or residual.numel() != tokens * hidden
                                 or residual.shape[-1:] != y.shape[1:]):
        raise ValueError(f"residual must be {y.dtype} or float32 [{tokens}, {hidden}], got {residual.dtype} "
                         f"{tuple(residual.shape)}")


def moe_combine(y: torch.Tensor, weights: torch.Tensor, order: MoEOrder,
                residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``residual[t] + sum over j of weights[t, j] * y[order.positions[t, j]]`` for every token, in the residual's dtype
    (y's without one): fp32 sums, one rounding. ``y`` [rows, hidden] holds the experts' rows in ``order``, all of them or
    the first ``order.offsets[-1]``; ``weights`` is float32 [..., top_k]; ``residual`` (optional) [..., hidden], in y's dtype
    or float32, gives the result its shape. A slot without a row adds nothing, whatever its weight. Differentiable in
    y, the weights and the residual (reverse mode, once); rows of y that no slot has get a gradient of zeros."""
    out = _lib.sparse().combine(y, weights, order, residual)
    if out is None:
        _check_combine(y, weights, order, residual)
        y, weights, residual, *order = _plain("moe_combine", y, weights, residual, *order)
        with _lib.device_guard(y.device):
            out = _lib.taken("moe_combine", _lib.sparse().combine(y, weights, tuple(order), residual))
    return out


# ------------------------------------------------------------ the layer's feed-forward half
class _ExpertsFn(torch.autograd.Function):
    """down(silu(gate) * up) of every expert's rows on frozen NF4 banks; kept for the backward: the gate and up
    projections' outputs."""

    @staticmethod
    def forward(ctx, rows, gate_up, gate_up_absmax, down, down_absmax, offsets, inter, blocksize):
        H = int(rows.shape[1])
        gu = nf4_grouped_gemm(rows, gate_up, gate_up_absmax, offsets, (2 * inter, H), blocksize)
        y = nf4_grouped_gemm(swiglu_fwd(gu), down, down_absmax, offsets, (H, inter), blocksize)
        if ctx.needs_input_grad[0]:
            ctx.save_for_backward(gu, gate_up, gate_up_absmax, down, down_absmax)
            ctx.offsets, ctx.inter, ctx.blocksize = offsets, inter, blocksize
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        gu, gate_up, gate_up_absmax, down, down_absmax = ctx.saved_tensors
        H, inter, bs = int(grad.shape[1]), ctx.inter, ctx.blocksize
        dh = nf4_grouped_gemm(grad, down, down_absmax, ctx.offsets, (H, inter), bs, backward=True)
        dx = nf4_grouped_gemm(swiglu_bwd(dh, gu), gate_up, gate_up_absmax, ctx.offsets, (2 * inter, H), bs, backward=True)
        return dx, None, None, None, None, None, None, None


class NF4MoE(nn.Module):
    """The sparse feed-forward half of a decoder layer on frozen NF4 expert banks:

        h = x + residual,  y = norm(h),  out = h + sum over a token's experts of w_e * down_e(silu(gate_e y) * up_e y)

    ``router`` maps rows [tokens, H] to logits [tokens, E] (an ``nn.Linear``); ``gate_up`` and ``down`` are
    ``(packed, QuantState)`` of the stacked banks [E, 2 I, H] ([gate; up] of each expert) and [E, H, I], as
    ``quantize_4bit`` makes them from 3-D weights. ``norm`` is an :class:`~stratum_amd.norm.RMSNorm` or None (y = x; out
    then has the residual added if one is given, and nothing else). The remaining arguments are those of
    :func:`moe_route`; ``bias`` becomes a float32 buffer, which ``.to(dtype)`` and ``.half()`` leave in 32 bits.

    Differentiable in x, the residual, the norm's weight and the router's parameters. The experts' row counts are read
    back once per call (the products' launch needs them)."""

    def __init__(self, router: nn.Module, gate_up: tuple, down: tuple, top_k: int, *, norm: Optional[nn.Module] = None,
                 score: str = "softmax", bias: Optional[torch.Tensor] = None, groups: int = 1, top_groups: int = 1,
                 group_score: str = "max", renormalize: bool = True, scale: float = 1.0):
        super().__init__()
        (gq, gs), (dq, ds) = gate_up, down
        if len(gs.shape) != 3 or len(ds.shape) != 3:
            raise ValueError("gate_up and down must be quantized from [E, 2 I, H] and [E, H, I] weights")
        E, two_i, H = (int(d) for d in gs.shape)
        if tuple(ds.shape) != (E, H, two_i // 2) or two_i % 2:
            raise ValueError(f"gate_up {tuple(gs.shape)} and down {tuple(ds.shape)} do not fit each other")
        if gs.blocksize != ds.blocksize:
            raise ValueError("gate_up and down must share one blocksize")
        if not (fused_supported(two_i, H, gs.blocksize, backward=True)
                and fused_supported(H, two_i // 2, gs.blocksize, backward=True)):
            raise ValueError(f"experts of [{two_i}, {H}], blocksize {gs.blocksize}: unsupported widths")
        self.num_experts, self.hidden, self.inter, self.blocksize = E, H, two_i // 2, gs.blocksize
        # plain attributes, as NF4Linear's: .to(dtype) and .half() leave the fp32 scales alone
        self.gate_up_packed, self.gate_up_absmax = gq.reshape(-1), gs.absmax.reshape(-1).float()
        self.down_packed, self.down_absmax = dq.reshape(-1), ds.absmax.reshape(-1).float()
        self.router, self.norm, self.top_k = router, norm, int(top_k)
        self.register_buffer("bias", bias.detach().float() if bias is not None else None)
        self.route = {"score": score, "groups": groups, "top_groups": top_groups, "group_score": group_score,
                      "renormalize": renormalize, "scale": scale}

    @classmethod
    def quantize(cls, router: nn.Module, gate_up: torch.Tensor, down: torch.Tensor, top_k: int, *, blocksize: int = 64,
                 **kwargs) -> "NF4MoE":
        """From dense banks [E, 2 I, H] and [E, H, I] (on the GPU, or copied there)."""
        def bank(w):
            return quantize_4bit(w.detach().to(w.device if w.is_cuda else "cuda"), blocksize=blocksize)
        return cls(router, bank(gate_up), bank(down), top_k, **kwargs)

    def experts(self, rows: torch.Tensor, order: MoEOrder) -> torch.Tensor:
        """The experts' outputs for *rows* in *order*: the first ``order.offsets[-1]`` of them."""
        offsets = order.offsets.cpu()  # the call's one synchronisation
        live = int(offsets[-1])
        if live != rows.shape[0]:
            rows = rows[:live]
        if live == 0:
            return rows
        return _ExpertsFn.apply(rows, self.gate_up_packed, self.gate_up_absmax, self.down_packed, self.down_absmax, offsets,
                                self.inter, self.blocksize)

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None,
                mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``x`` [..., H]; ``residual`` of its shape is added first; ``mask`` (bool [...]) is False for padding."""
        y, h = x, residual
        if self.norm is not None:
            y, h = (self.norm(x), x) if residual is None else self.norm(x, residual)
        rows = _rows(y, self.hidden)
        logits = self.router(rows)
        weights, experts = moe_route(logits, self.top_k, mask=mask.reshape(-1) if mask is not None else None,
                                     bias=self.bias.float() if self.bias is not None else None, **self.route)
        order = moe_sort(experts, self.num_experts)
        out = self.experts(moe_gather(rows, order), order)
        stream = _rows(h, self.hidden) if h is not None else None
        return moe_combine(out, weights, order, stream).reshape(x.shape)

    def _apply(self, fn, recurse=True):
        bias = self.bias
        super()._apply(fn, recurse)
        if bias is not None and self.bias.dtype != torch.float32:  # .to(dtype), .half(): it moves and stays as exact
            self.bias = bias.float().to(self.bias.device)
        return self

    def extra_repr(self) -> str:
        return (f"{self.num_experts} experts of [{self.hidden}, {self.inter}], top {self.top_k}, "
                f"nf4 blocksize={self.blocksize}, {self.route}")
