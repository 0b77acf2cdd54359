"""Root-mean-square norm with the residual's addition, as one operator with its gradients.

A decoder layer adds a branch to its residual stream and normalises the sum for the next branch. The
reference leaves both to transformers' modules (``stratum/model/qwen3.py``, ``stratum/model/llama.py``);
here they are one pass over the rows in each direction.
"""

from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
from torch.autograd import forward_ad

from . import _lib
from .functional import _on_device

__all__ = ["RMSNorm", "rms_norm"]


def _norm_operands(x, weight, eps, residual):
    """Checked operands, contiguous: (type, x, residual, weight)."""
    tag = _lib.dtype_tag(x.dtype)
    if not x.is_cuda:
        raise RuntimeError("rms_norm runs on the GPU kernels; its operands must be on the GPU")
    if x.dim() < 1:
        raise ValueError("rms_norm takes rows, got a scalar")
    cols = int(x.shape[-1])
    if tuple(weight.shape) != (cols,):
        raise ValueError(f"weight has shape {tuple(weight.shape)}, x has {cols} columns")
    if weight.dtype not in (x.dtype, torch.float32):
        raise ValueError(f"weight must be {x.dtype} or float32, got {weight.dtype}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    _on_device(x.device, weight=weight, residual=residual)
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"residual has shape {tuple(residual.shape)}, x has {tuple(x.shape)}")
        if residual.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"residual must be {x.dtype} or float32, got {residual.dtype}")
    return tag, x.contiguous(), residual.contiguous() if residual is not None else None, weight.contiguous()


def _size(t: torch.Tensor) -> tuple:
    """(rows, columns)."""
    cols = int(t.shape[-1])
    return (t.numel() // cols if cols else 0), cols


def _norm_fwd(x, weight, eps, residual, keep):
    """(y, h or None, rstd or None)."""
    tag, x2, r2, w = _norm_operands(x, weight, eps, residual)
    rows, cols = _size(x)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    h = torch.empty(x.shape, dtype=residual.dtype, device=x.device) if residual is not None else None
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device) if keep else None
    with _lib.device_guard(x.device):
        rc = _lib.lib().stm_rms_norm_fwd(
            x2.data_ptr(), r2.data_ptr() if r2 is not None else None, _lib.dtype_tag(r2.dtype) if r2 is not None else tag,
            w.data_ptr(), _lib.dtype_tag(w.dtype), y.data_ptr(), h.data_ptr() if h is not None else None,
            rstd.data_ptr() if keep else None, rows, cols, float(eps), tag, _lib.stream_handle(x.device))
    _lib.check(rc, "stm_rms_norm_fwd")
    return y, h, rstd


class _RMSNormFn(torch.autograd.Function):
    """Kept for the backward: h (x without a residual), the weight and 1 / rms of every row."""

    @staticmethod
    def forward(ctx, x, weight, eps, residual):
        y, h, rstd = _norm_fwd(x, weight, eps, residual, True)
        ctx.set_materialize_grads(False)
        ctx.dtype = x.dtype
        ctx.save_for_backward(x if h is None else h, weight, rstd)
        return y if h is None else (y, h)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight, rstd = ctx.saved_tensors
        need_x, need_w, _, need_r = ctx.needs_input_grad
        if dy is None:  # only the sum went on
            return (dh.to(ctx.dtype) if need_x and dh is not None else None), None, None, dh if need_r else None
        dev, tag = dy.device, _lib.dtype_tag(dy.dtype)
        d2, h2, w = dy.contiguous(), h.contiguous(), weight.contiguous()
        e2 = dh.contiguous() if dh is not None else None
        rows, cols = _size(dy)
        apart = need_r and h.dtype != dy.dtype
        dx = torch.empty(dy.shape, dtype=dy.dtype, device=dev) if need_x or (need_r and not apart) else None
        dr = torch.empty(dy.shape, dtype=h.dtype, device=dev) if apart else None
        dw = torch.empty(weight.shape, dtype=weight.dtype, device=dev) if need_w else None
        ws = None
        if need_w:
            nbytes = int(_lib.lib().stm_rms_norm_workspace_bytes(rows, cols))
            if nbytes < 0:
                _lib.check(nbytes, "stm_rms_norm_workspace_bytes")
            ws = torch.empty(nbytes // 4, dtype=torch.float32, device=dev)
        ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
        with _lib.device_guard(dev):
            rc = _lib.lib().stm_rms_norm_bwd(
                d2.data_ptr(), ptr(e2), h2.data_ptr(), _lib.dtype_tag(h.dtype), rstd.data_ptr(), w.data_ptr(),
                _lib.dtype_tag(w.dtype), ptr(dx), ptr(dr), ptr(dw), rows, cols, tag, ptr(ws),
                4 * ws.numel() if ws is not None else 0, _lib.stream_handle(dev))
        _lib.check(rc, "stm_rms_norm_bwd")
        return dx if need_x else None, dw, None, (dr if apart else dx) if need_r else None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None):
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension, in x's dtype (bf16, fp16 or fp32).

    With ``residual`` (x's shape; x's dtype or fp32) the rows are ``h = x + residual``, and the result is
    ``(y, h)``, h in the residual's dtype: y comes from the sum in 32 bits, each output is rounded once.
    ``weight``: [columns] in x's dtype or fp32. Differentiable in x, the residual and the weight (reverse
    mode; a forward-mode dual is refused); the weight's gradient is a sum in a fixed order. Kept for the
    backward: h (x without a residual) and 4 bytes a row."""
    grad = torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                        (residual is not None and residual.requires_grad))
    if not grad and all(t is None or forward_ad.unpack_dual(t).tangent is None for t in (x, weight, residual)):
        with torch.no_grad():
            y, h, _ = _norm_fwd(x, weight, eps, residual, False)
        return y if residual is None else (y, h)
    return _RMSNormFn.apply(x, weight, eps, residual)


class RMSNorm(nn.Module):
    """:func:`rms_norm` with a weight of its own: ``norm(x)``, or ``norm(x, residual)`` -> (y, h)."""

    def __init__(self, hidden: int, eps: float = 1e-6, dtype: Optional[torch.dtype] = None, device=None):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(hidden, dtype=dtype, device=device))

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        return rms_norm(x, self.weight, self.eps, residual)

    def extra_repr(self) -> str:
        return f"{self.weight.shape[0]}, eps={self.eps}"
