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


def _plain(what: str, *tensors) -> list:
    """The operands of an operator that has a node of its own: tensors of torch's own class (aliases of a subclass's),
    none of them a forward-mode dual."""
    out = []
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{what} is differentiable in reverse mode only")
        out.append(t if t is None or type(t) in (torch.Tensor, nn.Parameter) else t.as_subclass(torch.Tensor))
    return out


def _check(x, weight, eps, residual) -> None:
    if not x.is_cuda:
        raise RuntimeError("rms_norm runs on the GPU kernels; its operands must be on the GPU")
    _lib.dtype_tag(x.dtype)
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


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None):
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension, in x's dtype (bf16, fp16 or fp32).

    With ``residual`` (x's shape; x's dtype or fp32) the rows are ``h = x + residual``, and the result is
    ``(y, h)``, h in the residual's dtype: y comes from the sum in 32 bits, each output is rounded once.
    ``weight``: [columns] in x's dtype or fp32. Differentiable in x, the residual and the weight (reverse
    mode, once); the weight's gradient is a sum in a fixed order. Kept for the backward: h (x without a residual; x and
    the residual where h has 16 bits: the gradients are those of the sum, and do not depend on which of them are asked
    for) and 4 bytes a row."""
    out = _lib.sparse().norm(x, weight, eps, residual)
    if out is None:  # an operand to refuse or to convert, or another device than the current one
        _check(x, weight, eps, residual)
        x, weight, residual = _plain("rms_norm", x, weight, residual)
        with _lib.device_guard(x.device):
            out = _lib.taken("rms_norm", _lib.sparse().norm(x, weight, eps, residual))
    return out


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
