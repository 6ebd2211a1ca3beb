"""Layer norm on the MI355X kernels: a norm in front of a low-bit Linear, a
router or the expert loop.  The recipe's patterns keep every norm in high
precision (precision.py); this one is nano-train's LayerNorm
(src/layers.py:639-781).  Its DeepSeek model has RMSNorm, another operator.

layer_norm() is the operator with its gradients; LayerNorm is the module.
Statistics and sums are fp32 whatever the input's type; outputs and gradients
are rounded once.
"""

from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from . import _lib
from . import ops

MAX_WIDTH = 16384
_DTYPES = frozenset(ops._DTYPE_CODE)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
               eps: float = 1e-5) -> torch.Tensor:
    """y = (x - mean) / sqrt(var + eps) * weight + bias over the last axis of x
    [..., H], with the gradients of x, weight and bias under autograd.

    x bf16, fp16 or fp32 with rows of any pitch; weight and bias [H] (either
    may be None) share one of these types, which may differ from x's.  H <=
    16384.  The gradients of weight and bias are summed in a fixed order."""
    if not x.is_cuda:
        ops._require_device(x)
    dt = x.dtype
    if dt not in _DTYPES:
        ops._dtype_code(dt)
    H = x.shape[-1] if x.dim() else 0
    if not 1 <= H <= MAX_WIDTH:
        raise ValueError(f"layer_norm takes [..., H] with rows of 1 to {MAX_WIDTH} elements, not {tuple(x.shape)}")
    weight = _check_weight("weight", weight, x, H) if weight is not None else None
    bias = _check_weight("bias", bias, x, H) if bias is not None else None
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight and bias must share a dtype, not {weight.dtype} and {bias.dtype}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    return (_lib._autograd or _lib.autograd()).layer_norm(x, weight, bias, eps)


def _check_weight(name: str, t: torch.Tensor, x: torch.Tensor, H: int) -> torch.Tensor:
    if t.dtype not in _DTYPES:
        ops._dtype_code(t.dtype)
    if t.dim() != 1 or t.shape[0] != H:
        raise ValueError(f"{name} must be [{H}], not {tuple(t.shape)}")
    if t.device != x.device:
        raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    return t if t.stride(0) == 1 else t.contiguous()


class LayerNorm(nn.Module):
    """Layer norm over the last axis (src/layers.py:639-781)."""

    def __init__(self, hidden_size: int, eps: float = 1e-5, *, dtype: Optional[torch.dtype] = None, device=None):
        super().__init__()
        self.hidden_size = hidden_size
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(hidden_size, dtype=dtype, device=device))
        self.bias = nn.Parameter(torch.zeros(hidden_size, dtype=dtype, device=device))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, eps=self.eps)

    def extra_repr(self) -> str:
        return f"{self.hidden_size}, eps={self.eps}"
