"""Layer norm and root-mean-square norm on the MI355X kernels: a norm in front of
a low-bit Linear, a router or the expert loop.  The recipe's patterns keep every
norm in high precision (precision.py); these are nano-train's LayerNorm
(src/layers.py:639-781) and its DeepSeek model's RMSNorm.

layer_norm() and rms_norm() are the operators with their gradients, LayerNorm and
RMSNorm the modules; rms_norm_quant() gives the norm in 8 bits, as the low-bit
products take it.  Statistics and sums are fp32 whatever the input's type;
outputs and gradients are rounded once.
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


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, *, residual: Optional[torch.Tensor] = None,
             eps: float = 1e-6, checkpoint: Optional[str] = None):
    """y = s / sqrt(mean(s^2) + eps) * weight over the last axis of s = x +
    residual [..., H]: y without a residual, else (y, s), s rounded to x's type and
    the norm that of the rounded s.  With the gradients of x, weight and residual
    under autograd (s may be differentiated too).

    x bf16, fp16 or fp32 with rows of any pitch, residual of its type and shape;
    weight [H] of one of these types, or None.  H <= 16384.  The gradient of weight
    is summed in a fixed order.

    checkpoint None keeps s for the backward; "e4m3" keeps it in 8 bits (a power of
    two for each 128 columns, values rounded by at most 2^-4 of themselves where
    they are not 2^-14 of the tile's largest or less), and the gradients are those
    of the norm at the values kept, with the deviations of the true ones.  A
    value that is not finite is kept as NaN."""
    weight, keep = _check_rms("rms_norm", x, weight, residual, eps), ops.checkpoint_code(checkpoint)
    return (_lib._autograd or _lib.autograd()).rms_norm(x, weight, residual, eps, keep)


def rms_norm_quant(x: torch.Tensor, weight: Optional[torch.Tensor] = None, *, residual: Optional[torch.Tensor] = None,
                   eps: float = 1e-6, fmt: str = "e4m3", want_nan_rows: bool = False):
    """rms_norm() with y in 8 bits: a QTensor of [rows, H] (leading axes flattened,
    a scale for each 128 columns of a row, tile-major), or (QTensor, s) with a
    residual.  ops.gemm_blockscaled and moe.expert_mlp take it as it is.

    Codes and scales are laid out as those of ops.quant_tile_1x128 (fmt "e4m3" or
    "int_grid", 8 bits, round to nearest) and are of y's own value, rounded once: where y
    lies in the middle of two codes, the even one.  They have no gradient: where one
    is being recorded for x, weight or residual, the call is refused.  want_nan_rows
    as for ops.quant_tile_1x128 (the int grid needs it to carry a NaN on)."""
    weight = _check_rms("rms_norm_quant", x, weight, residual, eps)
    grid = ops.grid_code(fmt)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise RuntimeError("rms_norm_quant has no gradient: call it under torch.no_grad(), or rms_norm in training")
    codes, scales, nan, s = (_lib._autograd or _lib.autograd()).rms_norm_quant(x, weight, residual, eps, grid,
                                                                               int(want_nan_rows))
    q = ops.QTensor(codes, scales, 1, scales.shape[1], 0, grid, codes.shape[0], x.shape[-1], nan, None)
    return q if residual is None else (q, s)


def _check_rms(fn: str, x: torch.Tensor, weight, residual, eps: float):
    if not x.is_cuda:
        ops._require_device(x)
    dt = x.dtype
    if dt not in _DTYPES:
        ops._dtype_code(dt)
    H = x.shape[-1] if x.dim() else 0
    if not 1 <= H <= MAX_WIDTH:
        raise ValueError(f"{fn} takes [..., H] with rows of 1 to {MAX_WIDTH} elements, not {tuple(x.shape)}")
    if residual is not None:
        if residual.dtype != dt:
            raise TypeError(f"residual is {residual.dtype}, x {dt}")
        if residual.shape != x.shape:
            raise ValueError(f"residual must be {tuple(x.shape)}, not {tuple(residual.shape)}")
        if residual.device != x.device:
            raise ValueError(f"residual is on {residual.device}, x on {x.device}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    return _check_weight("weight", weight, x, H) if weight is not None else None


class RMSNorm(nn.Module):
    """Root-mean-square norm over the last axis: forward(x) is y, forward(x,
    residual) is (y, x + residual)."""

    def __init__(self, hidden_size: int, eps: float = 1e-6, *, checkpoint: Optional[str] = None,
                 dtype: Optional[torch.dtype] = None, device=None):
        super().__init__()
        ops.checkpoint_code(checkpoint)
        self.hidden_size, self.eps, self.checkpoint = hidden_size, eps, checkpoint
        self.weight = nn.Parameter(torch.ones(hidden_size, dtype=dtype, device=device))

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        return rms_norm(x, self.weight, residual=residual, eps=self.eps, checkpoint=self.checkpoint)

    def extra_repr(self) -> str:
        return f"{self.hidden_size}, eps={self.eps}" + (f", checkpoint={self.checkpoint!r}" if self.checkpoint else "")
