"""Layer norm on the MI355X kernels: the norm in front of a low-bit Linear, a
router or the expert loop, which the DeepSeek-V3 recipe keeps in high
precision (precision.py).

layer_norm() is the operator with its gradients; LayerNorm is the module
(src/layers.py:639-781 of nano-train).  Statistics and sums are fp32 whatever
the input's type; outputs and gradients are rounded once.
"""

from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib
from . import ops

MAX_WIDTH = 16384


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x as [T, H] with unit stride along H and rows that lie one behind the
    other (or are one row repeated): a copy only where no view gives that"""
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if x2.stride(1) != 1 or (x2.stride(0) != 0 and x2.stride(0) < x2.shape[1]):
        x2 = x2.contiguous()
    return x2


def _wdtype(x2, weight, bias) -> int:
    return ops._dtype_code((weight if weight is not None else bias if bias is not None else x2).dtype)


def _forward(x2: torch.Tensor, weight, bias, eps: float, stats: bool):
    """y and, for the backward, the rows' means and then their 1 / deviations in one tensor"""
    T, H = x2.shape
    y = torch.empty((T, H), dtype=x2.dtype, device=x2.device)
    mr = torch.empty(2 * T, dtype=torch.float32, device=x2.device) if stats else None
    at = mr.data_ptr() if stats else 0
    _lib.call("ntlb_layer_norm_forward", x2.data_ptr(), ops._dtype_code(x2.dtype), T, H, x2.stride(0),
              ops._ptr(weight), ops._ptr(bias), _wdtype(x2, weight, bias), eps, y.data_ptr(), H, at or None,
              at + 4 * T if at else None, ops._stream())
    return y, mr


def _backward(ctx, dy):
    x2, weight, bias, mr = ctx.saved_tensors
    T, H = x2.shape
    dev = x2.device
    d2 = _rows(dy)
    want_x, want_w, want_b = ctx.needs_input_grad[:3]
    dx = torch.empty((T, H), dtype=x2.dtype, device=dev) if want_x else None
    dw = torch.empty_like(weight) if want_w else None
    db = torch.empty_like(bias) if want_b else None
    xc = ops._dtype_code(x2.dtype)
    ws, need = None, 0
    if want_w or want_b:
        need = _lib.lib().ntlb_layer_norm_workspace_bytes(xc, T, H)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
    at = mr.data_ptr()
    _lib.call("ntlb_layer_norm_backward", x2.data_ptr(), xc, T, H, x2.stride(0), d2.data_ptr(), d2.stride(0), at,
              at + 4 * T, ops._ptr(weight), _wdtype(x2, weight, bias), ops._ptr(dx), H, ops._ptr(dw), ops._ptr(db),
              ops._ptr(ws), need, ops._stream())
    if want_x and dx.shape != ctx.shape:
        dx = dx.reshape(ctx.shape)
    return dx, dw, db, None


_backward_of_graph = once_differentiable(_backward)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x2 = _rows(x)
        y, mr = _forward(x2, weight, bias, eps, True)
        ctx.save_for_backward(x2, weight, bias, mr)
        ctx.shape = x.shape
        return y if x.dim() == 2 else y.reshape(x.shape)

    @staticmethod
    def backward(ctx, dy):
        # a gradient that is itself to be differentiated is refused there
        return (_backward_of_graph if torch.is_grad_enabled() else _backward)(ctx, dy)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
               eps: float = 1e-5) -> torch.Tensor:
    """y = (x - mean) / sqrt(var + eps) * weight + bias over the last axis of x
    [..., H], with the gradients of x, weight and bias under autograd.

    x bf16, fp16 or fp32 with rows of any pitch; weight and bias [H] (either
    may be None) share one of these types, which may differ from x's.  H <=
    16384.  The gradients of weight and bias are summed in a fixed order."""
    ops._require_device(x, weight, bias)
    if x.dim() < 1:
        raise ValueError("x must be [..., H]")
    H = x.shape[-1]
    if not 1 <= H <= MAX_WIDTH:
        raise ValueError(f"layer_norm takes rows of 1 to {MAX_WIDTH} elements, not {H}")
    ops._dtype_code(x.dtype)
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        ops._dtype_code(t.dtype)
        if t.shape != (H,):
            raise ValueError(f"{name} must be [{H}], not {tuple(t.shape)}")
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight and bias must share a dtype, not {weight.dtype} and {bias.dtype}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    weight = weight if weight is None or weight.stride(0) == 1 else weight.contiguous()
    bias = bias if bias is None or bias.stride(0) == 1 else bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _forward(_rows(x), weight, bias, float(eps), False)[0].reshape(x.shape)


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
