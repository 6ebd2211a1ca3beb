"""The language-model head's loss on the MI355X kernels: the product with the
vocabulary's weights, the softmax cross entropy and their gradients in one
operator, which never holds the logits of all words (the LM head is one of
the DeepSeek-V3 recipe's high-precision modules, precision.py).

linear_cross_entropy() is the operator; LMHeadLoss is the module.
"""

from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib
from . import ops
from .norm import _rows

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def _forward(x2, w, targets, ignore_index: int, reduction: int):
    T, H = x2.shape
    V = w.shape[0]
    L = _lib.lib()
    dev = x2.device
    state = torch.empty(int(L.ntlb_linear_xent_state_bytes(T, H)), dtype=torch.uint8, device=dev)
    need = int(L.ntlb_linear_xent_workspace_bytes(T, H, V, 0))
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
    loss = torch.empty(max(T, 1) if reduction == 0 else 1, dtype=torch.float32, device=dev)
    _lib.call("ntlb_linear_xent_forward", x2.data_ptr(), x2.stride(0), w.data_ptr(), w.stride(0), targets.data_ptr(),
              int(targets.dtype == torch.int64), T, H, V, ignore_index, reduction, loss.data_ptr(), state.data_ptr(),
              ws.data_ptr(), need, ops._stream())
    return (loss if T else loss[:0]) if reduction == 0 else loss, state


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, ignore_index, reduction):
        x2 = _rows(hidden.detach())
        w = ops._pad_cols(weight.detach(), 8)
        loss, state = _forward(x2, w, targets.reshape(-1).contiguous(), ignore_index, reduction)
        ctx.save_for_backward(w, state)
        ctx.meta = (hidden.shape, x2.shape[0], weight.shape, reduction)
        return loss.reshape(targets.shape if reduction == 0 else ())

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        w, state = ctx.saved_tensors
        shape, T, (V, H), reduction = ctx.meta
        dev = w.device
        dloss = dloss.reshape(-1).contiguous()
        dx = torch.empty((T, H), dtype=torch.bfloat16, device=dev) if ctx.needs_input_grad[0] else None
        dw = torch.empty((V, H), dtype=torch.bfloat16, device=dev) if ctx.needs_input_grad[1] else None
        need = int(_lib.lib().ntlb_linear_xent_workspace_bytes(max(T, 1), H, V, 1))
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        _lib.call("ntlb_linear_xent_backward", state.data_ptr(), w.data_ptr(), w.stride(0), T, H, V, reduction,
                  dloss.data_ptr(), ops._ptr(dx), H, ops._ptr(dw), H, ws.data_ptr(), need, ops._stream())
        return dx.reshape(shape) if dx is not None else None, dw, None, None, None


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *,
                         ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """The cross entropy (fp32) of softmax(hidden @ weight^T) at the targets,
    with the gradients of hidden and weight under autograd.

    hidden bf16 [..., H], weight bf16 [V, H], targets int32 or int64 of
    hidden's leading shape.  Positions with targets == ignore_index have loss 0
    and no gradient, and cost no product; their hidden rows are not read.
    reduction: "none" (the loss of each position), "sum", or "mean" over the
    positions that are not ignored (0 if there are none).  A target that is
    neither a word nor ignore_index makes its position's loss NaN, and the
    gradients with it.

    The logits are never kept: the backward forms them again, a piece of the
    vocabulary at a time.  A weight whose rows are not whole 16-byte pieces
    (H % 8 != 0) is copied to padded rows first."""
    ops._require_device(hidden, weight, targets)
    if reduction not in _REDUCTIONS:
        raise ValueError(f"unknown reduction {reduction!r}; expected 'none', 'sum' or 'mean'")
    if hidden.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise TypeError(f"linear_cross_entropy takes bfloat16 hidden and weight, not {hidden.dtype} and {weight.dtype}")
    if targets.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"targets must be int32 or int64, not {targets.dtype}")
    if hidden.dim() < 1 or weight.dim() != 2 or weight.shape[1] != hidden.shape[-1] or weight.numel() == 0:
        raise ValueError(f"hidden must be [..., H] and weight [V, H]; got {tuple(hidden.shape)}, {tuple(weight.shape)}")
    if targets.shape != hidden.shape[:-1]:
        raise ValueError(f"targets must be {tuple(hidden.shape[:-1])}, not {tuple(targets.shape)}")
    if not (hidden.device == weight.device == targets.device):
        raise ValueError(f"hidden, weight and targets are on {hidden.device}, {weight.device} and {targets.device}")
    red = _REDUCTIONS[reduction]
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        return _LinearCrossEntropy.apply(hidden, weight, targets, int(ignore_index), red)
    loss, _ = _forward(_rows(hidden), ops._pad_cols(weight, 8), targets.reshape(-1).contiguous(),
                       int(ignore_index), red)
    return loss.reshape(targets.shape if red == 0 else ())


class LMHeadLoss(nn.Module):
    """The head's weight [V, H] and its loss: forward(hidden, targets)."""

    def __init__(self, hidden_size: int, vocab_size: int, *, ignore_index: int = -100, reduction: str = "mean",
                 weight: Optional[nn.Parameter] = None, device=None):
        super().__init__()
        if weight is None:
            weight = nn.Parameter(torch.empty(vocab_size, hidden_size, dtype=torch.bfloat16, device=device))
            nn.init.normal_(weight, std=0.02)
        elif weight.shape != (vocab_size, hidden_size):
            raise ValueError(f"weight must be [{vocab_size}, {hidden_size}], not {tuple(weight.shape)}")
        self.weight = weight
        self.ignore_index, self.reduction = ignore_index, reduction

    def forward(self, hidden: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
        return linear_cross_entropy(hidden, self.weight, targets, ignore_index=self.ignore_index,
                                    reduction=self.reduction)
