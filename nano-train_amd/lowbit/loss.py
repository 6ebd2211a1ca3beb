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

from . import _lib
from . import ops

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


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
    vocabulary at a time.  Their gradient is rounded to bf16 as the operand of the
    gradients' products, as it is where a bf16 model keeps its logits: with the
    rounding of the results that is up to 1.4 times the latter alone.  Up to 64
    positions it keeps 16 bits, and adds nothing.  A weight whose rows are not whole 16-byte pieces
    (H % 8 != 0), or over 2^22 values apart, is copied to padded rows first.  At
    most 2^22 positions."""
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
    return (_lib._autograd or _lib.autograd()).linear_xent(hidden, weight, targets, ignore_index,
                                                           _REDUCTIONS[reduction])


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
