"""The parts of an expert or a dense MLP that stay in high precision, on the
MI355X kernels.

grouped_matmul() is one Linear per expert over rows sorted by expert
(src/models/moe.py:888-962, :1062-1097) in bf16, with its gradients; swiglu() is
silu(gate) * up of a product's output that holds both (ExpertMLP.forward,
moe.py:190-193).  Both can keep what their backward reads in 8 bits.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from . import ops


def swiglu(x: torch.Tensor, *, block: int = 0, checkpoint: Optional[str] = None) -> torch.Tensor:
    """silu(gate) * up [..., I] of x [..., 2I], which holds both, with its
    gradient under autograd.

    block 0: gate is the first half of the columns; a multiple of 128 that divides
    I: gate and up alternate in blocks of that many columns (128: the row order of
    moe.stack_gate_up).  x bf16, fp16 or fp32 with rows of any pitch; fp32 inside,
    rounded once.

    checkpoint None keeps x for the backward; "e4m3" keeps gate and up in 8 bits (a
    power of two for each 128 columns, values rounded by at most 2^-4 of
    themselves where they are not 2^-14 of the tile's largest or less), and the
    gradient is that at the values kept.  A value that is not finite is kept as
    NaN."""
    if not x.is_cuda:
        ops._require_device(x)
    if x.dtype not in ops._DTYPE_CODE:
        ops._dtype_code(x.dtype)
    n = x.shape[-1] if x.dim() else 0
    if n < 2 or n % 2:
        raise ValueError(f"swiglu takes [..., 2I], not {tuple(x.shape)}")
    if block and (block < 0 or block % 128 or (n // 2) % block):
        raise ValueError(f"block must be 0 or a multiple of 128 that divides {n // 2}, not {block}")
    return (_lib._autograd or _lib.autograd()).swiglu(x, block, ops.checkpoint_code(checkpoint))


def grouped_matmul(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, *,
                   checkpoint: Optional[str] = None) -> torch.Tensor:
    """y[r] = weight[e] @ x[r] for the rows r of expert e, with the gradients of x
    and weight under autograd.

    x bf16 [R, K], its rows sorted by expert; weight bf16 [E, N, K]; offsets int32
    [E + 1], not decreasing, on x's device: expert e has the rows offsets[e] ..
    offsets[e + 1] - 1, any number of them, offsets[0] being 0.  Rows at or past offsets[E]
    (a capacity's spare rows) are not read; y and the gradient of x are zero there.  The
    gradient of an expert without rows is zero.  Sums are fp32, results rounded once.
    x and weight of any strides: what is not in rows of whole 16-byte pieces (K % 8,
    for the backward N % 8) is copied to padded rows first.  E <= 4096.

    checkpoint None keeps x for the weight's gradient; "e4m3" keeps it in 8 bits (a
    power of two for each 128 columns, values rounded by at most 2^-4 of
    themselves where they are not 2^-14 of the tile's largest or less), and that gradient is
    the one at the values kept.  A value that is not finite is kept as NaN."""
    ops._require_device(x, weight, offsets)
    if x.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise TypeError(f"grouped_matmul takes bfloat16 x and weight, not {x.dtype} and {weight.dtype}")
    if x.dim() != 2 or weight.dim() != 3 or weight.numel() == 0 or weight.shape[2] != x.shape[1]:
        raise ValueError(f"x must be [R, K] and weight [E, N, K]; got {tuple(x.shape)}, {tuple(weight.shape)}")
    if offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.shape[0] != weight.shape[0] + 1:
        raise ValueError(f"offsets must be int32 [{weight.shape[0] + 1}], not {offsets.dtype} {tuple(offsets.shape)}")
    if not (x.device == weight.device == offsets.device):
        raise ValueError(f"x, weight and offsets are on {x.device}, {weight.device} and {offsets.device}")
    if offsets.stride(0) != 1:
        offsets = offsets.contiguous()
    return (_lib._autograd or _lib.autograd()).grouped_matmul(x, weight, offsets, ops.checkpoint_code(checkpoint))
