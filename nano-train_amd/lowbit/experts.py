"""The parts of an expert or a dense MLP that stay in high precision, on the
MI355X kernels.

swiglu() is silu(gate) * up of a product's output that holds both
(ExpertMLP.forward, src/models/moe.py:190-193), with its gradient.
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
