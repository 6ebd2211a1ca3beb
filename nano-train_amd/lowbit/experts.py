"""The parts of an expert or a dense MLP that stay in high precision, on the
MI355X kernels.

grouped_matmul() is one Linear per expert over rows sorted by expert
(src/models/moe.py:888-962, :1062-1097) in bf16, with its gradients; swiglu() is
silu(gate) * up of a product's output that holds both (ExpertMLP.forward,
moe.py:190-193).  Both can keep what their backward reads in 8 bits.
local_moe_bf16() is the routed expert loop of them, moe.local_moe() without codes.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from . import moe
from . import ops


def swiglu(x: torch.Tensor, *, block: int = 0, checkpoint: Optional[str] = None) -> torch.Tensor:
    """silu(gate) * up [..., I] of x [..., 2I], which holds both, with its
    gradient under autograd.

    block 0: gate is the first half of the columns; a multiple of 128 that divides
    I: gate and up alternate in blocks of that many columns (128: the row order of
    moe.stack_gate_up).  x bf16, fp16 or fp32 with rows of any pitch; fp32 inside,
    rounded once.  A gate below -174 (of which sigmoid is 3e-76) gives 0.

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
    offsets[e + 1] - 1, any number of them, offsets[0] being 0.  (One below 0 or below one
    before it counts as that, one past R as R.)  Rows at or past offsets[E]
    (a capacity's spare rows) are not read; y and the gradient of x are zero there.  The
    gradient of an expert without rows is zero.  Sums are fp32, in an order that R, E,
    N and K alone decide, results rounded once.  x and weight of any strides: what is
    not in rows of whole 16-byte pieces (K % 8, for the backward N % 8) is copied to
    padded rows first.  E <= 4096.

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


class _Dispatch(torch.autograd.Function):
    """tokens[token_indices] of every expert (moe.py:1086, :488): the rows of the
    routing's order.  Rows past the kept ones hold any token; nothing reads them."""

    @staticmethod
    def forward(ctx, tokens, routing, expert_ids):
        T, k = tokens.shape[0], routing.top_k
        ctx.routing, ctx.shape = routing, tokens.shape
        ctx.save_for_backward(routing.pos, expert_ids)
        return tokens.index_select(0, routing.inv.clamp(0, max(T * k - 1, 0)) // k)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_rows):
        pos, expert_ids = ctx.saved_tensors
        T, H = ctx.shape
        d_rows = d_rows.contiguous().view(-1).view(-1, H)
        out = torch.empty((T, H), dtype=d_rows.dtype, device=d_rows.device)
        if T:
            ids = expert_ids.contiguous()
            _lib.call("ntlb_moe_token_grad", d_rows.data_ptr(), H, ops._dtype_code(d_rows.dtype), pos.data_ptr(),
                      ids.data_ptr(), 1 if ids.dtype == torch.int64 else 0, T, ctx.routing.top_k, H, out.data_ptr(), H,
                      ops._stream())
        return out, None, None


class _Combine(torch.autograd.Function):
    """output[token_indices] += expert_out * weights (moe.py:1087-1088, :489-490)"""

    @staticmethod
    def forward(ctx, rows, topk_w, routing, expert_ids):
        ctx.routing = routing
        ctx.save_for_backward(rows, topk_w, routing.pos)
        return moe.combine_rows(rows, routing, expert_ids, topk_w, expert_ids.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        rows, topk_w, pos = ctx.saved_tensors
        T, k, H = topk_w.shape[0], ctx.routing.top_k, rows.shape[1]
        w = topk_w.contiguous()
        d_rows = torch.empty((rows.shape[0], H), dtype=rows.dtype, device=rows.device)
        d_w = torch.empty(w.shape, dtype=w.dtype, device=w.device)
        if T:
            d_out = d_out.contiguous().view(-1).view(T, H)
            _lib.call("ntlb_moe_combine_backward", d_out.data_ptr(), H, rows.data_ptr(), rows.stride(0),
                      ops._dtype_code(rows.dtype), pos.data_ptr(), w.data_ptr(), ops._dtype_code(w.dtype), T, k, H,
                      d_rows.data_ptr(), H, d_w.data_ptr(), ops._stream())
        return d_rows, d_w, None, None


def local_moe_bf16(tokens: torch.Tensor, expert_ids: torch.Tensor, topk_w: torch.Tensor, w_gate_up: torch.Tensor,
                   w_down: torch.Tensor, *, capacity: int = 0, checkpoint: Optional[str] = None) -> torch.Tensor:
    """The single-rank routed expert loop with its products in bf16 (moe.py:1062-1093,
    LocalRoutedMoE.forward :476-491, ExpertMLP.forward :190-193): moe.local_moe()'s
    arguments, shapes and capacity, without codes in its products, and the gradients of
    tokens, routing weights and expert weights under autograd, all of them on one
    device, which need not be the current one.  grouped_matmul(), swiglu(block=128),
    grouped_matmul() and the weighted sum of each token's rows.

    checkpoint "e4m3" keeps the rows of both products and the projections between
    them in 8 bits for the backward, 1/2 of what the bf16 loop keeps beside the
    down projection's output."""
    ops._require_device(tokens, expert_ids, topk_w, w_gate_up, w_down)
    if any(t.device != tokens.device for t in (expert_ids, topk_w, w_gate_up, w_down)):
        raise ValueError(f"tokens are on {tokens.device}, expert_ids, topk_w, w_gate_up and w_down on {expert_ids.device}, "
                         f"{topk_w.device}, {w_gate_up.device} and {w_down.device}")
    if tokens.dim() != 2 or expert_ids.dim() != 2 or topk_w.shape != expert_ids.shape or expert_ids.shape[0] != tokens.shape[0]:
        raise ValueError("tokens must be [T, H], expert_ids and topk_w [T, k]")
    if tokens.dtype != torch.bfloat16 or w_gate_up.dtype != torch.bfloat16 or w_down.dtype != torch.bfloat16:
        raise TypeError("local_moe_bf16 takes bf16 tokens and bf16 expert weights")
    if w_gate_up.dim() != 3 or w_gate_up.shape[1] % 256 or w_gate_up.shape[2] != tokens.shape[1] \
            or w_down.shape != (w_gate_up.shape[0], tokens.shape[1], w_gate_up.shape[1] // 2):
        raise ValueError(f"weights must be w_gate_up [E, 2I, H] (2I % 256 == 0) and w_down [E, H, I]; got "
                         f"{tuple(w_gate_up.shape)}, {tuple(w_down.shape)}")
    if expert_ids.shape[1] > 8:
        raise ValueError("local_moe_bf16 supports top_k <= 8")
    ops.checkpoint_code(checkpoint)
    with torch.cuda.device(tokens.device):  # the gather and the sum launch on the current device's stream
        routing = moe.route_by_expert(expert_ids, w_gate_up.shape[0], capacity=int(capacity), topk_w=topk_w)
        rows = _Dispatch.apply(tokens, routing, expert_ids)
        gate_up = grouped_matmul(rows, w_gate_up, routing.offsets, checkpoint=checkpoint)
        h = swiglu(gate_up, block=128, checkpoint=checkpoint)
        return _Combine.apply(grouped_matmul(h, w_down, routing.offsets, checkpoint=checkpoint), topk_w, routing,
                              expert_ids)
