"""Routing to experts on the MI355X kernels: the scores, the choice and the
weights in front of the expert loop (moe.local_moe, moe.local_moe_forward,
ep.pack_dispatch), which the DeepSeek-V3 recipe keeps in high precision.

route_tokens() is the operator with its gradient; TopKRouter is the module
(TopKRouter, src/models/moe.py:196-350 of nano-train): the gate product, the
routing, and the balance bias with its update.
"""

from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import _lib
from . import ops
from .norm import _rows

MAX_EXPERTS = 1024
MAX_TOP_K = 16
MAX_GROUPS = 16
_SCORES = {"softmax": 0, "sigmoid": 1}


def _forward(z: torch.Tensor, k: int, sigmoid: int, bias, groups: int, kept: int, renorm: int, scale: float):
    T, E = z.shape
    ids = torch.empty((T, k), dtype=torch.int32, device=z.device)
    w = torch.empty((T, k), dtype=torch.float32, device=z.device)
    _lib.call("ntlb_route_topk", z.data_ptr(), ops._dtype_code(z.dtype), T, E, z.stride(0), k, sigmoid, ops._ptr(bias),
              groups, kept, renorm, scale, ids.data_ptr(), w.data_ptr(), ops._stream())
    return ids, w


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, k, sigmoid, groups, kept, renorm, scale):
        z = _rows(logits.detach())
        ids, w = _forward(z, k, sigmoid, bias, groups, kept, renorm, scale)
        ctx.save_for_backward(z, ids)
        ctx.cfg = (k, sigmoid, renorm, scale, logits.shape)
        ctx.mark_non_differentiable(ids)
        lead = logits.shape[:-1]
        return ids.reshape(*lead, k), w.reshape(*lead, k)

    @staticmethod
    @once_differentiable
    def backward(ctx, _d_ids, dw):
        z, ids = ctx.saved_tensors
        k, sigmoid, renorm, scale, shape = ctx.cfg
        T, E = z.shape
        dw = dw.contiguous()
        dz = torch.empty((T, E), dtype=z.dtype, device=z.device)
        _lib.call("ntlb_route_topk_backward", z.data_ptr(), ops._dtype_code(z.dtype), T, E, z.stride(0), k, sigmoid,
                  renorm, scale, ids.data_ptr(), dw.data_ptr(), dz.data_ptr(), E, ops._stream())
        return dz.reshape(shape), None, None, None, None, None, None, None


def route_tokens(logits: torch.Tensor, top_k: int, *, score: str = "softmax", bias: Optional[torch.Tensor] = None,
                 n_groups: int = 1, topk_groups: Optional[int] = None, renormalize: bool = True, scale: float = 1.0):
    """(expert_ids int32 [..., top_k], weights fp32 [..., top_k]) of the
    router's logits [..., E], bf16, fp16 or fp32 with rows of any pitch.

    Scores are softmax(logits) or sigmoid(logits) in fp32.  The experts are
    chosen by score + bias (fp32 [E], e.g. a balance bias; it does not enter
    the weights and has no gradient), highest first, equal ones lowest index
    first.  With topk_groups < n_groups, the experts form n_groups equal runs
    and only those of the topk_groups best groups can be chosen, a group's
    score being the sum of its two highest choices.  A weight is scale times
    the chosen score, renormalize dividing by the chosen scores' sum + 1e-20.
    Under autograd the weights carry the gradient of the logits.

    Experts that must not be chosen take bias -inf: they are chosen only when
    fewer than top_k others remain.  NaN logits order highest; ids are always
    distinct and in range.  E <= 1024, top_k <= 16, n_groups <= 16."""
    ops._require_device(logits, bias)
    if score not in _SCORES:
        raise ValueError(f"unknown score {score!r}; expected 'softmax' or 'sigmoid'")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= MAX_EXPERTS:
        raise ValueError(f"logits must be [..., E] with 1 to {MAX_EXPERTS} experts, not {tuple(logits.shape)}")
    ops._dtype_code(logits.dtype)
    E = logits.shape[-1]
    kept = n_groups if topk_groups is None else topk_groups
    if not 1 <= n_groups <= MAX_GROUPS or E % n_groups:
        raise ValueError(f"{E} experts cannot form {n_groups} equal groups (at most {MAX_GROUPS})")
    if not 1 <= kept <= n_groups:
        raise ValueError(f"topk_groups must be 1 to {n_groups}, not {kept}")
    if not 1 <= top_k <= min(MAX_TOP_K, kept * (E // n_groups)):
        raise ValueError(f"top_k must be 1 to {min(MAX_TOP_K, kept * (E // n_groups))}, not {top_k}")
    if bias is not None:
        if bias.shape != (E,) or bias.dtype != torch.float32 or bias.device != logits.device:
            raise ValueError(f"bias must be float32 [{E}] on {logits.device}, not {bias.dtype} {tuple(bias.shape)} "
                             f"on {bias.device}")
        bias = bias.detach()
        if bias.stride(0) != 1:
            bias = bias.contiguous()
    args = (int(top_k), _SCORES[score], bias, int(n_groups), int(kept), int(bool(renormalize)), float(scale))
    if torch.is_grad_enabled() and logits.requires_grad:
        return _Route.apply(logits, bias, args[0], args[1], *args[3:])
    ids, w = _forward(_rows(logits), *args)
    lead = logits.shape[:-1]
    return ids.reshape(*lead, top_k), w.reshape(*lead, top_k)


class TopKRouter(nn.Module):
    """The gate product and route_tokens() of its logits; forward(tokens [T, H])
    returns (expert_ids, weights) as moe.local_moe takes them.

    The gate weight stays in its own dtype (fp32 by default: the recipe's
    routers are not low-bit) and the product runs in it.  balance_bias, when
    asked for, is a buffer that update_bias() moves against the experts' load."""

    def __init__(self, hidden_size: int, n_experts: int, top_k: int, *, score: str = "softmax",
                 balance_bias: bool = False, n_groups: int = 1, topk_groups: Optional[int] = None,
                 renormalize: bool = True, scale: float = 1.0, dtype: torch.dtype = torch.float32, device=None):
        super().__init__()
        self.n_experts, self.top_k = n_experts, top_k
        self.cfg = dict(score=score, n_groups=n_groups, topk_groups=topk_groups, renormalize=renormalize, scale=scale)
        self.weight = nn.Parameter(torch.empty(n_experts, hidden_size, dtype=dtype, device=device))
        nn.init.normal_(self.weight, std=0.02)
        self.register_buffer("balance_bias",
                             torch.zeros(n_experts, dtype=torch.float32, device=device) if balance_bias else None)

    def logits(self, tokens: torch.Tensor) -> torch.Tensor:
        return F.linear(tokens.to(self.weight.dtype), self.weight)

    def forward(self, tokens: torch.Tensor):
        return route_tokens(self.logits(tokens), self.top_k, bias=self.balance_bias, **self.cfg)

    @torch.no_grad()
    def update_bias(self, expert_ids: torch.Tensor, rate: float = 1e-3) -> None:
        """balance_bias += rate * sign(mean load - load) over one batch's ids."""
        if self.balance_bias is None:
            raise RuntimeError("the router has no balance bias")
        load = torch.bincount(expert_ids.reshape(-1).long(), minlength=self.n_experts).float()
        self.balance_bias += rate * torch.sign(load.mean() - load)
