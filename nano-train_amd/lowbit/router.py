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

from . import _lib
from . import ops

MAX_EXPERTS = 1024
MAX_TOP_K = 16
MAX_GROUPS = 16
_SCORES = {"softmax": 0, "sigmoid": 1}


def route_tokens(logits: torch.Tensor, top_k: int, *, score: str = "softmax", bias: Optional[torch.Tensor] = None,
                 n_groups: int = 1, topk_groups: Optional[int] = None, renormalize: bool = True, scale: float = 1.0):
    """(expert_ids int32 [..., top_k], weights fp32 [..., top_k]) of the
    router's logits [..., E], bf16, fp16 or fp32 with rows of any pitch.

    Scores are softmax(logits) or sigmoid(logits) in fp32 (0 below 2^-126).  The experts are
    chosen by score + bias (fp32 [E], e.g. a balance bias; it does not enter
    the weights and has no gradient), highest first, equal ones lowest index
    first.  With topk_groups < n_groups, the experts form n_groups equal runs
    and only those of the topk_groups best groups can be chosen, a group's
    score being the sum of its two highest choices.  A weight is scale times
    the chosen score, renormalize dividing by the chosen scores' sum + 1e-20.
    Under autograd the weights carry the gradient of the logits.

    Experts that must not be chosen take bias -inf, or logits of -inf: they are
    chosen only when fewer than top_k others remain.  NaN logits order highest;
    ids are always distinct and in range.  E <= 1024, top_k <= 16, n_groups <= 16."""
    if not logits.is_cuda:
        ops._require_device(logits)
    if score not in _SCORES:
        raise ValueError(f"unknown score {score!r}; expected 'softmax' or 'sigmoid'")
    E = logits.shape[-1] if logits.dim() else 0
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"logits must be [..., E] with 1 to {MAX_EXPERTS} experts, not {tuple(logits.shape)}")
    ops._dtype_code(logits.dtype)
    kept = n_groups if topk_groups is None else topk_groups
    if not 1 <= n_groups <= MAX_GROUPS or E % n_groups:
        raise ValueError(f"{E} experts cannot form {n_groups} equal groups (at most {MAX_GROUPS})")
    if not 1 <= kept <= n_groups:
        raise ValueError(f"topk_groups must be 1 to {n_groups}, not {kept}")
    most = min(MAX_TOP_K, kept * (E // n_groups))
    if not 1 <= top_k <= most:
        raise ValueError(f"top_k must be 1 to {most}, not {top_k}")
    if bias is not None:
        if bias.dtype != torch.float32 or bias.dim() != 1 or bias.shape[0] != E or bias.device != logits.device:
            raise ValueError(f"bias must be float32 [{E}] on {logits.device}, not {bias.dtype} {tuple(bias.shape)} "
                             f"on {bias.device}")
        bias = bias.detach()
        if bias.stride(0) != 1:
            bias = bias.contiguous()
    return (_lib._autograd or _lib.autograd()).route(logits, bias, top_k, _SCORES[score], n_groups, kept,
                                                     bool(renormalize), scale)


class TopKRouter(nn.Module):
    """The gate product and route_tokens() of its logits; forward(tokens [T, H])
    returns (expert_ids, weights) as moe.local_moe takes them.

    The gate weight stays in its own dtype (fp32 by default: the recipe's
    routers are not low-bit) and the product runs in it.  balance_bias, when
    asked for, is a buffer that update_bias() moves against the experts' load; it
    stays fp32 when the module's type is changed."""

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

    def _apply(self, fn, *args, **kwargs):
        before = self.balance_bias
        super()._apply(fn, *args, **kwargs)
        if before is not None and self.balance_bias.dtype != torch.float32:
            # fewer bits would swallow its steps, and route_tokens() takes it in fp32
            self.balance_bias = before.to(self.balance_bias.device)
        return self

    def logits(self, tokens: torch.Tensor) -> torch.Tensor:
        return F.linear(tokens.to(self.weight.dtype), self.weight)

    def forward(self, tokens: torch.Tensor):
        return route_tokens(self.logits(tokens), self.top_k, bias=self.balance_bias, **self.cfg)

    @torch.no_grad()
    def update_bias(self, expert_ids: torch.Tensor, rate: float = 1e-3) -> None:
        """balance_bias += rate * sign(mean load - load) over one batch's ids;
        what is no expert's id (a dropped assignment's, say) is not counted."""
        if self.balance_bias is None:
            raise RuntimeError("the router has no balance bias")
        ids, E = expert_ids.reshape(-1).long(), self.n_experts
        # bincount would ask the device for its length: the host would wait, and a graph could not hold the call
        load = torch.zeros(E + 1, dtype=torch.int64, device=ids.device)
        load.scatter_add_(0, torch.where((ids >= 0) & (ids < E), ids, E), torch.ones_like(ids))
        load = load[:E].float()
        self.balance_bias += rate * torch.sign(load.mean() - load)
