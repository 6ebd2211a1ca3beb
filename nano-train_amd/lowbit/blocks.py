"""The MoE layer and the loss of a small language model on this package's
kernels: routed experts and a head as nano-train's models have them
(src/models/deepseek.py, src/models/moe.py; the norm is LayerNorm, where
deepseek.py has RMSNorm), with the low-bit expert products in the middle and the
parts that stay in high precision around them.

  MoEBlock   x + experts(norm(x)): norm.LayerNorm, router.TopKRouter,
             moe.local_moe
  MoELM      embedding, MoEBlocks, a last norm, loss.LMHeadLoss
"""

from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from . import moe
from .loss import LMHeadLoss, linear_cross_entropy
from .norm import LayerNorm
from .router import TopKRouter


class MoEBlock(nn.Module):
    """A pre-norm routed expert layer with its residual, bf16 [..., hidden].

    hidden and intermediate are multiples of 128 (moe.local_moe).  Router
    options go to TopKRouter; fmt and rounding choose the experts' codes.
    last_ids holds the expert ids of the last forward, for update_bias()."""

    def __init__(self, hidden: int, intermediate: int, n_experts: int, top_k: int, *, fmt: str = "e4m3",
                 rounding: str = "nearest", capacity_factor: float = 0.0, eps: float = 1e-5, device=None, **router):
        super().__init__()
        if hidden % 128 or intermediate % 128:
            raise ValueError(f"hidden {hidden} and intermediate {intermediate} must be multiples of 128")
        if top_k > 8:
            raise ValueError("the expert loop supports top_k <= 8")
        bf = dict(dtype=torch.bfloat16, device=device)
        self.norm = LayerNorm(hidden, eps, **bf)
        self.router = TopKRouter(hidden, n_experts, top_k, device=device, **router)
        gate, up = (0.02 * torch.randn(n_experts, intermediate, hidden, **bf) for _ in range(2))
        self.w_gate_up = nn.Parameter(moe.stack_gate_up(gate, up))
        self.w_down = nn.Parameter(0.02 * torch.randn(n_experts, hidden, intermediate, **bf))
        self.fmt, self.rounding, self.capacity_factor = fmt, rounding, capacity_factor
        self.last_ids: Optional[torch.Tensor] = None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        t = self.norm(x).reshape(-1, x.shape[-1])
        ids, w = self.router(t)
        self.last_ids = ids
        capacity = 0
        if self.capacity_factor > 0:
            capacity = moe.compute_capacity(self.capacity_factor, t.shape[0], self.router.top_k, self.router.n_experts)
        y = moe.local_moe(t, ids, w, self.w_gate_up, self.w_down, capacity=capacity, fmt=self.fmt,
                          rounding=self.rounding)
        return x + y.reshape(x.shape)


class MoELM(nn.Module):
    """Next-token model of MoEBlocks: forward(tokens [..., S], targets [..., S])
    is the loss; score(tokens, targets) each position's log-likelihood.  The
    embedding and the head share one weight [vocab, hidden]."""

    def __init__(self, vocab: int, hidden: int, intermediate: int, n_experts: int, top_k: int, n_layers: int = 1, *,
                 ignore_index: int = -100, device=None, **block):
        super().__init__()
        self.head = LMHeadLoss(hidden, vocab, ignore_index=ignore_index, device=device)
        self.blocks = nn.ModuleList(MoEBlock(hidden, intermediate, n_experts, top_k, device=device, **block)
                                    for _ in range(n_layers))
        self.norm = LayerNorm(hidden, dtype=torch.bfloat16, device=device)

    def hidden(self, tokens: torch.Tensor) -> torch.Tensor:
        x = torch.nn.functional.embedding(tokens, self.head.weight)
        for block in self.blocks:
            x = block(x)
        return self.norm(x)

    def forward(self, tokens: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
        return self.head(self.hidden(tokens), targets)

    @torch.no_grad()
    def score(self, tokens: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
        return -linear_cross_entropy(self.hidden(tokens), self.head.weight, targets,
                                     ignore_index=self.head.ignore_index, reduction="none")
