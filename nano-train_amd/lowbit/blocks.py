"""The MoE layer and the loss of a small language model on this package's
kernels: routed experts and a head as nano-train's models have them
(src/models/deepseek.py, src/models/moe.py), with the low-bit expert products in
the middle and the parts that stay in high precision around them.

  MoEBlock   x + experts(norm(x)): norm.LayerNorm or RMSNorm, router.TopKRouter,
             moe.local_moe or, in bf16, experts.local_moe_bf16
  MoELM      embedding, MoEBlocks, a last norm, loss.LMHeadLoss
"""

from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from . import moe
from . import ops
from .experts import local_moe_bf16
from .loss import LMHeadLoss, linear_cross_entropy
from .norm import LayerNorm, RMSNorm
from .router import TopKRouter


def _norm(kind: str, hidden: int, eps: float, checkpoint: Optional[str], **kw) -> nn.Module:
    if kind == "layer":
        return LayerNorm(hidden, eps, **kw)
    if kind == "rms":
        return RMSNorm(hidden, eps, checkpoint=checkpoint, **kw)
    raise ValueError(f"unknown norm {kind!r}; expected 'layer' or 'rms'")


class MoEBlock(nn.Module):
    """A pre-norm routed expert layer with its residual, bf16 [..., hidden].

    hidden and intermediate are multiples of 128 (moe.local_moe).  norm is "layer"
    or "rms".  products: the experts', "lowbit" (fmt and rounding choose their codes)
    or "bf16", for a layer that the recipe leaves in high precision.  checkpoint "e4m3" keeps what the rms
    norm and the bf16 experts need for their backward in 8 bits.  Router options go
    to TopKRouter.  last_ids holds the expert ids of the last forward, for
    update_bias()."""

    def __init__(self, hidden: int, intermediate: int, n_experts: int, top_k: int, *, fmt: str = "e4m3",
                 rounding: str = "nearest", capacity_factor: float = 0.0, eps: float = 1e-5, norm: str = "layer",
                 products: str = "lowbit", checkpoint: Optional[str] = None, device=None, **router):
        super().__init__()
        if hidden % 128 or intermediate % 128:
            raise ValueError(f"hidden {hidden} and intermediate {intermediate} must be multiples of 128")
        if top_k > 8:
            raise ValueError("the expert loop supports top_k <= 8")
        if products not in ("lowbit", "bf16"):
            raise ValueError(f"unknown products {products!r}; expected 'lowbit' or 'bf16'")
        ops.checkpoint_code(checkpoint)
        if checkpoint and norm != "rms" and products != "bf16":
            raise ValueError("checkpoint is for the rms norm and the bf16 experts; this block has neither")
        bf = dict(dtype=torch.bfloat16, device=device)
        self.norm = _norm(norm, hidden, eps, checkpoint, **bf)
        self.router = TopKRouter(hidden, n_experts, top_k, device=device, **router)
        gate, up = (0.02 * torch.randn(n_experts, intermediate, hidden, **bf) for _ in range(2))
        self.w_gate_up = nn.Parameter(moe.stack_gate_up(gate, up))
        self.w_down = nn.Parameter(0.02 * torch.randn(n_experts, hidden, intermediate, **bf))
        self.fmt, self.rounding, self.capacity_factor = fmt, rounding, capacity_factor
        self.products, self.checkpoint = products, checkpoint
        self.last_ids: Optional[torch.Tensor] = None

    def forward(self, x: torch.Tensor, delta: Optional[torch.Tensor] = None, *, split: bool = False):
        """x + experts(norm(x)).  split: the block on x + delta (delta None: x) without the last
        sum: (the experts' output, x + delta), for the next block's x and delta; with
        the rms norm the norm then forms x + delta."""
        if not split:
            if delta is not None:
                x = x + delta
            return x + self._experts(self.norm(x))
        if delta is None:
            return self._experts(self.norm(x)), x
        if isinstance(self.norm, RMSNorm):
            t, x = self.norm(delta, x)
        else:
            x = x + delta
            t = self.norm(x)
        return self._experts(t), x

    def _experts(self, normed: torch.Tensor) -> torch.Tensor:
        t = normed.reshape(-1, normed.shape[-1])
        ids, w = self.router(t)
        self.last_ids = ids
        capacity = 0
        if self.capacity_factor > 0:
            capacity = moe.compute_capacity(self.capacity_factor, t.shape[0], self.router.top_k, self.router.n_experts)
        if self.products == "bf16":
            y = local_moe_bf16(t, ids, w, self.w_gate_up, self.w_down, capacity=capacity, checkpoint=self.checkpoint)
        else:
            y = moe.local_moe(t, ids, w, self.w_gate_up, self.w_down, capacity=capacity, fmt=self.fmt,
                              rounding=self.rounding)
        return y.reshape(normed.shape)


class MoELM(nn.Module):
    """Next-token model of MoEBlocks: forward(tokens [..., S], targets [..., S])
    is the loss; score(tokens, targets) each position's log-likelihood.  The
    embedding and the head share one weight [vocab, hidden].  Block options go to
    MoEBlock; norm is the last norm's kind too."""

    def __init__(self, vocab: int, hidden: int, intermediate: int, n_experts: int, top_k: int, n_layers: int = 1, *,
                 ignore_index: int = -100, norm: str = "layer", checkpoint: Optional[str] = None, device=None, **block):
        super().__init__()
        self.head = LMHeadLoss(hidden, vocab, ignore_index=ignore_index, device=device)
        self.blocks = nn.ModuleList(MoEBlock(hidden, intermediate, n_experts, top_k, norm=norm, checkpoint=checkpoint,
                                             device=device, **block) for _ in range(n_layers))
        self.norm = _norm(norm, hidden, 1e-5, checkpoint, dtype=torch.bfloat16, device=device)

    def hidden(self, tokens: torch.Tensor) -> torch.Tensor:
        x = torch.nn.functional.embedding(tokens, self.head.weight)
        if not isinstance(self.norm, RMSNorm) or not self.blocks:
            for block in self.blocks:
                x = block(x)
            return self.norm(x)
        delta = None
        for block in self.blocks:  # each sum of the residual stream is formed by the norm after it
            delta, x = block(x, delta, split=True)
        return self.norm(delta, x)[0]

    def forward(self, tokens: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
        return self.head(self.hidden(tokens), targets)

    @torch.no_grad()
    def score(self, tokens: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
        return -linear_cross_entropy(self.hidden(tokens), self.head.weight, targets,
                                     ignore_index=self.head.ignore_index, reduction="none")
