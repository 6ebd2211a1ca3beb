"""A small MoE language model trained on one GPU: norm, router, low-bit experts and head loss together.

    python nano-train_amd/examples/moe_lm.py --steps 60
    python nano-train_amd/examples/moe_lm.py --steps 60 --norm rms --products bf16 --checkpoint e4m3

The data is synthetic: the next word is a fixed permutation of the current one, and the first positions of every
sequence are a prompt that the loss leaves out.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))))

from lowbit.blocks import MoELM  # noqa: E402


def batch(g: torch.Generator, step_of: torch.Tensor, sequences: int, length: int, prompt: int):
    words = [torch.randint(0, step_of.numel(), (sequences,), generator=g)]
    for _ in range(length):
        words.append(step_of[words[-1]])
    w = torch.stack(words, 1)
    targets = w[:, 1:].clone()
    targets[:, :prompt] = -100
    return w[:, :-1].cuda(), targets.cuda()


def train(steps: int = 60, *, vocab: int = 500, hidden: int = 256, intermediate: int = 128, experts: int = 8,
          top_k: int = 2, layers: int = 2, sequences: int = 16, length: int = 32, prompt: int = 4, lr: float = 2e-3,
          seed: int = 0, log=None, **block):
    """The losses of `steps` steps and the trained model."""
    torch.manual_seed(seed)
    g = torch.Generator().manual_seed(seed)
    step_of = torch.randperm(vocab, generator=g)
    model = MoELM(vocab, hidden, intermediate, experts, top_k, layers, device="cuda", score="sigmoid",
                  balance_bias=True, n_groups=4, topk_groups=2, scale=1.5, **block)
    opt = torch.optim.AdamW(model.parameters(), lr=lr, weight_decay=0.0)
    losses = []
    for step in range(steps):
        tokens, targets = batch(g, step_of, sequences, length, prompt)
        opt.zero_grad(set_to_none=True)
        loss = model(tokens, targets)
        loss.backward()
        opt.step()
        for block in model.blocks:
            block.router.update_bias(block.last_ids)
        losses.append(loss.detach())
        if log and (step % 10 == 0 or step == steps - 1):
            log(f"step {step}: loss {float(loss.detach()):.4f}")
    return [float(x) for x in losses], model, step_of


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__)
    p.add_argument("--steps", type=int, default=60)
    p.add_argument("--seed", type=int, default=0)
    p.add_argument("--norm", choices=("layer", "rms"), default="layer")
    p.add_argument("--products", choices=("lowbit", "bf16"), default="lowbit", help="the experts' products")
    p.add_argument("--checkpoint", choices=("e4m3",), help="keep activations for the backward in 8 bits")
    a = p.parse_args()
    _, model, step_of = train(a.steps, seed=a.seed, log=print, norm=a.norm, products=a.products, checkpoint=a.checkpoint)
    # one token at a time, as a generation step calls the operators
    word = torch.tensor([[7]], device="cuda")
    right, wrong = step_of[7].item(), (step_of[7].item() + 1) % step_of.numel()
    ll = [float(model.score(word, torch.tensor([[w]], device="cuda"))) for w in (right, wrong)]
    print(f"log-likelihood of the word that follows: {ll[0]:.3f}, of another: {ll[1]:.3f}")


if __name__ == "__main__":
    main()
