"""GPU tests of the MoE block and the small language model: norm, router, experts and head loss in one training step."""

from __future__ import annotations

import os
import sys

import pytest
import torch

from conftest import PKG_PARENT

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(PKG_PARENT, "examples"))


def _block(dev, **kw):
    from lowbit.blocks import MoEBlock

    torch.manual_seed(3)
    return MoEBlock(256, 128, 8, 2, device=dev, **kw)


def test_block_is_its_parts(gpu_device):
    """the block's output and gradients are those of its operators called one by one"""
    from lowbit import moe
    from lowbit.norm import layer_norm
    from lowbit.router import route_tokens

    b = _block(gpu_device, score="sigmoid", n_groups=4, topk_groups=2, scale=1.5)
    x = torch.randn(3, 50, 256, device=gpu_device).bfloat16().requires_grad_(True)
    dy = torch.randn(3, 50, 256, device=gpu_device).bfloat16()
    y = b(x)
    y.backward(dy)
    x2 = x.detach().clone().requires_grad_(True)
    p = {n: q.detach().clone().requires_grad_(True) for n, q in b.named_parameters()}
    t = layer_norm(x2, p["norm.weight"], p["norm.bias"]).reshape(-1, 256)
    ids, w = route_tokens(torch.nn.functional.linear(t.float(), p["router.weight"]), 2, score="sigmoid", n_groups=4,
                          topk_groups=2, scale=1.5)
    want = x2 + moe.local_moe(t, ids, w, p["w_gate_up"], p["w_down"]).reshape(x.shape)
    want.backward(dy)
    assert torch.equal(y.detach(), want.detach()) and torch.equal(b.last_ids, ids)
    assert torch.equal(x.grad, x2.grad)
    for n, q in b.named_parameters():
        assert torch.equal(q.grad, p[n].grad) and q.grad.any(), n


def test_block_with_a_capacity_and_no_gradients(gpu_device):
    b = _block(gpu_device, capacity_factor=1.0, fmt="int_grid")
    x = torch.randn(64, 256, device=gpu_device).bfloat16()
    with torch.no_grad():
        y = b(x)
        one = b(x[:1])
    assert y.isfinite().all() and one.shape == (1, 256)


def test_block_refusals(gpu_device):
    from lowbit.blocks import MoEBlock

    with pytest.raises(ValueError, match="multiples of 128"):
        MoEBlock(200, 128, 8, 2, device=gpu_device)
    with pytest.raises(ValueError, match="top_k"):
        MoEBlock(256, 128, 16, 9, device=gpu_device)


def test_small_model_learns(gpu_device):
    """60 steps on a next-word permutation of 500 words: from ln 500 (6.2) or above to below a third of it, the balance
    bias moves, and single tokens score the right word above another"""
    import moe_lm

    losses, model, step_of = moe_lm.train(60)
    assert losses[0] > 5.5 and sum(losses[-5:]) / 5 < 2.1, (losses[0], losses[-5:])
    assert model.blocks[0].router.balance_bias.any()
    words = torch.arange(0, 40, device=gpu_device)[:, None]
    right = model.score(words, step_of[:40, None].cuda())
    wrong = model.score(words, ((step_of[:40, None] + 1) % 500).cuda())
    assert (right > wrong).float().mean() > 0.9
    one = model.score(words[:1], step_of[:1, None].cuda())
    assert one.shape == (1, 1)


@pytest.mark.parametrize("rounding", ["nearest", "stochastic"])
def test_one_token_and_a_gradient_of_any_pitch(gpu_device, rounding):
    """the experts' single row, whose incoming gradient has strides (1, 1), as a column's transposition leaves it"""
    from lowbit import moe

    b = _block(gpu_device)
    x, w = torch.randn(1, 256, device=gpu_device).bfloat16(), torch.rand(1, 2, device=gpu_device)
    ids = torch.tensor([[3, 5]], dtype=torch.int32, device=gpu_device)
    up = torch.randn(256, 1, device=gpu_device).bfloat16().t()
    assert up.stride() == (1, 1)
    got = []
    for u in (up, up.reshape(-1).clone().reshape(1, 256)):
        leaves = [x.clone().requires_grad_(True), w.clone().requires_grad_(True), b.w_gate_up, b.w_down]
        y = moe.local_moe(leaves[0], ids, leaves[1], *leaves[2:], rounding=rounding)
        got.append(torch.autograd.grad(y, leaves, u))
    assert all(torch.equal(p, q) for p, q in zip(*got))


@pytest.mark.parametrize("shape", [(0, 256), (2, 0, 256)])
@pytest.mark.parametrize("rounding", ["nearest", "stochastic"])
def test_no_tokens(gpu_device, shape, rounding):
    """an empty batch trains: gradients of the inputs' shapes, zero for the weights"""
    b = _block(gpu_device, rounding=rounding, score="sigmoid")
    x = torch.randn(*shape, device=gpu_device).bfloat16().requires_grad_(True)
    y = b(x)
    assert y.shape == shape
    y.sum().backward()
    assert x.grad.shape == shape
    for n, p in b.named_parameters():
        assert p.grad.shape == p.shape and not p.grad.any(), n
    with torch.no_grad():
        assert b(x).shape == shape


def test_small_model_without_positions(gpu_device):
    from lowbit.blocks import MoELM

    m = MoELM(50, 256, 128, 8, 2, device=gpu_device)
    none = torch.zeros(2, 0, dtype=torch.int64, device=gpu_device)
    loss = m(none, none)
    loss.backward()
    assert float(loss.detach()) == 0 and all(p.grad is None or not p.grad.any() for p in m.parameters())
    assert m.score(none, none).shape == (2, 0)
