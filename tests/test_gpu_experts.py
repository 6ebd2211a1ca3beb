"""GPU tests of the routed expert loop in bf16 (lowbit.experts.local_moe_bf16) against the loop over experts in 64 bits, and
of a block and a small model made of it, the rms norm and activations kept in 8 bits.

Bounds: every stage rounds to bf16 (2^-8 of its result): the projections, h, the experts' outputs, the products with the
routing weights and their sums; the reference here forms all of them in 64 bits, so results are compared by their
2-norm: six roundings of independent sign come to at most 6 x 2^-8 of it.  With 8 bits kept, each value that a
weight's gradient sums is off by up to 2^-4, on average over signs far less; the norm of such a gradient is held to 2^-4.
"""

from __future__ import annotations

import os
import sys

import pytest
import torch

from conftest import PKG_PARENT

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(PKG_PARENT, "examples"))

V = 2.0 ** -8


def _inputs(T, E, k, H, I, dev, seed=0):
    from lowbit import moe

    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, generator=g).bfloat16().to(dev)
    gate, up = ((torch.randn(E, I, H, generator=g) / H ** 0.5).bfloat16().to(dev) for _ in range(2))
    down = (torch.randn(E, H, I, generator=g) / I ** 0.5).bfloat16().to(dev)
    ids = torch.rand(T, E, generator=g).argsort(1)[:, :k].int().to(dev)
    w = torch.rand(T, k, generator=g).to(dev)
    dy = torch.randn(T, H, generator=g).bfloat16().to(dev)
    return x, ids, w, moe.stack_gate_up(gate, up), down, dy


def _reference(x, ids, w, w_gate_up, w_down, keep):
    """the loop over experts; keep[e]: which (token, slot) pairs of expert e count"""
    from lowbit import moe

    out = torch.zeros_like(x)
    gate, up = moe.split_gate_up(w_gate_up)
    for e in range(w_down.shape[0]):
        t, s = keep[e]
        if t.numel() == 0:
            continue
        H = x.shape[1]
        a, b = x[t] @ gate[e].reshape(-1, H).t(), x[t] @ up[e].reshape(-1, H).t()
        out = out.index_add(0, t, (torch.nn.functional.silu(a) * b @ w_down[e].t()) * w[t, s][:, None])
    return out


def _pairs(ids, w, E, capacity):
    keep = []
    for e in range(E):
        t, s = (ids == e).nonzero(as_tuple=True)
        if capacity and t.numel() > capacity:
            top = torch.topk(w[t, s], capacity).indices
            t, s = t[top], s[top]
        keep.append((t, s))
    return keep


def _far(a, b):
    return float((a.double() - b).norm() / b.norm())


@pytest.mark.parametrize("T,E,k,H,I,capacity", [(40, 6, 2, 256, 128, 0), (500, 8, 3, 128, 256, 0), (500, 8, 3, 128, 256, 90),
                                                (1, 32, 8, 256, 128, 0), (300, 3, 1, 384, 128, 0)])
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_values_and_gradients(gpu_device, T, E, k, H, I, capacity, checkpoint):
    from lowbit.experts import local_moe_bf16

    x, ids, w, gu, down, dy = _inputs(T, E, k, H, I, gpu_device, T + E)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, gu, down)]
    y = local_moe_bf16(leaves[0], ids, *leaves[1:], capacity=capacity, checkpoint=checkpoint)
    got = torch.autograd.grad(y, leaves, dy)
    wide = [t.double().requires_grad_(True) for t in (x, w, gu, down)]
    want_y = _reference(wide[0], ids, *wide[1:], _pairs(ids, w, E, capacity))
    want = torch.autograd.grad(want_y, wide, dy.double())
    assert _far(y.detach(), want_y.detach()) < 6 * V
    for name, a, b in zip(("tokens", "weights", "gate_up", "down"), got, want):
        assert a.dtype == (torch.float32 if name == "weights" else torch.bfloat16) and a.shape == b.shape
        assert _far(a, b) < (6 * V if not checkpoint or name == "weights" else 6 * V + 2.0 ** -4), name
    with torch.no_grad():
        assert torch.equal(local_moe_bf16(x, ids, w, gu, down, capacity=capacity), y)


def test_what_is_kept(gpu_device):
    """with 8 bits no row of both products nor of the projections stays in bf16"""
    from lowbit.experts import local_moe_bf16

    x, ids, w, gu, down, _ = _inputs(64, 4, 2, 256, 128, gpu_device)
    kept = {}
    for checkpoint in (None, "e4m3"):
        saved = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
            local_moe_bf16(x.requires_grad_(True), ids, w, gu.requires_grad_(True), down.requires_grad_(True),
                           checkpoint=checkpoint)
        seen = {t.data_ptr(): t for t in saved if t.data_ptr() not in (gu.data_ptr(), down.data_ptr())}
        kept[checkpoint] = sum(t.numel() * t.element_size() for t in seen.values() if t.numel() >= 128 * 128)
    out = 128 * 256 * 2  # the down projection's rows, for the routing weights' gradient
    assert kept[None] - out == 128 * 2 * (256 + 256 + 128) and kept["e4m3"] - out == 128 * (256 + 256 + 128)


def test_a_row_of_any_pitch_and_no_tokens(gpu_device):
    from lowbit.experts import local_moe_bf16

    x, ids, w, gu, down, dy = _inputs(1, 4, 2, 256, 128, gpu_device)
    got = []
    for u in (dy, dy.reshape(256, 1).t()):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, gu, down)]
        got.append(torch.autograd.grad(local_moe_bf16(leaves[0], ids, *leaves[1:]), leaves, u))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    leaves = [t.clone().requires_grad_(True) for t in (x[:0], w[:0], gu, down)]
    y = local_moe_bf16(leaves[0], ids[:0], *leaves[1:], checkpoint="e4m3")
    assert y.shape == (0, 256)
    y.sum().backward()
    assert [t.grad.shape for t in leaves] == [t.shape for t in leaves] and not leaves[2].grad.any()


def test_an_expert_named_twice_and_long_ids(gpu_device):
    """a token's slots count one by one, also where they name the same expert; ids of 64 bits are the same ids"""
    from lowbit.experts import local_moe_bf16

    x, _, w, gu, down, dy = _inputs(30, 4, 2, 256, 128, gpu_device, 3)
    ids = (torch.arange(60, device=gpu_device, dtype=torch.int32).view(30, 2) // 2) % 4  # both slots alike
    leaves = [t.clone().requires_grad_(True) for t in (x, w, gu, down)]
    y = local_moe_bf16(leaves[0], ids, *leaves[1:])
    got = torch.autograd.grad(y, leaves, dy)
    wide = [t.double().requires_grad_(True) for t in (x, w, gu, down)]
    want_y = _reference(wide[0], ids, *wide[1:], _pairs(ids, w, 4, 0))
    want = torch.autograd.grad(want_y, wide, dy.double())
    assert _far(y.detach(), want_y.detach()) < 6 * V
    assert all(_far(a, b) < 6 * V for a, b in zip(got, want))
    again = local_moe_bf16(leaves[0], ids.long(), *leaves[1:])
    assert torch.equal(again, y)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(again, leaves, dy), got))


def test_second_gradient_is_refused(gpu_device):
    from lowbit.experts import local_moe_bf16

    x, ids, w, gu, down, _ = _inputs(16, 4, 2, 256, 128, gpu_device)
    for which in range(4):
        leaves = [t.clone().requires_grad_(i == which) for i, t in enumerate((x, w, gu, down))]
        y = local_moe_bf16(leaves[0], ids, *leaves[1:])
        (d,) = torch.autograd.grad(y.square().sum(), leaves[which], create_graph=True)
        with pytest.raises(RuntimeError):
            d.square().sum().backward()


def test_refusals(gpu_device):
    from lowbit.blocks import MoEBlock
    from lowbit.experts import local_moe_bf16

    x, ids, w, gu, down, _ = _inputs(8, 4, 2, 256, 128, gpu_device)
    with pytest.raises(RuntimeError, match="ROCm device"):
        local_moe_bf16(x.cpu(), ids, w, gu, down)
    with pytest.raises(TypeError, match="bf16"):
        local_moe_bf16(x.float(), ids, w, gu, down)
    for bad in ((x, ids[:4], w, gu, down), (x, ids, w[:, :1], gu, down), (x, ids, w, gu[:, :128], down), (x, ids, w, gu, gu)):
        with pytest.raises(ValueError):
            local_moe_bf16(*bad)
    with pytest.raises(ValueError, match="checkpoint"):
        local_moe_bf16(x, ids, w, gu, down, checkpoint="fp8")
    with pytest.raises(ValueError, match="norm"):
        MoEBlock(256, 128, 8, 2, norm="batch", device=gpu_device)
    with pytest.raises(ValueError, match="products"):
        MoEBlock(256, 128, 8, 2, products="fp32", device=gpu_device)
    with pytest.raises(ValueError, match="neither"):
        MoEBlock(256, 128, 8, 2, checkpoint="e4m3", device=gpu_device)


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_block_is_its_parts(gpu_device, checkpoint):
    from lowbit.blocks import MoEBlock
    from lowbit.experts import local_moe_bf16
    from lowbit.norm import rms_norm
    from lowbit.router import route_tokens

    torch.manual_seed(3)
    b = MoEBlock(256, 128, 8, 2, device=gpu_device, norm="rms", products="bf16", checkpoint=checkpoint, score="sigmoid")
    x = torch.randn(3, 50, 256, device=gpu_device).bfloat16().requires_grad_(True)
    dy = torch.randn(3, 50, 256, device=gpu_device).bfloat16()
    y = b(x)
    y.backward(dy)
    x2 = x.detach().clone().requires_grad_(True)
    p = {n: q.detach().clone().requires_grad_(True) for n, q in b.named_parameters()}
    t = rms_norm(x2, p["norm.weight"], eps=1e-5, checkpoint=checkpoint).reshape(-1, 256)
    ids, w = route_tokens(torch.nn.functional.linear(t.float(), p["router.weight"]), 2, score="sigmoid")
    want = x2 + local_moe_bf16(t, ids, w, p["w_gate_up"], p["w_down"], checkpoint=checkpoint).reshape(x.shape)
    want.backward(dy)
    assert torch.equal(y.detach(), want.detach()) and torch.equal(x.grad, x2.grad)
    for n, q in b.named_parameters():
        assert torch.equal(q.grad, p[n].grad) and q.grad.any(), n


@pytest.mark.parametrize("norm", ["layer", "rms"])
def test_the_residual_joins_the_norm(gpu_device, norm):
    """blocks after one another: the sum in the next norm is the sum of forward(), bit for bit"""
    from lowbit.blocks import MoELM

    torch.manual_seed(1)
    m = MoELM(90, 256, 128, 4, 2, 3, device=gpu_device, norm=norm, products="bf16")
    words = torch.randint(0, 90, (2, 12), device=gpu_device)
    with torch.no_grad():
        x = torch.nn.functional.embedding(words, m.head.weight)
        for block in m.blocks:
            x = block(x)
        assert torch.equal(m.hidden(words), m.norm(x))
        x = torch.randn(5, 256, device=gpu_device).bfloat16()
        d = torch.randn(5, 256, device=gpu_device).bfloat16()
        y, total = m.blocks[0](x, d, split=True)
        assert torch.equal(total, x + d) and torch.equal(total + y, m.blocks[0](x + d)) and torch.equal(total + y, m.blocks[0](x, d))
        assert MoELM(90, 256, 128, 4, 2, 0, device=gpu_device, norm=norm).hidden(words).shape == (2, 12, 256)


@pytest.mark.parametrize("options", [dict(norm="rms"), dict(norm="rms", products="bf16", checkpoint="e4m3")])
def test_example_runs(gpu_device, options):
    import moe_lm

    losses, model, step_of = moe_lm.train(3, **options)
    assert all(torch.isfinite(torch.tensor(losses)))
    for n, p in model.named_parameters():
        assert p.grad is not None and p.grad.isfinite().all() and p.grad.any(), n
    assert model.score(torch.tensor([[7]], device=gpu_device), step_of[7].reshape(1, 1).cuda()).isfinite().all()


@pytest.mark.parametrize("capacity", [0, 20])
def test_generation_replays_in_a_graph(gpu_device, capacity):
    """the loop without gradients, captured: every replay is the eager result of the tokens, ids and weights then there"""
    from lowbit.experts import local_moe_bf16

    x, ids, w, gu, down, _ = _inputs(60, 6, 2, 256, 128, gpu_device)
    with torch.no_grad():
        local_moe_bf16(x, ids, w, gu, down, capacity=capacity)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = local_moe_bf16(x, ids, w, gu, down, capacity=capacity)
        for seed in range(1, 5):
            for t, new in zip((x, ids, w), _inputs(60, 6, 2, 256, 128, gpu_device, seed)):
                t.copy_(new)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, local_moe_bf16(x, ids, w, gu, down, capacity=capacity)), seed
