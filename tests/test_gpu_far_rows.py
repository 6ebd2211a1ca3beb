"""GPU tests of the RMS norm, SwiGLU and the grouped products on buffers of more than 2^32 values: the last rows are those
that the operator gives for a copy of them alone (each row is its own result), and the grouped products' the definition in
64 bits, with the bounds of their own tests."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U, V = 2.0 ** -24, 2.0 ** -8


def _random(dev, *sizes, seed=0):
    g = torch.Generator(dev).manual_seed(seed)
    return torch.randn(*sizes, generator=g, device=dev, dtype=torch.bfloat16)


def test_rms_norm(gpu_device):
    from lowbit.norm import rms_norm, rms_norm_quant

    T, H, n = (1 << 32) // 7168 + 300, 7168, 70
    x, w = _random(gpu_device, T, H), _random(gpu_device, H, seed=1)
    far = x[-n:].clone()
    for checkpoint in (None, "e4m3"):
        grads = []
        for rows in (x, far):
            leaf = rows.requires_grad_(True)
            y = rms_norm(leaf, w, checkpoint=checkpoint)
            grads.append((y.detach()[-n:].clone(), torch.autograd.grad(y, leaf, y.detach())[0][-n:].clone()))
            del y, leaf
        assert all(torch.equal(a, b) for a, b in zip(*grads)), checkpoint
        del grads
    with torch.no_grad():
        q, p = rms_norm_quant(x, w), rms_norm_quant(far, w)
        assert torch.equal(q.codes[-n:], p.codes) and torch.equal(q.scales[:, T - n:T], p.scales[:, :n])


def test_swiglu(gpu_device):
    from lowbit.experts import swiglu

    T, I, n = (1 << 31) // 5120 + 300, 5120, 70
    x = _random(gpu_device, T, 2 * I)
    far = x[-n:].clone()
    for block, checkpoint in ((0, None), (128, "e4m3")):
        got = []
        for rows in (x, far):
            leaf = rows.requires_grad_(True)
            h = swiglu(leaf, block=block, checkpoint=checkpoint)
            got.append((h.detach()[-n:].clone(), torch.autograd.grad(h, leaf, h.detach())[0][-n:].clone()))
            del h, leaf
        assert all(torch.equal(a, b) for a, b in zip(*got)), (block, checkpoint)


def _close(got, want, n, mags):
    assert ((got.double() - want).abs() <= 2 * n * U * mags + V * want.abs()).all()


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_grouped_rows(gpu_device, checkpoint):
    """many rows: the last ones' y and dx, the last expert's dW"""
    from _kept import kept
    from lowbit.experts import grouped_matmul

    K, N, n = 4096, 136, 200
    R = (1 << 32) // K + 1000
    x, w, dy = _random(gpu_device, R, K), _random(gpu_device, 3, N, K, seed=1), _random(gpu_device, R, N, seed=2)
    offsets = torch.tensor([0, R // 2, R - n, R], dtype=torch.int32, device=gpu_device)
    lx, lw = x.requires_grad_(True), w.requires_grad_(True)
    y = grouped_matmul(lx, lw, offsets, checkpoint=checkpoint)
    dx, dw = torch.autograd.grad(y, (lx, lw), dy)
    xe, we, de = x.detach()[-n:].double(), w.detach()[2].double(), dy[-n:].double()
    _close(y.detach()[-n:], xe @ we.t(), K, xe.abs() @ we.t().abs())
    _close(dx[-n:], de @ we, N, de.abs() @ we.abs())
    xk = kept(xe) if checkpoint else xe
    _close(dw[2], de.t() @ xk, n, de.t().abs() @ xk.abs())


def test_grouped_weights(gpu_device):
    """many weights: the last expert's y, dx and dW, by streaming, by tiles of 128 and of 256"""
    from lowbit.experts import grouped_matmul

    N, K = 2048, 4096
    E = (1 << 32) // (N * K) + 2
    w = _random(gpu_device, E, N, K)
    for n in (2, 100, 300):
        counts = torch.full((E,), n)
        offsets = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).int().to(gpu_device)
        x, dy = _random(gpu_device, E * n, K, seed=n), _random(gpu_device, E * n, N, seed=n + 1)
        lx, lw = x.requires_grad_(True), w.requires_grad_(True)
        y = grouped_matmul(lx, lw, offsets)
        dx, dw = torch.autograd.grad(y, (lx, lw), dy)
        xe, we, de = x.detach()[-n:].double(), w.detach()[-1].double(), dy[-n:].double()
        _close(y.detach()[-n:], xe @ we.t(), K, xe.abs() @ we.t().abs())
        _close(dx[-n:], de @ we, N, de.abs() @ we.abs())
        _close(dw[-1], de.t() @ xe, n, de.t().abs() @ xe.abs())
        del y, dx, dw
