"""GPU tests of lowbit.experts.swiglu against the definition in 64 bits.

Bounds, with u = 2^-24: of 16-bit inputs the sigmoid's exponential is off by (|g| + 4) u (its rounded argument and the
exponential itself) and the reciprocal by 2 u, of fp32 inputs both by 4 u; products add one u each.  The derivative's
factor 1 + g (1 - sig) adds that error of (1 - sig) times |g|.  The result is rounded once (2^-24, 2^-11 fp16, 2^-8 bf16, and the
least step of fp16 and fp32; the unit's reciprocal gives no numbers below 2^-126, where 1 / (1 + t) is none).
"""

from __future__ import annotations

import pytest
import torch

from _kept import kept, values

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}


def _inputs(T, I, dtype, seed, dev, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn(T, 2 * I, generator=g)
    return x.to(dtype).to(dev), torch.randn(T, I, generator=g).to(dtype).to(dev)


def _parts(x, block):
    T, I = x.shape[0], x.shape[1] // 2
    b = block or I
    v = x.reshape(T, I // b, 2, b)
    return v[:, :, 0].reshape(T, I), v[:, :, 1].reshape(T, I)


def _joined(a, b, block):
    T, I = a.shape
    n = block or I
    return torch.stack([a.reshape(T, I // n, n), b.reshape(T, I // n, n)], 2).reshape(T, 2 * I)


def _check(got, want, bound, what):
    bound = bound + ROUND[got.dtype] * want.abs() + 2 * LEAST[got.dtype]
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), (what, int(bad.sum()), float(((got.double() - want).abs() / bound).nan_to_num(1e9).max()))


def _check_all(h, dx, x, dh, block, checkpoint):
    gate, up = (t.double() for t in _parts(x, block))
    off = 12 * U + 2 * U * gate.abs()
    want = torch.sigmoid(gate) * gate * up
    _check(h, want, want.abs() * off, "h")
    if dx is None:
        return
    if checkpoint:
        gate, up = kept(gate), kept(up)
    off = 12 * U + 2 * U * gate.abs()
    sig, d = torch.sigmoid(gate), dh.double()
    rest = torch.sigmoid(-gate)
    a = d * up * sig
    dg, du = a * (1 + gate * rest), d * gate * sig
    bound = _joined(a.abs() * (1 + (gate * rest).abs()) * (off + 4 * U) * 2, du.abs() * off, block)
    _check(dx, _joined(dg, du, block), bound, "dx")


SIZES = [(1, 1, 0), (1, 2048, 0), (3, 5, 0), (7, 64, 0), (130, 1003, 0), (33, 256, 128), (8, 2048, 128), (5, 18432, 0),
         (65, 768, 384), (2, 129, 0), (4, 128, 128), (700, 130, 0)]


@pytest.mark.parametrize("T,I,block", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_values_and_gradients(gpu_device, T, I, block, dtype):
    from lowbit.experts import swiglu

    x, dh = _inputs(T, I, dtype, 7 * T + I, gpu_device)
    with torch.no_grad():
        h0 = swiglu(x, block=block)
    for checkpoint in (None, "e4m3"):
        leaf = x.clone().requires_grad_(True)
        h = swiglu(leaf, block=block, checkpoint=checkpoint)
        (dx,) = torch.autograd.grad(h, leaf, dh)
        assert torch.equal(h.detach(), h0) and dx.dtype == dtype and dx.shape == x.shape
        _check_all(h0, dx, x, dh, block, checkpoint)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("I,block", [(5, 0), (129, 0), (1003, 0), (256, 128), (768, 256)])
def test_kept_codes(gpu_device, dtype, I, block):
    from lowbit.experts import swiglu

    x, dh = _inputs(6, I, dtype, I, gpu_device)
    x = x * torch.logspace(-5, 3, 2 * I, device=gpu_device).to(dtype)
    x[3] = 0
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
        swiglu(x.requires_grad_(True), block=block, checkpoint="e4m3")
    assert len(saved) == 2 and all(t.dtype is torch.uint8 for t in saved)
    codes, exps = sorted(saved, key=lambda t: -t.numel())
    q = values(codes, exps)
    q, codes = q.reshape(6, 2, -1), codes.reshape(6, 2, -1)
    for i, part in enumerate(_parts(x.detach(), block)):
        assert torch.equal(q[:, i, :I].nan_to_num(1234.0), kept(part).nan_to_num(1234.0)) and not codes[:, i, I:].any()


@pytest.mark.parametrize("which", ["pitch", "offset", "transposed", "repeated", "3d", "dh_pitch"])
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_strides(gpu_device, which, checkpoint):
    from lowbit.experts import swiglu

    T, I = 30, 501
    x0, dh0 = _inputs(T, I + 8, torch.bfloat16, 5, gpu_device)
    n = 2 * I
    x, dh = {"pitch": (x0[:, :n], dh0[:, :I].contiguous()), "offset": (x0[:, 3:3 + n], dh0[:, :I]),
             "transposed": (x0[:, :n].t().contiguous().t(), dh0[:, :I]),
             "repeated": (x0[:1, :n].expand(T, n), dh0[:, :I]),
             "3d": (x0[:, :n].reshape(5, 6, n), dh0[:, :I].reshape(5, 6, I)),
             "dh_pitch": (x0[:, :n].contiguous(), dh0[:1, 1:1 + I].expand(T, I))}[which]
    leaf = x.detach().requires_grad_(True)
    h = swiglu(leaf, checkpoint=checkpoint)
    (dx,) = torch.autograd.grad(h, leaf, dh)
    assert h.shape == (*x.shape[:-1], I) and dx.shape == x.shape
    _check_all(h.detach().reshape(T, I), dx.reshape(T, n), x.reshape(T, n), dh.reshape(T, I), 0, checkpoint)


def test_far_gates_and_values_that_are_not_finite(gpu_device):
    """gates far off zero neither overflow nor lose their small results; NaN and infinity stay with their element,
    also in the tile that is kept"""
    from lowbit.experts import swiglu

    gates = [-1e30, -200.0, -104.0, -88.0, -60.0, -20.0, -1.278, -0.0, 0.0, 1e-30, 20.0, 90.0, 200.0, 1e30]
    x = torch.tensor([gates + [1.5] * len(gates)], device=gpu_device)
    dh = torch.ones(1, len(gates), device=gpu_device)
    leaf = x.clone().requires_grad_(True)
    h = swiglu(leaf)
    (dx,) = torch.autograd.grad(h, leaf, dh)
    _check_all(h.detach(), dx, x, dh, 0, None)
    x, dh = _inputs(4, 200, torch.bfloat16, 3, gpu_device)
    whole = swiglu(x)
    x[1, 7], x[2, 203], x[3, 130] = float("nan"), float("inf"), float("inf")
    at = torch.zeros(4, 200, dtype=torch.bool, device=gpu_device)
    at[1, 7] = at[2, 3] = at[3, 130] = True
    for checkpoint in (None, "e4m3"):
        leaf = x.clone().requires_grad_(True)
        h = swiglu(leaf, checkpoint=checkpoint)
        assert torch.equal(h.detach()[~at], whole[~at]) and not h.detach()[at].isfinite().any()
        (dx,) = torch.autograd.grad(h, leaf, dh)
        ok = ~torch.cat([at, at], 1)
        assert dx[ok].isfinite().all()


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_no_rows(gpu_device, checkpoint):
    from lowbit.experts import swiglu

    x = torch.empty(0, 64, device=gpu_device, requires_grad=True)
    h = swiglu(x, checkpoint=checkpoint)
    assert h.shape == (0, 32)
    h.sum().backward()
    assert x.grad.shape == (0, 64)


def test_gradient_against_differences(gpu_device):
    """central differences of the kernel's own fp32 outputs, the h^2 term removed"""
    from lowbit.experts import swiglu

    step = 2.0 ** -6
    x, dh = _inputs(16, 100, torch.float32, 17, gpu_device)
    p = torch.randn(16, 200, generator=torch.Generator().manual_seed(2)).to(gpu_device)
    f = lambda k: (swiglu(x + k * p).double() * dh.double()).sum()  # noqa: E731
    leaf = x.clone().requires_grad_(True)
    h = swiglu(leaf)
    (dx,) = torch.autograd.grad(h, leaf, dh)
    want = (dx.double() * p.double()).sum()
    d1, d2 = (f(step) - f(-step)) / (2 * step), (f(2 * step) - f(-2 * step)) / (4 * step)
    scale = float((h.detach().double() * dh.double()).abs().sum())
    assert abs(float((4 * d1 - d2) / 3 - want)) <= abs(float(d1 - d2)) + 32 * U * scale / step


def test_other_stream_graph_and_second_uses(gpu_device):
    from lowbit.experts import swiglu

    x, dh = _inputs(50, 515, torch.bfloat16, 21, gpu_device)
    leaf = x.clone().requires_grad_(True)

    def step():
        h = swiglu(leaf, checkpoint="e4m3")
        return h.detach(), *torch.autograd.grad(h, leaf, dh)

    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        with torch.no_grad():
            leaf.copy_(torch.randn(50, 1030, generator=torch.Generator().manual_seed(k)).to(x))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))
    moved = leaf * 1
    h = swiglu(moved)
    with torch.no_grad():
        moved.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(h, leaf, dh)
    (dx,) = torch.autograd.grad(swiglu(leaf).square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def test_refusals(gpu_device):
    from lowbit.experts import swiglu

    x = torch.randn(4, 512, device=gpu_device)
    with pytest.raises(RuntimeError, match="ROCm device"):
        swiglu(torch.randn(4, 32))
    with pytest.raises(ValueError, match="2I"):
        swiglu(x[:, :31])
    with pytest.raises(ValueError, match="2I"):
        swiglu(x[:, :0])
    with pytest.raises(TypeError, match="dtype"):
        swiglu(x.double())
    for block in (64, -128, 384):
        with pytest.raises(ValueError, match="block"):
            swiglu(x, block=block)
    with pytest.raises(ValueError, match="checkpoint"):
        swiglu(x, checkpoint="int8")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_far_gates_keep_what_the_type_holds(gpu_device, dtype, checkpoint):
    """the sigmoid of a gate below -87.3 lies under the normal numbers of fp32 and of bf16, its product with the gate, up
    and the incoming gradient need not: each comes out within the bounds, up to gates of -174"""
    from lowbit.experts import swiglu

    gates = torch.tensor([-60.0, -80.0, -87.0, -87.5, -88.0, -90.0, -92.0, -96.0, -103.0, -104.0, -120.0, -144.0, -160.0,
                          60.0, 88.0, 104.0, 160.0] + [-168.0, -174.0] * (checkpoint is None))
    ups = torch.tensor([1.0, -3.0, 1e10, -1e20, 1e30, 2.5e38])
    incoming = torch.tensor([1.0, -1e5, 1e25])
    rows = torch.cartesian_prod(gates, ups, incoming)
    # neither dh up nor h past the largest number
    rows = rows[(rows[:, 1:].prod(1).abs() < 3e38) & ((rows[:, 0] < 0) | (rows[:, 1:].prod(1).abs() < 1e36))]
    # one value a row: a kept tile is its own
    x = rows[:, :2].to(dtype).to(gpu_device)
    dh = rows[:, 2:].to(dtype).to(gpu_device)
    leaf = x.clone().requires_grad_(True)
    h = swiglu(leaf, checkpoint=checkpoint)
    (dx,) = torch.autograd.grad(h, leaf, dh)
    _check_all(h.detach(), dx, x, dh, 0, checkpoint)


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_more_rows_than_a_launch_has_tiles(gpu_device, checkpoint):
    """fp32 rows of one tile each, whose threads in one launch would be 2^32"""
    from lowbit.experts import swiglu

    T = (1 << 27) + 3
    x = torch.randn(T, 2, generator=torch.Generator(gpu_device).manual_seed(1), device=gpu_device).requires_grad_(True)
    h = swiglu(x, checkpoint=checkpoint)
    (dx,) = torch.autograd.grad(h, x, torch.ones_like(h))
    for part in (slice(0, 5000), slice((1 << 26) - 5000, (1 << 26) + 5000), slice(T - 5000, T)):
        _check_all(h.detach()[part], dx[part], x.detach()[part], torch.ones_like(h[part]).detach(), 0, checkpoint)
    with torch.no_grad():  # no row left out: fp32's own formula, both sides off by less than 32 u
        want = x[:, :1] / (1 + torch.exp(-x[:, :1])) * x[:, 1:]
        assert ((h - want).abs() <= 64 * U * want.abs() + 2.0 ** -126).all()
