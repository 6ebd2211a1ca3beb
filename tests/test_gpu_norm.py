"""GPU tests of lowbit.norm.layer_norm against the definition in 64 bits.

Bounds, with u = 2^-24 (fp32 arithmetic) and v the output type's rounding
(2^-24, 2^-11 fp16, 2^-8 bf16; fp16 adds its least step): a thread adds at most 64 values in sequence
and the tree over the threads adds fewer than 64 steps more, so a row sum is
off by at most 128 u times the sum of magnitudes.  That moves the mean by 128 u
mean|x| and xh by d = 256 u (r mean|x| + |xh|) (mean, its square in the
variance, root, product).  y = xh w + b and the gradients follow from that by
the triangle inequality; dw and db add T rows in some order (T u times the sum
of magnitudes).  Every comparison is elementwise against these bounds.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 0.0, torch.float16: 2.0 ** -24, torch.bfloat16: 0.0}


def _inputs(T, H, dtype, wdtype, seed, dev):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, generator=g) * torch.exp(0.5 * torch.randn(H, generator=g)) + torch.randn(T, 1, generator=g)
    w = 1 + 0.2 * torch.randn(H, generator=g)
    b = 0.3 * torch.randn(H, generator=g)
    dy = torch.randn(T, H, generator=g)
    return x.to(dtype).to(dev), w.to(wdtype).to(dev), b.to(wdtype).to(dev), dy.to(dtype).to(dev)


def _stats(x, eps):
    x = x.double()
    m = x.mean(1, keepdim=True)
    r = 1 / torch.sqrt(((x - m) ** 2).mean(1, keepdim=True) + eps)
    xh = (x - m) * r
    return xh, r, 256 * U * (r * x.abs().mean(1, keepdim=True) + xh.abs())


def _check(got, want, bound, what):
    bound = bound + ROUND[got.dtype] * want.abs() + LEAST[got.dtype] + 1e-37
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (what, int(bad.sum()), float((off / bound).nan_to_num(1e9).max()))


def _check_forward(y, x, w, b, eps):
    xh, r, d = _stats(x, eps)
    wd = torch.ones_like(xh[0]) if w is None else w.double()
    bd = torch.zeros_like(xh[0]) if b is None else b.double()
    want = xh * wd + bd
    _check(y, want, d * wd.abs() + 4 * U * ((xh * wd).abs() + bd.abs()), "y")


def _check_backward(dx, dw, db, x, w, dy, eps):
    xh, r, d = _stats(x, eps)
    T, H = x.shape
    e = dy.double()
    t = e if w is None else e * w.double()
    s0, s1 = t.mean(1, keepdim=True), (t * xh).mean(1, keepdim=True)
    if dx is not None:
        off1 = 256 * U * (t * xh).abs().mean(1, keepdim=True) + (t.abs() * d).mean(1, keepdim=True)
        bound = r * (256 * U * (t.abs() + t.abs().mean(1, keepdim=True) + (xh * s1).abs()) + d * s1.abs()
                     + xh.abs() * off1) + 512 * U * r * (t - s0 - xh * s1).abs()
        _check(dx, r * (t - s0 - xh * s1), bound, "dx")
    if dw is not None:
        _check(dw, (e * xh).sum(0), (T + 8) * U * (e * xh).abs().sum(0) + (e.abs() * d).sum(0), "dw")
    if db is not None:
        _check(db, e.sum(0), (T + 8) * U * e.abs().sum(0), "db")


SIZES = [(1, 1), (1, 7168), (3, 5), (7, 64), (2, 513), (130, 1541), (33, 4104), (5, 16384), (1100, 512), (257, 1000),
         (1, 9000), (520, 7168), (4099, 24), (700, 2047)]
TYPES = [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float32, torch.float32),
         (torch.bfloat16, torch.float32)]


@pytest.mark.parametrize("T,H", SIZES)
@pytest.mark.parametrize("dtype,wdtype", TYPES)
def test_values_and_gradients(gpu_device, T, H, dtype, wdtype):
    from lowbit.norm import layer_norm

    x, w, b, dy = _inputs(T, H, dtype, wdtype, 31 * T + H, gpu_device)
    with torch.no_grad():
        y0 = layer_norm(x, w, b, eps=1e-5)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves, eps=1e-5)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(y.detach(), y0)
    assert y.dtype == dtype and dx.dtype == dtype and dw.dtype == wdtype
    _check_forward(y.detach(), x, w, b, 1e-5)
    _check_backward(dx, dw, db, x, w, dy, 1e-5)
    again = torch.autograd.grad(layer_norm(*leaves, eps=1e-5), leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))


@pytest.mark.parametrize("which", ["pitch", "offset", "transposed", "repeated", "3d", "dy_pitch"])
def test_strides(gpu_device, which):
    """rows of a larger matrix, rows off 16 bytes, a transposed matrix, one row repeated, more axes"""
    from lowbit.norm import layer_norm

    T, H = 70, 1001
    x, w, b, dy = _inputs(T, H + 7, torch.bfloat16, torch.bfloat16, 5, gpu_device)
    w, b = w[:H], b[:H]
    if which == "pitch":
        xv, dv = x[:, :H], dy[:, :H].contiguous()
    elif which == "offset":
        xv, dv = x[:, 3:3 + H], dy[:, 1:1 + H]
    elif which == "transposed":
        xv, dv = x[:, :H].t().contiguous().t(), dy[:, :H]
    elif which == "repeated":
        xv, dv = x[:1, :H].expand(T, H), dy[:, :H]
    elif which == "3d":
        xv, dv = x[:, :H].reshape(7, 10, H), dy[:, :H].reshape(7, 10, H)
    else:
        xv, dv = x[:, :H].contiguous(), dy[:1, :H].expand(T, H)
    xl, wl, bl = xv.detach().requires_grad_(True), w.clone().requires_grad_(True), b.clone().requires_grad_(True)
    y = layer_norm(xl, wl, bl)
    dx, dw, db = torch.autograd.grad(y, (xl, wl, bl), dv)
    assert y.shape == xv.shape and dx.shape == xv.shape
    xr, dr = xv.reshape(-1, H), dv.reshape(-1, H)
    _check_forward(y.detach().reshape(-1, H), xr, w, b, 1e-5)
    _check_backward(dx.reshape(-1, H), dw, db, xr, w, dr, 1e-5)


@pytest.mark.parametrize("has_w,has_b", [(False, False), (True, False), (False, True)])
def test_without_weight_or_bias(gpu_device, has_w, has_b):
    from lowbit.norm import layer_norm

    x, w, b, dy = _inputs(40, 300, torch.float16, torch.float32, 9, gpu_device)
    w, b = (w.requires_grad_(True) if has_w else None), (b.requires_grad_(True) if has_b else None)
    xl = x.clone().requires_grad_(True)
    y = layer_norm(xl, w, b, eps=1e-3)
    y.backward(dy)
    _check_forward(y.detach(), x, w if w is None else w.detach(), b if b is None else b.detach(), 1e-3)
    _check_backward(xl.grad, w.grad if has_w else None, b.grad if has_b else None, x,
                    w if w is None else w.detach(), dy, 1e-3)


@pytest.mark.parametrize("need", [(True, False, False), (False, True, False), (False, False, True), (False, True, True)])
def test_each_gradient_alone(gpu_device, need):
    from lowbit.norm import layer_norm

    x, w, b, dy = _inputs(65, 770, torch.bfloat16, torch.bfloat16, 11, gpu_device)
    leaves = [t.clone().requires_grad_(n) for t, n in zip((x, w, b), need)]
    layer_norm(*leaves).backward(dy)
    assert [t.grad is not None for t in leaves] == list(need)
    _check_backward(*[t.grad for t in leaves], x, w, dy, 1e-5)


def test_rows_off_centre_and_constant_rows(gpu_device):
    """mean 4096 times the deviation: E[x^2] - mean^2 would lose the variance; a constant row gives exactly b"""
    from lowbit.norm import layer_norm

    g = torch.Generator().manual_seed(3)
    x = (torch.randn(6, 2000, generator=g) + 4096.0).to(gpu_device)
    x[2] = 17.25
    x[3] = 0.0
    w, b = torch.randn(2000, generator=g).to(gpu_device), torch.randn(2000, generator=g).to(gpu_device)
    y = layer_norm(x, w, b)
    _check_forward(y, x, w, b, 1e-5)
    assert torch.equal(y[2], b) and torch.equal(y[3], b)


def test_nan_and_infinity_stay_in_their_rows(gpu_device):
    from lowbit.norm import layer_norm

    x, w, b, dy = _inputs(9, 600, torch.bfloat16, torch.bfloat16, 13, gpu_device)
    clean = layer_norm(x, w, b)
    x[2, 5], x[4, 599], x[7, 0] = float("nan"), float("inf"), float("-inf")
    xl = x.clone().requires_grad_(True)
    y = layer_norm(xl, w, b)
    y.backward(dy)
    bad = torch.zeros(9, dtype=torch.bool, device=gpu_device)
    bad[[2, 4, 7]] = True
    assert torch.equal(y.detach()[~bad], clean[~bad])
    assert y.detach()[bad].isnan().all() and xl.grad[bad].isnan().all() and xl.grad[~bad].isfinite().all()


def test_no_rows(gpu_device):
    from lowbit.norm import layer_norm

    x = torch.empty(0, 96, device=gpu_device, requires_grad=True)
    w, b = (torch.ones(96, device=gpu_device, requires_grad=True) for _ in range(2))
    y = layer_norm(x, w, b)
    assert y.shape == (0, 96)
    y.sum().backward()
    assert x.grad.shape == (0, 96) and not w.grad.any() and not b.grad.any()


def test_gradients_against_differences(gpu_device):
    """d/ds of f(s) = <y(x + s p, w + s q, b + s c), dy> by central differences of the kernel's own fp32 outputs.
    With h = 2^-6 the cubic term is below h^2 |f'''| / 6 (here < 2% of |p| |dx| scale) and rounding below
    2 u sum|y dy| / 2h."""
    from lowbit.norm import layer_norm

    T, H, h = 24, 200, 2.0 ** -6
    x, w, b, dy = _inputs(T, H, torch.float32, torch.float32, 17, gpu_device)
    g = torch.Generator().manual_seed(18)
    p, q, c = (torch.randn(*s, generator=g).to(gpu_device) for s in ((T, H), (H,), (H,)))
    f = lambda s: (layer_norm(x + s * p, w + s * q, b + s * c).double() * dy.double()).sum()  # noqa: E731
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    want = sum((u.double() * v.double()).sum() for u, v in zip(grads, (p, q, c)))
    d1 = (f(h) - f(-h)) / (2 * h)
    d2 = (f(2 * h) - f(-2 * h)) / (4 * h)
    best = (4 * d1 - d2) / 3  # the h^2 term removed
    scale = float((y.detach().double() * dy.double()).abs().sum())
    assert abs(float(best - want)) <= abs(float(d1 - d2)) + 8 * U * scale / h


def test_second_gradient_is_refused(gpu_device):
    from lowbit.norm import layer_norm

    x = torch.randn(4, 8, device=gpu_device, requires_grad=True)
    (dx,) = torch.autograd.grad(layer_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def test_other_stream_and_graph(gpu_device):
    from lowbit.norm import layer_norm

    x, w, b, _ = _inputs(50, 1030, torch.bfloat16, torch.bfloat16, 21, gpu_device)
    want = layer_norm(x, w, b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = layer_norm(x, w, b)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer_norm(x, w, b)
    for k in range(3):
        x.copy_(torch.randn(50, 1030, generator=torch.Generator().manual_seed(k)).to(x))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, layer_norm(x, w, b))


def test_module(gpu_device):
    from lowbit.norm import LayerNorm

    m = LayerNorm(48, dtype=torch.bfloat16, device=gpu_device)
    x = torch.randn(5, 48, device=gpu_device).bfloat16()
    _check_forward(m(x).detach(), x, m.weight.detach(), m.bias.detach(), 1e-5)
    assert set(m.state_dict()) == {"weight", "bias"}


def test_refusals(gpu_device):
    from lowbit.norm import layer_norm

    x = torch.randn(4, 32, device=gpu_device)
    with pytest.raises(RuntimeError, match="ROCm device"):
        layer_norm(torch.randn(4, 32))
    with pytest.raises(ValueError, match="16384"):
        layer_norm(torch.randn(1, 16385, device=gpu_device))
    with pytest.raises(ValueError, match="weight"):
        layer_norm(x, torch.ones(31, device=gpu_device))
    with pytest.raises(TypeError, match="dtype"):
        layer_norm(x.double())
    with pytest.raises(TypeError, match="share"):
        layer_norm(x, torch.ones(32, device=gpu_device), torch.ones(32, device=gpu_device).half())
    with pytest.raises(ValueError, match="eps"):
        layer_norm(x, eps=-1.0)
