"""GPU tests of lowbit.loss.linear_cross_entropy against the definition in 64 bits.

Bounds, with u = 2^-24 and S_t = max over the words of sum_h |x_th w_vh|: a
logit adds H exact products in fp32, H roundings of at most u S each, taken as
independent: off by at most e = 4 sqrt(H) u S (four deviations).  A loss moves
by at most twice that, plus 16 u of |logsumexp| and the logit (exp, log, the
joins).  dz = u_t (p - 1[y]) is off by 4 e + 32 u |lse| relative to u_t p and
rounded to bf16 once (2^-8); dX and dW follow elementwise by the triangle
inequality over their sums, with 4 sqrt(n) u for the n additions and the
output's 2^-8.  The roundings of dz and of the output are independent, each of
at most 2^-8 and 2^-8 / sqrt(3) in the mean square, so a gradient as a whole is
within 2^-8 in the Frobenius norm.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
B = 2.0 ** -8
IGNORE = -100


def _inputs(T, H, V, seed, dev, ignored=0.0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, H, generator=g) * 0.05).bfloat16()
    y = torch.randint(0, V, (T,), generator=g)
    x = ((torch.randn(T, H, generator=g) + 20.0 / math.sqrt(H) * torch.rand(T, 1, generator=g) * w[y].float()) * scale)
    y = torch.where(torch.rand(T, generator=g) < ignored, IGNORE, y)
    return x.bfloat16().to(dev), w.to(dev), y.to(dev), g


def _check(x, w, y, loss, dx, dw, reduction, dloss, ignore=IGNORE):
    """loss / dx / dw (each may be None) of 2-D x against 64 bits"""
    T, H = x.shape
    V = w.shape[0]
    live = y != ignore
    xd, wd = torch.where(live[:, None], x.double(), 0.0), w.double()
    z = xd @ wd.t()
    lse = torch.logsumexp(z, 1)
    at = torch.where(live, y, 0).long()[:, None]
    each = torch.where(live, lse - z.gather(1, at)[:, 0], 0.0)
    n = max(1, int(live.sum()))
    e = 4 * math.sqrt(H) * U * (xd.abs() @ wd.abs().t()).amax(1)
    off = torch.where(live, 2 * e + 16 * U * (lse.abs() + z.gather(1, at)[:, 0].abs()), 0.0)
    if loss is not None:
        if reduction == "none":
            want, bound = each, off
        else:
            div = n if reduction == "mean" else 1
            want, bound = each.sum() / div, (off.sum() + 4 * math.sqrt(n) * U * each.sum()) / div
        assert loss.dtype == torch.float32 and ((loss.double() - want).abs() <= bound).all()
    if dx is None and dw is None:
        return
    up = (dloss.double() if reduction == "none" else (dloss.double() / (n if reduction == "mean" else 1)).expand(T))
    up = torch.where(live, up, 0.0)[:, None]
    p = torch.softmax(z, 1)
    dz = p.clone().scatter_add_(1, at, torch.full_like(up, -1.0)) * up
    err = B * dz.abs() + up.abs() * p * (4 * e + 32 * U * lse.abs())[:, None]
    for got, want, mag, er, terms in ((dx, lambda m: m @ wd, lambda m: m @ wd.abs(), err, V),
                                      (dw, lambda m: m.t() @ xd, lambda m: m.t() @ xd.abs(), err, n)):
        if got is None:
            continue
        want = want(dz)
        bound = mag(er) + 4 * math.sqrt(terms) * U * mag(dz.abs()) + B * want.abs() + 1e-37
        diff = (got.double() - want).abs()
        assert got.dtype == torch.bfloat16 and (diff <= bound).all(), float((diff / bound).max())
        if want.norm() > 0:
            assert diff.norm() <= B * want.norm(), float(diff.norm() / want.norm())


SIZES = [(1, 64, 256), (1, 8, 1), (3, 5, 7), (16, 1024, 3001), (257, 1000, 5003), (300, 513, 700), (64, 72, 260),
         (1003, 520, 2111), (513, 192, 20011), (37, 2048, 9000), (255, 64, 257), (600, 1541, 500), (2049, 300, 1023)]


@pytest.mark.parametrize("T,H,V", SIZES)
@pytest.mark.parametrize("reduction,ignored", [("mean", 0.0), ("none", 0.4), ("sum", 0.05)])
def test_loss_and_gradients(gpu_device, T, H, V, reduction, ignored):
    from lowbit.loss import linear_cross_entropy

    x, w, y, g = _inputs(T, H, V, T + H + V, gpu_device, ignored)
    with torch.no_grad():
        l0 = linear_cross_entropy(x, w, y, reduction=reduction)
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = linear_cross_entropy(xl, wl, y, reduction=reduction)
    dl = (torch.randn(T, generator=g) if reduction == "none" else torch.tensor(0.7)).to(gpu_device)
    dx, dw = torch.autograd.grad(loss, (xl, wl), dl, retain_graph=True)
    assert loss.shape == ((T,) if reduction == "none" else ()) and torch.equal(loss.detach(), l0)
    _check(x, w, y, loss.detach(), dx, dw, reduction, dl)
    again = torch.autograd.grad(loss, (xl, wl), dl)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])


def test_several_pieces_of_the_vocabulary(gpu_device):
    from lowbit.loss import linear_cross_entropy

    T, H, V = 8192, 64, 40001
    x, w, y, _ = _inputs(T, H, V, 3, gpu_device, 0.02)
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = linear_cross_entropy(xl, wl, y)
    dx, dw = torch.autograd.grad(loss, (xl, wl))
    _check(x, w, y, loss.detach(), dx, dw, "mean", torch.ones((), device=gpu_device))


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_all_ignored(gpu_device, reduction):
    from lowbit.loss import linear_cross_entropy

    x, w, y, _ = _inputs(70, 96, 300, 4, gpu_device)
    y[:] = IGNORE
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = linear_cross_entropy(xl, wl, y, reduction=reduction)
    assert not loss.detach().any()
    loss.sum().backward()
    assert not xl.grad.any() and not wl.grad.any() and xl.grad.isfinite().all()


def test_ignored_rows_cannot_pass_on_a_nan(gpu_device):
    """ignored rows hold NaN and infinity; the ignore index may lie inside the vocabulary"""
    from lowbit.loss import linear_cross_entropy

    x, w, y, _ = _inputs(400, 200, 900, 5, gpu_device)
    y[::3] = 17
    x[::3] = float("nan")
    x[3] = float("inf")
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = linear_cross_entropy(xl, wl, y, ignore_index=17, reduction="sum")
    dx, dw = torch.autograd.grad(loss, (xl, wl))
    assert not dx[::3].any()
    _check(x.nan_to_num(0.0, 0.0), w, y, loss.detach(), dx, dw, "sum", torch.ones((), device=gpu_device), ignore=17)


def test_a_target_outside_the_vocabulary_is_loud(gpu_device):
    from lowbit.loss import linear_cross_entropy

    x, w, y, _ = _inputs(50, 64, 300, 6, gpu_device)
    want = linear_cross_entropy(x, w, y, reduction="none")
    y[7], y[9] = 300, -1
    xl = x.clone().requires_grad_(True)
    loss = linear_cross_entropy(xl, w, y, reduction="none")
    bad = torch.zeros(50, dtype=torch.bool, device=gpu_device)
    bad[[7, 9]] = True
    assert loss.detach()[bad].isnan().all() and torch.equal(loss.detach()[~bad], want[~bad])
    loss.sum().backward()
    assert xl.grad[bad].isnan().all() and xl.grad[~bad].isfinite().all()


def test_nan_and_infinite_rows(gpu_device):
    from lowbit.loss import linear_cross_entropy

    x, w, y, _ = _inputs(20, 64, 700, 7, gpu_device)
    want = linear_cross_entropy(x, w, y, reduction="none")
    x[3, 5], x[8, 0] = float("nan"), float("inf")
    loss = linear_cross_entropy(x, w, y, reduction="none")
    bad = torch.zeros(20, dtype=torch.bool, device=gpu_device)
    bad[[3, 8]] = True
    assert loss[bad].isnan().all() and torch.equal(loss[~bad], want[~bad])


def test_large_logits(gpu_device):
    """logits of several hundred: exp overflows without the maximum taken off"""
    from lowbit.loss import linear_cross_entropy

    x, w, y, _ = _inputs(130, 512, 1500, 8, gpu_device, scale=300.0)
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = linear_cross_entropy(xl, wl, y, reduction="none")
    dl = torch.ones(130, device=gpu_device)
    dx, dw = torch.autograd.grad(loss, (xl, wl), dl)
    assert loss.max() > 300
    _check(x, w, y, loss.detach(), dx, dw, "none", dl)


@pytest.mark.parametrize("which", ["pitch", "offset", "repeated", "3d", "weight_pitch", "weight_offset", "weight_t",
                                   "int32", "targets_strided"])
def test_strides_and_types(gpu_device, which):
    from lowbit.loss import linear_cross_entropy

    T, H, V = 60, 256, 800
    x, w, y, _ = _inputs(T, H + 16, V, 9, gpu_device, 0.1)
    xv, wv, yv = x[:, :H].contiguous(), w[:, :H].contiguous(), y
    if which == "pitch":
        xv = x[:, :H]
    elif which == "offset":
        xv = x[:, 5:5 + H]
    elif which == "repeated":
        xv = x[:1, :H].expand(T, H)
    elif which == "3d":
        xv, yv = x[:, :H].reshape(6, 10, H), y.reshape(6, 10)
    elif which == "weight_pitch":
        wv = w[:, 8:8 + H]
    elif which == "weight_offset":
        wv = w[:, 3:3 + H]
    elif which == "weight_t":
        wv = w[:, :H].t().contiguous().t()
    elif which == "int32":
        yv = y.int()
    else:
        yv = torch.stack([y, y + 1], 1)[:, 0]
    xl, wl = xv.detach().requires_grad_(True), wv.detach().requires_grad_(True)
    loss = linear_cross_entropy(xl, wl, yv, reduction="sum")
    dx, dw = torch.autograd.grad(loss, (xl, wl))
    assert dx.shape == xv.shape and dw.shape == wv.shape
    _check(xv.reshape(T, H), wv, yv.reshape(T), loss.detach(), dx.reshape(T, H), dw, "sum",
           torch.ones((), device=gpu_device))


@pytest.mark.parametrize("which", ["hidden", "weight"])
def test_one_gradient_alone(gpu_device, which):
    from lowbit.loss import linear_cross_entropy

    x, w, y, _ = _inputs(90, 128, 1000, 10, gpu_device, 0.2)
    xl, wl = x.clone().requires_grad_(which == "hidden"), w.clone().requires_grad_(which == "weight")
    loss = linear_cross_entropy(xl, wl, y)
    loss.backward()
    assert (xl.grad is None) == (which != "hidden") and (wl.grad is None) == (which != "weight")
    _check(x, w, y, loss.detach(), xl.grad, wl.grad, "mean", torch.ones((), device=gpu_device))


def test_no_positions(gpu_device):
    from lowbit.loss import linear_cross_entropy

    x = torch.empty(0, 64, device=gpu_device, dtype=torch.bfloat16, requires_grad=True)
    w = torch.randn(100, 64, device=gpu_device).bfloat16().requires_grad_(True)
    y = torch.empty(0, dtype=torch.int64, device=gpu_device)
    for reduction in ("mean", "sum", "none"):
        loss = linear_cross_entropy(x, w, y, reduction=reduction)
        dx, dw = torch.autograd.grad(loss.sum(), (x, w))
        assert float(loss.detach().sum()) == 0 and dx.shape == (0, 64) and not dw.any()


def test_gradient_against_differences(gpu_device):
    """central differences of the kernel's own losses along directions that bf16 holds exactly: x and w are whole
    multiples of 2^-6 and the steps of 2^-5, all below 2 in magnitude.  The h^2 term is removed by h and 2h; the
    gradients are bf16 (2^-8 of the magnitudes that meet) and the losses off by 2 e each."""
    from lowbit.loss import linear_cross_entropy

    T, H, V, h = 20, 32, 50, 2.0 ** -5
    g = torch.Generator().manual_seed(11)
    q = lambda *s: (torch.randint(-64, 65, s, generator=g).float() / 64).to(gpu_device)  # noqa: E731
    x, w = q(T, H), q(V, H)
    sx = torch.randint(-1, 2, (T, H), generator=g).float().to(gpu_device)
    sw = torch.randint(-1, 2, (V, H), generator=g).float().to(gpu_device)
    y = torch.randint(0, V, (T,), generator=g).to(gpu_device)
    f = lambda a, b: linear_cross_entropy((x + a * sx).bfloat16(), (w + b * sw).bfloat16(), y,  # noqa: E731
                                          reduction="none").double().sum()
    xl, wl = x.bfloat16().requires_grad_(True), w.bfloat16().requires_grad_(True)
    dx, dw = torch.autograd.grad(linear_cross_entropy(xl, wl, y, reduction="sum"), (xl, wl))
    assert torch.equal((x + 2 * h * sx).bfloat16().float(), x + 2 * h * sx)
    p = torch.softmax(x.double() @ w.double().t(), 1)
    dz = p.scatter_add(1, y[:, None], torch.full((T, 1), -1.0, dtype=torch.float64, device=gpu_device)).abs()
    e = 4 * math.sqrt(H) * U * float((x.abs() @ w.abs().t()).max()) + 32 * U * 10
    for a, b, got, mag in ((1, 0, (dx.double() * sx).sum(), (dz @ w.double().abs() * sx.abs()).sum()),
                           (0, 1, (dw.double() * sw).sum(), (dz.t() @ x.double().abs() * sw.abs()).sum())):
        d1 = (f(a * h, b * h) - f(-a * h, -b * h)) / (2 * h)
        d2 = (f(2 * a * h, 2 * b * h) - f(-2 * a * h, -2 * b * h)) / (4 * h)
        # independent roundings of bf16, far fewer than their worst sum: their magnitudes' sum bounds them
        assert abs(float((4 * d1 - d2) / 3 - got)) <= abs(float(d1 - d2)) + 2 * B * float(mag) + 4 * T * e / h


def test_other_stream_and_graph(gpu_device):
    from lowbit.loss import linear_cross_entropy

    x, w, y, _ = _inputs(100, 320, 3000, 12, gpu_device, 0.3)
    want = linear_cross_entropy(x, w, y)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = linear_cross_entropy(x, w, y)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = linear_cross_entropy(x, w, y)
    for k in range(3):
        x2, _, y2, _ = _inputs(100, 320, 3000, 20 + k, gpu_device, 0.2 * k)
        x.copy_(x2)
        y.copy_(y2)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, linear_cross_entropy(x, w, y))


def test_module(gpu_device):
    from lowbit.loss import LMHeadLoss

    x, w, y, _ = _inputs(30, 64, 500, 13, gpu_device)
    m = LMHeadLoss(64, 500, weight=torch.nn.Parameter(w))
    m(x, y).backward()
    _check(x, w, y, None, None, m.weight.grad, "mean", torch.ones((), device=gpu_device))
    assert LMHeadLoss(64, 500, device=gpu_device).weight.dtype == torch.bfloat16
    with pytest.raises(ValueError, match="weight"):
        LMHeadLoss(64, 501, weight=m.weight)


def test_refusals(gpu_device):
    from lowbit.loss import linear_cross_entropy

    x, w, y, _ = _inputs(4, 64, 100, 14, gpu_device)
    with pytest.raises(RuntimeError, match="ROCm device"):
        linear_cross_entropy(x.cpu(), w.cpu(), y.cpu())
    with pytest.raises(TypeError, match="bfloat16"):
        linear_cross_entropy(x.float(), w, y)
    with pytest.raises(TypeError, match="int32 or int64"):
        linear_cross_entropy(x, w, y.float())
    with pytest.raises(ValueError, match="reduction"):
        linear_cross_entropy(x, w, y, reduction="max")
    with pytest.raises(ValueError, match="weight"):
        linear_cross_entropy(x, w[:, :32], y)
    with pytest.raises(ValueError, match="targets"):
        linear_cross_entropy(x, w, y[:3])


@pytest.mark.parametrize("n", [3, 331, 1000])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_a_common_factor_is_not_rounded(gpu_device, n, reduction):
    """the factor 1 / n of a mean enters in fp32: rounded into the operands it would scale the whole gradient, so the
    part of the gradient along the true one is looked at, where independent roundings average out: (dx, want) /
    (want, want) - 1 is a weighted mean of n * H relative errors of at most 2 * 2^-8 and at most 2^-8 correlated
    in a row through p - 1; with the labels' p below 1/8 the latter's error is at most 2^-8 / 8"""
    from lowbit.loss import linear_cross_entropy

    g = torch.Generator().manual_seed(n)
    H, V = 256, 4000
    x, w = torch.randn(n, H, generator=g).bfloat16().to(gpu_device), (torch.randn(V, H, generator=g) * 0.05).bfloat16().to(gpu_device)
    y = torch.randint(0, V, (n,), generator=g).to(gpu_device)
    xl = x.clone().requires_grad_(True)
    loss = linear_cross_entropy(xl, w, y, reduction=reduction)
    (dx,) = torch.autograd.grad(loss, xl, torch.full((n,), 1.0 / n, device=gpu_device) if reduction == "none" else None)
    p = torch.softmax(x.double() @ w.double().t(), 1)
    assert p.gather(1, y[:, None]).max() < 0.125
    want = p.scatter_add(1, y[:, None], torch.full((n, 1), -1.0, dtype=torch.float64, device=gpu_device)) @ w.double() / n
    part = float((dx.double() * want).sum() / (want * want).sum()) - 1
    assert abs(part) <= B / 8 + 4 * 2 * B / math.sqrt(n * H)


@pytest.mark.parametrize("live", [1, 63, 64, 65, 128, 129])
@pytest.mark.parametrize("T", [200, 1100])
def test_memory_past_the_live_rows_takes_no_part(gpu_device, T, live):
    """the contraction over positions ends inside a block of 64: whatever the workspace held there before, here NaN"""
    from lowbit.loss import linear_cross_entropy

    x, w, y, _ = _inputs(T, 200, 3000, live, gpu_device)
    y[torch.randperm(T, generator=torch.Generator().manual_seed(live))[live:].to(gpu_device)] = IGNORE
    x[y == IGNORE] = float("nan")
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    for _ in range(2):
        torch.cuda.empty_cache()
        junk = [torch.full((16 << 20,), float("nan"), device=gpu_device) for _ in range(4)]
        junk += [torch.full((64 << 10,), float("nan"), device=gpu_device) for _ in range(64)]
        del junk
        loss = linear_cross_entropy(xl, wl, y)
        dx, dw = torch.autograd.grad(loss, (xl, wl))
        _check(torch.where((y == IGNORE)[:, None], torch.zeros_like(x), x), w, y, loss.detach(), dx, dw, "mean",
               torch.ones((), device=gpu_device))


@pytest.mark.parametrize("T", [1, 5, 1000])
@pytest.mark.parametrize("scale", [1.0, 30.0])
def test_few_rows_of_many_words(gpu_device, T, scale):
    """hundreds of tiles' pairs to a row, of far apart maxima"""
    from lowbit.loss import linear_cross_entropy

    x, w, y, _ = _inputs(T, 64, 40001, T, gpu_device, 0.2, scale)
    for reduction in ("none", "sum"):
        with torch.no_grad():
            _check(x, w, y, linear_cross_entropy(x, w, y, reduction=reduction), None, None, reduction, None)
    w2 = w.clone()
    w2[:39000] = -float("inf")  # rows of -inf, inf and NaN products: the pairs of whole tiles hold no number
    x2 = x.abs()
    x2[x2 == 0] = 1.0
    live = y != IGNORE
    y2 = torch.where(live, 39000 + y % 1001, y)
    z = x2.double() @ w[39000:].double().t()
    want = torch.logsumexp(z, 1) - z.gather(1, torch.where(live, y2 - 39000, 0)[:, None])[:, 0]
    with torch.no_grad():
        got = linear_cross_entropy(x2, w2, y2, reduction="none").double()
    e = 4 * math.sqrt(64) * U * (x2.double().abs() @ w[39000:].double().abs().t()).amax(1)
    bound = 2 * e + 16 * U * (torch.logsumexp(z, 1).abs() + z.abs().amax(1))
    assert ((got - want).abs() <= bound)[live].all() and (got[~live] == 0).all()


def test_too_large_is_refused():
    """before anything is read or launched"""
    from lowbit import _lib

    p = 4096
    for T, H, V, ldw in (((1 << 22) + 1, 64, 64, 64), (8, (1 << 20) + 8, 64, (1 << 20) + 8), (8, 64, (1 << 30) + 1, 64),
                         (1 << 22, 64, 1 << 19, 64), (8, 1 << 20, 1 << 18, 1 << 20), (1 << 22, 4096, 64, 4096)):
        with pytest.raises(_lib.LowBitKernelError, match="too large"):
            _lib.call("ntlb_linear_xent_forward", p, H, p, ldw, p, 1, T, H, V, -100, 2, p, p, p, 1 << 60, 0)


@pytest.mark.parametrize("T,H,V", [(1, 7168, 300), (3, 6413, 265), (16, 4096, 1000), (17, 2000, 129), (129, 2500, 700), (300, 5000, 257),
                                   (5, 1280, 66001)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_a_divided_contraction(gpu_device, T, H, V, reduction):
    """few tiles of long rows, whose contraction workgroups share: the sums come in a fixed order, call after call and
    whatever the memory held, with ignored rows and none at all"""
    from lowbit.loss import linear_cross_entropy

    x, w, y, g = _inputs(T, H, V, T + H, gpu_device, 0.3)
    dl = (torch.randn(T, generator=g) if reduction == "none" else torch.tensor(1.3)).to(gpu_device)
    first = None
    for k in range(4):
        junk = torch.full((8 << 20,), float("nan"), device=gpu_device)
        del junk
        xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        loss = linear_cross_entropy(xl, wl, y, reduction=reduction)
        got = (loss.detach(), *torch.autograd.grad(loss, (xl, wl), dl))
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))
    _check(x, w, y, *first, reduction, dl)
    none = torch.full_like(y, IGNORE)
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = linear_cross_entropy(xl, wl, none, reduction=reduction)
    assert (loss == 0).all()
    assert all((t == 0).all() for t in torch.autograd.grad(loss, (xl, wl), dl))


@pytest.mark.parametrize("R,H,pitch,off", [(1, 1, 1, 0), (5, 7, 7, 1), (70000, 3, 5, 0), (300, 345, 345, 0), (33, 1000, 1003, 3), (9, 8, 8, 2),
                                           (4, 20001, 20001, 0)])
def test_pad_rows(gpu_device, R, H, pitch, off):
    """each value to its place, zeros past H, nothing past the rows"""
    from lowbit import _lib

    src = torch.randint(-32768, 32767, (off + R * pitch,), dtype=torch.int16, device=gpu_device)
    Hp = (H + 7) // 8 * 8 + 8 * (R % 2)
    out = torch.full((R + 1, Hp), 77, dtype=torch.int16, device=gpu_device)
    s = torch.cuda.current_stream().cuda_stream
    _lib.call("ntlb_pad_rows", src.data_ptr() + 2 * off, pitch, R, H, out.data_ptr(), Hp, s)
    x = src[off:].as_strided((R, H), (pitch, 1)) if pitch else None
    assert torch.equal(out[:R, :H], x) and (out[:R, H:] == 0).all() and (out[R] == 77).all()


def test_pad_rows_refuses():
    from lowbit import _lib

    for args in ((4096, 8, -1, 8, 4096, 8, 0), (4096, 8, 4, 8, 4096, 7, 0), (4096, 8, 4, 9, 4096, 8, 0), (4096, 8, 4, 8, 4098, 8, 0),
                 (0, 8, 4, 8, 4096, 8, 0)):
        with pytest.raises(ValueError, match="ntlb_pad_rows"):
            _lib.call("ntlb_pad_rows", *args)


@pytest.mark.parametrize("T,H,V", [(5, 4096, 300), (40, 2048, 1000), (1100, 256, 3000), (20, 1280, 66001)])
@pytest.mark.parametrize("reduction", [0, 2])
def test_both_directions_replay_in_a_graph(gpu_device, T, H, V, reduction):
    """the calls of a step captured once, with contractions divided or not, and replayed over new values and dirty
    memory: every replay equals the eager step"""
    from lowbit import _lib
    from lowbit.loss import linear_cross_entropy

    L = _lib.lib()
    new = lambda n: torch.full((n,), 255, dtype=torch.uint8, device=gpu_device)  # noqa: E731
    x, w, y, _ = _inputs(T, H, V, 1, gpu_device, 0.3)
    loss = torch.empty(T if reduction == 0 else 1, device=gpu_device)
    dl = torch.rand(T if reduction == 0 else 1, device=gpu_device)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    state, fws, bws = (new(n) for n in (L.ntlb_linear_xent_state_bytes(T, H), max(16, L.ntlb_linear_xent_workspace_bytes(T, H, V, 0)),
                                        L.ntlb_linear_xent_workspace_bytes(T, H, V, 1)))

    def step():
        s = torch.cuda.current_stream().cuda_stream
        _lib.call("ntlb_linear_xent_forward", x.data_ptr(), H, w.data_ptr(), H, y.data_ptr(), 1, T, H, V, IGNORE, reduction,
                  loss.data_ptr(), state.data_ptr(), fws.data_ptr(), fws.numel(), s)
        _lib.call("ntlb_linear_xent_backward", state.data_ptr(), w.data_ptr(), H, T, H, V, reduction, dl.data_ptr(),
                  dx.data_ptr(), H, dw.data_ptr(), H, bws.data_ptr(), bws.numel(), s)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in range(4):
        x2, w2, y2, _ = _inputs(T, H, V, 30 + k, gpu_device, 0.25 * k)
        x.copy_(x2)
        w.copy_(w2)
        y.copy_(y2)
        state.fill_(255)
        fws.fill_(255)
        bws.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        want = linear_cross_entropy(xl, wl, y, reduction=("none", "sum", "mean")[reduction])
        gx, gw = torch.autograd.grad(want, (xl, wl), dl if reduction == 0 else dl[0])
        assert torch.equal(loss, want.detach().reshape(-1)) and torch.equal(dx, gx) and torch.equal(dw, gw)


@pytest.mark.parametrize("T", [1, 40, 64, 65, 300])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("others", ["zero", "bad", "one"])
def test_incoming_gradients_that_are_no_numbers(gpu_device, T, bad, others):
    """a position whose incoming gradient is infinite or NaN passes it on, whatever the others' are; so does none that is
    ignored"""
    from lowbit.loss import linear_cross_entropy

    x, w, y, _ = _inputs(T, 128, 500, 31, gpu_device)
    at = T // 2
    dl = torch.full((T,), {"zero": 0.0, "bad": bad, "one": 1.0}[others], device=gpu_device)
    dl[at] = bad
    rows = dl != dl if bad != bad else dl == bad
    for which in ("both", "hidden", "weight"):
        xl, wl = x.clone().requires_grad_(which != "weight"), w.clone().requires_grad_(which != "hidden")
        linear_cross_entropy(xl, wl, y, reduction="none").backward(dl)
        if which != "weight":
            assert not xl.grad[rows].isfinite().any() and xl.grad[~rows].isfinite().all()
            assert others == "one" or not xl.grad[~rows].any()
        if which != "hidden":
            assert not wl.grad.isfinite().any()
    y[at] = IGNORE
    rows[at] = False
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    linear_cross_entropy(xl, wl, y, reduction="none").backward(dl)
    assert not xl.grad[at].any()
    if not rows.any():
        assert xl.grad.isfinite().all() and wl.grad.isfinite().all()
        assert others == "one" or not (xl.grad.any() or wl.grad.any())


@pytest.mark.parametrize("H", [64, 1000])
def test_an_empty_batch_stays_inside_its_state(gpu_device, H):
    from lowbit import _lib

    V = 300
    L = _lib.lib()
    nb, nw = L.ntlb_linear_xent_state_bytes(0, H), L.ntlb_linear_xent_workspace_bytes(0, H, V, 1)
    state = torch.full((nb + 65536,), 255, dtype=torch.uint8, device=gpu_device)
    ws = torch.full((nw + 65536,), 255, dtype=torch.uint8, device=gpu_device)
    w, dw = torch.randn(V, H, device=gpu_device).bfloat16(), torch.full((V, H), 7.0, device=gpu_device).bfloat16()
    loss, dl = torch.ones(1, device=gpu_device), torch.ones(1, device=gpu_device)
    s = torch.cuda.current_stream().cuda_stream
    _lib.call("ntlb_linear_xent_forward", None, H, w.data_ptr(), H, None, 1, 0, H, V, IGNORE, 2, loss.data_ptr(),
              state.data_ptr(), ws.data_ptr(), 0, s)
    _lib.call("ntlb_linear_xent_backward", state.data_ptr(), w.data_ptr(), H, 0, H, V, 2, dl.data_ptr(), None, H, dw.data_ptr(), H,
              ws.data_ptr(), nw, s)
    assert float(loss) == 0 and not dw.any()
    assert (state[nb:] == 255).all() and (ws[nw:] == 255).all()


@pytest.mark.parametrize("reduction", [0, 1, 2])
def test_an_empty_batch_reads_no_incoming_gradient(gpu_device, reduction):
    from lowbit import _lib

    H, V = 72, 300
    L = _lib.lib()
    new = lambda n: torch.full((n,), 255, dtype=torch.uint8, device=gpu_device)  # noqa: E731
    w, dw = torch.randn(V, H, device=gpu_device).bfloat16(), torch.full((V, H), 7.0, device=gpu_device).bfloat16()
    state, ws = new(L.ntlb_linear_xent_state_bytes(0, H)), new(L.ntlb_linear_xent_workspace_bytes(1, H, V, 1))
    loss = torch.ones(1, device=gpu_device)
    s = torch.cuda.current_stream().cuda_stream
    _lib.call("ntlb_linear_xent_forward", None, H, w.data_ptr(), H, None, 1, 0, H, V, IGNORE, reduction, loss.data_ptr(),
              state.data_ptr(), ws.data_ptr(), ws.numel(), s)
    _lib.call("ntlb_linear_xent_backward", state.data_ptr(), w.data_ptr(), H, 0, H, V, reduction, None, None, H, dw.data_ptr(), H,
              ws.data_ptr(), ws.numel(), s)
    assert not dw.any() and (reduction == 0 or float(loss) == 0)


@pytest.mark.parametrize("T", [3, 64, 200])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_no_live_position_passes_nothing_on(gpu_device, T, reduction):
    """all ignored: zero gradients, whatever the incoming one"""
    from lowbit.loss import linear_cross_entropy

    x, w, y, _ = _inputs(T, 64, 300, 41, gpu_device)
    y[:] = IGNORE
    for up in (float("nan"), float("inf")):
        xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        loss = linear_cross_entropy(xl, wl, y, reduction=reduction)
        dx, dw = torch.autograd.grad(loss, (xl, wl), torch.full_like(loss, up))
        assert not dx.any() and not dw.any()


@pytest.mark.parametrize("T", [5, 40, 64, 70, 300])
@pytest.mark.parametrize("which", ["weight", "both"])
def test_words_without_probability_take_no_gradient(gpu_device, T, which):
    """positive hidden rows and words of -inf: their logits are -inf and their p is 0, so their rows of dW are 0 (dX, a sum
    with 0 times -inf, is NaN by definition), whatever fills the tiles' rows past the live ones"""
    from lowbit.loss import linear_cross_entropy

    x, w, y, _ = _inputs(T, 96, 700, 51, gpu_device, 0.2 if T > 5 else 0.0)
    x = x.abs() + 2.0 ** -6
    y = torch.where(y == IGNORE, y, y % 400 + 300)
    wf = w[300:].clone()
    w[:300] = -float("inf")
    xl, wl = x.clone().requires_grad_(which == "both"), w.clone().requires_grad_(True)
    loss = linear_cross_entropy(xl, wl, y)
    loss.backward()
    assert not wl.grad[:300].any()
    _check(x, wf, torch.where(y == IGNORE, y, y - 300), loss.detach(), None, wl.grad[300:], "mean", torch.ones((), device=gpu_device))


@pytest.mark.parametrize("T", [5, 40, 300])
@pytest.mark.parametrize("V", [257, 40001])
@pytest.mark.parametrize("top", [200.0, 24.0, -200.0])
def test_confident_positions(gpu_device, T, V, top):
    """x_t picks one column of the weight, whose bf16 values are the logits without a rounding; the label's is `top`, the
    largest, and the others' exponentials add to 1e-7 ... 1 of its own.  A term exp(z - top) is off by 64 u of itself (its
    exponent, below 50, by a rounding and log2(e)'s), and the additions that hold the 1 of the largest, at most 24 before
    the tiles' pairs are joined, by u each; the logarithm by 4 u of itself.  So a loss is within 72 u of itself and 24 u,
    however large the logits, and never negative.  dz, read off dW (ceil(T / 64) equal rows to a column): the same in p,
    8 u more at p - 1, and the roundings of dz and of dW to bf16"""
    from lowbit.loss import linear_cross_entropy

    g = torch.Generator().manual_seed(V + T)
    H = 64
    eps = 10.0 ** -(7 * torch.rand(H, generator=g, dtype=torch.float64))
    w = (top - torch.log(V / eps) + 0.5 * torch.randn(V, H, generator=g, dtype=torch.float64)).clamp(max=top - 1).bfloat16()
    word = torch.randint(0, V, (H,), generator=g)
    w[word, torch.arange(H)] = top
    x = torch.zeros(T, H, dtype=torch.bfloat16)
    x[torch.arange(T), torch.arange(T) % H] = 1.0
    x, w, y = x.to(gpu_device), w.to(gpu_device), word[torch.arange(T) % H].to(gpu_device)
    d = (w.double() - top).t()[torch.arange(T, device=gpu_device) % H]  # z - the label's
    rest = torch.exp(d).scatter_(1, y[:, None], 0.0).sum(1)
    want = torch.log1p(rest)
    wl = w.clone().requires_grad_(True)
    each = linear_cross_entropy(x, w, y, reduction="none")
    loss = linear_cross_entropy(x, wl, y, reduction="sum")
    bound = 72 * U * want + 24 * U
    assert (each >= 0).all() and ((each.double() - want).abs() <= bound).all(), float(((each.double() - want).abs() / bound).max())
    assert abs(float(loss.detach().double() - want.sum())) <= float(bound.sum() + 4 * math.sqrt(T) * U * want.sum())
    (dw,) = torch.autograd.grad(loss, wl)
    p = torch.exp(d) / (1 + rest)[:, None]
    dz = p.scatter(1, y[:, None], -(rest / (1 + rest))[:, None])
    off = (p * (72 * U * (1 + rest) + 24 * U)[:, None]).scatter_add(1, y[:, None], torch.full_like(want, 8 * U)[:, None])
    want = dz.t() @ x.double()
    bound = (2 * B + B * B) * want.abs() + (1 + B) * 1.01 * (off.t() @ x.double()) + 1e-37
    assert ((dw.double() - want).abs() <= bound).all(), float(((dw.double() - want).abs() / bound).max())


@pytest.mark.parametrize("pitch", [(1 << 22) + 8, (1 << 22) + 3])
def test_a_weight_of_very_long_rows(gpu_device, pitch):
    """rows further apart than the products' copies reach: the weight goes through padded rows"""
    from lowbit.loss import linear_cross_entropy

    x, w, y, _ = _inputs(20, 64, 5, 61, gpu_device)
    far = torch.zeros(5 * pitch, dtype=torch.bfloat16, device=gpu_device).as_strided((5, 64), (pitch, 1))
    far.copy_(w)
    got, want = [], []
    for out, weight in ((got, far), (want, w)):
        xl, wl = x.clone().requires_grad_(True), weight.detach().requires_grad_(True)
        loss = linear_cross_entropy(xl, wl, y)
        out += [loss.detach(), *torch.autograd.grad(loss, (xl, wl))]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_too_large_is_refused_alike_from_python(gpu_device):
    """the package's own error, as other entry points raise it, before a launch"""
    from lowbit import _lib
    from lowbit.loss import linear_cross_entropy

    T = (1 << 22) + 1
    x = torch.zeros(1, 8, dtype=torch.bfloat16, device=gpu_device).expand(T, 8)
    w = torch.zeros(16, 8, dtype=torch.bfloat16, device=gpu_device)
    y = torch.zeros(1, dtype=torch.int64, device=gpu_device).expand(T)
    for wl in (w, w.clone().requires_grad_(True)):
        with pytest.raises(_lib.LowBitKernelError, match="too large"):
            linear_cross_entropy(x, wl, y)
    assert float(linear_cross_entropy(x[:3], w, y[:3])) > 0  # the next call is none the worse
