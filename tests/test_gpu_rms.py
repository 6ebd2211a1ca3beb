"""GPU tests of lowbit.norm.rms_norm and rms_norm_quant against the definition in 64 bits.

Bounds, with u = 2^-24 (fp32 arithmetic) and v the output type's rounding (2^-24, 2^-11 fp16, 2^-8 bf16; fp16 adds its
least step): a thread adds at most 64 squares in sequence and the tree over the threads fewer than 64 more, all of one
sign, so the mean of squares is off by at most 130 u of itself and r by 70 u with its root and division; xh = s r and y =
xh w by 80 u.  mean(t xh) is off by 256 u of the mean of magnitudes.  dw adds T rows in some order.  Every comparison
is elementwise against these bounds.
"""

from __future__ import annotations

import pytest
import torch

from _kept import kept, values

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 0.0, torch.float16: 2.0 ** -24, torch.bfloat16: 0.0}


def _inputs(T, H, dtype, wdtype, seed, dev):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, generator=g) * torch.exp(0.5 * torch.randn(H, generator=g))
    res = torch.randn(T, H, generator=g)
    w = 1 + 0.2 * torch.randn(H, generator=g)
    dy, ds = torch.randn(T, H, generator=g), torch.randn(T, H, generator=g)
    return [t.to(d).to(dev) for t, d in ((x, dtype), (res, dtype), (w, wdtype), (dy, dtype), (ds, dtype))]


def _check(got, want, bound, what):
    bound = bound + ROUND[got.dtype] * want.abs() + LEAST[got.dtype] + 1e-37
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (what, int(bad.sum()), float((off / bound).nan_to_num(1e9).max()))


def _r(s, eps):
    return 1 / torch.sqrt(s.double().square().mean(1, keepdim=True) + eps)


def _check_forward(y, s, w, eps):
    want = s.double() * _r(s, eps) * (1.0 if w is None else w.double())
    _check(y, want, 80 * U * want.abs(), "y")


def _check_backward(dx, dw, s, held, w, dy, ds, eps):
    """held: s as the backward reads it"""
    r, T = _r(s, eps), s.shape[0]
    xh, e = held.double() * r, dy.double()
    t = e if w is None else e * w.double()
    m = (t * xh).mean(1, keepdim=True)
    if dx is not None:
        a = r * (t - xh * m)
        off = 256 * U * ((t * xh).abs().mean(1, keepdim=True) + m.abs())
        bound = r * (4 * U * t.abs() + xh.abs() * off + 256 * U * (xh * m).abs()) + 128 * U * a.abs()
        want = a if ds is None else a + ds.double()
        _check(dx, want, bound + 4 * U * (want.abs() + a.abs()), "dx")
    if dw is not None:
        _check(dw, (e * xh).sum(0), (T + 136) * U * (e * xh).abs().sum(0), "dw")


SIZES = [(1, 1), (1, 7168), (3, 5), (7, 64), (2, 513), (130, 1541), (33, 4104), (5, 16384), (1100, 512), (257, 1000),
         (1, 9000), (520, 7168), (4099, 24), (700, 2047), (3, 129), (5, 127), (4, 8200)]
TYPES = [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float32, torch.float32),
         (torch.bfloat16, torch.float32)]


@pytest.mark.parametrize("T,H", SIZES)
@pytest.mark.parametrize("dtype,wdtype", TYPES)
def test_values_and_gradients(gpu_device, T, H, dtype, wdtype):
    from lowbit.norm import rms_norm

    x, res, w, dy, ds = _inputs(T, H, dtype, wdtype, 31 * T + H, gpu_device)
    total = (x.float() + res.float()).to(dtype)
    for residual in (False, True):
        for checkpoint in (None, "e4m3"):
            leaves = [t.clone().requires_grad_(True) for t in (x, res, w)]
            lx, lr, lw = leaves
            if residual:
                y, s = rms_norm(lx, lw, residual=lr, eps=1e-5, checkpoint=checkpoint)
                dx, dres, dw = torch.autograd.grad((y, s), leaves, (dy, ds))
                assert torch.equal(s.detach(), total) and torch.equal(dx, dres)
            else:
                y = rms_norm(lx, lw, eps=1e-5, checkpoint=checkpoint)
                dx, dw = torch.autograd.grad(y, (lx, lw), dy)
            with torch.no_grad():
                again = rms_norm(x, w, residual=res if residual else None, eps=1e-5, checkpoint=checkpoint)
            assert torch.equal(y.detach(), again[0] if residual else again)
            assert y.dtype == dtype and dx.dtype == dtype and dw.dtype == wdtype
            at = total if residual else x
            _check_forward(y.detach(), at, w, 1e-5)
            _check_backward(dx, dw, at, kept(at) if checkpoint else at, w, dy, ds if residual else None, 1e-5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("H", [3, 64, 129, 1000, 1541, 7168])
def test_kept_codes(gpu_device, dtype, H):
    """what the operator keeps is the definition's 8 bits of s, bit for bit, zero past H; nothing of 16 or more bits stays"""
    from lowbit.norm import rms_norm

    x, res, w, dy, ds = _inputs(9, H, dtype, dtype, H, gpu_device)
    x, res = x * torch.logspace(-6, 4, H, device=gpu_device).to(dtype), res * 0
    x[2], x[4, 0] = 0, 448.0
    x[5, :H // 2] = float(torch.finfo(dtype).tiny) if dtype is not torch.float16 else 2.0 ** -24
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
        y, s = rms_norm(x.requires_grad_(True), w, residual=res, checkpoint="e4m3")
    big = [t for t in saved if t.numel() >= s.numel() and t.dtype is not torch.uint8]
    assert not big
    codes = max((t for t in saved if t.dtype is torch.uint8), key=lambda t: t.numel())
    (exps,) = [t for t in saved if t.dtype is torch.uint8 and t is not codes]
    assert codes.shape[1] % 128 == 0 and not codes[:, H:].any()
    q = values(codes, exps)
    assert torch.equal(q[:, :H].nan_to_num(1234.0), kept(s.detach()).nan_to_num(1234.0))  # fp16 reaches infinity


def test_kept_values_that_are_not_finite(gpu_device):
    """kept as NaN, beside a tile whose other values are kept as if they were not there; other rows' gradients are whole"""
    from lowbit.norm import rms_norm

    x, _, w, dy, _ = _inputs(6, 300, torch.bfloat16, torch.bfloat16, 4, gpu_device)
    x[1, 3], x[2, 299], x[4, 130] = float("nan"), float("inf"), float("-inf")
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
        y = rms_norm(x.requires_grad_(True), w, checkpoint="e4m3")
    codes, exps = sorted((t for t in saved if t.dtype is torch.uint8), key=lambda t: -t.numel())
    q = values(codes, exps)
    assert torch.equal(q[:, :300].nan_to_num(1234.0), kept(x.detach()).nan_to_num(1234.0))
    (dx,) = torch.autograd.grad(y, x, dy)
    assert dx[[0, 3, 5]].isfinite().all() and dx[[1, 2, 4]].isnan().any(1).all()


@pytest.mark.parametrize("which", ["pitch", "offset", "transposed", "repeated", "3d", "dy_pitch"])
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_strides(gpu_device, which, checkpoint):
    from lowbit.norm import rms_norm

    T, H = 70, 1001
    ts = _inputs(T, H + 7, torch.bfloat16, torch.bfloat16, 5, gpu_device)
    w = ts[2][:H]
    make = {"pitch": lambda t: t[:, :H], "offset": lambda t: t[:, 3:3 + H], "transposed": lambda t: t[:, :H].t().contiguous().t(),
            "repeated": lambda t: t[:1, :H].expand(T, H), "3d": lambda t: t[:, :H].reshape(7, 10, H),
            "dy_pitch": lambda t: t[:, :H].contiguous()}[which]
    x, res, dy, ds = (make(ts[i]) for i in (0, 1, 3, 4))
    if which == "dy_pitch":
        dy, ds = ts[3][:, 1:1 + H], ts[4][:1, :H].expand(T, H)
    lx, lr, lw = x.detach().requires_grad_(True), res.detach().requires_grad_(True), w.clone().requires_grad_(True)
    y, s = rms_norm(lx, lw, residual=lr, checkpoint=checkpoint)
    dx, dres, dw = torch.autograd.grad((y, s), (lx, lr, lw), (dy, ds))
    assert y.shape == s.shape == dx.shape == dres.shape == x.shape
    s2 = s.detach().reshape(-1, H)
    assert torch.equal(s2, (x.float() + res.float()).bfloat16().reshape(-1, H))
    _check_forward(y.detach().reshape(-1, H), s2, w, 1e-6)
    _check_backward(dx.reshape(-1, H), dw, s2, kept(s2) if checkpoint else s2, w, dy.reshape(-1, H), ds.reshape(-1, H), 1e-6)


@pytest.mark.parametrize("need", [(True, False, False), (False, True, False), (False, False, True), (True, False, True)])
@pytest.mark.parametrize("used", ["y", "s", "both"])
def test_each_gradient_alone(gpu_device, need, used):
    """of the leaves that want one, from either result alone"""
    from lowbit.norm import rms_norm

    x, res, w, dy, ds = _inputs(65, 770, torch.bfloat16, torch.bfloat16, 11, gpu_device)
    leaves = [t.clone().requires_grad_(n) for t, n in zip((x, res, w), need)]
    y, s = rms_norm(leaves[0], leaves[2], residual=leaves[1])
    f = {"y": (y * dy).sum(), "s": (s * ds).sum(), "both": (y * dy).sum() + (s * ds).sum()}[used]
    f.backward()
    assert [t.grad is not None for t in leaves] == [need[0], need[1], need[2] and used != "s"]
    at, want_ds = s.detach(), ds if used == "both" else None
    for t in leaves[:2]:
        if t.grad is not None:
            if used == "s":
                assert torch.equal(t.grad, ds)
            else:
                _check_backward(t.grad, None, at, at, w, dy, want_ds, 1e-6)
    if leaves[2].grad is not None:
        _check_backward(None, leaves[2].grad, at, at, w, dy, None, 1e-6)


def test_without_weight(gpu_device):
    from lowbit.norm import rms_norm

    x, res, _, dy, _ = _inputs(40, 300, torch.float16, torch.float16, 9, gpu_device)
    lx = x.clone().requires_grad_(True)
    y = rms_norm(lx, eps=1e-3)
    y.backward(dy)
    _check_forward(y.detach(), x, None, 1e-3)
    _check_backward(lx.grad, None, x, x, None, dy, None, 1e-3)


def test_zero_rows_and_rows_that_are_not_finite(gpu_device):
    from lowbit.norm import rms_norm

    x, res, w, dy, ds = _inputs(9, 600, torch.bfloat16, torch.bfloat16, 13, gpu_device)
    x[1] = 0
    clean = rms_norm(x, w)
    assert not clean[1].any()
    x[2, 5], x[4, 599], x[7, 0] = float("nan"), float("inf"), float("-inf")
    xl = x.clone().requires_grad_(True)
    y = rms_norm(xl, w)
    y.backward(dy)
    bad = torch.zeros(9, dtype=torch.bool, device=gpu_device)
    bad[[2, 4, 7]] = True
    assert torch.equal(y.detach()[~bad], clean[~bad]) and xl.grad[~bad].isfinite().all()
    assert y.detach()[2].isnan().all() and y.detach()[4, 599].isnan() and y.detach()[7, 0].isnan()


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_no_rows(gpu_device, checkpoint):
    from lowbit.norm import rms_norm, rms_norm_quant

    x, res = (torch.empty(0, 96, device=gpu_device, requires_grad=True) for _ in range(2))
    w = torch.ones(96, device=gpu_device, requires_grad=True)
    y, s = rms_norm(x, w, residual=res, checkpoint=checkpoint)
    assert y.shape == s.shape == (0, 96)
    (y.sum() + s.sum()).backward()
    assert x.grad.shape == res.grad.shape == (0, 96) and not w.grad.any()
    with torch.no_grad():
        q, s = rms_norm_quant(x, w, residual=res)
    assert q.rows == 0 and q.codes.shape == (0, 128) and s.shape == (0, 96)


def test_gradients_against_differences(gpu_device):
    """d/dh of f = <y(x + h p, r + h p', w + h q), dy> + <s, ds> by central differences of the kernel's own fp32 outputs;
    the h^2 term removed, what remains is far below the difference of the two quotients; rounding: below 2 u sum|y dy| / h"""
    from lowbit.norm import rms_norm

    T, H, h = 24, 200, 2.0 ** -6
    x, res, w, dy, ds = _inputs(T, H, torch.float32, torch.float32, 17, gpu_device)
    g = torch.Generator().manual_seed(18)
    p, p2, q = (torch.randn(*s, generator=g).to(gpu_device) for s in ((T, H), (T, H), (H,)))

    def f(k):
        y, s = rms_norm(x + k * p, w + k * q, residual=res + k * p2)
        return (y.double() * dy.double()).sum() + (s.double() * ds.double()).sum()

    leaves = [t.clone().requires_grad_(True) for t in (x, res, w)]
    y, s = rms_norm(leaves[0], leaves[2], residual=leaves[1])
    grads = torch.autograd.grad((y, s), leaves, (dy, ds))
    want = sum((a.double() * b.double()).sum() for a, b in zip(grads, (p, p2, q)))
    d1, d2 = (f(h) - f(-h)) / (2 * h), (f(2 * h) - f(-2 * h)) / (4 * h)
    scale = float((y.detach().double() * dy.double()).abs().sum() + (s.detach().double() * ds.double()).abs().sum())
    assert abs(float((4 * d1 - d2) / 3 - want)) <= abs(float(d1 - d2)) + 8 * U * scale / h


def _exact_codes(s, w, fmt):
    """the code values of s w over its tiles' scales in 64 bits, and how near each lies to the middle of two (0: a tie)"""
    from _kept import round_e4m3

    p, qmax = s.double() * w.double(), 448.0 if fmt == "e4m3" else 127.0
    v = torch.cat([t * qmax / t.abs().amax(1, keepdim=True).clamp(min=1e-300) for t in p.split(128, 1)], 1)
    if fmt == "e4m3":
        q = round_e4m3(v)
        a, b = round_e4m3(v * (1 - 4 * U)), round_e4m3(v * (1 + 4 * U))
    else:
        q, a, b = v.round(), (v * (1 - 4 * U)).round(), (v * (1 + 4 * U)).round()
    return q, a, b


def _code_values(q, H):
    if q.grid == 1:
        return q.codes[:, :H].view(torch.float8_e4m3fn).double()
    return q.codes[:, :H].view(torch.int8).double()


@pytest.mark.parametrize("fmt", ["e4m3", "int_grid"])
@pytest.mark.parametrize("T,H", [(1, 7168), (3, 5), (37, 129), (130, 1541), (2, 16384), (300, 1000), (64, 128), (9, 2)])
@pytest.mark.parametrize("dtype,wdtype", TYPES)
def test_codes_are_the_nearest(gpu_device, fmt, T, H, dtype, wdtype):
    """of bf16 values and weights, whose products and their multiples by 448 or 127 have 24 bits, every code is the exact
    quotient's, ties included (no other quotient of such numbers is nearer to a tie than 2^-23 of itself); of others it is where
    the quotient is not within 4 u of the middle of two codes"""
    from lowbit.norm import rms_norm_quant

    x, res, w, _, _ = _inputs(T, H, dtype, wdtype, T + H, gpu_device)
    total = (x.float() + res.float()).to(dtype)
    for residual, at in ((None, x), (res, total)):
        q = rms_norm_quant(x, w, residual=residual, fmt=fmt, want_nan_rows=True)
        q = q if residual is None else q[0]
        got, (want, low, high) = _code_values(q, H), _exact_codes(at, w, fmt)
        if dtype == wdtype == torch.bfloat16:
            assert torch.equal(got, want)
        else:
            assert ((got == want) | (got == low) | (got == high)).all()
        top = torch.stack([p.abs().amax(1) for p in (at.double() * w.double()).split(128, 1)]) * _r(at, 1e-6)[:, 0]
        want = top / (448.0 if fmt == "e4m3" else 127.0)
        assert ((q.scales[:, :T].double() - want).abs() <= 80 * U * want).all()
        assert not q.codes[:, H:].any() and not q.nan_rows.any()
        assert (q.rows, q.K, q.s_row, q.s_col, q.shift) == (T, H, 1, q.scales.shape[1], 0)


@pytest.mark.parametrize("fmt", ["e4m3", "int_grid"])
def test_codes_of_special_rows_are_the_quantizers(gpu_device, fmt):
    """zeros, NaN, infinities, magnitudes at fp32's ends: codes, scales and NaN rows are quant_tile_1x128's of y"""
    from lowbit import ops
    from lowbit.norm import rms_norm, rms_norm_quant

    x, res, w, _, _ = _inputs(12, 300, torch.float32, torch.float32, 5, gpu_device)
    x[1], res[1] = 0, 0
    x[2, 150], x[3, 0], res[4, 299] = float("nan"), float("inf"), float("-inf")
    x[5], res[5] = x[5] * 1e-30, 0
    x[6, :128], res[6] = 0, 0
    x[7] *= 1e30
    x[8, 3] = 1e18
    w = w.clone()
    w[200] = 0
    for eps in (0.0, 1e-6):
        y, s = rms_norm(x, w, residual=res, eps=eps)
        q, s2 = rms_norm_quant(x, w, residual=res, eps=eps, fmt=fmt, want_nan_rows=True)
        assert torch.equal(s.view(torch.int32), s2.view(torch.int32))
        want = ops.quant_tile_1x128(y, fmt=fmt, want_nan_rows=True)
        assert torch.equal(q.nan_rows, want.nan_rows)
        odd = torch.tensor([1, 2, 3, 4, 7], device=gpu_device)  # row 7: its squares pass fp32, so that y is 0
        assert torch.equal(q.codes[odd], want.codes[odd]) and torch.equal(q.scales[:, odd], want.scales[:, odd])
        rest = torch.tensor([5, 6, 8, 9, 10, 11], device=gpu_device)
        a, b = q.scales[:, rest].double(), want.scales[:, rest].double()
        assert ((a - b).abs() <= 4 * U * b).all()
        if eps:
            got, ref = _code_values(q, 300)[rest], _exact_codes(s[rest], w, fmt)
            assert ((got == ref[0]) | (got == ref[1]) | (got == ref[2])).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,H", [(1, 7168), (5, 333), (200, 1024)])
def test_codes_of_16_bit_inputs(gpu_device, dtype, T, H):
    """y in 64 bits over the tile's scale, to half a step of e4m3 (2^-4 of the value, 2^-10 of the scale below its normal
    numbers); the scale is off by 80 u, which a value near the middle of two steps adds once more"""
    from lowbit import ops
    from lowbit.norm import rms_norm_quant

    x, res, w, _, _ = _inputs(T, H, dtype, dtype, T, gpu_device)
    q, s = rms_norm_quant(x, w, residual=res)
    assert torch.equal(s, (x.float() + res.float()).to(dtype))
    y = s.double() * _r(s, 1e-6) * w.double()
    tiles = (H + 127) // 128
    top = torch.stack([p.abs().amax(1) for p in y.split(128, 1)])
    scale = q.scales[:, :T].double()
    assert ((scale - top / 448).abs() <= 100 * U * top / 448).all()
    each = scale.t().repeat_interleave(128, 1)[:, :H]
    got = ops.dequant(q, out_dtype=torch.float32).double()
    assert ((got - y).abs() <= (2.0 ** -4 + 200 * U) * y.abs() + each * 2.0 ** -10 * (1 + 200 * U)).all()
    assert tiles * 128 == q.codes.shape[1] and not q.codes[:, H:].any()


def test_the_codes_go_into_a_product(gpu_device):
    """norm, codes, blockwise product: the product of what the codes stand for"""
    from lowbit import ops
    from lowbit.norm import rms_norm_quant

    x, res, w, _, _ = _inputs(70, 1024, torch.bfloat16, torch.bfloat16, 3, gpu_device)
    g = torch.Generator().manual_seed(1)
    wq, _ = ops.quant_block_128x128((0.02 * torch.randn(256, 1024, generator=g)).bfloat16().to(gpu_device), fmt="e4m3")
    q, _ = rms_norm_quant(x.reshape(7, 10, 1024), w, residual=res.reshape(7, 10, 1024))
    got = ops.gemm_blockscaled(q, wq, out_dtype=torch.float32)
    a, b = ops.dequant(q, out_dtype=torch.float32).double(), ops.dequant(wq, out_dtype=torch.float32).double()
    bound = 1024 * 2 * U * (a.abs() @ b.abs().t())
    assert ((got.double() - a @ b.t()).abs() <= bound).all()


def test_second_gradient_and_tangents_are_refused(gpu_device):
    import torch.autograd.forward_ad as fw
    from lowbit.norm import rms_norm

    x = torch.randn(4, 8, device=gpu_device, requires_grad=True)
    (dx,) = torch.autograd.grad(rms_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
    with fw.dual_level(), pytest.raises(NotImplementedError):
        rms_norm(fw.make_dual(x.detach(), torch.ones_like(x)))


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_other_stream_and_graph(gpu_device, checkpoint):
    """forward and backward on another stream, and replayed from a graph"""
    from lowbit.norm import rms_norm

    x, res, w, dy, ds = _inputs(50, 1030, torch.bfloat16, torch.bfloat16, 21, gpu_device)
    leaves = [t.clone().requires_grad_(True) for t in (x, res, w)]

    def step():
        y, s = rms_norm(leaves[0], leaves[2], residual=leaves[1], checkpoint=checkpoint)
        return (y.detach(), s.detach(), *torch.autograd.grad((y, s), leaves, (dy, ds)))

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
            leaves[0].copy_(torch.randn(50, 1030, generator=torch.Generator().manual_seed(k)).to(x))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_results_may_be_changed_only_where_nothing_reads_them(gpu_device):
    """s is read by the backward: a change in place is noticed; y may change, and with 8 bits kept s may too"""
    from lowbit.norm import rms_norm

    x, res, w, dy, _ = _inputs(5, 64, torch.float32, torch.float32, 2, gpu_device)
    leaves = [t.clone().requires_grad_(True) for t in (x, res, w)]
    y, s = rms_norm(leaves[0], leaves[2], residual=leaves[1])
    with torch.no_grad():
        s.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, leaves, dy)
    y, s = rms_norm(leaves[0], leaves[2], residual=leaves[1], checkpoint="e4m3")
    first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    with torch.no_grad():
        s.mul_(2)
    again = torch.autograd.grad(y, leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, leaves, dy)


def test_x_is_its_own_residual(gpu_device):
    """s = 2 x, and x has the gradients of both places"""
    from lowbit.norm import rms_norm

    g = torch.Generator().manual_seed(2)
    x, dy, ds = (torch.randn(9, 200, generator=g).to(gpu_device) for _ in range(3))
    a, b, c = (x.clone().requires_grad_(True) for _ in range(3))
    one, two = rms_norm(a, residual=a), rms_norm(b, residual=c)
    assert torch.equal(one[1], 2 * x) and torch.equal(one[0], two[0])
    (da,) = torch.autograd.grad(one, a, (dy, ds))
    db, dc = torch.autograd.grad(two, (b, c), (dy, ds))
    assert torch.equal(db, dc) and torch.equal(da, 2 * db)
    torch.autograd.backward(rms_norm(b, residual=c), (dy, ds))
    assert torch.equal(b.grad, db) and torch.equal(c.grad, db) and b.grad.data_ptr() != c.grad.data_ptr()


def test_module(gpu_device):
    from lowbit.norm import RMSNorm

    m = RMSNorm(48, dtype=torch.bfloat16, device=gpu_device)
    x = torch.randn(5, 48, device=gpu_device).bfloat16()
    _check_forward(m(x).detach(), x, m.weight.detach(), 1e-6)
    y, s = m(x, x)
    assert torch.equal(s.detach(), x + x) and set(m.state_dict()) == {"weight"}


def test_refusals(gpu_device):
    from lowbit.norm import RMSNorm, rms_norm, rms_norm_quant

    x = torch.randn(4, 32, device=gpu_device)
    for f in (rms_norm, rms_norm_quant):
        with pytest.raises(RuntimeError, match="ROCm device"):
            f(torch.randn(4, 32))
        with pytest.raises(ValueError, match="16384"):
            f(torch.randn(1, 16385, device=gpu_device))
        with pytest.raises(ValueError, match="weight"):
            f(x, torch.ones(31, device=gpu_device))
        with pytest.raises(TypeError, match="dtype"):
            f(x.double())
        with pytest.raises(TypeError, match="residual"):
            f(x, residual=x.half())
        with pytest.raises(ValueError, match="residual"):
            f(x, residual=x[:1])
        with pytest.raises(ValueError, match="residual"):
            f(x, residual=x.cpu())
        with pytest.raises(ValueError, match="eps"):
            f(x, eps=-1.0)
    with pytest.raises(ValueError, match="checkpoint"):
        rms_norm(x, checkpoint="int8")
    with pytest.raises(ValueError, match="checkpoint"):
        RMSNorm(8, checkpoint="fp8")
    with pytest.raises(ValueError, match="format"):
        rms_norm_quant(x, fmt="e5m2")
    with pytest.raises(RuntimeError, match="no gradient"):
        rms_norm_quant(x, torch.ones(32, device=gpu_device, requires_grad=True))
