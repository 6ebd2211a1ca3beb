"""GPU tests of lowbit.experts.grouped_matmul against the definition in 64 bits, expert by expert.

Bounds, with u = 2^-24: products of bf16 values are exact in fp32, a sum of n of them in any order is off by at most 2 n u
of the sum of magnitudes (the matrix unit may drop bits below fp32's last one once an addition); the result is rounded to
bf16 (2^-8).  Every comparison is elementwise.
"""

from __future__ import annotations

import pytest
import torch

from _kept import kept, values

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
V = 2.0 ** -8


def _inputs(counts, K, N, seed, dev, spare=0):
    g = torch.Generator().manual_seed(seed)
    R = sum(counts) + spare
    x = torch.randn(R, K, generator=g) * torch.exp(0.5 * torch.randn(K, generator=g))
    w = 0.05 * torch.randn(len(counts), N, K, generator=g)
    dy = torch.randn(R, N, generator=g)
    offsets = torch.tensor([0] + counts).cumsum(0).int()
    return [t.bfloat16().to(dev) for t in (x, w, dy)] + [offsets.to(dev)]


def _check(got, want, n, mags, what):
    bound = 2 * n * U * mags + V * want.abs() + 1e-37
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[:4].tolist(),
                           float(((got.double() - want).abs() / bound).nan_to_num(1e9).max()))


def _check_all(y, dx, dw, x, w, dy, offsets, checkpoint=None):
    ends = offsets.tolist()
    K, N = x.shape[1], w.shape[1]
    assert y.shape == (x.shape[0], N)
    assert not y[ends[-1]:].any() and (dx is None or not dx[ends[-1]:].any())
    for e in range(w.shape[0]):
        part = slice(ends[e], ends[e + 1])
        xe, we, n = x[part].double(), w[e].double(), ends[e + 1] - ends[e]
        if n == 0:
            assert dw is None or not dw[e].any()
            continue
        _check(y[part], xe @ we.t(), K, xe.abs() @ we.t().abs(), ("y", e))
        if dx is not None:
            de = dy[part].double()
            _check(dx[part], de @ we, N, de.abs() @ we.abs(), ("dx", e))
        if dw is not None:
            de = dy[part].double()
            xk = kept(xe) if checkpoint else xe
            _check(dw[e], de.t() @ xk, n, de.t().abs() @ xk.abs(), ("dw", e))


CASES = [  # rows of each expert, K, N, spare rows
    ([1], 8, 8, 0), ([1], 7168, 16, 0), ([3, 0, 5], 64, 24, 2), ([0, 0, 1, 0], 200, 130, 0), ([5, 0, 11, 1], 1000, 345, 7),
    ([0, 0], 72, 40, 9), ([16, 17, 33, 65, 1], 264, 264, 0), ([300, 7, 0, 129], 520, 384, 30), ([1003, 1], 129, 257, 0),
    ([128, 256, 384], 256, 512, 0), ([700, 513, 255, 257], 1024, 768, 1), ([2, 1] * 50, 96, 72, 3), ([90] * 70, 64, 136, 0),
    ([2500, 2600], 320, 2304, 0), ([1] * 8, 7168, 512, 0), ([40, 3, 64, 100], 2049, 100, 0), ([1, 1], 1, 1, 1),
    # the contraction in ranges: of y, of dx, of both; rows behind, no rows, a last quad cut
    ([160], 4096, 128, 0), ([0, 90, 0, 133], 1111, 77, 9), ([200], 72, 4096, 40), ([257, 40], 1025, 1027, 0), ([70, 0], 7168, 1, 3),
]


@pytest.mark.parametrize("counts,K,N,spare", CASES)
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_values_and_gradients(gpu_device, counts, K, N, spare, checkpoint):
    from lowbit.experts import grouped_matmul

    x, w, dy, offsets = _inputs(counts, K, N, 3 * K + N, gpu_device, spare)
    if spare:
        x[-spare:], dy[-spare:] = float("nan"), float("nan")  # not read
    lx, lw = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = grouped_matmul(lx, lw, offsets, checkpoint=checkpoint)
    dx, dw = torch.autograd.grad(y, (lx, lw), dy)
    with torch.no_grad():
        assert torch.equal(grouped_matmul(x, w, offsets, checkpoint=checkpoint), y)
    _check_all(y.detach(), dx, dw, x, w, dy, offsets, checkpoint)
    again = torch.autograd.grad(grouped_matmul(lx, lw, offsets, checkpoint=checkpoint), (lx, lw), dy)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


@pytest.mark.parametrize("counts,K,N", [([1] * 4095 + [3], 16, 8), ([2], 1 << 22, 3), ([3, 0], 8, 1 << 22), ([1 << 20, 5], 8, 8),
                                        ([0] * 64 + [70] + [0] * 70 + [9], 320, 128)])
def test_the_largest_of_each_size(gpu_device, counts, K, N):
    from lowbit.experts import grouped_matmul

    g = torch.Generator(gpu_device).manual_seed(K + N)
    R, E = sum(counts), len(counts)
    x, w, dy = (torch.randn(*size, generator=g, device=gpu_device).bfloat16() for size in ((R, K), (E, N, K), (R, N)))
    offsets = torch.tensor([0] + counts).cumsum(0).int().to(gpu_device)
    lx, lw = x.requires_grad_(True), w.requires_grad_(True)
    y = grouped_matmul(lx, lw, offsets)
    dx, dw = torch.autograd.grad(y, (lx, lw), dy)
    ends = offsets.tolist()
    for e in [0, E // 2, E - 1]:
        part = slice(ends[e], ends[e + 1])
        n = ends[e + 1] - ends[e]
        if n == 0:
            assert not dw[e].any()
            continue
        xe, we, de = x.detach()[part].double(), w.detach()[e].double(), dy[part].double()
        _check(y.detach()[part], xe @ we.t(), K, xe.abs() @ we.t().abs(), ("y", e))
        _check(dx[part], de @ we, N, de.abs() @ we.abs(), ("dx", e))
        _check(dw[e], de.t() @ xe, n, de.t().abs() @ xe.abs(), ("dw", e))


def test_calls_side_by_side(gpu_device):
    """two streams at once, each with ranges of a contraction: every call has sums of its own"""
    from lowbit.experts import grouped_matmul

    sets = [_inputs([60, 0, 77], 2048, 264, seed, gpu_device) for seed in (1, 2)]
    with torch.no_grad():
        want = [grouped_matmul(x, w, o) for x, w, _, o in sets]
        streams = [torch.cuda.Stream() for _ in sets]
        torch.cuda.synchronize()
        got = [[], []]
        for _ in range(20):
            for i, (x, w, _, o) in enumerate(sets):
                with torch.cuda.stream(streams[i]):
                    got[i].append(grouped_matmul(x, w, o))
        torch.cuda.synchronize()
    assert all(torch.equal(t, want[i]) for i in range(2) for t in got[i])


@pytest.mark.parametrize("which", ["pitch", "offset", "transposed", "weights_t", "weights_shared", "weights_slice", "dy_pitch",
                                   "dy_repeated", "x_repeated"])
def test_strides(gpu_device, which):
    from lowbit.experts import grouped_matmul

    counts, K, N = [30, 0, 100, 7], 136, 72
    x, w, dy, offsets = _inputs(counts, K + 16, N + 16, 5, gpu_device)
    x, w, dy = {
        "pitch": lambda: (x[:, :K], w[:, :N, :K], dy[:, :N]),
        "offset": lambda: (x[:, 3:3 + K], w[:, 1:1 + N, 5:5 + K], dy[:, 1:1 + N]),
        "transposed": lambda: (x[:, :K].t().contiguous().t(), w[:, :N, :K].contiguous(), dy[:, :N].t().contiguous().t()),
        "weights_t": lambda: (x[:, :K].contiguous(), w[:, :N, :K].transpose(1, 2).contiguous().transpose(1, 2), dy[:, :N]),
        "weights_shared": lambda: (x[:, :K], w[:1, :N, :K].expand(4, N, K), dy[:, :N]),
        "weights_slice": lambda: (x[:, :K], torch.cat([w, w])[::2, :N, :K], dy[:, :N]),
        "dy_pitch": lambda: (x[:, :K].contiguous(), w[:, :N, :K].contiguous(), dy[:, 8:8 + N]),
        "dy_repeated": lambda: (x[:, :K].contiguous(), w[:, :N, :K].contiguous(), dy[:1, :N].expand(137, N)),
        "x_repeated": lambda: (x[:1, :K].expand(137, K), w[:, :N, :K].contiguous(), dy[:, :N]),
    }[which]()
    lx, lw = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    y = grouped_matmul(lx, lw, offsets)
    dx, dw = torch.autograd.grad(y, (lx, lw), dy)
    _check_all(y.detach(), dx, dw, x, w, dy, offsets)


def test_one_row_and_offsets_of_any_stride(gpu_device):
    from lowbit.experts import grouped_matmul

    x, w, dy, _ = _inputs([1], 64, 32, 1, gpu_device)
    one = x.reshape(64, 1).t()
    assert one.stride() == (1, 1)
    off = torch.tensor([0, 9, 1, 9], dtype=torch.int32, device=gpu_device)[::2]
    lx, lw = one.detach().requires_grad_(True), w.clone().requires_grad_(True)
    y = grouped_matmul(lx, lw, off)
    dx, dw = torch.autograd.grad(y, (lx, lw), dy.reshape(32, 1).t())
    _check_all(y.detach(), dx, dw, x, w, dy, off.contiguous())


@pytest.mark.parametrize("need", [(True, False), (False, True)])
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_each_gradient_alone_keeps_the_other_operand_only(gpu_device, need, checkpoint):
    from lowbit.experts import grouped_matmul

    x, w, dy, offsets = _inputs([65, 3], 256, 128, 7, gpu_device)
    lx, lw = x.clone().requires_grad_(need[0]), w.clone().requires_grad_(need[1])
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
        y = grouped_matmul(lx, lw, offsets, checkpoint=checkpoint)
    kinds = sorted(str(t.dtype) for t in saved)
    assert kinds == (["torch.bfloat16", "torch.int32"] if need[0] or not checkpoint else ["torch.int32"] + ["torch.uint8"] * 2)
    y.backward(dy)
    assert (lx.grad is not None, lw.grad is not None) == need
    _check_all(y.detach(), lx.grad, lw.grad, x, w, dy, offsets, checkpoint)


@pytest.mark.parametrize("K", [8, 100, 129, 1000, 7168])
def test_kept_codes(gpu_device, K):
    from lowbit.experts import grouped_matmul

    x, w, _, offsets = _inputs([5, 4], K, 16, K, gpu_device)
    x = x * torch.logspace(-6, 6, K, device=gpu_device).bfloat16()
    x[2], x[3, 0], x[4, K - 1], x[5, K // 2] = 0, 448.0, float("nan"), float("inf")
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
        grouped_matmul(x, w.requires_grad_(True), offsets, checkpoint="e4m3")
    codes, exps = sorted((t for t in saved if t.dtype is torch.uint8), key=lambda t: -t.numel())
    assert torch.equal(values(codes, exps)[:, :K].nan_to_num(1234.0), kept(x).nan_to_num(1234.0))
    assert not codes[:, K:].any()


def test_values_that_are_not_finite_stay_with_their_rows_and_experts(gpu_device):
    from lowbit.experts import grouped_matmul

    for counts in ([4, 5, 6], [300, 200, 250]):
        x, w, dy, offsets = _inputs(counts, 136, 144, 3, gpu_device)
        clean = grouped_matmul(x, w, offsets)
        row, n = counts[0] + 1, sum(counts)
        x[row, 3], w[2, 5, 7] = float("inf"), float("nan")
        for checkpoint in (None, "e4m3"):
            lx, lw = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
            y = grouped_matmul(lx, lw, offsets, checkpoint=checkpoint)
            dx, dw = torch.autograd.grad(y, (lx, lw), dy)
            last = counts[0] + counts[1]
            ok = torch.ones(n, 144, dtype=torch.bool, device=gpu_device)
            ok[row], ok[last:, 5] = False, False
            assert torch.equal(y.detach()[ok], clean[ok]) and not y.detach()[row].isfinite().any()
            assert y.detach()[last:, 5].isnan().all()
            assert dx[:last].isfinite().all() and dx[last:, 7].isnan().all() and dx[last:, 8].isfinite().all()
            assert dw[0].isfinite().all() and dw[2].isfinite().all()
            assert not dw[1, :, 3].isfinite().any() and dw[1, :, 4].isfinite().all()


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_no_rows(gpu_device, checkpoint):
    from lowbit.experts import grouped_matmul

    x = torch.empty(0, 64, device=gpu_device, dtype=torch.bfloat16, requires_grad=True)
    w = torch.randn(3, 40, 64, device=gpu_device).bfloat16().requires_grad_(True)
    off = torch.zeros(4, dtype=torch.int32, device=gpu_device)
    y = grouped_matmul(x, w, off, checkpoint=checkpoint)
    assert y.shape == (0, 40)
    y.sum().backward()
    assert x.grad.shape == (0, 64) and w.grad.shape == w.shape and not w.grad.any()


def test_offsets_past_the_rows_count_as_their_number(gpu_device):
    from lowbit.experts import grouped_matmul

    for counts in ([7, 4], [300, 290]):
        x, w, dy, offsets = _inputs(counts, 64, 136, 2, gpu_device)
        far = offsets.clone()
        far[-1] = 2 ** 31 - 1
        lx, lw = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        y = grouped_matmul(lx, lw, far)
        dx, dw = torch.autograd.grad(y, (lx, lw), dy)
        _check_all(y.detach(), dx, dw, x, w, dy, offsets)


def test_gradients_against_differences(gpu_device):
    """y is linear in x and in w: <dx, p> = <y(p, w), dy> and <dw, q> = <y(x, q), dy>, each side's roundings counted"""
    from lowbit.experts import grouped_matmul

    counts, K, N = [40, 1, 23], 200, 88
    x, w, dy, offsets = _inputs(counts, K, N, 8, gpu_device)
    p, q, _, _ = _inputs(counts, K, N, 9, gpu_device)
    lx, lw = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(grouped_matmul(lx, lw, offsets), (lx, lw), dy)
    for grad, by, y in ((dx, p, grouped_matmul(p, w, offsets)), (dw, q, grouped_matmul(x, q, offsets))):
        a, b = grad.double() * by.double(), y.double() * dy.double()
        # each side's values are off by V of themselves and 2 n u of their magnitudes, far less here
        assert abs(float(a.sum() - b.sum())) <= 1.1 * V * float(a.abs().sum() + b.abs().sum())


@pytest.mark.parametrize("counts,K,N", [([3, 0, 9], 264, 136), ([600, 200, 0, 300], 264, 136), ([100, 0, 150], 1032, 520)])
def test_other_stream_and_graph(gpu_device, counts, K, N):
    """both directions on another stream and replayed from a graph, over new rows, new offsets among them"""
    from lowbit.experts import grouped_matmul

    x, w, dy, offsets = _inputs(counts, K, N, 4, gpu_device)
    lx, lw = x.clone().requires_grad_(True), w.clone().requires_grad_(True)

    def step():
        y = grouped_matmul(lx, lw, offsets, checkpoint="e4m3")
        return y.detach(), *torch.autograd.grad(y, (lx, lw), dy)

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
    n = len(counts)
    for k in range(4):
        other = _inputs([c for c in counts[k % n:] + counts[:k % n]], K, N, 40 + k, gpu_device)
        with torch.no_grad():
            lx.copy_(other[0])
            offsets.copy_(other[3])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))
    _check_all(*out, lx.detach(), w, dy, offsets, "e4m3")


def test_graph_rules(gpu_device):
    from lowbit.experts import grouped_matmul

    x, w, dy, offsets = _inputs([9, 4], 64, 40, 4, gpu_device)
    leaves = [x.clone().requires_grad_(True), w.clone().requires_grad_(True)]
    for i in range(3):
        moved = [t * 1 for t in leaves] + [offsets.clone()]
        y = grouped_matmul(*moved)
        with torch.no_grad():
            moved[i].mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, leaves, dy)
    y = grouped_matmul(*leaves, offsets)
    first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(y, leaves, dy)))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, leaves, dy)
    (dx,) = torch.autograd.grad(grouped_matmul(*leaves, offsets).square().sum(), leaves[0], create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def test_refusals(gpu_device):
    from lowbit.experts import grouped_matmul

    x, w, _, off = _inputs([3, 4], 64, 40, 4, gpu_device)
    for a, b, c in ((x.cpu(), w, off), (x, w.cpu(), off), (x, w, off.cpu())):
        with pytest.raises(RuntimeError, match="ROCm device"):
            grouped_matmul(a, b, c)
    with pytest.raises(TypeError, match="bfloat16"):
        grouped_matmul(x.float(), w, off)
    with pytest.raises(TypeError, match="bfloat16"):
        grouped_matmul(x, w.half(), off)
    for bad in (x[:, :63], x[None], x[0]):
        with pytest.raises(ValueError, match="must be"):
            grouped_matmul(bad, w, off)
    with pytest.raises(ValueError, match="must be"):
        grouped_matmul(x, w[:0], off)
    for bad in (off.long(), off[:2], off[None]):
        with pytest.raises(ValueError, match="offsets"):
            grouped_matmul(x, w, bad)
    with pytest.raises(ValueError, match="checkpoint"):
        grouped_matmul(x, w, off, checkpoint="int8")
    many = w[:1, :1, :1].expand(4097, 1, 64)
    with pytest.raises(RuntimeError, match="too large"):
        grouped_matmul(x, many, torch.zeros(4098, dtype=torch.int32, device=gpu_device))


@pytest.mark.parametrize("table,R,K,N", [
    ([0, 4096, 0, 4096], 4096, 64, 136),  # more row tiles, were the experts apart, than rows have
    ([0, 300, 100, 700, 650, 900], 1000, 72, 40), ([0, -5, 600, -9, 2 ** 31 - 1, 0], 700, 64, 264),
    ([0, 3, 1, 5, 4, 4, 12, 2, 9], 14, 200, 130),  # few rows
    ([0, 160, 0], 170, 4096, 128),  # the contraction in ranges
    ([0] + [(37 * e) % 1001 for e in range(200)], 1100, 64, 136),  # experts past the first 64
    ([0] + [(5 * e) % 131 for e in range(200)], 140, 64, 24),
])
def test_offsets_that_decrease(gpu_device, table, R, K, N):
    """an offset below one before it counts as that one: every row has one expert or none, and its result"""
    from lowbit.experts import grouped_matmul

    E = len(table) - 1
    x, w, dy, _ = _inputs([R] + [0] * (E - 1), K, N, R + E, gpu_device)
    offsets = torch.tensor(table, dtype=torch.int32, device=gpu_device)
    lx, lw = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    unwritten = [torch.full((R, n), float("nan"), dtype=torch.bfloat16, device=gpu_device) for n in (N, K)]
    del unwritten  # the memory that the results take next
    y = grouped_matmul(lx, lw, offsets)
    dx, dw = torch.autograd.grad(y, (lx, lw), dy)
    _check_all(y.detach(), dx, dw, x, w, dy, offsets.cummax(0).values.clamp(0, R))


def test_a_row_of_many_experts_and_columns(gpu_device):
    """few rows whose weights, by 16 columns of every expert a workgroup, would take more threads than a launch has"""
    from lowbit.experts import grouped_matmul

    E, N, K, R = 4096, 65536, 8, 10
    x, w, _, _ = _inputs([R], K, N, 5, gpu_device)
    counts = torch.zeros(E, dtype=torch.int32, device=gpu_device)
    counts[torch.randperm(E, generator=torch.Generator().manual_seed(1))[:R - 2].to(gpu_device)] = 1
    counts[E - 1] += 2
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0).int()])
    with torch.no_grad():
        y = grouped_matmul(x, w.expand(E, N, K), offsets)
    _check(y, x.double() @ w[0].double().t(), K, x.double().abs() @ w[0].double().t().abs(), "y")


def _long(n, rows, cols, seed, dev):
    """a [rows, n] and b [cols, n] of -1, 0 and 1 in bf16 with a b^T exact in fp32 and in bf16, whatever the order: of each
    64 columns one is not zero in a.  Those columns' products cancel in pairs that lie anywhere, but for 66 of them: the
    sums stay below 128, and without any one of the columns each sum is another."""
    g = torch.Generator().manual_seed(seed)
    steps = n // 64
    at = torch.arange(steps) * 64 + torch.randint(0, 64, (steps,), generator=g)
    sa, sb = (torch.randint(0, 2, (m, steps), generator=g) * 2 - 1 for m in (rows, cols))
    order = torch.randperm(steps, generator=g)
    half = (steps - 66) // 2
    sa[:, order[half:2 * half]] = -sa[:, order[:half]]
    sb[:, order[half:2 * half]] = sb[:, order[:half]]
    a = torch.zeros(rows, n)
    a[:, at] = sa.float()
    b = torch.randint(0, 2, (cols, n), generator=g) * 2.0 - 1
    b[:, at] = sb.float()
    want = (sa.double() @ sb.double().t()).float()
    assert want.any() and want.abs().max() < 128
    for lost in (slice(0, 1), slice(steps - 1, steps), slice(0, steps // 16), slice(steps // 2, steps), slice(0, steps)):
        short = want - (sa[:, lost].double() @ sb[:, lost].double().t()).float()
        assert not torch.equal(short, want), lost  # a sum that leaves columns out is told
    return a.bfloat16().to(dev), b.bfloat16().to(dev), want.to(dev)


@pytest.mark.parametrize("n,rows", [(1 << 22, 2), (1 << 18, 40), (1 << 16, 300)])
def test_long_contractions_are_whole(gpu_device, n, rows):
    """sums over the largest K, N and number of rows, exact: by streaming, by ranges, by one tile"""
    from lowbit.experts import grouped_matmul

    offsets = torch.tensor([0, rows, rows], dtype=torch.int32, device=gpu_device)
    x, w, want = _long(n, rows, 5, 1, gpu_device)
    with torch.no_grad():
        y = grouped_matmul(x, w.expand(2, 5, n), offsets)
    assert torch.equal(y.float(), want)
    dy, w, want = _long(n, rows, 16, 2, gpu_device)  # dx = dy W
    lx = torch.zeros(rows, 16, dtype=torch.bfloat16, device=gpu_device, requires_grad=True)
    (dx,) = torch.autograd.grad(grouped_matmul(lx, w.t().contiguous().expand(2, n, 16), offsets), lx, dy)
    assert torch.equal(dx.float(), want)


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_an_expert_of_many_rows_is_whole(gpu_device, checkpoint):
    """dW over 2^20 rows, exact"""
    from lowbit.experts import grouped_matmul

    n = 1 << 20
    dy, x, want = _long(n, 24, 40, 3, gpu_device)
    x, dy = (torch.cat([t.t(), torch.ones_like(t[:, :5]).t()]) for t in (x, dy))  # and an expert of five rows
    offsets = torch.tensor([0, n, n + 5], dtype=torch.int32, device=gpu_device)
    lw = torch.zeros(2, 24, 40, dtype=torch.bfloat16, device=gpu_device, requires_grad=True)
    (dw,) = torch.autograd.grad(grouped_matmul(x, lw, offsets, checkpoint=checkpoint), lw, dy)
    assert torch.equal(dw[0].float(), want) and (dw[1] == 5).all()
