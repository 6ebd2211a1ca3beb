"""GPU tests of lowbit.router.route_tokens against the definition in 64 bits.

The ids are compared as whole numbers wherever the 64-bit order of the choices
does not hang on the last bits of a 32-bit score: a row is compared when each
gap between consecutive chosen experts (and to the first one left out, and
between the groups at the edge) is 0 or at least 4e-6 of the choice and score,
which is over ten times what fp32 scores can be off (two roundings of exp, the
sum of at most 1024 terms in a tree, the division, the addition of the bias:
under 16 u = 1e-6 relative).  The inputs are such that at least 90% of the rows
are.  Weights and gradients, for the kernel's own ids: 64 u of the magnitudes
that enter plus the output's rounding.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 1e-37, torch.float16: 2.0 ** -24, torch.bfloat16: 1e-37}
EPS = 1e-20


def _scores(z, score):
    z = z.double()
    if score == "sigmoid":
        return torch.sigmoid(z)
    return torch.nan_to_num(torch.softmax(z, -1), nan=0.0) if z.isneginf().all(-1).any() else torch.softmax(z, -1)


def _reference(z, k, score, bias, G, Gk):
    """ids [T, k] in 64 bits and which rows' order is clear"""
    p = _scores(z, score)
    c = p if bias is None else p + bias.double()
    T, E = c.shape
    clear = torch.ones(T, dtype=torch.bool, device=z.device)
    if Gk < G:
        gs = c.reshape(T, G, E // G).sort(dim=2, descending=True).values[:, :, :2].sum(2)
        o = gs.sort(dim=1, descending=True, stable=True)
        gap = o.values[:, Gk - 1] - o.values[:, Gk]
        clear &= (gap == 0) | (gap > 8e-6 * (o.values[:, Gk - 1].abs() + 1e-3))
        kept = torch.zeros(T, G, dtype=torch.bool, device=z.device).scatter_(1, o.indices[:, :Gk], True)
        c = torch.where(kept.repeat_interleave(E // G, 1), c, float("-inf"))
    o = c.sort(dim=1, descending=True, stable=True)
    n = min(k + 1, E)
    v, pv = o.values[:, :n], p.gather(1, o.indices[:, :n])
    gap = v[:, :-1] - v[:, 1:]
    tie = (gap == 0) | (v[:, :-1] == v[:, 1:])
    clear &= (tie | (gap > 4e-6 * (v[:, :-1].abs() + pv[:, :-1]))).all(1)
    return o.indices[:, :k].int(), clear


def _check_ids(ids, z, k, score, bias, G, Gk, share=0.9):
    want, clear = _reference(z, k, score, bias, G, Gk)
    assert clear.float().mean() >= share
    assert torch.equal(ids[clear], want[clear])
    srt = ids.sort(1).values
    assert (ids >= 0).all() and (ids < z.shape[1]).all() and (srt[:, 1:] > srt[:, :-1]).all()


def _check_weights(w, dz, z, ids, score, renorm, scale, dw=None):
    zd = z.double().requires_grad_(True)
    p = _scores(zd, score).gather(1, ids.long())
    s = p.sum(1, keepdim=True) + EPS
    want = scale * (p / s if renorm else p)
    assert ((w.double() - want).abs() <= 64 * U * want.abs() + 1e-37).all()
    if dw is None:
        return
    (gz,) = torch.autograd.grad(want, zd, dw.double())
    d = scale * dw.double().abs()
    pd = p.detach()
    if renorm:
        sd = s.detach()
        d = (d + (d * pd).sum(1, keepdim=True) / sd) / sd  # magnitudes that meet at a chosen score
    allp = _scores(z, score)
    if score == "softmax":
        dp = torch.zeros_like(allp).scatter_(1, ids.long(), d)
        mag = allp * (dp + (d * pd).sum(1, keepdim=True))
    else:
        mag = torch.zeros_like(allp).scatter_(1, ids.long(), d * pd * (1 - pd))
    bound = 64 * U * mag + ROUND[dz.dtype] * gz.abs() + LEAST[dz.dtype]
    assert ((dz.double() - gz).abs() <= bound).all()


def _inputs(T, E, dtype, seed, dev, biased):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(T, E, generator=g) * 1.5).to(dtype).to(dev)
    b = (0.1 * torch.randn(E, generator=g)).to(dev) if biased else None
    return z, b, g


# T, E, k, score, bias, groups, kept groups, renormalize, scale
CASES = [
    (1, 1, 1, "softmax", False, 1, 1, False, 1.0),
    (1, 256, 8, "sigmoid", True, 8, 4, True, 2.5),
    (4, 8, 8, "softmax", False, 1, 1, True, 1.0),
    (777, 32, 8, "softmax", False, 1, 1, True, 1.0),
    (1001, 60, 6, "softmax", False, 1, 1, False, 16.0),
    (333, 64, 4, "sigmoid", False, 4, 2, True, 1.0),
    (501, 96, 5, "softmax", True, 8, 3, True, 1.0),
    (259, 160, 6, "softmax", False, 8, 3, False, 16.0),
    (2000, 256, 8, "sigmoid", True, 8, 4, True, 2.5),
    (77, 250, 16, "sigmoid", False, 1, 1, True, 1.0),
    (64, 255, 1, "softmax", True, 15, 2, False, 1.0),
    (130, 384, 8, "sigmoid", True, 1, 1, True, 2.5),
    (41, 512, 12, "softmax", True, 16, 7, True, 1.0),
    (70, 1000, 16, "sigmoid", True, 10, 4, True, 1.0),
    (9, 1024, 3, "softmax", False, 1, 1, False, 1.0),
    (33, 16, 2, "sigmoid", True, 16, 5, True, 1.0),
    (50, 48, 16, "softmax", False, 3, 1, False, 1.0),
    (70001, 24, 2, "softmax", True, 1, 1, True, 1.0),
]


@pytest.mark.parametrize("T,E,k,score,biased,G,Gk,renorm,scale", CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_ids_weights_gradient(gpu_device, T, E, k, score, biased, G, Gk, renorm, scale, dtype):
    from lowbit.router import route_tokens

    z, b, g = _inputs(T, E, dtype, T + E, gpu_device, biased)
    dw = torch.randn(T, k, generator=g).to(gpu_device)
    zl = z.clone().requires_grad_(True)
    kw = dict(score=score, bias=b, n_groups=G, topk_groups=Gk, renormalize=renorm, scale=scale)
    ids, w = route_tokens(zl, k, **kw)
    assert ids.dtype == torch.int32 and w.dtype == torch.float32 and ids.shape == w.shape == (T, k)
    (dz,) = torch.autograd.grad(w, zl, dw)
    assert dz.dtype == dtype
    _check_ids(ids, z, k, score, b, G, Gk)
    _check_weights(w.detach(), dz, z, ids, score, renorm, scale, dw)
    with torch.no_grad():
        ids0, w0 = route_tokens(z, k, **kw)
    assert torch.equal(ids, ids0) and torch.equal(w.detach(), w0)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_ties_go_to_the_lowest_index(gpu_device, score):
    from lowbit.router import route_tokens

    z = torch.zeros(5, 200, device=gpu_device)
    z[1, 50:] = 1.0
    z[2, ::3] = 2.0
    z[3] = -0.0
    z[3, ::2] = 0.0
    z[4, 7], z[4, 150] = 3.0, 3.0
    ids, _ = route_tokens(z, 8, score=score)
    assert ids[0].tolist() == list(range(8)) and ids[3].tolist() == list(range(8))
    assert ids[1].tolist() == list(range(50, 58))
    assert ids[2].tolist() == list(range(0, 24, 3))
    assert ids[4].tolist() == [7, 150, 0, 1, 2, 3, 4, 5]
    ids, _ = route_tokens(z, 8, score=score, n_groups=8, topk_groups=2)
    assert ids[0].tolist() == list(range(8))  # equal groups: the first two


def test_masked_experts(gpu_device):
    """logits and biases of -inf; rows with fewer than top_k experts left, and with none"""
    from lowbit.router import route_tokens

    inf = float("inf")
    z = torch.randn(6, 64, generator=torch.Generator().manual_seed(1)).to(gpu_device)
    z[0, 10:] = -inf
    z[1, 3:] = -inf
    z[2] = -inf
    z[3] = torch.finfo(torch.float32).min
    zl = z.clone().requires_grad_(True)
    ids, w = route_tokens(zl, 8, score="softmax")
    w.sum().backward()
    assert (ids[0] < 10).all() and sorted(ids[1].tolist()) == list(range(8))
    assert w[1].detach()[3:].eq(0).all() and abs(float(w[1].detach().sum()) - 1) < 1e-6
    assert ids[2].tolist() == list(range(8)) and w[2].eq(0).all()
    assert ids[3].tolist() == list(range(8)) and (w[3] - 0.125).abs().max() < 1e-6
    assert zl.grad.isfinite().all() and zl.grad[2].eq(0).all()
    b = torch.zeros(64, device=gpu_device)
    b[5:] = -inf
    ids, w = route_tokens(z[4:], 8, score="sigmoid", bias=b, renormalize=False)
    assert all(sorted(r[:5]) == [0, 1, 2, 3, 4] and r[5:] == [5, 6, 7] for r in ids.tolist())
    assert torch.allclose(w, torch.sigmoid(z[4:].gather(1, ids.long())), rtol=1e-6, atol=0)
    b[:] = -inf
    ids, _ = route_tokens(z[4:], 8, score="sigmoid", bias=b, n_groups=4, topk_groups=1)
    assert ids.tolist() == [list(range(8))] * 2


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("G,Gk", [(1, 1), (8, 2)])
def test_nan_and_infinite_logits_give_valid_ids(gpu_device, score, G, Gk):
    from lowbit.router import route_tokens

    z = torch.randn(40, 256, generator=torch.Generator().manual_seed(2)).to(gpu_device)
    clean, wc = route_tokens(z, 8, score=score, n_groups=G, topk_groups=Gk)
    z[3, 17] = float("nan")
    z[9] = float("nan")
    z[11, 100] = float("inf")
    z[20] = float("inf")
    z[30, :5] = 200.0
    ids, w = route_tokens(z, 8, score=score, n_groups=G, topk_groups=Gk)
    srt = ids.sort(1).values
    assert (ids >= 0).all() and (ids < 256).all() and (srt[:, 1:] > srt[:, :-1]).all()
    same = torch.ones(40, dtype=torch.bool, device=gpu_device)
    same[[3, 9, 11, 20, 30]] = False
    assert torch.equal(ids[same], clean[same]) and torch.equal(w[same], wc[same])
    assert w[3].isnan().any() and w[9].isnan().all()
    if score == "sigmoid":
        assert ids[3, 0] == 17 and w[11].isfinite().all()


@pytest.mark.parametrize("which", ["pitch", "offset", "transposed", "repeated", "3d"])
def test_strides(gpu_device, which):
    from lowbit.router import route_tokens

    T, E, k = 60, 90, 6
    z, _, g = _inputs(T, E + 5, torch.bfloat16, 3, gpu_device, False)
    zv = {"pitch": z[:, :E], "offset": z[:, 3:3 + E], "transposed": z[:, :E].t().contiguous().t(),
          "repeated": z[:1, :E].expand(T, E), "3d": z[:, :E].reshape(6, 10, E)}[which]
    dw = torch.randn(T, k, generator=g).to(gpu_device)
    zl = zv.detach().requires_grad_(True)
    ids, w = route_tokens(zl, k)
    (dz,) = torch.autograd.grad(w, zl, dw.reshape(w.shape))
    assert ids.shape == zv.shape[:-1] + (k,) and dz.shape == zv.shape
    zr, ids = zv.reshape(T, E), ids.reshape(T, k)
    _check_ids(ids, zr, k, "softmax", None, 1, 1)
    _check_weights(w.detach().reshape(T, k), dz.reshape(T, E), zr, ids, "softmax", True, 1.0, dw)


def test_gradient_against_differences(gpu_device):
    """central differences of the kernel's own weights where no choice changes, at h and 2h with the h^2 term removed;
    rounding is below 8 u scale / h"""
    from lowbit.router import route_tokens

    h = 2.0 ** -7
    for score, renorm in (("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)):
        # choices far apart, so that the steps do not reorder them
        g = torch.Generator().manual_seed(4)
        z = torch.stack([torch.randperm(40, generator=g).float() * 0.15 - 3 for _ in range(30)]).to(gpu_device)
        v = torch.randn(30, 40, generator=g).clamp(-2, 2).to(gpu_device)
        dw = torch.randn(30, 5, generator=g).to(gpu_device)
        zl = z.clone().requires_grad_(True)
        ids, w = route_tokens(zl, 5, score=score, renormalize=renorm, scale=2.0)
        (dz,) = torch.autograd.grad(w, zl, dw)

        def f(s):
            i, x = route_tokens(z + s * v, 5, score=score, renormalize=renorm, scale=2.0)
            assert torch.equal(i, ids)
            return (x.double() * dw.double()).sum()

        d1, d2 = (f(h) - f(-h)) / (2 * h), (f(2 * h) - f(-2 * h)) / (4 * h)
        scale = float((w.detach() * dw).abs().sum())
        want = float((dz.double() * v.double()).sum())
        assert abs(float((4 * d1 - d2) / 3) - want) <= abs(float(d1 - d2)) + 8 * U * scale / h


def test_no_tokens(gpu_device):
    from lowbit.router import route_tokens

    z = torch.empty(0, 32, device=gpu_device, requires_grad=True)
    ids, w = route_tokens(z, 4)
    assert ids.shape == w.shape == (0, 4)
    w.sum().backward()
    assert z.grad.shape == (0, 32)


def test_other_stream_and_graph(gpu_device):
    from lowbit.router import route_tokens

    z, b, _ = _inputs(100, 256, torch.float32, 8, gpu_device, True)
    kw = dict(score="sigmoid", bias=b, n_groups=8, topk_groups=4)
    want = route_tokens(z, 8, **kw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = route_tokens(z, 8, **kw)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = route_tokens(z, 8, **kw)
    for k in range(3):
        z.copy_(torch.randn(100, 256, generator=torch.Generator().manual_seed(k)).to(z))
        graph.replay()
        torch.cuda.synchronize()
        now = route_tokens(z, 8, **kw)
        assert torch.equal(out[0], now[0]) and torch.equal(out[1], now[1])


def test_module_routes_and_balances(gpu_device):
    from lowbit.router import TopKRouter

    torch.manual_seed(0)
    r = TopKRouter(64, 16, 2, score="sigmoid", balance_bias=True, device=gpu_device)
    x = torch.randn(500, 64, device=gpu_device) + 1.0
    ids, w = r(x)
    w.square().sum().backward()
    assert r.weight.grad.isfinite().all() and r.weight.grad.any()
    spread = lambda i: torch.bincount(i.reshape(-1).long(), minlength=16).float().std()  # noqa: E731
    first = spread(ids)
    for _ in range(60):
        with torch.no_grad():
            ids, _ = r(x)
        r.update_bias(ids, rate=0.01)
    assert spread(ids) < 0.5 * first


def test_refusals(gpu_device):
    from lowbit.router import TopKRouter, route_tokens

    z = torch.randn(4, 32, device=gpu_device)
    with pytest.raises(RuntimeError, match="ROCm device"):
        route_tokens(torch.randn(4, 32), 2)
    with pytest.raises(ValueError, match="score"):
        route_tokens(z, 2, score="tanh")
    with pytest.raises(ValueError, match="1024"):
        route_tokens(torch.randn(2, 1025, device=gpu_device), 2)
    for k in (0, 17, 33):
        with pytest.raises(ValueError, match="top_k"):
            route_tokens(z, k)
    with pytest.raises(ValueError, match="groups"):
        route_tokens(z, 2, n_groups=5)
    with pytest.raises(ValueError, match="topk_groups"):
        route_tokens(z, 2, n_groups=4, topk_groups=5)
    with pytest.raises(ValueError, match="top_k"):
        route_tokens(z, 9, n_groups=4, topk_groups=1)
    with pytest.raises(ValueError, match="bias"):
        route_tokens(z, 2, bias=torch.zeros(31, device=gpu_device))
    with pytest.raises(ValueError, match="bias"):
        route_tokens(z, 2, bias=torch.zeros(32, device=gpu_device, dtype=torch.float16))
    with pytest.raises(TypeError, match="dtype"):
        route_tokens(z.double(), 2)
    with pytest.raises(RuntimeError, match="balance bias"):
        TopKRouter(8, 4, 2, device=gpu_device).update_bias(torch.zeros(1, 2, device=gpu_device))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("k", [2, 5])
def test_gradients_nearly_alike_do_not_cancel(gpu_device, score, k):
    """dw of one large value and small differences: the renormalised weights' sum is one, so the large value has no part in
    the gradient.  Formed from differences, each of a few roundings, what is left is off by roundings of the differences'
    size; the sum d p would be off by roundings of the large value, a thousand times more"""
    from lowbit.router import route_tokens

    g = torch.Generator().manual_seed(k)
    z = torch.randn(64, 40, generator=g).to(gpu_device).requires_grad_(True)
    dw = (1024.0 + torch.randint(-64, 65, (64, k), generator=g) / 64.0).to(gpu_device)  # exact in fp32
    ids, w = route_tokens(z, k, score=score)
    (dz,) = torch.autograd.grad(w, z, dw)
    zd = z.detach().double().requires_grad_(True)
    p = (torch.softmax(zd, 1) if score == "softmax" else torch.sigmoid(zd)).gather(1, ids.long())
    (want,) = torch.autograd.grad(p / p.sum(1, keepdim=True), zd, dw.double())
    # |c| <= 2; c, its mean, their difference, p and its factors: at most 64 roundings of values below 4 |dw/dz|
    assert (dz.double() - want).abs().max() <= 64 * U * 4


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("G,Gk", [(1, 1), (8, 2), (3, 1)])
@pytest.mark.parametrize("renorm", [True, False])
def test_sigmoid_of_logits_far_below_zero(gpu_device, dtype, G, Gk, renorm):
    """scores that underflow, at -inf, the types' lowest values and below -85, beside k experts in each group that do not:
    those are chosen, and a low one weighs its sigmoid, never NaN"""
    from lowbit.router import route_tokens

    T, E, k = 300, 96, 6
    g = torch.Generator().manual_seed(21)
    low = torch.cat([torch.tensor([-float("inf"), torch.finfo(torch.float32).min, torch.finfo(torch.bfloat16).min, -65504.0,
                                   -1000.0, -200.0, -177.0]), torch.linspace(-180, -85, 401)])
    z = torch.randn(T, E, generator=g) * 1.5
    per = E // G
    keep = torch.rand(T, G, per, generator=g).argsort(-1).argsort(-1) < k  # k of each group's experts
    z = torch.where(keep.reshape(T, E), z, low[torch.randint(low.numel(), (T, E), generator=g)]).to(dtype).to(gpu_device)
    dw = torch.randn(T, k, generator=g).to(gpu_device)
    zl = z.clone().requires_grad_(True)
    for bias in (None, torch.zeros(E, device=gpu_device)):
        ids, w = route_tokens(zl, k, score="sigmoid", bias=bias, n_groups=G, topk_groups=Gk, renormalize=renorm)
        (dz,) = torch.autograd.grad(w, zl, dw)
        _check_ids(ids, z, k, "sigmoid", None, G, Gk)
        _check_weights(w.detach(), dz, z, ids, "sigmoid", renorm, 1.0, dw)
        assert dz.isfinite().all()


@pytest.mark.parametrize("low", [-float("inf"), torch.finfo(torch.float32).min, -1e5, -200.0, -178.5])
@pytest.mark.parametrize("biased", [False, True])
def test_sigmoid_of_masked_experts(gpu_device, low, biased):
    """fewer experts than top_k are left beside those masked by their logits (and by a bias of -inf): they come first,
    then the masked ones, lowest index first and of no weight"""
    from lowbit.router import route_tokens

    z = torch.full((3, 40), low)
    z[0, [30, 7, 12]] = torch.tensor([2.0, 1.0, 0.5])
    z[1, 39] = -3.0
    b = torch.zeros(40, device=gpu_device)
    if biased:
        b[[i for i in range(40) if i not in (7, 12, 30, 39)]] = -float("inf")
    zl = z.to(gpu_device).requires_grad_(True)
    for G, Gk in ((1, 1), (2, 2)):
        ids, w = route_tokens(zl, 8, score="sigmoid", bias=b if biased else None, n_groups=G, topk_groups=Gk)
        if biased:
            assert ids.tolist() == [[30, 7, 12, 39, 0, 1, 2, 3], [39, 7, 12, 30, 0, 1, 2, 3], [7, 12, 30, 39, 0, 1, 2, 3]]
        else:
            assert ids.tolist() == [[30, 7, 12, 0, 1, 2, 3, 4], [39, 0, 1, 2, 3, 4, 5, 6], list(range(8))]
        want = torch.zeros(3, 8, dtype=torch.float64)
        p = torch.sigmoid(torch.tensor([2.0, 1.0, 0.5], dtype=torch.float64))
        want[0, :3], want[1, 0] = p / p.sum(), 1.0
        assert (w.detach().cpu().double() - want).abs().max() <= 64 * U
        (dz,) = torch.autograd.grad(w.square().sum(), zl)
        assert dz.isfinite().all()


def test_sigmoid_from_minus_180_to_minus_85(gpu_device):
    """every expert's score where exp(-z) nears and passes the largest float: to 1e-37 the sigmoid, and in its order"""
    from lowbit.router import route_tokens

    z = torch.linspace(-180, -85, 16 * 4096).reshape(16, 4096).t().contiguous().to(gpu_device)
    ids, w = route_tokens(z, 16, score="sigmoid", renormalize=False)
    want = torch.sigmoid(z.double()).gather(1, ids.long())
    assert ((w.double() - want).abs() <= 64 * U * want + 1e-37).all() and (w >= 0).all()
    assert (w[:, 1:] <= w[:, :-1]).all()


def test_update_bias_does_not_wait_for_the_device(gpu_device):
    from lowbit.router import TopKRouter

    r = TopKRouter(64, 16, 2, score="sigmoid", balance_bias=True, device=gpu_device)
    ids = torch.randint(0, 16, (500, 2), device=gpu_device, dtype=torch.int32)
    load = torch.bincount(ids.reshape(-1).long(), minlength=16).float()
    torch.cuda.set_sync_debug_mode("error")
    try:
        r.update_bias(ids, rate=0.25)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    want = 0.25 * torch.sign(load.mean() - load)
    assert torch.equal(r.balance_bias, want)
    r.update_bias(torch.cat([ids.reshape(-1), torch.tensor([-1, 16, 1 << 30], dtype=torch.int32, device=gpu_device)]), rate=0.25)
    assert torch.equal(r.balance_bias, 2 * want)  # what is no expert's id is not counted


def test_the_balance_bias_stays_fp32(gpu_device):
    """a module's type is changed as a whole: the bias, whose steps fewer bits would swallow, keeps its own and its values"""
    from lowbit.router import TopKRouter

    r = TopKRouter(64, 16, 2, score="sigmoid", balance_bias=True)
    r.balance_bias += 0.1001
    r = r.to(gpu_device).bfloat16()
    assert r.weight.dtype == torch.bfloat16 and r.balance_bias.dtype == torch.float32 and r.balance_bias.is_cuda
    assert torch.equal(r.balance_bias.cpu(), torch.full((16,), 0.0) + 0.1001)
    ids, w = r(torch.randn(5, 64, device=gpu_device).bfloat16())
    assert ids.shape == (5, 2) and w.isfinite().all()
    assert TopKRouter(8, 4, 2).half().balance_bias is None
