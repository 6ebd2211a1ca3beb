"""Timed cases of the operators around the low-bit products of an MoE language model's training step.

The recipe keeps three parts of such a model in high precision: its norms, its routers and its head.  Each is one
operator here, called through a public entry point of ``lowbit``:

  norm    layer_norm(x, weight, bias): the norm in front of a low-bit Linear or of the expert loop; trained, also the
          gradients of x, weight and bias
  route   route_tokens(logits, top_k, ...): scores of a token's experts, the choice of groups and experts, and the
          routing weights that local_moe() takes; trained, also the gradient of the logits
  xent    linear_cross_entropy(hidden, weight, targets): the head's product and the softmax cross entropy over the
          vocabulary; trained, also the gradients of hidden and weight

``own`` False computes them in elementary torch operations in 32 bits, True by the package's kernels.  Every case is
made from its seed on the GPU.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
IGNORE = -100
RENORM_EPS = 1e-20  # added to a token's chosen scores' sum before the division

# the largest listed case (the 4096-token head) bounds what a drawn case may cost
MAX_FLOPS = 2.4e13
MAX_BYTES = 4.0e9


def listed():
    return [
        # a generation step: the one new token's norm before a 7168-wide projection
        dict(name="norm_fwd_1", op="norm", train=False, T=1, H=7168, dtype="bf16", wdtype="bf16"),
        # a training step's norm in front of the 7168-wide MLP, 8192 tokens
        dict(name="norm_train_8192", op="norm", train=True, T=8192, H=7168, dtype="bf16", wdtype="bf16"),
        # a small fp32 model whose sizes are no multiples of anything
        dict(name="norm_train_odd", op="norm", train=True, T=1003, H=1541, dtype="f32", wdtype="f32"),
        # many short rows: a long batch of a narrow fp16 model whose norm weights stay fp32
        dict(name="norm_train_narrow", op="norm", train=True, T=65536, H=512, dtype="f16", wdtype="f32"),
        # generation with 32 sequences: 256 experts in 8 groups, sigmoid scores with a balance bias, top 8 of 4 groups
        dict(name="route_fwd_32", op="route", train=False, T=32, E=256, k=8, score="sigmoid", bias=True, G=8, Gk=4,
             renorm=True, scale=2.5, dtype="f32"),
        # the router of the 4096-token expert loop: 32 experts, softmax scores, top 8
        dict(name="route_train_4096", op="route", train=True, T=4096, E=32, k=8, score="softmax", bias=False, G=1, Gk=1,
             renorm=True, scale=1.0, dtype="bf16"),
        # a large training batch over 256 experts in groups
        dict(name="route_train_65536", op="route", train=True, T=65536, E=256, k=8, score="sigmoid", bias=True, G=8,
             Gk=4, renorm=True, scale=2.5, dtype="f32"),
        # odd sizes: 60 experts, plain softmax weights of the top 6
        dict(name="route_train_odd", op="route", train=True, T=5001, E=60, k=6, score="softmax", bias=False, G=1, Gk=1,
             renorm=False, scale=1.0, dtype="f16"),
        # scoring: the log-likelihood of 16 positions under a 131072-token vocabulary, no gradients
        dict(name="xent_score_16", op="xent", train=False, T=16, H=4096, V=131072, ignored=0.0, reduction="none"),
        # a small model's training step, nothing a multiple of anything, 40% of the positions masked (prompts, padding)
        dict(name="xent_train_odd", op="xent", train=True, T=1003, H=1000, V=10007, ignored=0.4, reduction="mean"),
        # an ordinary head: 2048 tokens, 32768 words, a gradient of its own for each position
        dict(name="xent_train_2048", op="xent", train=True, T=2048, H=2048, V=32768, ignored=0.0, reduction="none"),
        # a large head: 4096 tokens 7168 wide, 131072 words
        dict(name="xent_train_4096", op="xent", train=True, T=4096, H=7168, V=131072, ignored=0.05, reduction="mean"),
    ]


def _size(rng, lo: int, hi: int, mult: int = 1) -> int:
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(mult, (v + mult // 2) // mult * mult)


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if w["flops"] <= MAX_FLOPS and w["bytes"] <= MAX_BYTES:
            return case


def _draw(rng):
    op = rng.choice(("norm", "route", "xent"))
    train = rng.random() < 0.67
    if op == "norm":
        dt = rng.choice(("bf16", "f16", "f32"))
        return dict(op=op, train=train, T=_size(rng, 1, 65536), H=_size(rng, 64, 8192, rng.choice((1, 8, 64))), dtype=dt,
                    wdtype=rng.choice((dt, "f32")))
    if op == "route":
        groups = rng.choice((1, 1, 2, 4, 8))
        E = groups * _size(rng, max(1, 8 // groups), 512 // groups)
        Gk = rng.randint(1, groups)
        k = rng.randint(1, min(8, Gk * (E // groups)))
        return dict(op=op, train=train, T=_size(rng, 1, 65536), E=E, k=k, score=rng.choice(("softmax", "sigmoid")),
                    bias=rng.random() < 0.5, G=groups, Gk=Gk,
                    renorm=k > 1 and rng.random() < 0.7,  # one weight renormalised is a constant
                    scale=rng.choice((1.0, 2.5)), dtype=rng.choice(("f32", "bf16", "f16")))
    m = rng.choice((1, 8, 64))  # model widths are round; small models' are not always
    return dict(op=op, train=train, T=_size(rng, 1, 8192), H=_size(rng, 128, 7168, m), V=_size(rng, 256, 131072, m),
                ignored=rng.choice((0.0, 0.05, 0.4)), reduction=rng.choice(("mean", "sum", "none")))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    return {"norm": _norm_inputs, "route": _route_inputs, "xent": _xent_inputs}[case["op"]](dict(case), g)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _norm_inputs(c, g):
    dt, wdt = DTYPES[c["dtype"]], DTYPES[c["wdtype"]]
    T, H = c["T"], c["H"]
    # a residual stream: channels of unequal size, rows off centre
    x = _randn(g, T, H) * torch.exp(0.7 * _randn(g, H)) + 0.5 * _randn(g, T, 1)
    s = dict(case=c, eps=1e-5, x=x.to(dt), w=(1.0 + 0.2 * _randn(g, H)).to(wdt), b=(0.1 * _randn(g, H)).to(wdt))
    if c["train"]:
        s["dy"] = _randn(g, T, H).to(dt)
        for k in ("x", "w", "b"):
            s[k].requires_grad_(True)
    return s


def _choices(c, logits, bias):
    """Scores and choices of every expert in 64 bits, and the choices with those of groups left out at -inf."""
    z = logits.double()
    p = torch.softmax(z, -1) if c["score"] == "softmax" else torch.sigmoid(z)
    ch = p if bias is None else p + bias.double()
    T, E, G = z.shape[0], c["E"], c["G"]
    if G == 1:
        return p, ch, ch, None
    best = ch.reshape(T, G, E // G).sort(dim=-1, descending=True).values[..., :2].sum(-1)
    order = best.sort(dim=-1, descending=True, stable=True)
    keep = torch.zeros(T, G, dtype=torch.bool, device=z.device).scatter_(1, order.indices[:, : c["Gk"]], True)
    return p, ch, torch.where(keep.repeat_interleave(E // G, 1), ch, float("-inf")), order.values


def _route_inputs(c, g):
    T, E, k = c["T"], c["E"], c["k"]
    dt = DTYPES[c["dtype"]]
    tilt = 0.5 * _randn(g, E)  # popular and unpopular experts
    bias = (-0.1 * tilt + 0.02 * _randn(g, E)) if c["bias"] else None  # what balancing has learnt against them
    logits = (_randn(g, T, E) + tilt).to(dt)
    # The expert ids are whole numbers, compared as such.  Rows where the order of two experts, or of two groups at
    # the edge of the choice, hangs on the last bits of a 32-bit score are drawn again; equal logits stay (ties).
    for _ in range(200):
        p, ch, masked, best = _choices(c, logits, bias)
        top = masked.sort(dim=-1, descending=True)
        n = min(k + 1, E)
        v, pv = top.values[:, :n], p.gather(1, top.indices[:, :n])
        gap = v[:, :-1] - v[:, 1:]
        near = (gap > 0) & (gap < 4e-6 * (v[:, :-1].abs() + pv[:, :-1]))
        bad = near.any(1) if n > 1 else torch.zeros(T, dtype=torch.bool, device=DEV)
        if best is not None and c["Gk"] < c["G"]:
            a, b = best[:, c["Gk"] - 1], best[:, c["Gk"]]
            bad |= (a - b > 0) & (a - b < 8e-6 * (a.abs() + 1e-3))
        rows = bad.nonzero()[:, 0]
        if rows.numel() == 0:
            break
        logits[rows] = (_randn(g, rows.numel(), E) + tilt).to(dt)
    else:
        raise RuntimeError("no separated routing inputs")
    s = dict(case=c, logits=logits, bias=bias)
    if c["train"]:
        s["dw"] = _randn(g, T, k)
        s["logits"].requires_grad_(True)
    return s


def _xent_inputs(c, g):
    T, H, V = c["T"], c["H"], c["V"]
    w = (0.02 * _randn(g, V, H)).to(torch.bfloat16)
    # words by Zipf's law, scattered over the vocabulary
    rank = torch.exp(torch.rand(T, generator=g, device=DEV, dtype=torch.float64) * math.log(V + 1)).long().clamp(1, V) - 1
    y = torch.randperm(V, generator=g, device=DEV)[rank]
    # hidden rows that have learnt something: they lean to their word's row by a varying amount
    lean = 3.0 / math.sqrt(H) * torch.rand(T, 1, generator=g, device=DEV)
    x = (_randn(g, T, H) + lean * 50.0 * w[y].float()).to(torch.bfloat16)
    y = torch.where(torch.rand(T, generator=g, device=DEV) < c["ignored"], IGNORE, y)
    s = dict(case=c, x=x, w=w, y=y)
    if c["train"]:
        if c["reduction"] == "none":
            s["dl"] = torch.rand(T, generator=g, device=DEV) / T
        s["x"].requires_grad_(True)
        s["w"].requires_grad_(True)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _norm_own, "route": _route_own, "xent": _xent_own}[op](state)
    with torch.no_grad():
        return {"norm": _norm_plain, "route": _route_plain, "xent": _xent_plain}[op](state)


def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nano-train_amd")
    if at not in sys.path:
        sys.path.insert(0, at)


def _norm_own(s):
    _package()
    from lowbit.norm import layer_norm

    if not s["case"]["train"]:
        return {"y": layer_norm(s["x"], s["w"], s["b"], eps=s["eps"])}
    y = layer_norm(s["x"], s["w"], s["b"], eps=s["eps"])
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}


def _route_own(s):
    _package()
    from lowbit.router import route_tokens

    c = s["case"]
    ids, w = route_tokens(s["logits"], c["k"], score=c["score"], bias=s["bias"], n_groups=c["G"], topk_groups=c["Gk"],
                          renormalize=c["renorm"], scale=c["scale"])
    if not c["train"]:
        return {"ids": ids, "w": w}
    (dl,) = torch.autograd.grad(w, (s["logits"],), s["dw"])
    return {"ids": ids, "w": w.detach(), "dlogits": dl}


def _xent_own(s):
    _package()
    from lowbit.loss import linear_cross_entropy

    c = s["case"]
    loss = linear_cross_entropy(s["x"], s["w"], s["y"], ignore_index=IGNORE, reduction=c["reduction"])
    if not c["train"]:
        return {"loss": loss}
    dx, dw = torch.autograd.grad(loss, (s["x"], s["w"]), s.get("dl"))
    return {"loss": loss.detach(), "dx": dx, "dw": dw}


def _norm_plain(s):
    x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
    d = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((d * d).mean(1, keepdim=True) + s["eps"])
    xhat = d * rstd
    y = (xhat * w + b).to(s["x"].dtype)
    if not s["case"]["train"]:
        return {"y": y}
    dy = s["dy"].float()
    t = dy * w
    dx = rstd * (t - t.mean(1, keepdim=True) - xhat * (t * xhat).mean(1, keepdim=True))
    return {"y": y, "dx": dx.to(s["x"].dtype), "dw": (dy * xhat).sum(0).to(s["w"].dtype), "db": dy.sum(0).to(s["b"].dtype)}


def _route_plain(s):
    c = s["case"]
    z = s["logits"].float()
    T, E, G, k = c["T"], c["E"], c["G"], c["k"]
    if c["score"] == "softmax":
        e = torch.exp(z - z.amax(1, keepdim=True))
        p = e / e.sum(1, keepdim=True)
    else:
        p = 1.0 / (1.0 + torch.exp(-z))
    ch = p if s["bias"] is None else p + s["bias"]
    if G > 1:  # a group's score: the sum of its two highest choices
        best = torch.sort(ch.reshape(T, G, E // G), dim=2, descending=True).values[:, :, :2].sum(2)
        groups = torch.sort(best, dim=1, descending=True, stable=True).indices[:, : c["Gk"]]
        out = torch.ones(T, G, dtype=torch.bool, device=z.device)
        out[torch.arange(T, device=z.device)[:, None], groups] = False
        ch = torch.where(out.repeat_interleave(E // G, 1), float("-inf"), ch)
    ids = torch.sort(ch, dim=1, descending=True, stable=True).indices[:, :k]
    chosen = torch.gather(p, 1, ids)
    total = chosen.sum(1, keepdim=True) + RENORM_EPS
    w = c["scale"] * (chosen / total if c["renorm"] else chosen)
    if not c["train"]:
        return {"ids": ids.int(), "w": w}
    dc = c["scale"] * s["dw"]
    if c["renorm"]:
        dc = (dc - (dc * chosen).sum(1, keepdim=True) / total) / total
    dp = torch.zeros_like(p)
    dp.scatter_(1, ids, dc)
    dz = p * (dp - (dp * p).sum(1, keepdim=True)) if c["score"] == "softmax" else dp * p * (1.0 - p)
    return {"ids": ids.int(), "w": w, "dlogits": dz.to(s["logits"].dtype)}


def _xent_plain(s):
    c = s["case"]
    x, w, y = s["x"].float(), s["w"].float(), s["y"]
    live = y != IGNORE
    at = torch.where(live, y, 0)[:, None]
    z = x @ w.t()
    z -= z.amax(1, keepdim=True)
    label = torch.gather(z, 1, at)[:, 0]
    e = z.exp_()
    total = e.sum(1, keepdim=True)
    each = torch.where(live, torch.log(total[:, 0]) - label, 0.0)
    n = live.sum().clamp(min=1).float()
    loss = {"none": each, "sum": each.sum(), "mean": each.sum() / n}[c["reduction"]]
    if not c["train"]:
        return {"loss": loss}
    up = s["dl"] if c["reduction"] == "none" else (1.0 / n if c["reduction"] == "mean" else torch.ones_like(n)).expand(c["T"])
    up = torch.where(live, up, 0.0)[:, None]
    dz = e.div_(total)
    dz.scatter_add_(1, at, torch.full_like(up, -1.0))
    dz *= up
    return {"loss": loss, "dx": (dz @ w).to(s["x"].dtype), "dw": (dz.t() @ x).to(s["w"].dtype)}


# ---------------------------------------------------------------------------
# the definitions in 64 bits, gradients by automatic differentiation
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "xent" and float(c["T"]) * c["V"] > 6e8:
        return None  # several 64-bit matrices of tokens by vocabulary
    if c["op"] == "norm":
        x, w, b = (s[k].detach().double().requires_grad_(True) for k in ("x", "w", "b"))
        var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        y = (x - mean) / torch.sqrt(var + s["eps"]) * w + b
        if not c["train"]:
            return {"y": y.detach()}
        dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"].double())
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    if c["op"] == "route":
        z = s["logits"].detach().double().requires_grad_(True)
        with torch.no_grad():
            ids = _choices(c, z, s["bias"])[2].sort(dim=-1, descending=True, stable=True).indices[:, : c["k"]]
        p = (torch.softmax(z, -1) if c["score"] == "softmax" else torch.sigmoid(z)).gather(1, ids)
        w = (p / (p.sum(-1, keepdim=True) + RENORM_EPS) if c["renorm"] else p) * c["scale"]
        if not c["train"]:
            return {"ids": ids.int(), "w": w.detach()}
        (dl,) = torch.autograd.grad(w, (z,), s["dw"].double())
        return {"ids": ids.int(), "w": w.detach(), "dlogits": dl}
    x, w = (s[k].detach().double().requires_grad_(True) for k in ("x", "w"))
    live = s["y"] != IGNORE
    z = x @ w.t()
    each = (torch.logsumexp(z, 1) - z.gather(1, s["y"].clamp(min=0)[:, None])[:, 0])[live]
    if c["reduction"] == "none":
        loss = torch.zeros(c["T"], dtype=torch.float64, device=z.device).masked_scatter(live, each)
    else:
        loss = each.sum() / (max(1, each.numel()) if c["reduction"] == "mean" else 1)
    if not c["train"]:
        return {"loss": loss.detach()}
    dx, dw = torch.autograd.grad(loss, (x, w), s["dl"].double() if c["reduction"] == "none" else None)
    return {"loss": loss.detach(), "dx": dx, "dw": dw}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    c = case
    T = c["T"]
    if c["op"] == "norm":
        e, ew, H = DTYPES[c["dtype"]].itemsize, DTYPES[c["wdtype"]].itemsize, c["H"]
        if not c["train"]:
            return {"bytes": 2 * T * H * e + 2 * H * ew, "flops": 8 * T * H}
        return {"bytes": 4 * T * H * e + 4 * H * ew, "flops": 20 * T * H}
    if c["op"] == "route":
        e, E, k = DTYPES[c["dtype"]].itemsize, c["E"], c["k"]
        fixed = 4 * E if c["bias"] else 0
        if not c["train"]:
            return {"bytes": T * (E * e + 8 * k) + fixed, "flops": T * 8 * E}
        return {"bytes": T * (2 * E * e + 12 * k) + fixed, "flops": T * 14 * E}
    H, V = c["H"], c["V"]
    out = 4 * T if c["reduction"] == "none" else 4
    if not c["train"]:
        return {"bytes": 2 * (T + V) * H + 8 * T + out, "flops": 2 * T * V * H + 4 * T * V}
    return {"bytes": 4 * (T + V) * H + 8 * T + out * (2 if c["reduction"] == "none" else 1), "flops": 6 * T * V * H + 6 * T * V}
