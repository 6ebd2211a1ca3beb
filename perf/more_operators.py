"""Timed cases of the operators of a model's layers that stay in high precision and keep their activations in 8 bits.

The low-bit recipe leaves layers in bf16 (its norms, a first or last layer's experts, whole models that are trained for
comparison).  What such a layer needs, each one operator here and called through a public entry point of ``lowbit``:

  norm     rms_norm(x, weight, residual=...): the root-mean-square norm with the residual's addition in front of it; trained,
           also the gradients; for generation rms_norm_quant(): the same with its output in e4m3 with a scale for each 128
           columns, as the low-bit products take it
  swiglu   swiglu(x): silu(gate) * up of a product's output that holds both; trained, also the gradient
  grouped  grouped_matmul(x, weight, offsets): rows sorted by expert times their own expert's weight, every number of rows;
           trained, also the gradients of x and weight

Where a case says keep = "e4m3", what the operator keeps of its input for the backward pass is held in 8 bits: 128 columns
of a row share a power of two, and the gradients are those of the values that the 8 bits stand for.

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
EPS = 1e-6
E4M3_MAX = 448.0
MIN_EXP = -126  # of a kept tile's power of two


def listed():
    return [
        # a generation step: the new token's hidden state joins the residual stream, normed for a low-bit 7168-wide product
        dict(name="norm_quant_1", op="norm", mode="quant", T=1, H=7168, dtype="bf16", wdtype="bf16", residual=True, keep=""),
        # a long prompt in front of the same product
        dict(name="norm_quant_8192", op="norm", mode="quant", T=8192, H=7168, dtype="bf16", wdtype="bf16", residual=True,
             keep=""),
        # a training step's pre-norm, 8192 tokens, the residual stream kept in 8 bits
        dict(name="norm_train_8192", op="norm", mode="train", T=8192, H=7168, dtype="bf16", wdtype="bf16", residual=True,
             keep="e4m3"),
        # a small fp32 model whose sizes are no multiples of anything, a norm without a residual
        dict(name="norm_train_odd", op="norm", mode="train", T=1003, H=1541, dtype="f32", wdtype="f32", residual=False,
             keep=""),
        # a generation step: one token in the MLPs of its 8 experts
        dict(name="swiglu_fwd_8", op="swiglu", mode="fwd", T=8, I=2048, block=0, dtype="bf16", keep=""),
        # the expert loop of 4096 tokens with 8 experts each, gate and up in alternating blocks of 128 columns
        dict(name="swiglu_train_32768", op="swiglu", mode="train", T=32768, I=2048, block=128, dtype="bf16", keep="e4m3"),
        # a dense MLP of 18432 columns, 8192 tokens
        dict(name="swiglu_train_8192", op="swiglu", mode="train", T=8192, I=18432, block=0, dtype="bf16", keep="e4m3"),
        # a small fp16 model, odd widths, nothing in 8 bits
        dict(name="swiglu_train_odd", op="swiglu", mode="train", T=5001, I=1003, block=0, dtype="f16", keep=""),
        # a generation step: one token's 8 of 32 experts, their gate and up weights
        dict(name="grouped_fwd_8", op="grouped", mode="fwd", R=8, E=32, busy=8, K=7168, N=4096, unused=0, keep=""),
        # generation with 32 sequences: 256 rows over all 32 experts
        dict(name="grouped_fwd_256", op="grouped", mode="fwd", R=256, E=32, busy=32, K=7168, N=4096, unused=0, keep=""),
        # a small model's training step: odd sizes, experts without rows, rows behind the last one that a capacity left
        dict(name="grouped_train_odd", op="grouped", mode="train", R=1003, E=7, busy=5, K=1000, N=345, unused=50,
             keep="e4m3"),
        # the gate and up projections of 4096 tokens with 8 of 32 experts each, the rows kept in 8 bits
        dict(name="grouped_train_32768", op="grouped", mode="train", R=32768, E=32, busy=32, K=7168, N=4096, unused=0,
             keep="e4m3"),
    ]


def _size(rng, lo: int, hi: int, mult: int = 1) -> int:
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(mult, (v + mult // 2) // mult * mult)


def draw(rng):
    most = work(listed()[-1])
    while True:
        case = _draw(rng)
        w = work(case)
        if w["flops"] <= most["flops"] and w["bytes"] <= most["bytes"]:
            return case


def _draw(rng):
    op = rng.choice(("norm", "swiglu", "grouped"))
    keep = rng.choice(("", "e4m3"))
    mult = rng.choice((1, 8, 128))
    if op == "norm":
        mode = rng.choice(("quant", "train", "train"))
        dt = rng.choice(("bf16", "bf16", "f16", "f32"))
        return dict(op=op, mode=mode, T=_size(rng, 1, 32768), H=_size(rng, 64, 8192, mult), dtype=dt,
                    wdtype=rng.choice((dt, "f32")), residual=rng.random() < 0.6, keep=keep if mode == "train" else "")
    if op == "swiglu":
        mode = rng.choice(("fwd", "train", "train"))
        I = _size(rng, 64, 18432, mult)
        return dict(op=op, mode=mode, T=_size(rng, 1, 32768), I=I, block=128 if I % 128 == 0 and rng.random() < 0.5 else 0,
                    dtype=rng.choice(("bf16", "bf16", "f16", "f32")), keep=keep if mode == "train" else "")
    mode = rng.choice(("fwd", "train", "train"))
    R, E = _size(rng, 1, 32768), _size(rng, 1, 64)
    unused = rng.choice((0, 0, R // 20))
    busy = min(rng.choice((E, rng.randint((E + 1) // 2, E))), R - unused)
    return dict(op=op, mode=mode, R=R, E=E, busy=busy, K=_size(rng, 64, 7168, mult), N=_size(rng, 64, 4096, mult),
                unused=unused, keep=keep if mode == "train" else "")


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    return {"norm": _norm_inputs, "swiglu": _swiglu_inputs, "grouped": _grouped_inputs}[case["op"]](dict(case), g)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _norm_inputs(c, g):
    dt, wdt = DTYPES[c["dtype"]], DTYPES[c["wdtype"]]
    T, H = c["T"], c["H"]
    # a residual stream: channels of unequal size
    x = _randn(g, T, H) * torch.exp(0.7 * _randn(g, H))
    s = dict(case=c, x=x.to(dt), w=(1.0 + 0.2 * _randn(g, H)).to(wdt), res=None)
    if c["residual"]:  # what the layer before added is the smaller of the two
        s["res"], s["x"] = s["x"], (0.3 * _randn(g, T, H)).to(dt)
    if c["mode"] == "train":
        s["dy"] = _randn(g, T, H).to(dt)
        s["ds"] = _randn(g, T, H).to(dt) if c["residual"] else None
        for k in ("x", "res", "w"):
            if s[k] is not None:
                s[k].requires_grad_(True)
    return s


def _swiglu_inputs(c, g):
    dt = DTYPES[c["dtype"]]
    T, I = c["T"], c["I"]
    x = (_randn(g, T, 2 * I) * torch.exp(0.5 * _randn(g, 2 * I))).to(dt)
    s = dict(case=c, x=x)
    if c["mode"] == "train":
        s["dh"] = _randn(g, T, I).to(dt)
        x.requires_grad_(True)
    return s


def _grouped_inputs(c, g):
    R, E, K, N, busy = c["R"], c["E"], c["K"], c["N"], c["busy"]
    used = R - c["unused"]
    # `busy` of the experts have rows, popular ones more (their rank to the power of -0.8)
    who = torch.randperm(E, generator=g, device=DEV)[:busy]
    p = torch.arange(1, busy + 1, device=DEV, dtype=torch.float64) ** -0.8
    more = torch.rand(used - busy, generator=g, device=DEV, dtype=torch.float64) * p.sum()
    ids = torch.searchsorted(p.cumsum(0), more).clamp(max=busy - 1)
    counts = torch.zeros(E, dtype=torch.int64, device=DEV)
    counts[who] = 1 + torch.bincount(ids, minlength=busy)
    offsets = torch.zeros(E + 1, dtype=torch.int32, device=DEV)
    offsets[1:] = counts.cumsum(0)
    w = torch.empty(E, N, K, dtype=torch.bfloat16, device=DEV)
    for e in range(E):
        w[e] = 0.02 * _randn(g, N, K)
    s = dict(case=c, x=(_randn(g, R, K) * torch.exp(0.5 * _randn(g, K))).to(torch.bfloat16), w=w, offsets=offsets,
             most=int(counts.max()))  # rows of the largest expert: the plain form pads every expert to it
    if c["mode"] == "train":
        s["dy"] = (0.1 * _randn(g, R, N)).to(torch.bfloat16)
        s["x"].requires_grad_(True)
        s["w"].requires_grad_(True)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _norm_own, "swiglu": _swiglu_own, "grouped": _grouped_own}[op](state)
    with torch.no_grad():
        return {"norm": _norm_plain, "swiglu": _swiglu_plain, "grouped": _grouped_plain}[op](state)


def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nano-train_amd")
    if at not in sys.path:
        sys.path.insert(0, at)


def _norm_own(s):
    _package()
    from lowbit.norm import rms_norm, rms_norm_quant

    c, H = s["case"], s["case"]["H"]
    if c["mode"] == "quant":
        q = rms_norm_quant(s["x"], s["w"], residual=s["res"], eps=EPS, fmt="e4m3")
        q, total = q if c["residual"] else (q, None)
        out = {"y": q.codes[:, :H].view(torch.float8_e4m3fn), "scales": q.scales[:, : c["T"]]}
        return {**out, "s": total} if c["residual"] else out
    y = rms_norm(s["x"], s["w"], residual=s["res"], eps=EPS, checkpoint=c["keep"] or None)
    if not c["residual"]:
        dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    y, total = y
    dx, dres, dw = torch.autograd.grad((y, total), (s["x"], s["res"], s["w"]), (s["dy"], s["ds"]))
    return {"y": y.detach(), "s": total.detach(), "dx": dx, "dres": dres, "dw": dw}


def _swiglu_own(s):
    _package()
    from lowbit.experts import swiglu

    c = s["case"]
    h = swiglu(s["x"], block=c["block"], checkpoint=c["keep"] or None)
    if c["mode"] == "fwd":
        return {"h": h}
    (dx,) = torch.autograd.grad(h, (s["x"],), s["dh"])
    return {"h": h.detach(), "dx": dx}


def _grouped_own(s):
    _package()
    from lowbit.experts import grouped_matmul

    c = s["case"]
    y = grouped_matmul(s["x"], s["w"], s["offsets"], checkpoint=c["keep"] or None)
    if c["mode"] == "fwd":
        return {"y": y}
    dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw}


def _tiles(x):
    """x [T, H] as [T, tiles, 128], zeros behind the last column."""
    T, H = x.shape
    n = (H + 127) // 128
    p = torch.zeros(T, n * 128, dtype=x.dtype, device=x.device)
    p[:, :H] = x
    return p.reshape(T, n, 128)


def _kept(x):
    """What 8 bits keep of the fp32 values x [T, H]: for each 128 columns the smallest power of two that brings their
    largest magnitude to 448 or less, the values over it as e4m3."""
    t = _tiles(x)
    m, e = torch.frexp(t.abs().amax(2, keepdim=True))  # m in [0.5, 1); 448 is 0.875 * 2^9
    k = torch.where(m > 0.875, e - 8, e - 9).clamp(min=MIN_EXP)
    q = (t * _power(-k)).to(torch.float8_e4m3fn).float()
    return (q * _power(k)).reshape(x.shape[0], -1)[:, : x.shape[1]]


def _power(k):
    """2^k in 32 bits, -127 < k < 128."""
    return ((k + 127) << 23).view(torch.float32)


def _norm_plain(s):
    c, dt = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    total = (x + s["res"].float()).to(dt) if c["residual"] else None
    t = total.float() if c["residual"] else x
    r = torch.rsqrt((t * t).mean(1, keepdim=True) + EPS)
    y = t * r * w
    if c["mode"] == "quant":
        tiles = _tiles(y)
        scale = tiles.abs().amax(2) / E4M3_MAX
        scale = torch.where(scale > 0, scale, 1.0)
        q = (tiles / scale[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        out = {"y": q.reshape(c["T"], -1)[:, : c["H"]], "scales": scale.t()}
        return {**out, "s": total} if c["residual"] else out
    dy = s["dy"].float()
    xh = (_kept(t) if c["keep"] else t) * r
    u = dy * w
    dx = r * (u - xh * (u * xh).mean(1, keepdim=True))
    dw = (dy * xh).sum(0).to(s["w"].dtype)
    if not c["residual"]:
        return {"y": y.to(dt), "dx": dx.to(dt), "dw": dw}
    dx = (dx + s["ds"].float()).to(dt)
    return {"y": y.to(dt), "s": total, "dx": dx, "dres": dx, "dw": dw}


def _halves(x, block):
    """gate and up of x [T, 2 I]: its halves, or alternating blocks of columns."""
    T, I = x.shape[0], x.shape[1] // 2
    b = block or I
    v = x.reshape(T, I // b, 2, b)
    return v[:, :, 0].reshape(T, I), v[:, :, 1].reshape(T, I)


def _swiglu_plain(s):
    c, dt = s["case"], s["x"].dtype
    T, I, b = c["T"], c["I"], c["block"] or c["I"]
    gate, up = _halves(s["x"].float(), c["block"])
    h = (gate / (1.0 + torch.exp(-gate)) * up).to(dt)
    if c["mode"] == "fwd":
        return {"h": h}
    dh = s["dh"].float()
    if c["keep"]:
        gate, up = _kept(gate), _kept(up)
    sig = 1.0 / (1.0 + torch.exp(-gate))
    dx = torch.empty(T, I // b, 2, b, device=dh.device)
    dx[:, :, 0] = (dh * up * sig * (1.0 + gate * (1.0 - sig))).reshape(T, I // b, b)
    dx[:, :, 1] = (dh * gate * sig).reshape(T, I // b, b)
    return {"h": h, "dx": dx.reshape(T, 2 * I).to(dt)}


def _grouped_plain(s):
    c = s["case"]
    R, E = c["R"], c["E"]
    # every expert's rows, padded with zeros to those of the largest one
    row = torch.arange(R, device=s["x"].device, dtype=torch.int32)
    e = torch.searchsorted(s["offsets"][1:].contiguous(), row, right=True)
    live = e < E
    at = torch.where(live, e * s["most"] + row - s["offsets"][e.clamp(max=E - 1)], 0)

    def pad(t):
        p = torch.zeros(E * s["most"], t.shape[1], device=t.device)
        return p.index_add_(0, at, torch.where(live[:, None], t, 0.0)).reshape(E, s["most"], -1)

    def rows(p):
        return torch.where(live[:, None], p.reshape(E * s["most"], -1)[at], 0.0).to(torch.bfloat16)

    x, w = s["x"].float(), s["w"].float()
    y = rows(torch.bmm(pad(x), w.transpose(1, 2).contiguous()))
    if c["mode"] == "fwd":
        return {"y": y}
    dy = pad(s["dy"].float())
    dx = rows(torch.bmm(dy, w))
    dw = torch.bmm(dy.transpose(1, 2).contiguous(), pad(_kept(x) if c["keep"] else x)).to(torch.bfloat16)
    return {"y": y, "dx": dx, "dw": dw}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _norm_exact, "swiglu": _swiglu_exact, "grouped": _grouped_exact}[case["op"]](s)


def _round_e4m3(v):
    """v to the nearest e4m3 value, ties to the even one: three bits behind the leading one, down to steps of 2^-9."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3.0)
    return torch.round(v / step) * step


def _columns(x, f):
    """f(128 columns) of x, the last ones as many as there are."""
    return torch.cat([f(part) for part in x.split(128, dim=1)], dim=1)


def _double_power(k):
    return ((k + 1023) << 52).view(torch.float64)


def _stands_for(x):
    def tile(v):
        top = v.abs().amax(1, keepdim=True)
        k = torch.ceil(torch.log2(top / E4M3_MAX))  # near a power of two the logarithm may say one more or less
        k = k.clamp(min=MIN_EXP).long()
        k = torch.where(top <= E4M3_MAX * _double_power(k - 1), k - 1, k)
        k = torch.where(top > E4M3_MAX * _double_power(k), k + 1, k).clamp(min=MIN_EXP)
        return _round_e4m3(v * _double_power(-k)) * _double_power(k)

    return _columns(x, tile)


def _norm_exact(s):
    c = s["case"]
    x, w = s["x"].detach().double(), s["w"].detach().double()
    if c["residual"]:
        x = (x + s["res"].detach().double()).to(s["x"].dtype).double()
    rms = torch.sqrt(x.square().mean(1, keepdim=True) + EPS)
    y = x / rms * w
    more = {"s": x} if c["residual"] else {}
    if c["mode"] == "quant":
        top = torch.stack([part.abs().amax(1) for part in y.split(128, dim=1)])
        return {"y": _columns(y, lambda v: _round_e4m3(v / v.abs().amax(1, keepdim=True) * E4M3_MAX)),
                "scales": top / E4M3_MAX, **more}
    xh = (_stands_for(x) if c["keep"] else x) / rms
    dy = s["dy"].double()
    dx = (dy * w - xh * (dy * w * xh).mean(1, keepdim=True)) / rms
    dw = (dy * xh).sum(0)
    if c["residual"]:
        dx = dx + s["ds"].double()
        more["dres"] = dx
    return {"y": y, "dx": dx, "dw": dw, **more}


def _swiglu_exact(s):
    c = s["case"]
    T, I = c["T"], c["I"]
    b = c["block"] or I
    col = torch.arange(I, device=DEV)
    at = col // b * 2 * b + col % b  # h's columns' places of gate in x; up's are b on
    x = s["x"].detach().double()
    h = torch.nn.functional.silu(x[:, at]) * x[:, at + b]
    if c["mode"] == "fwd":
        return {"h": h}
    gate, up = x[:, at], x[:, at + b]
    if c["keep"]:
        gate, up = _stands_for(gate), _stands_for(up)
    gate.requires_grad_(True)
    up.requires_grad_(True)
    dg, du = torch.autograd.grad(torch.nn.functional.silu(gate) * up, (gate, up), s["dh"].double())
    dx = torch.empty_like(x)
    dx[:, at], dx[:, at + b] = dg, du
    return {"h": h, "dx": dx}


def _grouped_exact(s):
    c = s["case"]
    x, w = s["x"].detach(), s["w"].detach()
    ends = s["offsets"].tolist()
    y = torch.zeros(c["R"], c["N"], dtype=torch.float64, device=DEV)
    train = c["mode"] == "train"
    if train:
        dx = torch.zeros(c["R"], c["K"], dtype=torch.float64, device=DEV)
        dw = torch.zeros(c["E"], c["N"], c["K"], dtype=torch.float64, device=DEV)
    for e in range(c["E"]):
        part = slice(ends[e], ends[e + 1])
        if ends[e] == ends[e + 1]:
            continue
        xe, we = x[part].double(), w[e].double()
        y[part] = torch.mm(xe, we.t())
        if train:
            dye = s["dy"][part].double()
            dx[part] = torch.mm(dye, we)
            dw[e] = torch.mm(dye.t(), _stands_for(xe) if c["keep"] else xe)
    return {"y": y, "dx": dx, "dw": dw} if train else {"y": y}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "norm":
        T, H, e, ew = c["T"], c["H"], DTYPES[c["dtype"]].itemsize, DTYPES[c["wdtype"]].itemsize
        if c["mode"] == "quant":
            return {"bytes": T * H * ((3 if c["residual"] else 1) * e + 1) + 4 * T * ((H + 127) // 128) + H * ew,
                    "flops": 8 * T * H}
        # the residual's gradient is x's
        return {"bytes": (7 if c["residual"] else 4) * T * H * e + 2 * H * ew, "flops": 18 * T * H}
    if c["op"] == "swiglu":
        n, e = c["T"] * c["I"], DTYPES[c["dtype"]].itemsize
        return {"bytes": 6 * n * e, "flops": 24 * n} if c["mode"] == "train" else {"bytes": 3 * n * e, "flops": 8 * n}
    used, K, N = c["R"] - c["unused"], c["K"], c["N"]
    if c["mode"] == "fwd":
        return {"bytes": 2 * (used * K + c["busy"] * N * K + c["R"] * N) + 4 * c["E"], "flops": 2 * used * N * K}
    return {"bytes": 4 * (c["R"] * (K + N)) + 2 * (c["busy"] + c["E"]) * N * K + 4 * c["E"], "flops": 6 * used * N * K}
