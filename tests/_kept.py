"""The 8 bits that operators keep of their inputs, in 64 bits and by the definition: 128 columns of a row share the
smallest power of two 2^k, k >= -126, with |x| <= 448 2^k; x 2^-k is rounded to e4m3, ties to the even value."""

from __future__ import annotations

import torch

_GRID = None


def power(k: torch.Tensor) -> torch.Tensor:
    """2^k in 64 bits by its exponent's bits (the device's pow is off by a unit for some k)"""
    return ((k.long() + 1023) << 52).view(torch.float64)


def values(codes: torch.Tensor, exps: torch.Tensor) -> torch.Tensor:
    """what kept codes [rows, tiles * 128] and their tiles' bytes stand for, in 64 bits"""
    return codes.view(torch.float8_e4m3fn).double() * power(exps.long() - 127).repeat_interleave(128, 1)


def _e4m3_grid():
    global _GRID
    if _GRID is None:
        vals = [m * 2.0 ** -9 for m in range(8)]
        vals += [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1]  # the last one is NaN
        _GRID = torch.tensor(vals, dtype=torch.float64)
    return _GRID


def round_e4m3(v: torch.Tensor) -> torch.Tensor:
    """the nearest of the 127 values of each sign (by search), a tie to the one of even index"""
    grid = _e4m3_grid().to(v.device)
    a = v.abs()
    hi = torch.searchsorted(grid, a).clamp(max=grid.numel() - 1)
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - a, a - grid[lo]
    take_hi = (up < down) | ((up == down) & (hi % 2 == 0))
    return torch.where(take_hi, grid[hi], grid[lo]) * torch.sign(v)


def kept(x: torch.Tensor) -> torch.Tensor:
    """what 8 bits keep of x [..., n], in 64 bits (NaN for what is not finite)"""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for c in range(0, x.shape[-1], 128):
        v = x[..., c:c + 128].double()
        ok = v.isfinite()
        f = torch.where(ok, v, 0.0)
        top = f.abs().amax(-1, keepdim=True)
        k = torch.full_like(top, -126.0)
        for j in range(120, -127, -1):  # the smallest power that will do
            k = torch.where(top <= 448.0 * 2.0 ** j, float(j), k)
        p = power(k)
        out[..., c:c + 128] = torch.where(ok, round_e4m3(f / p) * p, float("nan"))
    return out
