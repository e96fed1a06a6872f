"""64-bit statements of the 8-bit operators, written from their definition block by block."""
import math

import torch

TOP = {"e4m3": 8, "e5m2": 15}
GRID = {"e4m3": (3, -6), "e5m2": (2, -14)}      # fraction bits, smallest normal exponent


def exponent(amax: float, fmt: str) -> int:
    """Smallest e in [-127, 127] with amax <= 1.75 * 2^(top + e)."""
    if amax == 0:
        return -127
    frac, ex = math.frexp(amax)
    e = ex - 1 - TOP[fmt] + (1 if frac > 0.875 else 0)
    return max(-127, min(127, e))


def round_code(y: torch.Tensor, fmt: str) -> torch.Tensor:
    bits, low = GRID[fmt]
    _, ex = torch.frexp(y.abs())
    step = torch.ldexp(torch.ones_like(y), (ex - 1).clamp(min=low) - bits)
    return torch.round(y / step) * step


def quantize(x: torch.Tensor, fmt: str, tiles: bool):
    """[rows, cols] -> (codes in 64 bits [rows, cols], exponents [rows, blocks])."""
    x = x.double()
    rows, cols = x.shape
    code = torch.empty_like(x)
    exps = torch.full((rows, -(-cols // 128)), -127, dtype=torch.int32)
    for j in range(exps.shape[1]):
        c = slice(128 * j, min(128 * (j + 1), cols))
        r = 0
        while r < rows:
            rr = slice(r, min(r + 128, rows) if tiles else r + 1)
            part = x[rr, c]
            fin = part[torch.isfinite(part)].abs()
            e = exponent(float(fin.max()) if fin.numel() else 0.0, fmt)
            y = part * 2.0 ** -e
            q = round_code(torch.where(torch.isfinite(y), y, torch.zeros_like(y)), fmt)
            bad = torch.full_like(y, math.nan) if fmt == "e4m3" else y
            code[rr, c] = torch.where(torch.isfinite(y), q, bad)
            exps[rr, j] = e
            r = rr.stop
    return code, exps


def values(q) -> torch.Tensor:
    """The values of a BlockFp8 in 64 bits, on its device."""
    out = q.data[:, :q.cols].double()
    for j in range(-(-q.cols // 128)):
        out[:, 128 * j:128 * (j + 1)] *= q.scale[j // 4, :, j % 4].double()[:, None]
    return out


def check_product(out: torch.Tensor, a: torch.Tensor, b: torch.Tensor, base=None, rounds: int = 1):
    """out against a @ b^T (+ base) in 64 bits.

    Sums: K products (exact in fp32: 4-bit by 4-bit fractions) are added in fp32, each addition off by at most
    2^-23 of the magnitudes summed (truncating adders included), so (K + 2) 2^-23 sum |a b|; then half a step of the
    output type, relative to the result, for each rounding to it."""
    exact = a @ b.t()
    mag = a.abs() @ b.abs().t()
    if base is not None:
        exact, mag = exact + base.double(), mag + base.double().abs()
    half = torch.finfo(out.dtype).eps / 2
    tol = (a.shape[1] + 2) * 2.0 ** -23 * mag
    tol = tol * (1 + half) + rounds * half * exact.abs() + torch.finfo(out.dtype).tiny
    bad = (out.double() - exact).abs() > tol
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((out.double() - exact).abs() - tol).max()):.3g}"
