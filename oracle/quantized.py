"""8-bit rows restated in 64 bits on the CPU: e4m3 codes, one power of two per page and head.

Written from the format: 4 bits of exponent (bias 7), 3 of mantissa, no
infinities; a page's scale is the least 2^e that keeps its finite elements
within 448 * 2^e, e from -126 to 119 (448 * 2^119 is finite in fp32; 7 for rows
of half precision).
"""

from __future__ import annotations

import math

import torch


def decode(codes: torch.Tensor) -> torch.Tensor:
    """Values of e4m3 ``codes`` (uint8)."""
    c = codes.long()
    exponent, mantissa = (c >> 3) & 15, c & 7
    size = torch.where(exponent == 0, mantissa.double() * 2.0 ** -9, (8 + mantissa).double() * 2.0 ** (exponent.double() - 10))
    size = torch.where((c & 127) == 127, torch.nan, size)
    return torch.where(c >= 128, -size, size)


def values(codes: torch.Tensor, exponents: torch.Tensor, page: int) -> torch.Tensor:
    """Values of ``codes`` [..., rows, heads, dim] with ``exponents`` [..., pages, heads] of pages of ``page`` rows."""
    rows = torch.arange(codes.shape[-3]) // page
    return decode(codes) * 2.0 ** exponents.double()[..., rows, :][..., None]


def step(x: torch.Tensor) -> torch.Tensor:
    """The distance of neighbouring codes' values where ``x`` lies."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))).clamp(max=8)
    return 2.0 ** (e - 3)


def round_code(x: torch.Tensor) -> torch.Tensor:
    """``x`` (64 bits) rounded to the nearest e4m3 value, ties to even, at most 448."""
    s = step(x)
    return (torch.round(x / s) * s).clamp(-448, 448)


def exponent(top: float, most: int = 119) -> int:
    """e of the scale for finite elements up to ``top``."""
    if top == 0:
        return -126
    m, k = math.frexp(top)  # m in [0.5, 1), 448 = 0.875 * 2^9
    return max(-126, min(most, k - 9 + (m > 0.875)))


def store(x: torch.Tensor, most: int = 119, had: int = -126):
    """``(values / scale, e)`` of rows ``x`` [rows, dim] that go into a page whose cached rows have exponent ``had``."""
    finite = x[torch.isfinite(x)]
    e = max(had, exponent(float(finite.abs().max()) if finite.numel() else 0.0, most))
    y = torch.where(torch.isfinite(x), x, torch.nan)
    return y * 2.0 ** -e, e
