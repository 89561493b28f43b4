"""Queries on a paged cache restated in 64 bits on the CPU, one request and head at a time.

Written from the definitions: new token ``i`` of a request with ``length``
cached tokens, ``new`` of them new, is cached token ``p = length - new + i``.
"""

from __future__ import annotations

import math

import torch


def visible(length: int, new: int, *, causal=True, window=0, prefix=0) -> torch.Tensor:
    """``[new, length]`` truth values: which cached tokens each new one sees."""
    p = torch.arange(length - new, length)[:, None]
    j = torch.arange(length)[None, :]
    seen = torch.ones(new, length, dtype=torch.bool)
    if causal:
        seen &= j <= p
    if window:
        seen &= j > p - window
    return seen | (j < prefix)


def scores(q, k, *, scale, cap=0.0, slope=0.0):
    """``[new, length]`` scores of one head from ``q`` [new, D] and ``k`` [length, D]."""
    q, k = q.double(), k.double()
    x = scale * (q @ k.T)
    if cap:
        x = cap * torch.tanh(x / cap)
    new, length = x.shape
    away = (torch.arange(length - new, length)[:, None] - torch.arange(length)[None, :]).abs()
    return x - slope * away


def attention(q, k, v, *, scale, cap=0.0, slope=0.0, **mask):
    """``(out, lse, magnitude)`` of one head: magnitude is the same average over ``|v|``."""
    seen = visible(k.shape[0], q.shape[0], **mask)
    x = scores(q, k, scale=scale, cap=cap, slope=slope)
    out = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(out)
    lse = torch.full((q.shape[0],), -math.inf, dtype=torch.float64)
    for i in range(q.shape[0]):
        at = seen[i].nonzero()[:, 0]
        if at.numel() == 0:
            continue
        lse[i] = torch.logsumexp(x[i, at], 0)
        w = (x[i, at] - lse[i]).exp()
        out[i] = w @ v[at].double()
        mag[i] = w @ v[at].double().abs()
    return out, lse, mag


def key_weights(q, k, lse, *, scale, cap=0.0, slope=0.0, **mask):
    """``[length]`` sums over the new tokens of ``exp(score - lse)`` of one head."""
    seen = visible(k.shape[0], q.shape[0], **mask)
    w = (scores(q, k, scale=scale, cap=cap, slope=slope) - lse.double()[:, None]).exp()
    return torch.where(seen & (lse > -math.inf)[:, None], w, 0.0).sum(0)


def score_error(q, k, *, scale):
    """Bound of a score's error when its products are summed in 32 bits, in any order."""
    d = q.shape[1]
    size = (abs(scale) * (q.double().abs() @ k.double().abs().T)).max() if q.numel() and k.numel() else torch.tensor(0.0)
    return float(size) * (d + 4) * 2.0 ** -24


def rotate(x, positions, inv_freq, *, magnitude=1.0, interleaved=False):
    """``x`` [tokens, heads, D] turned by ``positions * inv_freq`` over its first ``2 len(inv_freq)`` elements."""
    x = x.double()
    half = inv_freq.numel()
    angle = positions.double()[:, None, None] * inv_freq.double()
    c, s = angle.cos() * magnitude, angle.sin() * magnitude
    y = x.clone()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def keep(weights, budget: int, first: int = 0, last: int = 0) -> list[int]:
    """Places kept of one request's ``weights`` (a list of floats), in order."""
    n = len(weights)
    if n <= budget:
        return list(range(n))
    middle = sorted(range(first, n - last), key=lambda j: (not math.isnan(weights[j]),
                                                            0.0 if math.isnan(weights[j]) else -weights[j], j))
    return sorted([*range(first), *middle[:budget - first - last], *range(n - last, n)])
