"""Random query batches over a paged pool, and what the oracle says of them (test helper)."""

from __future__ import annotations

from dataclasses import dataclass, field

import torch

from cachebridge_amd.online.queries import QueryBatch
from cachebridge_amd.plan import rows_from_stacked
from oracle import queries as oracle


@dataclass
class Case:
    lengths: list
    new: list
    heads: int
    kv_heads: int
    dim: int
    dtype: torch.dtype
    page: int
    q: torch.Tensor                 # CPU [tokens, heads, dim]
    k: torch.Tensor                 # CPU [layers, rows, kv_heads, dim]
    v: torch.Tensor
    slots: list                     # CPU int64 rows of each request's cached tokens
    batch: QueryBatch
    pool: tuple = field(default=())  # device k, v

    def spans(self):
        at = 0
        for b, (length, new) in enumerate(zip(self.lengths, self.new)):
            yield b, length, new, at
            at += new

    @property
    def tokens(self):
        return sum(self.new)


def make(lengths, new, *, heads=4, kv_heads=2, dim=64, dtype=torch.bfloat16, page=16, layers=1, seed=0, index="table",
         padding=0, spread=1.0, start=0, max_query=None, max_length=None, bounds=True):
    """A batch on the GPU. ``index``: "table" (flat [requests, width] block table), "offsets" (pages back to back,
    explicit offsets), "i32" / "i64" (slots with offsets) or "identity". ``padding`` rows of no request follow in q.
    ``start`` index tokens come before the first request's (offsets only)."""
    g = torch.Generator().manual_seed(seed)
    pages = [-(-n // page) for n in lengths]
    total = sum(pages) + 3
    n = sum(new) + padding
    rows = total * page + (start if index == "identity" else 0)
    q = (torch.randn(n, heads, dim, generator=g) * spread).to(dtype)
    k = torch.randn(layers, rows, kv_heads, dim, generator=g).to(dtype)
    v = torch.randn(layers, rows, kv_heads, dim, generator=g).to(dtype)
    order = torch.randperm(total, generator=g)
    kd, vd = k.cuda(), v.cuda()
    slots, at = [], 0
    qs = torch.tensor([0] + new).cumsum(0).to(torch.int32).cuda()
    ln = torch.tensor(lengths, dtype=torch.int32).cuda()
    more = {}
    if index in ("table", "offsets"):
        width = max(pages, default=0) + 1
        table = torch.full((len(lengths), width), -1, dtype=torch.int32)
        flat, offsets = [], []
        for b, (m, length) in enumerate(zip(pages, lengths)):
            mine = order[at:at + m]
            table[b, :m] = mine.int()
            # Back to back, a request may start inside its first page.
            inside = (5 * b) % page if index == "offsets" and length and length % page and length % page + (5 * b) % page <= page else 0
            offsets.append((start // page + at) * page + inside)
            flat.append(mine.int())
            t = torch.arange(length) + inside
            slots.append(mine[t // page] * page + t % page)
            at += m
        if index == "table":
            rows_d = rows_from_stacked(kd, vd, block_table=table.view(-1).cuda(), page_size=page)
            more["request_stride"] = width * page
        else:
            lead = torch.full((start // page,), -1, dtype=torch.int32)
            rows_d = rows_from_stacked(kd, vd, block_table=torch.cat([lead, *flat]).cuda(), page_size=page)
            more["offsets"] = torch.tensor(offsets, dtype=torch.int64).cuda()
    else:
        perm = torch.randperm(rows, generator=g)
        offsets, flat = [], [torch.full((start,), -1, dtype=torch.int64)]
        for length in lengths:
            mine = torch.arange(at, at + length) if index == "identity" else perm[at:at + length]
            offsets.append(start + at)
            slots.append(mine + (start if index == "identity" else 0))
            flat.append(mine)
            at += length
        more["offsets"] = torch.tensor(offsets, dtype=torch.int64).cuda()
        if index == "identity":
            rows_d = rows_from_stacked(kd, vd)
        else:
            kind = torch.int32 if index == "i32" else torch.int64
            rows_d = rows_from_stacked(kd, vd, index=torch.cat(flat).to(kind).cuda())
    if bounds:
        max_query = max(new, default=0) if max_query is None else max_query
    batch = QueryBatch(rows_d, qs, ln, max_query=max_query,
                       max_length=max(lengths, default=0) if max_length is None else max_length, **more)
    return Case(list(lengths), list(new), heads, kv_heads, dim, dtype, page, q, k, v, slots, batch, (kd, vd))


def check_attention(case: Case, out, lse=None, *, layer=0, scale=None, cap=0.0, slopes=None, prefix=None, **mask):
    """Compare with the oracle. Bounds, per element: the result's own rounding (u |o|), the weights' rounding before
    their product with V (u sum w |v|; in half precision also 2^-25 |v| a key, half a step below its normal range, for
    weights whose row sums to 1 or more), a weight's error from its score's (2 d each, in it and in the sum) and the
    fp32 sums' and exponentials' (n + 16 roundings)."""
    scale = case.dim ** -0.5 if scale is None else scale
    u = torch.finfo(case.dtype).eps / 2
    group = case.heads // case.kv_heads
    out = out.double().cpu()
    for b, length, new, at in case.spans():
        for h in range(case.heads):
            q = case.q[at:at + new, h]
            k, v = (x[layer, case.slots[b], h // group] for x in (case.k, case.v))
            how = dict(scale=scale, cap=cap, slope=0.0 if slopes is None else float(slopes[h]),
                       prefix=0 if prefix is None else int(prefix[b]), **mask)
            want, want_lse, mag = oracle.attention(q, k, v, **how)
            d = oracle.score_error(q, k, scale=scale) + 2.0 ** -21 * (cap + abs(how["slope"]) * length)
            small = 2.0 ** -25 * length * float(v.double().abs().max()) if case.dtype == torch.float16 and length else 0.0
            tol = u * want.abs() + u * mag + mag * (4 * d + (length + 16) * 2.0 ** -23) + small + 1e-30
            got = out[at:at + new, h]
            worst = ((got - want).abs() - tol).max() if new else torch.tensor(-1.0)
            assert worst <= 0, (b, h, float(worst), float((got - want).abs().max()))
            if lse is not None:
                z = lse[at:at + new, h].double().cpu()
                fin = torch.isfinite(want_lse)
                assert torch.equal(z[~fin], want_lse[~fin])
                gap = (z - want_lse)[fin].abs() - (d + (length + 16) * 2.0 ** -23 + 2.0 ** -22 * want_lse[fin].abs())
                assert gap.numel() == 0 or gap.max() <= 0, (b, h, float(gap.max()))


def check_weights(case: Case, before, after, lse, *, layer=0, scale=None, cap=0.0, slopes=None, prefix=None, **mask):
    """A weight's terms are off by their scores' errors and those of the difference and exponential (2^-21 of the
    score's size), its fp32 sum by one rounding a term."""
    scale = case.dim ** -0.5 if scale is None else scale
    group = case.heads // case.kv_heads
    want = before.double().cpu().clone()
    tol = torch.zeros_like(want)
    for b, length, new, at in case.spans():
        for h in range(case.heads):
            q, k = case.q[at:at + new, h], case.k[layer, case.slots[b], h // group]
            how = dict(scale=scale, cap=cap, slope=0.0 if slopes is None else float(slopes[h]),
                       prefix=0 if prefix is None else int(prefix[b]), **mask)
            z = lse[at:at + new, h].double().cpu()
            got = oracle.key_weights(q, k, z, **how)
            d = oracle.score_error(q, k, scale=scale) + 2.0 ** -21 * (cap + abs(how["slope"]) * length + 30)
            want[b, :length] += got
            tol[b, :length] += got * 2 * d
    tol += want.abs() * (sum(case.new) * case.heads + 16) * 2.0 ** -24 + 1e-30
    gap = ((after.double().cpu() - want).abs() - tol).max()
    assert gap <= 0, float(gap)
