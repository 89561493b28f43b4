"""Random query batches over an 8-bit paged pool (test helper)."""

from __future__ import annotations

import torch

from cachebridge_amd.online.queries import QueryBatch
from cachebridge_amd.plan import BlockScales, rows_from_stacked
from oracle import quantized as oracle

from . import query_cases

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def codes_of(x: torch.Tensor) -> torch.Tensor:
    return x.view(torch.uint8)


def device_scales(exponents: torch.Tensor) -> torch.Tensor:
    return (exponents + 127).to(torch.uint8).cuda().view(E8M0)


def make(lengths, new, *, page=16, scale_page=None, dtype=torch.bfloat16, index="table", seed=0, **kw) -> query_cases.Case:
    """``query_cases.make`` with its pool in 8 bits: values of about one, scales of 2^-8 to 2^-5 that differ from page to
    page and head to head. ``case.k`` and ``case.v`` are the cached values in 64 bits, ``case.pool`` the device's codes,
    ``case.scales`` its scales, ``case.exponents`` their exponents."""
    case = query_cases.make(lengths, new, page=page, dtype=dtype, index=index, seed=seed, **kw)
    scale_page = page if scale_page is None else scale_page
    g = torch.Generator().manual_seed(seed + 1000)
    layers, rows, heads = case.k.shape[:3]
    pages = -(-rows // scale_page)
    pool, scales, exponents, values = [], [], [], []
    for x in (case.k, case.v):
        e = torch.randint(-8, -4, (layers, pages, heads), generator=g)
        spread = 2.0 ** -e.double()[:, torch.arange(rows) // scale_page][..., None] * 0.5
        codes = (x.double() * spread).clamp(-448, 448).float().to(E4M3).view(torch.uint8)
        pool.append(codes.cuda().view(E4M3))
        scales.append(device_scales(e))
        exponents.append(e)
        values.append(oracle.values(codes, e, scale_page))
    old = case.batch
    table = {} if index == "identity" else \
        dict(block_table=old.rows.keep[-1], page_size=page) if index in ("table", "offsets") else dict(index=old.rows.keep[-1])
    described = rows_from_stacked(*pool, **table, scales=BlockScales(*scales, scale_page, dtype))
    case.batch = QueryBatch(described, *old._keep[:2], offsets=old._keep[2], request_stride=old.c.request_stride,
                            max_query=old.max_query, max_length=old.max_length)
    case.k, case.v = values
    case.pool, case.scales, case.exponents, case.scale_page = tuple(pool), tuple(scales), tuple(exponents), scale_page
    return case
