"""GPU: attention on 16-bit pools whose weights keep fp32."""

from __future__ import annotations

import pytest
import torch

from cachebridge_amd.online.queries import paged_attention
from oracle import queries as oracle

from .query_cases import make

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 128), (BF16, 256), (FP16, 64), (FP16, 128), (FP16, 256), (BF16, 512)])
@pytest.mark.parametrize("new", [[1, 1, 1], [90, 7, 33], [0, 290, 1]])
@pytest.mark.parametrize("how", [{}, dict(window=20, prefix=[4, 300, 33]), dict(cap=4.0, slopes=True, causal=False)])
def test_fp32_weights(how, new, dtype, dim):
    """The bounds of query_cases.check_attention without its terms for the weights' rounding."""
    case = make([190, 301, 33], new, heads=4, kv_heads=2, dim=dim, dtype=dtype, seed=3)
    how, dev = dict(how), {}
    prefix, slopes = how.pop("prefix", None), how.pop("slopes", None)
    if prefix:
        dev["prefix_lengths"] = torch.tensor(prefix, dtype=torch.int32).cuda()
    if slopes:
        slopes = 2.0 ** -torch.arange(1, 5).float()
        dev["slopes"] = slopes.cuda()
    out, lse = paged_attention(case.batch, 0, case.q.cuda(), return_lse=True, fp32_weights=True, **how, **dev)
    rounded = paged_attention(case.batch, 0, case.q.cuda(), **how, **dev)
    u = torch.finfo(dtype).eps / 2
    err = {"fp32": 0.0, "rounded": 0.0}
    for b, length, m, at in case.spans():
        for h in range(4 if m else 0):
            k, v = (x[0, case.slots[b], h // 2] for x in (case.k, case.v))
            more = dict(how, slope=float(slopes[h]) if slopes is not None else 0.0, prefix=prefix[b] if prefix else 0)
            want, z, mag = oracle.attention(case.q[at:at + m, h], k, v, scale=dim ** -0.5, **more)
            d = oracle.score_error(case.q[at:at + m, h], k, scale=dim ** -0.5) + 2.0 ** -21 * (how.get("cap", 0.0) + more["slope"] * length)
            got = out[at:at + m, h].double().cpu()
            assert ((got - want).abs() - (u * want.abs() + mag * (4 * d + (length + 16) * 2.0 ** -23) + 1e-30)).max() <= 0, (b, h)
            assert ((lse[at:at + m, h].double().cpu() - z).abs() - (d + (length + 16) * 2.0 ** -23 + 2.0 ** -22 * z.abs())).max() <= 0
            err["fp32"] += float((got - want).square().sum())
            err["rounded"] += float((rounded[at:at + m, h].double().cpu() - want).square().sum())
    assert err["fp32"] <= err["rounded"]
