"""GPU: steps over an 8-bit cache whose values are as large or as small as the format has them."""

from __future__ import annotations

import pytest
import torch

from cachebridge_amd.online.queries import paged_attention
from oracle import quantized, queries

from .quantized_cases import codes_of, make

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def rewrite(case, kind, codes, exponents):
    """The pool's codes (uint8) and exponents [layers, pages, heads] of K (0) or V (1), and the case's values of them."""
    codes_of(case.pool[kind]).copy_(codes)
    codes_of(case.scales[kind]).copy_((exponents + 127).to(torch.uint8))
    setattr(case, "kv"[kind], quantized.values(codes, exponents, case.scale_page))


def scored(case, key):
    """One of 32 cached tokens scores 6.5, the others 0: K is 6.5 in element 0 of the tokens for which key(j) holds, 0
    elsewhere, and q is 1 there."""
    codes = torch.zeros(case.k.shape, dtype=torch.uint8)
    for slots in case.slots:
        at = torch.tensor([key(j) for j in range(len(slots))])
        codes[:, slots[at], :, 0] = 0x4d  # 1.625 * 2^2
    rewrite(case, 0, codes, torch.zeros(case.exponents[0].shape, dtype=torch.long))
    case.q.zero_()
    case.q[:, :, 0] = 1.0


def check(case, out, **mask):
    """The bounds of query_cases.check_attention, with half of bf16's least step in place of its 1e-30."""
    for b, length, new, at in case.spans():
        for h in range(case.heads):
            k, v = (x[0, case.slots[b], h * case.kv_heads // case.heads] for x in (case.k, case.v))
            want, _, mag = queries.attention(case.q[at:at + new, h], k, v, scale=1.0, **mask)
            d = queries.score_error(case.q[at:at + new, h], k, scale=1.0)
            tol = 2.0 ** -8 * want.abs() + mag * (2.0 ** -8 + 4 * d + (length + 16) * 2.0 ** -23) + 2.0 ** -134
            gap = (out[at:at + new, h].double().cpu() - want).abs() - tol
            assert gap.max() <= 0, (b, h, float(gap.max()), float(want.abs().max()))


# New tokens, requests, heads, KV heads: one split that holds all of a request's keys (as many workgroups as a launch is
# cut for), or several.
CUTS = {"one-split": (1, 32, 32, 32), "splits": (1, 2, 4, 2), "rows": (7, 32, 96, 32), "rows-splits": (6, 1, 8, 2)}


@pytest.mark.parametrize("cut", list(CUTS))
def test_large_values_behind_low_scores(cut):
    """V at the largest scale, and scores that grow by 2^9.4 without the running maximum being renewed: weights times
    scales leave fp32, the result does not."""
    new, requests, heads, kv = CUTS[cut]
    case = make([300] * requests, [new] * requests, heads=heads, kv_heads=kv, dim=64, dtype=BF16, seed=2)
    scored(case, lambda j: j >= 128 and j % 32 == 5)
    g = torch.Generator().manual_seed(7)
    codes = torch.randint(0, 0x7f if cut == "one-split" else 0x50, case.v.shape, generator=g, dtype=torch.uint8)
    codes[..., 3] = 0
    rewrite(case, 1, codes, torch.full(case.exponents[1].shape, 119))
    check(case, paged_attention(case.batch, 0, case.q.cuda(), scale=1.0))


@pytest.mark.parametrize("cut", list(CUTS))
def test_small_values_of_many_small_weights(cut):
    """V at the least scale and most of the weight on tokens of 2^-9.4 each: weights times scales are below bf16's
    normal range, the result is not."""
    new, requests, heads, kv = CUTS[cut]
    case = make([900] * requests, [new] * requests, heads=heads, kv_heads=kv, dim=64, dtype=BF16, seed=3)
    scored(case, lambda j: j % 32 == 5 and j < 128)
    codes = torch.randint(0x40, 0x7f, case.v.shape, generator=torch.Generator().manual_seed(8), dtype=torch.uint8)
    rewrite(case, 1, codes, torch.full(case.exponents[1].shape, -126))
    check(case, paged_attention(case.batch, 0, case.q.cuda(), scale=1.0))


@pytest.mark.parametrize("cut", list(CUTS))
@pytest.mark.parametrize("far", [119, -126])
def test_scales_of_tokens_that_none_sees(far, cut):
    """Before the window, pages whose scale is far from the others' change no bit; neither does a page of nobody."""
    new, requests, heads, kv = CUTS[cut]
    case = make([300] * requests, [new] * requests, heads=heads, kv_heads=kv, dim=64, dtype=BF16, seed=4)
    want = paged_attention(case.batch, 0, case.q.cuda(), window=100)
    e = case.exponents[1].clone()
    seen = torch.zeros(e.shape[1], dtype=torch.bool)
    for slots in case.slots:
        seen[slots[300 - new - 99:] // 16] = True
    e[:, ~seen] = far
    assert int((~seen).sum()) >= 12 * requests
    rewrite(case, 1, codes_of(case.pool[1]).cpu(), e)
    assert torch.equal(paged_attention(case.batch, 0, case.q.cuda(), window=100), want)
