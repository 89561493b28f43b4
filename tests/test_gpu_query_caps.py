"""GPU: capped scores keep the accuracy of the score, whatever the cap."""

from __future__ import annotations

import pytest
import torch

from cachebridge_amd.online.queries import add_key_weights, paged_attention
from oracle import queries as oracle

from .query_cases import make

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 128), (BF16, 256), (FP16, 128), (FP32, 64), (BF16, 30)])
@pytest.mark.parametrize("new", [[1, 1, 1], [90, 7, 33], [180, 290, 33]])
@pytest.mark.parametrize("scale", [0.02, -0.25])
@pytest.mark.parametrize("cap", [1e-40, 1e-3, 2.0, 30.0, 50.0, 1e3, 1e6, 1e20, 3e38])
def test_capped_scores(cap, scale, new, dtype, dim):
    """Bounds as query_cases.check_attention and check_weights derive them, but for the cap: a score is off by its
    products' error and by 2^-20 of the largest score of the heads that share K (polynomial 2^-23 and some five
    roundings of the score itself; the forms of exp(2y) 3 2^-23 of the cap, taken where that largest score is 0.55 of
    the cap or more), not by a share of whatever the cap is."""
    lengths, heads = [190, 301, 33], 4
    case = make(lengths, new, heads=heads, kv_heads=2, dim=dim, dtype=dtype, seed=3, spread=3.0)
    q = case.q.cuda()
    out, lse = paged_attention(case.batch, 0, q, return_lse=True, cap=cap, scale=scale)
    weights = torch.zeros(3, 301).cuda()
    add_key_weights(case.batch, 0, q, lse, weights, cap=cap, scale=scale)
    out, lse, weights = out.double().cpu(), lse.double().cpu(), weights.double().cpu()
    u = torch.finfo(dtype).eps / 2
    want_w, tol_w = torch.zeros(3, 301, dtype=torch.float64), torch.zeros(3, 301, dtype=torch.float64)
    for b, length, m, at in case.spans():
        for h in range(heads):
            qh = case.q[at:at + m, h]
            k, v = (x[0, case.slots[b], h // 2] for x in (case.k, case.v))
            want, z, mag = oracle.attention(qh, k, v, scale=scale, cap=cap)
            size = max(float(oracle.scores(case.q[at:at + m, g], k, scale=scale, cap=cap).abs().max())
                       for g in range(heads) if g // 2 == h // 2)
            d = min(oracle.score_error(qh, k, scale=scale), 2.0 * size) + 2.0 ** -20 * size
            small = 2.0 ** -25 * length * float(v.double().abs().max()) if dtype == FP16 else 0.0
            tol = u * want.abs() + u * mag + mag * (4 * d + (length + 16) * 2.0 ** -23) + small + 1e-30
            assert ((out[at:at + m, h] - want).abs() - tol).max() <= 0, (b, h)
            gap = (lse[at:at + m, h] - z).abs() - (d + (length + 16) * 2.0 ** -23 + 2.0 ** -22 * z.abs())
            assert gap.max() <= 0, (b, h, float(gap.max()))
            got = oracle.key_weights(qh, k, lse[at:at + m, h], scale=scale, cap=cap)
            want_w[b, :length] += got
            tol_w[b, :length] += got * 2 * (d + 2.0 ** -21 * (size + 10))
    tol_w += want_w * (sum(new) * heads + 16) * 2.0 ** -24 + 1e-30
    assert ((weights - want_w).abs() - tol_w).max() <= 0
