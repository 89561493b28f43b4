"""GPU: evictions of requests whose cached or target rows are not all there."""

from __future__ import annotations

import math

import pytest
import torch

from cachebridge_amd.online.queries import (ERROR_CACHE_ROW, ERROR_TARGET_ROW, QueryBatch, evict_tokens,
                                            paged_attention)
from cachebridge_amd.plan import rows_from_stacked

from .query_cases import make

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def flagged(*, lose_source=(), lose_target=(), budget=20):
    """Two requests of 50 tokens, request 0 without some rows, into a pool full of NaN: (case, kept, target, its index, flag)."""
    case = make([50, 50], [1, 1], heads=2, kv_heads=2, dim=64, index="i32", seed=2)
    qs, ln, off = case.batch._keep
    index = case.batch.rows.keep[-1].clone()
    index[list(lose_source)] = -1
    batch = QueryBatch(rows_from_stacked(*case.pool, index=index), qs, ln, offsets=off, max_length=50)
    k, v = (torch.full((1, 128, 2, 64), math.nan, dtype=BF16).cuda() for _ in range(2))
    to = torch.randperm(128, generator=torch.Generator().manual_seed(3)).int()
    to[list(lose_target)] = 128
    grown = torch.zeros(2, dtype=torch.int32).cuda()
    target = QueryBatch(rows_from_stacked(k, v, index=to.cuda()), qs, grown, request_stride=64, max_length=64)
    flag = torch.zeros(1, dtype=torch.int32).cuda()
    w = torch.arange(100, dtype=torch.float32).view(2, 50).flip(1).cuda()
    kept = evict_tokens(batch, w, target, budget=budget, error_flag=flag)
    grown.copy_(kept.lengths)
    return case, kept, target, to, int(flag)


@pytest.mark.parametrize("budget", [20, 50])
def test_a_request_that_lost_kept_tokens_has_no_length(budget):
    case, kept, target, to, flag = flagged(lose_source=[7], budget=budget)
    assert flag == ERROR_CACHE_ROW
    assert kept.lengths.tolist() == [0, budget]
    assert kept.tokens.tolist() == [list(range(budget))] * 2
    # What a program goes on with is finite: the row that kept its NaN is nobody's.
    out = torch.full((2, 2, 64), 5.0, dtype=BF16).cuda()
    paged_attention(target, 0, case.q.cuda(), out=out, error_flag=torch.zeros(1, dtype=torch.int32).cuda())
    assert (out[0] == 5.0).all() and torch.isfinite(out[1]).all()
    at = to[64:64 + budget].long()
    assert torch.equal(target.rows.keep[0][0, at].cpu(), case.k[0, case.slots[1][:budget]])


def test_a_lost_row_of_a_token_that_is_not_kept_does_no_harm():
    case, kept, target, to, flag = flagged(lose_source=[30])
    assert flag == 0 and kept.lengths.tolist() == [20, 20]


def test_a_token_without_a_target_row_is_left_out_there_too():
    case, kept, target, to, flag = flagged(lose_target=[7])
    assert flag == ERROR_TARGET_ROW and kept.lengths.tolist() == [20, 20]
    again = torch.zeros(1, dtype=torch.int32).cuda()
    out = paged_attention(target, 0, case.q.cuda(), error_flag=again)
    assert int(again) == ERROR_CACHE_ROW and torch.isfinite(out).all()
