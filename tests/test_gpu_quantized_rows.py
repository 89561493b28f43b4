"""GPU: steps of several new tokens over an 8-bit cache, 17 to 32 query rows a KV head: two blocks of rows a wave."""

from __future__ import annotations

import pytest
import torch

from cachebridge_amd.online.queries import QueryBatch, paged_attention

from .quantized_cases import make
from .query_cases import check_attention
from .test_gpu_quantized_attention import attend
from .test_gpu_quantized_attention import test_rows_of_no_request_and_strides as rows_of_no_request_and_strides
from .test_gpu_quantized_attention import test_what_is_not_seen_never_counts as what_is_not_seen_never_counts
from .test_gpu_queries import MASKS

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16

# lengths, new tokens, (heads, KV heads): the longest request has 17 to 32 rows a KV head, others one block of them or none.
SHAPES = {
    "spec": ([190, 301, 33], [5, 8, 3], (8, 2)),
    "spec-wide": ([70, 512, 19], [4, 3, 1], (16, 2)),
    "full": ([32, 90, 64], [32, 17, 0], (2, 2)),
    "odd-group": ([75, 18, 6], [6, 4, 6], (15, 3)),
    "one-token": ([257, 1], [1, 1], (27, 1)),
    "splits": ([2100], [6], (4, 1)),
    "splits-long": ([5000, 40], [2, 1], (9, 1)),
    "many": ([40 + 3 * i for i in range(70)], [1 + i % 3 for i in range(70)], (16, 2)),
}


def rows_of(new, heads):
    return max(new) * heads[0] // heads[1]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [48, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_causal(shape, dim, dtype):
    lengths, new, heads = SHAPES[shape]
    assert 16 < rows_of(new, heads) <= 32
    case = make(lengths, new, heads=heads[0], kv_heads=heads[1], dim=dim, dtype=dtype, seed=len(shape) + dim)
    check_attention(case, *attend(case))


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 128), (BF16, 256), (FP16, 64), (FP16, 128), (FP16, 192)])
@pytest.mark.parametrize("mask", list(MASKS))
@pytest.mark.parametrize("shape", ["spec", "spec-wide"])
def test_masks(shape, mask, dtype, dim):
    lengths, new, heads = SHAPES[shape]
    case = make(lengths, new, heads=heads[0], kv_heads=heads[1], dim=dim, dtype=dtype, seed=3)
    how = dict(MASKS[mask])
    dev = {}
    if how.get("prefix"):
        dev["prefix_lengths"] = torch.tensor(how["prefix"], dtype=torch.int32).cuda()
    if how.get("slopes"):
        how["slopes"] = 2.0 ** -(1 + torch.arange(heads[0]).float() / 2)
        dev["slopes"] = how["slopes"].cuda()
    kw = {k: v for k, v in how.items() if k not in ("prefix", "slopes")}
    check_attention(case, *attend(case, **kw, **dev), **how)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,new", [(4, 9), (4, 12), (4, 16), (8, 7), (8, 5)])
def test_what_one_block_does_not_see_never_counts(heads, new, dim, dtype):
    """The heads share two KV heads: 18 to 32 rows. NaN that the first rows do not see and the last do is in the tile of both."""
    assert 16 < new * heads // 2 <= 32
    what_is_not_seen_never_counts(new, dim, heads, dtype)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("new", [[6, 10], [10, 2]])
def test_strides(new, dtype):
    rows_of_no_request_and_strides(new, dtype)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_a_captured_call_follows_the_lengths(dtype):
    """Three new tokens a request, eight heads a KV head: a captured call against the eager one, lengths as they grow."""
    case = make([600, 350], [3, 3], heads=16, kv_heads=2, dim=128, dtype=dtype, seed=5)
    old = case.batch
    lengths = torch.tensor([100, 3], dtype=torch.int32).cuda()
    batch = QueryBatch(old.rows, old._keep[0], lengths, request_stride=old.c.request_stride, max_length=600, max_query=3)
    q = case.q.cuda()
    paged_attention(batch, 0, q, return_lse=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = paged_attention(batch, 0, q, return_lse=True)
    for i in range(4):
        lengths += torch.tensor([150, 115], dtype=torch.int32).cuda() * (i > 0)
        graph.replay()
        torch.cuda.synchronize()
        want = paged_attention(batch, 0, q, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), i
        case.lengths = lengths.tolist()
        slots, case.slots = case.slots, [s[:n] for s, n in zip(case.slots, case.lengths)]
        check_attention(case, *got)
        case.slots = slots
