"""GPU: which requests, index tokens and rows of a query batch belong to whom."""

from __future__ import annotations

import pytest
import torch

from cachebridge_amd.online.queries import (ERROR_REQUEST, ERROR_TARGET_ROW, QueryBatch, Rotary, add_key_weights,
                                            evict_tokens, install_tokens, paged_attention)
from cachebridge_amd.online.delivery import _at_offset
from cachebridge_amd.plan import Rows, rows_from_stacked
from oracle import queries as oracle

from .query_cases import check_attention, make

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def int32(*x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def new_flag():
    return torch.zeros(1, dtype=torch.int32).cuda()


def close(got, q, k, v, **how):
    """One head's rows against the oracle: roundings of the result and of the weights, and fp32 sums of 100 terms."""
    want, _, mag = oracle.attention(q, k, v, scale=q.shape[1] ** -0.5, **how)
    u = torch.finfo(q.dtype).eps / 2
    return ((got.double().cpu() - want).abs() - (u * want.abs() + (u + 2.0 ** -14) * mag)).max() <= 0


def slots_of_32(index, g):
    """(rows arguments, pool row of each of 3 * 32 index tokens)."""
    if index == "identity":
        return {}, torch.arange(96)
    pages = torch.randperm(6, generator=g)
    t = torch.arange(96)
    return dict(block_table=pages.int().cuda(), page_size=16), pages[t // 16] * 16 + t % 16


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("index", ["identity", "table"])
def test_a_request_longer_than_its_stride_is_left_out(index, dtype):
    """Request 0 has 40 cached tokens where 32 are its own: the next ones are request 1's."""
    g = torch.Generator().manual_seed(1)
    dim, lengths = 64, [40, 30, 32]
    k, v = (torch.randn(1, 96, 2, dim, generator=g).to(dtype) for _ in range(2))
    fused = torch.randn(6, 8, dim, generator=g).to(dtype)
    more, slot = slots_of_32(index, g)
    kd, vd = k.cuda(), v.cuda()
    batch = QueryBatch(rows_from_stacked(kd, vd, **more), int32(0, 2, 4, 6), int32(*lengths), max_length=50, max_query=2,
                       request_stride=32)
    fd = fused.cuda()
    out = torch.full_like(fd[:, :4], 5.0)
    flag = new_flag()
    q = install_tokens(batch, 0, fd[:, :4], fd[:, 4:6], fd[:, 6:], Rotary.build(dim, 1e4), out=out, error_flag=flag)
    assert int(flag) == ERROR_REQUEST and (q[:2] == 5.0).all()
    stored = torch.cat([slot[32 * b + n - 2:32 * b + n] for b, n in ((1, 30), (2, 32))])
    assert torch.equal(vd[0, stored].cpu(), fused[2:, 6:])
    rest = torch.ones(96, dtype=torch.bool)
    rest[stored] = False
    for x, y in ((kd, k), (vd, v)):
        assert torch.equal(x[0].cpu()[rest], y[0][rest])

    out = torch.full_like(q, 7.0)
    flag = new_flag()
    _, lse = paged_attention(batch, 0, q, out=out, return_lse=True, error_flag=flag)
    assert int(flag) == ERROR_REQUEST and (out[:2] == 7.0).all()
    for b in (1, 2):
        at = slot[32 * b:32 * b + lengths[b]]
        for h in range(4):
            assert close(out[2 * b:2 * b + 2, h], q[2 * b:2 * b + 2, h].cpu(), kd[0, at, h // 2].cpu(), vd[0, at, h // 2].cpu())

    weights = torch.full((3, 50), 3.0).cuda()
    flag = new_flag()
    lse[:2] = 0.0
    add_key_weights(batch, 0, q, lse, weights, error_flag=flag)
    assert int(flag) == ERROR_REQUEST and (weights[0] == 3.0).all()
    assert (weights[1, :30] > 3.0).all() and (weights[1, 30:] == 3.0).all() and (weights[2, :32] > 3.0).all()

    tk, tv = torch.zeros_like(kd), torch.zeros_like(vd)
    target = QueryBatch(rows_from_stacked(tk, tv), int32(0, 2, 4, 6), int32(*lengths), max_length=50, request_stride=32)
    flag = new_flag()
    kept = evict_tokens(batch, weights, target, budget=20, error_flag=flag)
    assert int(flag) == ERROR_REQUEST and kept.lengths.tolist() == [0, 20, 20]
    assert (tk[0, :32] == 0).all() and torch.equal(tk[0, 32], kd[0, slot[32 + int(kept.tokens[1, 0])]])


def test_evicted_tokens_stay_within_their_request_s_stride():
    """A budget above the target's stride: what is past it is not copied over the next request's rows."""
    case = make([50, 20, 45], [1, 1, 1], heads=2, kv_heads=2, dim=64, seed=2)
    k, v = torch.zeros(1, 96, 2, 64, dtype=BF16).cuda(), torch.zeros(1, 96, 2, 64, dtype=BF16).cuda()
    target = QueryBatch(rows_from_stacked(k, v), *case.batch._keep[:2], request_stride=32, max_length=50)
    flag = new_flag()
    kept = evict_tokens(case.batch, torch.ones(3, 50).cuda(), target, budget=60, error_flag=flag)
    assert int(flag) == ERROR_TARGET_ROW and kept.lengths.tolist() == [50, 20, 45]
    for b, n in ((0, 32), (1, 20), (2, 32)):
        for got, src in ((k, case.k), (v, case.v)):
            assert torch.equal(got[0, 32 * b:32 * b + n].cpu(), src[0, case.slots[b][:n]])
    assert (k[0, 52:64] == 0).all()


def test_several_requests_need_places_of_their_own():
    case = make([30, 20], [1, 1], dim=64, index="i32")
    qs, ln, _ = case.batch._keep
    with pytest.raises(ValueError, match="offsets or a request_stride"):
        QueryBatch(case.batch.rows, qs, ln, max_length=30)
    QueryBatch(case.batch.rows, qs, ln, max_length=30, offsets=torch.zeros(2, dtype=torch.int64).cuda())  # one history


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("new", [1, 30, 200])
def test_bounds_far_above_the_lengths_without_a_stride(new, dtype):
    case = make([1500, 300, 210], [new, new, min(new, 7)], heads=4, kv_heads=2, dim=64, dtype=dtype, seed=new, index="offsets")
    qs, ln, off = case.batch._keep
    for bound in (1500, 40000, 1 << 20):
        batch = QueryBatch(case.batch.rows, qs, ln, offsets=off, max_length=bound, max_query=new)
        out, lse = paged_attention(batch, 0, case.q.cuda(), return_lse=True)
        check_attention(case, out, lse)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("bad", [0, 63, 70, 149])
def test_a_bad_request_among_many_is_flagged(bad, dtype):
    """Query tiles found by a search: whichever of the searched requests is outside the bounds."""
    lengths, new = [20 + b % 9 for b in range(150)], [1 + b % 3 for b in range(150)]
    new[5] = 20  # by-request places would be twenty times the tiles
    case = make(lengths, new, heads=64, kv_heads=2, dim=64, dtype=dtype, seed=5)
    qs, ln, _ = case.batch._keep
    ln = ln.clone()
    ln[bad] = 60
    batch = QueryBatch(case.batch.rows, qs, ln, max_length=50, max_query=20, request_stride=case.batch.c.request_stride)
    out = torch.full_like(case.q, 9.0).cuda()
    flag = new_flag()
    paged_attention(batch, 0, case.q.cuda(), out=out, error_flag=flag)
    assert int(flag) == ERROR_REQUEST
    mine = torch.zeros(case.tokens, dtype=torch.bool)
    mine[sum(new[:bad]):sum(new[:bad + 1])] = True
    want = paged_attention(case.batch, 0, case.q.cuda())
    assert (out[mine.cuda()] == 9.0).all() and torch.equal(out[~mine.cuda()], want[~mine.cuda()])


# Query starts, and the requests whose rows are their own; max_query is 8.
STARTS = {
    "falls": ([0, 8, 4, 12], [0]),               # request 1 falls, request 2 starts behind row 8
    "past the end": ([0, 100, 3, 6], []),         # requests 1 and 2 start before the 100th row
    "last past the end": ([0, 3, 100], [0]),
    "late": ([2, 1, 0, 8], []),                  # every later start is below the first
    "twice": ([0, 3, 1, 3, 3, 9, 8, 12], [0, 3, 4]),
    "negative": ([-2, 3, 7], [1]),
}


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("length,dtype", [(30, BF16), (30, FP32), (3000, BF16), (3000, FP32)])
@pytest.mark.parametrize("starts", list(STARTS))
def test_rows_of_falling_starts_have_one_owner(starts, length, dtype, many):
    """Install, attention (keys split or not) and key weights answer the same requests and leave all other rows.

    ``many``: 70 empty requests stand before them, and tiles are found by a search."""
    start, good = STARTS[starts]
    front = 70 if many else 0
    n, heads, dim = len(start) - 1, 4, 64
    case = make([length] * (n + front), [0] * (n + front), heads=heads, kv_heads=2, dim=dim, dtype=dtype, seed=7, page=16)
    qs = int32(*[start[0]] * front, *start)
    tokens = 12
    batch = QueryBatch(case.batch.rows, qs, case.batch._keep[1], max_length=length, max_query=8,
                       request_stride=case.batch.c.request_stride)
    g = torch.Generator().manual_seed(2)
    fused = torch.randn(tokens, 8, dim, generator=g).to(dtype).cuda()
    owner = {t: front + b for b in good for t in range(start[b], start[b + 1])}
    mine = torch.tensor([t in owner for t in range(tokens)])
    before = [x.clone() for x in case.pool]
    out = torch.full((tokens, heads, dim), 5.0, dtype=dtype).cuda()
    flag = new_flag()
    q = install_tokens(batch, 0, fused[:, :4], fused[:, 4:6], fused[:, 6:], Rotary.build(dim, 1e4), out=out, error_flag=flag)
    assert int(flag) == ERROR_REQUEST
    assert torch.equal((q == 5.0).all(-1).all(-1).cpu(), ~mine)
    stored = torch.zeros(before[0].shape[1], dtype=torch.bool)
    for b in good:
        m = start[b + 1] - start[b]
        at = case.slots[front + b][length - m:] if m else case.slots[front + b][:0]
        stored[at] = True
        assert torch.equal(case.pool[1][0, at].cpu(), fused[start[b]:start[b + 1], 6:].cpu())
    for x, y in zip(case.pool, before):
        assert torch.equal(x[0][~stored.cuda()], y[0][~stored.cuda()])

    out = torch.full_like(q, 7.0)
    flag = new_flag()
    _, lse = paged_attention(batch, 0, q, out=out, return_lse=True, error_flag=flag)
    assert int(flag) == ERROR_REQUEST
    assert torch.equal((out == 7.0).all(-1).all(-1).cpu(), ~mine)
    kc, vc = (x.cpu() for x in case.pool)
    for b in good:
        at = case.slots[front + b]
        for h in (0, 3):
            rows = slice(start[b], start[b + 1])
            assert start[b] == start[b + 1] or close(out[rows, h], q[rows, h].cpu(), kc[0, at, h // 2], vc[0, at, h // 2])

    lse[~mine.cuda()] = 0.0
    weights = torch.zeros(n + front, length).cuda()
    flag = new_flag()
    add_key_weights(batch, 0, q, lse, weights, error_flag=flag)
    assert int(flag) == ERROR_REQUEST
    want = torch.zeros(n + front)
    for b in owner.values():
        want[b] += heads
    # Each row's weights sum to one: fp32 sums of up to 3000 terms, and scores of at most 16.
    assert ((weights.sum(1).cpu() - want).abs() <= want * (3000 * 2.0 ** -23 + 2.0 ** -16)).all()


def test_outputs_whose_rows_share_memory_are_refused():
    case = make([30], [3], dim=64)
    q = case.q.cuda()
    for out in (q[:1].expand(3, 4, 64), q[:, :1].expand(3, 4, 64)):
        with pytest.raises(ValueError, match="share memory"):
            paged_attention(case.batch, 0, q, out=out)
        with pytest.raises(ValueError, match="share memory"):
            install_tokens(case.batch, 0, q, q[:, :2], q[:, 2:], Rotary.build(64, 1e4), out=out)
    # Inputs may: one row of queries for every token.
    got = paged_attention(case.batch, 0, q[:1].expand(3, 4, 64))
    assert torch.equal(got[0], paged_attention(case.batch, 0, q)[0])


def test_rows_have_to_say_how_long_their_index_is():
    """Without it every cached token would count as missing."""
    case = make([30], [3], dim=64, index="i32")
    rows = case.batch.rows
    qs, ln, _ = case.batch._keep
    with pytest.raises(ValueError, match="entries"):
        QueryBatch(Rows(rows.c, rows.dtype, rows.device, rows.keep), qs, ln, max_length=30)
    # Another offset into the same index.
    moved = _at_offset(rows, 10)
    flag = new_flag()
    out = paged_attention(QueryBatch(moved, int32(0, 3), int32(20), max_length=20), 0, case.q.cuda(), error_flag=flag)
    assert int(flag) == 0
    at = case.slots[0][10:]
    for h in range(4):
        assert close(out[:, h], case.q[:, h], case.k[0, at, h // 2], case.v[0, at, h // 2])


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("at,to", [(3, 50), (3, 640), (300, 690), (699, 0)])
def test_a_start_out_of_order_among_many(at, to, dtype):
    """Steps of 700 requests, one start misplaced: those that start below an earlier one are left out, the others are not."""
    n = 700
    case = make([9] * n, [1] * n, heads=4, kv_heads=2, dim=64, dtype=dtype, seed=4)
    start = list(range(n + 1))
    start[at] = to
    bad = [b for b in range(n) if not 0 <= start[b + 1] - start[b] <= 1 or start[b] < max(start[:b + 1])]
    batch = QueryBatch(case.batch.rows, int32(*start), case.batch._keep[1], max_length=9, max_query=1,
                       request_stride=case.batch.c.request_stride)
    q = case.q.cuda()
    want, want_lse = paged_attention(case.batch, 0, q, return_lse=True)
    flag, out = new_flag(), torch.full_like(q, 7.0)
    paged_attention(batch, 0, q, out=out, error_flag=flag)
    assert int(flag) == ERROR_REQUEST
    rows = [start[b] for b in range(n) if b not in bad and start[b + 1] > start[b]]
    mine = torch.zeros(n, dtype=torch.bool)
    mine[rows] = True
    assert torch.equal(out[mine.cuda()], want[mine.cuda()]) and (out[~mine.cuda()] == 7.0).all()
    weights = torch.zeros(2, n, 9).cuda()
    flag = new_flag()
    add_key_weights(case.batch, 0, q, want_lse, weights[0])
    add_key_weights(batch, 0, q, want_lse, weights[1], error_flag=flag)
    assert int(flag) == ERROR_REQUEST
    good = torch.tensor([b not in bad and start[b + 1] > start[b] for b in range(n)]).cuda()
    assert torch.equal(weights[1][good], weights[0][good]) and (weights[1][~good] == 0).all()


@pytest.mark.parametrize("fp32_weights", [False, True])
def test_a_captured_step_stops_at_the_stride(fp32_weights):
    """Two graphs of one step, replayed in turn while lengths grow: request 0 reaches its stride of 32 and is left out
    from then on, request 1 goes on as before."""
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(1, 96, 2, 64, generator=g).to(BF16).cuda() for _ in range(2))
    fused = torch.randn(2, 8, 64, generator=g).to(BF16).cuda()
    lengths, start, flag = int32(29, 9), int32(0, 1, 2), new_flag()
    batch = QueryBatch(rows_from_stacked(k, v), start, lengths, max_length=50, max_query=1, request_stride=32)
    alone = QueryBatch(rows_from_stacked(k, v), start, lengths, max_length=50, max_query=1, offsets=torch.tensor([64, 32]).cuda())
    spin, weights = Rotary.build(64, 1e4), torch.zeros(2, 50).cuda()
    out = torch.zeros(2, 4, 64, dtype=BF16).cuda()

    def step(batch):
        q = install_tokens(batch, 0, fused[:, :4], fused[:, 4:6], fused[:, 6:], spin, error_flag=flag)
        _, lse = paged_attention(batch, 0, q, out=out, return_lse=True, cap=20.0, fp32_weights=fp32_weights, error_flag=flag)
        add_key_weights(batch, 0, q, torch.nan_to_num(lse, neginf=-1e30), weights, cap=20.0, error_flag=flag)

    step(batch)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(batch)
        graphs.append(graph)
    for turn in range(6):
        lengths += 1
        flag.zero_()
        out.fill_(7.0)
        weights.zero_()
        before = k.clone(), v.clone()
        torch.cuda.synchronize()
        graphs[turn % 2].replay()
        torch.cuda.synchronize()
        past = 30 + turn > 32
        assert int(flag) == (ERROR_REQUEST if past else 0), turn
        assert bool((out[0] == 7.0).all()) == past and bool((weights[0] == 0).all()) == past
        changed = (v != before[1])[0].flatten(1).any(1).nonzero().flatten().tolist()
        assert set(changed) <= ({32 + 9 + turn} if past else {29 + turn, 32 + 9 + turn}), turn
        got, w = out[1].clone(), weights[1].clone()
        weights.zero_()
        step(alone)  # request 0 elsewhere: request 1 has the same bits
        assert torch.equal(out[1], got) and torch.equal(weights[1], w)
        k.copy_(before[0])
        v.copy_(before[1])
