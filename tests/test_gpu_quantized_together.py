"""GPU: 8-bit caches as they are used: a handed-off prefix quantized, answered and grown, captured steps, other streams,
caches past 2^32 bytes, calls that have nothing to do."""

from __future__ import annotations

import math

import pytest
import torch

from cachebridge_amd import QuantizedKVPool, pool_rows, synthetic
from cachebridge_amd.online.blocks import map_install_batch
from cachebridge_amd.online.queries import (ERROR_REQUEST, QueryBatch, Rotary, install_tokens, paged_attention,
                                            quantize_tokens)
from cachebridge_amd.plan import BlockScales, RequestSpan, rows_from_stacked
from oracle import quantized as oracle

from . import query_cases
from .quantized_cases import codes_of, make
from .query_cases import check_attention
from .test_gpu_query_handoff import check, tables

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def pool_values(pool, layer):
    """What layer's codes and scales stand for, in 64 bits on the CPU."""
    return [oracle.values(codes_of(x[layer]).cpu(), codes_of(s[layer]).cpu().int() - 127, pool.page_size)
            for x, s in ((pool.k_data, pool.k_scale), (pool.v_data, pool.v_scale))]


def state(pool):
    return [codes_of(x) for x in (pool.k_data, pool.v_data, pool.k_scale, pool.v_scale)]


def test_from_the_handoff_to_answers_in_8_bits():
    """A cohort's mapped prefixes go into an 8-bit pool of other pages, then prompts and steps grow and answer on them."""
    layers, page, history, new = 2, 32, [333, 250], [5, 40]
    sh = synthetic.shape("tp4", tokens=sum(history))
    sh.target_layers = layers
    h = synthetic.make_handoff(sh, target_pages=64)
    g = torch.Generator().manual_seed(3)
    table, offsets, slots = tables(history, torch.randperm(64, generator=g).tolist())
    spans = [RequestSpan(0, int(offsets[0]), history[0], 0, history[0]),
             RequestSpan(history[0], int(offsets[1]), history[1], 0, history[1])]
    map_install_batch(h.mapper, h.source_pool, h.source_slots, h.target_pool, spans, block_table=table, page_size=16)
    kv, dim, dtype = h.target_pool.head_num, h.target_pool.head_dim, h.target_pool.dtype
    lengths = torch.tensor(history, dtype=torch.int32).cuda()
    start = torch.zeros(3, dtype=torch.int32).cuda()
    prefix = QueryBatch(pool_rows(h.target_pool, block_table=table, page_size=16), start, lengths, offsets=offsets, max_length=333)

    pool = QuantizedKVPool(layer_num=layers, pages=40, head_num=kv, head_dim=dim, page_size=page, dtype=dtype, fill="zeros")
    order = torch.randperm(40, generator=g).int().view(2, 20)
    rows = pool_rows(pool, block_table=order.view(-1).cuda())
    grown = lengths.clone()
    flag = torch.zeros(1, dtype=torch.int32).cuda()
    batch = QueryBatch(rows, torch.tensor([0, 5, 45], dtype=torch.int32).cuda(), grown, request_stride=20 * page, max_length=600)
    assert quantize_tokens(prefix, batch, error_flag=flag).tolist() == history
    where = [torch.tensor([int(order[b, t // page]) * page + t % page for t in range(20 * page)]) for b in range(2)]
    for layer in range(layers):
        for x, y in zip(pool_values(pool, layer), (h.target_pool.k_buffer[layer], h.target_pool.v_buffer[layer])):
            for b, n in enumerate(history):
                want = y[slots[b]].double().cpu()
                got = x[where[b][:n]]
                # Half a step of the page's scale: at most 2^-4 of the value, or of 2^-6 times the scale (448 of which the
                # page's largest is above half of).
                top = want.abs().amax(-1).clamp(min=1e-9)
                for p in range(0, n, page):
                    size = want[p:p + page].abs().amax((0, 2))
                    assert ((got[p:p + page] - want[p:p + page]).abs() <= 2.0 ** -4 * want[p:p + page].abs() + (2.0 ** -10 * size / 224)[:, None]).all(), (layer, b, p)
                assert torch.isfinite(top).all()

    heads, spin, total = 4 * kv, Rotary.build(dim, 1e6), 45
    one = torch.tensor([0, 1, 2], dtype=torch.int32).cuda()
    step = QueryBatch(rows, one, grown, request_stride=20 * page, max_length=600, max_query=1)
    grown += torch.tensor(new, dtype=torch.int32).cuda()
    for who, count in ((batch, new), (step, [1, 1]), (step, [1, 1])):
        if who is step:
            grown += 1
        x = torch.randn(layers, sum(count), heads + 2 * kv, dim, generator=g).to(dtype).cuda()
        now = grown.tolist()
        for layer in range(layers):
            y = x[layer]
            q = install_tokens(who, layer, y[:, :heads], y[:, heads:heads + kv], y[:, heads + kv:], spin, error_flag=flag)
            out = paged_attention(who, layer, q, error_flag=flag)
            k, v = pool_values(pool, layer)
            at = 0
            for b, m in enumerate(count):
                mine = where[b][:now[b]]
                check(out[at:at + m], q[at:at + m].cpu(), k[mine], v[mine], dim)
                stored = y[at:at + m, heads + kv:].double().cpu()
                got = v[mine[-m:]]
                assert ((got - stored).abs() <= 2.0 ** -4 * stored.abs() + 2.0 ** -10 * v[mine].abs().max() / 224).all()
                at += m
    assert int(flag) == 0 and total == sum(new)
    with pytest.raises(ValueError):
        map_install_batch(h.mapper, h.source_pool, h.source_slots, pool, spans, block_table=order.view(-1).cuda(), page_size=page)


def steps(seed, *, dtype=BF16, page=16, heads=8, kv=2, dim=128, lengths=(70, 33, 250), room=24):
    """A pool, a step batch on it whose lengths may grow by `room`, and a step's rows."""
    case = make(list(lengths), [1] * len(lengths), heads=heads, kv_heads=kv, dim=dim, dtype=dtype, page=page, seed=seed)
    width = -(-(max(lengths) + room) // page)
    pool = QuantizedKVPool(layer_num=1, pages=width * len(lengths), head_num=kv, head_dim=dim, page_size=page, dtype=dtype, fill="zeros")
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(pool.pages, generator=g).int().cuda()
    grown = torch.tensor(lengths, dtype=torch.int32).cuda()
    plain = query_cases.make(list(lengths), [1] * len(lengths), heads=heads, kv_heads=kv, dim=dim, dtype=dtype, page=16, seed=seed)
    batch = QueryBatch(pool_rows(pool, block_table=table), torch.arange(len(lengths) + 1, dtype=torch.int32).cuda(), grown,
                       request_stride=width * page, max_length=max(lengths) + room, max_query=1)
    assert quantize_tokens(plain.batch, batch).tolist() == list(lengths)
    fused = torch.randn(room, len(lengths), heads + 2 * kv, dim, generator=g).to(dtype).cuda()
    return pool, batch, grown, fused, heads, kv, Rotary.build(dim, 1e4), case


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_captured_steps_follow_the_lengths(dtype):
    """Two captured steps (store and attend) on two pools, replayed in turn while lengths grow, with eager work and
    synchronizations between: every replay is the eager call."""
    runs = []
    for seed in (1, 2):
        pool, batch, grown, fused, heads, kv, spin, _ = steps(seed, dtype=dtype)
        twin = [x.clone() for x in (pool.k_data.view(torch.uint8), pool.v_data.view(torch.uint8), codes_of(pool.k_scale), codes_of(pool.v_scale))]
        row = fused[0].clone()

        def call(b=batch, r=row, h=heads, n=kv, s=spin):
            q = install_tokens(b, 0, r[:, :h], r[:, h:h + n], r[:, h + n:], s)
            return paged_attention(b, 0, q, return_lse=True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call()
        for x, y in zip(state(pool), twin):
            x.copy_(y)
        k, v, ks, vs = twin
        scales = BlockScales(ks.view(torch.float8_e8m0fnu), vs.view(torch.float8_e8m0fnu), 16, dtype)
        same = QueryBatch(rows_from_stacked(k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), block_table=batch.rows.keep[2],
                                            page_size=16, scales=scales), *batch._keep[:2], request_stride=batch.c.request_stride,
                          max_length=batch.max_length, max_query=1)
        runs.append((pool, grown, fused, row, graph, got, twin, same, call))
    for i in range(20):
        for pool, grown, fused, row, graph, got, twin, same, call in runs:
            grown += 1
            row.copy_(fused[i])
            graph.replay()
            if i % 3 == 0:
                torch.cuda.synchronize()
            torch.zeros(1 << 20, device="cuda").add_(1)  # eager work between the replays
            want = call(same, row)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), i
            assert all(torch.equal(x, y) for x, y in zip(state(pool), twin)), i


def test_a_captured_quantize_is_replayed():
    case = query_cases.make([100, 37], [1, 1], heads=2, kv_heads=2, dim=128, layers=3, seed=4)
    pool = QuantizedKVPool(layer_num=3, pages=20, head_num=2, head_dim=128)
    target = QueryBatch(pool_rows(pool, block_table=torch.randperm(20).int().cuda()), *case.batch._keep[:2], request_stride=160, max_length=100)
    out = torch.zeros(2, dtype=torch.int32).cuda()
    quantize_tokens(case.batch, target, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        quantize_tokens(case.batch, target, out=out)
    for i in range(4):
        for x in case.pool:
            x.mul_(1.37)
        for x in state(pool):
            x.fill_(3)
        out.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in state(pool)]
        for x in state(pool):
            x.fill_(3)
        assert torch.equal(quantize_tokens(case.batch, target), out) and out.tolist() == [100, 37]
        assert all(torch.equal(x, y) for x, y in zip(got, state(pool))), i


def test_on_another_stream_and_twice_the_same_bits():
    pool, batch, grown, fused, heads, kv, spin, _ = steps(5, lengths=(2000, 130), room=8)
    row = fused[0]
    before = [x.clone() for x in state(pool)]
    grown += 1
    q = install_tokens(batch, 0, row[:, :heads], row[:, heads:heads + kv], row[:, heads + kv:], spin)
    want = paged_attention(batch, 0, q, return_lse=True)
    after = [x.clone() for x in state(pool)]
    for x, y in zip(state(pool), before):
        x.copy_(y)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    q2 = install_tokens(batch, 0, row[:, :heads], row[:, heads:heads + kv], row[:, heads + kv:], spin, stream=side)
    got = paged_attention(batch, 0, q2, return_lse=True, stream=side)
    side.synchronize()
    assert torch.equal(q, q2) and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert all(torch.equal(x, y) for x, y in zip(state(pool), after))


@pytest.mark.parametrize("new", [1, 3, 40])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_bytes_past_32_bits(new, dtype):
    """A layer of 5 GB: pages on both sides of 2^32 bytes, stored and read; scales past the first pages."""
    kv, dim, page, rows = 16, 256, 64, 5 * (1 << 30) // 4096
    k, v = (torch.empty(1, rows, kv, dim, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    pages = rows // page
    scales = [torch.full((1, pages, kv), 99, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2)]
    far = (1 << 32) // 4096 // page  # the page that 2^32 bytes lie before
    mine = [3, far - 1, far, pages - 1]
    table = torch.tensor(mine, dtype=torch.int32).cuda()
    length = 4 * page - 7
    small = query_cases.make([length], [new], heads=kv, kv_heads=kv, dim=dim, dtype=dtype, seed=new)
    batch = QueryBatch(rows_from_stacked(k, v, block_table=table, page_size=page, scales=BlockScales(*scales, page, dtype)),
                       *small.batch._keep[:2], request_stride=4 * page, max_length=length)
    assert quantize_tokens(small.batch, batch).tolist() == [length]
    where = torch.cat([torch.arange(page) + p * page for p in mine])[:length]

    def held():
        return [torch.cat([oracle.values(codes_of(x[:, p * page:(p + 1) * page]).cpu(), codes_of(s[:, p:p + 1]).cpu().int() - 127, page)
                           for p in mine], 1)[0, :length] for x, s in ((k, scales[0]), (v, scales[1]))]
    for x, y in zip(held(), (small.k, small.v)):
        want = y[0, small.slots[0]].double()
        assert ((x - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** -10 * want.abs().max() / 224).all()
    fused = torch.randn(new, 3 * kv, dim, generator=torch.Generator().manual_seed(9)).to(dtype).cuda()
    q = install_tokens(batch, 0, fused[:, :kv], fused[:, kv:2 * kv], fused[:, 2 * kv:], Rotary.build(dim, 1e4))
    out = paged_attention(batch, 0, q)
    kk, vv = held()
    stored = fused[:, 2 * kv:].double().cpu()
    assert ((vv[-new:] - stored).abs() <= 2.0 ** -4 * stored.abs() + 2.0 ** -10 * vv.abs().max() / 224).all()
    check(out, q.cpu(), kk, vv, dim)
    assert where.numel() == length


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_bounds_do_not_change_what_is_stored(dtype):
    """Pages found by request (a bound on new tokens is known) or by token (none is): the same bits."""
    lengths, new, n = [70, 16, 5, 300], [7, 1, 5, 200], 213
    fused = torch.randn(n, 8, 64, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    got = []
    for bound in (200, None):
        case = make(lengths, new, heads=4, kv_heads=2, dim=64, dtype=dtype, seed=8, bounds=False, max_query=bound, max_length=300)
        flag = torch.zeros(1, dtype=torch.int32).cuda()
        q = install_tokens(case.batch, 0, fused[:, :4], fused[:, 4:6], fused[:, 6:], Rotary.build(64, 1e4), error_flag=flag)
        assert int(flag) == 0
        got.append([q, *(codes_of(x) for x in (*case.pool, *case.scales))])
    assert all(torch.equal(x, y) for x, y in zip(*got))


@pytest.mark.parametrize("many", [False, True])
def test_falling_query_starts_are_left_out(many):
    """Requests that start before an earlier one are not stored, and not answered."""
    count = 150 if many else 3
    case = make([30] * count, [4] * count, dim=64, seed=15)
    qs = torch.arange(count + 1, dtype=torch.int32) * 4
    qs[1], qs[2] = 8, 4  # request 0 has rows 0 to 7, 1 none that may be had, 2 starts before 1
    qs = qs.cuda()
    old = case.batch
    batch = QueryBatch(old.rows, qs, old._keep[1], max_length=30, max_query=8, request_stride=old.c.request_stride)
    before = [codes_of(x).clone() for x in (*case.pool, *case.scales)]
    n = case.tokens
    x = torch.randn(n, 8, 64, generator=torch.Generator().manual_seed(3)).to(BF16).cuda()
    q, out = torch.full((n, 4, 64), 7.0, dtype=BF16).cuda(), torch.full((n, 4, 64), 7.0, dtype=BF16).cuda()
    for error in range(2):
        flag = torch.zeros(1, dtype=torch.int32).cuda()
        if error == 0:
            install_tokens(batch, 0, x[:, :4], x[:, 4:6], x[:, 6:], Rotary.build(64, 1e4), out=q, error_flag=flag)
        else:
            paged_attention(batch, 0, x[:, :4], out=out, error_flag=flag)
        assert int(flag) == ERROR_REQUEST
    mine = torch.zeros(before[0].shape[1], dtype=torch.bool)
    mine[torch.cat([case.slots[b] for b in [0, *range(3, count)]])] = True
    for a, b in zip(case.pool, before):
        assert torch.equal(codes_of(a)[:, ~mine.cuda()], b[:, ~mine.cuda()])
    assert (q[:8] != 7.0).any() and (out[:8] != 7.0).any()
    if many:
        assert (q[12:] != 7.0).flatten(1).any(1).all() and (out[12:] != 7.0).flatten(1).any(1).all()


def test_nothing_to_do():
    case = make([20, 30], [0, 0], heads=2, kv_heads=2, dim=64, seed=1)
    before = [codes_of(x).clone() for x in (*case.pool, *case.scales)]
    x = torch.zeros(0, 6, 64, dtype=BF16).cuda()
    q = install_tokens(case.batch, 0, x[:, :2], x[:, 2:4], x[:, 4:], Rotary.build(64, 1e4))
    assert paged_attention(case.batch, 0, q).shape == (0, 2, 64)
    y = torch.full((3, 6, 64), 2.0, dtype=BF16).cuda()  # rows of no request
    out = torch.full((3, 2, 64), 5.0, dtype=BF16).cuda()
    install_tokens(case.batch, 0, y[:, :2], y[:, 2:4], y[:, 4:], Rotary.build(64, 1e4), out=out)
    paged_attention(case.batch, 0, y[:, :2], out=out)
    assert (out == 5.0).all()
    empty = torch.zeros(0, dtype=torch.int32).cuda()
    none = QueryBatch(case.batch.rows, torch.zeros(1, dtype=torch.int32).cuda(), empty, max_length=10)
    install_tokens(none, 0, y[:, :2], y[:, 2:4], y[:, 4:], Rotary.build(64, 1e4), out=out)
    paged_attention(none, 0, y[:, :2], out=out)
    plain = query_cases.make([20], [1], heads=2, kv_heads=2, dim=64, seed=1)
    assert quantize_tokens(QueryBatch(plain.batch.rows, torch.zeros(1, dtype=torch.int32).cuda(), empty, max_length=10), none).numel() == 0
    assert (out == 5.0).all() and all(torch.equal(codes_of(a), b) for a, b in zip((*case.pool, *case.scales), before))


@pytest.mark.parametrize("new", [1, 50])
def test_fp32_weights(new):
    """Asked for, they leave the result's own rounding and fp32 sums alone."""
    case = make([300], [new], heads=4, kv_heads=2, dim=128, dtype=BF16, seed=6)
    out = paged_attention(case.batch, 0, case.q.cuda(), fp32_weights=True)
    for h in range(4):
        from oracle import queries
        want, _, mag = queries.attention(case.q[:, h], case.k[0, case.slots[0], h // 2], case.v[0, case.slots[0], h // 2], scale=128 ** -0.5)
        d = queries.score_error(case.q[:, h], case.k[0, case.slots[0], h // 2], scale=128 ** -0.5)
        tol = 2.0 ** -8 * want.abs() + mag * (4 * d + 316 * 2.0 ** -23)
        assert ((out[:, h].double().cpu() - want).abs() - tol).max() <= 0


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_long_pages_and_shared_heads(dtype):
    """Pages of 512 tokens, whose rows are read twice, and keys and values that all heads share (a stride of zero)."""
    case = make([700], [690], heads=2, kv_heads=2, dim=128, dtype=dtype, page=512, seed=4)
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(690, n, 128, generator=g).to(dtype).cuda() for n in (2, 1, 1))
    spin = Rotary.build(128, 1e4)
    install_tokens(case.batch, 0, q, k.expand(-1, 2, -1), v.expand(-1, 2, -1), spin)
    shared = [codes_of(x).clone() for x in (*case.pool, *case.scales)]
    again = make([700], [690], heads=2, kv_heads=2, dim=128, dtype=dtype, page=512, seed=4)
    install_tokens(again.batch, 0, q, k.expand(-1, 2, -1).contiguous(), v.expand(-1, 2, -1).contiguous(), spin)
    assert all(torch.equal(codes_of(a), b) for a, b in zip((*again.pool, *again.scales), shared))
    values = oracle.values(codes_of(case.pool[1]).cpu(), codes_of(case.scales[1]).cpu().int() - 127, 512)[0, case.slots[0][10:]]
    want = v.double().cpu().expand(-1, 2, -1)
    assert ((values - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** -10 * max(float(want.abs().max()), 0.2) / 224).all()




@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("sections", [None, (24, 20, 20)])
def test_long_prompts_store_what_their_chunks_do(sections, quantized, dtype):
    """A prompt of 2500 tokens at once, its queries rotated in place, against chunks of 160 (whole pages): the same bits."""
    heads, kv, dim, n, page = 16, 2, 256, 2500, 32
    fused = torch.randn(n, heads + 2 * kv, dim, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    spin = Rotary.build(128, 1e4, sections=sections)
    places = torch.randint(0, 5000, (n,) if sections is None else (3, n), generator=torch.Generator().manual_seed(4)).cuda()
    got = []
    for step in (n, 160):
        case = (make if quantized else query_cases.make)([n], [n], heads=heads, kv_heads=kv, dim=dim, dtype=dtype, page=page, seed=5)
        rows = case.batch.rows
        x = fused.clone()
        for t in range(0, n, step):
            part = x[t:t + step]
            m = len(part)
            batch = QueryBatch(rows, torch.tensor([0, m], dtype=torch.int32).cuda(),
                               torch.tensor([t + m], dtype=torch.int32).cuda(), request_stride=n, max_length=n)
            flag = torch.zeros(1, dtype=torch.int32).cuda()
            install_tokens(batch, 0, part[:, :heads], part[:, heads:heads + kv], part[:, heads + kv:], spin,
                           positions=places[..., t:t + m].contiguous(), out=part[:, :heads], error_flag=flag)
            assert int(flag) == 0
        assert torch.equal(x[:, heads:], fused[:, heads:])
        got.append([x, *(rows.keep[:2] if not quantized else [codes_of(y) for y in (*case.pool, *case.scales)])])
    for a, b in zip(*got):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    # A turn keeps the lengths: an element is off by half a step, its square by twice that share, all else by far less.
    before, after = (x[:, :heads].double().cpu() for x in (fused, got[0][0]))
    assert not torch.equal(before, after)
    size = before.square().sum(-1)
    assert ((after.square().sum(-1) - size).abs() <= 1.01 * torch.finfo(dtype).eps * size).all()
