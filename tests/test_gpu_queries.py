"""GPU: queries on a paged cache against the 64-bit oracle, where they can go wrong."""

from __future__ import annotations

import math

import pytest
import torch

from cachebridge_amd.online.queries import (ERROR_CACHE_ROW, ERROR_REQUEST, ERROR_TARGET_ROW, QueryBatch, Rotary,
                                            add_key_weights, evict_tokens, install_tokens, paged_attention)
from cachebridge_amd.plan import rows_from_layers, rows_from_stacked
from oracle import queries as oracle

from .query_cases import check_attention, check_weights, make

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def attend(case, **kw):
    out, lse = paged_attention(case.batch, 0, case.q.cuda(), return_lse=True, **kw)
    return out, lse


# lengths, new tokens, (heads, kv heads)
SHAPES = {
    "one": ([1], [1], (2, 1)),
    "step": ([5, 130, 1, 64, 257], [1] * 5, (8, 2)),
    "step-wide": ([700, 33], [1, 1], (48, 1)),
    "question": ([37, 300], [37, 5], (4, 2)),
    "odd-group": ([75, 18], [40, 18], (15, 3)),
    "prompt": ([200], [200], (3, 3)),
    "empty": ([0, 40, 0, 17], [0, 3, 0, 17], (4, 2)),
    "no-new": ([50, 60], [0, 2], (4, 4)),
    "long": ([2100], [3], (4, 1)),
    "chunk-long": ([1500], [150], (4, 2)),
    "wide": ([420, 1, 300], [300, 1, 130], (4, 2)),
    "wide-long": ([1300], [260], (6, 2)),
    "wide-odd": ([333], [333], (5, 1)),
}


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_attention_causal(shape, dim, dtype):
    lengths, new, (heads, kv) = SHAPES[shape]
    case = make(lengths, new, heads=heads, kv_heads=kv, dim=dim, dtype=dtype, seed=len(shape) + dim)
    check_attention(case, *attend(case))


MASKS = {
    "full": dict(causal=False),
    "window1": dict(window=1),
    "window7": dict(window=7),
    "window64": dict(window=64),
    "window100-full": dict(window=100, causal=False),
    "prefix": dict(prefix=[50, 0, 33]),
    "sinks": dict(prefix=[4, 300, 33], window=20),
    "cap": dict(cap=5.0),
    "bias": dict(slopes=True),
    "all": dict(cap=3.0, slopes=True, prefix=[70, 9, 40], window=40, scale=0.3),
}


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 128), (BF16, 256), (FP16, 128), (FP32, 64)])
@pytest.mark.parametrize("mask", list(MASKS))
@pytest.mark.parametrize("new", [[1, 1, 1], [90, 7, 33], [180, 290, 33]])
def test_attention_and_weights_masks(new, mask, dtype, dim):
    case = make([190, 301, 33], new, heads=8, kv_heads=2, dim=dim, dtype=dtype, seed=3)
    how = dict(MASKS[mask])
    dev = {}
    if how.get("prefix"):
        dev["prefix_lengths"] = torch.tensor(how["prefix"], dtype=torch.int32).cuda()
    if how.get("slopes"):
        how["slopes"] = 2.0 ** -torch.arange(1, 9).float()
        dev["slopes"] = how["slopes"].cuda()
    kw = {k: v for k, v in how.items() if k not in ("prefix", "slopes")}
    out, lse = attend(case, **kw, **dev)
    check_attention(case, out, lse, **how)
    before = torch.rand(3, 301).cuda()
    after = before.clone()
    add_key_weights(case.batch, 0, case.q.cuda(), lse, after, **kw, **dev)
    check_weights(case, before, after, lse, **how)


@pytest.mark.parametrize("dim", [2, 30, 48, 80, 96, 130, 192, 320, 512])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_attention_and_weights_other_head_sizes(dim, dtype):
    case = make([70, 19], [20, 1], heads=4, kv_heads=2, dim=dim, dtype=dtype, seed=dim)
    out, lse = attend(case)
    check_attention(case, out, lse)
    before = torch.zeros(2, 80).cuda()
    after = before.clone()
    add_key_weights(case.batch, 0, case.q.cuda(), lse, after)
    check_weights(case, before, after, lse)


@pytest.mark.parametrize("index", ["table", "offsets", "i32", "i64", "identity"])
@pytest.mark.parametrize("page", [1, 16, 24])
def test_index_kinds(index, page):
    case = make([100, 37, 5], [9, 1, 5], dim=128, index=index, page=page, layers=2, seed=4, start=48)
    out, lse = paged_attention(case.batch, 1, case.q.cuda(), return_lse=True)
    check_attention(case, out, lse, layer=1)
    before = torch.zeros(3, 100).cuda()
    after = before.clone()
    add_key_weights(case.batch, 1, case.q.cuda(), lse, after)
    check_weights(case, before, after, lse, layer=1)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_many_ragged_requests(dtype):
    """More requests than lanes: query tiles are found by a search."""
    g = torch.Generator().manual_seed(9)
    lengths = torch.randint(0, 90, (150,), generator=g).tolist()
    new = [min(n, int(torch.randint(0, 4, (1,), generator=g))) for n in lengths]
    big = next(i for i, n in enumerate(lengths) if i > 70 and n > 60)
    new[big] = 60
    case = make(lengths, new, dim=64, dtype=dtype, seed=5)
    out, lse = attend(case)
    check_attention(case, out, lse)
    before = torch.zeros(150, max(lengths)).cuda()
    after = before.clone()
    add_key_weights(case.batch, 0, case.q.cuda(), lse, after)
    check_weights(case, before, after, lse)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("new,dim", [(1, 64), (20, 64), (150, 64), (20, 128), (150, 128), (20, 256), (150, 256)])
@pytest.mark.parametrize("heads", [4, 8])
def test_what_is_not_seen_never_counts(new, dim, heads, dtype):
    """Infinities and NaN behind the mask, past the length and in pages of nobody leave every row as it was."""
    case = make([170, 170], [new, new], heads=heads, dim=dim, dtype=dtype, seed=6)
    want, want_lse = attend(case, window=9)
    k, v = case.pool
    inside = torch.zeros(k.shape[1], dtype=torch.bool)
    for b in range(2):
        inside[case.slots[b]] = True
    for x, bad in ((k, math.nan), (v, math.nan)):
        x[:, ~inside.cuda()] = bad
    seen = 170 - new - 8  # the first token any new one sees
    for at, bad in ((0, math.inf), (1, -math.inf), (2, math.nan)):
        if at < seen:
            k[0, case.slots[0][at]] = bad
            v[0, case.slots[0][at]] = bad
    got, got_lse = attend(case, window=9)
    assert torch.equal(got, want) and torch.equal(got_lse, want_lse)
    # A value that only the last rows see: earlier rows stay, those rows get it.
    if new > 1:
        v[0, case.slots[0][169]] = math.inf
        v[0, case.slots[1][168], :, 3] = math.nan
        got, got_lse = attend(case, window=9)
        assert torch.equal(got_lse, want_lse)
        assert torch.equal(got[:new - 1], want[:new - 1])
        assert torch.isposinf(got[new - 1]).all()
        assert torch.equal(got[new:2 * new - 2], want[new:2 * new - 2])
        assert torch.isnan(got[2 * new - 2:, :, 3]).all()
        keep = [d for d in range(dim) if d != 3]
        assert torch.equal(got[2 * new - 2:, :, keep], want[2 * new - 2:, :, keep])


@pytest.mark.parametrize("new", [30, 300])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_infinite_values_of_both_signs_meet_as_nan(dim, new):
    case = make([30 + new], [new], dim=dim, seed=2)
    _, v = case.pool
    want, _ = attend(case)
    v[0, case.slots[0][40], 0, 5] = math.inf
    v[0, case.slots[0][50], 0, 5] = -math.inf
    got, _ = attend(case)
    assert torch.equal(got[:10], want[:10])
    assert torch.isposinf(got[10:20, :2, 5]).all() and torch.isnan(got[20:, :2, 5]).all()
    assert torch.equal(got[:, 2:], want[:, 2:])
    keep = [d for d in range(dim) if d != 5]
    assert torch.equal(got[..., keep], want[..., keep])


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, BF16), (128, FP16), (96, FP16)])
@pytest.mark.parametrize("how", [{}, dict(window=300, prefix=[37, 8]), dict(cap=4.0, causal=False)])
def test_large_launches(how, dim, dtype):
    """Enough scores for eight waves a workgroup; a sample of the rows against the oracle, values that are not finite
    and bad rows among them."""
    new, heads, lengths = [700, 40], 16, [2400, 500]
    case = make(lengths, new, heads=heads, kv_heads=2, dim=dim, dtype=dtype, seed=21, index="i32")
    how = dict(how)
    prefix = how.pop("prefix", None)
    more = {} if prefix is None else dict(prefix_lengths=torch.tensor(prefix, dtype=torch.int32).cuda())
    assert sum(new) * heads * (lengths[0] if prefix else min(lengths[0], how.get("window", 1 << 30))) >= 24 << 20
    out, lse = attend(case, **how, **more)
    u = torch.finfo(dtype).eps / 2
    def check(out, lse):
        for b, at, m in ((0, 0, 700), (1, 700, 40)):
            rows = sorted({0, 1, 31, 63, 64, 127, 128, 255, 256, 300, 511, 640, 699} & set(range(m)))
            for h in (0, 7, 8, 15):
                k, v = (x[0, case.slots[b], h // 8].double() for x in (case.k, case.v))
                seen = oracle.visible(lengths[b], m, **{x: y for x, y in how.items() if x != "cap"}, prefix=prefix[b] if prefix else 0)[rows]
                q = case.q[at:at + m, h].double()
                x = oracle.scores(q, k, scale=dim ** -0.5, cap=how.get("cap", 0.0))[rows].masked_fill(~seen, -math.inf)
                w = torch.softmax(x, 1)
                want, mag = w @ v, w @ v.abs()
                # The bounds of query_cases.check_attention.
                d = oracle.score_error(q, k, scale=dim ** -0.5) + 2.0 ** -21 * how.get("cap", 0.0)
                tol = u * want.abs() + u * mag + mag * (4 * d + (lengths[b] + 16) * 2.0 ** -23) + 2.0 ** -25 * lengths[b] * v.abs().max()
                got = out[at:at + m, h].double().cpu()[rows]
                assert ((got - want).abs() - tol).max() <= 0, (b, h)
                z = torch.logsumexp(x, 1)
                assert ((lse[at:at + m, h].double().cpu()[rows] - z).abs() - (d + (lengths[b] + 16) * 2.0 ** -23 + 2.0 ** -22 * z.abs())).max() <= 0
    check(out, lse)
    if how.get("causal", True) and prefix is None:
        _, v = case.pool
        v[0, case.slots[0][2100], 0, 5] = math.inf   # new token 400 and later ones see it
        v[0, case.slots[0][2200], 1, 6] = math.nan
        got, _ = attend(case, **how, **more)
        assert torch.equal(got[:400], out[:400]) and torch.equal(got[700:], out[700:])
        assert torch.isposinf(got[400:700, :8, 5]).all() and torch.isnan(got[500:700, 8:, 6]).all()
        assert torch.equal(got[400:500, 8:], out[400:500, 8:])
        keep = [d for d in range(dim) if d not in (5, 6)]
        assert torch.equal(got[..., keep], out[..., keep])


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_large_scores(dtype):
    """Rows whose maximum grows from tile to tile, by little and by much, and scores far from zero."""
    case = make([600], [70], dim=64, dtype=dtype, seed=8, spread=1.0)
    k = case.pool[0]
    grow = torch.linspace(0.1, 12.0, 600)
    case.k[0, case.slots[0]] = (case.q[-1, 0].float() * grow[:, None, None] * 0.5).to(dtype).expand(600, 2, 64)
    k.copy_(case.k)
    check_attention(case, *attend(case))
    check_attention(case, *attend(case, scale=-2.0), scale=-2.0)
    check_attention(case, *attend(case, scale=0.0), scale=0.0)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("new", [1, 40, 600])
def test_many_small_weights_keep_their_sum(new, dtype):
    """One token takes nearly all the weight; 65535 others have 1.02 * 2^-25 of its."""
    n, dim, w = 65536, 64, 1.02 * 2.0 ** -25
    k, v = torch.zeros(1, n, 1, dim, dtype=dtype).cuda(), torch.ones(1, n, 1, dim, dtype=dtype).cuda()
    k[0, 0], v[0, 0] = 1, 0
    start, lengths = torch.tensor([0, new]).int().cuda(), torch.tensor([n]).int().cuda()
    batch = QueryBatch(rows_from_stacked(k, v), start, lengths, max_length=n)
    out = paged_attention(batch, 0, torch.ones(new, 1, dim, dtype=dtype).cuda(), scale=-math.log(w) / dim, causal=False)
    want = (n - 1) * w / (1 + (n - 1) * w)
    # Scores of 17.3 in fp32: two roundings of 2^-24 of them, times as much again for the exponential. A weight's
    # rounding: half a step of the type; fp16 weights of 1.02 * 2^-17 (they count from 2^8) have a step of 2^-24.
    half = torch.finfo(dtype).eps / 2
    weight = {BF16: half, FP16: 2.0 ** -25 / (1.02 * 2.0 ** -17), FP32: half}[dtype]
    # fp32 sums of 65536 terms in chains of at most 65536 / 16, each step off by 2^-24.
    tolerance = weight + half + 4 * 17.4 * 2.0 ** -24 + 4096 * 2.0 ** -24
    assert ((out.double() / want - 1).abs() <= tolerance).all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_rows_of_no_request_and_strides(dtype):
    case = make([40, 90], [6, 11], heads=6, kv_heads=2, dim=128, dtype=dtype, seed=11, padding=5)
    wide = torch.full((22, 10, 128), 7.0, dtype=dtype).cuda()
    wide[:, 2:8] = case.q.cuda()
    out = torch.full((6, 22, 128), 3.0, dtype=dtype).cuda().transpose(0, 1)
    got, lse = paged_attention(case.batch, 0, wide[:, 2:8], out=out, return_lse=True)
    assert got is out
    check_attention(case, out[:17], lse[:17])
    assert (out[17:] == 3.0).all()
    # Alignment of two elements, not 16 bytes.
    odd = torch.zeros(22 * 6 * 128 + 1, dtype=dtype).cuda()[1:].view(22, 6, 128)
    odd.copy_(case.q)
    again = paged_attention(case.batch, 0, odd, out=torch.empty(22 * 6 * 128 + 1, dtype=dtype).cuda()[1:].view(22, 6, 128))
    check_attention(case, again[:17])
    w1, w2 = torch.zeros(2, 90).cuda(), torch.zeros(2, 200).cuda()[:, :90]
    add_key_weights(case.batch, 0, wide[:, 2:8], lse, w1)
    add_key_weights(case.batch, 0, odd, lse, w2)
    check_weights(case, torch.zeros(2, 90), w1, lse)
    check_weights(case, torch.zeros(2, 90), w2, lse)


def test_unaligned_pool():
    """Pool rows that do not start at 16 bytes: stacked buffers at an odd offset."""
    case = make([50], [7], dim=64, seed=12)
    k, v = (torch.zeros(x.numel() + 1, dtype=x.dtype).cuda()[1:].view(x.shape).copy_(x) for x in case.pool)
    table = torch.cat([torch.tensor([int(s) // 16 for s in case.slots[0][::16]], dtype=torch.int32)]).cuda()
    batch = QueryBatch(rows_from_stacked(k, v, block_table=table, page_size=16), torch.tensor([0, 7]).int().cuda(),
                       torch.tensor([50]).int().cuda(), max_length=50)
    out, lse = paged_attention(batch, 0, case.q.cuda(), return_lse=True)
    check_attention(case, out, lse)


def test_pool_of_one_buffer_per_layer():
    case = make([90, 20], [4, 20], dim=128, layers=3, seed=13)
    ks, vs = (list(x.clone().unbind(0)) for x in case.pool)
    old = case.batch
    rows = rows_from_layers([x.clone() for x in ks], [x.clone() for x in vs], block_table=old.rows.keep[-1], page_size=16)
    batch = QueryBatch(rows, *old._keep[:2], max_length=90, max_query=20, request_stride=old.c.request_stride)
    for layer in (0, 2):
        out, lse = paged_attention(batch, layer, case.q.cuda(), return_lse=True)
        check_attention(case, out, lse, layer=layer)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_bad_rows_and_requests_are_left_out_and_flagged(dtype):
    case = make([60, 60, 60, 60], [5, 5, 5, 5], dim=64, dtype=dtype, seed=14, index="i32")
    good, good_lse = attend(case)
    flag = torch.zeros(1, dtype=torch.int32).cuda()
    paged_attention(case.batch, 0, case.q.cuda(), error_flag=flag)
    assert int(flag) == 0
    old = case.batch
    index = old.rows.keep[-1].clone()
    index[3] = -1               # request 0, token 3
    index[60 + 10] = 1 << 30    # request 1, token 10
    rows = rows_from_stacked(*case.pool, index=index)
    qs, ln, off = (t.clone() for t in old._keep)
    ln[2] = 61                  # past max_length
    off[3] = 210                # its tokens run past the index: 30 are there
    batch = QueryBatch(rows, qs, ln, offsets=off, max_length=60, max_query=5)
    out = torch.full_like(case.q, 9.0).cuda()
    w = torch.zeros(4, 60).cuda()
    _, lse = paged_attention(batch, 0, case.q.cuda(), out=out, return_lse=True, error_flag=flag)
    assert int(flag) == ERROR_CACHE_ROW | ERROR_REQUEST
    assert (out[10:15] == 9.0).all()
    fl2 = torch.zeros(1, dtype=torch.int32).cuda()
    add_key_weights(batch, 0, case.q.cuda(), good_lse, w, error_flag=fl2)
    assert int(fl2) == ERROR_CACHE_ROW | ERROR_REQUEST
    assert w[0, 3] == 0 and w[1, 10] == 0 and (w[2] == 0).all() and (w[3, 30:] == 0).all() and (w[0, :3] > 0).all()
    # The first two requests as if the bad tokens were hidden.
    for b, hole in ((0, 3), (1, 10)):
        for h in range(case.heads):
            q, kk, vv = case.q[5 * b:5 * b + 5, h].double(), case.k[0, case.slots[b], h // 2].double(), case.v[0, case.slots[b], h // 2].double()
            x = oracle.scores(q, kk, scale=0.125)
            seen = oracle.visible(60, 5)
            seen[:, hole] = False
            want = torch.softmax(x.masked_fill(~seen, -math.inf), 1) @ vv
            assert (out[5 * b:5 * b + 5, h].double().cpu() - want).abs().max() < 2 ** -6


def test_falling_query_starts_are_refused_on_the_device():
    case = make([30, 30, 30], [4, 4, 4], dim=64, seed=15)
    qs = torch.tensor([0, 8, 4, 12], dtype=torch.int32).cuda()
    batch = QueryBatch(case.batch.rows, qs, case.batch._keep[1], max_length=30, max_query=8,
                       request_stride=case.batch.c.request_stride)
    flag = torch.zeros(1, dtype=torch.int32).cuda()
    paged_attention(batch, 0, case.q.cuda(), error_flag=flag)
    assert int(flag) == ERROR_REQUEST


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("dim,rotary", [(128, 128), (128, 64), (64, 64), (96, 96), (96, 48), (80, 20), (256, 256), (2, 2), (510, 6)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_install(dim, rotary, interleaved, dtype):
    case = make([70, 16, 1, 33], [7, 16, 1, 0], heads=6, kv_heads=2, dim=dim, dtype=dtype, layers=2, seed=dim + rotary)
    g = torch.Generator().manual_seed(1)
    fused = torch.randn(24, 10, dim, generator=g).to(dtype)
    q, k, v = fused[:, :6], fused[:, 6:8], fused[:, 8:]
    spin = Rotary.build(rotary, 1e4, dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32),
                        interleaved=interleaved)
    before = [x.clone() for x in case.pool]
    fd = fused.cuda()
    got = install_tokens(case.batch, 1, fd[:, :6], fd[:, 6:8], fd[:, 8:], spin)
    pos = torch.cat([torch.arange(n - m, n) for n, m in zip(case.lengths, case.new)])
    turned = dict(magnitude=spin.magnitude, interleaved=interleaved)
    inv = spin.inv_freq.cpu()
    u = torch.finfo(dtype).eps / 2
    # One rounding of the result; cosine, sine and the two products are fp32 (8 roundings of the pair's size).
    def near(a, x):
        want = oracle.rotate(x, pos, inv, **turned)
        size = x.double().abs().amax(-1, keepdim=True) * 2 * spin.magnitude
        assert ((a.double().cpu() - want).abs() - (u * want.abs() + 2.0 ** -21 * size + 2.0 ** -25)).max() <= 0
    near(got, q)
    assert torch.equal(fd.cpu(), fused)
    rows = torch.cat([s[n - m:] for s, n, m in zip(case.slots, case.lengths, case.new)])
    kd, vd = case.pool
    near(kd[1, rows], k)
    assert torch.equal(vd[1, rows].cpu(), v)
    rest = torch.ones(kd.shape[1], dtype=torch.bool)
    rest[rows] = False
    for x, y in zip(case.pool, before):
        assert torch.equal(x[0], y[0]) and torch.equal(x[1][rest.cuda()], y[1][rest.cuda()])
    # In place, and with positions given.
    far = torch.randint(0, 1 << 30, (24,), generator=g)
    qd = fd[:, :6]
    assert install_tokens(case.batch, 1, qd, fd[:, 6:8], fd[:, 8:], spin, positions=far.cuda(), out=qd) is qd
    pos = far
    near(qd, q)
    near(kd[1, rows], k)
    install_tokens(case.batch, 1, fused.cuda()[:, :6], fd[:, 6:8], fd[:, 8:], spin, positions=far.int().cuda(), out=qd)
    near(qd, q)


def test_install_leaves_bad_rows_and_requests_out():
    case = make([40, 40, 40], [2, 2, 2], heads=2, kv_heads=1, dim=64, seed=20, index="i64", padding=3)
    index = case.batch.rows.keep[-1].clone()
    index[39] = case.pool[0].shape[1]
    index[40 + 38] = -5
    ln = case.batch._keep[1].clone()
    ln[2] = 1
    batch = QueryBatch(rows_from_stacked(*case.pool, index=index), case.batch._keep[0], ln, offsets=case.batch._keep[2],
                       max_length=40, max_query=2)
    before = [x.clone() for x in case.pool]
    q = case.q.cuda()
    out = torch.full_like(q, 5.0)
    kv = torch.randn(9, 1, 64).to(BF16).cuda()
    flag = torch.zeros(1, dtype=torch.int32).cuda()
    install_tokens(batch, 0, q, kv, kv, Rotary.build(64, 1e4), out=out, error_flag=flag)
    assert int(flag) == ERROR_TARGET_ROW | ERROR_REQUEST
    assert (out[4:] == 5.0).all() and (out[:4] != 5.0).any()
    stored = torch.tensor([int(case.slots[0][38]), int(case.slots[1][39])])
    assert torch.equal(case.pool[1][0, stored].cpu(), kv[[0, 3]].cpu())
    rest = torch.ones(before[0].shape[1], dtype=torch.bool)
    rest[stored] = False
    for x, y in zip(case.pool, before):
        assert torch.equal(x[0][rest.cuda()], y[0][rest.cuda()])


def _evict_case(lengths, budget, first, last, weights, *, dtype=BF16, kv_heads=2, dim=64, layers=3, seed=0):
    case = make(lengths, [1 if n else 0 for n in lengths], heads=kv_heads, kv_heads=kv_heads, dim=dim, dtype=dtype, layers=layers, seed=seed)
    pages = [-(-min(n, budget) // 16) for n in lengths]
    k = torch.zeros(layers, (sum(pages) + 1) * 16, kv_heads, dim, dtype=dtype).cuda()
    v = torch.zeros_like(k)
    order = torch.randperm(sum(pages) + 1)
    offsets = torch.tensor([0] + pages).cumsum(0)[:-1] * 16
    target = QueryBatch(rows_from_stacked(k, v, block_table=order[:sum(pages)].int().cuda(), page_size=16),
                        *case.batch._keep[:2], max_length=max(lengths), offsets=offsets.cuda())
    kept = evict_tokens(case.batch, weights.cuda(), target, budget=budget, first=first, last=last)
    wt = weights.tolist()
    where = []
    for b, n in enumerate(lengths):
        want = oracle.keep(wt[b][:n], budget, first, last)
        assert int(kept.lengths[b]) == len(want)
        assert kept.tokens[b].tolist() == want + [-1] * (budget - len(want))
        got_w = kept.weights[b].cpu()
        assert torch.equal(torch.nan_to_num(got_w[:len(want)], 123.0), torch.nan_to_num(weights[b, want], 123.0))
        assert (got_w[len(want):] == 0).all()
        t = torch.arange(len(want))
        rows = order[int(offsets[b]) // 16 + t // 16] * 16 + t % 16
        where.append(rows)
        for got, src in ((k, case.k), (v, case.v)):
            assert torch.equal(got[:, rows].cpu(), src[:, case.slots[b][want]] if want else src[:, :0])
    rest = torch.ones(k.shape[1], dtype=torch.bool)
    rest[torch.cat(where)] = False
    assert (k[:, rest.cuda()] == 0).all() and (v[:, rest.cuda()] == 0).all()


@pytest.mark.parametrize("budget,first,last", [(1, 0, 0), (1, 0, 1), (10, 4, 6), (40, 4, 8), (64, 0, 0), (200, 3, 3), (333, 0, 9)])
def test_evict(budget, first, last):
    g = torch.Generator().manual_seed(budget)
    lengths = [333, 1, 64, 0, 200, 41]
    _evict_case(lengths, budget, first, last, torch.rand(6, 333, generator=g).square(), seed=budget)


@pytest.mark.parametrize("kind", ["zeros", "few", "signs", "special", "steps"])
def test_evict_ties_and_special_weights(kind):
    g = torch.Generator().manual_seed(3)
    w = torch.rand(2, 1500, generator=g)
    if kind == "zeros":
        w = torch.where(w < 0.9, torch.zeros(()), w)
        w[0, ::3] *= -0.0  # both zeros are one weight
    elif kind == "few":
        w = (w * 3).floor()
    elif kind == "signs":
        w = (w - 0.5) * torch.where(torch.rand(2, 1500, generator=g) < 0.5, 1e-40, 0.1)  # subnormals among them
    elif kind == "special":
        w[0, 5], w[0, 77], w[0, 700], w[1, 9] = math.nan, math.inf, -math.inf, math.nan
        w[1, 100:200] = math.inf
    else:
        w = 1.0 + (w * 4).floor() * 2.0 ** -23
    _evict_case([1500, 1300], 150, 2, 5, w, seed=1)


@pytest.mark.parametrize("dtype,kv_heads,dim", [(FP32, 1, 2), (FP16, 3, 6), (BF16, 1, 30), (FP32, 3, 66), (FP16, 8, 128)])
def test_evict_row_sizes(dtype, kv_heads, dim):
    w = torch.rand(2, 120, generator=torch.Generator().manual_seed(dim))
    _evict_case([120, 77], 50, 4, 4, w, dtype=dtype, kv_heads=kv_heads, dim=dim)


@pytest.mark.parametrize("n", [17000, 66000, 70001])
def test_evict_long_history(n):
    w = torch.rand(1, n, generator=torch.Generator().manual_seed(8))
    _evict_case([n], 5000, 4, 64, w, kv_heads=1, dim=8, layers=1)


def test_evict_bad_rows_are_flagged():
    case = make([50, 50], [1, 1], heads=2, kv_heads=2, dim=64, index="i32", seed=2)
    index = case.batch.rows.keep[-1].clone()
    index[7] = -1
    qs, ln, off = case.batch._keep
    bad_len = ln.clone()
    bad_len[1] = 51
    batch = QueryBatch(rows_from_stacked(*case.pool, index=index), qs, bad_len, offsets=off, max_length=50)
    k, v = torch.zeros(1, 64, 2, 64, dtype=BF16).cuda(), torch.zeros(1, 64, 2, 64, dtype=BF16).cuda()
    target = QueryBatch(rows_from_stacked(k, v), qs, ln, request_stride=32, max_length=50)
    flag = torch.zeros(1, dtype=torch.int32).cuda()
    w = torch.arange(100, dtype=torch.float32).view(2, 50).flip(1).cuda()
    kept = evict_tokens(batch, w, target, budget=20, error_flag=flag)
    assert int(flag) == ERROR_CACHE_ROW | ERROR_REQUEST
    assert kept.tokens[0].tolist() == list(range(20))
    assert (k[0, 7] == 0).all() and torch.equal(k[0, 8].cpu(), case.k[0, case.slots[0][8]])
    assert (k[0, 32:] == 0).all()


def test_evict_keeps_nothing_of_a_request_outside_the_bounds():
    case = make([50, 50, 50], [1, 1, 1], heads=2, kv_heads=2, dim=64, index="i32", seed=2)
    qs, ln, off = case.batch._keep
    ln = ln.clone()
    ln[0], ln[2] = -1, 51
    batch = QueryBatch(rows_from_stacked(*case.pool, index=case.batch.rows.keep[-1]), qs, ln, offsets=off, max_length=50)
    k, v = torch.zeros(1, 96, 2, 64, dtype=BF16).cuda(), torch.zeros(1, 96, 2, 64, dtype=BF16).cuda()
    target = QueryBatch(rows_from_stacked(k, v), qs, ln, request_stride=32, max_length=50)
    for budget in (20, 60):  # fewer than a request has, and more
        torch.full((64, 1 << 10), -7, dtype=torch.int32).cuda()  # what new tensors may be made of
        flag = torch.zeros(1, dtype=torch.int32).cuda()
        kept = evict_tokens(batch, torch.ones(3, 50).cuda(), target, budget=budget, error_flag=flag)
        assert int(flag) & ERROR_REQUEST and kept.lengths.tolist() == [0, min(budget, 50), 0]
        for b in (0, 2):
            assert (kept.tokens[b] == -1).all() and (kept.weights[b] == 0).all()
        # Request 1 has rows 32 to 32 + 49 at most; all others stay.
        assert (k[0, :32] == 0).all() and (k[0, 82:] == 0).all() and (k[0, 32:52] != 0).any()


def _serve(case, spin, fused, weights, stream=None):
    """One pass of all operators: store the new tokens, attend, add weights."""
    h, kv = case.heads, case.kv_heads
    q = install_tokens(case.batch, 0, fused[:, :h], fused[:, h:h + kv], fused[:, h + kv:], spin, stream=stream)
    out, lse = paged_attention(case.batch, 0, q, return_lse=True, stream=stream)
    add_key_weights(case.batch, 0, q, lse, weights, stream=stream)
    return q, out, lse


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (FP32, 64)])
def test_the_operators_together(dtype, dim):
    """Store, attend, weigh, evict, and go on from the kept tokens at their own positions."""
    case = make([150, 90], [9, 1], heads=4, kv_heads=2, dim=dim, dtype=dtype, seed=30)
    fused = torch.randn(10, 8, dim, generator=torch.Generator().manual_seed(4)).to(dtype)
    spin = Rotary.build(dim, 1e4)
    weights = torch.zeros(2, 150).cuda()
    q, out, lse = _serve(case, spin, fused.cuda(), weights)
    case.q, case.k, case.v = q.cpu(), case.pool[0].cpu(), case.pool[1].cpu()
    check_attention(case, out, lse)
    check_weights(case, torch.zeros(2, 150), weights, lse)
    # Each row's weights sum to one over what it sees.
    assert (weights.sum(1).cpu() - torch.tensor([36.0, 4.0])).abs().max() < 36 * 150 * 2.0 ** -22
    k, v = torch.zeros(1, 256, 2, dim, dtype=dtype).cuda(), torch.zeros(1, 256, 2, dim, dtype=dtype).cuda()
    rows = rows_from_stacked(k, v, block_table=torch.randperm(16).int().cuda(), page_size=16)
    qs = torch.tensor([0, 1, 2], dtype=torch.int32).cuda()
    grown = torch.tensor([41, 41], dtype=torch.int32).cuda()
    target = QueryBatch(rows, qs, grown, request_stride=128, max_length=41)
    kept = evict_tokens(case.batch, weights, target, budget=40, first=4, last=8)
    assert kept.lengths.tolist() == [40, 40]
    step = torch.randn(2, 8, dim, generator=torch.Generator().manual_seed(5)).to(dtype)
    sd = step.cuda()
    pos = torch.tensor([150, 90]).cuda()
    q2 = install_tokens(target, 0, sd[:, :4], sd[:, 4:6], sd[:, 6:], spin, positions=pos)
    out2 = paged_attention(target, 0, q2)
    table = rows.keep[-1].cpu().long()
    for b in range(2):
        t = torch.arange(41)
        at = table[b * 8 + t // 16] * 16 + t % 16
        src = case.slots[b][kept.tokens[b].cpu().long()]
        assert torch.equal(k[0, at[:40]].cpu(), case.k[0, src])
        for h in range(4):
            want, _, mag = oracle.attention(q2[b:b + 1, h].cpu(), k[0, at, h // 2].cpu(), v[0, at, h // 2].cpu(), scale=dim ** -0.5)
            u = torch.finfo(dtype).eps / 2
            assert ((out2[b, h].double().cpu() - want[0]).abs() - (u * want[0].abs() + (u + 2.0 ** -16) * mag[0])).max() <= 0


def test_other_stream_and_repeat():
    case = make([500, 90], [9, 30], heads=8, kv_heads=2, dim=128, seed=31)
    fused = torch.randn(39, 12, 128, generator=torch.Generator().manual_seed(4)).to(BF16).cuda()
    spin = Rotary.build(128, 1e6)
    w0 = torch.zeros(2, 500).cuda()
    want = _serve(case, spin, fused, w0)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    w1 = torch.zeros(2, 500).cuda()
    s.wait_stream(torch.cuda.current_stream())
    got = _serve(case, spin, fused, w1, stream=s)
    s.synchronize()
    for a, b in zip((*want, w0), (*got, w1)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dim,dtype", [(128, BF16), (64, FP32)])
def test_captured_graphs_follow_the_lengths(dim, dtype):
    """Two graphs captured from one batch, replayed in turn with eager work between; lengths grow between replays."""
    case = make([1000, 700], [1, 1], heads=8, kv_heads=1, dim=dim, dtype=dtype, seed=32)
    spin = Rotary.build(dim, 1e6)
    fused = torch.randn(2, 10, dim, generator=torch.Generator().manual_seed(4)).to(dtype).cuda()
    ln = case.batch._keep[1]
    ln.copy_(torch.tensor([990, 690]))
    weights = torch.zeros(2, 1000).cuda()
    _serve(case, spin, fused, weights)  # the library loads outside the capture
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = _serve(case, spin, fused, weights)
        graphs.append((g, got))
    for step in range(6):
        ln += 1
        pool = [x.clone() for x in case.pool]
        weights.zero_()
        want = [x.clone() for x in _serve(case, spin, fused, weights)] + [weights.clone()]
        stored = [x.clone() for x in case.pool]
        for x, y in zip(case.pool, pool):
            x.copy_(y)
        weights.zero_()
        torch.cuda.synchronize()
        g, got = graphs[step % 2]
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, (*got, weights)):
            assert torch.equal(a, b), step
        for x, y in zip(case.pool, stored):
            assert torch.equal(x, y)


def test_long_cache_offsets_pass_32_bits():
    """A request's index tokens and the pool's bytes past 2^32: identity rows at the end of a 9 GiB layer."""
    rows, dim = (9 << 30) // (128 * 2), 128
    k = torch.empty(1, rows, 1, dim, dtype=BF16, device="cuda")
    v = torch.empty_like(k)
    g = torch.Generator().manual_seed(3)
    kk, vv = torch.randn(100, dim, generator=g).to(BF16), torch.randn(100, dim, generator=g).to(BF16)
    k[0, rows - 100:, 0], v[0, rows - 100:, 0] = kk.cuda(), vv.cuda()
    q = torch.randn(2, 1, dim, generator=g).to(BF16)
    ln, qs = torch.tensor([100], dtype=torch.int32).cuda(), torch.tensor([0, 2], dtype=torch.int32).cuda()
    batch = QueryBatch(rows_from_stacked(k, v), qs, ln, offsets=torch.tensor([rows - 100]).cuda(), max_length=100)
    out = paged_attention(batch, 0, q.cuda())
    want, _, mag = oracle.attention(q[:, 0], kk, vv, scale=dim ** -0.5)
    assert ((out[:, 0].double().cpu() - want).abs() - (2.0 ** -8 * (want.abs() + mag))).max() <= 0
    # An offset past 2^32 index tokens lies outside the pool: nothing is read, all is flagged.
    flag = torch.zeros(1, dtype=torch.int32).cuda()
    far = QueryBatch(rows_from_stacked(k, v), qs, ln, offsets=torch.tensor([1 << 33]).cuda(), max_length=100)
    out, lse = paged_attention(far, 0, q.cuda(), return_lse=True, error_flag=flag)
    assert int(flag) == ERROR_CACHE_ROW and (out == 0).all() and torch.isneginf(lse).all()


def test_refusals_on_the_gpu():
    case = make([30], [3], dim=64)
    q = case.q.cuda()
    with pytest.raises(ValueError, match="layer"):
        paged_attention(case.batch, 1, q)
    with pytest.raises(ValueError, match="multiple of the KV heads"):
        paged_attention(case.batch, 0, q[:, :3])
    with pytest.raises(ValueError, match="head_dim"):
        paged_attention(case.batch, 0, q[..., :32])
    with pytest.raises(ValueError, match="last dimension"):
        paged_attention(case.batch, 0, q.transpose(1, 2).contiguous().transpose(1, 2))
    with pytest.raises(ValueError, match="window"):
        paged_attention(case.batch, 0, q, window=-1)
    with pytest.raises(ValueError, match="cap"):
        paged_attention(case.batch, 0, q, cap=-1.0)
    with pytest.raises(ValueError, match="scale"):
        paged_attention(case.batch, 0, q, scale=math.inf)
    with pytest.raises(ValueError, match="weights"):
        add_key_weights(case.batch, 0, q, torch.zeros(3, 4).cuda(), torch.zeros(1, 29).cuda())
    with pytest.raises(ValueError, match="lse"):
        add_key_weights(case.batch, 0, q, torch.zeros(4, 3).cuda(), torch.zeros(1, 30).cuda())
    with pytest.raises(ValueError, match="rotary_dim"):
        install_tokens(case.batch, 0, q, q[:, :2], q[:, :2], Rotary.build(66, 1e4))
    with pytest.raises(ValueError, match="budget"):
        evict_tokens(case.batch, torch.zeros(1, 30).cuda(), case.batch, budget=4, first=3, last=2)
    with pytest.raises(ValueError, match="positions"):
        install_tokens(case.batch, 0, q, q[:, :2], q[:, :2], Rotary.build(64, 1e4), positions=torch.zeros(2).long().cuda())
    assert paged_attention(case.batch, 0, q[:0]).shape == (0, 4, 64)


def test_integers_past_32_bits_are_refused():
    case = make([40], [2], heads=2, kv_heads=1, dim=64)
    qs, ln, off = case.batch._keep
    big = 1 << 32
    q = case.q.cuda()
    with pytest.raises(ValueError, match="layer"):
        paged_attention(case.batch, big, q)
    with pytest.raises(ValueError, match="window"):
        paged_attention(case.batch, 0, q, window=big + 5)
    for kw in (dict(max_length=big + 40), dict(max_length=40, max_query=-big), dict(max_length=40, request_stride=1 << 64)):
        with pytest.raises(ValueError, match=list(kw)[-1]):
            QueryBatch(case.batch.rows, qs, ln, **kw)
    with pytest.raises(ValueError, match="budget"):
        evict_tokens(case.batch, torch.zeros(1, 40).cuda(), case.batch, budget=big + 1)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("new", [1, 30, 200])
def test_bounds_far_above_the_lengths(new, dtype):
    case = make([1500, 300, 210], [new, new, min(new, 7)], heads=4, kv_heads=2, dim=64, dtype=dtype, seed=new)
    qs, ln, off = case.batch._keep
    for bound in (1500, 40000, 1 << 20):
        batch = QueryBatch(case.batch.rows, qs, ln, offsets=off, max_length=bound, max_query=new,
                           request_stride=case.batch.c.request_stride)
        out, lse = paged_attention(batch, 0, case.q.cuda(), return_lse=True)
        check_attention(case, out, lse)
