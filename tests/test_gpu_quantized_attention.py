"""GPU: attention over an 8-bit cache against the 64-bit oracle on the values that its codes and scales stand for.

The bounds are those of query_cases.check_attention: e4m3 values times powers of two are exact in every type used here."""

from __future__ import annotations

import math

import pytest
import torch

from cachebridge_amd.online.queries import ERROR_CACHE_ROW, ERROR_REQUEST, QueryBatch, add_key_weights, evict_tokens, paged_attention
from cachebridge_amd.plan import BlockScales, rows_from_stacked
from oracle import queries as oracle

from .quantized_cases import codes_of, make
from .query_cases import check_attention
from .test_gpu_queries import MASKS, SHAPES

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def attend(case, **kw):
    return paged_attention(case.batch, 0, case.q.cuda(), return_lse=True, **kw)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_causal(shape, dim, dtype):
    lengths, new, (heads, kv) = SHAPES[shape]
    case = make(lengths, new, heads=heads, kv_heads=kv, dim=dim, dtype=dtype, seed=len(shape) + dim)
    check_attention(case, *attend(case))


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 128), (BF16, 256), (FP16, 128), (FP32, 64)])
@pytest.mark.parametrize("mask", list(MASKS))
@pytest.mark.parametrize("new", [[1, 1, 1], [90, 7, 33], [180, 290, 33]])
def test_masks(new, mask, dtype, dim):
    case = make([190, 301, 33], new, heads=8, kv_heads=2, dim=dim, dtype=dtype, seed=3)
    how = dict(MASKS[mask])
    dev = {}
    if how.get("prefix"):
        dev["prefix_lengths"] = torch.tensor(how["prefix"], dtype=torch.int32).cuda()
    if how.get("slopes"):
        how["slopes"] = 2.0 ** -torch.arange(1, 9).float()
        dev["slopes"] = how["slopes"].cuda()
    kw = {k: v for k, v in how.items() if k not in ("prefix", "slopes")}
    check_attention(case, *attend(case, **kw, **dev), **how)


@pytest.mark.parametrize("dim", [2, 30, 40, 48, 72, 80, 96, 112, 130, 192, 208, 320, 512])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_other_head_sizes(dim, dtype):
    case = make([170, 19], [120, 1], heads=4, kv_heads=2, dim=dim, dtype=dtype, seed=dim)
    check_attention(case, *attend(case))
    step = make([170, 19, 33], [1, 1, 2], heads=4, kv_heads=2, dim=dim, dtype=dtype, seed=dim)
    check_attention(step, *attend(step))


@pytest.mark.parametrize("new", [[9, 1, 5], [1, 1, 1], [80, 30, 5]])
@pytest.mark.parametrize("index", ["table", "offsets", "i32", "i64", "identity"])
@pytest.mark.parametrize("page,scale_page", [(1, 1), (16, 16), (24, 24), (16, 40), (40, 16), (64, 1), (16, 7)])
def test_index_kinds_and_pages(index, page, scale_page, new):
    case = make([100, 37, 5], new, dim=128, index=index, page=page, scale_page=scale_page, layers=2, seed=4,
                start=48 // page * page)
    out, lse = paged_attention(case.batch, 1, case.q.cuda(), return_lse=True)
    check_attention(case, out, lse, layer=1)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_many_ragged_requests(dtype):
    g = torch.Generator().manual_seed(9)
    lengths = torch.randint(0, 90, (150,), generator=g).tolist()
    new = [min(n, int(torch.randint(0, 4, (1,), generator=g))) for n in lengths]
    big = next(i for i, n in enumerate(lengths) if i > 70 and n > 60)
    new[big] = 60
    case = make(lengths, new, dim=64, dtype=dtype, seed=5)
    check_attention(case, *attend(case))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("new,dim", [(1, 64), (20, 64), (150, 64), (1, 128), (20, 128), (150, 128), (20, 256), (150, 256)])
@pytest.mark.parametrize("heads", [4, 8])
def test_what_is_not_seen_never_counts(new, dim, heads, dtype):
    """NaN codes behind the mask, past the length and in pages of nobody, and scales of pages of nobody that are no
    scales, leave every row as it was; a row that sees a NaN value gets it."""
    case = make([170, 170], [new, new], heads=heads, dim=dim, dtype=dtype, seed=6)
    want, want_lse = attend(case, window=9)
    k, v = (codes_of(x) for x in case.pool)
    inside = torch.zeros(k.shape[1], dtype=torch.bool)
    for b in range(2):
        inside[case.slots[b]] = True
    k[:, ~inside.cuda()] = 0x7f
    v[:, ~inside.cuda()] = 0xff
    used = torch.zeros(case.scales[0].shape[1], dtype=torch.bool)
    used[torch.cat(case.slots) // 16] = True
    for s in case.scales:
        codes_of(s)[:, ~used.cuda()] = 255
    seen = 170 - new - 8  # the first token any new one sees
    for at, bad in ((0, 0x7f), (1, 0xff)):
        if at < seen:
            k[0, case.slots[0][at]] = bad
            v[0, case.slots[0][at]] = bad
    got, got_lse = attend(case, window=9)
    assert torch.equal(got, want) and torch.equal(got_lse, want_lse)
    if new > 1:
        v[0, case.slots[0][169]] = 0xff
        v[0, case.slots[1][168], :, 3] = 0x7f
        got, got_lse = attend(case, window=9)
        assert torch.equal(got_lse, want_lse)
        assert torch.equal(got[:new - 1], want[:new - 1])
        assert torch.isnan(got[new - 1]).all()
        assert torch.equal(got[new:2 * new - 2], want[new:2 * new - 2])
        assert torch.isnan(got[2 * new - 2:, :, 3]).all()
        keep = [d for d in range(dim) if d != 3]
        assert torch.equal(got[2 * new - 2:, :, keep], want[2 * new - 2:, :, keep])


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, BF16), (128, FP16), (96, FP16), (256, BF16)])
@pytest.mark.parametrize("how", [{}, dict(window=300, prefix=[37, 8]), dict(cap=4.0, causal=False)])
def test_large_launches(how, dim, dtype):
    """Enough scores for eight waves a workgroup; a sample of the rows against the oracle, NaN among the values."""
    new, heads, lengths = [700, 40], 16, [2400, 500]
    case = make(lengths, new, heads=heads, kv_heads=2, dim=dim, dtype=dtype, seed=21, index="i32")
    how = dict(how)
    prefix = how.pop("prefix", None)
    more = {} if prefix is None else dict(prefix_lengths=torch.tensor(prefix, dtype=torch.int32).cuda())
    out, lse = attend(case, **how, **more)
    u = torch.finfo(dtype).eps / 2
    for b, at, m in ((0, 0, 700), (1, 700, 40)):
        rows = sorted({0, 1, 31, 63, 64, 127, 128, 255, 256, 300, 511, 640, 699} & set(range(m)))
        for h in (0, 7, 8, 15):
            k, v = (x[0, case.slots[b], h // 8] for x in (case.k, case.v))
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
    if how.get("causal", True) and prefix is None:
        v = codes_of(case.pool[1])
        v[0, case.slots[0][2100], 0, 5] = 0x7f   # new token 400 and later ones see it
        v[0, case.slots[0][2200], 1, 6] = 0xff
        got, _ = attend(case, **how, **more)
        assert torch.equal(got[:400], out[:400]) and torch.equal(got[700:], out[700:])
        assert torch.isnan(got[400:700, :8, 5]).all() and torch.isnan(got[500:700, 8:, 6]).all()
        keep = [d for d in range(dim) if d not in (5, 6)]
        assert torch.equal(got[..., keep], out[..., keep])


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("new", [1, 40])
def test_scales_far_apart(new, dtype):
    """Pages whose scales differ by 2^12: values of 2^-8 beside values of 2^4, with weights on both."""
    case = make([200], [new], heads=4, kv_heads=2, dim=64, dtype=dtype, seed=12)
    for i, s in enumerate(case.scales):
        e = case.exponents[i].clone()
        e[:, ::2] = -16
        e[:, 1::2] = -5 if i == 0 else -4
        codes_of(s).copy_((e + 127).to(torch.uint8))
        from oracle import quantized
        setattr(case, "kv"[i], quantized.values(codes_of(case.pool[i]).cpu(), e, 16))
    check_attention(case, *attend(case))


@pytest.mark.parametrize("new", [3, 70])
def test_large_scales(new):
    """bf16 values near 2^100 and 2^-100: scales at both ends of what is stored."""
    case = make([100], [new], heads=2, kv_heads=2, dim=64, dtype=BF16, seed=13)
    for i, (s, e) in enumerate(zip(case.scales, (-100, 90))):
        codes_of(s).fill_(e + 127)
        from oracle import quantized
        setattr(case, "kv"[i], quantized.values(codes_of(case.pool[i]).cpu(), torch.full_like(case.exponents[i], e), 16))
    out, lse = attend(case, scale=2.0 ** 92)
    check_attention(case, out, lse, scale=2.0 ** 92)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("new", [[6, 11], [1, 1], [40, 90]])
def test_rows_of_no_request_and_strides(new, dtype):
    case = make([40, 90], new, heads=6, kv_heads=2, dim=128, dtype=dtype, seed=11, padding=5)
    n = sum(new)
    wide = torch.full((n + 5, 10, 128), 7.0, dtype=dtype).cuda()
    wide[:, 2:8] = case.q.cuda()
    out = torch.full((6, n + 5, 128), 3.0, dtype=dtype).cuda().transpose(0, 1)
    got, lse = paged_attention(case.batch, 0, wide[:, 2:8], out=out, return_lse=True)
    assert got is out
    check_attention(case, out[:n], lse[:n])
    assert (out[n:] == 3.0).all()
    odd = torch.zeros((n + 5) * 6 * 128 + 1, dtype=dtype).cuda()[1:].view(n + 5, 6, 128)
    odd.copy_(case.q)
    again = paged_attention(case.batch, 0, odd, out=torch.empty((n + 5) * 6 * 128 + 1, dtype=dtype).cuda()[1:].view(n + 5, 6, 128))
    check_attention(case, again[:n])


@pytest.mark.parametrize("new", [1, 30])
def test_unaligned_pool(new):
    case = make([50], [new], dim=64, seed=12)
    k, v = (torch.zeros(x.numel() + 3, dtype=torch.uint8).cuda()[3:].view(x.shape).copy_(codes_of(x)).view(x.dtype) for x in case.pool)
    table = torch.tensor([int(s) // 16 for s in case.slots[0][::16]], dtype=torch.int32).cuda()
    batch = QueryBatch(rows_from_stacked(k, v, block_table=table, page_size=16, scales=BlockScales(*case.scales, 16)),
                       torch.tensor([0, new]).int().cuda(), torch.tensor([50]).int().cuda(), max_length=50)
    out, lse = paged_attention(batch, 0, case.q.cuda(), return_lse=True)
    check_attention(case, out, lse)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("new", [5, 1])
def test_bad_rows_and_requests_are_left_out_and_flagged(new, dtype):
    case = make([60] * 4, [new] * 4, dim=64, dtype=dtype, seed=14, index="i32")
    flag = torch.zeros(1, dtype=torch.int32).cuda()
    paged_attention(case.batch, 0, case.q.cuda(), error_flag=flag)
    assert int(flag) == 0
    old = case.batch
    index = old.rows.keep[2].clone()
    index[3] = -1               # request 0, token 3
    index[60 + 10] = 1 << 30    # request 1, token 10
    rows = rows_from_stacked(*case.pool, index=index, scales=old.rows.scales)
    qs, ln, off = (t.clone() for t in old._keep)
    ln[2] = 61                  # past max_length
    off[3] = 210                # its tokens run past the index: 30 are there
    batch = QueryBatch(rows, qs, ln, offsets=off, max_length=60, max_query=5)
    out = torch.full_like(case.q, 9.0).cuda()
    paged_attention(batch, 0, case.q.cuda(), out=out, error_flag=flag)
    assert int(flag) == ERROR_CACHE_ROW | ERROR_REQUEST
    assert (out[2 * new:3 * new] == 9.0).all()
    u = torch.finfo(dtype).eps / 2
    for b, hole in ((0, 3), (1, 10)):
        for h in range(case.heads):
            q, k, v = case.q[new * b:new * b + new, h], case.k[0, case.slots[b], h // 2], case.v[0, case.slots[b], h // 2]
            x = oracle.scores(q, k, scale=0.125)
            seen = oracle.visible(60, new)
            seen[:, hole] = False
            w = torch.softmax(x.masked_fill(~seen, -math.inf), 1)
            tol = u * (w @ v).abs() + (w @ v.abs()) * (u + 4 * oracle.score_error(q, k, scale=0.125) + 76 * 2.0 ** -23)
            assert ((out[new * b:new * b + new, h].double().cpu() - w @ v).abs() - tol).max() <= 0


def test_tokens_of_other_types_and_other_operators_are_refused():
    case = make([40, 40], [2, 2], dim=64, dtype=FP16, seed=1)
    with pytest.raises(ValueError, match="float16"):
        paged_attention(case.batch, 0, case.q.to(BF16).cuda())
    w = torch.zeros(2, 40).cuda()
    with pytest.raises(ValueError, match="8-bit"):
        add_key_weights(case.batch, 0, case.q.cuda(), torch.zeros(4, 4).cuda(), w)
    with pytest.raises(ValueError, match="8-bit"):
        evict_tokens(case.batch, w, case.batch, budget=4)
