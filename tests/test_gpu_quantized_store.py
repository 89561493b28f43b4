"""GPU: rows that go into an 8-bit cache, from a prefix or as new tokens, against the 64-bit oracle."""

from __future__ import annotations

import math

import pytest
import torch

from cachebridge_amd import QuantizedKVPool, pool_rows
from cachebridge_amd.online.queries import (ERROR_CACHE_ROW, ERROR_REQUEST, ERROR_TARGET_ROW, QueryBatch, Rotary,
                                            install_tokens, paged_attention, quantize_tokens)
from cachebridge_amd.plan import BlockScales, rows_from_stacked
from oracle import quantized as oracle
from oracle import queries as rotation

from . import query_cases
from .quantized_cases import E4M3, codes_of, device_scales, make

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def most(dtype):
    return 7 if dtype == FP16 else 119


def exact(got, want):
    """Codes whose values are ``want`` (NaN where it is)."""
    v = oracle.decode(got)
    return torch.equal(torch.nan_to_num(v, 1e9), torch.nan_to_num(oracle.round_code(want), 1e9))


def target_for(case, page, *, room=0, order_seed=5, dtype=None):
    """An 8-bit pool of marked codes and a batch over it with pages for the case's requests."""
    layers, _, kv, dim = case.k.shape
    pages = [-(-(n + room) // page) for n in case.lengths]
    width = max(pages, default=0) + 1
    pool = QuantizedKVPool(layer_num=layers, pages=sum(pages) + 2, head_num=kv, head_dim=dim, page_size=page,
                           dtype=dtype or case.dtype)
    for x in (pool.k_data, pool.v_data):
        codes_of(x).fill_(0x55)
    for x in (pool.k_scale, pool.v_scale):
        codes_of(x).fill_(99)
    order = torch.randperm(sum(pages) + 2, generator=torch.Generator().manual_seed(order_seed))
    table, at = torch.full((len(pages), width), -1, dtype=torch.int32), 0
    for b, m in enumerate(pages):
        table[b, :m] = order[at:at + m].int()
        at += m
    rows = pool_rows(pool, block_table=table.view(-1).cuda())
    batch = QueryBatch(rows, *case.batch._keep[:2], request_stride=width * page, max_length=case.batch.max_length + room,
                       max_query=case.batch.max_query)
    return pool, table, batch


def check_quantized(case, pool, table, page, skip=()):
    """Every request's tokens, all layers: exact codes and scales; everything else as it was."""
    for x, src, s in ((pool.k_data, case.k, pool.k_scale), (pool.v_data, case.v, pool.v_scale)):
        codes, bytes_ = codes_of(x).cpu(), codes_of(s).cpu()
        left, left_scale = torch.ones(codes.shape[1], dtype=torch.bool), torch.ones(bytes_.shape[1], dtype=torch.bool)
        for b, n in enumerate(case.lengths):
            if b in skip:
                continue
            for p in range(-(-n // page)):
                at, stop = int(table[b, p]), min(n, (p + 1) * page)
                rows = slice(at * page, at * page + stop - p * page)
                left[rows], left_scale[at] = False, False
                for l in range(codes.shape[0]):
                    for h in range(codes.shape[2]):
                        want, e = oracle.store(src[l, case.slots[b][p * page:stop], h].double(), most(case.dtype))
                        assert int(bytes_[l, at, h]) == e + 127, (b, p, l, h)
                        assert exact(codes[l, rows, h], want), (b, p, l, h)
        assert (codes[:, left] == 0x55).all() and (bytes_[:, left_scale] == 99).all()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("page", [1, 16, 24, 64, 300])
@pytest.mark.parametrize("dim,kv", [(128, 2), (64, 3), (40, 1)])
def test_quantize(dim, kv, page, dtype):
    case = query_cases.make([130, 0, 1, 64, 257], [1, 0, 1, 1, 1], heads=kv, kv_heads=kv, dim=dim, dtype=dtype, layers=2, seed=dim + page)
    pool, table, target = target_for(case, page)
    flag = torch.zeros(1, dtype=torch.int32).cuda()
    got = quantize_tokens(case.batch, target, error_flag=flag)
    assert got.tolist() == case.lengths and int(flag) == 0
    check_quantized(case, pool, table, page)


@pytest.mark.parametrize("dim", [2, 6, 8, 30, 72, 80, 96, 256, 330, 512])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_quantize_head_sizes(dim, dtype):
    case = query_cases.make([50, 33], [1, 1], heads=2, kv_heads=2, dim=dim, dtype=dtype, seed=dim)
    pool, table, target = target_for(case, 32)
    quantize_tokens(case.batch, target)
    check_quantized(case, pool, table, 32)


@pytest.mark.parametrize("index", ["offsets", "i32", "i64", "identity"])
def test_quantize_from_other_indices(index):
    case = query_cases.make([100, 37, 5], [1, 1, 1], dim=128, index=index, layers=2, seed=4, start=48)
    pool, table, target = target_for(case, 16)
    quantize_tokens(case.batch, target)
    check_quantized(case, pool, table, 16)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_quantize_special_values(dtype):
    """Zeros of both signs, every code's value and what lies between, subnormals, the largest, infinities and NaN."""
    case = query_cases.make([96], [1], heads=2, kv_heads=2, dim=64, dtype=dtype, seed=3)
    v = oracle.decode(torch.arange(256, dtype=torch.uint8))
    v = v[torch.isfinite(v)]
    fine = v.sort().values.unique()
    step = fine[1:] - fine[:-1]
    line = torch.cat([v, fine[:-1] + step / 2, fine[:-1] + step / 4, fine[:-1] + step * 0.75, -torch.zeros(8).double()])
    line = torch.cat([line, torch.zeros(-line.numel() % 128, dtype=torch.float64)]).view(-1, 1, 64)
    rows = case.slots[0]
    big = float(torch.finfo(dtype).max)
    def put(first, x):
        x = x.to(dtype)
        case.k[0, rows[first:first + x.shape[0]]] = x
        case.v[0, rows[first:first + x.shape[0]]] = -x
    assert line.shape[0] <= 16
    put(0, line.expand(-1, 2, -1))                     # page 0: scale 1
    put(16, torch.zeros(16, 2, 64))                    # page 1: nothing but zeros
    put(32, torch.full((1, 2, 64), big))               # page 2: the largest
    put(33, torch.full((1, 2, 64), big * 0.87))
    put(48, torch.full((1, 2, 64), math.inf))          # pages 3 and 4: what is not finite beside what is
    put(49, torch.full((1, 2, 64), -math.inf))
    put(64, torch.full((16, 2, 64), math.nan))         # nothing finite
    put(80, torch.full((16, 2, 64), float(torch.finfo(dtype).tiny)) * torch.arange(64) / 16)  # subnormals
    for x, y in zip(case.pool, (case.k, case.v)):
        x.copy_(y)
    pool, table, target = target_for(case, 16)
    assert quantize_tokens(case.batch, target).tolist() == [96]
    check_quantized(case, pool, table, 16)
    zero = codes_of(pool.v_data)[0, int(table[0, 1]) * 16:int(table[0, 1]) * 16 + 16]
    assert (zero == 0x80).all() and int(codes_of(pool.k_scale)[0, int(table[0, 1]), 0]) == 1
    bad = codes_of(pool.k_data)[0, int(table[0, 3]) * 16:int(table[0, 3]) * 16 + 2]
    assert (bad & 0x7f == 0x7f).all()


def test_quantize_leaves_out_and_flags():
    case = query_cases.make([50] * 6, [1] * 6, heads=2, kv_heads=2, dim=64, index="i32", layers=2, seed=2)
    index = case.batch.rows.keep[-1].clone()
    index[7] = -1                      # request 0, token 7 has no row
    qs, ln, off = (t.clone() for t in case.batch._keep)
    ln[1], ln[2] = 51, -1              # outside the bounds
    batch = QueryBatch(rows_from_stacked(*case.pool, index=index), qs, ln, offsets=off, max_length=50)
    pool, table, target = target_for(case, 16)
    table[3, 1] = -1                   # request 3's tokens 16 to 31 have no page
    table[4, 2] = pool.pages
    starts = torch.arange(6) * table.shape[1] * 16
    starts[5] += 8                     # not at a page's first slot
    target = QueryBatch(pool_rows(pool, block_table=table.view(-1).cuda()), qs, ln, offsets=starts.cuda(), max_length=50)
    flag = torch.zeros(1, dtype=torch.int32).cuda()
    got = quantize_tokens(batch, target, error_flag=flag)
    assert got.tolist() == [0, 0, 0, 50, 50, 0]
    assert int(flag) == ERROR_CACHE_ROW | ERROR_TARGET_ROW | ERROR_REQUEST
    codes = codes_of(pool.k_data).cpu()
    own = {b: torch.cat([torch.arange(16) + int(p) * 16 for p in table[b] if 0 <= p < pool.pages]) for b in range(6)}
    for b in (1, 2, 5):
        assert (codes[:, own[b]] == 0x55).all()
    assert (codes[:, own[0][7]] == 0x55).all() and (codes[:, own[0][8]] != 0x55).any()
    # Past a request's stride nothing is stored: the next request's pages begin there.
    pool, table, _ = target_for(case, 16)
    tight = QueryBatch(pool_rows(pool, block_table=table[:, :2].contiguous().view(-1).cuda()), qs, ln, request_stride=32, max_length=50)
    flag.zero_()
    ln.fill_(50)
    got = quantize_tokens(case.batch, tight, error_flag=flag)
    assert got.tolist() == [50] * 6 and int(flag) == ERROR_TARGET_ROW
    codes = codes_of(pool.k_data).cpu()
    for b in range(6):
        for p in range(4):
            at = int(table[b, p])
            if at >= 0:
                assert (codes[:, at * 16:at * 16 + 16] == 0x55).all() == (p >= 2)


def test_quantize_other_pools_are_refused():
    case = query_cases.make([20], [1], heads=2, kv_heads=2, dim=64, seed=2)
    pool, table, target = target_for(case, 16)
    with pytest.raises(ValueError, match="8-bit"):
        quantize_tokens(case.batch, case.batch)
    with pytest.raises(ValueError, match="8-bit"):
        quantize_tokens(target, target)
    with pytest.raises(ValueError, match="dtype"):
        quantize_tokens(case.batch, target_for(case, 16, dtype=FP16)[2])
    with pytest.raises(ValueError, match="block table"):
        quantize_tokens(case.batch, QueryBatch(pool_rows(pool, block_table=table.view(-1).cuda(), page_size=32), *case.batch._keep[:2], max_length=20))
    with pytest.raises(ValueError, match="block table"):
        quantize_tokens(case.batch, QueryBatch(pool_rows(pool), *case.batch._keep[:2], max_length=20))


# ---------------------------------------------------------------------------
# New tokens
# ---------------------------------------------------------------------------


def check_stored(case, before, fused, heads, kv, turned, layer, page):
    """The 8-bit pool after new tokens, against what it held: values, scales and every code that is none of them."""
    dim = case.dim
    for x, s, at, kind in ((case.pool[0], case.scales[0], heads, 0), (case.pool[1], case.scales[1], heads + kv, 1)):
        codes, bytes_ = codes_of(x).cpu(), codes_of(s).cpu()
        old_codes, old_bytes = before[kind]
        left = torch.ones_like(codes, dtype=torch.bool)
        left_scale = torch.ones_like(bytes_, dtype=torch.bool)
        t = 0
        for b, (n, m) in enumerate(zip(case.lengths, case.new)):
            place = n - m
            while place < n:
                page0 = place // page * page
                stop = min(n, page0 + page)
                rows = case.slots[b][place:stop]
                cached = case.slots[b][page0:place]
                where = int(rows[0]) // page
                left_scale[layer, where] = False
                for h in range(kv):
                    want = turned(fused[t:t + stop - place, at + h], slice(t, t + stop - place)) if kind == 0 else fused[t:t + stop - place, at + h].double()
                    had = int(old_bytes[layer, where, h]) - 127 if len(cached) else -126
                    y, e = oracle.store(want, most(case.dtype), had)
                    assert int(bytes_[layer, where, h]) == e + 127, (b, place, h, kind)
                    got = oracle.decode(codes[layer, rows, h])
                    # K: cosine, sine and two products in fp32 (8 roundings of the pair's size), then half a step.
                    size = fused[t:t + stop - place, at + h].double().abs().amax(-1, keepdim=True) * 2 * turned.magnitude
                    slack = 2.0 ** -21 * size * 2.0 ** -e + 2.0 ** -25 if kind == 0 else 0.0
                    off = (got - y.clamp(-448, 448)).abs()
                    assert (off <= oracle.step(y.abs() + slack) / 2 + slack).all(), (b, place, h, kind)
                    if kind == 1:
                        assert exact(codes[layer, rows, h], y)
                    again = oracle.decode(old_codes[layer, cached, h]) * 2.0 ** (had - e)
                    assert exact(codes[layer, cached, h], again)
                    left[layer, rows, h] = False
                    left[layer, cached, h] = False
                t += stop - place
                place = stop
        assert torch.equal(codes[left], old_codes[left]) and torch.equal(bytes_[left_scale], old_bytes[left_scale])


class Turned:
    def __init__(self, positions, spin, axes=None):
        self.magnitude, self.spin, self.inv = spin.magnitude, spin, spin.inv_freq.cpu()
        self.positions, self.axes = positions, axes

    def __call__(self, x, tokens=slice(None)):
        x = x.double()
        if self.axes is None:
            return rotation.rotate(x[:, None] if x.ndim == 2 else x, self.positions[tokens], self.inv, magnitude=self.magnitude,
                                   interleaved=self.spin.interleaved).view(x.shape)
        # A pair at a time, by its own axis.
        y, half = x.clone(), self.inv.numel()
        for i in range(half):
            a, b = (2 * i, 2 * i + 1) if self.spin.interleaved else (i, half + i)
            angle = self.positions[self.axes[i]][tokens].double() * self.inv[i]
            c, s = angle.cos() * self.magnitude, angle.sin() * self.magnitude
            if x.ndim == 3:
                c, s = c[:, None], s[:, None]
            y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        return y


def near(got, want, x, magnitude, dtype):
    u = torch.finfo(dtype).eps / 2
    size = x.double().abs().amax(-1, keepdim=True) * 2 * magnitude
    assert ((got.double().cpu() - want).abs() - (u * want.abs() + 2.0 ** -21 * size + 2.0 ** -25)).max() <= 0


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("dim,rotary", [(128, 128), (128, 64), (64, 64), (96, 48), (80, 20), (256, 64), (2, 2), (510, 6), (512, 512)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_install(dim, rotary, interleaved, dtype):
    case = make([70, 16, 1, 33, 100], [7, 16, 1, 0, 40], heads=6, kv_heads=2, dim=dim, dtype=dtype, layers=2, seed=dim + rotary)
    g = torch.Generator().manual_seed(1)
    fused = torch.randn(64, 10, dim, generator=g)
    fused[:3] *= 30  # the first page's scales grow
    fused = fused.to(dtype)
    spin = Rotary.build(rotary, 1e4, dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32), interleaved=interleaved)
    before = [(codes_of(x).cpu().clone(), codes_of(s).cpu().clone()) for x, s in zip(case.pool, case.scales)]
    fd = fused.cuda()
    flag = torch.zeros(1, dtype=torch.int32).cuda()
    got = install_tokens(case.batch, 1, fd[:, :6], fd[:, 6:8], fd[:, 8:], spin, error_flag=flag)
    assert int(flag) == 0 and torch.equal(fd.cpu(), fused)
    turned = Turned(torch.cat([torch.arange(n - m, n) for n, m in zip(case.lengths, case.new)]), spin)
    near(got, turned(fused[:, :6]), fused[:, :6], spin.magnitude, dtype)
    check_stored(case, before, fused, 6, 2, turned, 1, 16)


@pytest.mark.parametrize("page", [1, 7, 24, 64, 128])
@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (FP32, 64), (BF16, 30)])
def test_install_pages(dtype, dim, page):
    case = make([300, 65, 5], [290, 3, 5], heads=2, kv_heads=1, dim=dim, dtype=dtype, page=page, seed=page)
    fused = torch.randn(298, 4, dim, generator=torch.Generator().manual_seed(page)).to(dtype)
    spin = Rotary.build(dim, 1e6)
    before = [(codes_of(x).cpu().clone(), codes_of(s).cpu().clone()) for x, s in zip(case.pool, case.scales)]
    fd = fused.cuda()
    qd = fd[:, :2]
    assert install_tokens(case.batch, 0, qd, fd[:, 2:3], fd[:, 3:], spin, out=qd) is qd
    turned = Turned(torch.cat([torch.arange(n - m, n) for n, m in zip(case.lengths, case.new)]), spin)
    near(qd, turned(fused[:, :2]), fused[:, :2], 1.0, dtype)
    check_stored(case, before, fused, 2, 1, turned, 0, page)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
@pytest.mark.parametrize("cyclic", [False, True])
@pytest.mark.parametrize("dtype,dim,sections,interleaved", [(BF16, 128, (24, 20, 20), False), (FP16, 64, (11, 11, 10), True),
                                                            (FP32, 96, (16, 8), False), (BF16, 80, (5, 3, 3), True)])
def test_axes(dtype, dim, sections, interleaved, cyclic, kind):
    """Positions of several axes, into an 8-bit and a 16- or 32-bit pool."""
    lengths, new, n = [70, 40], [37, 1], 38
    g = torch.Generator().manual_seed(2)
    fused = torch.randn(n, 8, dim, generator=g).to(dtype)
    pos = torch.randint(0, 1 << 20, (len(sections), n), generator=g).to(kind)
    spin = Rotary.build(2 * sum(sections), 1e4, interleaved=interleaved, sections=sections, cyclic=cyclic)
    turned = Turned(pos, spin, list(spin.axes))
    fd = fused.cuda()
    case = make(lengths, new, heads=4, kv_heads=2, dim=dim, dtype=dtype, seed=1)
    before = [(codes_of(x).cpu().clone(), codes_of(s).cpu().clone()) for x, s in zip(case.pool, case.scales)]
    got = install_tokens(case.batch, 0, fd[:, :4], fd[:, 4:6], fd[:, 6:], spin, positions=pos.cuda())
    near(got, turned(fused[:, :4]), fused[:, :4], 1.0, dtype)
    check_stored(case, before, fused, 4, 2, turned, 0, 16)
    plain = query_cases.make(lengths, new, heads=4, kv_heads=2, dim=dim, dtype=dtype, seed=1)
    again = install_tokens(plain.batch, 0, fd[:, :4], fd[:, 4:6], fd[:, 6:], spin, positions=pos.cuda())
    assert torch.equal(again, got)
    rows = torch.cat([s[a - m:] for s, a, m in zip(plain.slots, lengths, new)])
    near(plain.pool[0][0, rows], turned(fused[:, 4:6]), fused[:, 4:6], 1.0, dtype)
    assert torch.equal(plain.pool[1][0, rows].cpu(), fused[:, 6:])
    # Without positions every axis has the token's place; equal rows say the same.
    place = torch.cat([torch.arange(a - m, a) for a, m in zip(lengths, new)]).to(kind).cuda()
    one = install_tokens(plain.batch, 0, fd[:, :4], fd[:, 4:6], fd[:, 6:], spin._replace(axes=None))
    for p in (None, place.expand(len(sections), -1).contiguous()):
        assert torch.equal(install_tokens(plain.batch, 0, fd[:, :4], fd[:, 4:6], fd[:, 6:], spin, positions=p), one)


def test_axes_that_do_not_fit_are_refused():
    case = query_cases.make([20], [3], heads=2, kv_heads=1, dim=64, seed=1)
    x = torch.zeros(3, 4, 64, dtype=BF16).cuda()
    spin = Rotary.build(64, 1e4, sections=(16, 8, 8))
    def call(spin, positions):
        return install_tokens(case.batch, 0, x[:, :2], x[:, 2:3], x[:, 3:], spin, positions=positions)
    for bad in (torch.zeros(3).int(), torch.zeros(2, 3).int(), torch.zeros(3, 4).int(), torch.zeros(3, 3)):
        with pytest.raises(ValueError):
            call(spin, bad.cuda())
    with pytest.raises(ValueError, match="contiguous"):
        call(spin, torch.zeros(3, 3, 2).int().cuda()[..., 0])
    for bad in (spin.axes[:-1], list(spin.axes), bytes([9] * 32)):
        with pytest.raises(ValueError, match="axes"):
            call(spin._replace(axes=bad), None)
    with pytest.raises(ValueError, match="1-D"):
        call(spin._replace(axes=None), torch.zeros(3, 3).int().cuda())


def test_install_leaves_bad_rows_and_requests_out():
    case = make([40] * 4, [2] * 4, heads=2, kv_heads=1, dim=64, seed=20, padding=3)
    table = case.batch.rows.keep[2].clone().view(4, -1)
    table[0, 2] = case.pool[0].shape[1] // 16
    qs, ln, _ = case.batch._keep
    ln = ln.clone()
    ln[2] = 1
    offsets = torch.arange(4) * table.shape[1] * 16
    offsets[3] -= 8
    batch = QueryBatch(rows_from_stacked(*case.pool, block_table=table.view(-1), page_size=16, scales=case.batch.rows.scales), qs, ln,
                       offsets=offsets.cuda(), max_length=40, max_query=2)
    before = [codes_of(x).cpu().clone() for x in (*case.pool, *case.scales)]
    out = torch.full_like(case.q, 5.0).cuda()
    kv = torch.randn(11, 1, 64).to(BF16).cuda()
    flag = torch.zeros(1, dtype=torch.int32).cuda()
    install_tokens(batch, 0, case.q.cuda(), kv, kv, Rotary.build(64, 1e4), out=out, error_flag=flag)
    assert int(flag) == ERROR_TARGET_ROW | ERROR_REQUEST
    assert (out[4:] == 5.0).all()
    assert all((out[t] != 5.0).any() for t in range(4))
    mine = case.slots[1][32:40]
    for x, y in zip(case.pool, before):
        rest = torch.ones(y.shape[1], dtype=torch.bool)
        rest[mine] = False
        assert torch.equal(codes_of(x).cpu()[0][rest], y[0][rest])
        assert not torch.equal(codes_of(x).cpu()[0][case.slots[1][38:]], y[0][case.slots[1][38:]])
    with pytest.raises(ValueError, match="block table"):
        slots = QueryBatch(rows_from_stacked(*case.pool, scales=case.batch.rows.scales), qs, ln, offsets=offsets.cuda(), max_length=40)
        install_tokens(slots, 0, case.q.cuda(), kv, kv, Rotary.build(64, 1e4))


def test_a_page_grows_token_by_token():
    """A page filled one token a call, each larger than the ones before: scales grow, cached codes are rounded again,
    and what is stored stays within half a step of the page's scale for each time it grew, and one."""
    dim, page = 64, 16
    pool = QuantizedKVPool(layer_num=1, pages=2, head_num=1, head_dim=dim, page_size=page)
    table = torch.tensor([1], dtype=torch.int32).cuda()
    qs, length = torch.tensor([0, 1], dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int32).cuda()
    batch = QueryBatch(pool_rows(pool, block_table=table), qs, length, max_length=page, max_query=1)
    spin = Rotary.build(dim, 1e4)
    rows = (torch.randn(page, 3, dim, generator=torch.Generator().manual_seed(1)) * 1.7 ** torch.arange(page)[:, None, None]).to(BF16)
    rd, held, had = rows.cuda(), torch.zeros(0, dim, dtype=torch.float64), -126
    for i in range(page):
        length.fill_(i + 1)
        install_tokens(batch, 0, rd[i:i + 1, :1], rd[i:i + 1, 1:2], rd[i:i + 1, 2:], spin)
        new, e = oracle.store(rows[i:i + 1, 2].double(), had=had if i else -126)
        held = torch.cat([oracle.round_code(held * 2.0 ** (had - e)), oracle.round_code(new)])
        had = e
        assert int(codes_of(pool.v_scale)[0, 1, 0]) == e + 127
        assert torch.equal(oracle.decode(codes_of(pool.v_data)[0, page:page + i + 1, 0].cpu()), held)
    assert (codes_of(pool.v_scale)[0, 0] == 1).all()
    # Going on from a shorter request: the page's later slots count no more.
    length.fill_(5)
    small = (rows[:1] * 0.01).cuda()
    before = codes_of(pool.v_data)[0, page + 5:2 * page].clone()
    install_tokens(batch, 0, small[:, :1], small[:, 1:2], small[:, 2:], spin)
    assert int(codes_of(pool.v_scale)[0, 1, 0]) == had + 127 and torch.equal(codes_of(pool.v_data)[0, page + 5:2 * page], before)
    length.fill_(1)  # and from a page's first slot its scale is chosen anew
    install_tokens(batch, 0, small[:, :1], small[:, 1:2], small[:, 2:], spin)
    assert int(codes_of(pool.v_scale)[0, 1, 0]) == oracle.store(small[:, 2].double().cpu())[1] + 127
