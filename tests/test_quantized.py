"""8-bit caches without a GPU: argument checks before any HIP call, layouts, axes, the oracle's rounding."""

from __future__ import annotations

import ctypes

import pytest
import torch

from cachebridge_amd import QuantizedKVPool, _lib, pool_rows
from cachebridge_amd.online.queries import Rotary
from cachebridge_amd.plan import BlockScales, rows_from_stacked
from oracle import quantized as oracle

from .test_abi import _c_layout
from .test_queries import FAKE, batch, heads, lib, ref, refused, scores  # noqa: F401

BF16 = _lib.CB_DTYPE_BF16


def paged(**kw):
    """A block table of pages of 16 over 256 rows of 2 heads of 128."""
    return batch(**dict(dict(index_kind=3, index=FAKE, index_entries=64, page_size=16, request_stride=128), **kw))


def scale_pages(**kw):
    s = _lib.CbPageScales(FAKE, FAKE, 32, 2, 16, 16)
    for name, value in kw.items():
        setattr(s, name, value)
    return s


def rotation(**kw):
    r = _lib.CbRotation(FAKE, None, None, 8, 128, 0, 0, 1, 1.0)
    for name, value in kw.items():
        setattr(r, name, value)
    return r


def at(x):
    return None if x is None else ctypes.addressof(x)


def install(lib, b=None, s=None, layer=0, dtype=BF16, dim=128, q=None, out=None, k=None, v=None, turn=None):
    q, out, k, v = heads() if q is None else q, heads() if out is None else out, heads(2) if k is None else k, heads(2) if v is None else v
    return lib.cb_install_quantized(ref(paged() if b is None else b), ref(scale_pages() if s is None else s), layer, dtype, dim,
                                    at(q), at(out), at(k), at(v),
                                    ref(rotation() if turn is None else turn), None, None)


BAD_SCALES = [
    (dict(k=None), "null scales"), (dict(v=None), "null scales"), (dict(page_size=0), "page_size"),
    (dict(page_size=(1 << 20) + 1), "page_size"), (dict(pages=15), "do not cover"), (dict(pages=-1), "do not cover"),
    (dict(pages=1 << 31), "do not cover"), (dict(page_stride=1), "page_stride"), (dict(layer_stride=-1), "layer_stride"),
]


@pytest.mark.parametrize("kw,text", BAD_SCALES)
def test_bad_scales_are_refused(lib, kw, text):  # noqa: F811
    s, need = scale_pages(**kw), ctypes.c_int64(0)
    refused(lib, install(lib, s=s), text)
    refused(lib, lib.cb_quantize_tokens(ref(batch(request_stride=100)), ref(paged()), ref(s), BF16, 128, FAKE, None, None), text)
    refused(lib, lib.cb_quantized_attention(ref(paged()), ref(s), 0, BF16, 128, ref(scores()), ref(heads()), ref(heads()),
                                            None, None, 0, None, None), text)
    refused(lib, lib.cb_quantized_attention_workspace_bytes(ref(paged()), ref(s), BF16, 128, ref(scores()), 4, ctypes.byref(need)), text)


@pytest.mark.parametrize("kw,text", [
    (dict(b=paged(index_kind=0)), "block table"), (dict(b=paged(index_kind=1)), "block table"),
    (dict(b=paged(page_size=32)), "block table"), (dict(b=paged(request_stride=0)), "request_stride"),
    (dict(layer=2), "layer"), (dict(dim=127), "head_dim"), (dict(dim=256), "shorter"), (dict(dtype=7), "dtype"),
    (dict(q=heads(0)), "q needs"), (dict(k=heads(4)), "k has 4 heads"), (dict(v=heads(2, data=None)), "null v data"),
    (dict(out=heads(head_stride=0)), "share memory"), (dict(turn=rotation(rotary_dim=130)), "rotary_dim"),
    (dict(turn=rotation(inv_freq=None)), "inv_freq"), (dict(turn=rotation(magnitude=float("nan"))), "magnitude"),
    (dict(turn=rotation(positions=FAKE, positions_kind=0)), "positions"),
    (dict(turn=rotation(pair_axis=bytes(63) + b"\3", axes=3)), "pair 63 turns by axis 3 of 3"),
    (dict(turn=rotation(pair_axis=bytes(64), axes=0)), "axes"), (dict(turn=rotation(pair_axis=bytes(64), axes=9)), "axes"),
    (dict(turn=rotation(pair_axis=bytes(64), axes=2, positions=FAKE, positions_kind=1, axis_stride=7)), "shorter"),
])
def test_install_refusals(lib, kw, text):  # noqa: F811
    refused(lib, install(lib, **kw), text)


def test_rotated_install_refusals(lib):  # noqa: F811
    def call(turn, b=None):
        many, kv = heads(), heads(2)
        return lib.cb_install_rotated(ref(batch(request_stride=100) if b is None else b), 0, BF16, 128, at(many), at(many), at(kv),
                                      at(kv), ref(turn), None, None)
    refused(lib, call(None), "null rotation")
    refused(lib, call(rotation(pair_axis=b"\1" * 64, axes=1)), "axis 1 of 1")
    refused(lib, call(rotation(), batch(request_stride=0)), "request_stride")


def test_quantize_refusals(lib):  # noqa: F811
    def call(b=None, t=None, dtype=BF16, dim=128, lengths=FAKE):
        return lib.cb_quantize_tokens(ref(batch(request_stride=100) if b is None else b), ref(paged() if t is None else t),
                                      ref(scale_pages()), dtype, dim, lengths, None, None)
    refused(lib, call(lengths=None), "lengths_out")
    refused(lib, call(dtype=_lib.CB_DTYPE_F64), "dtype")
    refused(lib, call(dim=130), "shorter")
    refused(lib, call(t=paged(num_requests=2)), "requests")
    refused(lib, call(t=paged(num_layers=3)), "layers")
    refused(lib, call(t=paged(heads=1)), "KV heads")
    refused(lib, call(t=paged(page_size=8)), "block table")
    refused(lib, call(t=paged(index_kind=0)), "block table")
    refused(lib, call(t=paged(request_stride=0)), "request_stride")
    refused(lib, call(b=batch(max_length=1 << 30, request_stride=1 << 30, num_requests=1 << 20), t=paged(num_requests=1 << 20)), "too many")


def test_attention_refusals(lib):  # noqa: F811
    def call(b=None, s=None, q=None, out=None, dim=128, dtype=BF16, layer=0):
        return lib.cb_quantized_attention(ref(paged() if b is None else b), ref(scale_pages()), layer, dtype, dim,
                                          ref(scores() if s is None else s), ref(heads() if q is None else q),
                                          ref(heads() if out is None else out), None, None, 0, None, None)
    refused(lib, lib.cb_quantized_attention(ref(paged()), ref(scale_pages()), 0, BF16, 128, ref(scores()), None, ref(heads()),
                                            None, None, 0, None, None), "null q")
    refused(lib, call(q=heads(3)), "multiple")
    refused(lib, call(out=heads(2)), "out has 2 heads")
    refused(lib, call(layer=2), "layer")
    refused(lib, call(s=scores(window=-1)), "window")
    refused(lib, call(dtype=9), "dtype")
    long = paged(max_length=100000, request_stride=1 << 20)
    need = ctypes.c_int64(0)
    assert lib.cb_quantized_attention_workspace_bytes(ref(long), ref(scale_pages()), BF16, 128, ref(scores()), 4, ctypes.byref(need)) == 0
    assert need.value > 0
    refused(lib, call(b=long), "workspace")


@pytest.mark.parametrize("cls,cname", [(_lib.CbRotation, "cb_rotation"), (_lib.CbPageScales, "cb_page_scales")])
def test_struct_layouts(cls, cname):
    fields = [name for name, _ in cls._fields_]
    size, *offsets = _c_layout(cname, fields)
    assert ctypes.sizeof(cls) == size and [getattr(cls, f).offset for f in fields] == offsets


def test_pool_describes_its_pages():
    pool = QuantizedKVPool(layer_num=3, pages=5, head_num=2, head_dim=64, page_size=24, device="cpu", fill="zeros")
    assert pool.size == 120 and pool.k_scale.shape == (3, 5, 2) and (pool.v_scale.view(torch.uint8) == 1).all()
    table = torch.zeros(5, dtype=torch.int32)
    rows = pool_rows(pool, block_table=table)
    assert rows.scales.dtype == torch.bfloat16 and rows.c.page_size == 24 and rows.c_scales.pages == 5
    part = pool.rows(block_table=table, layers=slice(1, 3))
    assert part.num_layers == 2 and part.c_scales.k == pool.k_scale[1].data_ptr()
    with pytest.raises(ValueError, match="dtype"):
        QuantizedKVPool(layer_num=1, pages=1, head_num=1, head_dim=64, dtype=torch.float64, device="cpu")
    with pytest.raises(ValueError, match="page_size"):
        QuantizedKVPool(layer_num=1, pages=1, head_num=1, head_dim=64, page_size=0, device="cpu")


def test_scales_that_do_not_fit_their_pool_are_refused():
    codes = torch.zeros(2, 32, 2, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    good = torch.ones(2, 2, 2, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    rows_from_stacked(codes, codes, scales=BlockScales(good, good, 16))
    for k, page, of, text in ((good.float(), 16, codes, "e8m0"), (good[:, :1], 16, codes, "contiguous|scales must be"),
                              (good, 8, codes, "scales must be"), (good, 0, codes, "page_size"),
                              (good, 16, codes.view(torch.uint8), "e4m3"), (good.transpose(0, 1), 16, codes, "contiguous")):
        with pytest.raises(ValueError, match=text):
            rows_from_stacked(of, of, scales=BlockScales(k, good, page))
    with pytest.raises(ValueError, match="dtype"):
        rows_from_stacked(codes, codes, scales=BlockScales(good, good, 16, torch.float64))


def test_axes_of_pairs():
    assert Rotary.axis_of_pairs((2, 1, 3)) == bytes([0, 0, 1, 2, 2, 2])
    assert Rotary.axis_of_pairs((4, 2, 2), cyclic=True) == bytes([0, 1, 2, 0, 1, 2, 0, 0])
    assert Rotary.axis_of_pairs((3, 3, 2), cyclic=True) == bytes([0, 1, 2, 0, 1, 2, 0, 1])
    assert Rotary.axis_of_pairs((5,)) == bytes(5)
    for bad in ((), (0, 0), (-1, 3), (1,) * 9):
        with pytest.raises(ValueError):
            Rotary.axis_of_pairs(bad)
    with pytest.raises(ValueError, match="largest"):
        Rotary.axis_of_pairs((1, 4), cyclic=True)
    with pytest.raises(ValueError, match="pairs"):
        Rotary.build(64, 1e4, sections=(16, 15), device="cpu")
    assert Rotary.build(64, 1e4, sections=(16, 8, 8), device="cpu").axes == bytes([0] * 16 + [1] * 8 + [2] * 8)


def test_oracle_codes():
    """Every code's value, rounding between neighbours, and the least scale, against torch's own conversion."""
    codes = torch.arange(256, dtype=torch.uint8)
    v = oracle.decode(codes)
    assert torch.equal(torch.nan_to_num(v, 1e9), torch.nan_to_num(codes.view(torch.float8_e4m3fn).double(), 1e9))
    fine = v[torch.isfinite(v)].sort().values.unique()
    assert torch.equal(oracle.round_code(fine), fine)
    between = torch.cat([fine[:-1] + (fine[1:] - fine[:-1]) * f for f in (0.25, 0.5, 0.75)])
    assert torch.equal(oracle.round_code(between), between.float().to(torch.float8_e4m3fn).double())
    for top, e in ((448.0, 0), (448.0001, 1), (1.75, -8), (1.8, -7), (0.0, -126), (2.0 ** -140, -126), (2.9e38, 119)):
        assert oracle.exponent(top) == e and (e == -126 or 448.0 * 2.0 ** e >= top > 448.0 * 2.0 ** (e - 1))
    assert oracle.exponent(3.3e38) == 119  # 448 * 2^119 and no more: twice that is no fp32 value
    assert oracle.exponent(65504.0, 99) == 8 and oracle.exponent(65504.0, 7) == 7
