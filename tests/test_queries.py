"""Queries on a paged cache without a GPU: argument checks before any HIP call, frequencies, the oracle, the code object."""

from __future__ import annotations

import ctypes
import math
import re
import struct
import subprocess

import pytest
import torch

from cachebridge_amd import _lib
from cachebridge_amd.online.queries import QueryBatch, Rotary
from cachebridge_amd.plan import rows_from_stacked
from cachebridge_amd.rope import _inverse_frequency, rope_frequencies
from oracle import queries as oracle

from .test_abi import _c_layout
from .test_code_object import _tool

FAKE = 1 << 20  # a pointer that is never followed: every call here fails before a launch


@pytest.fixture(scope="module")
def lib(built_library):
    return _lib.load()


def batch(**kw):
    b = _lib.CbQueryBatch()
    c = b.cache
    c.k_base = c.v_base = FAKE
    c.layer_stride, c.row_stride, c.rows, c.num_layers, c.heads = 1 << 16, 256, 256, 2, 2
    b.query_start = b.lengths = FAKE
    b.num_requests, b.num_tokens, b.max_query, b.max_length = 3, 8, 4, 100
    for name, value in kw.items():
        setattr(c if hasattr(c, name) else b, name, value)
    return b


def heads(n=4, dim=128, data=FAKE, **kw):
    h = _lib.CbHeads(data, n * dim, dim, n, 0)
    for name, value in kw.items():
        setattr(h, name, value)
    return h


def scores(**kw):
    s = _lib.CbScores(0.1, 0.0, 0, 1)
    for name, value in kw.items():
        setattr(s, name, value)
    return s


def refused(lib, rc, text):
    assert rc == _lib.CB_EINVAL
    assert re.search(text, lib.cb_last_error().decode()), lib.cb_last_error()


def ref(x):
    return None if x is None else ctypes.byref(x)


def attend(lib, b=None, layer=0, dtype=_lib.CB_DTYPE_BF16, dim=128, s=None, q=None, out=None, work=None, work_bytes=0):
    return lib.cb_paged_attention(ref(batch() if b is None else b), layer, dtype, dim, ref(scores() if s is None else s),
                                  ref(heads() if q is None else q), ref(heads() if out is None else out), None, work,
                                  work_bytes, None, None)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=7), "dtype"), (dict(dim=127), "head_dim"), (dict(dim=514), "head_dim"), (dict(dim=0), "head_dim"),
    (dict(layer=2), "layer"), (dict(layer=-1), "layer"), (dict(dim=256), "shorter"),
    (dict(s=scores(scale=math.nan)), "scale"), (dict(s=scores(cap=-1.0)), "cap"), (dict(s=scores(cap=math.inf)), "cap"),
    (dict(s=scores(window=-3)), "window"), (dict(q=heads(3)), "multiple"), (dict(q=heads(0)), "multiple"),
    (dict(out=heads(2)), "out has 2 heads"), (dict(q=heads(data=None)), "null q data"),
    (dict(q=heads(data=FAKE + 1)), "aligned"), (dict(out=heads(head_stride=-1)), "negative stride"),
    (dict(b=batch(head_offset=1)), "head_offset"), (dict(b=batch(heads=0)), "KV heads"),
    (dict(b=batch(rows=1 << 31)), "rows"), (dict(b=batch(rows=0)), "rows"), (dict(b=batch(k_base=None)), "required"),
    (dict(b=batch(k_base=FAKE + 1)), "aligned"), (dict(b=batch(num_requests=-1)), "negative"),
    (dict(b=batch(max_query=9)), "max_query"), (dict(b=batch(max_length=(1 << 30) + 1)), "max_length"),
    (dict(b=batch(max_length=-1)), "max_length"), (dict(b=batch(lengths=None)), "null"),
    (dict(b=batch(query_start=None)), "null"), (dict(b=batch(request_stride=-1)), "request_stride"),
    (dict(b=batch(index_kind=3, index=FAKE)), "page_size"), (dict(b=batch(index_kind=3, index=FAKE, page_size=1 << 21)), "page_size"),
    (dict(b=batch(index_kind=2)), "index pointer"), (dict(b=batch(index_kind=1, index=FAKE, index_entries=-1)), "index_entries"),
    (dict(b=batch(index_kind=9)), "index_kind"), (dict(b=batch(index_offset=-1)), "index_offset"),
])
def test_attention_refusals(lib, kw, text):
    refused(lib, attend(lib, **kw), text)


def test_attention_needs_its_workspace(lib):
    b = batch(max_length=100000, rows=200000)
    need = ctypes.c_int64(0)
    assert lib.cb_attention_workspace_bytes(ref(b), _lib.CB_DTYPE_BF16, 128, ref(scores()), 4, ctypes.byref(need)) == 0
    assert need.value > 0
    for work, n in ((None, need.value), (FAKE, need.value - 1), (FAKE + 16, need.value)):
        refused(lib, attend(lib, b, work=work, work_bytes=n), "workspace")
    b = batch(num_tokens=0, max_query=0)
    assert lib.cb_attention_workspace_bytes(ref(b), _lib.CB_DTYPE_BF16, 128, ref(scores()), 4, ctypes.byref(need)) == 0
    assert need.value == 0
    refused(lib, lib.cb_attention_workspace_bytes(ref(b), 0, 128, ref(scores()), 4, None), "null")


def test_null_descriptions(lib):
    b, s, h = batch(), scores(), heads()
    refused(lib, lib.cb_paged_attention(None, 0, 0, 128, ref(s), ref(h), ref(h), None, None, 0, None, None), "null batch")
    refused(lib, lib.cb_paged_attention(ref(b), 0, 0, 128, None, ref(h), ref(h), None, None, 0, None, None), "null scores")
    refused(lib, lib.cb_paged_attention(ref(b), 0, 0, 128, ref(s), None, ref(h), None, None, 0, None, None), "null q")
    refused(lib, lib.cb_paged_attention(ref(b), 0, 0, 128, ref(s), ref(h), None, None, None, 0, None, None), "null out")
    refused(lib, lib.cb_add_key_weights(ref(b), 0, 0, 128, ref(s), ref(h), None, FAKE, 100, None, None), "null lse")
    refused(lib, lib.cb_add_key_weights(ref(b), 0, 0, 128, ref(s), ref(h), FAKE, FAKE, 99, None, None), "max_length")


def install(lib, b=None, dim=128, rot=128, inv=FAKE, mag=1.0, pos=None, kind=0, q=None, k=None):
    return lib.cb_install_tokens(ref(batch() if b is None else b), 0, 0, dim, ref(heads() if q is None else q),
                                 ref(heads()), ref(heads(2) if k is None else k), ref(heads(2)), inv, rot, 0, mag, pos,
                                 kind, None, None)


@pytest.mark.parametrize("kw,text", [
    (dict(rot=0), "rotary_dim"), (dict(rot=7), "rotary_dim"), (dict(rot=130), "rotary_dim"), (dict(inv=None), "inv_freq"),
    (dict(mag=math.inf), "magnitude"), (dict(pos=FAKE, kind=0), "positions"), (dict(pos=FAKE, kind=3), "positions"),
    (dict(k=heads(4)), "k has 4 heads"), (dict(q=heads(6)), "q_out has 4 heads"),
])
def test_install_refusals(lib, kw, text):
    refused(lib, install(lib, **kw), text)


def evict(lib, b=None, t=None, budget=10, first=1, last=1, stride=100, kept=FAKE):
    return lib.cb_evict_tokens(ref(batch() if b is None else b), ref(batch() if t is None else t), 0, 128, FAKE, stride,
                               budget, first, last, kept, FAKE, FAKE, None, None)


@pytest.mark.parametrize("kw,text", [
    (dict(budget=0), "budget"), (dict(first=6, last=5), "within the budget"), (dict(first=-1), "within the budget"),
    (dict(stride=99), "max_length"), (dict(kept=None), "null"), (dict(t=batch(num_requests=2)), "requests"),
    (dict(t=batch(heads=1, row_stride=256)), "layers or KV heads"), (dict(t=batch(num_layers=1)), "layers or KV heads"),
])
def test_evict_refusals(lib, kw, text):
    refused(lib, evict(lib, **kw), text)


@pytest.mark.parametrize("cls,cname", [(_lib.CbQueryBatch, "cb_query_batch"), (_lib.CbHeads, "cb_heads"),
                                       (_lib.CbScores, "cb_scores")])
def test_struct_layouts_match_the_c_compiler(cls, cname):
    fields = [name for name, _ in cls._fields_]
    size, *offsets = _c_layout(cname, fields)
    assert ctypes.sizeof(cls) == size
    assert [getattr(cls, f).offset for f in fields] == offsets


def test_batches_live_on_a_gpu():
    x = torch.zeros(1, 32, 2, 64)
    with pytest.raises(ValueError, match="GPU"):
        QueryBatch(rows_from_stacked(x, x), torch.tensor([0, 1]).int(), torch.tensor([4]).int(), max_length=4)


def test_frequencies_are_the_tables_in_64_bits():
    yarn = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=8192, beta_fast=16, attn_factor=1.1)
    for scaling in (None, yarn):
        inv, magnitude = rope_frequencies(128, 1e6, scaling)
        table, m = _inverse_frequency(128, 1e6, scaling)
        # The tables' exponent is off by 2^-24 relative, which its power magnifies by ln(theta) < 14.
        assert inv.dtype == torch.float64 and ((inv / table.double() - 1).abs() < 16 * 2.0 ** -22).all()
        assert magnitude == pytest.approx(m)
    assert torch.equal(rope_frequencies(64, 1e4, dict(type="linear", factor=8))[0], rope_frequencies(64, 1e4, None)[0] / 8)
    llama = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=8192)
    inv, plain = rope_frequencies(128, 5e5, llama)[0], rope_frequencies(128, 5e5, None)[0]
    wave = 2 * math.pi / plain
    assert torch.equal(inv[wave < 8192 / 4], plain[wave < 8192 / 4])
    assert torch.equal(inv[wave > 8192], plain[wave > 8192] / 8)
    mid = (wave > 8192 / 4) & (wave < 8192)
    smooth = (8192 / wave[mid] - 1.0) / 3.0
    assert torch.allclose(inv[mid], (1 - smooth) * plain[mid] / 8 + smooth * plain[mid], rtol=1e-14)
    for bad in (dict(rope_type="dynamic", factor=2), dict(rope_type="yarn", factor=1, original_max_position_embeddings=10),
                dict(rope_type="linear", factor=0), dict(llama, low_freq_factor=4.0)):
        with pytest.raises(ValueError):
            rope_frequencies(64, 1e4, bad)
    with pytest.raises(ValueError, match="even"):
        rope_frequencies(63, 1e4, None)
    spin = Rotary.build(32, 1e4, interleaved=True, device="cpu")
    assert spin.interleaved and spin.inv_freq.shape == (16,) and spin.magnitude == 1.0


def test_oracle_agrees_with_dense_torch():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(n, 32, generator=g, dtype=torch.float64) for n in (9, 30, 30))
    want = torch.nn.functional.scaled_dot_product_attention(q[None], k[None], v[None], attn_mask=oracle.visible(30, 9)[None])
    out, lse, mag = oracle.attention(q, k, v, scale=32 ** -0.5)
    assert torch.allclose(out, want[0], atol=1e-12) and (mag >= out.abs() - 1e-12).all()
    assert oracle.key_weights(q, k, lse, scale=32 ** -0.5).sum().item() == pytest.approx(9.0)
    # Rotations keep lengths and differences of positions.
    inv, _ = rope_frequencies(32, 1e4, None)
    for pairs in (False, True):
        a = oracle.rotate(q[:, None], torch.arange(9) + 100, inv, interleaved=pairs)
        b = oracle.rotate(k[:9, None], torch.arange(9) + 90, inv, interleaved=pairs)
        c = oracle.rotate(q[:, None], torch.arange(9) + 10, inv, interleaved=pairs)
        d = oracle.rotate(k[:9, None], torch.arange(9), inv, interleaved=pairs)
        assert torch.allclose((a * b).sum(-1), (c * d).sum(-1))
    assert oracle.keep([1.0, 5.0, 5.0, 0.0, math.nan, 2.0], 4, first=1, last=1) == [0, 1, 4, 5]


def test_no_query_kernel_uses_scratch(built_library, tmp_path):
    """Every code object of the library, not its first alone: no private segment, no spills."""
    fatbin = tmp_path / "fatbin.bin"
    subprocess.run([_tool("llvm-objcopy"), f"--dump-section=.hip_fatbin={fatbin}", str(built_library),
                    str(tmp_path / "copy.so")], check=True, capture_output=True)
    data = fatbin.read_bytes()
    kernels = {}
    for n, start in enumerate(m.start() for m in re.finditer(b"__CLANG_OFFLOAD_BUNDLE__", data)):
        count, at = struct.unpack_from("<Q", data, start + 24)[0], start + 32
        for _ in range(count):
            offset, size, name = struct.unpack_from("<QQQ", data, at)
            triple = data[at + 24:at + 24 + name].decode()
            at += 24 + name
            if "gfx950" not in triple:
                continue
            code = tmp_path / f"code{n}.co"
            code.write_bytes(data[start + offset:start + offset + size])
            notes = subprocess.run([_tool("llvm-readelf"), "--notes", str(code)], check=True, capture_output=True,
                                   text=True).stdout
            for block in notes.split(".name:")[1:]:
                fields = dict(re.findall(r"\.(private_segment_fixed_size|vgpr_spill_count):\s+(\d+)", block))
                if "private_segment_fixed_size" in fields:
                    kernels[block.split()[0]] = {k: int(v) for k, v in fields.items()}
    names = " ".join(kernels)
    for expected in ("map_install_stream_kernel", "install_tokens_kernel", "attend_any_kernel", "attend_tile_kernel",
                     "attend_step_kernel", "join_few_kernel", "join_splits_kernel", "key_weights_any_kernel",
                     "key_weights_kernel", "select_tokens_kernel", "move_rows_kernel"):
        assert expected in names, expected
    assert not {n: m for n, m in kernels.items() if any(m.values())}
