"""Bounds of the query calls without a GPU: what is refused before any launch."""

from __future__ import annotations

import ctypes

import pytest

from cachebridge_amd import _lib

from .test_queries import FAKE, attend, batch, evict, heads, lib, ref, refused, scores  # noqa: F401


def test_requests_that_store_rows_need_places_of_their_own(lib):  # noqa: F811
    """Neither offsets nor a stride: all three requests would store to the same rows."""
    h, kv = heads(), heads(2)
    rc = lib.cb_install_tokens(ref(batch()), 0, 0, 128, ref(h), ref(h), ref(kv), ref(kv), FAKE, 128, 0, 1.0, None,
                               _lib.CB_INDEX_IDENTITY, None, None)
    refused(lib, rc, "offsets or a request_stride")
    refused(lib, evict(lib, b=batch(request_stride=100)), "target need offsets or a request_stride")


@pytest.mark.parametrize("strides", [(0, 128), (512, 0), (511, 128), (512, 127), (128, 512), (128, 128), (100, 1000),
                                     (300, 600), (200, 401)])
def test_outputs_whose_rows_share_memory_are_refused(lib, strides):  # noqa: F811
    """8 tokens of 4 heads of 128 elements."""
    out = heads(token_stride=strides[0], head_stride=strides[1])
    refused(lib, attend(lib, out=out), "out has rows that share memory")
    h, kv, b = heads(), heads(2), batch(request_stride=100)
    rc = lib.cb_install_tokens(ref(b), 0, 0, 128, ref(h), ref(out), ref(kv), ref(kv), FAKE, 128, 0, 1.0, None, 0, None, None)
    refused(lib, rc, "q_out has rows that share memory")


@pytest.mark.parametrize("strides", [(512, 128), (640, 128), (128, 1024), (130, 1100), (1024, 256), (256, 5000),
                                     (384, 128 + 384 * 8), (400, 1300)])
def test_outputs_with_rows_apart_are_taken(lib, strides):  # noqa: F811
    """400 and 1300: later heads start between the first head's tokens. What is refused then is the workspace, which comes later."""
    dim = 128 if strides != (400, 1300) else 100
    t, h = ([i * s for i in range(n)] for n, s in ((8, strides[0]), (4, strides[1])))
    places = sorted(x + y for x in t for y in h)
    assert all(b - a >= dim for a, b in zip(places, places[1:])), "the case itself"
    b = batch(max_length=100000, rows=200000, row_stride=256)
    refused(lib, attend(lib, b, dim=dim, q=heads(dim=dim), out=heads(token_stride=strides[0], head_stride=strides[1])), "workspace")


def test_launches_past_32_bits_of_threads_are_refused(lib):  # noqa: F811
    """Bounds that the arguments allow, but no grid: 2^32 threads or more."""
    s, q, kv, far = scores(), heads(), heads(2), 1 << 30
    b = batch(max_length=far, request_stride=far, rows=far)
    rc = lib.cb_add_key_weights(ref(b), 0, 0, 128, ref(s), ref(q), FAKE, FAKE, far, None, None)
    refused(lib, rc, "too many cached tokens")
    refused(lib, evict(lib, b=b, t=b, budget=far, stride=far), "too large")
    b = batch(num_tokens=1 << 27, request_stride=far)
    rc = lib.cb_install_tokens(ref(b), 0, 0, 128, ref(q), ref(q), ref(kv), ref(kv), FAKE, 128, 0, 1.0, None, 0, None, None)
    refused(lib, rc, "too many tokens")
    b = batch(max_length=far, request_stride=far, rows=far, num_requests=32, num_tokens=32, max_query=1)
    need = ctypes.c_int64(0)
    assert lib.cb_attention_workspace_bytes(ref(b), 0, 128, ref(s), 4, ctypes.byref(need)) == 0
    refused(lib, attend(lib, b, work=FAKE, work_bytes=need.value), "too many query tiles")
