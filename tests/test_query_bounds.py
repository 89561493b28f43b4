"""Bounds of the query calls without a GPU: what is refused before any launch."""

from __future__ import annotations

from cachebridge_amd import _lib

from .test_queries import FAKE, batch, evict, heads, lib, ref, refused  # noqa: F401


def test_requests_that_store_rows_need_places_of_their_own(lib):  # noqa: F811
    """Neither offsets nor a stride: all three requests would store to the same rows."""
    h, kv = heads(), heads(2)
    rc = lib.cb_install_tokens(ref(batch()), 0, 0, 128, ref(h), ref(h), ref(kv), ref(kv), FAKE, 128, 0, 1.0, None,
                               _lib.CB_INDEX_IDENTITY, None, None)
    refused(lib, rc, "offsets or a request_stride")
    refused(lib, evict(lib, b=batch(request_stride=100)), "target need offsets or a request_stride")
