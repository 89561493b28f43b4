"""Queries on an installed prefix: the new tokens of a batch of requests over a paged pool.

Once ``install_unpublished`` has published a request's history, the target
model answers on it, layer by layer:

- ``install_tokens``: rotate the new tokens' queries and keys to their
  positions and store their K/V rows into the requests' pages;
- ``paged_attention``: attention of the new tokens over the cached ones (a
  prompt's chunk or a decoding step: windows, prefixes that see themselves
  whole, capped scores, biases by distance, grouped heads);
- ``add_key_weights``: add to each cached token the attention it got;
- ``evict_tokens``: keep the first, the last and the heaviest tokens of long
  histories, copied in order to other pages.

``QueryBatch`` describes the batch once for all layers. Its lengths and
offsets are device tensors that the kernels read, so a captured graph follows
their values; only the bounds ``max_query`` and ``max_length`` are fixed by
the host. A request outside these bounds is left out and flagged in
``error_flag`` (an int32 tensor, bits ``ERROR_CACHE_ROW``,
``ERROR_TARGET_ROW`` and ``ERROR_REQUEST``), as are cached tokens without a
valid pool row; nothing is read or written for them.

All work is asynchronous on ``stream`` (default: the current one). Inputs
belong to the caller and must stay as they are until that stream is done with
them. No counterpart in the reference, whose target engine answers the
queries (``cb/online/admission.py:466-499`` hands over after publication).
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import NamedTuple

import torch

from .. import _lib
from ..plan import Rows, io_dtype_code
from ..rope import rope_frequencies

_raw_stream = _lib._raw_stream

ERROR_CACHE_ROW = _lib.CB_ERROR_CACHE_ROW
ERROR_TARGET_ROW = _lib.CB_ERROR_TARGET_ROW
ERROR_REQUEST = _lib.CB_ERROR_REQUEST


class _On:
    """A launch's device and stream, entered: allocations and launches inside use them.

    Yields the stream's handle. With the batch's device current and no stream
    named, which every layer of a model's step is, nothing is entered: a
    context object would cost as much host time as the launch itself.
    """

    __slots__ = ("handle", "_context")

    def __init__(self, batch: "QueryBatch", stream: torch.cuda.Stream | None):
        index = batch.device.index
        if stream is not None:
            if stream.device.index != index:
                raise ValueError("stream belongs to another device than the batch")
            self._context = torch.cuda.stream(stream)
            self.handle = _lib.stream_handle(stream)
            return
        current = index == torch.cuda.current_device()
        self._context = None if current else torch.cuda.device(index)
        self.handle = int(torch.cuda.current_stream(index).cuda_stream) if _raw_stream is None else _raw_stream(index)

    def __enter__(self) -> int:
        if self._context is not None:
            self._context.__enter__()
        return self.handle

    def __exit__(self, *exc):
        if self._context is not None:
            self._context.__exit__(*exc)


def _device_vector(t: torch.Tensor, name: str, dtypes, device, entries: int | None) -> int:
    if t.ndim != 1 or t.dtype not in dtypes or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name} must be a contiguous 1-D tensor of {' or '.join(map(str, dtypes))} on {device}")
    if entries is not None and t.numel() != entries:
        raise ValueError(f"{name} must have {entries} entries")
    return t.data_ptr()


class QueryBatch:
    """New tokens of a batch of requests, and where their cached tokens are.

    ``rows`` describes the pool and its index (``pool_rows`` or
    ``rows_from_stacked`` with a block table, slot vector or neither). Request
    ``b`` has rows ``query_start[b]`` to ``query_start[b + 1] - 1`` (int32) of
    the token tensors; they are the last of its ``lengths[b]`` (int32) cached
    tokens. Its cached token ``j`` is index token ``offsets[b] + j`` (int64,
    the target offset of a ``RequestSpan``), or ``b * request_stride + j``: for
    a ``[requests, width]`` block table given flat, ``width * page_size``. A
    request longer than ``request_stride`` would reach into the next one's
    tokens: it is outside the batch's bounds. What ``offsets`` leave each
    request is the caller's to keep to.
    ``max_query`` and ``max_length`` bound the new and cached tokens of any
    request (default bounds read nothing from the device: ``max_query`` is
    every token row, so give it where it is known; a decoding step divides its
    keys by ``max_length``, so a bound far above the lengths costs time, and
    memory: its calls allocate ``max_length / 2048 * tokens * heads *
    head_dim`` floats, 1 GB for 64 tokens with 64 heads of 128 and a bound of
    2^20).
    """

    def __init__(self, rows: Rows, query_start: torch.Tensor, lengths: torch.Tensor, *, max_length: int,
                 max_query: int | None = None, offsets: torch.Tensor | None = None, request_stride: int = 0):
        if rows.device.type != "cuda":
            raise ValueError("the query batch lives on a GPU device")
        for t in rows.keep:
            if t.ndim == 1 and not t.is_contiguous():
                raise ValueError("pool indices must be contiguous")
        if rows.c.k_layers and any(t.data_ptr() % 16 for t in rows.keep if t.ndim == 3):
            raise ValueError("pool layers must be 16-byte aligned")
        if rows.c.index_kind != _lib.CB_INDEX_IDENTITY and rows.index_entries < 1:
            raise ValueError("rows do not say how many entries their index has")
        requests = lengths.numel()
        # The C fields are 32 bits wide, and ctypes drops what does not fit.
        if not 0 <= max_length <= 1 << 30:
            raise ValueError("max_length must be 0 to 2^30")
        if max_query is not None and max_query < 0:
            raise ValueError("max_query must not be negative")
        if not 0 <= request_stride <= 1 << 31:
            raise ValueError("request_stride must be 0 to 2^31")
        if requests > 1 and offsets is None and request_stride == 0:
            raise ValueError("several requests need offsets or a request_stride")
        c = _lib.CbQueryBatch()
        c.cache = rows.c
        c.index_entries = rows.index_entries
        c.query_start = _device_vector(query_start, "query_start", (torch.int32,), rows.device, requests + 1)
        c.lengths = _device_vector(lengths, "lengths", (torch.int32,), rows.device, None)
        if offsets is not None:
            c.offsets = _device_vector(offsets, "offsets", (torch.int64,), rows.device, requests)
        c.request_stride = request_stride
        c.num_requests = requests
        c.max_length = max_length
        self.head_dim = rows.c.row_stride // max(rows.c.heads, 1)
        self.c = c
        self.rows = rows
        self.requests = requests
        self.max_query = None if max_query is None else int(max_query)
        self.max_length = int(max_length)
        self.device = rows.device
        self.dtype = rows.dtype
        self._code = io_dtype_code(rows.dtype)
        self._keep = (query_start, lengths, offsets)

    @property
    def kv_heads(self) -> int:
        return self.c.cache.heads

    def _layer(self, layer: int) -> int:
        if not 0 <= layer < self.rows.num_layers:
            raise ValueError(f"layer {layer} outside the cache")
        return layer

    def _tokens(self, n: int):
        """The C description for token tensors of ``n`` rows (a copy: calls may run side by side)."""
        c = _lib.CbQueryBatch.from_buffer_copy(self.c)
        c.num_tokens = n
        c.max_query = n if self.max_query is None else min(self.max_query, n)
        return ctypes.byref(c)

    def _heads(self, t: torch.Tensor, name: str, tokens: int | None = None, heads: int | None = None) -> _lib.CbHeads:
        shape = t.shape
        if len(shape) != 3 or t.dtype != self.dtype or t.device != self.device:
            raise ValueError(f"{name} must be [tokens, heads, head_dim] of {self.dtype} on {self.device}")
        n, h, d = shape
        if d != self.head_dim:
            raise ValueError(f"{name} must have the pool's head_dim {self.head_dim}")
        if (tokens is not None and n != tokens) or (heads is not None and h != heads):
            raise ValueError(f"{name} must have {tokens} tokens and {heads} heads")
        st, sh, sd = t.stride()
        if sd != 1 and d > 1:
            raise ValueError(f"{name} must be contiguous in its last dimension")
        return _lib.CbHeads(t.data_ptr(), st, sh, h, 0)


class Rotary(NamedTuple):
    """Rotation of new tokens: radians per position of each pair (float64, on
    the batch's device), the magnitude of scaled contexts, and whether pairs
    are neighbours instead of halves of the rotated part. The rotated part is
    the head's first ``2 * len(inv_freq)`` elements."""

    inv_freq: torch.Tensor
    magnitude: float = 1.0
    interleaved: bool = False

    @classmethod
    def build(cls, rotary_dim: int, theta: float, scaling: dict | None = None, *, interleaved: bool = False,
              device="cuda") -> "Rotary":
        """Frequencies of ``rope_frequencies`` (plain, linear, YaRN or Llama 3 scaling)."""
        inv, magnitude = rope_frequencies(rotary_dim, theta, scaling)
        return cls(inv.to(device), magnitude, interleaved)


def _flag_pointer(batch: QueryBatch, error_flag: torch.Tensor | None):
    if error_flag is None:
        return None
    if error_flag.dtype != torch.int32 or error_flag.numel() < 1 or error_flag.device != batch.device:
        raise ValueError(f"error_flag must be an int32 tensor on {batch.device}")
    return error_flag.data_ptr()


def install_tokens(batch: QueryBatch, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rotary: Rotary,
                   *, positions: torch.Tensor | None = None, out: torch.Tensor | None = None,
                   error_flag: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """Rotate the new tokens' ``q`` and ``k`` and store their K/V rows into ``layer`` of the pool.

    ``q`` is ``[tokens, heads, head_dim]``, ``k`` and ``v`` ``[tokens,
    kv_heads, head_dim]``, of any token and head strides (views of a fused
    projection). Returns the rotated ``q``: ``out``, which may be ``q``, or a
    new tensor. ``positions`` (int32 or int64, one per token row) replaces the
    tokens' places in the cache where these differ, as after an eviction. Rows
    of no request are neither stored nor written.
    """
    n, heads, dim = q.shape if q.ndim == 3 else (0, 0, 0)
    cq = batch._heads(q, "q")
    ck = batch._heads(k, "k", n, batch.kv_heads)
    cv = batch._heads(v, "v", n, batch.kv_heads)
    inv = rotary.inv_freq
    _device_vector(inv, "inv_freq", (torch.float64,), batch.device, None)
    kind, pos = 0, None
    if positions is not None:
        pos = _device_vector(positions, "positions", (torch.int32, torch.int64), batch.device, n)
        kind = _lib.CB_INDEX_I64 if positions.dtype == torch.int64 else _lib.CB_INDEX_I32
    flag = _flag_pointer(batch, error_flag)
    with _On(batch, stream) as handle:
        if out is None:
            out = q.new_empty((n, heads, dim))
        co = batch._heads(out, "out", n, heads)
        _lib.check(_lib.load().cb_install_tokens(
            batch._tokens(n), batch._layer(layer), batch._code, dim, ctypes.byref(cq), ctypes.byref(co), ctypes.byref(ck),
            ctypes.byref(cv), inv.data_ptr(), 2 * inv.numel(), int(rotary.interleaved), rotary.magnitude, pos, kind,
            flag, handle))
        batch.rows.hold_for(stream)
    return out


def _scores(batch: QueryBatch, heads: int, dim: int, scale, causal, window, cap, slopes, prefix_lengths):
    if not 0 <= window <= 0x7FFFFFFF:
        raise ValueError("window must be 0 to 2^31 - 1")
    c = _lib.CbScores(dim ** -0.5 if scale is None else scale, cap, window, int(causal))
    if not math.isfinite(c.scale):
        raise ValueError("scale must be finite")
    if slopes is not None:
        c.slopes = _device_vector(slopes, "slopes", (torch.float32,), batch.device, heads)
    if prefix_lengths is not None:
        c.prefix_lengths = _device_vector(prefix_lengths, "prefix_lengths", (torch.int32,), batch.device,
                                          batch.requests)
    return c


def paged_attention(batch: QueryBatch, layer: int, q: torch.Tensor, *, scale: float | None = None, causal: bool = True,
                    window: int = 0, cap: float = 0.0, slopes: torch.Tensor | None = None,
                    prefix_lengths: torch.Tensor | None = None, fp32_weights: bool = False,
                    out: torch.Tensor | None = None, return_lse: bool = False, error_flag: torch.Tensor | None = None,
                    stream: torch.cuda.Stream | None = None):
    """Attention of the new tokens over the cached ones of their requests.

    New token at place ``p`` of its request sees cached token ``j`` if ``j <
    prefix_lengths[b]``, or if ``j <= p`` (unless not ``causal``) and ``j > p -
    window`` (unless ``window`` is 0). Scores are ``scale * (q . k)`` (default
    ``head_dim ** -0.5``), then ``cap * tanh(x / cap)`` with a ``cap``, then
    minus ``slopes[h] * |p - j|`` (fp32, one per query head). Query head ``h``
    reads KV head ``h // (heads // kv_heads)``.

    Returns ``[tokens, heads, head_dim]`` (``out`` or a new tensor), with
    ``return_lse`` also fp32 ``[tokens, heads]`` logarithms of the sums of
    exponentials. A token that sees nothing gets zeros and ``-inf``; rows of no
    request are not written. What a token does not see never reaches its row,
    NaN and infinities in the cache included. Scores, statistics and sums are
    fp32; the weights of a 16-bit pool are rounded to its type for their product
    with V, which adds about as much error as the result's own rounding, unless
    ``fp32_weights``, which takes fp32 products (8 to 13 times as long for
    prompts, 2 to 4 times for steps and short questions).
    """
    n, heads, dim = q.shape if q.ndim == 3 else (0, 0, 0)
    cq = batch._heads(q, "q")
    scores = _scores(batch, heads, dim, scale, causal, window, cap, slopes, prefix_lengths)
    scores.fp32_weights = bool(fp32_weights)
    flag = _flag_pointer(batch, error_flag)
    lib = _lib.load()
    with _On(batch, stream) as handle:
        if out is None:
            out = q.new_empty((n, heads, dim))
        co = batch._heads(out, "out", n, heads)
        lse = q.new_empty((n, heads), dtype=torch.float32) if return_lse else None
        c = batch._tokens(n)
        need = ctypes.c_int64(0)
        _lib.check(lib.cb_attention_workspace_bytes(c, batch._code, dim, ctypes.byref(scores), heads,
                                                    ctypes.byref(need)))
        work = q.new_empty(need.value, dtype=torch.uint8) if need.value else None
        _lib.check(lib.cb_paged_attention(
            c, batch._layer(layer), batch._code, dim, ctypes.byref(scores), ctypes.byref(cq), ctypes.byref(co),
            None if lse is None else lse.data_ptr(), None if work is None else work.data_ptr(), need.value, flag,
            handle))
        batch.rows.hold_for(stream)
    return (out, lse) if return_lse else out


def add_key_weights(batch: QueryBatch, layer: int, q: torch.Tensor, lse: torch.Tensor, weights: torch.Tensor, *,
                    scale: float | None = None, causal: bool = True, window: int = 0, cap: float = 0.0,
                    slopes: torch.Tensor | None = None, prefix_lengths: torch.Tensor | None = None,
                    error_flag: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None) -> None:
    """Add to ``weights[b, j]`` the attention cached token ``j`` got from the new tokens, over all heads.

    ``lse`` is what ``paged_attention`` returned for the same ``q`` and
    arguments (fp32 ``[tokens, heads]``, contiguous); ``weights`` is fp32
    ``[requests, >= max_length]`` and keeps what no new token sees. The order
    of every sum is fixed: the same call gives the same bits.
    """
    n, heads, dim = q.shape if q.ndim == 3 else (0, 0, 0)
    cq = batch._heads(q, "q")
    if lse.shape != (n, heads) or lse.dtype != torch.float32 or not lse.is_contiguous() or lse.device != batch.device:
        raise ValueError("lse must be a contiguous float32 [tokens, heads] tensor on the batch's device")
    stride = _weights_stride(batch, weights)
    scores = _scores(batch, heads, dim, scale, causal, window, cap, slopes, prefix_lengths)
    flag = _flag_pointer(batch, error_flag)
    with _On(batch, stream) as handle:
        _lib.check(_lib.load().cb_add_key_weights(
            batch._tokens(n), batch._layer(layer), batch._code, dim, ctypes.byref(scores), ctypes.byref(cq), lse.data_ptr(),
            weights.data_ptr(), stride, flag, handle))
        batch.rows.hold_for(stream)


def _weights_stride(batch: QueryBatch, weights: torch.Tensor) -> int:
    if weights.ndim != 2 or weights.dtype != torch.float32 or weights.device != batch.device:
        raise ValueError("weights must be a float32 [requests, max_length] tensor on the batch's device")
    if weights.shape[0] != batch.requests or weights.shape[1] < batch.max_length:
        raise ValueError("weights must cover every request and max_length cached tokens")
    if weights.shape[1] > 1 and weights.stride(1) != 1:
        raise ValueError("weights must be contiguous in its last dimension")
    return max(weights.stride(0), batch.max_length) if batch.requests < 2 else weights.stride(0)


@dataclass
class KeptTokens:
    """What an eviction kept: ``tokens`` and ``weights`` ``[requests, budget]``
    (then -1 and 0), ``lengths`` ``[requests]``. ``tokens`` holds the places the
    kept tokens had, which stay their positions. A length is 0 for a request
    outside the batch's bounds, and for one whose kept tokens are not all in
    the target because a cached row is missing: its target rows then hold in
    part what they held before, and ``tokens`` and ``weights`` only tell what
    was chosen."""

    tokens: torch.Tensor
    lengths: torch.Tensor
    weights: torch.Tensor


def evict_tokens(batch: QueryBatch, weights: torch.Tensor, target: QueryBatch, *, budget: int, first: int = 0,
                 last: int = 0, error_flag: torch.Tensor | None = None,
                 stream: torch.cuda.Stream | None = None) -> KeptTokens:
    """Keep at most ``budget`` cached tokens of each request and copy their rows, all layers, to ``target``.

    Kept are the ``first`` first and ``last`` last tokens and, of the others,
    those of the largest ``weights`` (fp32 ``[requests, >= max_length]``; equal
    ones: the lower place first; NaN counts above every number). They go, in
    order, to tokens 0, 1, ... of the same request of ``target``, a batch over
    unpublished pages of the same or another pool (its lengths are not read; a
    token past its ``request_stride`` is not copied and sets
    ``ERROR_TARGET_ROW``).
    Its rows must not be rows that kept tokens are read from. A request of at
    most ``budget`` tokens is copied whole.

    The other calls take a cached token's place for its position where they
    use a window or ``slopes``, and ``install_tokens`` alone takes
    ``positions``: on an evicted cache, windows and slopes measure the places
    that are left. Models with either should not go on from one.
    """
    stride = _weights_stride(batch, weights)
    if target.device != batch.device or target.dtype != batch.dtype:
        raise ValueError("batch and target must share device and dtype")
    if target.requests != batch.requests:
        raise ValueError("batch and target must have the same requests")
    dim = batch.head_dim
    if target.kv_heads != batch.kv_heads or target.head_dim != dim or target.rows.num_layers != batch.rows.num_layers:
        raise ValueError("batch and target must share layers, KV heads and head_dim")
    if not 1 <= budget <= 1 << 30 or first < 0 or last < 0 or first + last > budget:
        raise ValueError("budget must be 1 to 2^30 and hold the first and last tokens")
    flag = _flag_pointer(batch, error_flag)
    b, dev = batch.requests, batch.device
    with _On(batch, stream) as handle:
        kept = KeptTokens(torch.empty((b, budget), dtype=torch.int32, device=dev),
                          torch.empty(b, dtype=torch.int32, device=dev),
                          torch.empty((b, budget), dtype=torch.float32, device=dev))
        _lib.check(_lib.load().cb_evict_tokens(
            batch._tokens(0), target._tokens(0), batch._code, dim, weights.data_ptr(), stride, budget, first, last,
            kept.tokens.data_ptr(), kept.lengths.data_ptr(), kept.weights.data_ptr(), flag, handle))
        batch.rows.hold_for(stream)
        target.rows.hold_for(stream)
    return kept
