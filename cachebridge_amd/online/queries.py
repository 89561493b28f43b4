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
  histories, copied in order to other pages;
- ``quantize_tokens``: move histories into the pages of a ``QuantizedKVPool``
  (e4m3 codes, a scale for each page and head), on which ``install_tokens`` and
  ``paged_attention`` go on at half the bytes of a 16-bit pool.

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
import functools
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
    Over 8-bit rows (``rows`` with scales) token tensors are of the scales'
    ``dtype``.
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
        self.scales = rows.c_scales
        if rows.c_scales is None:
            self.dtype = rows.dtype
        else:
            self.dtype = rows.scales.dtype
            self._scales = ctypes.byref(rows.c_scales)
        self._code = io_dtype_code(self.dtype)
        self._keep = (query_start, lengths, offsets)
        self._by_tokens = {}

    @property
    def kv_heads(self) -> int:
        return self.c.cache.heads

    def _layer(self, layer: int) -> int:
        if not 0 <= layer < self.rows.num_layers:
            raise ValueError(f"layer {layer} outside the cache")
        return layer

    def _tokens(self, n: int):
        """The C description for token tensors of ``n`` rows (one for each ``n`` and bound, not written again: calls
        may run side by side)."""
        ref = self._by_tokens.get((n, self.max_query))
        if ref is None:
            c = _lib.CbQueryBatch.from_buffer_copy(self.c)
            c.num_tokens = n
            c.max_query = n if self.max_query is None else min(self.max_query, n)
            if len(self._by_tokens) >= 64:
                self._by_tokens = {}
            ref = self._by_tokens[n, self.max_query] = ctypes.byref(c)
        return ref

    def _heads(self, t: torch.Tensor, name: str, tokens: int | None = None, heads: int | None = None) -> _lib.CbHeads:
        data, token_stride, head_stride, h = self._row(t, name, tokens, heads)
        return _lib.CbHeads(data, token_stride, head_stride, h, 0)

    def _row(self, t: torch.Tensor, name: str, tokens: int | None = None, heads: int | None = None):
        """A token tensor's address, token and head stride and heads, checked: the words of a ``cb_heads``."""
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
        return t.data_ptr(), st, sh, h


# The cb_heads of q and out, or of q, out, k and v, four words each (the last one heads, its upper half reserved).
_TwoHeads = ctypes.c_int64 * 8
_FourHeads = ctypes.c_int64 * 16


class _Rotation(NamedTuple):
    inv_freq: torch.Tensor
    magnitude: float = 1.0
    interleaved: bool = False


class Rotary(_Rotation):
    """Rotation of new tokens: radians per position of each pair (float64, on
    the batch's device), the magnitude of scaled contexts, and whether pairs
    are neighbours instead of halves of the rotated part. The rotated part is
    the head's first ``2 * len(inv_freq)`` elements.

    ``axes`` (bytes, one per pair) makes positions of several axes, such as time,
    height and width of image patches: pair ``i`` turns by the position along
    axis ``axes[i]``. It is an attribute beside the tuple's three fields, which
    unpack as those of a rotation of one axis.
    """

    axes: bytes | None = None

    def __new__(cls, inv_freq: torch.Tensor, magnitude: float = 1.0, interleaved: bool = False,
                axes: bytes | None = None) -> "Rotary":
        self = super().__new__(cls, inv_freq, magnitude, interleaved)
        self.axes = axes
        return self

    def __getnewargs__(self):
        return (*self, self.axes)

    def _replace(self, **fields) -> "Rotary":
        axes = fields.pop("axes", self.axes)
        return type(self)(*super()._replace(**fields), axes)

    def __eq__(self, other):
        return self.axes == getattr(other, "axes", None) and super().__eq__(other)

    def __ne__(self, other):
        return not self == other

    def __hash__(self):
        return hash((*self, self.axes))

    def __repr__(self):
        return f"Rotary({', '.join(f'{k}={v!r}' for k, v in self._asdict().items())}, axes={self.axes!r})"

    @staticmethod
    def axis_of_pairs(sections, *, cyclic: bool = False) -> bytes:
        """The axis of each pair, ``sections[a]`` pairs of axis ``a``.

        In blocks, axis after axis, or ``cyclic``: the axes in turn from pair to
        pair, axis 0 in place of one whose pairs are used up (which needs the
        first section to be the largest).
        """
        sections = [int(n) for n in sections]
        if not 1 <= len(sections) <= 8 or min(sections) < 0 or sum(sections) < 1:
            raise ValueError("a rotation has 1 to 8 axes of some pairs")
        if not cyclic:
            return bytes(a for a, n in enumerate(sections) for _ in range(n))
        axes = [i % len(sections) if i // len(sections) < sections[i % len(sections)] else 0
                for i in range(sum(sections))]
        if any(axes.count(a) != n for a, n in enumerate(sections)):
            raise ValueError("cyclic axes need the first section to be the largest")
        return bytes(axes)

    @classmethod
    def build(cls, rotary_dim: int, theta: float, scaling: dict | None = None, *, interleaved: bool = False,
              sections=None, cyclic: bool = False, device="cuda") -> "Rotary":
        """Frequencies of ``rope_frequencies`` (plain, linear, YaRN or Llama 3 scaling), with ``sections`` the axes of
        ``axis_of_pairs`` over ``rotary_dim / 2`` pairs."""
        inv, magnitude = rope_frequencies(rotary_dim, theta, scaling)
        axes = None if sections is None else cls.axis_of_pairs(sections, cyclic=cyclic)
        if axes is not None and len(axes) != inv.numel():
            raise ValueError(f"the sections must have rotary_dim / 2 = {inv.numel()} pairs")
        return cls(inv.to(device), magnitude, interleaved, axes)


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
    tokens' places in the cache where these differ, as after an eviction; with
    ``rotary.axes`` it is ``[axes, tokens]``, contiguous. Rows of no request are
    neither stored nor written.

    Into an 8-bit pool, K/V rows are rounded to e4m3 under their page's and
    head's scale: the least power of two that keeps every finite element within
    448 times it. A page that holds cached tokens keeps its scale unless the new
    rows need a larger one, to which the cached ones are then rounded. Infinities
    and NaN are stored as NaN. Such a batch needs a block table of the pool's
    page size, and requests that start at a page's first slot.
    """
    n, heads, dim = q.shape if q.ndim == 3 else (0, 0, 0)
    rq = batch._row(q, "q")
    rk = batch._row(k, "k", n, batch.kv_heads)
    rv = batch._row(v, "v", n, batch.kv_heads)
    inv = _device_vector(rotary.inv_freq, "inv_freq", (torch.float64,), batch.device, None)
    pos, kind = _positions(batch, rotary, positions, n)
    flag = _flag_pointer(batch, error_flag)
    with _On(batch, stream) as handle:
        if out is None:
            out = q.new_empty((n, heads, dim))
        rows = _FourHeads(*rq, *batch._row(out, "out", n, heads), *rk, *rv)
        at = ctypes.addressof(rows)
        lib, layer, code = _lib.load(), batch._layer(layer), batch._code
        if batch.scales is None and rotary.axes is None:
            _lib.check(lib.cb_install_tokens(
                batch._tokens(n), layer, code, dim, at, at + 32, at + 64, at + 96, inv, 2 * rotary.inv_freq.numel(),
                int(rotary.interleaved), rotary.magnitude, pos, kind, flag, handle))
        else:
            turn = ctypes.byref(_rotation(rotary, inv, pos, kind, n))
            if batch.scales is None:
                _lib.check(lib.cb_install_rotated(batch._tokens(n), layer, code, dim, at, at + 32, at + 64, at + 96,
                                                  turn, flag, handle))
            else:
                _lib.check(lib.cb_install_quantized(batch._tokens(n), batch._scales, layer, code, dim, at, at + 32,
                                                    at + 64, at + 96, turn, flag, handle))
        batch.rows.hold_for(stream)
    return out


@functools.lru_cache(maxsize=64)
def _axis_count(axes: bytes) -> int:
    """The axes that pairs turn by: a step of many layers asks at every one."""
    return max(axes, default=0) + 1


def _positions(batch: QueryBatch, rotary: Rotary, positions: torch.Tensor | None, n: int):
    """The positions' address and index kind, None and 0 without any; the rotation's axes checked."""
    axes = rotary.axes
    if axes is None:
        if positions is None:
            return None, 0
        at = _device_vector(positions, "positions", (torch.int32, torch.int64), batch.device, n)
    else:
        if not isinstance(axes, bytes) or len(axes) != rotary.inv_freq.numel() or _axis_count(axes) > 8:
            raise ValueError("axes must be bytes, 0 to 7, one for each pair of inv_freq")
        if positions is None:
            return None, 0
        shape = positions.shape
        if len(shape) != 2 or shape[0] < _axis_count(axes) or shape[1] != n:
            raise ValueError("positions must be [axes, tokens] with one row for each of the rotation's axes")
        if positions.dtype not in (torch.int32, torch.int64) or not positions.is_contiguous() or positions.device != batch.device:
            raise ValueError(f"positions must be a contiguous tensor of torch.int32 or torch.int64 on {batch.device}")
        at = positions.data_ptr()
    return at, _lib.CB_INDEX_I64 if positions.dtype == torch.int64 else _lib.CB_INDEX_I32


def _rotation(rotary: Rotary, inv: int, pos: int | None, kind: int, n: int) -> _lib.CbRotation:
    axes, dim, spin = rotary.axes, 2 * rotary.inv_freq.numel(), int(rotary.interleaved)
    count = 1 if axes is None else _axis_count(axes)
    return _lib.CbRotation(inv, pos, axes, n, dim, spin, kind, count, rotary.magnitude)


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
    fp32; with 16-bit tokens the weights are rounded to their type for their
    product with V, which adds about as much error as the result's own rounding,
    unless ``fp32_weights``, which takes fp32 products (6 to 14 times as long for
    prompts, 2 to 10 times for steps and short questions). Over an 8-bit pool the
    cached values are codes times scales, ``q`` and the result are of the scales'
    ``dtype``, calls of up to 32 query rows a KV head keep 16 bits of a weight in
    any case, and ``fp32_weights`` takes 7 to 16 times as long for prompts, 2 to 18
    times for steps and short questions. fp32 tokens, and head sizes that are no
    multiple of 16 (on 16-bit pools: of 8) or above 256, go to that kernel too.
    """
    n, heads, dim = q.shape if q.ndim == 3 else (0, 0, 0)
    rq = batch._row(q, "q")
    scores = _scores(batch, heads, dim, scale, causal, window, cap, slopes, prefix_lengths)
    scores.fp32_weights = bool(fp32_weights)
    flag = _flag_pointer(batch, error_flag)
    lib = _lib.load()
    with _On(batch, stream) as handle:
        if out is None:
            out = q.new_empty((n, heads, dim))
        rows = _TwoHeads(*rq, *batch._row(out, "out", n, heads))
        at = ctypes.addressof(rows)
        lse = q.new_empty((n, heads), dtype=torch.float32) if return_lse else None
        c = batch._tokens(n)
        need = ctypes.c_int64(0)
        scored = (batch._code, dim, ctypes.byref(scores))
        if batch.scales is None:
            _lib.check(lib.cb_attention_workspace_bytes(c, *scored, heads, ctypes.byref(need)))
        else:
            _lib.check(lib.cb_quantized_attention_workspace_bytes(c, batch._scales, *scored, heads, ctypes.byref(need)))
        work = q.new_empty(need.value, dtype=torch.uint8) if need.value else None
        to = (at, at + 32, None if lse is None else lse.data_ptr(), None if work is None else work.data_ptr(), need.value,
              flag, handle)
        if batch.scales is None:
            _lib.check(lib.cb_paged_attention(c, batch._layer(layer), *scored, *to))
        else:
            _lib.check(lib.cb_quantized_attention(c, batch._scales, batch._layer(layer), *scored, *to))
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
    _plain_pool(batch)
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


def _plain_pool(batch: QueryBatch) -> None:
    if batch.scales is not None:
        raise ValueError("8-bit pools are read by paged_attention alone; weigh and evict before quantize_tokens")


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
    _plain_pool(batch)
    _plain_pool(target)
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


def quantize_tokens(batch: QueryBatch, target: QueryBatch, *, out: torch.Tensor | None = None,
                    error_flag: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """Move the cached tokens of each request, all layers, to tokens 0, 1, ... of the same request of ``target``.

    ``target`` is a batch over unpublished pages of an 8-bit pool whose
    ``dtype`` is ``batch``'s, with a block table of the pool's page size and
    requests that start at a page's first slot (its lengths are not read; a token
    past its ``request_stride`` is not copied and sets ``ERROR_TARGET_ROW``).
    Every page and head gets the least scale that keeps its finite elements
    within 448 times it; slots behind a request's last token keep their codes.

    Returns int32 ``[requests]`` lengths (``out`` or a new tensor): a request's
    own, or 0 where it is outside the batch's bounds or some cached token has no
    row (``ERROR_REQUEST``, ``ERROR_CACHE_ROW``): its pages then hold in part
    what they held before.
    """
    _plain_pool(batch)
    if target.scales is None:
        raise ValueError("target must be a batch over an 8-bit pool")
    if target.device != batch.device or target.dtype != batch.dtype:
        raise ValueError("batch and target must share device and dtype")
    if target.requests != batch.requests:
        raise ValueError("batch and target must have the same requests")
    dim = batch.head_dim
    if target.kv_heads != batch.kv_heads or target.head_dim != dim or target.rows.num_layers != batch.rows.num_layers:
        raise ValueError("batch and target must share layers, KV heads and head_dim")
    flag = _flag_pointer(batch, error_flag)
    with _On(batch, stream) as handle:
        if out is None:
            out = torch.empty(batch.requests, dtype=torch.int32, device=batch.device)
        _lib.check(_lib.load().cb_quantize_tokens(
            batch._tokens(0), target._tokens(0), target._scales, batch._code, dim,
            _device_vector(out, "out", (torch.int32,), batch.device, batch.requests), flag, handle))
        batch.rows.hold_for(stream)
        target.rows.hold_for(stream)
    return out
