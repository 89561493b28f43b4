// Requests of a query batch, their cached tokens and rows, and the checks that
// every call on one makes: what the sources behind cb_query_batch share.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "../../include/cachebridge_hip.h"
#include "cb_common.h"

namespace {

typedef __bf16 io_bf16;
typedef _Float16 io_f16;
typedef float f32x16 __attribute__((ext_vector_type(16)));

// Helpers that take a request or a key range by reference are always inlined: a
// call would put the struct, and what the caller keeps, into scratch memory.
#define CB_INLINE __device__ __attribute__((always_inline)) inline

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -INFINITY;

// ---------------------------------------------------------------------------
// Requests, their cached tokens and their rows
// ---------------------------------------------------------------------------

struct QBatch {
  const int32_t* query_start;
  const int32_t* lengths;
  const int64_t* offsets;
  int64_t request_stride;
  int64_t index_offset;
  int64_t entries;
  const void* index;
  int64_t rows;
  int64_t row_stride_b;
  int32_t kind;
  int32_t page_size;
  int32_t page_shift;  // log2(page_size), or -1
  int32_t requests;
  int32_t tokens;
  int32_t max_query;
  int32_t max_length;
  int32_t* err;
};

struct Request {
  int q0;        // first token row
  int n;         // new tokens
  int length;    // cached tokens, the new ones included
  int64_t first; // index entry of cached token 0 (block tables: its page's)
  uint32_t rem;  // block tables: cached token 0's slot in its page
  bool ok;
};

CB_INLINE void flag(int32_t* err, int bits) {
  if (err) atomicOr(err, bits);
}

// The request's index position alone (eviction: no new tokens involved).
CB_INLINE void place_request(const QBatch& B, int b, Request& r) {
  const int64_t start = (B.offsets ? B.offsets[b] : b * B.request_stride);
  r.ok = start >= 0 && start <= (int64_t{1} << 61);
  const int64_t u = r.ok ? start + B.index_offset : 0;
  r.first = u;
  r.rem = 0;
  if (B.kind == CB_INDEX_BLOCK_TABLE) {
    r.first = B.page_shift >= 0 ? u >> B.page_shift : u / B.page_size;
    r.rem = static_cast<uint32_t>(u - r.first * B.page_size);
  }
}

// One request by itself. Whether an earlier one starts behind it is for its
// callers: own_request, or load_requests for 64 at a time.
CB_INLINE Request load_request(const QBatch& B, int b) {
  Request r;
  place_request(B, b, r);
  const int64_t q0 = B.query_start[b], q1 = B.query_start[b + 1];
  const int length = B.lengths[b];
  r.ok = r.ok && q0 >= 0 && q1 >= q0 && q1 <= B.tokens && q1 - q0 <= B.max_query && length <= B.max_length &&
         q1 - q0 <= length;
  r.q0 = static_cast<int>(q0);
  r.n = r.ok ? static_cast<int>(q1 - q0) : 0;
  r.length = r.ok ? length : 0;
  return r;
}

// Pool row of cached token j, or -1 where its index entry or the row it names
// is out of range. The arithmetic within a request is 32 bits wide (at most
// 2^30 tokens); the request's own start is 64.
CB_INLINE int64_t cache_row(const QBatch& B, const Request& r, int j) {
  int64_t row;
  if (B.kind == CB_INDEX_BLOCK_TABLE) {
    const uint32_t x = r.rem + static_cast<uint32_t>(j);
    const uint32_t page = B.page_shift >= 0 ? x >> B.page_shift : x / static_cast<uint32_t>(B.page_size);
    const int64_t e = r.first + page;
    if (e >= B.entries) return -1;
    const int64_t p = reinterpret_cast<const CB_GLOBAL int32_t*>(as_global(B.index))[e];
    row = p * B.page_size + static_cast<int64_t>(x - page * static_cast<uint32_t>(B.page_size));
    if (p < 0) return -1;
  } else {
    const int64_t e = r.first + j;
    if (B.kind == CB_INDEX_IDENTITY) {
      row = e;
    } else {
      if (e >= B.entries) return -1;
      row = B.kind == CB_INDEX_I32 ? reinterpret_cast<const CB_GLOBAL int32_t*>(as_global(B.index))[e]
                                   : reinterpret_cast<const CB_GLOBAL int64_t*>(as_global(B.index))[e];
    }
  }
  return row >= 0 && row < B.rows ? row : -1;
}

// Whether request b starts before an earlier one, b the same in all lanes:
// this lane's largest start of those up to b's is above b's in some lane. Where
// query starts fall, such a request is outside the bounds, which leaves requests
// that own rows apart from each other whatever the starts are. MANY: past the
// first 64, four starts a lane and load, for kernels of short workgroups (steps of
// 2048 requests of 300: 152 us for 163; 148 without a look at the earlier starts).
template <bool MANY>
CB_INLINE int starts_to(const QBatch& B, int b) {
  const int lane = threadIdx.x & (kWave - 1);
  const CB_GLOBAL int32_t* start = reinterpret_cast<const CB_GLOBAL int32_t*>(as_global(B.query_start));
  int top = start[min(lane, b)];
  if constexpr (MANY) {
    typedef int32_t four __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll 2
    for (int i = kWave; i < b; i += 4 * kWave) {
      const four x = *reinterpret_cast<const CB_GLOBAL four*>(start + min(i + 4 * lane, b - 3));
      top = max(max(top, max(x[0], x[1])), max(x[2], x[3]));
    }
  } else {
#pragma unroll 2
    for (int i = kWave; i < b; i += kWave) top = max(top, start[min(i + lane, b)]);
  }
  return top;
}

// Request b, the same in all lanes, with its place among the others (asked for
// ahead of its own fields, so that both wait together).
template <bool MANY = false>
CB_INLINE Request own_request(const QBatch& B, int b) {
  const int top = starts_to<MANY>(B, b);
  Request r = load_request(B, b);
  if (__any(top > r.q0)) {
    r.ok = false;
    r.n = r.length = 0;
  }
  return r;
}

// Requests b0 to b0 + 63, one a lane (past the last one: it again, without
// tokens), as own_request has them, for a wave that goes through all of them in
// order. top: the largest start so far, at first 0.
CB_INLINE Request load_requests(const QBatch& B, int b0, int& top) {
  const int lane = threadIdx.x & (kWave - 1), b = min(b0 + lane, B.requests - 1);
  Request r = load_request(B, b);
  const int start = r.q0;
  top = max(top, start);
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int up = __shfl_up(top, d);
    top = lane >= d ? max(top, up) : top;
  }
  const bool fell = top > start;
  r.ok = r.ok & !fell;
  r.n = (fell | (b0 + lane >= B.requests)) ? 0 : r.n;
  top = __shfl(top, kWave - 1);
  return r;
}

// Flags requests that are outside the bounds; called by one wave.
CB_INLINE void flag_requests(const QBatch& B) {
  int top = 0;
  for (int b0 = 0; b0 < B.requests; b0 += kWave)
    if (!load_requests(B, b0, top).ok) flag(B.err, CB_ERROR_REQUEST);
}

// A request of its fields, as load_request has it: its token rows, cached tokens and
// first index token.
CB_INLINE Request request_of(const QBatch& B, int64_t q0, int64_t q1, int length, int64_t start) {
  Request r;
  r.ok = start >= 0 && start <= (int64_t{1} << 61);
  const int64_t u = r.ok ? start + B.index_offset : 0;
  r.first = u;
  r.rem = 0;
  if (B.kind == CB_INDEX_BLOCK_TABLE) {
    r.first = B.page_shift >= 0 ? u >> B.page_shift : u / B.page_size;
    r.rem = static_cast<uint32_t>(u - r.first * B.page_size);
  }
  r.ok = r.ok && q0 >= 0 && q1 >= q0 && q1 <= B.tokens && q1 - q0 <= B.max_query && length <= B.max_length &&
         q1 - q0 <= length;
  r.q0 = static_cast<int>(q0);
  r.n = r.ok ? static_cast<int>(q1 - q0) : 0;
  r.length = r.ok ? length : 0;
  return r;
}

// Requests b0 to b0 + 63, one a lane, as they stand in memory.
struct Fields {
  int start, end, length;
  int64_t first;
};
CB_INLINE Fields load_fields(const QBatch& B, int b0) {
  const int b = min(b0 + static_cast<int>(threadIdx.x & (kWave - 1)), B.requests - 1);
  return {B.query_start[b], B.query_start[b + 1], B.lengths[b], B.offsets ? B.offsets[b] : b * B.request_stride};
}

// What lane `lane` (the same in all) holds.
CB_INLINE int lane_value(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }
CB_INLINE int64_t lane_value(int64_t x, int lane) {
  return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(lane_value(static_cast<int>(x >> 32), lane))) << 32 |
                              static_cast<uint32_t>(lane_value(static_cast<int>(x), lane)));
}

// The request that token row t belongs to; false if none does. The first whose
// rows hold t decides: if an earlier one starts behind it, so does one for any
// later that holds t. Called by whole waves, t the same in all lanes. f: the first
// 64 requests' fields, which a caller may have asked for ahead of other loads;
// the request is made of its lane's, with nothing more to wait for.
CB_INLINE bool request_of_row(const QBatch& B, int t, Fields f, Request& r) {
  const int lane = threadIdx.x & (kWave - 1);
  int top = -2147483647;  // this lane's starts so far
  for (int b0 = 0; b0 < B.requests; b0 += kWave) {
    if (b0) f = load_fields(B, b0);
    const uint64_t hit = __ballot((b0 + lane < B.requests) & (f.start <= t) & (t < f.end));
    if (hit) {
      const int l = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<unsigned long long>(hit)) - 1);
      const int mine = lane_value(f.start, l);
      if (__any((top > mine) | ((lane < l) & (f.start > mine)))) return false;
      r = request_of(B, mine, lane_value(f.end, l), lane_value(f.length, l), lane_value(f.first, l));
      return r.ok;
    }
    top = max(top, f.start);
  }
  return false;
}

// The request that token row t belongs to, or `requests` if none does. The
// first whose rows hold t decides: if an earlier one starts behind it, so does
// one for any later that holds t. Called by whole waves, t the same in all lanes.
CB_INLINE int request_of_token(const QBatch& B, int t) {
  const int lane = threadIdx.x & (kWave - 1);
  int top = -2147483647;  // this lane's starts so far
  for (int b0 = 0; b0 < B.requests; b0 += kWave) {
    const int b = min(b0 + lane, B.requests - 1);
    const int start = B.query_start[b], end = B.query_start[b + 1];
    const uint64_t hit = __ballot((b0 + lane < B.requests) & (start <= t) & (t < end));
    if (hit) {
      const int l = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<unsigned long long>(hit)) - 1);
      const int mine = __shfl(start, l);
      return __any((top > mine) | ((lane < l) & (start > mine))) ? B.requests : b0 + l;
    }
    top = max(top, start);
  }
  return B.requests;
}

// ---------------------------------------------------------------------------
// Elements
// ---------------------------------------------------------------------------

template <typename IO>
__device__ inline float to_f32(IO x) {
  return static_cast<float>(x);
}
template <typename IO>
__device__ inline IO from_f32(float x) {
  return static_cast<IO>(x);  // round to nearest even
}
template <typename IO>
__device__ inline IO load_elem(const char* p) {
  return gload<IO>(as_global(static_cast<const void*>(p)));
}
template <typename IO>
__device__ inline void store_elem(char* p, IO v) {
  gstore<IO>(as_global(static_cast<void*>(p)), v);
}

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ inline float log2_fast(float x) { return __builtin_amdgcn_logf(x); }

struct Strided {
  char* data;
  int64_t token_b, head_b;
};

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

int elem_bytes(int32_t dtype) {
  return dtype == CB_DTYPE_F32 ? 4 : dtype == CB_DTYPE_BF16 || dtype == CB_DTYPE_F16 ? 2 : 0;
}

// Index entries that are a request's own: with starts request_stride apart, its
// stride, and what lies behind belongs to the next request. Offsets are the
// caller's, one request has the index to itself, and a stride of zero shares
// one history among all (which calls that store rows refuse).
int64_t request_span(const cb_query_batch& b) {
  return b.offsets || b.num_requests < 2 || b.request_stride == 0 ? int64_t{1} << 30 : b.request_stride;
}

bool shares_rows(const cb_query_batch& b) { return !b.offsets && b.num_requests > 1 && b.request_stride == 0; }

// cache_bytes: bytes of an element of the cache where they are not dtype's.
int check_batch(const cb_query_batch* batch, int32_t dtype, int32_t head_dim, int32_t* err, bool queries, QBatch* B,
                DevRows* rows, int cache_bytes = 0) {
  if (!batch) return fail(CB_EINVAL, "null batch");
  if (!elem_bytes(dtype)) return fail(CB_EINVAL, "bad dtype");
  const int eb = cache_bytes ? cache_bytes : elem_bytes(dtype);
  if (head_dim < 2 || head_dim > 512 || head_dim % 2) return fail(CB_EINVAL, "head_dim must be even, 2 to 512");
  int rc;
  if ((rc = to_dev_rows(batch->cache, eb, rows, eb))) return rc;
  const cb_rows& c = batch->cache;
  if (c.heads < 1) return fail(CB_EINVAL, "the cache needs KV heads");
  if (c.head_offset != 0) return fail(CB_EINVAL, "the cache's head_offset must be 0");
  if (c.row_stride < static_cast<int64_t>(c.heads) * head_dim)
    return fail(CB_EINVAL, "the cache's rows are shorter than heads * head_dim");
  if (c.rows > 0x7fffffff) return fail(CB_EINVAL, "more than 2^31 - 1 cache rows");
  if (c.index_kind == CB_INDEX_BLOCK_TABLE && c.page_size > (1 << 20)) return fail(CB_EINVAL, "page_size above 2^20");
  if (c.index_kind != CB_INDEX_IDENTITY && batch->index_entries < 0) return fail(CB_EINVAL, "negative index_entries");
  if (batch->num_requests < 0 || batch->num_tokens < 0) return fail(CB_EINVAL, "negative batch size");
  if (batch->request_stride < 0) return fail(CB_EINVAL, "negative request_stride");
  if (batch->request_stride > (int64_t{1} << 31)) return fail(CB_EINVAL, "request_stride above 2^31");
  if (batch->max_length < 0 || batch->max_length > (1 << 30)) return fail(CB_EINVAL, "max_length must be 0 to 2^30");
  if (batch->num_requests > 0 && (!batch->lengths || (queries && !batch->query_start)))
    return fail(CB_EINVAL, "null query_start or lengths");
  if (queries && (batch->max_query < 0 || batch->max_query > batch->num_tokens))
    return fail(CB_EINVAL, "max_query must be 0 to num_tokens");
  B->query_start = batch->query_start;
  B->lengths = batch->lengths;
  B->offsets = batch->offsets;
  B->request_stride = batch->request_stride;
  B->index_offset = c.index_offset;
  B->entries = batch->index_entries;
  B->index = c.index;
  B->rows = c.rows;
  B->row_stride_b = rows->row_stride_b;
  B->kind = c.index_kind;
  B->page_size = c.index_kind == CB_INDEX_BLOCK_TABLE ? c.page_size : 1;
  B->page_shift = (B->page_size & (B->page_size - 1)) ? -1 : __builtin_ctz(static_cast<unsigned>(B->page_size));
  B->requests = batch->num_requests;
  B->tokens = batch->num_tokens;
  B->max_query = batch->max_query;
  B->max_length = static_cast<int32_t>(std::min<int64_t>(batch->max_length, request_span(*batch)));
  B->err = err;
  return CB_OK;
}

int check_heads(const char* name, const cb_heads* h, int32_t heads, int eb, int32_t tokens, Strided* out) {
  if (!h) return fail(CB_EINVAL, "null %s", name);
  if (h->heads != heads) return fail(CB_EINVAL, "%s has %d heads, %d expected", name, h->heads, heads);
  if (tokens > 0 && !h->data) return fail(CB_EINVAL, "null %s data", name);
  if (h->token_stride < 0 || h->head_stride < 0) return fail(CB_EINVAL, "negative stride of %s", name);
  if (reinterpret_cast<uintptr_t>(h->data) % eb) return fail(CB_EINVAL, "%s is not aligned to its elements", name);
  *out = Strided{static_cast<char*>(h->data), h->token_stride * eb, h->head_stride * eb};
  return CB_OK;
}

// Whether two rows of a token tensor lie on one another: rows of an output that
// do would be stored by several workgroups at once.
bool rows_overlap(const cb_heads& h, int64_t tokens, int64_t dim) {
  const int64_t ts = h.token_stride, hs = h.head_stride;
  if (tokens < 2 && h.heads < 2) return false;
  if ((hs >= dim || h.heads < 2) && (ts >= (h.heads - 1) * hs + dim || tokens < 2)) return false;  // heads within tokens
  if ((ts >= dim || tokens < 2) && (hs >= (tokens - 1) * ts + dim || h.heads < 2)) return false;   // tokens within heads
  if (tokens > 1 && ts < dim) return true;
  for (int64_t i = 1; i < h.heads; ++i) {  // head i of token 0 against the tokens of head 0 beside it
    const int64_t at = i * hs, t = ts > 0 ? std::min(at / ts, tokens - 1) : 0;
    if (at - t * ts < dim || (t + 1 < tokens && (t + 1) * ts - at < dim)) return true;
  }
  return false;
}

int check_output(const char* name, const cb_heads* h, int32_t heads, int eb, int32_t tokens, int32_t dim, Strided* out) {
  if (int rc = check_heads(name, h, heads, eb, tokens, out)) return rc;
  if (rows_overlap(*h, tokens, dim)) return fail(CB_EINVAL, "%s has rows that share memory", name);
  return CB_OK;
}

bool aligned16(const Strided& s) {
  return (reinterpret_cast<uintptr_t>(s.data) | static_cast<uintptr_t>(s.token_b) | static_cast<uintptr_t>(s.head_b)) % 16 == 0;
}

// Pools of one buffer per layer hold allocations of their own, which are
// 16-byte aligned; a stacked pool's bases and layer stride are checked.
bool rows_aligned16(const DevRows& r, int head_bytes) {
  if (r.row_stride_b % 16 || head_bytes % 16) return false;
  if (r.k_layers) return true;
  return (reinterpret_cast<uintptr_t>(r.k_base) | reinterpret_cast<uintptr_t>(r.v_base) | static_cast<uintptr_t>(r.layer_stride_b)) % 16 == 0;
}

// HIP counts a launch's threads in 32 bits.
bool launch_fits(int64_t workgroups, int threads) { return workgroups <= 0xffffffffll / threads; }

int ceil_div(int64_t a, int64_t b) { return static_cast<int>((a + b - 1) / b); }

}  // namespace
