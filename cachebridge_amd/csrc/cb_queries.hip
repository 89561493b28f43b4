// Queries on an installed prefix for MI355X (gfx950): new tokens rotated and
// stored into a paged cache, attention over it, the attention each cached
// token got, and eviction by it. The C ABI is in include/cachebridge_hip.h.
//
// Layout shared by the score kernels. A request's new tokens and the G query
// heads of one KV head form rows r = i * G + g of one matrix (i: new token),
// so that K and V are read once per KV head whatever the number of heads and
// new tokens. Scores are computed transposed, S^T = K Q^T: an MFMA result
// holds one query row per lane and several keys per lane, so the softmax
// statistics of a row stay in its lane (plus one exchange among the lanes that
// share the row), and P^T is the next product's second operand as it stands:
// O^T += V^T P^T sums over keys, whose order within a step is free as long as
// both operands use the same one.

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

// ---------------------------------------------------------------------------
// New tokens: rotation and store
// ---------------------------------------------------------------------------

struct Strided {
  char* data;
  int64_t token_b, head_b;
};

struct InstallArgs {
  QBatch batch;
  DevRows cache;
  int32_t layer;
  int32_t head_dim, rotary_dim, interleaved;
  int32_t q_heads, kv_heads;
  int32_t slices;  // waves per token
  Strided q, q_out, k, v;
  const double* inv_freq;
  const void* positions;
  int32_t positions_kind;
  float magnitude;
};

constexpr int kInstallWaves = 4;
constexpr int kMaxPairs = 256;  // head_dim <= 512

// sin and cos of `turns` revolutions. The angle is reduced to an eighth of a
// turn either side of a quarter's multiple in 64 bits (positions times a
// frequency reach thousands of radians, where 32 bits leave no digits of the
// phase), then both are Taylor polynomials, |x| <= pi/4: in fp32 for 16-bit
// rows, first terms left out x^11/11! and x^12/12! below 2^-29; in fp64 for fp32
// rows, x^15/15! and x^16/16! below 2^-45.
template <typename T>
__device__ inline void sincos_turns(double turns, T* sn, T* cs) {
  const double q = __builtin_rint(turns * 4.0);
  const T x = static_cast<T>((turns - q * 0.25) * 6.283185307179586476925);
  const int quadrant = static_cast<int>(static_cast<int64_t>(q) & 3);
  const T y = x * x, one = 1;
  T s = 0, c = 0;
  if constexpr (sizeof(T) == 8) {
    s = y * y * (one / -39916800 + y * (one / 6227020800));
    c = y * y * (one / 479001600 + y * (one / -87178291200));
  }
  s = x + x * y * (-one / 6 + y * (one / 120 + y * (-one / 5040 + y * (one / 362880) + s)));
  c = one + y * (-one / 2 + y * (one / 24 + y * (-one / 720 + y * (one / 40320 + y * (-one / 3628800) + c))));
  const T a = (quadrant & 1) ? c : s, b = (quadrant & 1) ? s : c;
  *sn = (quadrant & 2) ? -a : a;
  *cs = (quadrant == 1 || quadrant == 2) ? -b : b;
}

// V elements as one access where V * sizeof(IO) is 16, else element by element.
template <typename IO, int V>
__device__ inline void load_vec(const char* p, float* out) {
  if constexpr (V * sizeof(IO) == 16) {
    typedef IO vec __attribute__((ext_vector_type(V)));
    const vec x = gload<vec>(as_global(static_cast<const void*>(p)));
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = static_cast<float>(x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = to_f32(load_elem<IO>(p + i * sizeof(IO)));
  }
}
template <typename IO, int V>
__device__ inline void store_vec(char* p, const float* in) {
  if constexpr (V * sizeof(IO) == 16) {
    typedef IO vec __attribute__((ext_vector_type(V)));
    vec x;
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = from_f32<IO>(in[i]);
    gstore<vec>(as_global(static_cast<void*>(p)), x);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) store_elem<IO>(p + i * sizeof(IO), from_f32<IO>(in[i]));
  }
}

// y_a = x_a cos - x_b sin, y_b = x_b cos + x_a sin for the pairs (a, b) of the
// rotated part, angles position * inv_freq. One wave per (token, slice of its
// heads' elements): lanes compute the token's angles once into LDS, then each
// item is V pairs of a head (two vectors) or V elements that are copied; slices
// are cut to an item a lane, so that a wave waits for memory once. Every element
// is read once and written once. 64 tokens of 64 query and 8 KV heads of 128 in bf16
// take 4.8 us, the latency of a launch and of three dependent loads; 2048 of 16
// and 2 (21 MB) 9.3 us, that latency and the bytes' time at a copy's rate.
template <typename IO, int V>
__global__ __launch_bounds__(kInstallWaves * kWave) void install_tokens_kernel(InstallArgs a) {
  // fp32 rows are rotated in fp64 and rounded once: in fp32 the cosine, sine and two
  // products would each round to the digits that are stored (2048 tokens of 16 and 2
  // heads of 128 13.9 us for 13.6).
  typedef std::conditional_t<sizeof(IO) == 4, double, float> T;
  typedef T pair __attribute__((ext_vector_type(2)));
  __shared__ pair turn[kInstallWaves][kMaxPairs];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kInstallWaves + wave;
  if (a.batch.err && blockIdx.x == gridDim.x - 1) {  // a workgroup more than there are tokens for
    if (wave == 0) flag_requests(a.batch);
    return;
  }
  const int t = static_cast<int>(unit / a.slices), slice = static_cast<int>(unit % a.slices);
  if (t >= a.batch.tokens) return;
  const int b = request_of_token(a.batch, t);
  if (b >= a.batch.requests) return;
  const Request r = load_request(a.batch, b);
  if (!r.ok) return;
  const int p = r.length - r.n + (t - r.q0);
  const int64_t row = cache_row(a.batch, r, p);
  if (row < 0 && lane == 0) flag(a.batch.err, CB_ERROR_TARGET_ROW);
  int64_t pos = p;
  if (a.positions)
    pos = a.positions_kind == CB_INDEX_I64 ? static_cast<const int64_t*>(a.positions)[t]
                                           : static_cast<const int32_t*>(a.positions)[t];
  const int pairs = a.rotary_dim / 2;
  for (int i = lane; i < pairs; i += kWave) {
    T s, c;
    sincos_turns(static_cast<double>(pos) * a.inv_freq[i] * 0.15915494309189533577, &s, &c);
    turn[wave][i] = pair{c * a.magnitude, s * a.magnitude};
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const int rot_items = pairs / V, pass_items = (a.head_dim - a.rotary_dim) / V, head_items = rot_items + pass_items;
  const int v_items = a.head_dim / V;
  const int turned = (a.q_heads + a.kv_heads) * head_items;
  const int total = turned + a.kv_heads * v_items;
  const int per = (total + a.slices - 1) / a.slices;
  const int stop = min(total, (slice + 1) * per);
  char* krow = const_cast<char*>((const char*)layer_base(a.cache, 0, a.layer)) + row * a.cache.row_stride_b;
  char* vrow = const_cast<char*>((const char*)layer_base(a.cache, 1, a.layer)) + row * a.cache.row_stride_b;
  constexpr int E = sizeof(IO);
  for (int idx = slice * per + lane; idx < stop; idx += kWave) {
    const char* src;
    char* dst;
    int item;
    if (idx < turned) {
      const int head = idx / head_items;
      item = idx - head * head_items;
      if (head < a.q_heads) {
        src = a.q.data + t * a.q.token_b + head * a.q.head_b;
        dst = a.q_out.data + t * a.q_out.token_b + head * a.q_out.head_b;
      } else {
        src = a.k.data + t * a.k.token_b + (head - a.q_heads) * a.k.head_b;
        dst = krow + static_cast<int64_t>(head - a.q_heads) * a.head_dim * E;
        if (row < 0) continue;
      }
    } else {
      if (row < 0) continue;
      const int head = (idx - turned) / v_items;
      const int off = (idx - turned - head * v_items) * V;
      float x[V];
      load_vec<IO, V>(a.v.data + t * a.v.token_b + head * a.v.head_b + off * E, x);
      store_vec<IO, V>(vrow + (static_cast<int64_t>(head) * a.head_dim + off) * E, x);
      continue;
    }
    if (item >= rot_items) {
      const int off = a.rotary_dim + (item - rot_items) * V;
      float x[V];
      load_vec<IO, V>(src + off * E, x);
      store_vec<IO, V>(dst + off * E, x);
      continue;
    }
    const int first = item * V;
    const int oa = a.interleaved ? 2 * first : first, ob = a.interleaved ? oa + V : first + pairs;
    float x[2 * V], y[2 * V];
    load_vec<IO, V>(src + oa * E, x);
    load_vec<IO, V>(src + ob * E, x + V);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const pair cs = turn[wave][first + i];
      if (a.interleaved) {
        y[2 * i] = static_cast<float>(x[2 * i] * cs.x - x[2 * i + 1] * cs.y);
        y[2 * i + 1] = static_cast<float>(x[2 * i + 1] * cs.x + x[2 * i] * cs.y);
      } else {
        y[i] = static_cast<float>(x[i] * cs.x - x[i + V] * cs.y);
        y[i + V] = static_cast<float>(x[i + V] * cs.x + x[i] * cs.y);
      }
    }
    store_vec<IO, V>(dst + oa * E, y);
    store_vec<IO, V>(dst + ob * E, y + V);
  }
}

// ---------------------------------------------------------------------------
// Scores: tiles of query rows, the cached tokens they see
// ---------------------------------------------------------------------------

struct ScoreArgs {
  QBatch batch;
  DevRows cache;
  int32_t layer;
  int32_t head_dim, q_heads, kv_heads, group;
  Strided q;
  float scale, cap;
  int32_t window, causal;
  const float* slopes;
  const int32_t* prefix;
  float inner;   // scale / cap, finite
  float gentle;  // raw products below it have |inner x| < kSmallAngle
  int32_t mod;  // scores are more than a product times a positive scale
};

struct AttendArgs {
  ScoreArgs s;
  Strided out;
  float* lse;
  float* part_out;   // [splits][tokens * q_heads][head_dim], each normalised
  float* part_lse;   // [splits][tokens * q_heads], log2
  int32_t tile_slots;     // query tiles launched per KV head
  int32_t request_slots;  // tiles per request if tiles are laid out by request, else 0
  int32_t splits;       // workgroups that may share a tile's keys
  int32_t least_tiles;  // key tiles that each has at least
  uint32_t by_splits;   // ceil(2^32 / splits), or 0: all have least_tiles
};

// Tile `i` of the launch: its request, and which of the request's tiles (the
// last first: under a causal mask it has the most keys). Returns false if
// there is none.
template <bool MANY = false>
CB_INLINE bool find_tile(const AttendArgs& a, int i, int rows_per_tile, Request& r, int& b, int& tile) {
  const QBatch& B = a.s.batch;
  const int G = a.s.group;
  if (a.request_slots > 0) {
    b = i / a.request_slots;
    r = own_request<MANY>(B, b);
    const int tiles = static_cast<int>((static_cast<int64_t>(r.n) * G + rows_per_tile - 1) / rows_per_tile);
    tile = tiles - 1 - (i - b * a.request_slots);
    if (!r.ok && threadIdx.x == 0 && i == b * a.request_slots) flag(B.err, CB_ERROR_REQUEST);
    return tile >= 0;
  }
  const int lane = threadIdx.x & (kWave - 1);
  int64_t before = 0;
  int top = 0;
  for (int b0 = 0; b0 < B.requests; b0 += kWave) {
    const Request m = load_requests(B, b0, top);
    // The last place looks at every request: where one is left out, the others'
    // tiles end before it (their rows' whole tiles and one more each).
    if (i == a.tile_slots - 1 && !m.ok && threadIdx.x < kWave) flag(B.err, CB_ERROR_REQUEST);
    int64_t sum = (static_cast<int64_t>(m.n) * G + rows_per_tile - 1) / rows_per_tile;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int64_t up = __shfl_up(sum, d);
      if (lane >= d) sum += up;
    }
    const uint64_t hit = __ballot(before + sum > i);
    if (hit) {
      const int l = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<unsigned long long>(hit)) - 1);
      b = b0 + l;
      r = load_request(B, b);
      const int64_t end = before + __shfl(sum, l);
      tile = static_cast<int>(end - 1 - i);
      return true;
    }
    before += __shfl(sum, kWave - 1);
  }
  return false;
}

// Cached tokens that query rows [row0, row1] of a request may see: [0, na) if
// a prefix stands apart from the window, then [lb, hb). They are walked in
// tiles of KT keys, those of the prefix first.
struct KeyRange {
  int na, lb, hb;
  int ta, tiles;
  int np;      // prefix length within the cache
  int p0, p1;  // cached token of the first and last row
};

template <int KT>
CB_INLINE KeyRange key_range(const ScoreArgs& s, const Request& r, int b, int row0, int row1) {
  KeyRange k;
  k.np = s.prefix ? max(0, min(s.prefix[b], r.length)) : 0;
  k.p0 = r.length - r.n + row0 / s.group;
  k.p1 = r.length - r.n + row1 / s.group;
  const int lo = s.window > 0 ? max(0, k.p0 - s.window + 1) : 0;
  const int hi = s.causal ? k.p1 + 1 : r.length;
  k.na = s.window > 0 ? min(k.np, lo) : 0;
  k.lb = lo;
  k.hb = max(hi, k.np);
  if (k.np < lo) k.hb = hi;
  k.ta = (k.na + KT - 1) / KT;
  k.tiles = k.ta + (k.hb - k.lb + KT - 1) / KT;
  return k;
}

template <int KT>
CB_INLINE int tile_start(const KeyRange& k, int t) {
  return t < k.ta ? t * KT : k.lb + (t - k.ta) * KT;
}
CB_INLINE int tile_end(const KeyRange& k, int t) { return t < k.ta ? k.na : k.hb; }

// Key tiles of each split of a tile that has `tiles`: its own keys in equal
// parts, whatever the bound that the launch was made for (64 new tokens over 4096
// in 8 requests, with parts cut by a bound of 32768: 131 us; by their own keys 35).
// The product is the quotient, or more by its 32 bits' error.
CB_INLINE int split_tiles(const AttendArgs& a, int tiles) {
  if (a.splits == 1) return tiles;
  return max(a.least_tiles, static_cast<int>(__umulhi(static_cast<uint32_t>(tiles + a.splits - 1), a.by_splits)));
}

// Whether every row of the tile sees every key of [start, stop).
CB_INLINE bool sees_all(const ScoreArgs& s, const KeyRange& k, int start, int stop) {
  if (stop <= k.np) return true;
  return (!s.causal || stop <= k.p0 + 1) && (s.window == 0 || start > k.p1 - s.window);
}

// Without branches (bitwise operators): lanes differ in p and j.
CB_INLINE bool sees(const ScoreArgs& s, const KeyRange& k, int p, int j) {
  const int above = s.window > 0 ? p - s.window : -1, below = s.causal ? p : 0x7fffffff;
  return (j < k.np) | ((j <= below) & (j > above));
}

// tanh y = y + y t q(t) with t = y^2, for |y| < kSmallAngle: q is the polynomial
// of third degree whose largest relative error in tanh is least (1.2e-7, by the
// exchange of extrema). The forms of exp(2y) that serve above are off by some
// 2^-22 of the cap: a cap of 10^4 would leave a score of 10 eleven of its bits.
constexpr float kSmallAngle = 0.625f;
constexpr float kTanh3 = -0.3333234124f, kTanh5 = 0.1330817506f, kTanh7 = -0.05194790459f, kTanh9 = 0.01519537339f;
CB_INLINE float tanh_rest(float t) {  // t q(t)
  return t * __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(kTanh9, t, kTanh7), t, kTanh5), t, kTanh3);
}

// cap * tanh(x / cap); away from zero tanh y = (1 - e) / (1 + e), e = exp(-2|y|).
CB_INLINE float capped(float x, float cap) {
  const float y = x / cap;
  if (fabsf(y) < kSmallAngle) return __builtin_fmaf(x, tanh_rest(y * y), x);
  const float e = exp2_fast(-2.0f * kLog2e * fabsf(y));
  return copysignf(cap * (1.0f - e) / (1.0f + e), x);
}

// A raw product's score, in natural units.
CB_INLINE float natural_score(const ScoreArgs& s, float dot, float slope, int p, int j) {
  float x = dot * s.scale;
  if (s.cap > 0) x = capped(x, s.cap);
  return x - slope * fabsf(static_cast<float>(p - j));
}

// Raw products of one lane (16 keys of a block that starts at cached token
// `start`, register e: key 8 (e / 4) + 4 h + e % 4) to scores times `unit`.
// Capped: where no lane's angle reaches kSmallAngle, which is the rule, the
// polynomial (READY: by factors made ahead, four registers, seven instructions,
// else nine). A block of 32 rows and keys with larger ones takes tanh y = 1 - 2 /
// (exp(2y) + 1), two transcendental operations that hold for either sign: it is
// off by 3 2^-23 of the cap, so by less than 2^-20 of the block's largest score,
// where the products' own sums are off by more. 8192 tokens with 16 heads of 128 take
// 419 us with blocks of the first kind and 428 with all of the second; with a
// selection by element the latter took 599, with the second form alone both 414.
template <bool READY>
CB_INLINE void modify_scores(const ScoreArgs& s, f32x16& x, float unit, float slope, int p, int start, int h) {
  const float by = s.scale * unit;
  if (s.cap > 0) {
    float far = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) far = fmaxf(far, fabsf(x[e]));
    if (__all(far < s.gentle)) {
      const float k3 = kTanh3 * by, k5 = kTanh5 * by, k7 = kTanh7 * by, k9 = kTanh9 * by;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float y = x[e] * s.inner, t = y * y, w = x[e] * by;
        if constexpr (READY)
          x[e] *= __builtin_fmaf(t, __builtin_fmaf(t, __builtin_fmaf(t, __builtin_fmaf(t, k9, k7), k5), k3), by);
        else
          x[e] = __builtin_fmaf(w, tanh_rest(t), w);
        if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      const float in = 2.0f * kLog2e * s.inner, out = s.cap * unit;
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = __builtin_fmaf(-2.0f * out, __builtin_amdgcn_rcpf(exp2_fast(x[e] * in) + 1.0f), out);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] *= by;
  }
  if (s.slopes) {
    const float by = slope * unit, away = static_cast<float>(p - start - 4 * h);
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = __builtin_fmaf(-by, fabsf(away - static_cast<float>(8 * (e >> 2) + (e & 3))), x[e]);
  }
}

// ---------------------------------------------------------------------------
// Rows of a tile's keys
// ---------------------------------------------------------------------------

// A tile's pool rows in LDS: one wave resolves them, a key a lane, so that the
// waves that stage the tile only look them up.
template <int KT, int SLOTS = 4>
struct TileRows {
  int row[SLOTS][KT];  // pool row of each key of tile t in slot t % SLOTS, 0 where there is none
  uint32_t valid[SLOTS][(KT + 31) / 32];  // keys that are there
};

// The index word that names key `lane` of a tile, loaded a tile before it is
// needed (identity: the row itself; -1 past the end).
template <int KT>
CB_INLINE int64_t fetch_entry(const QBatch& B, const Request& r, int start, int end) {
  const int j = start + (threadIdx.x & (kWave - 1));
  int64_t e = r.first + j;
  if (B.kind == CB_INDEX_IDENTITY) return j < end ? e : -1;
  if (B.kind == CB_INDEX_BLOCK_TABLE) {
    const uint32_t x = r.rem + static_cast<uint32_t>(j);
    e = r.first + (B.page_shift >= 0 ? x >> B.page_shift : x / static_cast<uint32_t>(B.page_size));
  }
  const bool in = (j < end) & (e < B.entries);
  if (B.entries <= 0) return -1;
  const int64_t at = in ? e : 0;
  const int64_t got = B.kind == CB_INDEX_I64 ? reinterpret_cast<const CB_GLOBAL int64_t*>(as_global(B.index))[at]
                                             : reinterpret_cast<const CB_GLOBAL int32_t*>(as_global(B.index))[at];
  return in ? got : -1;
}

template <int KT, int SLOTS>
CB_INLINE void place_rows(const QBatch& B, const Request& r, int64_t entry, int start, int end, TileRows<KT, SLOTS>& rows, int slot) {
  const int lane = threadIdx.x & (kWave - 1), j = start + lane;
  int64_t row = entry;
  if (B.kind == CB_INDEX_BLOCK_TABLE) {
    const uint32_t x = r.rem + static_cast<uint32_t>(j), ps = static_cast<uint32_t>(B.page_size);
    row = row < 0 ? -1 : row * ps + (B.page_shift >= 0 ? x & (ps - 1) : x % ps);
  }
  const bool ok = (row >= 0) & (row < B.rows) & (lane < KT) & (j < end);
  if (__any(!ok & (j < end) & (lane < KT))) flag(B.err, CB_ERROR_CACHE_ROW);
  if (lane < KT) rows.row[slot][lane] = ok ? static_cast<int>(row) : 0;
  const uint64_t valid = __ballot(ok);
  if (lane < (KT + 31) / 32) rows.valid[slot][lane] = static_cast<uint32_t>(valid >> (32 * lane));
}

// ---------------------------------------------------------------------------
// General attention: any even head_dim up to 512, any type, fp32 products
// (16x16x4 MFMA: lane l holds A[l % 16][l / 16] and B[l / 16][l % 16], its
// result rows 4 (l / 16) + e of column l % 16). A workgroup's four waves share
// tiles of 16 keys in LDS, 16 query rows each; the next tile's elements are
// loaded into registers (VE at a time: 16 bytes where rows allow it, else one)
// while a tile is used. Rows in LDS are DP + 4 floats apart, which puts the 16
// rows and 4 columns of an operand in distinct banks. A prompt of 250 fp32
// tokens with 4 heads of 64 takes 14.0 us and its join 5.8 us: at this size the
// two barriers and the row lookup of each tile bound it, not its 37 MFLOP; with
// a tile's loads waited for in place it was 41 us.
// ---------------------------------------------------------------------------

constexpr int kAnyWaves = 4;
constexpr int kAnyRows = 16 * kAnyWaves;
constexpr int kAnyKeys = 16;

__device__ inline f32x4 mfma4(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// Elements 4 e + g of a row of `dim`, zeros past it; loaded at clamped places
// and selected after, so that no load waits for another.
template <typename IO, int N>
CB_INLINE void load_spread(const char* row, int dim, int g, float (&x)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) x[e] = to_f32(load_elem<IO>(row + min(4 * e + g, dim - 1) * static_cast<int>(sizeof(IO))));
#pragma unroll
  for (int e = 0; e < N; ++e) x[e] = 4 * e + g < dim ? x[e] : 0.0f;
}

__device__ inline bool not_finite(float x) { return !(fabsf(x) < INFINITY); }

template <typename IO, int DP, int VE>
__global__ __launch_bounds__(kAnyWaves * kWave, DP == 64 ? 3 : DP == 128 ? 2 : 1) void attend_any_kernel(AttendArgs a) {
  constexpr int KT = kAnyKeys, LD = DP + 4, NB = DP / 16, NT = kAnyWaves * kWave, MW = DP / 32;
  // A 512-element row's sums and queries fill the registers: no tile waits there.
  constexpr bool AHEAD = DP <= 256;
  constexpr int NC = AHEAD ? (KT * DP / VE + NT - 1) / NT : 1;
  typedef IO vec __attribute__((ext_vector_type(VE)));
  __shared__ __align__(16) float lk[KT * LD];
  __shared__ __align__(16) float lv[KT * LD];
  __shared__ TileRows<KT> tile_rows;
  __shared__ uint32_t marks[2][kAnyRows * MW];
  __shared__ uint32_t odd[2];
  const ScoreArgs& s = a.s;
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int c = lane & 15, g = lane >> 4;
  const int head = blockIdx.x % s.kv_heads;
  const int rest = blockIdx.x / s.kv_heads;
  const int split = rest / a.tile_slots;
  Request r;
  int b, tile;
  if (!find_tile(a, rest % a.tile_slots, kAnyRows, r, b, tile)) return;
  const int rows = r.n * s.group;
  const int row0 = tile * kAnyRows, row1 = min(rows, row0 + kAnyRows) - 1;
  const KeyRange kr = key_range<KT>(s, r, b, row0, row1);
  const int per = split_tiles(a, kr.tiles), t0 = split * per, t1 = min(kr.tiles, t0 + per);
  if (a.splits > 1 && t0 >= t1) return;

  auto entry_of = [&](int t) { return t < t1 ? fetch_entry<KT>(s.batch, r, tile_start<KT>(kr, t), tile_end(kr, t)) : -1; };
  auto place = [&](int64_t entry, int t) {
    if (t < t1) place_rows(s.batch, r, entry, tile_start<KT>(kr, t), tile_end(kr, t), tile_rows, t & 3);
  };
  int64_t entry = -1;
  if (wave == 0) {
    const int64_t e0 = entry_of(t0), e1 = entry_of(t0 + 1);
    entry = entry_of(t0 + 2);
    place(e0, t0);
    place(e1, t0 + 1);
  }
  // Elements past head_dim are zeros for good: no tile writes them.
  for (int x = threadIdx.x; x < KT * LD; x += NT) lk[x] = lv[x] = 0.0f;
  for (int x = threadIdx.x; x < 2 * kAnyRows * MW; x += NT) (&marks[0][0])[x] = 0;
  if (threadIdx.x < 2) odd[threadIdx.x] = 0;

  const int row = row0 + 16 * wave + c;  // this lane's query row
  const bool live = row < rows;
  const int i = min(row, rows - 1) / s.group;
  const int qh = head * s.group + min(row, rows - 1) - i * s.group;
  const int p = r.length - r.n + i;
  const int D = s.head_dim;
  const char* qp = s.q.data + static_cast<int64_t>(r.q0 + i) * s.q.token_b + qh * s.q.head_b;
  float q[DP / 4];
  load_spread<IO>(qp, D, g, q);
  const float slope = s.slopes ? s.slopes[qh] : 0.0f;

  gcptr kbase = layer_base(s.cache, 0, s.layer) + static_cast<int64_t>(head) * D * sizeof(IO);
  gcptr vbase = layer_base(s.cache, 1, s.layer) + static_cast<int64_t>(head) * D * sizeof(IO);
  const int per_row = D / VE;
  int key_of[NC], elem_of[NC];  // this thread's chunks of a tile
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int x = n * NT + threadIdx.x;
    key_of[n] = x / per_row;
    elem_of[n] = (x - key_of[n] * per_row) * VE;
  }
  vec rk[NC], rv[NC];
  auto load = [&](int t) __attribute__((always_inline)) {
    if constexpr (!AHEAD) return;
    const uint32_t valid = tile_rows.valid[t & 3][0];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const bool in = (key_of[n] < KT) && ((valid >> key_of[n]) & 1);
      rk[n] = rv[n] = vec(static_cast<IO>(0.0f));
      if (in) {
        const int64_t off = static_cast<int64_t>(tile_rows.row[t & 3][key_of[n]]) * s.batch.row_stride_b + elem_of[n] * static_cast<int>(sizeof(IO));
        rk[n] = gload<vec>(kbase + off);
        rv[n] = gload<vec>(vbase + off);
      }
    }
  };
  auto store = [&](int t) __attribute__((always_inline)) {
    if constexpr (!AHEAD) {
      const uint32_t valid = tile_rows.valid[t & 3][0];
#pragma unroll 1
      for (int k = wave; k < KT; k += kAnyWaves) {
        const bool in = (valid >> k) & 1;
        const int64_t off = static_cast<int64_t>(tile_rows.row[t & 3][k]) * s.batch.row_stride_b;
#pragma unroll 2
        for (int d = lane; d < D; d += kWave) {
          lk[k * LD + d] = in ? static_cast<float>(gload<IO>(kbase + off + d * static_cast<int>(sizeof(IO)))) : 0.0f;
          lv[k * LD + d] = in ? static_cast<float>(gload<IO>(vbase + off + d * static_cast<int>(sizeof(IO)))) : 0.0f;
        }
      }
      return;
    }
#pragma unroll
    for (int n = 0; n < NC; ++n)
      if (key_of[n] < KT) {
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          lk[key_of[n] * LD + elem_of[n] + e] = static_cast<float>(rk[n][e]);
          lv[key_of[n] * LD + elem_of[n] + e] = static_cast<float>(rv[n][e]);
        }
      }
  };
  f32x4 o[NB];
#pragma unroll
  for (int d = 0; d < NB; ++d) o[d] = f32x4{0, 0, 0, 0};
  float m = kNegInf, l = 0;
  __syncthreads();
  if (t0 < t1) load(t0);
  for (int t = t0; t < t1; ++t) {
    const int start = tile_start<KT>(kr, t), end = tile_end(kr, t);
    __syncthreads();
    store(t);
    if (t + 1 < t1) {
      load(t + 1);
      if (wave == 0) {
        place(entry, t + 2);
        entry = entry_of(t + 3);
      }
    }
    const uint32_t valid = tile_rows.valid[t & 3][0];
    const bool all = sees_all(s, kr, start, min(end, start + KT)), whole = all && valid == 0xffffu;
    __syncthreads();
    if (!all) {
      // Values that are not finite leave the tile, noted for the rows that see
      // them (as in the 16-bit kernels).
      bool strange = false;
      for (int x = threadIdx.x; x < KT * LD; x += NT) strange |= not_finite(lv[x]);
      if (strange) odd[0] = odd[1] = 1;
      __syncthreads();
      if (odd[0]) {
        for (int x = lane; x < 16 * D; x += kWave) {
          const int y = x / D, d = x - y * D, at = row0 + 16 * wave + y;
          if (at >= rows) break;
          const int mine = r.length - r.n + at / s.group;
          bool up = false, down = false;
          for (int k = 0; k < KT; ++k) {
            const float v = lv[k * LD + d];
            const bool seen = sees(s, kr, mine, start + k) & ((valid >> k) & 1);
            up |= seen & ((v != v) | (v == INFINITY));
            down |= seen & ((v != v) | (v == kNegInf));
          }
          if (up) atomicOr(&marks[0][(16 * wave + y) * MW + (d >> 5)], 1u << (d & 31));
          if (down) atomicOr(&marks[1][(16 * wave + y) * MW + (d >> 5)], 1u << (d & 31));
        }
        __syncthreads();
        for (int x = threadIdx.x; x < KT * LD; x += NT) lv[x] = not_finite(lv[x]) ? 0.0f : lv[x];
        if (threadIdx.x == 0) odd[0] = 0;
        __syncthreads();
      }
    }
    f32x4 st = {0, 0, 0, 0}, st2 = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < DP / 4; e += 2) {
      st = mfma4(lk[c * LD + 4 * e + g], q[e], st);
      st2 = mfma4(lk[c * LD + 4 * e + 4 + g], q[e + 1], st2);
    }
    float x[4], top = kNegInf;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int k = 4 * g + e;
      const float y = natural_score(s, st[e] + st2[e], slope, p, start + k) * kLog2e;
      const bool in = whole | (sees(s, kr, p, start + k) & ((valid >> k) & 1));
      x[e] = in ? y : kNegInf;
      top = fmaxf(top, x[e]);
    }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const float m1 = fmaxf(m, top);
    const float mu = m1 == kNegInf ? 0.0f : m1;
    const float alpha = exp2_fast(m - mu);
    m = m1;
    float pr[4];
    l *= alpha;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      pr[e] = exp2_fast(x[e] - mu);
      l += pr[e];
    }
#pragma unroll
    for (int d = 0; d < NB; ++d) {
      o[d] *= alpha;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[d] = mfma4(lv[(4 * g + e) * LD + 16 * d + c], pr[e], o[d]);
    }
  }
  __syncthreads();
  if (odd[1]) {
#pragma unroll
    for (int d = 0; d < NB; ++d) {
      const int at = (16 * wave + c) * MW + (d >> 1);
      const uint32_t up = marks[0][at] >> (16 * (d & 1) + 4 * g), down = marks[1][at] >> (16 * (d & 1) + 4 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[d][e] += (up >> e) & 1 ? INFINITY : 0.0f;
        o[d][e] += (down >> e) & 1 ? kNegInf : 0.0f;
      }
    }
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (!live) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const float lse2 = l == 0.0f ? kNegInf : m + log2_fast(l);
  const int64_t at = static_cast<int64_t>(r.q0 + i) * s.q_heads + qh;
  if (a.splits > 1) {
    const int64_t slot = static_cast<int64_t>(split) * s.batch.tokens * s.q_heads + at;
    float* po = a.part_out + slot * D;
#pragma unroll
    for (int d = 0; d < NB; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (16 * d + 4 * g + e < D) po[16 * d + 4 * g + e] = o[d][e] * inv;
    if (g == 0) a.part_lse[slot] = lse2;
    return;
  }
  char* op = a.out.data + static_cast<int64_t>(r.q0 + i) * a.out.token_b + qh * a.out.head_b;
#pragma unroll
  for (int d = 0; d < NB; ++d)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (16 * d + 4 * g + e < D)
        store_elem<IO>(op + (16 * d + 4 * g + e) * static_cast<int>(sizeof(IO)), from_f32<IO>(o[d][e] * inv));
  if (a.lse && g == 0) a.lse[at] = lse2 * kLn2;
}

// How many splits the tile of a (token, head) has; -1 for rows of no request.
template <int KT>
CB_INLINE int row_splits(const AttendArgs& a, int t, int qh, int rows_per_tile) {
  const ScoreArgs& s = a.s;
  const int b = request_of_token(s.batch, t);
  if (b >= s.batch.requests) return -1;
  const Request r = load_request(s.batch, b);
  if (!r.ok) return -1;
  const int row = (t - r.q0) * s.group + qh % s.group;
  const int row0 = row / rows_per_tile * rows_per_tile;
  const KeyRange kr = key_range<KT>(s, r, b, row0, min(r.n * s.group, row0 + rows_per_tile) - 1);
  const int per = split_tiles(a, kr.tiles);
  return per > 0 ? (kr.tiles + per - 1) / per : 0;
}

// Joins few splits: out = sum 2^(lse_z - lse) out_z, a wave a row. Lane z holds
// split z's statistics, then every lane E elements of the row. Taken where
// there are rows enough for all CUs: with 128 new tokens (2048 rows of 128) over
// 4096 it takes 6.6 us where a workgroup a row takes 7.9, with 64 times 16
// tokens 13.4 against 37.2, with 1000 rows of 64 5.0 against 5.8; with 37 tokens
// (592 rows) 5.9 against 5.1, with 4 9.0 against 5.0.
constexpr int kJoinFew = 16;    // splits up to which, and
constexpr int kJoinRows = 768;  // rows from which it is taken

template <typename IO, int KT, int E>
__global__ __launch_bounds__(256) void join_few_kernel(AttendArgs a, int rows_per_tile) {
  typedef float vec __attribute__((ext_vector_type(E)));
  const ScoreArgs& s = a.s;
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t step = static_cast<int64_t>(s.batch.tokens) * s.q_heads;
  if (at >= step) return;
  const int t = static_cast<int>(at / s.q_heads), qh = static_cast<int>(at % s.q_heads);
  const float got = a.part_lse[min(lane, a.splits - 1) * step + at];  // before what it waits for is known
  const int n = __builtin_amdgcn_readfirstlane(row_splits<KT>(a, t, qh, rows_per_tile));
  if (n < 0) return;
  const float lse = lane < n ? got : kNegInf;
  float top = lse;
#pragma unroll
  for (int d = 1; d < kJoinFew; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  top = __shfl(top, 0);
  const float mu = top == kNegInf ? 0.0f : top;
  const float w = exp2_fast(lse - mu);
  float total = w;
#pragma unroll
  for (int d = 1; d < kJoinFew; d <<= 1) total += __shfl_xor(total, d);
  total = __shfl(total, 0);
  const int D = s.head_dim, d0 = lane * E;
  float o[E] = {};
  if (d0 < D) {
    for (int z = 0; z < n; ++z) {
      // Read from lanes that may hold no element and are off here.
      const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), z));
      const float* from = a.part_out + (z * step + at) * D + d0;
      if (f == 0.0f) continue;
      if (D % E == 0) {
        const vec x = *reinterpret_cast<const vec*>(from);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] += f * x[e];
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (d0 + e < D) o[e] += f * from[e];
      }
    }
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  char* op = a.out.data + static_cast<int64_t>(t) * a.out.token_b + qh * a.out.head_b;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (d0 + e < D) store_elem<IO>(op + (d0 + e) * static_cast<int>(sizeof(IO)), from_f32<IO>(o[e] * inv));
  if (a.lse && lane == 0) a.lse[at] = total == 0.0f ? kNegInf : (top + log2_fast(total)) * kLn2;
}

// Joins many splits, a workgroup a row: threads of one group of LANES hold four
// elements each of a split's row, the groups take splits in turn and meet in
// LDS in group order.
constexpr int kJoinThreads = 256;

template <typename IO, int KT, int LANES>
__global__ __launch_bounds__(kJoinThreads) void join_splits_kernel(AttendArgs a, int rows_per_tile) {
  constexpr int GROUPS = kJoinThreads / LANES;
  __shared__ float red[2][kJoinThreads / kWave];
  __shared__ f32x4 sums[GROUPS][LANES];
  const ScoreArgs& s = a.s;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int64_t at = blockIdx.x;
  const int t = static_cast<int>(at / s.q_heads), qh = static_cast<int>(at % s.q_heads);
  const int n = row_splits<KT>(a, t, qh, rows_per_tile);
  if (n < 0) return;
  const int64_t step = static_cast<int64_t>(s.batch.tokens) * s.q_heads;
  const float* lse = a.part_lse + at;
  float top = kNegInf;
  for (int z = threadIdx.x; z < n; z += kJoinThreads) top = fmaxf(top, lse[z * step]);
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  if (lane == 0) red[0][wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoinThreads / kWave; ++w) top = fmaxf(top, red[0][w]);
  const float mu = top == kNegInf ? 0.0f : top;
  float total = 0;
  for (int z = threadIdx.x; z < n; z += kJoinThreads) total += exp2_fast(lse[z * step] - mu);
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) total += __shfl_xor(total, d);
  if (lane == 0) red[1][wave] = total;
  const int g = threadIdx.x / LANES, x = threadIdx.x % LANES;
  const int D = s.head_dim;
  f32x4 o = {0, 0, 0, 0};
  const bool vector = D % 4 == 0;
  for (int z = g; z < n; z += GROUPS) {
    const float w = exp2_fast(lse[z * step] - mu);
    if (w == 0.0f || 4 * x >= D) continue;
    const float* from = a.part_out + (z * step + at) * D + 4 * x;
    if (vector) {
      o += w * *reinterpret_cast<const f32x4*>(from);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (4 * x + e < D) o[e] += w * from[e];
    }
  }
  sums[g][x] = o;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < kJoinThreads / kWave; ++w) total += red[1][w];
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  char* op = a.out.data + static_cast<int64_t>(t) * a.out.token_b + qh * a.out.head_b;
  for (int d = threadIdx.x; d < D; d += kJoinThreads) {
    float sum = 0;
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) sum += sums[k][d / 4][d & 3];
    store_elem<IO>(op + d * static_cast<int>(sizeof(IO)), from_f32<IO>(sum * inv));
  }
  if (a.lse && threadIdx.x == 0) a.lse[at] = total == 0.0f ? kNegInf : (top + log2_fast(total)) * kLn2;
}

// ---------------------------------------------------------------------------
// Attention in 16-bit types, head_dim a multiple of 8 up to 256 (padded with
// zeros to DP = 64, 128 or 256).
//
// One wave computes 32 query rows against tiles of KT keys with
// v_mfma_f32_32x32x16 (result register e of lane l: row 8 (e / 4) + 4 (l / 32)
// + e % 4, column l % 32): S^T = K Q^T has a query row per lane pair, so a
// lane sees half of its row's keys of a tile. Packed in register order, eight
// of its weights are the second operand of a step of 16 keys, in the key order
// {4h .. 4h+3, 8+4h .. 8+4h+3} (h = l / 32); V^T is read in the same order by
// transposing LDS reads, so weights never leave their lane.
//
// K and V rows come through LDS by DMA (global_load_lds_dwordx4: the LDS side
// is 16 bytes a lane in lane order, the global side any address a lane, which
// gathers rows of pages for free). A row's 16-byte chunks sit at positions
// chunk ^ f(key): the readers' lanes then hit distinct banks (K: 16 rows of
// one chunk; V: 4 rows of 4 chunks).
// ---------------------------------------------------------------------------

typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

#define CB_LDS_SPACE __attribute__((address_space(3)))

// An LDS address as the byte offset that DMA takes.
template <typename T>
__device__ inline CB_LDS_SPACE T* lds_at(uint32_t offset) {
  return (CB_LDS_SPACE T*)static_cast<uintptr_t>(offset);
}

template <typename IO>
struct Half;
template <>
struct Half<io_bf16> {
  typedef io_bf16 x8 __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kExponent = 0x7f807f80u, kCarry = 0x00800080u, kInf = 0x7f80u;
  static constexpr float kRoom = 0, kLag = 1024;
  static __device__ inline f32x16 mul(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  static __device__ inline uint32_t pack(float a, float b) { return pack_bf16(a, b); }
};
template <>
struct Half<io_f16> {
  typedef io_f16 x8 __attribute__((ext_vector_type(8)));
  typedef io_f16 x2 __attribute__((ext_vector_type(2)));
  static constexpr uint32_t kExponent = 0x7c007c00u, kCarry = 0x04000400u, kInf = 0x7c00u;
  // Weights count from 2^8, not 1: the many small ones of a long request keep
  // eight more bits above the type's least step of 2^-24.
  static constexpr float kRoom = 8, kLag = 32768;
  static __device__ inline f32x16 mul(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  }
  static __device__ inline uint32_t pack(float a, float b) {
    const f32x2 f = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, x2));  // round to nearest even
  }
};

// What the DMA reads for keys without a row and elements past head_dim.
__device__ const uint4 g_zeros[1] = {};

constexpr int kMaxDp = 256;

template <int DP>
__device__ inline int swizzle_k(int key) {
  return DP == 64 ? (key >> 1) & 7 : key & 15;
}
template <int DP>
__device__ inline int swizzle_v(int key) {
  return DP == 64 ? ((key >> 1) & 1) << 2 : (key & 3) << 2;
}

__device__ inline void dma16(gcptr src, uint32_t lds) {
  const uint32_t la = __builtin_amdgcn_readfirstlane(lds);
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
               :: "v"(reinterpret_cast<uint64_t>(src)), "s"(la) : "memory", "m0");
}

// s_waitcnt operands (gfx9 layout): everything, or the LDS DMA alone.
constexpr int wait_vm(int n) { return (n & 15) | 0x70 | 0xf00 | ((n >> 4) << 14); }
constexpr int kWaitAll = 0x0070;     // vmcnt 0, expcnt 7, lgkmcnt 0
__device__ inline void wait_and_meet() {
  __builtin_amdgcn_s_waitcnt(kWaitAll);
  asm volatile("s_barrier" ::: "memory");
}

// One wave's part of a tile's DMA: N instructions for K and as many for V,
// number u covering bytes [(first + u) * 1024, + 1024) of a tile.
template <typename IO, int DP, int KT, int N, int SLOTS>
struct Stager {
  static constexpr int C = DP / 8;  // 16-byte chunks a row
  gcptr kbase, vbase;               // the head's rows in the layer
  uint32_t stride;

  __device__ inline void init(const ScoreArgs& s, int head) {
    const int64_t off = static_cast<int64_t>(head) * s.head_dim * 2;
    kbase = layer_base(s.cache, 0, s.layer) + off;
    vbase = layer_base(s.cache, 1, s.layer) + off;
    stride = static_cast<uint32_t>(s.batch.row_stride_b);
  }
  // VALUE: the tile's V rows, else its K rows, to LDS at `to`.
  template <bool VALUE>
  CB_INLINE void issue(const ScoreArgs& s, const TileRows<KT, SLOTS>& rows, int slot, int first, uint32_t to) const {
    const int lane = threadIdx.x & (kWave - 1), pos = lane % C;
    uint32_t whole = ~0u;
#pragma unroll
    for (int k = 0; k < KT / 32; ++k) whole &= rows.valid[slot][k];
    const bool plain = (__builtin_amdgcn_readfirstlane(whole) == ~0u) & (s.head_dim == DP);
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int k = (first + u) * (kWave / C) + lane / C;
      const int c = pos ^ (VALUE ? swizzle_v<DP>(k) : swizzle_k<DP>(k));
      const uint32_t row = static_cast<uint32_t>(rows.row[slot][k]);
      gcptr at = (VALUE ? vbase : kbase) + static_cast<uint64_t>(row) * stride + c * 16;
      if (!plain) {
        const bool ok = (rows.valid[slot][k >> 5] >> (k & 31)) & 1;
        at = (ok & (c * 8 < s.head_dim)) ? at : as_global(static_cast<const void*>(g_zeros));
      }
      dma16(at, to + (first + u) * 1024);
    }
  }
};

// Whether a 16-byte chunk holds an infinity or NaN.
template <typename IO>
__device__ inline bool has_not_finite(u32x4 x) {
  uint32_t any = 0;
#pragma unroll
  for (int u = 0; u < 4; ++u) any |= ((x[u] & Half<IO>::kExponent) + Half<IO>::kCarry) & 0x80008000u;
  return any != 0;
}

// Zeros in place of the values of a chunk that are not finite.
template <typename IO>
__device__ inline u32x4 finite_part(u32x4 x) {
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const uint32_t c = ((x[u] & Half<IO>::kExponent) + Half<IO>::kCarry) & 0x80008000u;
    x[u] &= ~((c & 0x8000u ? 0xffffu : 0u) | (c & 0x80000000u ? 0xffff0000u : 0u));
  }
  return x;
}

// The operands of one row of `dim` elements: chunks 2 k + h of 16 bytes, zeros
// past dim. Loads are at clamped places and selected after: as branches each
// would wait for the one before.
template <int KS>
CB_INLINE void load_operands(const char* row, int dim, int h, bool vector, u32x4 (&x)[KS]) {
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    const char* at = row + 2 * min(16 * k + 8 * h, dim - 8);
    if (vector) {
      x[k] = gload<u32x4>(as_global(static_cast<const void*>(at)));
    } else {
#pragma unroll
      for (int w = 0; w < 4; ++w)
        x[k][w] = load_elem<uint16_t>(at + 4 * w) | static_cast<uint32_t>(load_elem<uint16_t>(at + 4 * w + 2)) << 16;
    }
  }
#pragma unroll
  for (int k = 0; k < KS; ++k) x[k] = 16 * k + 8 * h < dim ? x[k] : u32x4{0, 0, 0, 0};
}

// 32 query rows of one wave: their operands, statistics and sums.
template <typename IO, int DP, int KT, bool MOD>
struct RowBlock {
  typedef Half<IO> H;
  static constexpr int KB = KT / 32, DB = DP / 32, KS = DP / 16;
  u32x4 q[KS];
  f32x16 o[DB];
  float m, l;
  float slope;
  int row, i, qh, p;  // this lane's query row
  bool live;

  __device__ inline void init(const ScoreArgs& s, const Request& r, int head, int row0, bool vector) {
    const int lane = threadIdx.x & (kWave - 1), h = lane >> 5;
    const int rows = r.n * s.group;
    row = row0 + (lane & 31);
    live = row < rows;
    const int at = min(row, rows - 1);
    i = at / s.group;
    qh = head * s.group + at - i * s.group;
    p = r.length - r.n + i;
    const char* qp = s.q.data + static_cast<int64_t>(r.q0 + i) * s.q.token_b + qh * s.q.head_b;
    load_operands<KS>(qp, s.head_dim, h, vector, q);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] = 0;
    m = kNegInf;
    l = 0;
    slope = 0;
    if constexpr (MOD) slope = s.slopes ? s.slopes[qh] : 0.0f;
  }

  // LDS addresses within a tile that depend on the lane alone.
  struct Lanes {
    uint32_t k[DP == 64 ? 4 : 8];  // K chunk 2 ks + h of row l % 32; ks + 8: 256 bytes on
    uint32_t v[DP == 64 ? 2 : 4];  // V rows 4h + (l % 16) / 4, block db; db + 4: 256 bytes on
  };
  static __device__ inline Lanes lanes() {
    Lanes a;
    const int lane = threadIdx.x & (kWave - 1), h = lane >> 5, c = lane & 31;
#pragma unroll
    for (int ks = 0; ks < (DP == 64 ? 4 : 8); ++ks) a.k[ks] = c * DP * 2 + ((2 * ks + h) ^ swizzle_k<DP>(c)) * 16;
    const int l16 = lane & 15, key = 4 * h + (l16 >> 2);
#pragma unroll
    for (int db = 0; db < (DP == 64 ? 2 : 4); ++db)
      a.v[db] = key * DP * 2 + ((db * 4 + ((lane >> 4) & 1) * 2 + ((l16 & 3) >> 1)) ^ swizzle_v<DP>(key)) * 16 + (l16 & 1) * 8;
    return a;
  }

  static __device__ inline u32x4 k_frag(const Lanes& a, int kb, int ks) {
    return *lds_at<const u32x4>(a.k[ks & 7] + kb * 32 * DP * 2 + (ks >> 3) * 256);
  }
  static __device__ inline u32x4 v_frag(const Lanes& a, int step, int db) {
    const uint32_t at = a.v[db & 3] + step * 16 * DP * 2 + (db >> 2) * 256;
    const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_at<i16x4>(at));
    const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_at<i16x4>(at + 8 * DP * 2));
    const uint2 x = __builtin_bit_cast(uint2, lo), y = __builtin_bit_cast(uint2, hi);
    return u32x4{x.x, x.y, y.x, y.y};
  }

  // Raw products of the rows with a tile of KT keys. Operands are read from
  // LDS a few steps ahead of their use; the scheduling barriers keep the
  // compiler from moving the reads back to it, where each would be waited for.
  CB_INLINE void products(const Lanes& a, f32x16 (&st)[KB]) {
    constexpr int STEPS = KB * KS, AHEAD = 4;
    u32x4 f[AHEAD];
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) f[n] = k_frag(a, n % KB, n / KB);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) st[kb][e] = 0;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < STEPS; ++n) {
      st[n % KB] = H::mul(f[n % AHEAD], q[n / KB], st[n % KB]);
      if (n + AHEAD < STEPS) f[n % AHEAD] = k_frag(a, (n + AHEAD) % KB, (n + AHEAD) / KB);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // Raw products of the tile that starts at cached token `start` made ready
  // for their weights: modified and masked. `whole`: every row sees every key.
  // `valid`: keys that are there, 32 a word.
  CB_INLINE void ready(const ScoreArgs& s, const KeyRange& kr, f32x16 (&st)[KB], int start, bool whole,
                       const uint32_t* valid) {
    const int h = (threadIdx.x & (kWave - 1)) >> 5;
    // Scores times scale2 are in the log2 domain (MOD: scale2 is 1 and they
    // are put there at once).
    if constexpr (MOD) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) modify_scores<true>(s, st[kb], kLog2e, slope, p, start + 32 * kb, h);
    }
    if (!whole) {
      asm volatile("");  // a branch: as selects, every tile would pay for the mask (250 instructions)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const uint32_t there = valid[kb] >> (4 * h);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int k = 8 * (e >> 2) + (e & 3), j = start + 32 * kb + 4 * h + k;
          const bool in = sees(s, kr, p, j) & ((there >> k) & 1);
          st[kb][e] = in ? st[kb][e] : kNegInf;
        }
      }
    }
  }

  // Weights by the maximum that stands, packed as the next product's operands,
  // and their sum (of the weights as they were). The rounding to 16 bits is
  // the price of 16-bit products with V: over random keys it adds as much as the
  // result's own rounding does (bf16 errors of 2.4e-3 of the result where fp32 weights
  // leave 1.7e-3, fp16 2.7e-4 and 2.1e-4); a second product for the part rounded
  // off would be half as many matrix steps again. Calls that ask for fp32 weights
  // take attend_any_kernel: a step of 64 requests of 2048 151 us for 42, a prompt
  // of 4096 (16 heads of 128) 1126 for 135.
  CB_INLINE float try_weights(const f32x16 (&st)[KB], float scale2, u32x4 (&w)[KB][2]) const {
    const float mu = m == kNegInf ? 0.0f : m;
    float sum = 0;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const float x = exp2_fast(__builtin_fmaf(st[kb][e], scale2, -mu)), y = exp2_fast(__builtin_fmaf(st[kb][e + 1], scale2, -mu));
        sum += x + y;
        w[kb][e >> 3][(e & 7) >> 1] = H::pack(x, y);
      }
    return sum;
  }
  // A row's maximum is looked for only if a lane's weights show that it has
  // grown by much (their sum tells) or is not known yet: up to kLag, weights
  // lose no digits in fp32 sums or 16 bits (m is the maximum less kRoom). Vector instructions that are not
  // exponentials cost the matrix unit their time here (16 ns a product alone or
  // beside 2 exponentials a wave, 26 ns with 6 multiply-adds more), so the
  // maxima of every tile would.
  CB_INLINE void weights(const f32x16 (&st)[KB], float scale2, u32x4 (&w)[KB][2]) {
    float sum = try_weights(st, scale2, w);
    if (__any(!(sum < H::kLag) | (m == kNegInf))) {
      float top = kNegInf;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, st[kb][e]);
      top = __builtin_fmaf(top, scale2, -H::kRoom);
      const float m1 = fmaxf(m, fmaxf(top, __shfl_xor(top, 32)));
      const float alpha = m1 == kNegInf ? 1.0f : exp2_fast(m - m1);
      m = m1;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < DB; ++d) o[d] *= alpha;
      sum = try_weights(st, scale2, w);
    }
    l += sum;
  }

  // The first operands of a tile's values, read before its weights are made.
  static constexpr int kValuesAhead = 4;
  struct Values {
    u32x4 f[kValuesAhead];
  };
  // Lane addresses within the tiles at lk and lv: the rest of an address then
  // fits the instruction.
  static CB_INLINE Lanes place(const Lanes& a, uint32_t lk, uint32_t lv) {
    Lanes at = a;
#pragma unroll
    for (int x = 0; x < (DP == 64 ? 4 : 8); ++x) {
      at.k[x] += lk;
      asm("" : "+v"(at.k[x]));
    }
#pragma unroll
    for (int x = 0; x < (DP == 64 ? 2 : 4); ++x) {
      at.v[x] += lv;
      asm("" : "+v"(at.v[x]));
    }
    return at;
  }

  static CB_INLINE Values first_values(const Lanes& a) {
    Values v;
#pragma unroll
    for (int n = 0; n < kValuesAhead; ++n) v.f[n] = v_frag(a, n / DB, n % DB);
    __builtin_amdgcn_sched_barrier(0);
    return v;
  }
  CB_INLINE void add_values(const Lanes& a, const u32x4 (&w)[KB][2], Values& v) {
    constexpr int STEPS = 2 * KB * DB;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < STEPS; ++n) {
      const int t = n / DB, d = n % DB;
      o[d] = H::mul(v.f[n % kValuesAhead], w[t >> 1][t & 1], o[d]);
      if (n + kValuesAhead < STEPS) v.f[n % kValuesAhead] = v_frag(a, (n + kValuesAhead) / DB, (n + kValuesAhead) % DB);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // Adds the infinities that were taken out of V tiles (see mark_not_finite).
  __device__ inline void add_marks(const uint32_t* up, const uint32_t* down) {
    const int lane = threadIdx.x & (kWave - 1), h = lane >> 5;
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      const uint32_t u = up[(lane & 31) * DB + d], w = down[(lane & 31) * DB + d];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int bit = 8 * (e >> 2) + 4 * h + (e & 3);
        o[d][e] += (u >> bit) & 1 ? INFINITY : 0.0f;
        o[d][e] += (w >> bit) & 1 ? kNegInf : 0.0f;
      }
    }
  }

  __device__ inline void finish(const AttendArgs& a, const Request& r, int split, bool vector) {
    const ScoreArgs& s = a.s;
    const int h = (threadIdx.x & (kWave - 1)) >> 5;
    l += __shfl_xor(l, 32);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const float lse2 = l == 0.0f ? kNegInf : m + log2_fast(l);
    if (!live) return;
    const int64_t at = static_cast<int64_t>(r.q0 + i) * s.q_heads + qh;
    if (a.splits > 1) {
      const int64_t slot = static_cast<int64_t>(split) * s.batch.tokens * s.q_heads + at;
      gptr po = as_global(static_cast<void*>(a.part_out + slot * s.head_dim));
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (32 * d + 8 * g < s.head_dim)
            gstore<f32x4>(po + (32 * d + 8 * g + 4 * h) * 4,
                          f32x4{o[d][4 * g] * inv, o[d][4 * g + 1] * inv, o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv});
      if (h == 0) a.part_lse[slot] = lse2;
      return;
    }
    char* op = a.out.data + static_cast<int64_t>(r.q0 + i) * a.out.token_b + qh * a.out.head_b;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        if (32 * d + 8 * g < s.head_dim) {
          char* to = op + (32 * d + 8 * g + 4 * h) * 2;
          const uint2 x = make_uint2(H::pack(o[d][4 * g] * inv, o[d][4 * g + 1] * inv), H::pack(o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv));
          if (vector) {
            gstore<uint2>(as_global(static_cast<void*>(to)), x);
          } else {
            store_elem<uint16_t>(to, static_cast<uint16_t>(x.x));
            store_elem<uint16_t>(to + 2, static_cast<uint16_t>(x.x >> 16));
            store_elem<uint16_t>(to + 4, static_cast<uint16_t>(x.y));
            store_elem<uint16_t>(to + 6, static_cast<uint16_t>(x.y >> 16));
          }
        }
    if (a.lse && h == 0) a.lse[at] = lse2 * kLn2;
  }
};

// A tile that some rows see and others do not: a weight of zero times an
// infinity would be NaN in rows that do not see the value. Such values are
// taken out of the tile and noted, a bit per (row, element), for the rows that
// see their key; the sums get them at the end (+inf, -inf, both for NaN).

// One wave notes, for its 32 rows (marks [32][DP / 32], lane l < 32 owns row
// l's words), every such value of the V tile at lv.
template <typename IO, int DP, int KT>
CB_INLINE void mark_not_finite(uint32_t lv, int np, int below, int above, int start, int end,
                                                          CB_LDS_SPACE uint32_t* up, CB_LDS_SPACE uint32_t* down) {
  constexpr int C = DP / 8;
  const int lane = threadIdx.x & (kWave - 1);
  for (int n = 0; n < KT * C / kWave; ++n) {
    const u32x4 x = *lds_at<const u32x4>(lv + (n * kWave + lane) * 16);
    uint64_t hits = __ballot(has_not_finite<IO>(x));
    while (hits) {
      const int at = __ffsll(static_cast<unsigned long long>(hits)) - 1;
      hits &= hits - 1;
      const int chunk = n * kWave + at, key = chunk / C, d0 = ((chunk % C) ^ swizzle_v<DP>(key)) * 8, j = start + key;
      const bool seen = (j < end) & ((j < np) | ((j <= below) & (j > above)));
      for (int e = 0; e < 8; ++e) {
        const uint32_t word = __shfl(e < 4 ? (e < 2 ? x[0] : x[1]) : (e < 6 ? x[2] : x[3]), at);
        const uint32_t v = (word >> (16 * (e & 1))) & 0xffffu, mag = v & 0x7fffu;
        const bool nan = mag > Half<IO>::kInf, inf = mag == Half<IO>::kInf;
        const uint32_t bit = 1u << ((d0 + e) & 31);
        const int w = (lane & 31) * (DP / 32) + ((d0 + e) >> 5);
        if (seen & (lane < 32) & (nan | (inf & (v < 0x8000u)))) up[w] |= bit;
        if (seen & (lane < 32) & (nan | (inf & (v >= 0x8000u)))) down[w] |= bit;
      }
    }
  }
}

// Many query rows: a workgroup's NW waves hold 32 rows each and share K and V
// tiles, double buffered: while a tile is used the next one arrives. 2048 new
// tokens over 32768 (16 heads of 128, 2 KV heads, bf16, 533 GFLOP) take 529 us
// once the clocks have settled (up to 696 in the first 40 passes after a pause;
// calls of 531 to 571 with the join on several cards), 1.0 PFLOP/s, where a library
// product of 8192^3 reaches 1.21. What bounds it:
// matrix steps and vector instructions that are not exponentials do not overlap
// (see RowBlock::weights), so a tile costs its products plus its multiply-adds,
// packs and sums. 32 rows a wave: 64 have twice the products a K or V operand
// read, but took twice the time (1080 us; one wave a SIMD is left, and nothing
// runs while it waits). 64 keys a tile where they fit two workgroups' LDS:
// 32 took 847 us where 64 took 640.
template <typename IO, int DP, int KT, int NW, bool MOD>
__global__ __launch_bounds__(NW * kWave, DP == 256 ? 1 : 2) void attend_tile_kernel(AttendArgs a, int vector) {
  constexpr int kTile = KT * DP * 2, N = kTile / 1024 / NW;
  static_assert(N >= 1 && kTile % (1024 * NW) == 0, "a tile is whole DMA instructions of every wave");
  __shared__ __align__(1024) char tiles[4 * kTile];  // K, V of one buffer, K, V of the other
  __shared__ TileRows<KT> tile_rows;
  __shared__ uint32_t marks[2][NW][32 * (DP / 32)];
  __shared__ uint32_t odd[2];  // this tile holds values that are not finite; some tile did
  const ScoreArgs& s = a.s;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int head = blockIdx.x % s.kv_heads, rest = blockIdx.x / s.kv_heads;
  const int split = rest / a.tile_slots;
  Request r;
  int b, tile;
  if (!find_tile(a, rest % a.tile_slots, 32 * NW, r, b, tile)) return;
  const int rows = r.n * s.group, row0 = tile * 32 * NW;
  const KeyRange kr = key_range<KT>(s, r, b, row0, min(rows, row0 + 32 * NW) - 1);
  const int per = split_tiles(a, kr.tiles), t0 = split * per, t1 = min(kr.tiles, t0 + per);
  if (a.splits > 1 && t0 >= t1) return;

  typedef RowBlock<IO, DP, KT, MOD> Block;
  Block blk;
  blk.init(s, r, head, row0 + 32 * wave, vector);
  const typename Block::Lanes lanes = Block::lanes();
  const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((CB_LDS_SPACE char*)tiles));
  const float scale2 = MOD ? 1.0f : s.scale * kLog2e;
  Stager<IO, DP, KT, N, 4> stage;
  stage.init(s, head);
  const int first = wave * N;
  if (threadIdx.x < 2) odd[threadIdx.x] = 0;
  for (int w = threadIdx.x; w < 2 * NW * DP; w += NW * kWave) (&marks[0][0][0])[w] = 0;
  auto entry_of = [&](int t) { return t < t1 ? fetch_entry<KT>(s.batch, r, tile_start<KT>(kr, t), tile_end(kr, t)) : -1; };
  auto place = [&](int64_t entry, int t) {
    if (t < t1) place_rows(s.batch, r, entry, tile_start<KT>(kr, t), tile_end(kr, t), tile_rows, t & 3);
  };
  int64_t entry = -1;
  if (wave == 0) {
    const int64_t e0 = entry_of(t0), e1 = entry_of(t0 + 1);
    entry = entry_of(t0 + 2);
    place(e0, t0);
    place(e1, t0 + 1);
  }
  __syncthreads();
  if (t0 < t1) {
    stage.template issue<false>(s, tile_rows, t0 & 3, first, lds);
    stage.template issue<true>(s, tile_rows, t0 & 3, first, lds + kTile);
  }
  uint32_t buf = 0;
  for (int t = t0; t < t1; ++t) {
    wait_and_meet();
    if (wave == 0) place(entry, t + 2);
    if (t + 1 < t1) {
      const uint32_t to = lds + (buf ^ (2 * kTile));
      stage.template issue<false>(s, tile_rows, (t + 1) & 3, first, to);
      stage.template issue<true>(s, tile_rows, (t + 1) & 3, first, to + kTile);
    }
    if (wave == 0) entry = entry_of(t + 3);
    const int start = tile_start<KT>(kr, t), end = tile_end(kr, t);
    uint32_t valid[KT / 32], every = ~0u;
#pragma unroll
    for (int k = 0; k < KT / 32; ++k) every &= valid[k] = tile_rows.valid[t & 3][k];
    const bool all = sees_all(s, kr, start, min(end, start + KT));
    const bool whole = all && __builtin_amdgcn_readfirstlane(every) == ~0u;
    if (!all) {
      const uint32_t lv = lds + buf + kTile + (threadIdx.x & (kWave - 1)) * 16;
      bool strange = false;
#pragma unroll
      for (int u = 0; u < N; ++u) strange |= has_not_finite<IO>(*lds_at<const u32x4>(lv + (first + u) * 1024));
      if (strange) odd[0] = odd[1] = 1;
      __syncthreads();
      if (odd[0]) {
        mark_not_finite<IO, DP, KT>(lds + buf + kTile, kr.np, s.causal ? blk.p : 0x7fffffff, s.window > 0 ? blk.p - s.window : -1,
                                    start, end, (CB_LDS_SPACE uint32_t*)marks[0][wave], (CB_LDS_SPACE uint32_t*)marks[1][wave]);
        __syncthreads();
#pragma unroll
        for (int u = 0; u < N; ++u) {
          CB_LDS_SPACE u32x4* at = lds_at<u32x4>(lv + (first + u) * 1024);
          *at = finite_part<IO>(*at);
        }
        if (threadIdx.x == 0) odd[0] = 0;
        __syncthreads();
      }
    }
    f32x16 st[KT / 32];
    u32x4 w[KT / 32][2];
    const typename Block::Lanes at = Block::place(lanes, lds + buf, lds + buf + kTile);
    blk.products(at, st);
    blk.ready(s, kr, st, start, whole, valid);
    typename Block::Values v = Block::first_values(at);
    blk.weights(st, scale2, w);
    blk.add_values(at, w, v);
    buf ^= 2 * kTile;
  }
  __syncthreads();
  if (odd[1]) blk.add_marks(marks[0][wave], marks[1][wave]);
  blk.finish(a, r, split, vector);
}

// Few query rows (a decoding step): one block of 32 rows, whose keys the NW
// waves of a workgroup and the splits divide. Bound by memory, so each wave
// streams tiles of 32 keys through LDS of its own without barriers: two tiles
// of K and V are in flight, the next K is asked for as soon as the products
// have read its place, the next V after its sums. The rows that the index
// names are resolved into LDS first, so that the loop's only vector memory
// operations are the DMA, whose count tells what has arrived. One request of
// 32768 tokens (64 heads of 128, 8 KV heads, bf16, 134 MB) takes 31.7 us, 4.2 TB/s; four
// times the bytes (64 requests of 8192, 16 heads and 2 KV heads) 107 us, 5.0
// TB/s, a large copy's rate. 64 ragged requests of 2550 on average (167 MB) take
// 46 us, 3.6 TB/s: ragged lengths leave CUs without work at the end.
constexpr int kStepTiles = 64;  // tiles a split holds at most

template <typename IO, int DP, int NW, bool MOD>
__global__ __launch_bounds__(NW * kWave, 1) void attend_step_kernel(AttendArgs a, int vector) {
  constexpr int KT = 32, kTile = KT * DP * 2, N = kTile / 1024, C = DP / 8, LD = DP + 4;
  static_assert(4 * kTile >= 32 * LD * 4, "a wave's sums fit its tiles");
  __shared__ __align__(1024) char tiles[NW * 4 * kTile];  // a wave's K, K, V, V
  __shared__ int key_rows[kStepTiles * KT];
  __shared__ uint32_t marks[2][NW][32 * (DP / 32)];
  __shared__ float stats[2][NW][32];
  const ScoreArgs& s = a.s;
  const QBatch& B = s.batch;
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int head = blockIdx.x % s.kv_heads, rest = blockIdx.x / s.kv_heads;
  const int split = rest / a.tile_slots;
  Request r;
  int b, tile;
  if (!find_tile<true>(a, rest % a.tile_slots, 32, r, b, tile)) return;
  const int rows = r.n * s.group, row0 = tile * 32;
  const KeyRange kr = key_range<KT>(s, r, b, row0, min(rows, row0 + 32) - 1);
  const int per = min(split_tiles(a, kr.tiles), kStepTiles), t0 = split * per, t1 = min(kr.tiles, t0 + per);
  if (a.splits > 1 && t0 >= t1) return;

  for (int k = threadIdx.x; k < (t1 - t0) * KT; k += NW * kWave) {
    const int t = t0 + k / KT, j = tile_start<KT>(kr, t) + k % KT;
    int64_t row = -1;
    if (j < tile_end(kr, t)) {
      row = cache_row(B, r, j);
      if (row < 0) flag(B.err, CB_ERROR_CACHE_ROW);
    }
    key_rows[k] = static_cast<int>(row);
  }
  for (int w = threadIdx.x; w < 2 * NW * DP; w += NW * kWave) (&marks[0][0][0])[w] = 0;
  typedef RowBlock<IO, DP, KT, MOD> Block;
  Block blk;
  blk.init(s, r, head, row0, vector);
  const typename Block::Lanes lanes = Block::lanes();
  const float scale2 = MOD ? 1.0f : s.scale * kLog2e;
  const int64_t off = static_cast<int64_t>(head) * s.head_dim * 2;
  gcptr kbase = layer_base(s.cache, 0, s.layer) + off, vbase = layer_base(s.cache, 1, s.layer) + off;
  gcptr zero = as_global(static_cast<const void*>(g_zeros));
  const uint32_t stride = static_cast<uint32_t>(B.row_stride_b);
  const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((CB_LDS_SPACE char*)tiles)) + wave * 4 * kTile;
  wait_and_meet();

  const int n = t1 - t0 > wave ? (t1 - t0 - wave + NW - 1) / NW : 0;  // this wave's tiles: t0 + wave, + NW, ...
  auto request = [&](int i, gcptr base, uint32_t to, bool value) __attribute__((always_inline)) {
    const int at = (wave + i * NW) * KT;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int k = u * (kWave / C) + lane / C;
      const int row = key_rows[at + k];
      const int c = (lane % C) ^ (value ? swizzle_v<DP>(k) : swizzle_k<DP>(k));
      gcptr from = ((row >= 0) & (c * 8 < s.head_dim)) ? base + static_cast<uint64_t>(static_cast<uint32_t>(row)) * stride + c * 16 : zero;
      dma16(from, to + u * 1024);
    }
  };
  bool some_mark = false;
  if (n > 0) {
    request(0, kbase, lds, false);
    request(0, vbase, lds + 2 * kTile, true);
  }
  if (n > 1) {
    request(1, kbase, lds + kTile, false);
    request(1, vbase, lds + 3 * kTile, true);
  }
  uint32_t buf = 0;
  for (int i = 0; i < n; ++i) {
    const int t = t0 + wave + i * NW, start = tile_start<KT>(kr, t), end = tile_end(kr, t);
    const uint32_t valid = static_cast<uint32_t>(__ballot(key_rows[(t - t0) * KT + (lane & 31)] >= 0));
    if (i + 1 < n) __builtin_amdgcn_s_waitcnt(wait_vm(3 * N));
    else __builtin_amdgcn_s_waitcnt(wait_vm(N));
    asm volatile("" ::: "memory");
    f32x16 st[1];
    u32x4 w[1][2];
    const uint32_t lv = lds + 2 * kTile + buf;
    const typename Block::Lanes at = Block::place(lanes, lds + buf, lv);
    blk.products(at, st);
    if (i + 2 < n) {
      __builtin_amdgcn_s_waitcnt(0xc07f);  // the products' LDS reads
      request(i + 2, kbase, lds + buf, false);
    }
    const bool all = sees_all(s, kr, start, min(end, start + KT));
    blk.ready(s, kr, st, start, all & (valid == ~0u), &valid);
    blk.weights(st, scale2, w);
    if (i + 2 < n) __builtin_amdgcn_s_waitcnt(wait_vm(3 * N));
    else if (i + 1 < n) __builtin_amdgcn_s_waitcnt(wait_vm(2 * N));
    else __builtin_amdgcn_s_waitcnt(wait_vm(0));
    asm volatile("" ::: "memory");
    if (!all) {
      bool strange = false;
#pragma unroll
      for (int u = 0; u < N; ++u) strange |= has_not_finite<IO>(*lds_at<const u32x4>(lv + u * 1024 + lane * 16));
      if (__any(strange)) {
        some_mark = true;
        mark_not_finite<IO, DP, KT>(lv, kr.np, s.causal ? blk.p : 0x7fffffff, s.window > 0 ? blk.p - s.window : -1, start, end,
                                    (CB_LDS_SPACE uint32_t*)marks[0][wave], (CB_LDS_SPACE uint32_t*)marks[1][wave]);
#pragma unroll
        for (int u = 0; u < N; ++u) {
          CB_LDS_SPACE u32x4* at = lds_at<u32x4>(lv + u * 1024 + lane * 16);
          *at = finite_part<IO>(*at);
        }
      }
    }
    typename Block::Values v = Block::first_values(at);
    blk.add_values(at, w, v);
    if (i + 2 < n) {
      __builtin_amdgcn_s_waitcnt(0xc07f);
      request(i + 2, vbase, lv, true);
    }
    buf ^= kTile;
  }
  if (some_mark) blk.add_marks(marks[0][wave], marks[1][wave]);

  // The waves' sums meet in LDS, each wave's in its own tiles.
  blk.l += __shfl_xor(blk.l, 32);
  const int c = lane & 31, h = lane >> 5;
  float* mine = reinterpret_cast<float*>(tiles + wave * 4 * kTile) + c * LD;
  if (blk.live) {
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(mine + 32 * d + 8 * g + 4 * h) =
            f32x4{blk.o[d][4 * g], blk.o[d][4 * g + 1], blk.o[d][4 * g + 2], blk.o[d][4 * g + 3]};
  }
  if (h == 0) {
    stats[0][wave][c] = blk.m;
    stats[1][wave][c] = blk.l;
  }
  __syncthreads();
  const int D = s.head_dim, live = min(32, rows - row0), pairs = D / 2;
  for (int x = threadIdx.x; x < live * pairs; x += NW * kWave) {
    const int y = x / pairs, d = 2 * (x - y * pairs);
    float m = kNegInf;
#pragma unroll
    for (int w = 0; w < NW; ++w) m = fmaxf(m, stats[0][w][y]);
    const float mu = m == kNegInf ? 0.0f : m;
    float l = 0, o0 = 0, o1 = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = exp2_fast(stats[0][w][y] - mu);
      const float* from = reinterpret_cast<const float*>(tiles + w * 4 * kTile) + y * LD + d;
      l += f * stats[1][w][y];
      // A wave that saw nothing of this row has nothing to add.
      o0 += f != 0.0f ? f * from[0] : 0.0f;
      o1 += f != 0.0f ? f * from[1] : 0.0f;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const float lse2 = l == 0.0f ? kNegInf : m + log2_fast(l);
    const int row = row0 + y, i = row / s.group, qh = head * s.group + row - i * s.group;
    const int64_t at = static_cast<int64_t>(r.q0 + i) * s.q_heads + qh;
    if (a.splits > 1) {
      const int64_t slot = static_cast<int64_t>(split) * B.tokens * s.q_heads + at;
      *reinterpret_cast<float2*>(a.part_out + slot * D + d) = make_float2(o0 * inv, o1 * inv);
      if (d == 0) a.part_lse[slot] = lse2;
    } else {
      char* op = a.out.data + static_cast<int64_t>(r.q0 + i) * a.out.token_b + qh * a.out.head_b + d * 2;
      const uint32_t packed = Half<IO>::pack(o0 * inv, o1 * inv);
      if (vector) {
        gstore<uint32_t>(as_global(static_cast<void*>(op)), packed);
      } else {
        store_elem<uint16_t>(op, static_cast<uint16_t>(packed));
        store_elem<uint16_t>(op + 2, static_cast<uint16_t>(packed >> 16));
      }
      if (a.lse && d == 0) a.lse[at] = lse2 * kLn2;
    }
  }
}

// ---------------------------------------------------------------------------
// Weights of cached tokens
// ---------------------------------------------------------------------------

struct WeightArgs {
  ScoreArgs s;
  const float* lse;
  float* weights;
  int64_t weights_stride;
  int32_t key_slots;        // workgroups launched per request
  int32_t waves_per_block;  // 16-bit kernel: waves that share a block of 32 keys (1, 2 or 4)
};

// The new tokens of a request that may see any of the cached tokens
// [start, start + keys): all below a prefix, else those between.
CB_INLINE void query_range(const ScoreArgs& s, const Request& r, int np, int start, int keys, int* i0, int* i1) {
  *i0 = 0;
  *i1 = r.n;
  if (start < np) return;
  const int first = r.length - r.n;
  if (s.causal) *i0 = min(r.n, max(0, start - first));
  if (s.window > 0) *i1 = max(*i0, static_cast<int>(min(static_cast<int64_t>(r.n), static_cast<int64_t>(start) + keys - 1 + s.window - first)));
}

// w_j = sum over rows of exp(score - lse): one workgroup owns a key, so its sum
// needs no atomics and has one order.
//
// General form: a workgroup owns 16 keys of a request, its waves take every
// fourth block of 16 query rows of each KV head; partial sums meet in LDS in
// wave order.
template <typename IO, int DP>
__global__ __launch_bounds__(kAnyWaves * kWave, 1) void key_weights_any_kernel(WeightArgs a) {
  __shared__ float sums[kAnyWaves][16];
  const ScoreArgs& s = a.s;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int c = lane & 15, g = lane >> 4;
  const int b = blockIdx.x / a.key_slots, start = (blockIdx.x % a.key_slots) * 16;
  const Request r = own_request(s.batch, b);
  if (!r.ok && start == 0 && threadIdx.x == 0) flag(s.batch.err, CB_ERROR_REQUEST);
  if (start >= r.length) return;
  const int np = s.prefix ? max(0, min(s.prefix[b], r.length)) : 0;
  KeyRange kr{};
  kr.np = np;
  int i0, i1;
  query_range(s, r, np, start, 16, &i0, &i1);
  const int D = s.head_dim;
  const int64_t mine = start + c < r.length ? cache_row(s.batch, r, start + c) : -1;
  if (start + c < r.length && mine < 0 && wave == 0 && g == 0) flag(s.batch.err, CB_ERROR_CACHE_ROW);
  const uint64_t rows_ok = __ballot(mine >= 0);
  float sum[4] = {0, 0, 0, 0};
  for (int head = 0; head < s.kv_heads; ++head) {
    const char* kp = (const char*)layer_base(s.cache, 0, s.layer) + static_cast<int64_t>(head) * D * sizeof(IO) + (mine >= 0 ? mine : 0) * s.cache.row_stride_b;
    float k[DP / 4];
    load_spread<IO>(kp, D, g, k);
#pragma unroll
    for (int e = 0; e < DP / 4; ++e) k[e] = mine >= 0 ? k[e] : 0.0f;
    for (int row0 = i0 * s.group + 16 * wave; row0 < i1 * s.group; row0 += kAnyRows) {
      const int row = min(row0 + c, i1 * s.group - 1);
      const int i = row / s.group, qh = head * s.group + row % s.group, p = r.length - r.n + i;
      const char* qp = s.q.data + static_cast<int64_t>(r.q0 + i) * s.q.token_b + qh * s.q.head_b;
      f32x4 st = {0, 0, 0, 0};
      float q[DP / 4];
      load_spread<IO>(qp, D, g, q);
#pragma unroll
      for (int e = 0; e < DP / 4; ++e) st = mfma4(k[e], q[e], st);
      const float lse = a.lse[static_cast<int64_t>(r.q0 + i) * s.q_heads + qh];
      const float slope = s.slopes ? s.slopes[qh] : 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = start + 4 * g + e;
        const bool in = (row0 + c < i1 * s.group) & (lse != kNegInf) & sees(s, kr, p, j);
        // The difference first: what is near the row's maximum keeps its bits.
        const float w = exp2_fast((natural_score(s, st[e], slope, p, j) - lse) * kLog2e);
        sum[e] += in ? w : 0.0f;
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) sum[e] += __shfl_xor(sum[e], d);
    if (c == 0) sums[wave][4 * g + e] = sum[e];
  }
  __syncthreads();
  if (threadIdx.x < 16 && start + static_cast<int>(threadIdx.x) < r.length && ((rows_ok >> threadIdx.x) & 1)) {
    float add = 0;
#pragma unroll
    for (int w = 0; w < kAnyWaves; ++w) add += sums[w][threadIdx.x];
    a.weights[b * a.weights_stride + start + threadIdx.x] += add;
  }
}

// 16-bit form: a wave holds 32 keys of one KV head as MFMA operands in
// registers and walks blocks of 32 query rows, whose operands come straight
// from memory (the few rows of a batch stay in cache); S^T keeps a row a lane
// pair, so a key's sum over rows is a sum over lanes, made once at the end.
// The waves that share a block of keys (4 if there are 4 or more blocks of
// rows to walk, else fewer, so that none idles) meet in LDS in wave order.
// 32 tokens over 32768 (16 heads of 128, 2 KV heads, bf16, 17 MB, 4.3 GFLOP)
// take 28.3 us, 64 ragged steps over 2550 on average (85 MB) 31.0 us. Bound by
// vector instructions and the address unit: a block of 32 rows and 32 keys has 8
// products and some 260 other instructions, and four lanes of an operand's load
// touch as many rows. Keys and rows through LDS of the wave's own took 26.0 and
// 42.6 us a call for 28.5 and 32.5: fewer waves then have loads in flight.
constexpr int kWeightWaves = 4;

template <typename IO, int DP, bool MOD>
__global__ __launch_bounds__(kWeightWaves * kWave, DP < 256 ? 4 : MOD ? 2 : 3) void key_weights_kernel(WeightArgs a, int vector) {
  typedef Half<IO> H;
  constexpr int KS = DP / 16;
  __shared__ float sums[kWeightWaves][32];
  const ScoreArgs& s = a.s;
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int h = lane >> 5, c = lane & 31;
  const int b = blockIdx.x / a.key_slots;
  const int share = a.waves_per_block, sub = wave % share;
  const int wide = 32 * (kWeightWaves / share);  // keys of the workgroup
  const int first_key = (blockIdx.x % a.key_slots) * wide, start = first_key + 32 * (wave / share);
  const Request r = load_request(s.batch, b);
  if (first_key >= r.length && first_key > 0) return;
  // Asked for by the waves that store, and looked at where they do: waited for
  // here by all it took the step 34.0 us a call, not 31.7.
  // At head 256 there is no register left for it (a step of 64 requests of 2048 161 us for 164).
  int top = sub == 0 ? starts_to<true>(s.batch, b) : 0;
  if constexpr (DP == 256) top = __any(top > r.q0) ? 0x7fffffff : -1;
  KeyRange kr{};
  kr.np = s.prefix ? max(0, min(s.prefix[b], r.length)) : 0;
  int i0 = 0, i1 = 0;
  if (start < r.length) query_range(s, r, kr.np, start, 32, &i0, &i1);
  const int j = start + c;
  const int64_t mine = j < r.length ? cache_row(s.batch, r, j) : -1;
  if ((j < r.length) & (mine < 0) & (sub == 0) & (h == 0)) flag(s.batch.err, CB_ERROR_CACHE_ROW);
  const uint32_t there = static_cast<uint32_t>(__ballot(mine >= 0));
  const int D = s.head_dim;
  const int low = i0 * s.group, high = i1 * s.group, blocks = (high - low + 31) / 32;
  float sum[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) sum[e] = 0;
  int held = -1;
  u32x4 k[KS];
  for (int item = sub; item < s.kv_heads * blocks; item += share) {
    const int head = item / blocks, row0 = low + (item - head * blocks) * 32;
    if (head != held) {
      held = head;
      gcptr kp = layer_base(s.cache, 0, s.layer) + static_cast<int64_t>(head) * D * 2 + mine * s.batch.row_stride_b;
#pragma unroll
      for (int x = 0; x < KS; ++x) {
        const int d = 16 * x + 8 * h;
        k[x] = u32x4{0, 0, 0, 0};
        if ((mine >= 0) & (d < D)) k[x] = gload<u32x4>(kp + 2 * d);
      }
    }
    const int row = row0 + c, at = min(row, high - 1), i = at / s.group, qh = head * s.group + at - i * s.group;
    const int p = r.length - r.n + i;
    const char* qp = s.q.data + static_cast<int64_t>(r.q0 + i) * s.q.token_b + qh * s.q.head_b;
    float lse = a.lse[static_cast<int64_t>(r.q0 + i) * s.q_heads + qh];
    // Nothing is added by lanes past the last row and rows that see nothing.
    lse = ((row >= high) | (lse == kNegInf)) ? INFINITY : lse;
    float slope = 0;
    if constexpr (MOD) slope = s.slopes ? s.slopes[qh] : 0.0f;
    f32x16 st;
#pragma unroll
    for (int e = 0; e < 16; ++e) st[e] = 0;
#pragma unroll
    for (int x = 0; x < KS; ++x) {
      const int d = 16 * x + 8 * h;
      u32x4 q = {0, 0, 0, 0};
      if (d < D) {
        if (vector) {
          q = gload<u32x4>(as_global(static_cast<const void*>(qp + 2 * d)));
        } else {
#pragma unroll
          for (int w = 0; w < 4; ++w)
            q[w] = load_elem<uint16_t>(qp + 2 * d + 4 * w) | static_cast<uint32_t>(load_elem<uint16_t>(qp + 2 * d + 4 * w + 2)) << 16;
        }
      }
      st = H::mul(k[x], q, st);
    }
    kr.p0 = r.length - r.n + row0 / s.group;
    kr.p1 = r.length - r.n + min(row0 + 31, high - 1) / s.group;
    const bool whole = sees_all(s, kr, start, start + 32);
    if constexpr (MOD) modify_scores<false>(s, st, 1.0f, slope, p, start, h);
    // The difference first: what is near the row's maximum keeps its bits.
    auto weight = [&](int e) { return exp2_fast((MOD ? st[e] - lse : __builtin_fmaf(st[e], s.scale, -lse)) * kLog2e); };
    if (whole) {
#pragma unroll
      for (int e = 0; e < 16; ++e) sum[e] += weight(e);
    } else {
      asm volatile("");  // a branch, as in RowBlock::ready
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float w = weight(e);
        sum[e] += sees(s, kr, p, start + 8 * (e >> 2) + 4 * h + (e & 3)) ? w : 0.0f;
      }
    }
  }
  // Sums over the 32 lanes of a half: each exchange halves what a lane holds.
#pragma unroll
  for (int n = 8, d = 16; n >= 1; n >>= 1, d >>= 1) {
    const bool up = (lane & d) != 0;
#pragma unroll
    for (int e = 0; e < n; ++e) {
      const float keep = up ? sum[e + n] : sum[e], give = up ? sum[e] : sum[e + n];
      sum[e] = keep + __shfl_xor(give, d);
    }
  }
  sum[0] += __shfl_xor(sum[0], 1);
  // Lane bits 4, 3, 2, 1 chose register bits 3, 2, 1, 0.
  const int e = (lane >> 1) & 15;
  if ((lane & 1) == 0) sums[wave][8 * (e >> 2) + 4 * h + (e & 3)] = sum[0];
  __syncthreads();
  const bool ok = r.ok && !__any(top > r.q0);
  if (!ok && first_key == 0 && threadIdx.x == 0) flag(s.batch.err, CB_ERROR_REQUEST);
  if (ok && sub == 0 && h == 0 && j < r.length && ((there >> c) & 1)) {
    float add = 0;
    for (int w = 0; w < share; ++w) add += sums[wave + w][c];
    a.weights[b * a.weights_stride + j] += add;
  }
}

// ---------------------------------------------------------------------------
// Eviction
// ---------------------------------------------------------------------------

struct EvictArgs {
  QBatch batch, target;
  const float* weights;
  int64_t weights_stride;
  int32_t budget, first, last;
  int32_t target_span;  // index entries of the target that are a request's own
  int32_t* kept;
  int32_t* kept_lengths;
  float* kept_weights;
};

// The request's cached tokens, or -1 if it is outside the batch's bounds.
CB_INLINE int evict_length(const EvictArgs& a, int b) {
  Request r;
  place_request(a.batch, b, r);
  const int length = a.batch.lengths[b];
  return (r.ok & (length >= 0) & (length <= a.batch.max_length)) ? length : -1;
}

constexpr int kSelectWaves = 16;
constexpr int kSelectThreads = kSelectWaves * kWave;

// Orders fp32 as unsigned integers; both zeros are one value, every NaN the largest.
__device__ inline uint32_t rank_of(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w == 0.0f ? 0.0f : w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Bins of a digit, eight copies each: weights often share a digit (many
// zeros, one exponent), and lanes that add to one bin take turns, so lane l
// adds to copy l % 8 (in banks of its own) and a wave of one digit takes 8
// turns, not 64.
constexpr int kBins = 2048, kBinCopies = 8, kCopyStride = kBins + 8;

// One workgroup per request. The smallest rank that is still kept is found
// digit by digit from the top (11, 11 and 10 bits): a histogram of the ranks
// that share the digits so far, then the bin in which the count from the top
// reaches what is needed. Counts are integers, so the order of the adds does
// not matter. R ranks a lane stay in registers (R * 1024 tokens between the
// first and the last), R = 0 reads the weights again on every pass. 4096 of
// 16384 tokens take 23 us, 700 of some 2000 in 16 requests 15 us: three rounds
// of clearing, adding and scanning bins with a barrier between each, on one CU a
// request. Adds of equal digits gathered by ballots first took 37 us.
template <int R>
__global__ __launch_bounds__(kSelectThreads) void select_tokens_kernel(EvictArgs a) {
  __shared__ __align__(16) int bins[kCopyStride * kBinCopies];
  __shared__ int totals[2][kSelectWaves];
  __shared__ int found[2];
  const int b = blockIdx.x;
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int length = evict_length(a, b);
  if (length < 0 && threadIdx.x == 0) flag(a.batch.err, CB_ERROR_REQUEST);  // nothing of it is kept
  const int64_t slot0 = static_cast<int64_t>(b) * a.budget;
  const float* w = a.weights + b * a.weights_stride;
  int32_t* kept = a.kept + slot0;
  float* kept_weights = a.kept_weights + slot0;
  const int n = max(0, min(length, a.budget));
  if (threadIdx.x == 0) a.kept_lengths[b] = n;
  for (int j = n + threadIdx.x; j < a.budget; j += kSelectThreads) {
    kept[j] = -1;
    kept_weights[j] = 0.0f;
  }
  const bool choose = length > a.budget;
  const int head = choose ? a.first : n, tail = choose ? a.last : 0;
  for (int j = threadIdx.x; j < head; j += kSelectThreads) {
    kept[j] = j;
    kept_weights[j] = w[j];
  }
  for (int j = threadIdx.x; j < tail; j += kSelectThreads) {
    kept[n - tail + j] = length - tail + j;
    kept_weights[n - tail + j] = w[length - tail + j];
  }
  const int need = choose ? n - head - tail : 0;
  if (need > 0) {
    // Wave v's share of the middle: groups of 64 tokens, in order.
    const int mid = length - head - tail;
    const int groups = (mid + kWave - 1) / kWave;
    const int per = (groups + kSelectWaves - 1) / kSelectWaves;
    const int g0 = wave * per, g1 = min(groups, g0 + per);
    const float* wm = w + head;
    // Every rank is above 0, which stands for no token.
    auto read = [&](int g) { return g < g1 && g * kWave + lane < mid ? rank_of(wm[g * kWave + lane]) : 0u; };
    uint32_t k[R > 0 ? R : 1];
    if constexpr (R > 0) {
#pragma unroll
      for (int i = 0; i < R; ++i) k[i] = read(g0 + i);
    }
    auto each = [&](auto&& use) __attribute__((always_inline)) {
      if constexpr (R > 0) {
#pragma unroll
        for (int i = 0; i < R; ++i)
          if (g0 + i < g1) use(g0 + i, k[i]);
      } else {
        for (int g = g0; g < g1; ++g) use(g, read(g));
      }
    };
    uint32_t base = 0, known = 0;
    int left = need;
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, size = pass == 2 ? 1024 : kBins;
      for (int x = threadIdx.x; x < kCopyStride * kBinCopies / 4; x += kSelectThreads) reinterpret_cast<int4*>(bins)[x] = make_int4(0, 0, 0, 0);
      __syncthreads();
      each([&](int, uint32_t r) {
        if ((r != 0) & ((r & known) == base)) atomicAdd(bins + (lane & 7) * kCopyStride + ((r >> shift) & (size - 1)), 1);
      });
      __syncthreads();
      // Thread x holds the x-th pair of bins from the top.
      const int hi = size - 1 - 2 * static_cast<int>(threadIdx.x);
      int c1 = 0, c0 = 0;
      if (hi > 0) {
#pragma unroll
        for (int x = 0; x < kBinCopies; ++x) {
          c1 += bins[x * kCopyStride + hi];
          c0 += bins[x * kCopyStride + hi - 1];
        }
      }
      int sum = c1 + c0;
#pragma unroll
      for (int d = 1; d < kWave; d <<= 1) {
        const int up = __shfl_up(sum, d);
        sum += lane >= d ? up : 0;
      }
      if (lane == kWave - 1) totals[0][wave] = sum;
      __syncthreads();
      int before = sum - c1 - c0;
#pragma unroll
      for (int v = 0; v < kSelectWaves; ++v) before += v < wave ? totals[0][v] : 0;
      if ((before < left) & (before + c1 + c0 >= left)) {
        const bool upper = before + c1 >= left;
        found[0] = upper ? hi : hi - 1;
        found[1] = upper ? before : before + c1;
      }
      __syncthreads();
      base |= static_cast<uint32_t>(found[0]) << shift;
      known |= static_cast<uint32_t>(size - 1) << shift;
      left -= found[1];
    }
    // Ranks above `base` are kept, and of those equal to it the first `left`.
    int above = 0, equal = 0;
    each([&](int, uint32_t r) {
      above += __popcll(__ballot(r > base));
      equal += __popcll(__ballot(r == base));
    });
    if (lane == 0) {
      totals[0][wave] = above;
      totals[1][wave] = equal;
    }
    __syncthreads();
    int above_before = 0, equal_before = 0;
#pragma unroll
    for (int v = 0; v < kSelectWaves; ++v) {
      above_before += v < wave ? totals[0][v] : 0;
      equal_before += v < wave ? totals[1][v] : 0;
    }
    const uint64_t below = (uint64_t{1} << lane) - 1;
    each([&](int g, uint32_t r) {
      const uint64_t ma = __ballot(r > base), me = __ballot(r == base);
      const int ea = equal_before + __popcll(me & below);
      const int at = head + above_before + __popcll(ma & below) + min(ea, left);
      if ((r > base) | ((r == base) & (ea < left))) {
        const int j = g * kWave + lane;
        kept[at] = head + j;
        kept_weights[at] = wm[j];
      }
      above_before += __popcll(ma);
      equal_before += __popcll(me);
    });
  }
}

struct MoveArgs {
  EvictArgs e;
  DevRows src, dst;
  int32_t chunks_per_row;
  int32_t tokens_per_block;
  int32_t blocks_per_request;
};

// Every layer's K and V rows of the kept tokens. A workgroup moves a run of
// one request's tokens in one layer; each thread resolves the rows of four
// chunks, then has the four loads in flight, then stores. Bound by memory: 4096
// tokens of 64 layers of 2 heads of 128 in bf16 (537 MB read and written) take
// 113 us, 4.8 TB/s; 16 requests' 700 of 62 layers 284 us, 5.0 TB/s, a plain
// copy's rate.
template <typename V>
__global__ __launch_bounds__(256) void move_rows_kernel(MoveArgs a) {
  constexpr int U = 4;
  const EvictArgs& e = a.e;
  const int layer = blockIdx.y >> 1, kind = blockIdx.y & 1;
  const int b = blockIdx.x / a.blocks_per_request, at0 = (blockIdx.x - b * a.blocks_per_request) * a.tokens_per_block;
  const int n = min(evict_length(e, b), e.budget);
  if (at0 >= n) return;
  Request src, dst;
  place_request(e.batch, b, src);
  place_request(e.target, b, dst);
  const int32_t* kept = e.kept + static_cast<int64_t>(b) * e.budget;
  gcptr sbase = layer_base(a.src, kind, layer);
  gptr dbase = const_cast<gptr>(layer_base(a.dst, kind, layer));
  const int stop = min(n, at0 + a.tokens_per_block);
  const int total = max(0, min(stop, e.target_span) - at0) * a.chunks_per_row;  // past the span: the next request's
  for (int base = threadIdx.x; base < total; base += blockDim.x * U) {
    int64_t from[U], to[U];
    int at[U], chunk[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int idx = min(base + u * static_cast<int>(blockDim.x), total - 1);
      at[u] = at0 + idx / a.chunks_per_row;
      chunk[u] = idx % a.chunks_per_row;
      from[u] = kept[at[u]];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      from[u] = cache_row(e.batch, src, static_cast<int>(from[u]));
      to[u] = dst.ok ? cache_row(e.target, dst, at[u]) : -1;
    }
    bool ok[U];
    V v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = base + u * static_cast<int>(blockDim.x) < total;
      if (in & (chunk[u] == 0) & (blockIdx.y == 0) & ((from[u] < 0) | (to[u] < 0))) {
        flag(e.batch.err, (from[u] < 0 ? CB_ERROR_CACHE_ROW : 0) | (to[u] < 0 ? CB_ERROR_TARGET_ROW : 0));
        // Its target row, if there is one, keeps what it held: the request's length says that it may not be used.
        if (from[u] < 0) e.kept_lengths[b] = 0;
      }
      ok[u] = in & (from[u] >= 0) & (to[u] >= 0);
      if (ok[u]) v[u] = gload<V>(sbase + from[u] * a.src.row_stride_b + chunk[u] * static_cast<int>(sizeof(V)));
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (ok[u]) gstore<V>(dbase + to[u] * a.dst.row_stride_b + chunk[u] * static_cast<int>(sizeof(V)), v[u]);
  }
  if (stop > e.target_span && blockIdx.y == 0 && threadIdx.x == 0) flag(e.batch.err, CB_ERROR_TARGET_ROW);
}

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

int check_batch(const cb_query_batch* batch, int32_t dtype, int32_t head_dim, int32_t* err, bool queries, QBatch* B,
                DevRows* rows) {
  if (!batch) return fail(CB_EINVAL, "null batch");
  const int eb = elem_bytes(dtype);
  if (!eb) return fail(CB_EINVAL, "bad dtype");
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

int check_scores(const cb_query_batch* batch, int32_t layer, int32_t dtype, int32_t head_dim, const cb_scores* sc,
                 int32_t q_heads, int32_t* err, ScoreArgs* s) {
  int rc;
  if ((rc = check_batch(batch, dtype, head_dim, err, true, &s->batch, &s->cache))) return rc;
  if (!sc) return fail(CB_EINVAL, "null scores");
  if (layer < 0 || layer >= batch->cache.num_layers) return fail(CB_EINVAL, "layer %d outside the cache", layer);
  const int kv = batch->cache.heads;
  if (q_heads < 1 || q_heads % kv) return fail(CB_EINVAL, "query heads must be a positive multiple of the KV heads");
  if (!std::isfinite(sc->scale)) return fail(CB_EINVAL, "scale must be finite");
  if (!std::isfinite(sc->cap) || sc->cap < 0) return fail(CB_EINVAL, "cap must be finite and not negative");
  if (sc->window < 0) return fail(CB_EINVAL, "negative window");
  if (static_cast<int64_t>(batch->max_query) * (q_heads / kv) > 0x3fffffff) return fail(CB_EINVAL, "too many query rows");
  s->layer = layer;
  s->head_dim = head_dim;
  s->q_heads = q_heads;
  s->kv_heads = kv;
  s->group = q_heads / kv;
  s->scale = sc->scale;
  s->cap = sc->cap;
  // Bounded so that a product of zero stays zero however small the cap is.
  s->inner = sc->cap > 0 ? std::max(-1e38f, std::min(1e38f, sc->scale / sc->cap)) : 0.0f;
  s->gentle = kSmallAngle / std::fabs(s->inner);
  s->window = sc->window;
  s->causal = sc->causal != 0;
  s->slopes = sc->slopes;
  s->prefix = sc->prefix_lengths;
  // The plain form takes a row's maximum before the scale: that needs one above zero.
  s->mod = s->cap > 0 || s->slopes || !(s->scale > 0);
  return CB_OK;
}

// HIP counts a launch's threads in 32 bits.
bool launch_fits(int64_t workgroups, int threads) { return workgroups <= 0xffffffffll / threads; }

int ceil_div(int64_t a, int64_t b) { return static_cast<int>((a + b - 1) / b); }

// Workgroups of four waves that a launch is split into at least: two a CU. 512 new
// tokens over 32768 take 262, 173 and 185 us with 256, 512 and 1024, 64 requests of
// 8 new tokens over 2048 47, 38.5 and 39 us.
constexpr int kTargetGroups = 512;

// How the launch is cut: query tiles, and key splits where the tiles alone
// would leave CUs idle.
struct AttendShape {
  bool half;  // the 16-bit kernels
  bool step;  // of these, the one for few rows
  int waves;
  int rows_per_tile, keys_per_tile;
  int64_t tile_slots;
  int request_slots, splits, least_tiles;
};

// Whether the 16-bit kernels take the call: whole 16-byte chunks of rows.
bool takes_half(const ScoreArgs& s, int32_t dtype) {
  return dtype != CB_DTYPE_F32 && s.head_dim % 8 == 0 && s.cache.row_stride_b <= 0xffffffffll && s.head_dim <= kMaxDp && rows_aligned16(s.cache, s.head_dim * 2);
}

// Waves of attend_tile_kernel: eight share a tile's staging among twice the
// rows, if there are that many and a head's registers leave two waves a SIMD.
// That pays once a launch has work for all CUs (16 query heads, 2 KV heads,
// kernel and join, eight waves against four): 256 new tokens over 4096 cached
// 41.1 / 37.1 us, 64 over 32768 46.1 / 49.2, 1024 over 4096 63 / 70, 256 over
// 32768 106 / 120; 1000 of 1000 with 8 heads 39.4 / 34.1.
constexpr int kWideRows = 512;               // query rows per KV head, and
constexpr int64_t kWideScores = 24ll << 20;  // scores of the launch, from which eight are taken
// Query rows per KV head up to which attend_step_kernel is taken: one block of
// rows, so that K and V are read once. This kernel against the tile kernel, each
// with its join, 8 query heads a KV head: 64 ragged requests of 2550 on average 52 /
// 100 us; one request of 32768 38 / 38. Where all lengths are alike the tile
// kernel is ahead: 64 of 2048 42 / 35, with four new tokens 57 / 40.
constexpr int kStepRows = 32;
// Its workgroups: one request has all its splits at work, of several requests many
// are shorter than the bound that splits are cut by. With the join, 512, 1024
// and 2048: 64 ragged requests 73, 52, 67 us; 64 of 2048 33, 42, 42; one request of
// 32768 38 with 512 and 47 with 1024.
constexpr int kStepGroups = 512, kStepGroupsRagged = 1024;
constexpr int kStepWaves = 2;

AttendShape attend_shape(const ScoreArgs& s, int32_t dtype, bool fp32_weights) {
  AttendShape h{};
  h.half = !fp32_weights && takes_half(s, dtype);
  const QBatch& B = s.batch;
  h.step = h.half && static_cast<int64_t>(B.max_query) * s.group <= kStepRows;
  const int64_t seen = s.window > 0 && s.causal && !s.prefix ? std::min<int64_t>(B.max_length, s.window) : B.max_length;
  h.waves = h.half && s.head_dim <= 128 && static_cast<int64_t>(B.max_query) * s.group >= kWideRows &&
                    static_cast<int64_t>(B.tokens) * s.q_heads * seen >= kWideScores
                ? 8 : 4;
  h.rows_per_tile = h.step ? 32 : h.half ? 32 * h.waves : kAnyRows;
  h.keys_per_tile = !h.half ? kAnyKeys : !h.step && s.head_dim <= (s.mod ? 64 : 128) ? 64 : 32;
  const int per_request = std::max(1, ceil_div(static_cast<int64_t>(B.max_query) * s.group, h.rows_per_tile));
  const int64_t by_request = static_cast<int64_t>(per_request) * B.requests;
  const int64_t packed = ceil_div(static_cast<int64_t>(B.tokens) * s.group, h.rows_per_tile) + static_cast<int64_t>(B.requests);
  h.request_slots = by_request <= packed ? per_request : 0;
  h.tile_slots = std::min(by_request, packed);
  int64_t keys = B.max_length;
  if (s.window > 0 && s.causal && !s.prefix) keys = std::min<int64_t>(keys, static_cast<int64_t>(s.window) + std::min<int64_t>(B.max_query, h.rows_per_tile / s.group + 2));
  const int key_tiles = std::max(1, ceil_div(keys, h.keys_per_tile) + (s.prefix ? 1 : 0));
  const int64_t groups = h.tile_slots * s.kv_heads;
  const int64_t target = !h.step ? kTargetGroups * 4 / h.waves : B.requests > 1 ? kStepGroupsRagged : kStepGroups;
  h.least_tiles = h.half ? 8 : 2;
  h.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(target / std::max<int64_t>(1, groups), key_tiles / h.least_tiles)));
  if (h.step) {
    // Parts of one size for all requests, cut by the bound: their workgroups end
    // together (64 ragged requests 47 us, with parts by each one's own keys 68).
    h.splits = std::max(h.splits, ceil_div(key_tiles, kStepTiles));
    h.least_tiles = ceil_div(key_tiles, h.splits);
    h.splits = ceil_div(key_tiles, h.least_tiles);
  }
  return h;
}

int64_t round256(int64_t x) { return (x + 255) / 256 * 256; }

int64_t attend_workspace(const ScoreArgs& s, const AttendShape& h) {
  if (h.splits <= 1) return 0;
  const int64_t rows = static_cast<int64_t>(h.splits) * s.batch.tokens * s.q_heads;
  return round256(rows * s.head_dim * 4) + round256(rows * 4);
}

bool joins_by_wave(int splits, int64_t rows) { return splits <= kJoinFew && rows >= kJoinRows; }

template <typename IO, int KT>
void launch_join(const AttendArgs& a, const AttendShape& h, hipStream_t st) {
  if (h.splits <= 1) return;
  const int64_t rows = static_cast<int64_t>(a.s.batch.tokens) * a.s.q_heads;
  if (joins_by_wave(h.splits, rows)) {
    const dim3 grid(static_cast<unsigned>((rows + 3) / 4));
    if (a.s.head_dim <= 128) hipLaunchKernelGGL((join_few_kernel<IO, KT, 2>), grid, dim3(256), 0, st, a, h.rows_per_tile);
    else hipLaunchKernelGGL((join_few_kernel<IO, KT, 8>), grid, dim3(256), 0, st, a, h.rows_per_tile);
    return;
  }
  const dim3 grid(static_cast<unsigned>(rows));
  if (a.s.head_dim <= 128) hipLaunchKernelGGL((join_splits_kernel<IO, KT, 32>), grid, dim3(kJoinThreads), 0, st, a, h.rows_per_tile);
  else hipLaunchKernelGGL((join_splits_kernel<IO, KT, 128>), grid, dim3(kJoinThreads), 0, st, a, h.rows_per_tile);
}

template <typename IO, int DP>
void launch_any(const AttendArgs& a, unsigned grid, hipStream_t st) {
  constexpr int VE = 16 / sizeof(IO);
  if constexpr (DP == 512) hipLaunchKernelGGL((attend_any_kernel<IO, DP, 1>), dim3(grid), dim3(kAnyWaves * kWave), 0, st, a);
  else if (a.s.head_dim % VE == 0 && rows_aligned16(a.s.cache, a.s.head_dim * static_cast<int>(sizeof(IO))))
    hipLaunchKernelGGL((attend_any_kernel<IO, DP, VE>), dim3(grid), dim3(kAnyWaves * kWave), 0, st, a);
  else
    hipLaunchKernelGGL((attend_any_kernel<IO, DP, 1>), dim3(grid), dim3(kAnyWaves * kWave), 0, st, a);
}
template <typename IO, int DP, int KT, bool MOD>
void launch_half(const AttendArgs& a, const AttendShape& h, unsigned grid, hipStream_t st) {
  const int vector = aligned16(a.s.q) && aligned16(a.out);
  if (h.step) hipLaunchKernelGGL((attend_step_kernel<IO, DP, kStepWaves, MOD>), dim3(grid), dim3(kStepWaves * kWave), 0, st, a, vector);
  else if (DP <= 128 && h.waves == 8) hipLaunchKernelGGL((attend_tile_kernel<IO, DP, KT, DP <= 128 ? 8 : 4, MOD>), dim3(grid), dim3(8 * kWave), 0, st, a, vector);
  else hipLaunchKernelGGL((attend_tile_kernel<IO, DP, KT, 4, MOD>), dim3(grid), dim3(4 * kWave), 0, st, a, vector);
  if (h.step) launch_join<IO, 32>(a, h, st);
  else launch_join<IO, KT>(a, h, st);
}
template <typename IO>
void launch_attend(const AttendArgs& a, const AttendShape& h, bool mod, unsigned grid, hipStream_t st) {
  const int d = a.s.head_dim;
  if constexpr (sizeof(IO) == 2) {
    if (h.half) {
      if (mod) {
        if (d <= 64) launch_half<IO, 64, 64, true>(a, h, grid, st);
        else if (d <= 128) launch_half<IO, 128, 32, true>(a, h, grid, st);
        else launch_half<IO, 256, 32, true>(a, h, grid, st);
      } else {
        if (d <= 64) launch_half<IO, 64, 64, false>(a, h, grid, st);
        else if (d <= 128) launch_half<IO, 128, 64, false>(a, h, grid, st);
        else launch_half<IO, 256, 32, false>(a, h, grid, st);
      }
      return;
    }
  }
  if (d <= 64) launch_any<IO, 64>(a, grid, st);
  else if (d <= 128) launch_any<IO, 128>(a, grid, st);
  else if (d <= 256) launch_any<IO, 256>(a, grid, st);
  else launch_any<IO, 512>(a, grid, st);
  launch_join<IO, kAnyKeys>(a, h, st);
}

template <typename IO, int DP>
void launch_weights_any(const WeightArgs& a, unsigned grid, hipStream_t st) {
  hipLaunchKernelGGL((key_weights_any_kernel<IO, DP>), dim3(grid), dim3(kAnyWaves * kWave), 0, st, a);
}
template <typename IO, int DP>
void launch_weights_half(const WeightArgs& a, bool mod, unsigned grid, hipStream_t st) {
  const int vector = aligned16(a.s.q);
  if (mod) hipLaunchKernelGGL((key_weights_kernel<IO, DP, true>), dim3(grid), dim3(kWeightWaves * kWave), 0, st, a, vector);
  else hipLaunchKernelGGL((key_weights_kernel<IO, DP, false>), dim3(grid), dim3(kWeightWaves * kWave), 0, st, a, vector);
}
template <typename IO>
void launch_weights(const WeightArgs& a, bool mod, unsigned grid, hipStream_t st) {
  const int d = a.s.head_dim;
  if constexpr (sizeof(IO) == 2) {
    if (a.waves_per_block) {
      if (d <= 64) launch_weights_half<IO, 64>(a, mod, grid, st);
      else if (d <= 128) launch_weights_half<IO, 128>(a, mod, grid, st);
      else launch_weights_half<IO, 256>(a, mod, grid, st);
      return;
    }
  }
  if (d <= 64) launch_weights_any<IO, 64>(a, grid, st);
  else if (d <= 128) launch_weights_any<IO, 128>(a, grid, st);
  else if (d <= 256) launch_weights_any<IO, 256>(a, grid, st);
  else launch_weights_any<IO, 512>(a, grid, st);
}

template <typename IO>
void launch_install(const InstallArgs& a, bool wide, unsigned grid, hipStream_t st) {
  if (wide) hipLaunchKernelGGL((install_tokens_kernel<IO, 16 / sizeof(IO)>), dim3(grid), dim3(kInstallWaves * kWave), 0, st, a);
  else hipLaunchKernelGGL((install_tokens_kernel<IO, 1>), dim3(grid), dim3(kInstallWaves * kWave), 0, st, a);
}

}  // namespace

extern "C" {

int cb_install_tokens(const cb_query_batch* batch, int32_t layer, int32_t dtype, int32_t head_dim, const cb_heads* q,
                      const cb_heads* q_out, const cb_heads* k, const cb_heads* v, const double* inv_freq,
                      int32_t rotary_dim, int32_t interleaved, float magnitude, const void* positions,
                      int32_t positions_kind, int32_t* d_error_flag, void* stream) {
  InstallArgs a{};
  int rc;
  if ((rc = check_batch(batch, dtype, head_dim, d_error_flag, true, &a.batch, &a.cache))) return rc;
  if (layer < 0 || layer >= batch->cache.num_layers) return fail(CB_EINVAL, "layer %d outside the cache", layer);
  if (!q) return fail(CB_EINVAL, "null q");
  const int eb = elem_bytes(dtype), kv = batch->cache.heads, n = batch->num_tokens;
  if (q->heads < 1 || q->heads > (1 << 16)) return fail(CB_EINVAL, "q needs 1 to 65536 heads");
  if ((rc = check_heads("q", q, q->heads, eb, n, &a.q)) || (rc = check_output("q_out", q_out, q->heads, eb, n, head_dim, &a.q_out)) ||
      (rc = check_heads("k", k, kv, eb, n, &a.k)) || (rc = check_heads("v", v, kv, eb, n, &a.v)))
    return rc;
  if (rotary_dim < 2 || rotary_dim > head_dim || rotary_dim % 2)
    return fail(CB_EINVAL, "rotary_dim must be even, 2 to head_dim");
  if (!inv_freq) return fail(CB_EINVAL, "null inv_freq");
  if (!std::isfinite(magnitude)) return fail(CB_EINVAL, "magnitude must be finite");
  if (positions && positions_kind != CB_INDEX_I32 && positions_kind != CB_INDEX_I64)
    return fail(CB_EINVAL, "positions must be int32 or int64");
  if (shares_rows(*batch)) return fail(CB_EINVAL, "several requests need offsets or a request_stride");
  if (n == 0 || batch->num_requests == 0) return CB_OK;
  a.layer = layer;
  a.head_dim = head_dim;
  a.rotary_dim = rotary_dim;
  a.interleaved = interleaved != 0;
  a.q_heads = q->heads;
  a.kv_heads = kv;
  a.inv_freq = inv_freq;
  a.positions = positions;
  a.positions_kind = positions_kind;
  a.magnitude = magnitude;
  const int vec = 16 / eb;
  const bool wide = (rotary_dim / 2) % vec == 0 && head_dim % vec == 0 && aligned16(a.q) && aligned16(a.q_out) &&
                    aligned16(a.k) && aligned16(a.v) && rows_aligned16(a.cache, head_dim * eb);
  const int items = (q->heads + kv) * (head_dim - rotary_dim / 2) / (wide ? vec : 1) + kv * head_dim / (wide ? vec : 1);
  a.slices = std::max(1, std::min(64, ceil_div(items, kWave)));  // an item a lane: one round of memory latency
  const int64_t grid = (static_cast<int64_t>(n) * a.slices + kInstallWaves - 1) / kInstallWaves + (d_error_flag ? 1 : 0);
  if (!launch_fits(grid, kInstallWaves * kWave)) return fail(CB_EINVAL, "too many tokens");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == CB_DTYPE_BF16) launch_install<io_bf16>(a, wide, static_cast<unsigned>(grid), st);
  else if (dtype == CB_DTYPE_F16) launch_install<io_f16>(a, wide, static_cast<unsigned>(grid), st);
  else launch_install<float>(a, wide, static_cast<unsigned>(grid), st);
  CB_HIP(hipGetLastError());
  return CB_OK;
}

int cb_attention_workspace_bytes(const cb_query_batch* batch, int32_t dtype, int32_t head_dim, const cb_scores* scores,
                                 int32_t query_heads, int64_t* bytes) {
  if (!bytes) return fail(CB_EINVAL, "null bytes");
  ScoreArgs s{};
  int rc;
  if ((rc = check_scores(batch, 0, dtype, head_dim, scores, query_heads, nullptr, &s))) return rc;
  *bytes = s.batch.tokens && s.batch.requests ? attend_workspace(s, attend_shape(s, dtype, scores->fp32_weights != 0)) : 0;
  return CB_OK;
}

int cb_paged_attention(const cb_query_batch* batch, int32_t layer, int32_t dtype, int32_t head_dim,
                       const cb_scores* scores, const cb_heads* q, const cb_heads* out, float* lse, void* d_workspace,
                       int64_t workspace_bytes, int32_t* d_error_flag, void* stream) {
  if (!q) return fail(CB_EINVAL, "null q");
  AttendArgs a{};
  int rc;
  if ((rc = check_scores(batch, layer, dtype, head_dim, scores, q->heads, d_error_flag, &a.s))) return rc;
  const int eb = elem_bytes(dtype), n = batch->num_tokens;
  if ((rc = check_heads("q", q, q->heads, eb, n, &a.s.q)) || (rc = check_output("out", out, q->heads, eb, n, head_dim, &a.out))) return rc;
  if (n == 0 || batch->num_requests == 0) return CB_OK;
  const AttendShape h = attend_shape(a.s, dtype, scores->fp32_weights != 0);
  const int64_t need = attend_workspace(a.s, h);
  if (need > 0 && (!d_workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(d_workspace) % 256))
    return fail(CB_EINVAL, "attention needs a 256-byte aligned workspace of %lld bytes", static_cast<long long>(need));
  a.lse = lse;
  a.request_slots = h.request_slots;
  a.splits = h.splits;
  a.least_tiles = h.least_tiles;
  a.by_splits = h.splits > 1 && !h.step ? static_cast<uint32_t>(((int64_t{1} << 32) + h.splits - 1) / h.splits) : 0;
  if (need > 0) {
    a.part_out = static_cast<float*>(d_workspace);
    a.part_lse = reinterpret_cast<float*>(static_cast<char*>(d_workspace) +
                                          round256(static_cast<int64_t>(h.splits) * n * q->heads * head_dim * 4));
  }
  const int64_t grid = h.tile_slots * h.splits * a.s.kv_heads;
  const int64_t rows = static_cast<int64_t>(n) * q->heads;
  if (!launch_fits(grid, (h.step ? kStepWaves : h.waves) * kWave) || rows > 0x7fffffff ||
      (h.splits > 1 && !joins_by_wave(h.splits, rows) && !launch_fits(rows, kJoinThreads)))
    return fail(CB_EINVAL, "too many query tiles");
  a.tile_slots = static_cast<int32_t>(h.tile_slots);
  const bool mod = a.s.mod;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == CB_DTYPE_BF16) launch_attend<io_bf16>(a, h, mod, static_cast<unsigned>(grid), st);
  else if (dtype == CB_DTYPE_F16) launch_attend<io_f16>(a, h, mod, static_cast<unsigned>(grid), st);
  else launch_attend<float>(a, h, mod, static_cast<unsigned>(grid), st);
  CB_HIP(hipGetLastError());
  return CB_OK;
}

int cb_add_key_weights(const cb_query_batch* batch, int32_t layer, int32_t dtype, int32_t head_dim,
                       const cb_scores* scores, const cb_heads* q, const float* lse, float* weights,
                       int64_t weights_stride, int32_t* d_error_flag, void* stream) {
  if (!q) return fail(CB_EINVAL, "null q");
  WeightArgs a{};
  int rc;
  if ((rc = check_scores(batch, layer, dtype, head_dim, scores, q->heads, d_error_flag, &a.s))) return rc;
  const int eb = elem_bytes(dtype), n = batch->num_tokens;
  if ((rc = check_heads("q", q, q->heads, eb, n, &a.s.q))) return rc;
  if (weights_stride < batch->max_length) return fail(CB_EINVAL, "weights rows are shorter than max_length");
  if (n == 0 || batch->num_requests == 0 || batch->max_length == 0) return CB_OK;
  if (!lse || !weights) return fail(CB_EINVAL, "null lse or weights");
  a.lse = lse;
  a.weights = weights;
  a.weights_stride = weights_stride;
  int keys = 16;
  if (takes_half(a.s, dtype)) {
    const int64_t blocks = static_cast<int64_t>(a.s.kv_heads) * ceil_div(static_cast<int64_t>(batch->max_query) * a.s.group, 32);
    a.waves_per_block = blocks >= 4 ? 4 : blocks >= 2 ? 2 : 1;
    keys = 32 * (kWeightWaves / a.waves_per_block);
  }
  a.key_slots = ceil_div(batch->max_length, keys);
  const int64_t grid = static_cast<int64_t>(a.key_slots) * batch->num_requests;
  if (!launch_fits(grid, kWeightWaves * kWave)) return fail(CB_EINVAL, "too many cached tokens");
  const bool mod = a.s.mod;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == CB_DTYPE_BF16) launch_weights<io_bf16>(a, mod, static_cast<unsigned>(grid), st);
  else if (dtype == CB_DTYPE_F16) launch_weights<io_f16>(a, mod, static_cast<unsigned>(grid), st);
  else launch_weights<float>(a, mod, static_cast<unsigned>(grid), st);
  CB_HIP(hipGetLastError());
  return CB_OK;
}

int cb_evict_tokens(const cb_query_batch* batch, const cb_query_batch* target, int32_t dtype, int32_t head_dim,
                    const float* weights, int64_t weights_stride, int32_t budget, int32_t first, int32_t last,
                    int32_t* kept, int32_t* kept_lengths, float* kept_weights, int32_t* d_error_flag, void* stream) {
  EvictArgs a{};
  MoveArgs m{};
  int rc;
  if ((rc = check_batch(batch, dtype, head_dim, d_error_flag, false, &a.batch, &m.src)) ||
      (rc = check_batch(target, dtype, head_dim, d_error_flag, false, &a.target, &m.dst)))
    return rc;
  if (target->num_requests != batch->num_requests) return fail(CB_EINVAL, "batch and target differ in requests");
  if (target->cache.heads != batch->cache.heads || target->cache.num_layers != batch->cache.num_layers)
    return fail(CB_EINVAL, "batch and target differ in layers or KV heads");
  if (budget < 1 || budget > (1 << 30)) return fail(CB_EINVAL, "budget must be 1 to 2^30");
  if (first < 0 || last < 0 || static_cast<int64_t>(first) + last > budget)
    return fail(CB_EINVAL, "first + last must be within the budget");
  if (weights_stride < batch->max_length) return fail(CB_EINVAL, "weights rows are shorter than max_length");
  if (batch->num_requests == 0) return CB_OK;
  if ((!weights && batch->max_length > 0) || !kept || !kept_lengths || !kept_weights) return fail(CB_EINVAL, "null weights or kept");
  if (shares_rows(*target)) return fail(CB_EINVAL, "several requests of target need offsets or a request_stride");
  const int eb = elem_bytes(dtype);
  const int64_t row_bytes = static_cast<int64_t>(batch->cache.heads) * head_dim * eb;
  if (row_bytes > (1 << 24)) return fail(CB_EINVAL, "rows above 16 MB");
  a.weights = weights;
  a.weights_stride = weights_stride;
  a.budget = budget;
  a.first = first;
  a.last = last;
  a.target_span = static_cast<int32_t>(std::min<int64_t>(request_span(*target), 1 << 30));
  a.kept = kept;
  a.kept_lengths = kept_lengths;
  a.kept_weights = kept_weights;
  const bool wide = row_bytes % 16 == 0 && rows_aligned16(m.src, 16) && rows_aligned16(m.dst, 16);
  const int chunk = wide ? 16 : eb;
  m.e = a;
  m.chunks_per_row = static_cast<int32_t>(row_bytes / chunk);
  m.tokens_per_block = std::max(1, 1024 / m.chunks_per_row);
  m.blocks_per_request = ceil_div(std::min(budget, std::max(batch->max_length, 1)), m.tokens_per_block);
  const int64_t blocks = static_cast<int64_t>(m.blocks_per_request) * batch->num_requests;
  if (!launch_fits(blocks, 256) || !launch_fits(batch->num_requests, kSelectThreads) || batch->cache.num_layers > 32767)
    return fail(CB_EINVAL, "eviction too large");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 requests(static_cast<unsigned>(batch->num_requests));
  const int64_t middle = static_cast<int64_t>(batch->max_length) - first - last;
  if (middle <= 16 * kSelectThreads) hipLaunchKernelGGL(select_tokens_kernel<16>, requests, dim3(kSelectThreads), 0, st, a);
  else if (middle <= 64 * kSelectThreads) hipLaunchKernelGGL(select_tokens_kernel<64>, requests, dim3(kSelectThreads), 0, st, a);
  else hipLaunchKernelGGL(select_tokens_kernel<0>, requests, dim3(kSelectThreads), 0, st, a);
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(2 * batch->cache.num_layers));
  if (wide) hipLaunchKernelGGL(move_rows_kernel<uint4>, grid, dim3(256), 0, st, m);
  else if (eb == 4) hipLaunchKernelGGL(move_rows_kernel<uint32_t>, grid, dim3(256), 0, st, m);
  else hipLaunchKernelGGL(move_rows_kernel<uint16_t>, grid, dim3(256), 0, st, m);
  CB_HIP(hipGetLastError());
  return CB_OK;
}

}  // extern "C"
