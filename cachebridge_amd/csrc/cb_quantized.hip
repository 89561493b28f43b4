// Queries on an 8-bit cache for MI355X (gfx950): prefixes quantized into it, new
// tokens rotated and stored into it, attention over it. The C ABI and the
// format are in include/cachebridge_hip.h: e4m3 codes, one power of two as
// scale for each layer, page and KV head, K and V apart.
//
// A scale that is a power of two costs a floating-point code nothing: codes
// are exact multiples of it, a page whose scale grows only rounds those of its
// codes again that become subnormal, and bf16 holds every value exactly.

#include "cb_attend.h"
#include "cb_rotate.h"

namespace {

// ---------------------------------------------------------------------------
// Codes and scales
// ---------------------------------------------------------------------------

struct PageScales {
  uint8_t* k;
  uint8_t* v;
  int64_t layer_stride, page_stride;
  int64_t pages;
  int32_t page_size;
  int32_t page_shift;  // log2(page_size), or -1

  CB_INLINE CB_GLOBAL uint8_t* at(int kind, int layer, int64_t page, int head) const {
    return reinterpret_cast<CB_GLOBAL uint8_t*>(as_global(static_cast<void*>(kind ? v : k))) + layer * layer_stride + page * page_stride + head;
  }
  CB_INLINE int64_t page_of(int64_t row) const {
    const uint32_t x = static_cast<uint32_t>(row);  // rows are below 2^31
    return page_shift >= 0 ? x >> page_shift : x / static_cast<uint32_t>(page_size);
  }
};

__device__ inline float scale_value(uint32_t byte) { return __uint_as_float(byte << 23); }

struct ScaledCache {
  typedef uint8_t elem;
  static constexpr bool kScaled = true;
  PageScales scales;
  CB_INLINE float scale(int kind, int layer, int64_t row, int head) const {
    return scale_value(*scales.at(kind, layer, scales.page_of(row), head));
  }
  static __device__ inline float value(uint8_t x) { return __builtin_amdgcn_cvt_f32_fp8(x, 0); }
};

constexpr float kMaxCode = 448.0f;
constexpr int kLeastExponent = -126, kMostExponent = 127, kMostExponentF16 = 7;

__device__ inline float finite_size(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.0f;
}

// The least e with top <= 448 * 2^e, 448 being 1.75 * 2^8.
__device__ inline int needed_exponent(float top, int most) {
  const uint32_t u = __float_as_uint(top);
  const int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return u == 0 ? kLeastExponent : max(kLeastExponent, min(most, e));
}

// 2^-e for e in [-126, 127], exact but for the last, whose reciprocal is subnormal.
__device__ inline float inverse_scale(int e) { return __uint_as_float(e < 127 ? static_cast<uint32_t>(127 - e) << 23 : 1u << 22); }

// An element over the scale, ready to be rounded: what the scale's bound leaves
// out stays at 448, what is not finite becomes NaN.
__device__ inline float scaled(float x, float inv) {
  const float y = __builtin_amdgcn_fmed3f(x * inv, -kMaxCode, kMaxCode);
  return fabsf(x) < INFINITY ? y : __uint_as_float(0x7fc00000u);
}

__device__ inline uint32_t pack_codes(float a, float b, float c, float d) {
  return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
}

// V codes to `to`, as one or a few stores where V allows it.
template <int V>
CB_INLINE void store_codes(gptr to, const float* x, float inv) {
  if constexpr (V % 4 == 0) {
    typedef uint32_t words __attribute__((ext_vector_type(V / 4)));
    words w;
#pragma unroll
    for (int i = 0; i < V / 4; ++i)
      w[i] = pack_codes(scaled(x[4 * i], inv), scaled(x[4 * i + 1], inv), scaled(x[4 * i + 2], inv), scaled(x[4 * i + 3], inv));
    gstore<words>(to, w);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) gstore<uint8_t>(to + i, static_cast<uint8_t>(pack_codes(scaled(x[i], inv), 0, 0, 0)));
  }
}

CB_INLINE float wave_max(float x) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) x = fmaxf(x, __shfl_xor(x, d));
  return x;
}

// The pool page that holds page `page` of request r, or -1. Called for block
// tables of the scales' page size.
CB_INLINE int64_t pool_page(const QBatch& B, const PageScales& s, const Request& r, int page) {
  const int64_t e = r.first + page;
  if (e >= B.entries) return -1;
  const int64_t p = reinterpret_cast<const CB_GLOBAL int32_t*>(as_global(B.index))[e];
  return p >= 0 && (p + 1) * s.page_size <= B.rows ? p : -1;
}

// ---------------------------------------------------------------------------
// A prefix into the 8-bit cache
// ---------------------------------------------------------------------------

struct QuantizeArgs {
  QBatch batch, target;
  DevRows src, dst;
  PageScales scales;
  int32_t head_dim, heads;
  int32_t pages;        // of a request, at most
  int32_t target_span;  // index entries of the target that are a request's own
  int32_t most;         // a scale's largest exponent
  uint32_t page_groups;
  int32_t* lengths;
};

// Request b's places on both sides and its cached tokens, or -1 if it is outside the bounds.
CB_INLINE int quantize_request(const QuantizeArgs& a, int b, Request& src, Request& dst) {
  place_request(a.batch, b, src);
  place_request(a.target, b, dst);
  const int length = a.batch.lengths[b];
  return (src.ok & dst.ok & (dst.rem == 0) & (length >= 0) & (length <= a.batch.max_length)) ? length : -1;
}

// One workgroup looks through a request's index on both sides, so that its length
// has one writer.
CB_INLINE void report_request(const QuantizeArgs& a, int b) {
  __shared__ int missing;
  Request src, dst;
  const int length = quantize_request(a, b, src, dst);
  if (threadIdx.x == 0) missing = 0;
  __syncthreads();
  bool gone = false, nowhere = length > a.target_span;
#pragma unroll 4
  for (int j = threadIdx.x; j < length; j += blockDim.x) gone |= cache_row(a.batch, src, j) < 0;
  for (int p = threadIdx.x; p * a.scales.page_size < min(length, a.target_span); p += blockDim.x)
    nowhere |= pool_page(a.target, a.scales, dst, p) < 0;
  if (nowhere) flag(a.batch.err, CB_ERROR_TARGET_ROW);
  if (gone) {
    flag(a.batch.err, CB_ERROR_CACHE_ROW);
    missing = 1;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    if (length < 0) flag(a.batch.err, CB_ERROR_REQUEST);
    a.lengths[b] = missing || length < 0 ? 0 : length;
  }
}

// A wave a page and head of one layer's K or V: V elements a lane and step, the
// page's largest by an exchange among the lanes, then the codes. Pages of up
// to 64 * KEEP vectors stay in registers between the two, longer ones are read
// again (from L2).
template <typename IO, int V, int KEEP>
__global__ __launch_bounds__(256) void quantize_tokens_kernel(QuantizeArgs a) {
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  if (blockIdx.x >= a.page_groups) {
    if (blockIdx.y == 0) report_request(a, blockIdx.x - a.page_groups);
    return;
  }
  const int layer = blockIdx.y >> 1, kind = blockIdx.y & 1;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + wave;
  const int head = static_cast<int>(unit % a.heads);
  const int64_t rest = unit / a.heads;
  const int page = static_cast<int>(rest % a.pages);
  const int64_t b = rest / a.pages;
  if (b >= a.batch.requests) return;
  Request src, dst;
  const int length = min(quantize_request(a, static_cast<int>(b), src, dst), a.target_span);
  const int ps = a.scales.page_size, j0 = page * ps;
  if (j0 >= length) return;
  const int64_t to_page = pool_page(a.target, a.scales, dst, page);
  if (to_page < 0) return;
  const int per = a.head_dim / V, total = min(ps, length - j0) * per;
  gcptr from = layer_base(a.src, kind, layer) + static_cast<int64_t>(head) * a.head_dim * static_cast<int>(sizeof(IO));
  gptr to = const_cast<gptr>(layer_base(a.dst, kind, layer)) + to_page * ps * a.dst.row_stride_b + static_cast<int64_t>(head) * a.head_dim;
  float x[KEEP][V];
  bool has[KEEP];
  auto load = [&](int base) __attribute__((always_inline)) {
    int64_t row[KEEP];
#pragma unroll
    for (int u = 0; u < KEEP; ++u) {
      const int at = min(base + u * kWave + lane, total - 1);
      row[u] = cache_row(a.batch, src, j0 + at / per);
      has[u] = (row[u] >= 0) & (base + u * kWave + lane < total);
    }
#pragma unroll
    for (int u = 0; u < KEEP; ++u) {
      const int at = min(base + u * kWave + lane, total - 1);
      const char* p = (const char*)from + max(row[u], int64_t{0}) * a.src.row_stride_b + (at % per) * V * static_cast<int>(sizeof(IO));
      constexpr int W = V * sizeof(IO) % 16 == 0 ? 16 / sizeof(IO) : 1;
#pragma unroll
      for (int w = 0; w < V / W; ++w) load_vec<IO, W>(p + w * W * sizeof(IO), x[u] + w * W);
    }
  };
  float top = 0;
  for (int base = 0; base < total; base += KEEP * kWave) {
    load(base);
#pragma unroll
    for (int u = 0; u < KEEP; ++u)
#pragma unroll
      for (int i = 0; i < V; ++i) top = fmaxf(top, has[u] ? finite_size(x[u][i]) : 0.0f);
  }
  const int e = needed_exponent(wave_max(top), a.most);
  const float inv = inverse_scale(e);
  for (int base = 0; base < total; base += KEEP * kWave) {
    if (total > KEEP * kWave) load(base);
#pragma unroll
    for (int u = 0; u < KEEP; ++u) {
      const int at = base + u * kWave + lane;
      if (has[u]) store_codes<V>(to + (at / per) * a.dst.row_stride_b + (at % per) * V, x[u], inv);
    }
  }
  if (lane == 0) *a.scales.at(kind, layer, to_page, head) = static_cast<uint8_t>(e + 127);
}

// ---------------------------------------------------------------------------
// New tokens into the 8-bit cache
// ---------------------------------------------------------------------------

struct InstallQuantizedArgs {
  InstallArgs i;
  PageScales scales;
  int32_t most;
  uint32_t page_groups;
};

template <int V>
constexpr int kTurns = V == 8 ? 512 : kMaxPairs;  // pairs that 64 items turn, and those of one row at least

// The new rows of one page, head and kind (0: K, 1: V): a wave. Token row t is
// the page's first new one. Items of 2 V elements (both vectors of V pairs, or
// two neighbours) lie one a lane in rounds of whole rows; up to KEEP rounds
// stay in registers until the page's scale is known, more are read (and turned)
// twice.
template <typename IO, int V, int KEEP>
CB_INLINE void store_page(const InstallQuantizedArgs& q, const Request& r, int t, int head, int kind, turn_pair<IO>* turn) {
  const InstallArgs& a = q.i;
  const int lane = threadIdx.x & (kWave - 1);
  const int ps = q.scales.page_size, i0 = t - r.q0, p0 = r.length - r.n + i0;
  const int page = q.scales.page_shift >= 0 ? p0 >> q.scales.page_shift : p0 / ps, slot = p0 - page * ps;
  const int rows = min(ps - slot, r.n - i0);
  const int64_t to_page = pool_page(a.batch, q.scales, r, page);
  if (to_page < 0) {
    if (lane == 0) flag(a.batch.err, CB_ERROR_TARGET_ROW);
    return;
  }
  CB_GLOBAL uint8_t* scale = q.scales.at(kind, a.layer, to_page, head);
  const int had = slot > 0 ? static_cast<int>(*scale) - 127 : kLeastExponent;
  const int D = a.head_dim, pairs = a.rotary_dim / 2;
  gptr to = const_cast<gptr>(layer_base(a.cache, kind, a.layer)) + to_page * ps * a.cache.row_stride_b + static_cast<int64_t>(head) * D;
  const Strided& from = kind ? a.v : a.k;
  const char* base = from.data + t * from.token_b + head * from.head_b;

  const int turned = kind ? 0 : pairs / V, straight = kind ? 0 : a.rotary_dim;
  const int plain = (D - straight) / V, items = turned + (plain + 1) / 2;
  const int per_round = max(1, kWave / items), parts = (items + kWave - 1) / kWave;
  const int rounds = (rows + per_round - 1) / per_round * parts;
  struct Item {
    int row, first, second;  // elements of the two vectors
    bool on, two;
  };
  auto item = [&](int n) __attribute__((always_inline)) {
    Item m;
    const int row0 = n / parts * per_round, part = n - n / parts * parts;
    const int in = parts == 1 ? lane / items : 0, k = parts == 1 ? lane - in * items : part * kWave + lane;
    m.row = row0 + in;
    m.on = (in < per_round) & (m.row < rows) & (k < items);
    if (k < turned) {
      m.first = a.interleaved ? 2 * k * V : k * V;
      m.second = a.interleaved ? m.first + V : m.first + pairs;
      m.two = true;
    } else {
      m.first = straight + 2 * (k - turned) * V;
      m.second = m.first + V;
      m.two = 2 * (k - turned) + 1 < plain;
    }
    return m;
  };
  auto load = [&](int n, float (&y)[2 * V]) __attribute__((always_inline)) {
    const int row0 = n / parts * per_round;
    if (kind == 0 && n % parts == 0) {
      const int all = min(per_round, rows - row0) * pairs;
      for (int x = lane; x < all; x += kWave) {
        const int at = row0 + x / pairs;
        turn[x] = turn_of<turn_pair<IO>, turn_t<IO>>(a, t + at, p0 + at, x % pairs);
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    const Item m = item(n);
    float x[2 * V] = {};
    if (m.on) {
      const char* at = base + m.row * from.token_b;
      load_vec<IO, V>(at + m.first * static_cast<int>(sizeof(IO)), x);
      if (m.two) load_vec<IO, V>(at + m.second * static_cast<int>(sizeof(IO)), x + V);
    }
#pragma unroll
    for (int i = 0; i < 2 * V; ++i) y[i] = x[i];
    if (kind == 0) {
      const int k = a.interleaved ? m.first / 2 : m.first;
      if (m.on & (m.first < straight)) turn_pairs<V>(x, turn + (m.row - row0) * pairs + k, a.interleaved, y);
      __builtin_amdgcn_wave_barrier();  // before the next round's angles
    }
  };
  float y[KEEP][2 * V];
  float top = 0;
  for (int n0 = 0; n0 < rounds; n0 += KEEP)
#pragma unroll
    for (int u = 0; u < KEEP; ++u)
      if (n0 + u < rounds) {
        load(n0 + u, y[u]);
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) top = fmaxf(top, finite_size(y[u][i]));
      }
  const int e = max(had, needed_exponent(wave_max(top), q.most));
  const float inv = inverse_scale(e);
  for (int n0 = 0; n0 < rounds; n0 += KEEP)
#pragma unroll
    for (int u = 0; u < KEEP; ++u)
      if (n0 + u < rounds) {
        if (rounds > KEEP) load(n0 + u, y[u]);
        const Item m = item(n0 + u);
        gptr at = to + (slot + m.row) * a.cache.row_stride_b;
        if (m.on) store_codes<V>(at + m.first, y[u], inv);
        if (m.on & m.two) store_codes<V>(at + m.second, y[u] + V, inv);
      }
  if (e > had && slot > 0) {  // cached tokens of a page whose scale grows
    const float by = inverse_scale(min(e - had, 127));
    const int words = D / 2;
    for (int x = lane; x < slot * words; x += kWave) {
      gptr at = to + x / words * a.cache.row_stride_b + x % words * 2;
      const uint32_t c0 = gload<uint8_t>(at), c1 = gload<uint8_t>(at + 1);
      const uint32_t c = pack_codes(__builtin_amdgcn_cvt_f32_fp8(c0, 0) * by, __builtin_amdgcn_cvt_f32_fp8(c1, 0) * by, 0, 0);
      gstore<uint8_t>(at, static_cast<uint8_t>(c));
      gstore<uint8_t>(at + 1, static_cast<uint8_t>(c >> 8));
    }
  }
  if (lane == 0 && (e > had || slot == 0)) *scale = static_cast<uint8_t>(e + 127);
}

// One launch, two kinds of workgroups: those of a wave a (token, head, K or V),
// which store a page's new rows if the token is the first of them, and those that
// rotate the queries (install_rows).
template <typename IO, int V>
__global__ __launch_bounds__(kInstallWaves * kWave) void install_quantized_kernel(InstallQuantizedArgs q) {
  __shared__ turn_pair<IO> turn[kInstallWaves][kTurns<V>];
  const InstallArgs& a = q.i;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  if (blockIdx.x >= q.page_groups) {
    if (a.batch.err && blockIdx.x == gridDim.x - 1) {  // a workgroup more than there are tokens for
      if (wave == 0) flag_requests(a.batch);
      return;
    }
    install_rows<IO, V, false, true>(a, static_cast<int64_t>(blockIdx.x - q.page_groups) * kInstallWaves + wave, turn[wave]);
    return;
  }
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kInstallWaves + wave;
  const int t = static_cast<int>(unit / (2 * a.kv_heads)), rest = static_cast<int>(unit % (2 * a.kv_heads));
  if (t >= a.batch.tokens) return;
  const int b = request_of_token(a.batch, t);
  if (b >= a.batch.requests) return;
  const Request r = load_request(a.batch, b);
  if (!r.ok) return;
  if (r.rem != 0) {  // it shares a page with what lies before it
    flag(a.batch.err, CB_ERROR_REQUEST);
    return;
  }
  const int p = r.length - r.n + (t - r.q0);
  if (t > r.q0 && p % q.scales.page_size != 0) return;
  store_page<IO, V, 2>(q, r, t, rest >> 1, rest & 1, turn[wave]);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

int check_scales(const cb_page_scales* scales, const cb_query_batch& batch, PageScales* s) {
  if (!scales || !scales->k || !scales->v) return fail(CB_EINVAL, "null scales");
  if (scales->page_size < 1 || scales->page_size > (1 << 20)) return fail(CB_EINVAL, "page_size must be 1 to 2^20");
  if (scales->pages < 0 || scales->pages > 0x7fffffff || scales->pages * scales->page_size < batch.cache.rows)
    return fail(CB_EINVAL, "the scales' pages do not cover the cache's rows");
  if (scales->page_stride < batch.cache.heads) return fail(CB_EINVAL, "page_stride below the KV heads");
  if (scales->layer_stride < 0) return fail(CB_EINVAL, "negative layer_stride");
  s->k = scales->k;
  s->v = scales->v;
  s->layer_stride = scales->layer_stride;
  s->page_stride = scales->page_stride;
  s->pages = scales->pages;
  s->page_size = scales->page_size;
  s->page_shift = (s->page_size & (s->page_size - 1)) ? -1 : __builtin_ctz(static_cast<unsigned>(s->page_size));
  return CB_OK;
}

// A cache that rows are stored into: each page must be one request's.
int check_pages(const cb_query_batch& batch, const PageScales& s, const char* name) {
  if (batch.cache.index_kind != CB_INDEX_BLOCK_TABLE || batch.cache.page_size != s.page_size)
    return fail(CB_EINVAL, "%s must have a block table of the scales' page_size", name);
  if (shares_rows(batch)) return fail(CB_EINVAL, "several requests of %s need offsets or a request_stride", name);
  return CB_OK;
}

int most_exponent(int32_t dtype) { return dtype == CB_DTYPE_F16 ? kMostExponentF16 : kMostExponent; }

AttendShape quantized_shape(const ScoreArgs& s) {
  AttendShape h{};
  h.waves = kAnyWaves;
  h.rows_per_tile = kAnyRows;
  h.keys_per_tile = kAnyKeys;
  const QBatch& B = s.batch;
  const int per_request = std::max(1, ceil_div(static_cast<int64_t>(B.max_query) * s.group, h.rows_per_tile));
  const int64_t by_request = static_cast<int64_t>(per_request) * B.requests;
  const int64_t packed = ceil_div(static_cast<int64_t>(B.tokens) * s.group, h.rows_per_tile) + static_cast<int64_t>(B.requests);
  h.request_slots = by_request <= packed ? per_request : 0;
  h.tile_slots = std::min(by_request, packed);
  int64_t keys = B.max_length;
  if (s.window > 0 && s.causal && !s.prefix) keys = std::min<int64_t>(keys, static_cast<int64_t>(s.window) + std::min<int64_t>(B.max_query, h.rows_per_tile / s.group + 2));
  const int key_tiles = std::max(1, ceil_div(keys, h.keys_per_tile) + (s.prefix ? 1 : 0));
  const int64_t groups = h.tile_slots * s.kv_heads;
  h.least_tiles = 2;
  h.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(512 / std::max<int64_t>(1, groups), key_tiles / h.least_tiles)));
  return h;
}

template <typename IO>
void launch_quantized(const AttendArgs& a, const ScaledCache& cache, const AttendShape& h, unsigned grid, hipStream_t st) {
  const int d = a.s.head_dim;
  if (d <= 64) launch_any<IO, 64>(a, cache, grid, st);
  else if (d <= 128) launch_any<IO, 128>(a, cache, grid, st);
  else if (d <= 256) launch_any<IO, 256>(a, cache, grid, st);
  else launch_any<IO, 512>(a, cache, grid, st);
  launch_join<IO, kAnyKeys>(a, h, st);
}

template <typename IO>
void launch_store(const InstallQuantizedArgs& q, bool wide, unsigned grid, hipStream_t st) {
  if (wide) hipLaunchKernelGGL((install_quantized_kernel<IO, 16 / sizeof(IO)>), dim3(grid), dim3(kInstallWaves * kWave), 0, st, q);
  else hipLaunchKernelGGL((install_quantized_kernel<IO, 1>), dim3(grid), dim3(kInstallWaves * kWave), 0, st, q);
}

template <typename IO>
void launch_quantize(const QuantizeArgs& a, int vec, dim3 grid, hipStream_t st) {
  if (vec == 16) hipLaunchKernelGGL((quantize_tokens_kernel<IO, 16, 4>), grid, dim3(256), 0, st, a);
  else if (vec == 8) hipLaunchKernelGGL((quantize_tokens_kernel<IO, 8, 4>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((quantize_tokens_kernel<IO, 2, 4>), grid, dim3(256), 0, st, a);
}

}  // namespace

extern "C" {

int cb_install_quantized(const cb_query_batch* batch, const cb_page_scales* scales, int32_t layer, int32_t dtype,
                         int32_t head_dim, const cb_heads* q, const cb_heads* q_out, const cb_heads* k, const cb_heads* v,
                         const cb_rotation* rotation, int32_t* d_error_flag, void* stream) {
  InstallQuantizedArgs a{};
  int rc;
  if ((rc = check_batch(batch, dtype, head_dim, d_error_flag, true, &a.i.batch, &a.i.cache, 1)) ||
      (rc = check_scales(scales, *batch, &a.scales)) || (rc = check_pages(*batch, a.scales, "the batch")) ||
      (rc = check_install(batch, layer, dtype, head_dim, q, q_out, k, v, rotation, &a.i)))
    return rc;
  const int eb = elem_bytes(dtype), n = batch->num_tokens, rotary_dim = a.i.rotary_dim;
  if (n == 0 || batch->num_requests == 0) return CB_OK;
  const int vec = 16 / eb;
  const bool wide = (rotary_dim / 2) % vec == 0 && head_dim % vec == 0 && aligned16(a.i.q) && aligned16(a.i.q_out) &&
                    aligned16(a.i.k) && aligned16(a.i.v) && rows_aligned16(a.i.cache, 16) && head_dim % 8 == 0;
  const int items = a.i.q_heads * (head_dim - rotary_dim / 2) / (wide ? vec : 1);
  a.i.slices = std::max(1, std::min(64, ceil_div(items, kWave)));
  a.most = most_exponent(dtype);
  const int64_t pages = (static_cast<int64_t>(n) * 2 * a.i.kv_heads + kInstallWaves - 1) / kInstallWaves;
  const int64_t grid = pages + (static_cast<int64_t>(n) * a.i.slices + kInstallWaves - 1) / kInstallWaves + (d_error_flag ? 1 : 0);
  if (!launch_fits(grid, kInstallWaves * kWave)) return fail(CB_EINVAL, "too many tokens");
  a.page_groups = static_cast<uint32_t>(pages);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == CB_DTYPE_BF16) launch_store<io_bf16>(a, wide, static_cast<unsigned>(grid), st);
  else if (dtype == CB_DTYPE_F16) launch_store<io_f16>(a, wide, static_cast<unsigned>(grid), st);
  else launch_store<float>(a, wide, static_cast<unsigned>(grid), st);
  CB_HIP(hipGetLastError());
  return CB_OK;
}

int cb_quantize_tokens(const cb_query_batch* batch, const cb_query_batch* target, const cb_page_scales* scales,
                       int32_t dtype, int32_t head_dim, int32_t* lengths_out, int32_t* d_error_flag, void* stream) {
  QuantizeArgs a{};
  int rc;
  if ((rc = check_batch(batch, dtype, head_dim, d_error_flag, false, &a.batch, &a.src)) ||
      (rc = check_batch(target, dtype, head_dim, d_error_flag, false, &a.target, &a.dst, 1)) ||
      (rc = check_scales(scales, *target, &a.scales)))
    return rc;
  if (target->num_requests != batch->num_requests) return fail(CB_EINVAL, "batch and target differ in requests");
  if (target->cache.heads != batch->cache.heads || target->cache.num_layers != batch->cache.num_layers)
    return fail(CB_EINVAL, "batch and target differ in layers or KV heads");
  if (batch->num_requests == 0) return CB_OK;
  if (!lengths_out) return fail(CB_EINVAL, "null lengths_out");
  if ((rc = check_pages(*target, a.scales, "target"))) return rc;
  if (batch->cache.num_layers > 32767) return fail(CB_EINVAL, "more than 32767 layers");
  a.head_dim = head_dim;
  a.heads = batch->cache.heads;
  a.target_span = static_cast<int32_t>(std::min<int64_t>(request_span(*target), 1 << 30));
  a.most = most_exponent(dtype);
  a.lengths = lengths_out;
  a.pages = std::max(1, ceil_div(a.batch.max_length, a.scales.page_size));
  const int eb = elem_bytes(dtype);
  const bool aligned = rows_aligned16(a.src, head_dim * eb) && rows_aligned16(a.dst, 16);
  const int vec = aligned && head_dim % 16 == 0 ? 16 : aligned && head_dim % 8 == 0 ? 8 : 2;
  const int64_t units = static_cast<int64_t>(a.pages) * a.heads * batch->num_requests;
  const int64_t groups = (units + 3) / 4;
  if (!launch_fits(groups + batch->num_requests, 256)) return fail(CB_EINVAL, "too many pages");
  a.page_groups = static_cast<uint32_t>(groups);
  const dim3 grid(static_cast<unsigned>(groups + batch->num_requests), static_cast<unsigned>(2 * batch->cache.num_layers));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == CB_DTYPE_BF16) launch_quantize<io_bf16>(a, vec, grid, st);
  else if (dtype == CB_DTYPE_F16) launch_quantize<io_f16>(a, vec, grid, st);
  else launch_quantize<float>(a, vec, grid, st);
  CB_HIP(hipGetLastError());
  return CB_OK;
}

int cb_quantized_attention_workspace_bytes(const cb_query_batch* batch, const cb_page_scales* scales, int32_t dtype,
                                           int32_t head_dim, const cb_scores* scores, int32_t query_heads, int64_t* bytes) {
  if (!bytes) return fail(CB_EINVAL, "null bytes");
  ScoreArgs s{};
  PageScales p{};
  int rc;
  if ((rc = check_scores(batch, 0, dtype, head_dim, scores, query_heads, nullptr, &s, 1)) || (rc = check_scales(scales, *batch, &p)))
    return rc;
  *bytes = s.batch.tokens && s.batch.requests ? attend_workspace(s, quantized_shape(s)) : 0;
  return CB_OK;
}

int cb_quantized_attention(const cb_query_batch* batch, const cb_page_scales* scales, int32_t layer, int32_t dtype,
                           int32_t head_dim, const cb_scores* scores, const cb_heads* q, const cb_heads* out, float* lse,
                           void* d_workspace, int64_t workspace_bytes, int32_t* d_error_flag, void* stream) {
  if (!q) return fail(CB_EINVAL, "null q");
  AttendArgs a{};
  ScaledCache cache{};
  int rc;
  if ((rc = check_scores(batch, layer, dtype, head_dim, scores, q->heads, d_error_flag, &a.s, 1)) ||
      (rc = check_scales(scales, *batch, &cache.scales)))
    return rc;
  const int eb = elem_bytes(dtype), n = batch->num_tokens;
  if ((rc = check_heads("q", q, q->heads, eb, n, &a.s.q)) || (rc = check_output("out", out, q->heads, eb, n, head_dim, &a.out))) return rc;
  if (n == 0 || batch->num_requests == 0) return CB_OK;
  const AttendShape h = quantized_shape(a.s);
  unsigned grid;
  if ((rc = cut_attention(a, h, h.waves * kWave, lse, d_workspace, workspace_bytes, &grid))) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == CB_DTYPE_BF16) launch_quantized<io_bf16>(a, cache, h, grid, st);
  else if (dtype == CB_DTYPE_F16) launch_quantized<io_f16>(a, cache, h, grid, st);
  else launch_quantized<float>(a, cache, h, grid, st);
  CB_HIP(hipGetLastError());
  return CB_OK;
}

}  // extern "C"
