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

// Bytes above the largest that is ever stored read as it: 448 times that is
// finite, and a value that no row sees must not become an infinity.
constexpr float kMaxCode = 448.0f;
constexpr int kLeastExponent = -126, kMostExponent = 119, kMostExponentF16 = 7;

__device__ inline float scale_value(uint32_t byte, int most = kMostExponent) {
  return __uint_as_float(min(byte, static_cast<uint32_t>(most + 127)) << 23);
}

// The scales of one layer and head.
struct HeadScales {
  const CB_GLOBAL uint8_t* k;
  const CB_GLOBAL uint8_t* v;
  uint32_t page_stride, page_size;
  int32_t page_shift;

  CB_INLINE HeadScales(const PageScales& s, int layer, int head)
      : k(s.at(0, layer, 0, head)), v(s.at(1, layer, 0, head)), page_stride(s.page_stride), page_size(s.page_size), page_shift(s.page_shift) {}
  // Where the scale of pool row `row` is: its page's, pages times page_stride being below 2^32.
  CB_INLINE uint32_t at(int row) const {
    return (page_shift >= 0 ? static_cast<uint32_t>(row) >> page_shift : static_cast<uint32_t>(row) / page_size) * page_stride;
  }
};

struct ScaledCache {
  typedef uint8_t elem;
  static constexpr bool kScaled = true;
  PageScales scales;
  CB_INLINE float scale(int kind, int layer, int64_t row, int head) const {
    return scale_value(*scales.at(kind, layer, scales.page_of(row), head));
  }
  static __device__ inline float value(uint8_t x) { return __builtin_amdgcn_cvt_f32_fp8(x, 0); }
};

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

// 2^-e for e in [-126, 126].
__device__ inline float inverse_scale(int e) { return __uint_as_float(static_cast<uint32_t>(127 - e) << 23); }

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
// tables of the scales' page size. In two parts, so that other loads may be asked
// for between them.
CB_INLINE int page_entry(const QBatch& B, const Request& r, int page) {
  const int64_t e = r.first + page;
  return e < B.entries ? reinterpret_cast<const CB_GLOBAL int32_t*>(as_global(B.index))[e] : -1;
}
CB_INLINE int64_t page_of_entry(const QBatch& B, const PageScales& s, int entry) {
  const int64_t p = entry;
  return p >= 0 && (p + 1) * s.page_size <= B.rows ? p : -1;
}
CB_INLINE int64_t pool_page(const QBatch& B, const PageScales& s, const Request& r, int page) {
  return page_of_entry(B, s, page_entry(B, r, page));
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

// code = round(x / 2^e), e from the largest |x| of the page. Every element is read
// once (2 or 4 bytes) and written once (1): the copy rate bounds it. A wave a page
// and head of one layer's K or V: V elements a lane and step, the page's largest
// by an exchange among the lanes, then the codes. No barrier and no LDS: a page of
// 16 tokens of 128 is two vectors a lane, and waves that are at work on other pages hide
// its lookups. Pages of up to 64 * KEEP vectors stay in registers between
// the two, longer ones are read again (from L2). KEEP is the least of 2, 4 and 8
// that holds the page: 4096 tokens of 64 layers, 2 heads, 96
// us (KEEP 2; 403 MB, 4.2 TB/s with cold caches, 86 us in a row of calls); 16 fp16
// requests, 62 layers, pages of 32 340 us (KEEP 4; 1.5 GB, 4.5 TB/s).
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
  IO x[KEEP][V];
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
      for (int w = 0; w < V / W; ++w) {
        typedef IO vec __attribute__((ext_vector_type(W)));
        const vec y = gload<vec>(as_global(static_cast<const void*>(p + w * W * sizeof(IO))));
#pragma unroll
        for (int e = 0; e < W; ++e) x[u][w * W + e] = y[e];
      }
    }
  };
  float top = 0;
  for (int base = 0; base < total; base += KEEP * kWave) {
    load(base);
#pragma unroll
    for (int u = 0; u < KEEP; ++u)
#pragma unroll
      for (int i = 0; i < V; ++i) top = fmaxf(top, has[u] ? finite_size(to_f32(x[u][i])) : 0.0f);
  }
  const int e = needed_exponent(wave_max(top), a.most);
  const float inv = inverse_scale(e);
  for (int base = 0; base < total; base += KEEP * kWave) {
    if (total > KEEP * kWave) load(base);
#pragma unroll
    for (int u = 0; u < KEEP; ++u) {
      const int at = base + u * kWave + lane;
      float y[V];
#pragma unroll
      for (int i = 0; i < V; ++i) y[i] = to_f32(x[u][i]);
      if (has[u]) store_codes<V>(to + (at / per) * a.dst.row_stride_b + (at % per) * V, y, inv);
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
  int32_t page_slots;  // pages of a request that its new tokens may be in, or 0: a unit for each token
};

template <int V>
constexpr int kTurns = V == 8 ? 512 : kMaxPairs;  // pairs that 64 items turn, and those of one row at least

// The new rows of one page, head and kind (0: K, 1: V): a team of TW waves, one or
// the whole workgroup. Token row t is the page's first new one. Items of 2 V
// elements (both vectors of V pairs, or two neighbours) lie one a lane in rounds
// of whole rows, which the waves take in turn; up to KEEP rounds of a wave stay in
// registers until the page's scale is known, more are read (and turned) twice.
// Cached codes of the page, where a larger scale needs them rounded again, are
// read only then: a step in 16 meets a new page, and most others keep the scale.
template <typename IO, int V, int TW, int KEEP, typename AXES>
CB_INLINE void store_page(const InstallQuantizedArgs& q, const AXES& axes, const Request& r, int t, int head, int kind, turn_pair<IO>* turn) {
  __shared__ float tops[TW];
  const InstallArgs& a = q.i;
  const int lane = threadIdx.x & (kWave - 1), wave = TW > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) : 0;
  const int member = wave * kWave + lane;
  const int ps = q.scales.page_size, i0 = t - r.q0, p0 = r.length - r.n + i0;
  const int page = q.scales.page_shift >= 0 ? p0 >> q.scales.page_shift : p0 / ps, slot = p0 - page * ps;
  const int rows = min(ps - slot, r.n - i0);
  const int entry = page_entry(a.batch, r, page);  // on its way with the rows
  const int D = a.head_dim, pairs = a.rotary_dim / 2;
  const Strided& from = kind ? a.v : a.k;
  const char* base = from.data + t * from.token_b + head * from.head_b;

  const int turned = kind ? 0 : pairs / V, straight = kind ? 0 : a.rotary_dim;
  const int plain = (D - straight) / V, items = turned + (plain + 1) / 2;
  const int per_round = max(1, kWave / items), parts = (items + kWave - 1) / kWave;
  // This wave's rounds: groups of per_round rows, every TW-th from its own, parts each.
  const int groups = (rows + per_round - 1) / per_round, rounds = (max(groups - wave, 0) + TW - 1) / TW * parts;
  auto first_row = [&](int n) { return (wave + n / parts * TW) * per_round; };
  struct Item {
    int row, first, second;  // elements of the two vectors
    bool on, two;
  };
  auto item = [&](int n) __attribute__((always_inline)) {
    Item m;
    const int row0 = first_row(n), part = n - n / parts * parts;
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
    const int row0 = first_row(n);
    if (kind == 0 && n % parts == 0) {
      const int all = min(per_round, rows - row0) * pairs;
      for (int x = lane; x < all; x += kWave) {
        const int at = row0 + x / pairs;
        turn[x] = turn_of<turn_pair<IO>, turn_t<IO>>(a, p0 + at, load_angle(a, axes, t + at, x % pairs));
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
      if (m.on & (m.first < straight)) turn_pairs<V>(y, turn + (m.row - row0) * pairs + k, a.interleaved);
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
  const int64_t to_page = page_of_entry(a.batch, q.scales, entry);
  if (to_page < 0) {
    if (member == 0) flag(a.batch.err, CB_ERROR_TARGET_ROW);
    return;
  }
  CB_GLOBAL uint8_t* scale = q.scales.at(kind, a.layer, to_page, head);
  const int had = slot > 0 ? max(kLeastExponent, min(q.most, static_cast<int>(*scale) - 127)) : kLeastExponent;
  gptr to = const_cast<gptr>(layer_base(a.cache, kind, a.layer)) + to_page * ps * a.cache.row_stride_b + static_cast<int64_t>(head) * D;
  top = wave_max(top);
  if constexpr (TW > 1) {
    if (lane == 0) tops[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TW; ++w) top = fmaxf(top, tops[w]);
  }
  const int e = max(had, needed_exponent(top, q.most));
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
    const float by = inverse_scale(min(e - had, 126));  // codes times 2^-126 are zeros
    const int words = D / 2;
    for (int x = member; x < slot * words; x += TW * kWave) {
      gptr at = to + x / words * a.cache.row_stride_b + x % words * 2;
      const uint32_t c0 = gload<uint8_t>(at), c1 = gload<uint8_t>(at + 1);
      const uint32_t c = pack_codes(__builtin_amdgcn_cvt_f32_fp8(c0, 0) * by, __builtin_amdgcn_cvt_f32_fp8(c1, 0) * by, 0, 0);
      gstore<uint8_t>(at, static_cast<uint8_t>(c));
      gstore<uint8_t>(at + 1, static_cast<uint8_t>(c >> 8));
    }
  }
  if (member == 0 && (e > had || slot == 0)) *scale = static_cast<uint8_t>(e + 127);
}

// One launch, two kinds of workgroups: those whose teams of TW waves have a (page,
// head, K or V) each and store its new rows, and those that rotate the queries
// (install_rows). Pages are counted by request; where the bound on a request's new
// tokens leaves more of them than there are tokens, a team goes by a token and
// works if it is its page's first new one.
// A chunk's pages are whole: one wave a page of 64 took 93 us for 2048 tokens, a
// workgroup of four 13.7 and of eight 10.2 to 11.3 (20 MB, 4.2 us at the rate of a copy: the
// rest is one chain of row, largest, barrier, code). A step's pages have one new row,
// which one wave has in one round: 64 requests, heads (64, 8) 6.4 us, launch and the
// same chain without the barrier.
constexpr int kTeamWaves = 8;

template <typename IO, int V, int TW, typename AXES>
__global__ __launch_bounds__((TW > 1 ? TW : kInstallWaves) * kWave) void install_quantized_kernel(InstallQuantizedArgs q, AXES axes) {
  constexpr int W = TW > 1 ? TW : kInstallWaves;
  __shared__ turn_pair<IO> turn[W][kTurns<V>];
  const InstallArgs& a = q.i;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  if (blockIdx.x >= q.page_groups) {
    if (a.batch.err && blockIdx.x == gridDim.x - 1) {  // a workgroup more than there are tokens for
      if (wave == 0) flag_requests(a.batch);
      return;
    }
    install_rows<IO, V, 1, false, true>(a, axes, static_cast<int64_t>(blockIdx.x - q.page_groups) * W + wave, turn[wave]);
    return;
  }
  const int64_t unit = TW > 1 ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * W + wave;
  const int64_t place = unit / (2 * a.kv_heads);
  const int rest = static_cast<int>(unit - place * 2 * a.kv_heads), ps = q.scales.page_size;
  int t;
  Request r;
  if (q.page_slots) {
    const int64_t b = place / q.page_slots;
    if (b >= a.batch.requests) return;
    r = own_request<true>(a.batch, static_cast<int>(b));
    const int p0 = r.length - r.n, page = p0 / ps + static_cast<int>(place - b * q.page_slots);
    t = r.q0 + max(0, page * ps - p0);
    if (!r.ok || t >= r.q0 + r.n) return;
  } else {
    if (place >= a.batch.tokens) return;
    t = static_cast<int>(place);
    if (!request_of_row(a.batch, t, load_fields(a.batch, 0), r) || (t > r.q0 && (r.length - r.n + t - r.q0) % ps != 0)) return;
  }
  if (r.rem != 0) {  // it shares a page with what lies before it
    flag(a.batch.err, CB_ERROR_REQUEST);
    return;
  }
  store_page<IO, V, TW, 2>(q, axes, r, t, rest >> 1, rest & 1, turn[wave]);
}

// ---------------------------------------------------------------------------
// Attention in 16-bit types over codes, head_dim a multiple of 16 up to 256
// (padded with zeros to DP = 64, 128 or 256). Codes become elements of the matrix
// products in registers, K times its scale: e4m3 times a power of two is exact
// in bf16, and in fp16 down to half its least step.
// ---------------------------------------------------------------------------

typedef int i32x2 __attribute__((ext_vector_type(2)));

// 16 codes as 16 elements times `scale` (a power of two).
template <typename IO>
CB_INLINE void widen(u32x4 codes, float scale, u32x4& lo, u32x4& hi) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const int c = static_cast<int>(codes[w]);
    uint32_t x, y;
    if constexpr (std::is_same_v<IO, io_bf16>) {
      x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, scale, false));
      y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, scale, true));
    } else {
      x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, scale, false));
      y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, scale, true));
    }
    if (w < 2) {
      lo[2 * w] = x;
      lo[2 * w + 1] = y;
    } else {
      hi[2 * w - 4] = x;
      hi[2 * w - 3] = y;
    }
  }
}

template <typename IO>
constexpr int kMostRead = std::is_same_v<IO, io_f16> ? kMostExponentF16 : kMostExponent;

// Bits 7 of the bytes that are NaN codes.
__device__ inline uint32_t nan_codes(uint32_t x) { return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// A workgroup's request, the same in all lanes, in scalar registers: what follows
// from it (the tiles, their bounds and waits) is then scalar too.
CB_INLINE int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
CB_INLINE int64_t uniform(int64_t x) {
  return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(uniform(static_cast<int>(x >> 32)))) << 32 | static_cast<uint32_t>(uniform(static_cast<int>(x))));
}
CB_INLINE Request uniform(const Request& r) {
  Request u = r;
  u.q0 = uniform(r.q0);
  u.n = uniform(r.n);
  u.length = uniform(r.length);
  u.first = uniform(r.first);
  u.rem = static_cast<uint32_t>(uniform(static_cast<int>(r.rem)));
  return u;
}

// The launch's arguments (the kernel's first), read when this is called: held from the
// start, those that the end alone needs cost the main loop its scalar registers.
CB_INLINE AttendArgs late_args() {
  auto* from = reinterpret_cast<const CB_CONST uint32_t*>((const CB_CONST void*)__builtin_amdgcn_kernarg_segment_ptr());
  asm volatile("" : "+s"(from));
  struct Raw {
    uint32_t w[sizeof(AttendArgs) / 4];
  } raw;
#pragma unroll
  for (unsigned i = 0; i < sizeof(AttendArgs) / 4; ++i) raw.w[i] = from[i];
  return __builtin_bit_cast(AttendArgs, raw);
}

typedef float f32x8 __attribute__((ext_vector_type(8)));

template <typename IO>
CB_INLINE f32x4 mul16(u32x4 a, u32x4 b, f32x4 c) {
  typedef typename Half<IO>::x8 x8;
  if constexpr (std::is_same_v<IO, io_bf16>)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
}

// Places of an element tile's 16-byte chunks for ElemBlock's reads: K as for RowBlock
// (16 rows of one chunk), V eight keys of two chunks.
__device__ inline int swizzle_v16(int key) { return (key & 7) << 1; }

// 16 query rows of one wave over tiles of KT keys held as elements, with
// v_mfma_f32_16x16x32 (operands: lane l holds elements 8 (l / 16) .. + 7 of row or
// column l % 16; result register e of lane l: row 4 (l / 16) + e, column l % 16).
// S^T = K Q^T leaves a lane keys 16 kb + 4 g + e (g = l / 16) of query row l % 16,
// which for kb = 2 x and 2 x + 1 are the second operand of O^T += V^T P^T in the key
// order {4g .. 4g+3, 16+4g .. 16+4g+3} of block x. Half of RowBlock's rows take half
// of its registers, so that two waves share a SIMD where a head's 256 elements
// leave RowBlock one, and twice its reads a product.
template <typename IO, int DP, int KT, bool MOD>
struct ElemBlock {
  typedef Half<IO> H;
  static constexpr int KB = KT / 32, DB = DP / 16, KS = DP / 32;
  u32x4 q[KS];
  f32x4 o[DB];
  float m, l, slope;
  int i, qh, p;  // this lane's query row
  bool live;

  __device__ inline void init(const ScoreArgs& s, const Request& r, int head, int row0, bool vector) {
    const int lane = threadIdx.x & (kWave - 1), g = lane >> 4;
    const int rows = r.n * s.group, row = row0 + (lane & 15);
    live = row < rows;
    const int at = min(row, rows - 1);
    i = at / s.group;
    qh = head * s.group + at - i * s.group;
    p = r.length - r.n + i;
    const char* qp = s.q.data + static_cast<int64_t>(r.q0 + i) * s.q.token_b + qh * s.q.head_b;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const char* from = qp + 2 * min(32 * k + 8 * g, s.head_dim - 8);
      if (vector) {
        q[k] = gload<u32x4>(as_global(static_cast<const void*>(from)));
      } else {
#pragma unroll
        for (int w = 0; w < 4; ++w)
          q[k][w] = load_elem<uint16_t>(from + 4 * w) | static_cast<uint32_t>(load_elem<uint16_t>(from + 4 * w + 2)) << 16;
      }
    }
#pragma unroll
    for (int k = 0; k < KS; ++k) q[k] = 32 * k + 8 * g < s.head_dim ? q[k] : u32x4{0, 0, 0, 0};
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = f32x4{0, 0, 0, 0};
    m = kNegInf;
    l = slope = 0;
    if constexpr (MOD) slope = s.slopes ? s.slopes[qh] : 0.0f;
  }

  // LDS offsets within a tile that depend on the lane alone.
  struct Lanes {
    uint32_t k[DP == 64 ? 2 : 4];  // K chunk 4 ks + g of row l % 16; ks + 4: 256 bytes on
    uint32_t v[DP == 64 ? 4 : 8];  // V chunks 2 db and 2 db + 1 of this lane's key; db + 8: 256 bytes on
  };
  static __device__ inline Lanes lanes() {
    Lanes a;
    const int lane = threadIdx.x & (kWave - 1), g = lane >> 4, c = lane & 15;
#pragma unroll
    for (int ks = 0; ks < (DP == 64 ? 2 : 4); ++ks) a.k[ks] = c * DP * 2 + ((4 * ks + g) ^ swizzle_k<DP>(c)) * 16;
    const int key = 4 * g + (c >> 2);
#pragma unroll
    for (int d = 0; d < (DP == 64 ? 4 : 8); ++d) a.v[d] = key * DP * 2 + ((2 * d + ((c & 3) >> 1)) ^ place_v(key)) * 16 + (c & 1) * 8;
    return a;
  }
  static __device__ inline int place_v(int key) { return DP == 64 ? ((key >> 1) & 3) << 1 : swizzle_v16(key); }

  static CB_INLINE u32x4 k_frag(const Lanes& a, uint32_t lk, int kb, int ks) {
    return *lds_at<const u32x4>(lk + a.k[ks & 3] + kb * 16 * DP * 2 + (ks >> 2) * 256);
  }
  static CB_INLINE u32x4 v_frag(const Lanes& a, uint32_t lv, int x, int db) {
    const uint32_t at = lv + a.v[db & 7] + x * 32 * DP * 2 + (db >> 3) * 256;
    const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_at<i16x4>(at));
    const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_at<i16x4>(at + 16 * DP * 2));
    const uint2 y = __builtin_bit_cast(uint2, lo), z = __builtin_bit_cast(uint2, hi);
    return u32x4{y.x, y.y, z.x, z.y};
  }

  // Operands are read from LDS a few steps ahead of their use (as in RowBlock).
  static constexpr int kAhead = 4;
  CB_INLINE void products(const Lanes& a, uint32_t lk, f32x8 (&st)[KB]) {
    constexpr int B = KT / 16, STEPS = B * KS;
    u32x4 f[kAhead];
    f32x4 x[B];
#pragma unroll
    for (int n = 0; n < kAhead; ++n) f[n] = k_frag(a, lk, n % B, n / B);
#pragma unroll
    for (int kb = 0; kb < B; ++kb) x[kb] = f32x4{0, 0, 0, 0};
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < STEPS; ++n) {
      x[n % B] = mul16<IO>(f[n % kAhead], q[n / B], x[n % B]);
      if (n + kAhead < STEPS) f[n % kAhead] = k_frag(a, lk, (n + kAhead) % B, (n + kAhead) / B);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 8; ++e) st[kb][e] = x[2 * kb + (e >> 2)][e & 3];
  }

  // Modified and masked, as RowBlock::ready.
  CB_INLINE void ready(const ScoreArgs& s, const KeyRange& kr, f32x8 (&st)[KB], int start, bool whole, const uint32_t* valid) {
    const int g = (threadIdx.x & (kWave - 1)) >> 4;
    if constexpr (MOD) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) modify_scores<true, 8, 16>(s, st[kb], kLog2e, slope, p, start + 32 * kb, g);
    }
    if (!whole) {
      asm volatile("");  // a branch, not selects that every tile would pay for
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const uint32_t there = valid[kb] >> (4 * g);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int k = 16 * (e >> 2) + (e & 3);
          const bool in = sees(s, kr, p, start + 32 * kb + 4 * g + k) & ((there >> k) & 1);
          st[kb][e] = in ? st[kb][e] : kNegInf;
        }
      }
    }
  }

  CB_INLINE float try_weights(const f32x8 (&st)[KB], float scale2, u32x4 (&w)[KB]) const {
    const float mu = m == kNegInf ? 0.0f : m;
    float sum = 0;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float x = exp2_fast(__builtin_fmaf(st[kb][e], scale2, -mu)), y = exp2_fast(__builtin_fmaf(st[kb][e + 1], scale2, -mu));
        sum += x + y;
        w[kb][e >> 1] = H::pack(x, y);
      }
    return sum;
  }
  CB_INLINE void weights(const f32x8 (&st)[KB], float scale2, u32x4 (&w)[KB]) {
    float sum = try_weights(st, scale2, w);
    if (__any(!(sum < H::kLag) | (m == kNegInf))) {
      float top = kNegInf;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, st[kb][e]);
      top = __builtin_fmaf(top, scale2, -H::kRoom);
      top = fmaxf(top, __shfl_xor(top, 16));
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

  struct Values {
    u32x4 f[kAhead];
  };
  static CB_INLINE Values first_values(const Lanes& a, uint32_t lv) {
    Values v;
#pragma unroll
    for (int n = 0; n < kAhead; ++n) v.f[n] = v_frag(a, lv, n / DB, n % DB);
    __builtin_amdgcn_sched_barrier(0);
    return v;
  }
  CB_INLINE void add_values(const Lanes& a, uint32_t lv, const u32x4 (&w)[KB], Values& v) {
    constexpr int STEPS = KB * DB;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < STEPS; ++n) {
      o[n % DB] = mul16<IO>(v.f[n % kAhead], w[n / DB], o[n % DB]);
      if (n + kAhead < STEPS) v.f[n % kAhead] = v_frag(a, lv, (n + kAhead) / DB, (n + kAhead) % DB);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // One wave notes, a bit per (row, element), every NaN of the V tile at lv that its
  // rows see (codes stand for no infinities).
  CB_INLINE void mark_nan(uint32_t lv, const ScoreArgs& s, int np, int start, int end, CB_LDS_SPACE uint32_t* marks) const {
    constexpr int C = DP / 8;
    const int lane = threadIdx.x & (kWave - 1);
    const int below = s.causal ? p : 0x7fffffff, above = s.window > 0 ? p - s.window : -1;
    for (int n = 0; n < KT * C / kWave; ++n) {
      const u32x4 x = *lds_at<const u32x4>(lv + (n * kWave + lane) * 16);
      uint64_t hits = __ballot(has_not_finite<IO>(x));
      while (hits) {
        const int at = __ffsll(static_cast<unsigned long long>(hits)) - 1;
        hits &= hits - 1;
        const int chunk = n * kWave + at, key = chunk / C, d0 = ((chunk % C) ^ place_v(key)) * 8, j = start + key;
        const bool seen = (j < end) & ((j < np) | ((j <= below) & (j > above))) & (lane < 16);
        uint32_t bits = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t y = __shfl(x[w], at), c = ((y & H::kExponent) + H::kCarry) & 0x80008000u;
          bits |= (((c >> 15) & 1) | ((c >> 30) & 2)) << (2 * w);
        }
        if (seen) marks[(lane & 15) * (DP / 32) + (d0 >> 5)] |= bits << (d0 & 31);
      }
    }
  }
  CB_INLINE void add_marks(const uint32_t* marks) {
    const int lane = threadIdx.x & (kWave - 1), g = lane >> 4;
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      const uint32_t bits = marks[(lane & 15) * (DP / 32) + (d >> 1)] >> (16 * (d & 1) + 4 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[d][e] += (bits >> e) & 1 ? __uint_as_float(0x7fc00000u) : 0.0f;
    }
  }

  __device__ inline void finish(const AttendArgs& a, const Request& r, int split, bool vector) {
    const ScoreArgs& s = a.s;
    const int g = (threadIdx.x & (kWave - 1)) >> 4;
    l += __shfl_xor(l, 16);
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
        if (16 * d < s.head_dim) gstore<f32x4>(po + (16 * d + 4 * g) * 4, o[d] * inv);
      if (g == 0) a.part_lse[slot] = lse2;
      return;
    }
    char* op = a.out.data + static_cast<int64_t>(r.q0 + i) * a.out.token_b + qh * a.out.head_b;
#pragma unroll
    for (int d = 0; d < DB; ++d)
      if (16 * d < s.head_dim) {
        char* to = op + (16 * d + 4 * g) * 2;
        const uint2 x = make_uint2(H::pack(o[d][0] * inv, o[d][1] * inv), H::pack(o[d][2] * inv, o[d][3] * inv));
        if (vector) {
          gstore<uint2>(as_global(static_cast<void*>(to)), x);
        } else {
          store_elem<uint16_t>(to, static_cast<uint16_t>(x.x));
          store_elem<uint16_t>(to + 2, static_cast<uint16_t>(x.x >> 16));
          store_elem<uint16_t>(to + 4, static_cast<uint16_t>(x.y));
          store_elem<uint16_t>(to + 6, static_cast<uint16_t>(x.y >> 16));
        }
      }
    if (a.lse && g == 0) a.lse[at] = lse2 * kLn2;
  }
};

// A tile's keys in LDS, by slot t % 4: one wave resolves rows, another fetches scales.
template <int KT>
struct TileCodes {
  uint32_t off[4][KT];  // bytes from the head's first row, or the row itself where a layer has 2^32 or more; 0: no row
  uint32_t at[4][KT];   // place of its scales
  float scale[4][2][KT];
  uint32_t valid[4][(KT + 31) / 32];  // keys that are there
};

// DMA of 16 bytes a lane from base + off.
__device__ inline void dma16_at(gcptr base, uint32_t off, uint32_t lds) {
  const uint32_t la = __builtin_amdgcn_readfirstlane(lds);
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :: "v"(off), "s"(reinterpret_cast<uint64_t>(base)), "s"(la) : "memory", "m0");
}

constexpr int kTileWaves = 8;

// Many query rows: attend_tile_kernel's scheme on tiles that are widened once for
// all of a workgroup's waves. A tile's codes come to LDS by DMA, each wave reads
// the ones it asked for (16 a lane), and writes them as elements to where the
// 16-bit kernel's DMA would have put them; the tile after that is on its way
// while one is used. Keys without a row are read from row 0 and chunks past
// head_dim from the last one, and made zeros when they are widened: a tile that is
// whole pays nothing for either.
// The matrix unit bounds it, as it does the 16-bit kernel: a chunk of 2048 over
// 32768 with heads (16, 2) of 128 takes 540 to 625 us by the card's clock (533
// GFLOP, 440 us at the rate of a library's product; the 16-bit kernel 529 on the
// card where this took 537). Each wave widens an eighth of a tile, so that a tile's
// conversions are shared by 256 rows.
// RB: query rows a wave, 32 (RowBlock) or 16 (ElemBlock): twice the LDS reads a
// product, half the registers. 32 where a wave's registers leave two waves a SIMD
// (the chunk 588 us, 952 with 16). Heads of 256, where 32 rows leave one, and a head's
// few rows take 16: windows of 1024 over 8192 with capped scores 336 us where the
// 16-bit kernel with 32 takes 413.
template <typename IO, int DP, int KT, int RB, bool MOD>
__global__ __launch_bounds__(kTileWaves * kWave, 2) void attend_codes_kernel(AttendArgs a, ScaledCache cache, int vector) {
  typedef std::conditional_t<RB == 32, RowBlock<IO, DP, KT, MOD>, ElemBlock<IO, DP, KT, MOD>> Block;
  constexpr int NW = kTileWaves, C = DP / 16, kTile = KT * DP * 2, kCodes = KT * DP, kHalf = kCodes / 1024, M = 2 * kHalf / NW, N = kTile / 1024 / NW;
  static_assert(M >= 1 && 2 * kHalf % NW == 0 && N >= 1 && kTile % (1024 * NW) == 0, "a tile is whole DMA instructions of every wave");
  __shared__ __align__(1024) char tiles[4 * kTile];  // K, V of one buffer, K, V of the other
  __shared__ __align__(1024) char codes[2 * kCodes];
  __shared__ TileCodes<KT> keys;
  __shared__ uint32_t marks[RB / 16][NW][RB * (DP / 32)];
  __shared__ uint32_t odd[2];  // this tile holds values that are not finite; some tile did
  const ScoreArgs& s = a.s;
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int head = blockIdx.x % s.kv_heads, rest = blockIdx.x / s.kv_heads;
  const int split = rest / a.tile_slots;
  Request r;
  int b, tile;
  if (!find_tile(a, rest % a.tile_slots, RB * NW, r, b, tile)) return;
  r = uniform(r), b = uniform(b), tile = uniform(tile);
  const int rows = r.n * s.group, row0 = tile * RB * NW;
  const KeyRange kr = key_range<KT>(s, r, b, row0, min(rows, row0 + RB * NW) - 1);
  const int per = split_tiles(a, kr.tiles), t0 = split * per, t1 = min(kr.tiles, t0 + per);
  if (a.splits > 1 && t0 >= t1) return;

  Block blk;
  blk.init(s, r, head, row0 + RB * wave, vector);
  const typename Block::Lanes lanes = Block::lanes();
  const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((CB_LDS_SPACE char*)tiles));
  const uint32_t lds_codes = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((CB_LDS_SPACE char*)codes)) + wave * M * 1024;
  const float scale2 = MOD ? 1.0f : s.scale * kLog2e;
  if (threadIdx.x < 2) odd[threadIdx.x] = 0;
  for (int w = threadIdx.x; w < RB / 16 * NW * RB * (DP / 32); w += NW * kWave) (&marks[0][0][0])[w] = 0;
  const HeadScales hs(cache.scales, s.layer, head);
  const uint32_t stride = static_cast<uint32_t>(s.batch.row_stride_b);
  const bool small = static_cast<uint64_t>(s.batch.rows) * stride <= 0xffffffffull;
  auto entry_of = [&](int t) { return t < t1 ? fetch_entry<KT>(s.batch, r, tile_start<KT>(kr, t), tile_end(kr, t)) : -1; };
  auto place = [&](int64_t entry, int t) __attribute__((always_inline)) {
    if (t >= t1) return;
    const int j = tile_start<KT>(kr, t) + lane, end = tile_end(kr, t);
    int64_t row = entry;
    if (s.batch.kind == CB_INDEX_BLOCK_TABLE) {
      const uint32_t x = r.rem + static_cast<uint32_t>(j), ps = static_cast<uint32_t>(s.batch.page_size);
      row = row < 0 ? -1 : row * ps + (s.batch.page_shift >= 0 ? x & (ps - 1) : x % ps);
    }
    const bool ok = (row >= 0) & (row < s.batch.rows) & (lane < KT) & (j < end);
    if (__any(!ok & (j < end) & (lane < KT))) flag(s.batch.err, CB_ERROR_CACHE_ROW);
    const uint32_t at = ok ? static_cast<uint32_t>(row) : 0u;
    if (lane < KT) {
      keys.off[t & 3][lane] = small ? at * stride : at;
      keys.at[t & 3][lane] = hs.at(static_cast<int>(at));
    }
    const uint64_t valid = __ballot(ok);
    if (lane < (KT + 31) / 32) keys.valid[t & 3][lane] = static_cast<uint32_t>(valid >> (32 * lane));
  };
  // The scales of a tile's keys, K's and then V's, 64 a step.
  constexpr int SC = 2 * KT / kWave;
  uint32_t byte[SC];
  auto fetch_scales = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < SC; ++x) {
      const int at = x * kWave + lane, value = at / KT;
      byte[x] = (value ? hs.v : hs.k)[keys.at[t & 3][at % KT]];
    }
  };
  auto keep_scales = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < SC; ++x) (&keys.scale[t & 3][0][0])[x * kWave + lane] = scale_value(byte[x], kMostRead<IO>);
  };
  int64_t entry = -1;
  if (wave == 0) {
    const int64_t e0 = entry_of(t0), e1 = entry_of(t0 + 1), e2 = entry_of(t0 + 2);
    entry = entry_of(t0 + 3);
    place(e0, t0);
    place(e1, t0 + 1);
    place(e2, t0 + 2);
  }
  const int64_t off = static_cast<int64_t>(head) * s.head_dim;
  gcptr kbase = layer_base(s.cache, 0, s.layer) + off, vbase = layer_base(s.cache, 1, s.layer) + off;
  // DMA instruction u of a tile, M a wave: chunk lane % C of key (u % kHalf) * (64 / C) + lane / C, V from kHalf on.
  const int chunk = min(lane % C, s.head_dim / 16 - 1) * 16;
  auto ask = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const int u = wave * M + m, value = u >= kHalf, k = (u - value * kHalf) * (kWave / C) + lane / C;
      const uint32_t at = keys.off[t & 3][k];
      gcptr base = value ? vbase : kbase;
      if (small) dma16_at(base, at + chunk, lds_codes + m * 1024);
      else dma16(base + static_cast<uint64_t>(at) * stride + chunk, lds_codes + m * 1024);
    }
  };
  // This wave's codes of a tile, read before the barrier that the tile's turn begins with.
  u32x4 x[M];
  auto take = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(wait_vm(0));
    asm volatile("" ::: "memory");
#pragma unroll
    for (int m = 0; m < M; ++m) x[m] = *lds_at<const u32x4>(lds_codes + m * 1024 + lane * 16);
  };
  // Asks for the next tile's, then widens the taken ones, of tile t, to the buffer at `to`.
  auto put = [&](uint32_t to, int t) __attribute__((always_inline)) {
    if (t + 1 < t1) ask(t + 1);
    uint32_t every = ~0u;
#pragma unroll
    for (int k = 0; k < KT / 32; ++k) every &= keys.valid[t & 3][k];
    const bool plain = (uniform(static_cast<int>(every)) == -1) & (s.head_dim == DP);
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const int u = wave * M + m, value = u >= kHalf, k = (u - value * kHalf) * (kWave / C) + lane / C;
      if (!plain) {
        const bool there = ((keys.valid[t & 3][k >> 5] >> (k & 31)) & 1) & (lane % C * 16 < s.head_dim);
        x[m] = there ? x[m] : u32x4{0, 0, 0, 0};
      }
      u32x4 lo, hi;
      widen<IO>(x[m], keys.scale[t & 3][value][k], lo, hi);
      // Chunk 2 c of the widened row, and the one after: neighbours, as the swizzles leave the lowest bit or flip it for both.
      int swizzle = swizzle_k<DP>(k);
      if (value) {
        if constexpr (RB == 32) swizzle = swizzle_v<DP>(k);
        else swizzle = Block::place_v(k);
      }
      const uint32_t at = to + value * kTile + k * DP * 2 + ((2 * (lane % C)) ^ swizzle) * 16;
      *lds_at<u32x4>(at) = lo;
      *lds_at<u32x4>(at ^ 16) = hi;
    }
  };
  __syncthreads();
  if (wave == 1 && t0 < t1) {
    fetch_scales(t0);
    keep_scales(t0);
    if (t0 + 1 < t1) {
      fetch_scales(t0 + 1);
      keep_scales(t0 + 1);
    }
  }
  if (t0 < t1) {
    ask(t0);
    take();
  }
  wait_and_meet();
  if (t0 < t1) {
    put(lds, t0);
    if (t0 + 1 < t1) take();
  }
  uint32_t buf = 0;
  for (int t = t0; t < t1; ++t) {
    wait_and_meet();  // tile t is written, and this wave's codes of the next one are taken
    if (t + 1 < t1) put(lds + (buf ^ (2 * kTile)), t + 1);
    if (wave == 0) {
      place(entry, t + 3);
      entry = entry_of(t + 4);
    }
    if (wave == 1 && t + 2 < t1) fetch_scales(t + 2);
    const int start = tile_start<KT>(kr, t), end = tile_end(kr, t);
    uint32_t valid[KT / 32], every = ~0u;
#pragma unroll
    for (int k = 0; k < KT / 32; ++k) every &= valid[k] = keys.valid[t & 3][k];
    const bool all = sees_all(s, kr, start, min(end, start + KT));
    const bool whole = all && __builtin_amdgcn_readfirstlane(every) == ~0u;
    if (!all) {
      const uint32_t lv = lds + buf + kTile + lane * 16;
      const int first = wave * N;
      bool strange = false;
#pragma unroll
      for (int u = 0; u < N; ++u) strange |= has_not_finite<IO>(*lds_at<const u32x4>(lv + (first + u) * 1024));
      if (strange) odd[0] = odd[1] = 1;
      __syncthreads();
      if (odd[0]) {
        if constexpr (RB == 32)
          mark_not_finite<IO, DP, KT>(lds + buf + kTile, kr.np, s.causal ? blk.p : 0x7fffffff, s.window > 0 ? blk.p - s.window : -1,
                                      start, end, (CB_LDS_SPACE uint32_t*)marks[0][wave], (CB_LDS_SPACE uint32_t*)marks[1][wave]);
        else
          blk.mark_nan(lds + buf + kTile, s, kr.np, start, end, (CB_LDS_SPACE uint32_t*)marks[0][wave]);
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
    const uint32_t lk = lds + buf, lv = lk + kTile;
    if constexpr (RB == 32) {
      f32x16 st[KT / 32];
      u32x4 w[KT / 32][2];
      const typename Block::Lanes at = Block::place(lanes, lk, lv);
      blk.products(at, st);
      blk.ready(s, kr, st, start, whole, valid);
      typename Block::Values v = Block::first_values(at);
      blk.weights(st, scale2, w);
      blk.add_values(at, w, v);
    } else {
      f32x8 st[KT / 32];
      u32x4 w[KT / 32];
      blk.products(lanes, lk, st);
      blk.ready(s, kr, st, start, whole, valid);
      typename Block::Values v = Block::first_values(lanes, lv);
      blk.weights(st, scale2, w);
      blk.add_values(lanes, lv, w, v);
    }
    if (wave == 1 && t + 2 < t1) keep_scales(t + 2);
    if (t + 2 < t1) take();
    buf ^= 2 * kTile;
  }
  __syncthreads();
  if (odd[1]) {
    if constexpr (RB == 32) blk.add_marks(marks[0][wave], marks[1][wave]);
    else blk.add_marks(marks[0][wave]);
  }
  blk.finish(late_args(), r, split, vector);
}

// Places of 16-byte chunks within a row of codes in LDS, exchanged so that the
// lanes of a read hit distinct banks (K: one chunk of 16 rows; V: one of keys 0 to
// 7 and 16 to 23, or 8 to 15 and 24 to 31).
template <int DP>
__device__ inline int swizzle_code_k(int key) {
  return DP == 64 ? (key >> 2) & 3 : DP == 128 ? (key >> 1) & 7 : key & 15;
}
template <int DP>
__device__ inline int swizzle_code_v(int key) {
  return DP == 64    ? ((key >> 2) & 1) | ((key >> 3) & 2)
         : DP == 128 ? ((key >> 1) & 3) | ((key >> 2) & 4)
                     : (key & 7) | ((key >> 1) & 8);
}

// NB times 16 query rows of one wave over tiles of 32 keys held as codes, with
// v_mfma_f32_16x16x32 (operands: lane l holds elements 8 (l / 16) .. + 7 of row or
// column l % 16; result register e of lane l: row 4 (l / 16) + e, column l % 16). 16
// rows, not the 32 of RowBlock: a step has the query heads of one KV head, mostly 8
// or less, and what a row costs is paid for empty ones too. S^T = K Q^T leaves a
// lane keys 16 kb + 4 g + e (g = l / 16) of query row l % 16, which are the second
// operand of O^T += V^T P^T in the key order {4g .. 4g+3, 16+4g .. 16+4g+3}; V^T is
// read in that order by transposing LDS reads.
// K is widened with its scales, V without them: a value's scale goes into its
// weight, since a lane's codes of V are of eight keys. Weights times scales would
// leave fp16's range, so they are two bf16 terms for either type, 16 bits of each:
// a step of bf16 rows is then as near 64 bits as fp32 weights are (1.7e-3 of the
// result, its own rounding, where one term leaves 2.3e-3), for 0 to 5% of its time
// (64 requests of 8192 62 against 65 us).
template <typename IO, int DP, int NB, bool MOD>
struct CodeBlock {
  typedef Half<IO> H;
  static constexpr int DB = DP / 16, JS = DP / 64;  // result rows a column block; pairs of product steps
  u32x4 q[NB][2 * JS];
  f32x4 o[NB][DB];
  float m[NB], l[NB], slope[NB];
  int p[NB];  // cached token of this lane's query rows
  bool live[NB];

  __device__ inline void init(const ScoreArgs& s, const Request& r, int head, int row0, bool vector) {
    const int lane = threadIdx.x & (kWave - 1), g = lane >> 4;
    const int rows = r.n * s.group;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int row = row0 + 16 * n + (lane & 15);
      live[n] = row < rows;
      const int at = min(row, rows - 1), i = at / s.group, qh = head * s.group + at - i * s.group;
      p[n] = r.length - r.n + i;
      const char* qp = s.q.data + static_cast<int64_t>(r.q0 + i) * s.q.token_b + qh * s.q.head_b;
      // Elements 64 j + 16 g + 8 x .. + 7: those of a lane's 16 codes of K.
#pragma unroll
      for (int k = 0; k < 2 * JS; ++k) {
        const char* from = qp + 2 * min(64 * (k >> 1) + 16 * g + 8 * (k & 1), s.head_dim - 8);
        if (vector) {
          q[n][k] = gload<u32x4>(as_global(static_cast<const void*>(from)));
        } else {
#pragma unroll
          for (int w = 0; w < 4; ++w)
            q[n][k][w] = load_elem<uint16_t>(from + 4 * w) | static_cast<uint32_t>(load_elem<uint16_t>(from + 4 * w + 2)) << 16;
        }
      }
#pragma unroll
      for (int k = 0; k < 2 * JS; ++k) q[n][k] = 64 * (k >> 1) + 16 * g < s.head_dim ? q[n][k] : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int d = 0; d < DB; ++d) o[n][d] = f32x4{0, 0, 0, 0};
      m[n] = kNegInf;
      l[n] = slope[n] = 0;
      if constexpr (MOD) slope[n] = s.slopes ? s.slopes[qh] : 0.0f;
    }
  }

  // LDS offsets within a tile that depend on the lane alone.
  struct Lanes {
    uint32_t k[JS];  // K chunk 4 j + g of row l % 16
    uint32_t v[DB];  // V chunk db, this lane's half of it, of this lane's key
  };
  static __device__ inline Lanes lanes() {
    Lanes a;
    const int lane = threadIdx.x & (kWave - 1), g = lane >> 4, c = lane & 15;
#pragma unroll
    for (int j = 0; j < JS; ++j) a.k[j] = c * DP + ((4 * j + g) ^ swizzle_code_k<DP>(c)) * 16;
    const int i = c >> 1, key = 4 * g + (i & 3) + 4 * (i & 4);
#pragma unroll
    for (int d = 0; d < DB; ++d) a.v[d] = key * DP + (d ^ swizzle_code_v<DP>(key)) * 16 + (c & 1) * 8;
    return a;
  }

  // Raw products with the tile at lk; ks: the scales of keys l % 16 and 16 + l % 16.
  CB_INLINE void products(const Lanes& a, uint32_t lk, const float (&ks)[2], f32x8 (&st)[NB]) {
    f32x4 x[NB][2];
    u32x4 f[2][JS];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int j = 0; j < JS; ++j) f[kb][j] = *lds_at<const u32x4>(lk + a.k[j] + kb * 16 * DP);
#pragma unroll
    for (int n = 0; n < NB; ++n) x[n][0] = x[n][1] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < JS; ++j)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        u32x4 lo, hi;
        widen<IO>(f[kb][j], ks[kb], lo, hi);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          x[n][kb] = mul16<IO>(lo, q[n][2 * j], x[n][kb]);
          x[n][kb] = mul16<IO>(hi, q[n][2 * j + 1], x[n][kb]);
        }
      }
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int e = 0; e < 8; ++e) st[n][e] = x[n][e >> 2][e & 3];
  }

  // Modified and masked, as RowBlock::ready.
  CB_INLINE void ready(const ScoreArgs& s, const KeyRange& kr, f32x8 (&st)[NB], int start, bool whole, uint32_t valid) {
    const int g = (threadIdx.x & (kWave - 1)) >> 4;
    if constexpr (MOD) {
#pragma unroll
      for (int n = 0; n < NB; ++n) modify_scores<true, 8, 16>(s, st[n], kLog2e, slope[n], p[n], start, g);
    }
    if (!whole) {
      asm volatile("");  // a branch, not selects that every tile would pay for
      const uint32_t there = valid >> (4 * g);
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int k = 16 * (e >> 2) + (e & 3);
          const bool in = sees(s, kr, p[n], start + 4 * g + k) & ((there >> k) & 1);
          st[n][e] = in ? st[n][e] : kNegInf;
        }
    }
  }

  // As RowBlock's, but a weight is packed times its value's scale.
  CB_INLINE float try_weights(int n, const f32x8& st, float scale2, const f32x4 (&vs)[2], u32x4& w, u32x4& rest) const {
    const float mu = m[n] == kNegInf ? 0.0f : m[n];
    float sum = 0;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float x = exp2_fast(__builtin_fmaf(st[e], scale2, -mu)), y = exp2_fast(__builtin_fmaf(st[e + 1], scale2, -mu));
      sum += x + y;
      const float xs = x * vs[e >> 2][e & 3], ys = y * vs[e >> 2][(e & 3) + 1];
      const uint32_t hi = pack_bf16(xs, ys);
      w[e >> 1] = hi;
      rest[e >> 1] = pack_bf16(xs - lo_bf(hi), ys - hi_bf(hi));
    }
    return sum;
  }
  CB_INLINE void weights(const f32x8 (&st)[NB], float scale2, const f32x4 (&vs)[2], u32x4 (&w)[NB], u32x4 (&rest)[NB]) {
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      float sum = try_weights(n, st[n], scale2, vs, w[n], rest[n]);
      if (__any(!(sum < H::kLag) | (m[n] == kNegInf))) {
        float top = kNegInf;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, st[n][e]);
        top = __builtin_fmaf(top, scale2, -H::kRoom);
        top = fmaxf(top, __shfl_xor(top, 16));
        const float m1 = fmaxf(m[n], fmaxf(top, __shfl_xor(top, 32)));
        const float alpha = m1 == kNegInf ? 1.0f : exp2_fast(m[n] - m1);
        m[n] = m1;
        l[n] *= alpha;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[n][d] *= alpha;
        sum = try_weights(n, st[n], scale2, vs, w[n], rest[n]);
      }
      l[n] += sum;
    }
  }

  CB_INLINE void add_values(const Lanes& a, uint32_t lv, const u32x4 (&w)[NB], const u32x4 (&rest)[NB]) {
    i32x2 f[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) f[d] = __builtin_amdgcn_ds_read_tr8_b64_v2i32(lds_at<i32x2>(lv + a.v[d]));
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      u32x4 x;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        x[2 * k] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f[d][k], 1.0f, false));
        x[2 * k + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f[d][k], 1.0f, true));
      }
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        o[n][d] = mul16<io_bf16>(x, w[n], o[n][d]);
        o[n][d] = mul16<io_bf16>(x, rest[n], o[n][d]);
      }
    }
  }

  // NaN for the elements whose NaN values were taken out of the tiles.
  CB_INLINE void add_marks(const uint32_t* marks) {
    const int lane = threadIdx.x & (kWave - 1), g = lane >> 4;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const uint32_t bits = marks[(16 * n + (lane & 15)) * (DP / 32) + (d >> 1)] >> (16 * (d & 1) + 4 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][d][e] += (bits >> e) & 1 ? __uint_as_float(0x7fc00000u) : 0.0f;
      }
  }

  // The wave's sums into LDS, for join_sums.
  template <int NW>
  CB_INLINE void put_sums(float* sums, float (&stats)[2][NW][16 * NB], int wave) {
    constexpr int LD = DP + 4;
    const int lane = threadIdx.x & (kWave - 1), g = lane >> 4, c = lane & 15;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      l[n] += __shfl_xor(l[n], 16);
      l[n] += __shfl_xor(l[n], 32);
      if (live[n]) {
#pragma unroll
        for (int d = 0; d < DB; ++d) *reinterpret_cast<f32x4*>(sums + (16 * n + c) * LD + 16 * d + 4 * g) = o[n][d];
      }
      if (g == 0) {
        stats[0][wave][16 * n + c] = m[n];
        stats[1][wave][16 * n + c] = l[n];
      }
    }
  }
};

// One wave notes, for its rows, every NaN of the V tile of codes at lv that a row
// sees, and takes it out of the tile: a weight of zero times it would be NaN in rows
// that do not see it. Lane l notes for row l % 16 of column block l / 16.
template <int DP, int NB>
CB_INLINE void take_nan_out(uint32_t lv, int np, const int (&p)[NB], int window, int causal, int start, int end, CB_LDS_SPACE uint32_t* marks) {
  constexpr int C = DP / 16;
  const int lane = threadIdx.x & (kWave - 1), n = (lane >> 4) & 1;
  const int first = p[0], last = p[NB - 1], mine = n ? last : first;
  const int below = causal ? mine : 0x7fffffff, above = window > 0 ? mine - window : -1;
  for (int i = 0; i < 32 * C / kWave; ++i) {
    CB_LDS_SPACE u32x4* at = lds_at<u32x4>(lv + (i * kWave + lane) * 16);
    u32x4 x = *at;
    uint64_t hits = __ballot((nan_codes(x[0]) | nan_codes(x[1]) | nan_codes(x[2]) | nan_codes(x[3])) != 0);
    if (!hits) continue;
    while (hits) {
      const int who = __ffsll(static_cast<unsigned long long>(hits)) - 1;
      hits &= hits - 1;
      const int chunk = i * kWave + who, key = chunk / C, d0 = ((chunk % C) ^ swizzle_code_v<DP>(key)) * 16, j = start + key;
      const bool seen = (j < end) & ((j < np) | ((j <= below) & (j > above))) & (lane < 16 * NB);
      uint32_t bits = 0;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t nan = nan_codes(__shfl(x[w], who)) >> 7;
        bits |= ((nan & 1) | ((nan >> 7) & 2) | ((nan >> 14) & 4) | ((nan >> 21) & 8)) << (4 * w);
      }
      if (seen) marks[(lane & (16 * NB - 1)) * (DP / 32) + (d0 >> 5)] |= bits << (d0 & 31);
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) x[w] &= ~((nan_codes(x[w]) >> 7) * 0xffu);
    *at = x;
  }
}

// Waits for the K (else V) rows of the first of the last `left` tiles, X to S of
// them, N instructions each for K and for V.
template <int X, int S, int N>
CB_INLINE void wait_last(int left, bool value) {
  if (left == X) {
    if (value) __builtin_amdgcn_s_waitcnt(wait_vm(2 * (X - 1) * N));
    else __builtin_amdgcn_s_waitcnt(wait_vm((2 * X - 1) * N));
  } else if constexpr (X < S) {
    wait_last<X + 1, S, N>(left, value);
  }
}

// Few query rows: attend_step_kernel's scheme on tiles of codes. Each wave
// streams tiles of 32 keys through LDS of its own, S of them in flight.
// Reading K and V bounds it: 64 requests of 8192 with 268 MB take 56 to 66 us by
// card (4.1 to 4.8 TB/s, the rate of a copy). Shorter steps add 8 to 10 us for the
// chain of lookups before the first product and the sums after the last: 64
// ragged requests of 2550 28.9 us (17.7 at that rate), one of 32768 with 8 KV heads
// 19.3 (14.1).
// Two blocks of rows (17 to 32) of 128 elements hold 85,000 bytes of LDS, so one
// workgroup has the CU, one wave a SIMD and half as many bytes in flight: calls of 64
// requests of 2048 with heads (16, 2) take 29.5, 34.3, 65.7 and 72.9 us for one to four
// new tokens (8 to 32 rows), where a 16-bit pool takes 43.5, 48.8, 54.9 and 59.4.
// kCodeWaves 4, S 2: two waves take 33.7, 22.9 and 74.8 us for these three cases'
// 29.3, 19.4 and 62; blocks of 32 rows, with the LDS that they take, 42, 26.7 and 81.
// Splits cut for 512 or 2048 workgroups in place of 1024 are slower, for 256 the same
// within noise.
constexpr int kCodeTiles = 32;  // tiles a split holds at most
constexpr int kCodeWaves = 4;
// Weights times scales, and their low terms, have to stay normal in bf16, and their
// sums finite: weights reach 2^15 (H::kLag), codes 2^9, a split 2^10 keys. Scales
// of V beyond 2^+-80 are taken relative to the split's largest, which becomes 2^80,
// and the result is set right at its end: powers of two change no digit of what is
// within 2^190 of the largest. Looking for such scales takes 0.2 us of a step's 19.3.
constexpr int kFarScale = 80;

template <typename IO, int DP, int NB, bool MOD>
__global__ __launch_bounds__(kCodeWaves * kWave, DP == 256 ? 1 : 2) void step_codes_kernel(AttendArgs a, ScaledCache cache, int vector) {
  constexpr int NW = kCodeWaves, KT = 32, kTile = KT * DP, N = kTile / 1024, C = DP / 16, S = 2;
  constexpr int kSums = (16 * NB * (DP + 4) * 4 + 1023) / 1024 * 1024, kWaveBytes = 2 * S * kTile > kSums ? 2 * S * kTile : kSums;
  __shared__ __align__(1024) char tiles[NW * kWaveBytes];  // a wave's K tiles, then its V tiles; at the end its sums
  __shared__ int key_rows[kCodeTiles * KT];
  __shared__ __align__(16) float key_scales[2][kCodeTiles * KT];
  __shared__ uint32_t marks[NW][16 * NB * (DP / 32)];
  __shared__ float stats[2][NW][16 * NB];
  __shared__ int far_scale, top_scale;  // some scale of V is beyond 2^+-kFarScale; then the largest, a float's bits
  const ScoreArgs& s = a.s;
  const QBatch& B = s.batch;
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int head = blockIdx.x % s.kv_heads, rest = blockIdx.x / s.kv_heads;
  const int split = rest / a.tile_slots;
  Request r;
  int b, tile;
  if (!find_tile<true>(a, rest % a.tile_slots, 16 * NB, r, b, tile)) return;
  r = uniform(r), b = uniform(b), tile = uniform(tile);
  const int rows = r.n * s.group, row0 = tile * 16 * NB;
  const KeyRange kr = key_range<KT>(s, r, b, row0, min(rows, row0 + 16 * NB) - 1);
  const int per = min(split_tiles(a, kr.tiles), kCodeTiles), t0 = split * per, t1 = min(kr.tiles, t0 + per);
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
  if (threadIdx.x == 0) far_scale = top_scale = 0;
  for (int w = threadIdx.x; w < NW * NB * DP / 2; w += NW * kWave) (&marks[0][0])[w] = 0;
  typedef CodeBlock<IO, DP, NB, MOD> Block;
  Block blk;
  blk.init(s, r, head, row0, vector);
  const typename Block::Lanes lanes = Block::lanes();
  const float scale2 = MOD ? 1.0f : s.scale * kLog2e;
  const int64_t off = static_cast<int64_t>(head) * s.head_dim;
  gcptr kbase = layer_base(s.cache, 0, s.layer) + off, vbase = layer_base(s.cache, 1, s.layer) + off;
  gcptr zero = as_global(static_cast<const void*>(g_zeros));
  const uint32_t stride = static_cast<uint32_t>(B.row_stride_b);
  const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((CB_LDS_SPACE char*)tiles)) + wave * kWaveBytes;
  wait_and_meet();

  const int n = t1 - t0 > wave ? (t1 - t0 - wave + NW - 1) / NW : 0;  // this wave's tiles: t0 + wave, + NW, ...
  auto request = [&](int i, gcptr base, uint32_t to, bool value) __attribute__((always_inline)) {
    const int at = (wave + i * NW) * KT;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int k = u * (kWave / C) + lane / C;
      const int row = key_rows[at + k];
      const int c = (lane % C) ^ (value ? swizzle_code_v<DP>(k) : swizzle_code_k<DP>(k));
      gcptr from = ((row >= 0) & (c * 16 < s.head_dim)) ? base + static_cast<uint64_t>(static_cast<uint32_t>(row)) * stride + c * 16 : zero;
      dma16(from, to + u * 1024);
    }
  };
  // Waits until the K (else V) rows of the first of `left` tiles are there.
  auto arrived = [&](int left, bool value) __attribute__((always_inline)) {
    // In order of asking: K and V of S tiles; V is waited for with the K of a tile S on behind it, if there is one.
    if (!value ? left >= S : left > S) __builtin_amdgcn_s_waitcnt(wait_vm((2 * S - 1) * N));
    else wait_last<1, S, N>(left, value);
    asm volatile("" ::: "memory");
  };
  bool some_mark = false;
#pragma unroll 1
  for (int i = 0; i < S; ++i)
    if (i < n) {
      asm volatile("");
      request(i, kbase, lds + i * kTile, false);
      request(i, vbase, lds + (S + i) * kTile, true);
    }
  // The scales of keys, one without a row has no matter which.
  const HeadScales hs(cache.scales, s.layer, head);
  for (int k = threadIdx.x; k < (t1 - t0) * KT; k += NW * kWave) {
    const int row = key_rows[k];
    const uint32_t at = hs.at(max(row, 0)), value = hs.v[at];
    key_scales[0][k] = scale_value(hs.k[at], kMostRead<IO>);
    key_scales[1][k] = scale_value(value);
    if ((row >= 0) & (value - (127 - kFarScale) > 2u * kFarScale)) far_scale = 1;
  }
  __builtin_amdgcn_s_waitcnt(0xc07f);
  asm volatile("s_barrier" ::: "memory");
  auto scaled_down = [&]() { return uniform(far_scale) ? (uniform(top_scale) >> 23) - 127 - kFarScale : 0; };
  if (uniform(far_scale)) {
    auto each = [&](auto f) __attribute__((always_inline)) {
      for (int k = threadIdx.x; k < (t1 - t0) * KT; k += NW * kWave)
        if (key_rows[k] >= 0) f(key_scales[1][k]);
      __syncthreads();
    };
    each([&](float x) { atomicMax(&top_scale, __float_as_int(x)); });
    const int down = scaled_down();
    each([&](float& x) { x = __builtin_amdgcn_ldexpf(x, -down); });
  }
  uint32_t buf = 0;
  for (int i = 0; i < n; ++i) {
    const int t = t0 + wave + i * NW, start = tile_start<KT>(kr, t), end = tile_end(kr, t), at = (t - t0) * KT;
    const uint32_t valid = static_cast<uint32_t>(__ballot(key_rows[at + (lane & 31)] >= 0));
    float ks[2];
    f32x4 vs[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      ks[kb] = key_scales[0][at + 16 * kb + (lane & 15)];
      vs[kb] = *reinterpret_cast<const f32x4*>(&key_scales[1][at + 16 * kb + 4 * (lane >> 4)]);
    }
    arrived(n - i, false);
    f32x8 st[NB];
    u32x4 w[NB], low[NB];
    const uint32_t lk = lds + buf, lv = lk + S * kTile;
    blk.products(lanes, lk, ks, st);
    if (i + S < n) {
      __builtin_amdgcn_s_waitcnt(0xc07f);  // the products' LDS reads
      request(i + S, kbase, lk, false);
    }
    const bool all = sees_all(s, kr, start, min(end, start + KT));
    blk.ready(s, kr, st, start, all & (valid == ~0u), valid);
    blk.weights(st, scale2, vs, w, low);
    arrived(n - i, true);
    if (!all) {
      bool strange = false;
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const u32x4 x = *lds_at<const u32x4>(lv + u * 1024 + lane * 16);
        strange |= (nan_codes(x[0]) | nan_codes(x[1]) | nan_codes(x[2]) | nan_codes(x[3])) != 0;
      }
      if (__any(strange)) {
        some_mark = true;
        take_nan_out<DP, NB>(lv, kr.np, blk.p, s.window, s.causal, start, end, (CB_LDS_SPACE uint32_t*)marks[wave]);
      }
    }
    blk.add_values(lanes, lv, w, low);
    if (i + S < n) {
      __builtin_amdgcn_s_waitcnt(0xc07f);
      request(i + S, vbase, lv, true);
    }
    buf = buf + kTile == S * kTile ? 0 : buf + kTile;
  }
  if (some_mark) blk.add_marks(marks[wave]);
  blk.put_sums(reinterpret_cast<float*>(tiles + wave * kWaveBytes), stats, wave);
  __syncthreads();
  join_sums<DP, NW, 16 * NB, Half<IO>>(late_args(), r, head, row0, rows, split, vector, tiles, kWaveBytes, stats, scaled_down());
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
  if (scales->page_stride > 0xffffffffll / std::max<int64_t>(1, scales->pages)) return fail(CB_EINVAL, "a layer's scales above 2^32 bytes");
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

// Whether the kernels of 16-bit products take the call: whole 16-byte chunks of rows.
bool takes_codes(const ScoreArgs& s, int32_t dtype, const cb_scores& scores) {
  return !scores.fp32_weights && dtype != CB_DTYPE_F32 && s.head_dim <= kMaxDp && s.cache.row_stride_b <= 0xffffffffll &&
         rows_aligned16(s.cache, s.head_dim);
}

// Key tiles of 64 that a split has at least: 37 tokens over 4133 take 25.5, 19.8 and 17.6
// us with 8, 4 and 2 (the join 5.8, 5.8 and 6.1); with 1 the call takes 30.8 for 23.2.
constexpr int kCodeLeast = 2;

// attend_shape's waves are the 16-bit tile kernel's. Here a workgroup always has
// kTileWaves; they say which rows a wave has (8: 32, 4: 16), and launches of 16 rows a
// wave are cut for 512 workgroups, two a CU, where one has the CU.
AttendShape quantized_shape(const ScoreArgs& s, int32_t dtype, const cb_scores& scores) {
  AttendShape h = attend_shape(s, takes_codes(s, dtype, scores), kCodeLeast, kCodeTiles);
  // One block of rows a request: how many blocks there are does not change with its size.
  if (h.step && static_cast<int64_t>(s.batch.max_query) * s.group <= 16) h.rows_per_tile = 16;
  return h;
}

template <typename IO, int DP, int KT, bool MOD>
void launch_codes(const AttendArgs& a, const ScaledCache& cache, const AttendShape& h, unsigned grid, hipStream_t st) {
  const int vector = aligned16(a.s.q) && aligned16(a.out);
  if (h.step && h.rows_per_tile == 16) hipLaunchKernelGGL((step_codes_kernel<IO, DP, 1, MOD>), dim3(grid), dim3(kCodeWaves * kWave), 0, st, a, cache, vector);
  else if (h.step) hipLaunchKernelGGL((step_codes_kernel<IO, DP, 2, MOD>), dim3(grid), dim3(kCodeWaves * kWave), 0, st, a, cache, vector);
  else if (DP <= 128 && h.rows_per_tile == 32 * kTileWaves) hipLaunchKernelGGL((attend_codes_kernel<IO, DP, KT, DP <= 128 ? 32 : 16, MOD>), dim3(grid), dim3(kTileWaves * kWave), 0, st, a, cache, vector);
  else hipLaunchKernelGGL((attend_codes_kernel<IO, DP, KT, 16, MOD>), dim3(grid), dim3(kTileWaves * kWave), 0, st, a, cache, vector);
  if (h.step) launch_join<IO, 32>(a, h, st);
  else launch_join<IO, KT>(a, h, st);
}

template <typename IO>
void launch_quantized(const AttendArgs& a, const ScaledCache& cache, const AttendShape& h, unsigned grid, hipStream_t st) {
  const int d = a.s.head_dim;
  if constexpr (sizeof(IO) == 2) {
    if (h.half) {
      if (a.s.mod) {
        if (d <= 64) launch_codes<IO, 64, 64, true>(a, cache, h, grid, st);
        else if (d <= 128) launch_codes<IO, 128, 32, true>(a, cache, h, grid, st);
        else launch_codes<IO, 256, 32, true>(a, cache, h, grid, st);
      } else {
        if (d <= 64) launch_codes<IO, 64, 64, false>(a, cache, h, grid, st);
        else if (d <= 128) launch_codes<IO, 128, 64, false>(a, cache, h, grid, st);
        else launch_codes<IO, 256, 32, false>(a, cache, h, grid, st);
      }
      return;
    }
  }
  if (d <= 64) launch_any<IO, 64>(a, cache, grid, st);
  else if (d <= 128) launch_any<IO, 128>(a, cache, grid, st);
  else if (d <= 256) launch_any<IO, 256>(a, cache, grid, st);
  else launch_any<IO, 512>(a, cache, grid, st);
  launch_join<IO, kAnyKeys>(a, h, st);
}

template <typename IO, typename AXES>
void launch_store(const InstallQuantizedArgs& q, const AXES& axes, bool wide, bool teams, unsigned grid, hipStream_t st) {
  constexpr int V = 16 / sizeof(IO);
  const dim3 groups(grid), team(kTeamWaves * kWave), waves(kInstallWaves * kWave);
  if (wide && teams) hipLaunchKernelGGL((install_quantized_kernel<IO, V, kTeamWaves, AXES>), groups, team, 0, st, q, axes);
  else if (wide) hipLaunchKernelGGL((install_quantized_kernel<IO, V, 1, AXES>), groups, waves, 0, st, q, axes);
  else if (teams) hipLaunchKernelGGL((install_quantized_kernel<IO, 1, kTeamWaves, AXES>), groups, team, 0, st, q, axes);
  else hipLaunchKernelGGL((install_quantized_kernel<IO, 1, 1, AXES>), groups, waves, 0, st, q, axes);
}
template <typename AXES>
void launch_store_of(int32_t dtype, const InstallQuantizedArgs& q, const AXES& axes, bool wide, bool teams, unsigned grid, hipStream_t st) {
  if (dtype == CB_DTYPE_BF16) launch_store<io_bf16>(q, axes, wide, teams, grid, st);
  else if (dtype == CB_DTYPE_F16) launch_store<io_f16>(q, axes, wide, teams, grid, st);
  else launch_store<float>(q, axes, wide, teams, grid, st);
}

template <typename IO>
void launch_quantize(const QuantizeArgs& a, int vec, dim3 grid, hipStream_t st) {
  const int chunks = ceil_div(static_cast<int64_t>(a.scales.page_size) * a.head_dim, 16 * kWave);
  if (vec == 16 && chunks <= 2) hipLaunchKernelGGL((quantize_tokens_kernel<IO, 16, 2>), grid, dim3(256), 0, st, a);
  else if (vec == 16 && chunks > 4) hipLaunchKernelGGL((quantize_tokens_kernel<IO, 16, 8>), grid, dim3(256), 0, st, a);
  else if (vec == 16) hipLaunchKernelGGL((quantize_tokens_kernel<IO, 16, 4>), grid, dim3(256), 0, st, a);
  else if (vec == 8) hipLaunchKernelGGL((quantize_tokens_kernel<IO, 8, 4>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((quantize_tokens_kernel<IO, 2, 4>), grid, dim3(256), 0, st, a);
}

}  // namespace

extern "C" {

int cb_install_quantized(const cb_query_batch* batch, const cb_page_scales* scales, int32_t layer, int32_t dtype,
                         int32_t head_dim, const cb_heads* q, const cb_heads* q_out, const cb_heads* k, const cb_heads* v,
                         const cb_rotation* rotation, int32_t* d_error_flag, void* stream) {
  InstallQuantizedArgs a{};
  PairAxes axes{};
  bool many;
  int rc;
  if ((rc = check_batch(batch, dtype, head_dim, d_error_flag, true, &a.i.batch, &a.i.cache, 1)) ||
      (rc = check_scales(scales, *batch, &a.scales)) || (rc = check_pages(*batch, a.scales, "the batch")) ||
      (rc = check_install(batch, layer, dtype, head_dim, q, q_out, k, v, rotation, &a.i, &axes, &many)))
    return rc;
  const int eb = elem_bytes(dtype), n = batch->num_tokens, rotary_dim = a.i.rotary_dim;
  if (n == 0 || batch->num_requests == 0) return CB_OK;
  const int vec = 16 / eb;
  const bool wide = (rotary_dim / 2) % vec == 0 && head_dim % vec == 0 && aligned16(a.i.q) && aligned16(a.i.q_out) &&
                    aligned16(a.i.k) && aligned16(a.i.v) && rows_aligned16(a.i.cache, 16) && head_dim % 8 == 0;
  const InstallItems each = install_items(head_dim, rotary_dim, wide ? vec : 1);
  a.i.slices = std::max(1, std::min(64, ceil_div(a.i.q_heads * each.head, kWave)));
  a.most = most_exponent(dtype);
  // Pages of a request that max_query tokens may be in, wherever they begin; the whole workgroup has one where a
  // wave would go round more than twice.
  const int64_t ps = a.scales.page_size, most = batch->max_query;
  const int64_t slots = most < 1 ? 0 : (most + ps - 2) / ps + 1;
  a.page_slots = slots * batch->num_requests <= n ? static_cast<int32_t>(slots) : 0;
  const int64_t places = a.page_slots ? slots * batch->num_requests : n;
  const bool teams = std::min(ps, most) * std::max(each.head, each.value) > 2 * kWave;
  const int waves = teams ? kTeamWaves : kInstallWaves;
  const int64_t units = places * 2 * a.i.kv_heads, pages = teams ? units : (units + waves - 1) / waves;
  const int64_t grid = pages + (static_cast<int64_t>(n) * a.i.slices + waves - 1) / waves + (d_error_flag ? 1 : 0);
  if (!launch_fits(grid, waves * kWave)) return fail(CB_EINVAL, "too many tokens");
  a.page_groups = static_cast<uint32_t>(pages);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (many) launch_store_of(dtype, a, axes, wide, teams, static_cast<unsigned>(grid), st);
  else launch_store_of(dtype, a, OneAxis{}, wide, teams, static_cast<unsigned>(grid), st);
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
  *bytes = s.batch.tokens && s.batch.requests ? attend_workspace(s, quantized_shape(s, dtype, *scores)) : 0;
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
  const AttendShape h = quantized_shape(a.s, dtype, *scores);
  unsigned grid;
  if ((rc = cut_attention(a, h, (h.step ? kCodeWaves : h.half ? kTileWaves : kAnyWaves) * kWave, lse, d_workspace, workspace_bytes, &grid))) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == CB_DTYPE_BF16) launch_quantized<io_bf16>(a, cache, h, grid, st);
  else if (dtype == CB_DTYPE_F16) launch_quantized<io_f16>(a, cache, h, grid, st);
  else launch_quantized<float>(a, cache, h, grid, st);
  CB_HIP(hipGetLastError());
  return CB_OK;
}

}  // extern "C"
