// Attention of new tokens over cached ones: scores, masks, tiles of rows and
// keys, the general kernel, joins of split keys and the row blocks of the matrix
// kernels.
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

#pragma once

#include "cb_query_common.h"

namespace {

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
// `start`, register e: key 8 (e / 4) + 4 h + e % 4; or N keys, STEP (e / 4) + 4 h
// + e % 4) to scores times `unit`.
// Capped: where no lane's angle reaches kSmallAngle, which is the rule, the
// polynomial (READY: by factors made ahead, four registers, seven instructions,
// else nine). A block of 32 rows and keys with larger ones takes tanh y = 1 - 2 /
// (exp(2y) + 1), two transcendental operations that hold for either sign: it is
// off by 3 2^-23 of the cap, so by less than 2^-20 of the block's largest score,
// where the products' own sums are off by more. 8192 tokens with 16 heads of 128 take
// 419 us with blocks of the first kind and 428 with all of the second; with a
// selection by element the latter took 599, with the second form alone both 414.
template <bool READY, int N = 16, int STEP = 8, typename VEC = f32x16>
CB_INLINE void modify_scores(const ScoreArgs& s, VEC& x, float unit, float slope, int p, int start, int h) {
  const float by = s.scale * unit;
  if (s.cap > 0) {
    float far = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) far = fmaxf(far, fabsf(x[e]));
    if (__all(far < s.gentle)) {
      const float k3 = kTanh3 * by, k5 = kTanh5 * by, k7 = kTanh7 * by, k9 = kTanh9 * by;
#pragma unroll
      for (int e = 0; e < N; ++e) {
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
      for (int e = 0; e < N; ++e) x[e] = __builtin_fmaf(-2.0f * out, __builtin_amdgcn_rcpf(exp2_fast(x[e] * in) + 1.0f), out);
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] *= by;
  }
  if (s.slopes) {
    const float by = slope * unit, away = static_cast<float>(p - start - 4 * h);
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = __builtin_fmaf(-by, fabsf(away - static_cast<float>(STEP * (e >> 2) + (e & 3))), x[e]);
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

// CACHE: how the cache holds its elements, and what a row's are multiplied by.
template <typename IO>
struct PlainCache {
  typedef IO elem;
  static constexpr bool kScaled = false;
  CB_INLINE float scale(int, int, int64_t, int) const { return 1.0f; }
  static __device__ inline float value(IO x) { return static_cast<float>(x); }
};

template <typename IO, typename CACHE, int DP, int VE>
__global__ __launch_bounds__(kAnyWaves * kWave, DP == 64 ? 3 : DP == 128 ? 2 : 1) void attend_any_kernel(AttendArgs a, CACHE cache) {
  typedef typename CACHE::elem KV;
  constexpr int KT = kAnyKeys, LD = DP + 4, NB = DP / 16, NT = kAnyWaves * kWave, MW = DP / 32;
  // A 512-element row's sums and queries fill the registers: no tile waits there.
  constexpr bool AHEAD = DP <= 256;
  constexpr int NC = AHEAD ? (KT * DP / VE + NT - 1) / NT : 1;
  typedef KV vec __attribute__((ext_vector_type(VE)));
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

  gcptr kbase = layer_base(s.cache, 0, s.layer) + static_cast<int64_t>(head) * D * sizeof(KV);
  gcptr vbase = layer_base(s.cache, 1, s.layer) + static_cast<int64_t>(head) * D * sizeof(KV);
  const int per_row = D / VE;
  int key_of[NC], elem_of[NC];  // this thread's chunks of a tile
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int x = n * NT + threadIdx.x;
    key_of[n] = x / per_row;
    elem_of[n] = (x - key_of[n] * per_row) * VE;
  }
  vec rk[NC], rv[NC];
  float ks[NC], vs[NC];
  auto load = [&](int t) __attribute__((always_inline)) {
    if constexpr (!AHEAD) return;
    const uint32_t valid = tile_rows.valid[t & 3][0];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const bool in = (key_of[n] < KT) && ((valid >> key_of[n]) & 1);
      rk[n] = rv[n] = vec(static_cast<KV>(0));
      if constexpr (CACHE::kScaled) ks[n] = vs[n] = 1.0f;
      if (in) {
        const int at = tile_rows.row[t & 3][key_of[n]];
        if constexpr (CACHE::kScaled) {
          ks[n] = cache.scale(0, s.layer, at, head);
          vs[n] = cache.scale(1, s.layer, at, head);
        }
        const int64_t off = static_cast<int64_t>(at) * s.batch.row_stride_b + elem_of[n] * static_cast<int>(sizeof(KV));
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
        const int at = tile_rows.row[t & 3][k];
        const int64_t off = static_cast<int64_t>(at) * s.batch.row_stride_b;
        float kscale = 1.0f, vscale = 1.0f;
        if constexpr (CACHE::kScaled) {
          if (in) {
            kscale = cache.scale(0, s.layer, at, head);
            vscale = cache.scale(1, s.layer, at, head);
          }
        }
#pragma unroll 2
        for (int d = lane; d < D; d += kWave) {
          lk[k * LD + d] = in ? CACHE::value(gload<KV>(kbase + off + d * static_cast<int>(sizeof(KV)))) * kscale : 0.0f;
          lv[k * LD + d] = in ? CACHE::value(gload<KV>(vbase + off + d * static_cast<int>(sizeof(KV)))) * vscale : 0.0f;
        }
      }
      return;
    }
#pragma unroll
    for (int n = 0; n < NC; ++n)
      if (key_of[n] < KT) {
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float x = CACHE::value(rk[n][e]), y = CACHE::value(rv[n][e]);
          lk[key_of[n] * LD + elem_of[n] + e] = CACHE::kScaled ? x * ks[n] : x;
          lv[key_of[n] * LD + elem_of[n] + e] = CACHE::kScaled ? y * vs[n] : y;
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
// 4096 it takes 4.9 us where a workgroup a row takes 9.5, with 64 times 16
// tokens 13.3 against 45.7, with 1000 rows of 64 4.2 against 5.4; with 4 tokens (64
// rows of 16 splits) 5.2 against 4.2. Between them (37 tokens, 592 rows of 8 splits:
// 4.3 against 5.0) calls keep the order of sums that they have had.
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
  // U splits from z0 on: all their loads before any is used, past the last one the last again.
  auto add = [&](auto ahead, int z0) __attribute__((always_inline)) {
    constexpr int U = decltype(ahead)::value;
    float x[U][E];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float* from = a.part_out + (min(z0 + u, n - 1) * step + at) * D + d0;
      if (D % E == 0) {
        const vec y = *reinterpret_cast<const vec*>(from);
#pragma unroll
        for (int e = 0; e < E; ++e) x[u][e] = y[e];
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) x[u][e] = from[min(e, D - 1 - d0)];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // Read from lanes that may hold no element and are off here. A weight of zero takes nothing, NaN included.
      const float f = z0 + u < n ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), z0 + u)) : 0.0f;
      if (f == 0.0f) continue;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] += f * x[u][e];
    }
  };
  if (d0 < D) {
    if (n <= 2) {
      for (int z = 0; z < n; ++z) add(std::integral_constant<int, 1>{}, z);
    } else {
      for (int z = 0; z < n; z += 4) add(std::integral_constant<int, 4>{}, z);
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
// LDS in group order. Splits that are in flight together (eight a group where there
// are many) are what it waits for: a request of 32768 tokens with 64 heads 5.4 us
// (9.0 with splits in turn).
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
  // U splits of this group's from z0 on, as in join_few_kernel.
  auto add = [&](auto ahead, int z0) __attribute__((always_inline)) {
    constexpr int U = decltype(ahead)::value;
    f32x4 part[U];
    float w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int z = min(z0 + u * GROUPS, n - 1);
      w[u] = lse[z * step];
      const float* from = a.part_out + (z * step + at) * D;
      if (vector) {
        part[u] = *reinterpret_cast<const f32x4*>(from + min(4 * x, D - 4));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) part[u][e] = from[min(4 * x + e, D - 1)];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      w[u] = z0 + u * GROUPS < n ? exp2_fast(w[u] - mu) : 0.0f;
      o += w[u] == 0.0f ? f32x4{0, 0, 0, 0} : w[u] * part[u];
    }
  };
  if (n <= 2 * GROUPS) {
    for (int z = g; z < n; z += GROUPS) add(std::integral_constant<int, 1>{}, z);
  } else {
    for (int z = g; z < n; z += 8 * GROUPS) add(std::integral_constant<int, 8>{}, z);
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

// Sums of NW waves that lie in LDS, each wave's of its own keys (ROWS rows of DP + 4
// floats, `stride` bytes a wave, with their maxima and totals in stats), become the
// rows of the result or of a part. up: the power of two that sums lack.
template <int DP, int NW, int ROWS, typename H>
CB_INLINE void join_sums(const AttendArgs& a, const Request& r, int head, int row0, int rows, int split, int vector, const char* sums,
                         int stride, const float (&stats)[2][NW][ROWS], int up = 0) {
  constexpr int LD = DP + 4;
  const ScoreArgs& s = a.s;
  const int D = s.head_dim, live = min(ROWS, rows - row0), pairs = D / 2;
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
      const float* from = reinterpret_cast<const float*>(sums + w * stride) + y * LD + d;
      l += f * stats[1][w][y];
      // A wave that saw nothing of this row has nothing to add.
      o0 += f != 0.0f ? f * from[0] : 0.0f;
      o1 += f != 0.0f ? f * from[1] : 0.0f;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const float lse2 = l == 0.0f ? kNegInf : m + log2_fast(l);
    o0 = __builtin_amdgcn_ldexpf(o0 * inv, up);
    o1 = __builtin_amdgcn_ldexpf(o1 * inv, up);
    const int row = row0 + y, i = row / s.group, qh = head * s.group + row - i * s.group;
    const int64_t at = static_cast<int64_t>(r.q0 + i) * s.q_heads + qh;
    if (a.splits > 1) {
      const int64_t slot = static_cast<int64_t>(split) * s.batch.tokens * s.q_heads + at;
      *reinterpret_cast<float2*>(a.part_out + slot * D + d) = make_float2(o0, o1);
      if (d == 0) a.part_lse[slot] = lse2;
    } else {
      char* op = a.out.data + static_cast<int64_t>(r.q0 + i) * a.out.token_b + qh * a.out.head_b + d * 2;
      const uint32_t packed = H::pack(o0, o1);
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

// The sums of a workgroup's NW waves, each of its own keys, meet in LDS (each
// wave's in `stride` bytes of its own).
template <int DP, int NW, typename BLOCK>
CB_INLINE void join_waves(BLOCK& blk, const AttendArgs& a, const Request& r, int head, int row0, int rows, int split, int vector,
                          char* sums, int stride, float (&stats)[2][NW][32]) {
  constexpr int LD = DP + 4;
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  blk.l += __shfl_xor(blk.l, 32);
  const int c = lane & 31, h = lane >> 5;
  float* mine = reinterpret_cast<float*>(sums + wave * stride) + c * LD;
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
  join_sums<DP, NW, 32, typename BLOCK::H>(a, r, head, row0, rows, split, vector, sums, stride, stats);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

int check_scores(const cb_query_batch* batch, int32_t layer, int32_t dtype, int32_t head_dim, const cb_scores* sc,
                 int32_t q_heads, int32_t* err, ScoreArgs* s, int cache_bytes = 0) {
  int rc;
  if ((rc = check_batch(batch, dtype, head_dim, err, true, &s->batch, &s->cache, cache_bytes))) return rc;
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

constexpr int kStepTiles = 64;  // tiles a split holds at most

// Workgroups of four waves that a launch is split into at least: two a CU. 512 new
// tokens over 32768 take 262, 173 and 185 us with 256, 512 and 1024, 64 requests of
// 8 new tokens over 2048 47, 38.5 and 39 us.
constexpr int kTargetGroups = 512;

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

// half: the kernels of 16-bit products take the call.
// half_tiles: key tiles that a split of theirs has at least.
AttendShape attend_shape(const ScoreArgs& s, bool half, int half_tiles = 8, int step_tiles = kStepTiles) {
  AttendShape h{};
  h.half = half;
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
  h.least_tiles = h.half ? half_tiles : 2;
  h.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(target / std::max<int64_t>(1, groups), key_tiles / h.least_tiles)));
  if (h.step) {
    // Parts of one size for all requests, cut by the bound: their workgroups end
    // together (64 ragged requests 47 us, with parts by each one's own keys 68).
    h.splits = std::max(h.splits, ceil_div(key_tiles, step_tiles));
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

// What the workspace and the workgroups of a launch are: fills them in, refuses a
// workspace that is too small and launches past HIP's limits.
int cut_attention(AttendArgs& a, const AttendShape& h, int threads, float* lse, void* d_workspace, int64_t workspace_bytes,
                  unsigned* groups) {
  const int64_t need = attend_workspace(a.s, h);
  if (need > 0 && (!d_workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(d_workspace) % 256))
    return fail(CB_EINVAL, "attention needs a 256-byte aligned workspace of %lld bytes", static_cast<long long>(need));
  a.lse = lse;
  a.request_slots = h.request_slots;
  a.splits = h.splits;
  a.least_tiles = h.least_tiles;
  a.by_splits = h.splits > 1 && !h.step ? static_cast<uint32_t>(((int64_t{1} << 32) + h.splits - 1) / h.splits) : 0;
  const int64_t rows = static_cast<int64_t>(a.s.batch.tokens) * a.s.q_heads;
  if (need > 0) {
    a.part_out = static_cast<float*>(d_workspace);
    a.part_lse = reinterpret_cast<float*>(static_cast<char*>(d_workspace) + round256(h.splits * rows * a.s.head_dim * 4));
  }
  const int64_t grid = h.tile_slots * h.splits * a.s.kv_heads;
  if (!launch_fits(grid, threads) || rows > 0x7fffffff ||
      (h.splits > 1 && !joins_by_wave(h.splits, rows) && !launch_fits(rows, kJoinThreads)))
    return fail(CB_EINVAL, "too many query tiles");
  a.tile_slots = static_cast<int32_t>(h.tile_slots);
  *groups = static_cast<unsigned>(grid);
  return CB_OK;
}

template <typename IO, int DP, typename CACHE>
void launch_any(const AttendArgs& a, const CACHE& cache, unsigned grid, hipStream_t st) {
  constexpr int VE = 16 / sizeof(typename CACHE::elem);
  if constexpr (DP == 512) hipLaunchKernelGGL((attend_any_kernel<IO, CACHE, DP, 1>), dim3(grid), dim3(kAnyWaves * kWave), 0, st, a, cache);
  else if (a.s.head_dim % VE == 0 && rows_aligned16(a.s.cache, a.s.head_dim * static_cast<int>(sizeof(typename CACHE::elem))))
    hipLaunchKernelGGL((attend_any_kernel<IO, CACHE, DP, VE>), dim3(grid), dim3(kAnyWaves * kWave), 0, st, a, cache);
  else
    hipLaunchKernelGGL((attend_any_kernel<IO, CACHE, DP, 1>), dim3(grid), dim3(kAnyWaves * kWave), 0, st, a, cache);
}

}  // namespace
