// Rotation of new tokens and the store of their rows, for the kernels that do it.
#pragma once

#include "cb_query_common.h"

namespace {

// ---------------------------------------------------------------------------
// New tokens: rotation and store
// ---------------------------------------------------------------------------

constexpr int kInstallWaves = 4;
constexpr int kMaxPairs = 256;  // head_dim <= 512
constexpr int kMaxAxes = 8;

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

// Positions of one axis, or of several: rows of them, `stride` entries apart, and the
// axis of each pair. The latter are 256 bytes of a launch's arguments, which a step of
// 64 requests pays with 0.3 of its 5 us, so launches without axes go without.
struct OneAxis {
  CB_INLINE int64_t at(int, int t) const { return t; }
};
struct PairAxes {
  int64_t stride;
  uint8_t axis[kMaxPairs];
  CB_INLINE int64_t at(int pair, int t) const { return axis[pair] * stride + t; }
};


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

// Items of two vectors of V elements in a head of q or k, of these the turned ones
// first, and in a head of v.
struct InstallItems {
  int head, turned, value;
};
__host__ __device__ inline InstallItems install_items(int head_dim, int rotary_dim, int v) {
  const int turned = rotary_dim / 2 / v;
  return {turned + ((head_dim - rotary_dim) / v + 1) / 2, turned, (head_dim / v + 1) / 2};
}

// x / y, y the same in all lanes and mostly a power of two.
CB_INLINE int divide(int x, int y) { return (y & (y - 1)) == 0 ? x >> __builtin_ctz(y) : x / y; }

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

// What the rotation of IO rows is computed in: fp32 rows are rotated in fp64 and
// rounded once, since in fp32 the cosine, sine and two products would each round
// to the digits that are stored (2048 tokens of 16 and 2 heads of 128 13.9 us for
// 13.6).
template <typename IO>
using turn_t = std::conditional_t<sizeof(IO) == 4, double, float>;

template <typename IO>
using turn_pair = turn_t<IO> __attribute__((ext_vector_type(2)));

// What the angle of pair `i` of token row t is made of (the position where there is
// a row of them), and its cosine and sine, times the magnitude, at place p.
struct Angle {
  int64_t position;
  double inv_freq;
};
template <typename AXES>
CB_INLINE Angle load_angle(const InstallArgs& a, const AXES& axes, int t, int i) {
  Angle x{0, a.inv_freq[i]};
  if (a.positions) {
    const int64_t at = axes.at(i, t);
    x.position = a.positions_kind == CB_INDEX_I64 ? static_cast<const int64_t*>(a.positions)[at]
                                                  : static_cast<const int32_t*>(a.positions)[at];
  }
  return x;
}
template <typename PAIR, typename T>
CB_INLINE PAIR turn_of(const InstallArgs& a, int p, const Angle& x) {
  T s, c;
  sincos_turns(static_cast<double>(a.positions ? x.position : p) * x.inv_freq * 0.15915494309189533577, &s, &c);
  return PAIR{c * a.magnitude, s * a.magnitude};
}

// V pairs x (2 V elements: both vectors of the pairs, or neighbours) turned. Which
// of the two products a sum takes in unrounded is said, not left to the compiler:
// a token's bits are the same in all the kernels that turn it. In place: with a
// second array an install has 83 registers for 69 and 5 waves a SIMD for 7 (2048
// tokens of heads (16, 2) of 128 10.3 us for 9.1).
CB_INLINE float multiply_add(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
CB_INLINE double multiply_add(float a, double b, double c) { return __builtin_fma(static_cast<double>(a), b, c); }

template <int V, typename PAIR>
CB_INLINE void turn_pairs(float (&x)[2 * V], const PAIR* turn, bool interleaved) {
  auto pair = [&](int i, float& a, float& b) __attribute__((always_inline)) {
    const PAIR cs = turn[i];
    const float p = static_cast<float>(multiply_add(a, cs.x, -(b * cs.y)));
    b = static_cast<float>(multiply_add(b, cs.x, a * cs.y));
    a = p;
  };
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < V; ++i) pair(i, x[2 * i], x[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) pair(i, x[i], x[i + V]);
  }
}

// y_a = x_a cos - x_b sin, y_b = x_b cos + x_a sin for the pairs (a, b) of the
// rotated part, angles position * inv_freq. One wave per (token, slice of its
// heads' elements): lanes compute the token's angles once into LDS, then each
// item is two vectors of a head: those of V pairs, or two that are copied; slices
// are cut to U items a lane, so that a wave waits for memory once. Every element
// is read once and written once.
// KV: K and V rows go into the cache as they are, else queries alone are written.
// WHOLE: requests that do not start at a page's first slot are outside the bounds.
// What a wave reads of q, k and v depends on its token row alone: the loads are on
// their way while the row's request, place and cache row are looked up, which is
// one load of the batch's fields by all lanes and one index entry. What is left of a
// step is launch and that chain: 64 requests, heads (64, 8) of 128 4.9 us for 2.6 MB,
// 2048 tokens of (16, 2) 9.1 (21 MB).
// Above 8192 waves a lane takes two items, so that half as many waves look their
// row up: 2048 tokens of (16, 2) heads of 256 with three axes 15.2 us for 20.3 (38
// MB, 8.8 us at the rate of a copy; sines and cosines are 1 us of it).
template <typename IO, int V, int U, bool KV, bool WHOLE, typename AXES>
CB_INLINE void install_rows(const InstallArgs& a, const AXES& axes, int64_t unit, turn_pair<IO>* turn) {
  const int lane = threadIdx.x & (kWave - 1);
  const int t = static_cast<int>(unit / a.slices), slice = static_cast<int>(unit % a.slices);
  if (t >= a.batch.tokens) return;
  const Fields fields = load_fields(a.batch, 0);
  const int pairs = a.rotary_dim / 2, kv_heads = KV ? a.kv_heads : 0;
  const InstallItems n = install_items(a.head_dim, a.rotary_dim, V);
  const int turned = (a.q_heads + kv_heads) * n.head, total = turned + kv_heads * n.value;
  const int per = (total + a.slices - 1) / a.slices;
  const int stop = min(total, (slice + 1) * per);
  constexpr int E = sizeof(IO);
  struct Item {
    int64_t to;         // where its head's elements go, from q_out, or from the cache row of K or V
    int oa, ob, first;  // the two vectors; the first pair, or -1
    int kind;           // 0: q, 1: K, 2: V
    bool on, two;
  } item[U];
  float x[U][2 * V];
  auto load = [&](int idx) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      Item& m = item[u];
      const int at = min(idx + u * kWave, stop - 1);
      m.on = idx + u * kWave < stop;
      const char* src;
      int k;
      if (!KV || at < turned) {
        const int head = divide(at, n.head);
        k = at - head * n.head;
        m.kind = KV && head >= a.q_heads;
        if (m.kind) {
          src = a.k.data + t * a.k.token_b + (head - a.q_heads) * a.k.head_b;
          m.to = static_cast<int64_t>(head - a.q_heads) * a.head_dim * E;
        } else {
          src = a.q.data + t * a.q.token_b + head * a.q.head_b;
          m.to = t * a.q_out.token_b + head * a.q_out.head_b;
        }
        m.first = k < n.turned ? k * V : -1;
        m.oa = m.first < 0 ? a.rotary_dim + 2 * (k - n.turned) * V : a.interleaved ? 2 * m.first : m.first;
      } else {
        const int head = divide(at - turned, n.value);
        k = at - turned - head * n.value;
        m.kind = 2;
        src = a.v.data + t * a.v.token_b + head * a.v.head_b;
        m.to = static_cast<int64_t>(head) * a.head_dim * E;
        m.first = -1;
        m.oa = 2 * k * V;
      }
      m.ob = m.first < 0 || a.interleaved ? m.oa + V : m.first + pairs;
      m.two = m.first >= 0 || m.ob < a.head_dim;
      if (m.on) {
        load_vec<IO, V>(src + m.oa * E, x[u]);
        if (m.two) load_vec<IO, V>(src + m.ob * E, x[u] + V);
      }
    }
  };
  const int first = slice * per + lane;
  const Angle angle = load_angle(a, axes, t, min(lane, pairs - 1));
  if (first < stop) load(first);
  Request r;
  if (!request_of_row(a.batch, t, fields, r) || (WHOLE & (r.rem != 0))) return;
  const int p = r.length - r.n + (t - r.q0);
  int64_t row = -1;
  if constexpr (KV) {
    row = cache_row(a.batch, r, p);
    if (row < 0 && lane == 0) flag(a.batch.err, CB_ERROR_TARGET_ROW);
  }
  for (int i = lane; i < pairs; i += kWave) turn[i] = turn_of<turn_pair<IO>, turn_t<IO>>(a, p, i == lane ? angle : load_angle(a, axes, t, i));
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  char* krow = const_cast<char*>((const char*)layer_base(a.cache, 0, a.layer)) + row * a.cache.row_stride_b;
  char* vrow = const_cast<char*>((const char*)layer_base(a.cache, 1, a.layer)) + row * a.cache.row_stride_b;
  for (int idx = first; idx < stop; idx += U * kWave) {
    if (idx != first) load(idx);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Item& m = item[u];
      if (!m.on || (m.kind && row < 0)) continue;
      char* dst = (m.kind == 0 ? a.q_out.data : m.kind == 1 ? krow : vrow) + m.to;
      if (m.first >= 0) turn_pairs<V>(x[u], turn + m.first, a.interleaved);
      store_vec<IO, V>(dst + m.oa * E, x[u]);
      if (m.two) store_vec<IO, V>(dst + m.ob * E, x[u] + V);
    }
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

// The token tensors and the rotation of an install, checked; the batch and the
// cache are the caller's. many: pairs turn by positions of several axes.
int check_install(const cb_query_batch* batch, int32_t layer, int32_t dtype, int32_t head_dim, const cb_heads* q,
                  const cb_heads* q_out, const cb_heads* k, const cb_heads* v, const cb_rotation* rotation, InstallArgs* a,
                  PairAxes* axes, bool* many) {
  int rc;
  if (layer < 0 || layer >= batch->cache.num_layers) return fail(CB_EINVAL, "layer %d outside the cache", layer);
  if (!q) return fail(CB_EINVAL, "null q");
  const int eb = elem_bytes(dtype), kv = batch->cache.heads, n = batch->num_tokens;
  if (q->heads < 1 || q->heads > (1 << 16)) return fail(CB_EINVAL, "q needs 1 to 65536 heads");
  if ((rc = check_heads("q", q, q->heads, eb, n, &a->q)) || (rc = check_output("q_out", q_out, q->heads, eb, n, head_dim, &a->q_out)) ||
      (rc = check_heads("k", k, kv, eb, n, &a->k)) || (rc = check_heads("v", v, kv, eb, n, &a->v)))
    return rc;
  if (!rotation) return fail(CB_EINVAL, "null rotation");
  const cb_rotation& o = *rotation;
  if (o.rotary_dim < 2 || o.rotary_dim > head_dim || o.rotary_dim % 2)
    return fail(CB_EINVAL, "rotary_dim must be even, 2 to head_dim");
  if (!o.inv_freq) return fail(CB_EINVAL, "null inv_freq");
  if (!std::isfinite(o.magnitude)) return fail(CB_EINVAL, "magnitude must be finite");
  if (o.positions && o.positions_kind != CB_INDEX_I32 && o.positions_kind != CB_INDEX_I64)
    return fail(CB_EINVAL, "positions must be int32 or int64");
  *many = o.pair_axis && o.positions && o.axes > 1;
  if (o.pair_axis) {
    if (o.axes < 1 || o.axes > kMaxAxes) return fail(CB_EINVAL, "a rotation has 1 to %d axes", kMaxAxes);
    if (o.positions && o.axis_stride < n) return fail(CB_EINVAL, "axes of positions are shorter than num_tokens");
    for (int i = 0; i < o.rotary_dim / 2; ++i) {
      if (o.pair_axis[i] >= o.axes) return fail(CB_EINVAL, "pair %d turns by axis %d of %d", i, o.pair_axis[i], o.axes);
      axes->axis[i] = o.pair_axis[i];
    }
    axes->stride = o.axis_stride;
  }
  if (shares_rows(*batch)) return fail(CB_EINVAL, "several requests need offsets or a request_stride");
  a->layer = layer;
  a->head_dim = head_dim;
  a->rotary_dim = o.rotary_dim;
  a->interleaved = o.interleaved != 0;
  a->q_heads = q->heads;
  a->kv_heads = kv;
  a->inv_freq = o.inv_freq;
  a->positions = o.positions;
  a->positions_kind = o.positions_kind;
  a->magnitude = o.magnitude;
  return CB_OK;
}

}  // namespace
