// Queries on an installed prefix for MI355X (gfx950): new tokens rotated and
// stored into a paged cache, attention over it, the attention each cached
// token got, and eviction by it. The C ABI is in include/cachebridge_hip.h.

#include "cb_attend.h"
#include "cb_rotate.h"

namespace {

template <typename IO, int V, int U, typename AXES>
__global__ __launch_bounds__(kInstallWaves * kWave) void install_tokens_kernel(InstallArgs a, AXES axes) {
  __shared__ turn_pair<IO> turn[kInstallWaves][kMaxPairs];
  const int wave = threadIdx.x / kWave;
  if (a.batch.err && blockIdx.x == gridDim.x - 1) {  // a workgroup more than there are tokens for
    if (wave == 0) flag_requests(a.batch);
    return;
  }
  install_rows<IO, V, U, true, false>(a, axes, static_cast<int64_t>(blockIdx.x) * kInstallWaves + wave, turn[wave]);
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
template <typename IO, int DP, int NW, bool MOD>
__global__ __launch_bounds__(NW * kWave, 1) void attend_step_kernel(AttendArgs a, int vector) {
  constexpr int KT = 32, kTile = KT * DP * 2, N = kTile / 1024, C = DP / 8;
  static_assert(4 * kTile >= 32 * (DP + 4) * 4, "a wave's sums fit its tiles");
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

  join_waves<DP, NW>(blk, a, r, head, row0, rows, split, vector, tiles, 4 * kTile, stats);
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

// Whether the 16-bit kernels take the call: whole 16-byte chunks of rows.
bool takes_half(const ScoreArgs& s, int32_t dtype) {
  return dtype != CB_DTYPE_F32 && s.head_dim % 8 == 0 && s.cache.row_stride_b <= 0xffffffffll && s.head_dim <= kMaxDp && rows_aligned16(s.cache, s.head_dim * 2);
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
  if (d <= 64) launch_any<IO, 64>(a, PlainCache<IO>{}, grid, st);
  else if (d <= 128) launch_any<IO, 128>(a, PlainCache<IO>{}, grid, st);
  else if (d <= 256) launch_any<IO, 256>(a, PlainCache<IO>{}, grid, st);
  else launch_any<IO, 512>(a, PlainCache<IO>{}, grid, st);
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

constexpr int kManyWaves = 8192;  // of an install, from which a lane has two items

template <typename IO, typename AXES>
void launch_install(const InstallArgs& a, const AXES& axes, bool wide, int items, unsigned grid, hipStream_t st) {
  const dim3 groups(grid), threads(kInstallWaves * kWave);
  if (wide && items == 2) hipLaunchKernelGGL((install_tokens_kernel<IO, 16 / sizeof(IO), 2, AXES>), groups, threads, 0, st, a, axes);
  else if (wide) hipLaunchKernelGGL((install_tokens_kernel<IO, 16 / sizeof(IO), 1, AXES>), groups, threads, 0, st, a, axes);
  else hipLaunchKernelGGL((install_tokens_kernel<IO, 1, 1, AXES>), groups, threads, 0, st, a, axes);
}
template <typename AXES>
void launch_install_of(int32_t dtype, const InstallArgs& a, const AXES& axes, bool wide, int items, unsigned grid, hipStream_t st) {
  if (dtype == CB_DTYPE_BF16) launch_install<io_bf16>(a, axes, wide, items, grid, st);
  else if (dtype == CB_DTYPE_F16) launch_install<io_f16>(a, axes, wide, items, grid, st);
  else launch_install<float>(a, axes, wide, items, grid, st);
}

}  // namespace

extern "C" {

int cb_install_tokens(const cb_query_batch* batch, int32_t layer, int32_t dtype, int32_t head_dim, const cb_heads* q,
                      const cb_heads* q_out, const cb_heads* k, const cb_heads* v, const double* inv_freq,
                      int32_t rotary_dim, int32_t interleaved, float magnitude, const void* positions,
                      int32_t positions_kind, int32_t* d_error_flag, void* stream) {
  const cb_rotation rotation = {inv_freq, positions, nullptr, 0, rotary_dim, interleaved, positions_kind, 1, magnitude, 0};
  return cb_install_rotated(batch, layer, dtype, head_dim, q, q_out, k, v, &rotation, d_error_flag, stream);
}

int cb_install_rotated(const cb_query_batch* batch, int32_t layer, int32_t dtype, int32_t head_dim, const cb_heads* q,
                       const cb_heads* q_out, const cb_heads* k, const cb_heads* v, const cb_rotation* rotation,
                       int32_t* d_error_flag, void* stream) {
  InstallArgs a{};
  PairAxes axes{};
  bool many;
  int rc;
  if ((rc = check_batch(batch, dtype, head_dim, d_error_flag, true, &a.batch, &a.cache)) ||
      (rc = check_install(batch, layer, dtype, head_dim, q, q_out, k, v, rotation, &a, &axes, &many)))
    return rc;
  const int eb = elem_bytes(dtype), kv = a.kv_heads, n = batch->num_tokens, rotary_dim = a.rotary_dim;
  if (n == 0 || batch->num_requests == 0) return CB_OK;
  const int vec = 16 / eb;
  const bool wide = (rotary_dim / 2) % vec == 0 && head_dim % vec == 0 && aligned16(a.q) && aligned16(a.q_out) &&
                    aligned16(a.k) && aligned16(a.v) && rows_aligned16(a.cache, head_dim * eb);
  const InstallItems each = install_items(head_dim, rotary_dim, wide ? vec : 1);
  const int total = (a.q_heads + kv) * each.head + kv * each.value;
  // An item a lane: one round of memory latency; two where there are waves enough to fill the card.
  const int items = wide && static_cast<int64_t>(n) * ceil_div(total, kWave) >= kManyWaves ? 2 : 1;
  a.slices = std::max(1, std::min(64, ceil_div(total, items * kWave)));
  const int64_t grid = (static_cast<int64_t>(n) * a.slices + kInstallWaves - 1) / kInstallWaves + (d_error_flag ? 1 : 0);
  if (!launch_fits(grid, kInstallWaves * kWave)) return fail(CB_EINVAL, "too many tokens");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (many) launch_install_of(dtype, a, axes, wide, items, static_cast<unsigned>(grid), st);
  else launch_install_of(dtype, a, OneAxis{}, wide, items, static_cast<unsigned>(grid), st);
  CB_HIP(hipGetLastError());
  return CB_OK;
}

int cb_attention_workspace_bytes(const cb_query_batch* batch, int32_t dtype, int32_t head_dim, const cb_scores* scores,
                                 int32_t query_heads, int64_t* bytes) {
  if (!bytes) return fail(CB_EINVAL, "null bytes");
  ScoreArgs s{};
  int rc;
  if ((rc = check_scores(batch, 0, dtype, head_dim, scores, query_heads, nullptr, &s))) return rc;
  *bytes = s.batch.tokens && s.batch.requests ? attend_workspace(s, attend_shape(s, !scores->fp32_weights && takes_half(s, dtype))) : 0;
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
  const AttendShape h = attend_shape(a.s, !scores->fp32_weights && takes_half(a.s, dtype));
  unsigned grid;
  if ((rc = cut_attention(a, h, (h.step ? kStepWaves : h.waves) * kWave, lse, d_workspace, workspace_bytes, &grid))) return rc;
  const bool mod = a.s.mod;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == CB_DTYPE_BF16) launch_attend<io_bf16>(a, h, mod, grid, st);
  else if (dtype == CB_DTYPE_F16) launch_attend<io_f16>(a, h, mod, grid, st);
  else launch_attend<float>(a, h, mod, grid, st);
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
