// Attention backward with the probabilities computed again: P = exp(scale q k^T - lse),
//
//   D = rowsum(dout * out),  dV = P^T dout,  dP = dout V^T,  dS = P (dP - D),
//   dQ = scale dS K,  dK = scale dS^T Q, over all query heads that share the key head.
//
// Two kernels, each of which owns what it sums, so that no gradient is added up by atomics and the
// order of every sum is fixed: attention_bwd_keys holds dK and dV of 128 keys (32 a wave) in registers
// and walks over the queries of every head of the group; attention_bwd_queries holds dQ of 128 queries
// and walks over the keys.  Seven products instead of the five of a joint pass, without a
// read-modify-write of dQ in memory for every block of keys.
//
// As in the forward pass the scores' registers are the next product's operand: with a lane's
// column a key (bwd_keys: S = Q K^T) P and dS are operands of dV^T = dO^T P and dK^T = Q^T dS; with its
// column a query (bwd_queries: S^T = K Q^T) dS^T is the operand of dQ^T = K^T dS^T.  The other operand of
// these is a column of the tile in LDS (the transposing read).
//
// bwd_queries runs first and leaves each query's D in the workspace for bwd_keys.  Where blocks are too few for the
// compute units, both take ranges of what they walk over and leave float32 sums to be joined.
//
// 16-bit types: probabilities and dS are rounded to the type before their products (float16's dS in range, below),
// D comes from the rounded output.
//
// Measured on MI355X, bfloat16 8 x 1024 x 12 x 64, causal: queries 34.1 us, keys 48.0 (45 GFLOP together, 550
// TFLOP/s); 1 x 8192 x 16 x 128, all pairs: queries 790, keys 1280 us (1040 and 860 TFLOP/s of their products).  Matrix
// instructions, exponentials and transposing LDS reads of the key pass share the time; registers hold it to one or two
// waves a SIMD.  Float32 4 x 512 x 12 x 64: queries 31.4 + 6.3 us, keys 43.4 + 8.9.  Within a window (MASK, attention_device.h),
// bfloat16 8 x 1024 x 12 x 64, 256 keys and 4 sinks: queries 28.7, keys 38.4; of a key block's 34000 cycles there 7000 pass
// before the first tile and 4000 after the last.
#pragma once

#include <algorithm>
#include <cmath>

#include "attention_device.h"

namespace lwl {
namespace {

constexpr int kBlock = 128;  // keys (queries) of a workgroup: 32 for each of four waves
constexpr int kTile = kTileRows;  // queries (keys) of a tile
constexpr int kMostQuerySplits = 64;

// In dV's product the probabilities are 2^kLift times too large (exact, and taken back at the end): dV sums
// a key's probabilities over the queries, all of which may be small, and small ones are subnormal in
// float16 and flushed by the exponential in float32.
constexpr float kLift = 14.0f, kLower = 0x1p-14f;
// float16 holds the dS of a key times a power of two, `held`, that puts the largest met so far at 2^kHeldTop or
// more: unscaled, probabilities of long rows times small dout are subnormal or zero (relative error of dK,
// 2048 queries over 4096 keys, dout of 1e-4: 5.3e-2; 4.7e-3 so, which is dK's own rounding), and dS of large
// dout is infinite where dK fits.  As with the forward's maximum, a key is a lane's column: the sums are
// rescaled when a score's gradient leaves the range, and what leaves it at the bottom is 2^-36 of the largest.
// Until the first, 2^kHeldStart; the power is taken back with dK's scale.
template <class T>
constexpr bool kHold = __is_same(T, f16);
constexpr int kHeldStart = 60, kHeldTop = 12;
constexpr float kMostF16 = 65504.0f;
__device__ __forceinline__ int exponent_bits(float v) { return (int)(__float_as_uint(v) >> 23) & 0xff; }
// 16-bit products start from what is to be subtracted of them, S - lse / c with c = scale log2(e), and dP - D,
// which saves an operation a score.  Their sums then round at the size of lse / c: not for float32.
template <class T>
constexpr bool kFoldStats = sizeof(T) == 2;

// Head sizes up to 96 leave registers for two waves a SIMD, which overlap; 128 of a 16-bit type runs one, whose
// two halves of a tile the scheduler may interleave.
template <class T, int DP>
constexpr int kUnroll = sizeof(T) == 2 && DP > 96 ? 2 : 1;
template <class T, int DP>
constexpr int kKeysOccupancy = sizeof(T) == 2 && DP <= 96 ? 2 : 1;
// The key pass loads a product's operands from LDS just before it, where all of them ahead would not fit the
// registers.  At 96 that makes room for the second wave: bfloat16 4 x 2048 x 16 x 96, causal, 195 -> 153 us.
template <class T, int DP>
constexpr bool kLoadLate = sizeof(T) == 4 || DP == 96;

// float32 keeps of every query, beside D, the factor that makes its probabilities sum to 1.  lse is one rounded
// number, so exp2(s - lse) is off by the same 2^-24 |lse| for a whole row, more than all else here together; the
// query pass meets every key of a row, so it sums what it computes and passes 1 / sum on.
template <class T>
constexpr bool kRenorm = sizeof(T) == 4;
__device__ __forceinline__ float renorm_factor(float total) {
  return total == 0.0f ? 0.0f : 1.0f / total;  // 0: no keys
}

// The workspace: D of every query (float32: and its factor), then (256-byte aligned) the partial sums of a pass that
// is split: the query pass's until attention_bwd_join_queries has run, then the key pass's.
__host__ __device__ inline int64_t delta_floats(const AttnArgs& a) {
  return ((a.dtype == kF32 ? 2 : 1) * a.batch * a.heads * a.queries + 63) / 64 * 64;
}
__device__ __forceinline__ float* partials(const AttnArgs& a) { return a.work + delta_floats(a); }

// Within a window the key blocks that hold sinks (the first of them) have all later queries and the others a window's:
// the former are given their own number of ranges, and their partial sums follow the others'.
__host__ __device__ inline int64_t sink_blocks(const AttnArgs& a) {
  const int64_t sinks = a.sinks < a.keys ? a.sinks : a.keys;
  return (sinks + kBlock - 1) / kBlock;
}
__host__ __device__ inline int64_t partial_rows(const AttnArgs& a) { return a.batch * a.kv_heads * a.keys; }
// Whether some query sees a key: `seen` is the end of those that the last query sees.
template <int MASK>
__device__ __forceinline__ bool key_seen(const Allowed& w, int key, int seen) {
  return key < seen && (MASK != kWindow || key < w.sinks || key >= window_begin(w, 0));
}
// Where the partial sums of range `split` of key `key` of the key head number bk lie, two rows of dim.
template <int MASK>
__device__ __forceinline__ float* key_partial(const AttnArgs& a, int64_t bk, int64_t key, int split, bool sinks) {
  float* p = partials(a);
  if (MASK == kWindow && sinks) {
    const int64_t rows = sink_blocks(a) * kBlock;
    if (a.splits > 1) p += a.splits * partial_rows(a) * 2 * a.dim;
    return p + ((split * a.batch * a.kv_heads + bk) * rows + key) * 2 * a.dim;
  }
  return p + (split * partial_rows(a) + bk * a.keys + key) * 2 * a.dim;
}

template <class T, int DP, bool FAST, int MASK>
__global__ __launch_bounds__(256, (kKeysOccupancy<T, DP>)) void attention_bwd_keys(const AttnArgs a) {
  using Tile = BothWays<DP>;
  constexpr int KK = DP / 16, DT = DP / 32, PL = kTile * Tile::S;  // size of a plane
  __shared__ __attribute__((aligned(16))) Elem<T> lds_q[kBufs<T>][kPlanes<T> * PL];
  __shared__ __attribute__((aligned(16))) Elem<T> lds_g[kBufs<T>][kPlanes<T> * PL];
  constexpr int kStats = kRenorm<T> ? 3 : 2;  // lse, D and float32's factor, kTile of each
  __shared__ __attribute__((aligned(16))) float lds_stat[kBufs<T>][kStats][kTile];
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = uniform((int)threadIdx.x >> 6);
  const uint32_t kvh = (uint32_t)a.kv_heads, kvb = (uint32_t)a.batch * kvh, group = (uint32_t)a.heads / kvh;
  const uint32_t id = work_order(blockIdx.x, gridDim.x, (uint32_t)a.cus), bk = id % kvb;
  const int64_t b = uniform((int)(bk / kvh)), hk = uniform((int)(bk % kvh));
  uint32_t splits = (uint32_t)a.splits, part = id / kvb, first_block = 0;
  bool of_sinks = false;
  if constexpr (MASK == kWindow) {
    const uint32_t blocks = (uint32_t)sink_blocks(a);
    of_sinks = part < blocks * (uint32_t)a.sink_splits;
    if (of_sinks) {
      splits = (uint32_t)a.sink_splits;
    } else {
      part -= blocks * (uint32_t)a.sink_splits;
      first_block = blocks;
    }
  }
  const int split = uniform((int)(part % splits));
  // causal: the first keys have the most queries
  const int k0 = uniform((int)(first_block + part / splits)) * kBlock;
  const int dim = (int)a.dim;
  const Allowed allow = allowed_keys(a, b);
  const int queries = (int)a.queries;
  const int seen = key_end(allow, queries - 1);  // keys that some query sees
  const int wk0 = k0 + wave * 32, key = wk0 + (lane & 31);
  Opd<T> kf[KK], vf[KK];
  load_operand<T, DP, FAST>(kf, (const T*)a.k + b * a.ks[0] + hk * a.ks[1] + (int64_t)key * a.ks[2], dim,
                           key_seen<MASK>(allow, key, seen));
  load_operand<T, DP, FAST>(vf, (const T*)a.v + b * a.vs[0] + hk * a.vs[1] + (int64_t)key * a.vs[2], dim,
                           key_seen<MASK>(allow, key, seen));
  f32x16 dk[DT] = {}, dv[DT] = {};
  float held = __builtin_ldexpf(1.0f, kHeldStart);
  const float c = a.scale * kLog2E, inv_c = 1.0f / c;
  // queries before k0 - off see none of the block's keys (so none that sees nothing is ever read), those
  // before wk0 - off none of the wave's
  const int first = k0 >= seen ? queries : std::max(0, k0 - allow.off);
  const int wave_first = wk0 >= seen ? queries : wk0 - allow.off;
  // within a window, queries from here on see none of the block's keys, the wave's, this lane's
  int last = queries, wave_last = queries, lane_last = queries;
  if constexpr (MASK == kWindow) {
    const auto past = [&](int key) {  // a key's queries end here, sinks' never
      const int64_t p = (int64_t)key + allow.window - allow.off;
      return p < queries ? (int)p : queries;
    };
    if (k0 >= allow.sinks) last = past(std::min(k0 + kBlock, allow.len) - 1);
    if (wk0 >= allow.sinks) wave_last = past(std::min(wk0 + 32, allow.len) - 1);
    if (key >= allow.sinks) lane_last = past(key);
  }
  const T* qp = (const T*)a.q + b * a.qs[0] + hk * group * a.qs[1];
  const T* gp = (const T*)a.dout + b * a.dos[0] + hk * group * a.dos[1];
  const int64_t head0 = (b * a.heads + hk * group) * a.queries;
  TileLoader<T, DP, FAST> qt, gt;
  qt.init(qp, a.qs[2], dim, queries);
  gt.init(gp, a.dos[2], dim, queries);
  float sr = 0.0f;
  // Tiles of the first head, then of the next one of the group: one sequence, of which this workgroup
  // takes the tiles begin .. end.
  const int per_head = last > first ? (last - first + kTile - 1) / kTile : 0, tiles = per_head * (int)group;
  const int share = (tiles + (int)splits - 1) / (int)splits;
  const int begin = std::min(split * share, tiles), end = std::min(begin + share, tiles);
  auto fetch = [&](uint32_t fg, int fq) {
    qt.base = qp + fg * a.qs[1];
    gt.base = gp + fg * a.dos[1];
    qt.fetch(fq, last);
    gt.fetch(fq, last);
    if (threadIdx.x < kStats * kTile) {
      const int q = fq + (threadIdx.x & (kTile - 1));
      const bool is_d = threadIdx.x >= kTile, is_factor = threadIdx.x >= 2 * kTile;
      const float* stat = (is_d ? a.work : a.lse) + head0 + (int64_t)fg * queries;
      if (is_factor) stat += a.batch * a.heads * a.queries;
      sr = q < last ? stat[q] : (is_d ? 0.0f : INFINITY);  // past the last: no probabilities
      if constexpr (!kReadAhead<T, FAST>)
        sr = is_factor ? sr : is_d ? -sr : kFoldStats<T> ? (kLift - sr * kLog2E) * inv_c : kLift - sr * kLog2E;
    }
  };
  auto put = [&](int buf) {
    qt.template put<Tile>(lds_q[buf]);
    gt.template put<Tile>(lds_g[buf]);
    if constexpr (kReadAhead<T, FAST>) {  // not before, for it would wait for the tile's loads
      const bool is_d = threadIdx.x >= kTile, is_factor = threadIdx.x >= 2 * kTile;
      sr = is_factor ? sr : is_d ? -sr : kFoldStats<T> ? (kLift - sr * kLog2E) * inv_c : kLift - sr * kLog2E;
    }
    if (threadIdx.x < kStats * kTile) lds_stat[buf][threadIdx.x / kTile][threadIdx.x & (kTile - 1)] = sr;
  };
  int buf = 0;
  uint32_t g = begin < end ? (uint32_t)uniform(begin / per_head) : 0;
  int q0 = begin < end ? first + (begin - (int)g * per_head) * kTile : 0;
  if (begin < end) {
    fetch(g, q0);
    if constexpr (kBufs<T> == 2) put(0);
  }
  wait_operands<T, FAST>(kf);
  wait_operands<T, FAST>(vf);
  for (int i = begin; i < end; ++i) {
    __syncthreads();  // this tile is there, the one before has been read
    if constexpr (kBufs<T> == 1) {
      put(0);
      __syncthreads();
    }
    const bool head_ends = q0 + kTile >= last, more = i + 1 < end;
    const uint32_t next_g = head_ends ? g + 1 : g;
    const int next_q = head_ends ? first : q0 + kTile;
    if (more) fetch(next_g, next_q);
    if (q0 + kTile > wave_first && (MASK != kWindow || q0 < wave_last)) {
      // some pair of the tile is not allowed
      const bool masked = key_end(allow, q0) < wk0 + 32;
      const bool passed = MASK == kWindow && window_begin(allow, std::min(q0 + kTile, queries) - 1) > wk0 && wk0 + 32 > allow.sinks;
#pragma unroll kUnroll<T, DP>
      for (int t = 0; t < 2; ++t) {
        const int at = t * 32;
        const Elem<T>* lq = lds_q[buf] + at * Tile::S;
        const Elem<T>* lg = lds_g[buf] + at * Tile::S;
        f32x16 s, dp;
        {
          Opd<T> qf[KK], gf[KK];
#pragma unroll
          for (int r4 = 0; r4 < 4; ++r4) {
            const f32x4 l = *(const f32x4*)&lds_stat[buf][0][at + r4 * 8 + half * 4];
            const f32x4 d = *(const f32x4*)&lds_stat[buf][1][at + r4 * 8 + half * 4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              s[r4 * 4 + r] = kFoldStats<T> ? l[r] : 0.0f;
              dp[r4 * 4 + r] = kFoldStats<T> ? d[r] : 0.0f;
            }
          }
          const auto load_q = [&](int kk) { qf[kk] = lds_operand<T>(lq + Tile::at(lane & 31, kk * 16 + half * 8), PL); };
          const auto load_g = [&](int kk) { gf[kk] = lds_operand<T>(lg + Tile::at(lane & 31, kk * 16 + half * 8), PL); };
          if constexpr (kLoadLate<T, DP>) {
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
              load_q(kk);
              load_g(kk);
              s = mma32(qf[kk], kf[kk], s);
              dp = mma32(gf[kk], vf[kk], dp);
              fence_operands<T>();
              if (kk % 2) fence_schedule<T>();  // two steps' operands at a time
            }
          } else {
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
              load_q(kk);
              load_g(kk);
            }
            if constexpr (DP <= 64) fence_schedule<T>();
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
              s = mma32(qf[kk], kf[kk], s);
              dp = mma32(gf[kk], vf[kk], dp);
            }
          }
        }
        Opd<T> gc[2][DT], qc[2][DT];
        const auto load_columns = [&](int u, int d) {
          const int row = u * 16 + half * 4;
          gc[u][d] = lds_column_operand<T, Tile>(lg, PL, row, row + 8, d * 32 + (lane & 16));
          qc[u][d] = lds_column_operand<T, Tile>(lq, PL, row, row + 8, d * 32 + (lane & 16));
        };
        if constexpr (!kLoadLate<T, DP>) {
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int d = 0; d < DT; ++d) load_columns(u, d);
        }
        if constexpr (DP <= 96) fence_schedule<T>();
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if constexpr (kFoldStats<T>) {
            s[r] = exp2_hw(s[r] * c);
          } else {
            const int i = at + (r >> 2) * 8 + half * 4 + (r & 3);
            s[r] = exp2_hw(fmaf(s[r], c, lds_stat[buf][0][i])) * lds_stat[buf][kStats - 1][i];
            dp[r] += lds_stat[buf][1][i];
          }
          dp[r] *= s[r];
        }
        if constexpr (MASK == kWindow) {
          if (masked || passed) {
            // the queries from this key's position on, as far as its window reaches: their tile's bits
            const int from = key < allow.len ? key - allow.off : queries;
            const Seen seen = seen_keys(q0, lane_last, from, q0);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const uint32_t mask = bit_mask(t ? seen.w[1] : seen.w[0], (r >> 2) * 8 + (r & 3));
              s[r] = masked_term(s[r], mask);
              dp[r] = masked_term(dp[r], mask);
            }
          }
        } else if (masked) {
          // key < key_end(q), that is q >= key - off
          const int from = key < allow.len ? key - allow.off - q0 - at - half * 4 : kTile;
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if ((r >> 2) * 8 + (r & 3) < from) s[r] = dp[r] = 0.0f;
        }
        if constexpr (kHold<T>) {
          float most = 0.0f;
#pragma unroll
          for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(dp[r]));
          if (__any(most * held > kMostF16)) {
            most = max_halves(most);
            if (most * held > kMostF16) {
              const float next = __uint_as_float((uint32_t)(254 + kHeldTop - exponent_bits(most)) << 23);
              const int shrink = exponent_bits(next) - exponent_bits(held);
              held = next;
#pragma unroll
              for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) dk[d][r] = __builtin_ldexpf(dk[d][r], shrink);
            }
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) dp[r] *= held;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float e[8], f[8];
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            e[r] = s[u * 8 + r];
            f[r] = dp[u * 8 + r];
          }
          const Opd<T> p = operand_of<T>(e), ds = operand_of<T>(f);
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            if constexpr (kLoadLate<T, DP>) load_columns(u, d);
            dv[d] = mma32(gc[u][d], p, dv[d]);
            dk[d] = mma32(qc[u][d], ds, dk[d]);
            fence_operands<T>();
          }
        }
      }
    }
    if (kBufs<T> == 2 && more) put(buf ^ (kBufs<T> - 1));
    buf ^= kBufs<T> - 1;
    g = next_g;
    q0 = next_q;
  }
  if (key >= (int)a.keys) return;
  const float dk_scale = kHold<T> ? __builtin_ldexpf(a.scale * kLower, 127 - exponent_bits(held)) : a.scale * kLower;
  if (splits > 1) {  // summed by attention_bwd_join, which takes keys that no query sees for zeros
    if (!key_seen<MASK>(allow, key, seen)) return;
    float* sums = key_partial<MASK>(a, b * a.kv_heads + hk, key, split, of_sinks);
    store_result<float, DP, FAST>(sums, dk, dk_scale, dim);
    store_result<float, DP, FAST>(sums + dim, dv, kLower, dim);
    return;
  }
  store_result<T, DP, FAST>((T*)a.dk + b * a.dks[0] + hk * a.dks[1] + (int64_t)key * a.dks[2], dk, dk_scale, dim);
  store_result<T, DP, FAST>((T*)a.dv + b * a.dvs[0] + hk * a.dvs[1] + (int64_t)key * a.dvs[2], dv, kLower, dim);
}

template <class T, int DP, bool FAST, int MASK>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void attention_bwd_queries(const AttnArgs a) {
  // rows padded by 16 bytes: one tile in three is read by columns, and BothWays' addresses cost registers
  using Tile = Padded<DP>;
  constexpr int KK = DP / 16, DT = DP / 32, PL = kTile * Tile::S;  // size of a plane
  __shared__ __attribute__((aligned(16))) Elem<T> lds_k[kBufs<T>][kPlanes<T> * PL];
  __shared__ __attribute__((aligned(16))) Elem<T> lds_v[kBufs<T>][kPlanes<T> * PL];
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = uniform((int)threadIdx.x >> 6);
  const RowsWork w = rows_work(a);
  const int64_t b = w.b, hk = w.hk, h = w.h;
  const int q0 = w.block * kBlock;
  const int dim = (int)a.dim;
  const Allowed allow = allowed_keys(a, b);
  const int queries = (int)a.queries, wq0 = q0 + wave * 32, q = wq0 + (lane & 31);
  int q_end = q < queries ? key_end(allow, q) : 0;
  Walk<MASK, kTile> at;
  if constexpr (MASK == kWindow) {
    at = window_walk<kTile>(a, allow, q0, std::min(q0 + kBlock, queries) - 1, w.split, 0);
  } else {
    at.j = w.split * (int)a.split_len;
    at.end = std::min(key_end(allow, std::min(q0 + kBlock, queries) - 1), at.j + (int)a.split_len);
  }
  const int free_end = wq0 < queries ? key_end(allow, wq0) : 0;
  const int wave_end = wq0 < queries ? key_end(allow, std::min(wq0 + 32, queries) - 1) : 0;
  // within a window: of this lane's query, the wave's first and its last
  int q_begin = 0, wave_begin = 0, free_begin = 0;
  if constexpr (MASK == kWindow) {
    q_begin = window_begin(allow, std::min(q, queries - 1));
    if (allow.sinks == 0 && q_begin >= q_end) q_end = 0;  // past the last key by a window: it sees nothing
    wave_begin = window_begin(allow, std::min(wq0, queries - 1));
    free_begin = window_begin(allow, std::min(wq0 + 32, queries) - 1);
  }
  const T* kp = (const T*)a.k + b * a.ks[0] + hk * a.ks[1];
  const T* vp = (const T*)a.v + b * a.vs[0] + hk * a.vs[1];
  TileLoader<T, DP, FAST> kt, vt;
  kt.init(kp, a.ks[2], dim, (int)a.keys);
  vt.init(vp, a.vs[2], dim, (int)a.keys);
  if (at.live()) {
    kt.fetch(at.j, at.stop());
    vt.fetch(at.j, at.stop());
  }
  const int64_t row = (b * a.heads + h) * a.queries + q;
  // a query without keys has no probabilities: exp2(-infinity)
  float lse = q_end > 0 ? a.lse[row] * kLog2E : INFINITY;
  Opd<T> qf[KK], gf[KK];
  load_operand<T, DP, FAST>(qf, (const T*)a.q + b * a.qs[0] + h * a.qs[1] + (int64_t)q * a.qs[2], dim, q_end > 0);
  float delta = 0.0f, norm = 0.0f;
  Raw8<T> g_chunks[KK], o_chunks[KK];
  if constexpr (kReadAhead<T, FAST>) {
    load_chunks(g_chunks, (const T*)a.dout + b * a.dos[0] + h * a.dos[1] + (int64_t)q * a.dos[2], dim, q_end > 0);
    load_chunks(o_chunks, (const T*)a.out + b * a.os[0] + h * a.os[1] + (int64_t)q * a.os[2], dim, q_end > 0);
  }
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) {
    Raw8<T> gr, orow;
    if constexpr (!kReadAhead<T, FAST>) {
      load_chunk<T, FAST>(gr, (const T*)a.dout + b * a.dos[0] + h * a.dos[1] + (int64_t)q * a.dos[2], kk, dim, q_end > 0);
      load_chunk<T, FAST>(orow, (const T*)a.out + b * a.os[0] + h * a.os[1] + (int64_t)q * a.os[2], kk, dim, q_end > 0);
    } else {
      gr = g_chunks[kk];
      orow = o_chunks[kk];
    }
    gf[kk] = operand_of<T>(gr);
    float x[8], y[8];
    unpack8(x, gr);
    unpack8(y, orow);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      delta += x[r] * y[r];
      norm += x[r] * x[r];
    }
  }
  delta += other_half(delta);
  // float16 scores' gradients are held 2^-e times as large, 2^e about the length of this query's row of dout: they
  // are then not subnormal where gradients are small, and |dS| <= 4 max |v| (lengths again).  It costs nothing:
  // the power goes into lse and back out with dQ's scale.  Where values longer than 16000 take them past
  // float16's range all the same, the power is raised and what is summed so far taken down.
  float unscale = a.scale;
  if constexpr (__is_same(T, f16)) {
    norm += other_half(norm);
    if (norm > 0x1p-60f && norm < 0x1p60f) {
      const int e = (((int)(__float_as_uint(norm) >> 23) & 0xff) - 127) >> 1;
      lse += (float)e;
      unscale = ldexpf(a.scale, e);
    }
  }
  if (half == 0 && q < queries && w.split == 0) a.work[row] = delta;
  f32x16 dq[DT] = {};
  float total = 0.0f;  // of the query's probabilities
  const float c = a.scale * kLog2E;
  if (kBufs<T> == 2 && at.live()) {
    kt.template put<Tile>(lds_k[0]);
    vt.template put<Tile>(lds_v[0]);
  }
  wait_operands<T, FAST>(qf);
  wait_operands<T, FAST>(gf);
  int buf = 0;
  for (; at.live(); at.step(), buf ^= kBufs<T> - 1) {
    const int j0 = at.j;
    __syncthreads();  // this tile is there, the one before has been read
    if constexpr (kBufs<T> == 1) {
      kt.template put<Tile>(lds_k[0]);
      vt.template put<Tile>(lds_v[0]);
      __syncthreads();
    }
    const bool more = at.more();
    if (more) {
      kt.fetch(at.next(), at.next_stop());
      vt.fetch(at.next(), at.next_stop());
    }
    if (j0 < wave_end && (MASK != kWindow || j0 + kTile > wave_begin || j0 < allow.sinks)) {
#pragma unroll 1
      for (int t = 0; t < 2; ++t) {
        const Elem<T>* lk = lds_k[buf] + t * 32 * Tile::S;
        const Elem<T>* lv = lds_v[buf] + t * 32 * Tile::S;
        f32x16 s = {}, dp = {};
        {
          Opd<T> kf[KK], vf[KK];
          const auto load_k = [&](int kk) { kf[kk] = lds_operand<T>(lk + Tile::at(lane & 31, kk * 16 + half * 8), PL); };
          const auto load_v = [&](int kk) { vf[kk] = lds_operand<T>(lv + Tile::at(lane & 31, kk * 16 + half * 8), PL); };
          if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
              load_k(kk);
              load_v(kk);
              s = mma32(kf[kk], qf[kk], s);
              dp = mma32(vf[kk], gf[kk], dp);
              fence_operands<T>();
            }
          } else {
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) load_k(kk);
            // beyond 64 the two products one after the other, which holds half as many operands at a time
            if constexpr (DP > 64) {
              fence_schedule<T>();
#pragma unroll
              for (int kk = 0; kk < KK; ++kk) s = mma32(kf[kk], qf[kk], s);
            }
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) load_v(kk);
            fence_schedule<T>();
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
              if constexpr (DP <= 64) s = mma32(kf[kk], qf[kk], s);
              dp = mma32(vf[kk], gf[kk], dp);
            }
          }
        }
        Opd<T> kc[2][DT];
        const auto load_columns = [&](int u, int d) {
          kc[u][d] = lds_column_operand<T, Tile>(lk, PL, u * 16 + half * 4, u * 16 + half * 4 + 8, d * 32 + (lane & 16));
        };
        if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int d = 0; d < DT; ++d) load_columns(u, d);
        }
        fence_schedule<T>();
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[r] = exp2_hw(fmaf(s[r], c, -lse));
          if constexpr (!kRenorm<T>) s[r] *= dp[r] - delta;
        }
        // dp: may be NaN where masked
        if constexpr (MASK == kWindow) {
          if (j0 + kTile > std::min(free_end, at.stop()) ||
              (j0 < free_begin && std::min(j0 + kTile, at.stop()) > allow.sinks)) {
            const Seen seen = seen_keys(j0, std::min(q_end, at.stop()), q_begin, allow.sinks);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const uint32_t mask = bit_mask(t ? seen.w[1] : seen.w[0], (r >> 2) * 8 + (r & 3));
              s[r] = masked_term(s[r], mask);
              dp[r] = masked_term(dp[r], mask);
            }
          }
        } else if (j0 + kTile > free_end) {
          const int lim = q_end - j0 - t * 32 - half * 4;
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if ((r >> 2) * 8 + (r & 3) >= lim) s[r] = dp[r] = 0.0f;
        }
        if constexpr (kRenorm<T>) {
          float sum = 0.0f;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            sum += s[r];
            s[r] *= dp[r] - delta;
          }
          total += sum;
        }
        if constexpr (kHold<T>) {
          float most = 0.0f;
#pragma unroll
          for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(s[r]));
          if (__any(most > kMostF16)) {
            most = max_halves(most);
            const int n = most > kMostF16 ? exponent_bits(most) - 127 - kHeldTop : 0;
            lse += (float)n;
            unscale = __builtin_ldexpf(unscale, n);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = __builtin_ldexpf(s[r], -n);
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
              for (int r = 0; r < 16; ++r) dq[d][r] = __builtin_ldexpf(dq[d][r], -n);
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float e[8];
#pragma unroll
          for (int r = 0; r < 8; ++r) e[r] = s[u * 8 + r];
          const Opd<T> ds = operand_of<T>(e);
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            if constexpr (sizeof(T) == 4) load_columns(u, d);
            dq[d] = mma32(kc[u][d], ds, dq[d]);
            fence_operands<T>();
          }
        }
      }
    }
    if (kBufs<T> == 2 && more) {
      kt.template put<Tile>(lds_k[buf ^ (kBufs<T> - 1)]);
      vt.template put<Tile>(lds_v[buf ^ (kBufs<T> - 1)]);
    }
  }
  if constexpr (kRenorm<T>) total += other_half(total);
  if (q >= queries) return;
  const int64_t rows = a.batch * a.heads * a.queries;
  if (a.splits > 1) {  // summed by attention_bwd_join_queries
    const int64_t part = row * a.splits + w.split;
    if (kRenorm<T> && half == 0) partials(a)[rows * a.splits * dim + part] = total;
    store_result<float, DP, FAST>(partials(a) + part * dim, dq, unscale, dim);
    return;
  }
  if constexpr (kRenorm<T>) {
    const float factor = renorm_factor(total);
    if (half == 0) a.work[rows + row] = factor;
    unscale *= factor;
  }
  store_result<T, DP, FAST>((T*)a.dq + b * a.dqs[0] + h * a.dqs[1] + (int64_t)q * a.dqs[2], dq, unscale, dim);
}

// dQ of a query, and float32's factor, from the ranges of keys, in their order: a thread sums eight values.
template <class T>
__global__ __launch_bounds__(256) void attention_bwd_join_queries(const AttnArgs a) {
  const int dim = (int)a.dim, chunks = (dim + 7) / 8, rows_wg = 256 / chunks, r = threadIdx.x / chunks;
  const int col = (threadIdx.x - r * chunks) * 8, splits = a.splits;
  const int64_t rows = a.batch * a.heads * a.queries, row = (int64_t)blockIdx.x * rows_wg + r;
  if (r >= rows_wg || row >= rows) return;
  const float* part = partials(a) + row * splits * dim + col;
  float sum[8] = {}, factor = 1.0f;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    float v[8];
    load8(v, part + s * dim, dim - col);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] += v[i];
  }
  if constexpr (kRenorm<T>) {
    const float* totals = partials(a) + rows * splits * dim + row * splits;
    float total = 0.0f;
    for (int s = 0; s < splits; ++s) total += totals[s];
    factor = renorm_factor(total);
    if (col == 0) a.work[rows + row] = factor;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) sum[i] *= factor;
  const uint32_t queries = (uint32_t)a.queries, heads = (uint32_t)a.heads, bh = (uint32_t)row / queries;
  const uint32_t q = (uint32_t)row - bh * queries;
  const int64_t b = bh / heads, h = bh % heads;
  store8((T*)a.dq + b * a.dqs[0] + h * a.dqs[1] + (int64_t)q * a.dqs[2] + col, sum, dim - col);
}

// Keys of which some are in ranges: all, or the blocks of sinks.
template <int MASK>
__host__ __device__ inline int64_t join_keys(const AttnArgs& a) {
  if (MASK != kWindow || a.splits > 1) return a.keys;
  return std::min(a.keys, sink_blocks(a) * kBlock);
}

// dK and dV of a key from the ranges' partial sums, in the ranges' order: a thread sums eight values of them.
template <class T, int MASK>
__global__ __launch_bounds__(256) void attention_bwd_join(const AttnArgs a) {
  const int dim = (int)a.dim, chunks = (dim + 7) / 8, keys_wg = 128 / chunks, r = threadIdx.x / (2 * chunks);
  const int chunk = threadIdx.x - r * 2 * chunks;
  // within a window those of sinks only, where the others' are not in ranges
  const uint32_t keys = (uint32_t)join_keys<MASK>(a), kvh = (uint32_t)a.kv_heads, blocks = (keys + keys_wg - 1) / keys_wg;
  const uint32_t bk = blockIdx.x / blocks, key = (blockIdx.x - bk * blocks) * keys_wg + r;
  if (r >= keys_wg || key >= keys) return;
  const bool is_v = chunk >= chunks;
  const int col = (is_v ? chunk - chunks : chunk) * 8;
  const int64_t b = bk / kvh, hk = bk % kvh;
  const bool of_sinks = MASK == kWindow && key < sink_blocks(a) * kBlock;
  int splits = of_sinks ? a.sink_splits : a.splits;
  if (MASK == kWindow && splits == 1) return;  // written by the key pass
  const int64_t next = key_partial<MASK>(a, 0, 0, 1, of_sinks) - key_partial<MASK>(a, 0, 0, 0, of_sinks);
  const float* part = key_partial<MASK>(a, bk, key, 0, of_sinks) + (is_v ? dim : 0) + col;
  float sum[8] = {};
  const Allowed allow = allowed_keys(a, b);
  if (!key_seen<MASK>(allow, (int)key, key_end(allow, (int)a.queries - 1))) splits = 0;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    float v[8];
    load8(v, part + s * next, dim - col);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] += v[i];
  }
  T* dst = is_v ? (T*)a.dv + b * a.dvs[0] + hk * a.dvs[1] + (int64_t)key * a.dvs[2]
                : (T*)a.dk + b * a.dks[0] + hk * a.dks[1] + (int64_t)key * a.dks[2];
  store8(dst + col, sum, dim - col);
}

// Ranges of a query block's keys, where blocks are too few for the compute units: the estimate of the forward pass,
// with this pass's times, in us.  Of 1, 2, 3, 4, 10 ranges, with the join: float32 5 x 65 queries over up to 2641
// keys, 6 heads on 2, of size 32: 114, 66, 49, 41, 26 us, 11 are taken; float32 4 x 512 x 12 x 64: 46, 38, 42, 46,
// 56 us, 2; bfloat16 3 x 1807 x 4 x 96: 46, 39, 40, 41, 60 us, 3; 8 x 1024 x 12 x 64: 34, 53, 62, 72, 120 us, 1.
template <int MASK>
void plan_query_splits(AttnArgs& a) {
  const double unit = (double)((a.dim + 31) / 32 * 32) / 64, cus = (double)device_cus();
  const double alone = (a.dtype == kF32 ? 5.1 : 1.1) * unit, spread = (a.dtype == kF32 ? 4.8 : 1.0) * unit;
  // keys of the longest walk
  const int64_t keys = MASK == kWindow ? window_tiles(a, kBlock) * kTile : a.keys, tiles = (keys + kTile - 1) / kTile;
  const double wgs = (double)(a.batch * a.heads) * (double)((a.queries + kBlock - 1) / kBlock);
  const bool half = MASK != kWindow || keys >= a.keys;
  const double walked = (double)tiles * (half && ((a.causal && a.queries * 2 > a.keys) || a.lengths) ? 0.55 : 1.0);
  const double bytes = 8.0 * (double)(a.batch * a.heads) * (double)a.queries * (double)a.dim;
  double best = 0.0;
  int64_t splits = 1;
  for (int64_t n = 1; n <= std::min<int64_t>(tiles / 4 + 1, kMostQuerySplits); n = n < 4 ? n + 1 : n + n / 4) {
    const double walk = (double)((tiles + n - 1) / n + 1) * alone, all = wgs * ((double)n + walked) * spread / cus;
    const double t = std::max(walk, all) + (n > 1 ? 4.5 + (double)n * bytes / 18e6 : 0.0);
    // several only where they gain more than the estimate may be off by
    if (n == 1 || t < best * (splits == 1 ? 0.85 : 1.0)) {
      best = t;
      splits = n;
    }
  }
  a.split_len = splits > 1 ? ((keys + splits - 1) / splits + kTile - 1) / kTile * kTile : std::max<int64_t>(keys, 1);
  a.splits = splits > 1 ? (int)((keys + a.split_len - 1) / a.split_len) : 1;
}

// Workgroups of the key pass, planned, of the query pass with one range, and of the key pass's join.
template <int MASK>
int64_t key_workgroups(const AttnArgs& a) {
  int64_t blocks = (a.keys + kBlock - 1) / kBlock * a.splits;
  if (MASK == kWindow) blocks += sink_blocks(a) * (a.sink_splits - a.splits);
  return blocks * a.batch * a.kv_heads;
}
inline int64_t query_workgroups(const AttnArgs& a) { return a.batch * a.heads * ((a.queries + kBlock - 1) / kBlock); }
template <int MASK>
int64_t join_workgroups(const AttnArgs& a) {
  if (a.splits == 1 && !(MASK == kWindow && a.sink_splits > 1 && sink_blocks(a) > 0)) return 0;
  const int64_t keys_wg = 128 / ((a.dim + 7) / 8);
  return a.batch * a.kv_heads * ((join_keys<MASK>(a) + keys_wg - 1) / keys_wg);
}

template <class T, int DP, bool FAST, int MASK>
hipError_t launch(const AttnArgs& a, hipStream_t s) {
  const int64_t kgrid = key_workgroups<MASK>(a), qgrid = query_workgroups(a), jgrid = join_workgroups<MASK>(a);
  if (qgrid > 0) {
    AttnArgs by_keys = a;  // a's ranges are the key pass's
    plan_query_splits<MASK>(by_keys);
    hipLaunchKernelGGL((attention_bwd_queries<T, DP, FAST, MASK>), dim3((unsigned)(qgrid * by_keys.splits)), dim3(256), 0, s,
                       by_keys);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (by_keys.splits > 1) {
      const int64_t rows = a.batch * a.heads * a.queries, rows_wg = 256 / ((a.dim + 7) / 8);
      hipLaunchKernelGGL((attention_bwd_join_queries<T>), dim3((unsigned)((rows + rows_wg - 1) / rows_wg)), dim3(256), 0,
                         s, by_keys);
      e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
  }
  if (kgrid > 0) {
    hipLaunchKernelGGL((attention_bwd_keys<T, DP, FAST, MASK>), dim3((unsigned)kgrid), dim3(256), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (jgrid > 0) hipLaunchKernelGGL((attention_bwd_join<T, MASK>), dim3((unsigned)jgrid), dim3(256), 0, s, a);
  }
  return hipGetLastError();
}

template <class T, int DP, int MASK>
hipError_t run(const AttnArgs& a, hipStream_t s) {
  const bool fast = a.dim % 8 == 0 && fast_rows(a.q, a.qs, sizeof(T)) && fast_rows(a.k, a.ks, sizeof(T)) &&
                    fast_rows(a.v, a.vs, sizeof(T)) && fast_rows(a.dout, a.dos, sizeof(T));
  return fast ? launch<T, DP, true, MASK>(a, s) : launch<T, DP, false, MASK>(a, s);
}

template <class T, int MASK>
hipError_t run_dim(const AttnArgs& a, hipStream_t s) {
  switch ((a.dim + 31) / 32) {
    case 1: return run<T, 32, MASK>(a, s);
    case 2: return run<T, 64, MASK>(a, s);
    case 3: return run<T, 96, MASK>(a, s);
    case 4: return run<T, 128, MASK>(a, s);
  }
  return hipErrorInvalidValue;
}

// Ranges of a key block's queries (all query heads that share the key head in one sequence): what an estimate
// of the time makes shortest, in us, as in the forward pass: the longest walk alone, or all work spread over
// the compute units, in rounds where the works are equal; and with several ranges the join.
// Measured on MI355X, a tile of 64 queries: bfloat16 of head size 64 1.2 us when a compute unit has two
// workgroups and 1.6 alone, of size 128 2.8 us (one fits); float32 of size 64 6.8 us; and what a workgroup
// takes before its first tile and for its results, 7 and 10 us at size 64.  Of 1, 2, 3, 4 ranges, with the join:
// 4 x 512 x 12 x 64 in float32 60.9, 51.1, 59.1, 61.2 us, 2 are taken; float16 6 x 515 queries over up to 1531 keys,
// 12 heads on 4, of size 80: 70.4, 63.3, 77.7, 74.3 us, 2; bfloat16 8 x 1024 x 12 x 64: 47 us and up from 85, 1.
template <int MASK>
void plan_bwd_splits(AttnArgs& a) {
  const double unit = (double)((a.dim + 31) / 32 * 32) / 64, cus = (double)device_cus();
  const bool two = a.dtype != kF32 && a.dim <= 96;  // workgroups on a compute unit
  const double spread = (a.dtype == kF32 ? 6.8 : two ? 1.2 : 1.4) * unit;
  const double alone = (a.dtype == kF32 ? 6.8 : two ? 1.6 : 1.4) * unit;
  const double fixed = (a.dtype == kF32 ? 10.0 : 7.0) * unit, slots = two ? 2 * cus : cus;
  const int64_t group = a.heads / a.kv_heads, all_tiles = group * ((a.queries + kTile - 1) / kTile);
  int64_t tiles = all_tiles;
  if (MASK == kWindow)  // of the queries that a block's keys are in the window of
    tiles = std::min(tiles, group * ((std::min(a.window, a.queries) + kBlock - 1 + kTile - 1) / kTile));
  // with lengths, which only the device knows, about half of the blocks hold keys; the others take a little
  const double wgs = (double)(a.batch * a.kv_heads) * (double)((a.keys + kBlock - 1) / kBlock) * (a.lengths ? 0.7 : 1.0);
  const bool halves = a.causal && a.keys * 2 > a.queries && tiles == all_tiles;
  const double bytes = 16.0 * (double)(a.batch * a.kv_heads) * (double)a.keys * (double)a.dim;
  double best = 0.0;
  a.splits = 1;
  for (int64_t n = 1; n <= std::min<int64_t>(tiles / 4 + 1, 256); n = n < 4 ? n + 1 : n + n / 4) {
    const double walk = (double)((tiles + n - 1) / n), works = wgs * (double)n;
    const double whole = std::floor(works / slots), rest = works - whole * slots;
    const double round = walk * spread * slots / cus + fixed;
    const double all = halves ? 0.55 * wgs * (double)tiles / cus * spread + works / slots * fixed
                              : whole * round + (rest > cus ? round : rest > 0.0 ? walk * alone + fixed : 0.0);
    const double t = std::max(walk * alone + fixed, all) + (n > 1 ? 4.0 + (double)n * bytes / 11e6 : 0.0);
    if (n == 1 || t < best) {
      best = t;
      a.splits = (int)n;
    }
  }
  // Sinks' blocks walk over all later queries: in ranges where one alone, sharing its compute unit, would outlast all work
  // spread over the compute units and the join.  bfloat16, a training step with 4 sinks, us: 8 x 1024 x 12 x 64, window
  // 256, in 1, 2, 3 ranges 86, 92, 92, 1 is taken; 1 x 8192 x 12 x 64, window 512, in 1, 2, 4, 8, 16 ranges 289, 183, 130, 120,
  // 120, 8.
  a.sink_splits = 1;
  if (MASK == kWindow) {
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(all_tiles / 4, 256));
    const double sinks = (double)(a.batch * a.kv_heads * sink_blocks(a)), shared = two ? 1.8 * spread : alone;
    const double all = (wgs * (double)tiles + sinks * (double)all_tiles) * spread / cus + (wgs + sinks) / slots * fixed;
    const double part = 16.0 * sinks * (double)kBlock * (double)a.dim / 11e6;
    double least = 0.0;
    for (int64_t n = 1; n <= most; n = n < 4 ? n + 1 : n + n / 4) {
      const double walk = (double)((all_tiles + n - 1) / n) * shared + fixed;
      const double t = std::max(walk, all + (double)(n - 1) * sinks / slots * fixed) + (n > 1 ? 5.0 + (double)n * part : 0.0);
      if (n == 1 || t < least) {
        least = t;
        a.sink_splits = (int)n;
      }
    }
  }
}

// (The query pass's ranges, and their join, are only where its workgroups are few.)
template <int MASK>
bool bwd_fits(AttnArgs a) {
  // a block of keys has fewer than 512 ranges, sinks' and others, and 16 workgroups of the join
  if (a.batch * a.heads * ((std::max(a.queries, a.keys) + kBlock - 1) / kBlock) <= kMostWorkgroups / 1024) return true;
  plan_bwd_splits<MASK>(a);
  return std::max({key_workgroups<MASK>(a), query_workgroups(a), join_workgroups<MASK>(a)}) <= kMostWorkgroups;
}

template <int MASK>
int64_t bwd_work(const AttnArgs& args) {
  AttnArgs a = args, by_keys = args;
  plan_bwd_splits<MASK>(a);
  plan_query_splits<MASK>(by_keys);
  int64_t keys = a.splits > 1 ? (int64_t)a.splits * 2 * partial_rows(a) * a.dim : 0;
  if (MASK == kWindow && a.sink_splits > 1)
    keys += (int64_t)a.sink_splits * 2 * a.batch * a.kv_heads * sink_blocks(a) * kBlock * a.dim;
  const int64_t queries = by_keys.splits > 1 ? (int64_t)by_keys.splits * a.batch * a.heads * a.queries * (a.dim + 1) : 0;
  return delta_floats(a) + std::max(keys, queries);
}

template <int MASK>
hipError_t launch_bwd(AttnArgs a, hipStream_t s) {
  plan_bwd_splits<MASK>(a);
  a.cus = (int)device_cus();
  switch (a.dtype) {
    case kF32: return run_dim<float, MASK>(a, s);
    case kF16: return run_dim<f16, MASK>(a, s);
    case kBF16: return run_dim<bf16, MASK>(a, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace
}  // namespace lwl
