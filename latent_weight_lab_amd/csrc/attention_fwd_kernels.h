// Attention forward: out = softmax(scale q k^T) v in one pass over the keys, the scores never leaving
// registers, with the running maximum and sum of a softmax.
//
// attention_rows: a workgroup of four waves takes 128 queries of one head, 32 a wave, and walks over
// the keys in tiles of 64 that the waves share through LDS.  Scores are computed transposed,
// S^T = K Q^T, so that a lane holds scores of one query only: the maximum over 32 keys and the sum
// need no exchange among lanes but one with the lane's other half, and the probabilities are, as
// they lie in the result registers, the operand of O^T = V^T P^T (both operands may number a product's
// k in any one order; V's columns are read by the transposing LDS read in the order in which P's
// registers come).  The output is divided by the sum at the end.
//
// attention_token: when the queries that share a key head are at most 16 (decoding), reading the
// cache is all the work.  Each wave takes 32 keys at a time straight from memory into operand
// registers (values through its own piece of LDS for the transposing read), without barriers, the
// next 32 keys' loads in flight.
//
// Where heads and rows give too few workgroups, ranges of keys are given to different workgroups,
// which leave normalized float32 outputs and log sums; attention_join weighs them.
//
// MASK says which pairs count (attention_device.h): all that lengths and causal order leave, a window, or a tree's.  Within
// a window a block of queries walks over the sinks' tiles and its windows' only (Walk).  A tree's block of rows are the
// nodes of all query heads that share a key head, so that the cache is read once for them, and its ranges are cut
// by the sequences' lengths (tree_share).
//
// What is subtracted from the scores is the maximum less kLift when it was last raised, and it is raised
// only for a score more than kSlack above that maximum: probabilities then stay below 2^(kLift +
// kSlack) = 2^14, the accumulators are rarely rescaled, and of float16's range the upper part is used, so
// that a probability 2^-20 of the largest keeps its digits.  The first value is -FLT_MAX, not -infinity, so
// that a row with no allowed key sums zeros: exp2(-inf + FLT_MAX) is 0 and nothing is NaN.
//
// 16-bit types: a probability is rounded to the type, half a step at most, as the operand of its product with the values;
// the sum that the output is divided by takes it as it was.
//
// Measured on MI355X: prompts are bound by the matrix cores and by what stands between their instructions, the
// exponentials (a quarter of the vector rate) and LDS reads: bfloat16 1 x 8192 x 16 on 4 x 128, causal, 297 us, 925
// TFLOP/s of the pairs needed, where a library product of 8192^3 runs at 1030; 8 x 1024 x 12 x 64 23 us, 560 TFLOP/s,
// two rounds of walks of unequal lengths.  Float32 4 x 512 x 12 x 64 22.6 us and 5.7 for the join.  Tokens are bound
// by memory: bfloat16 64 sequences of up to 1024 tokens x 12 x 64 19.6 us (101 MB, 5.2 TB/s), float32 38.3 us (202 MB,
// 5.3 TB/s); float16 2 x 65536 x 4 x 128 42.6 us (268 MB, 6.3 TB/s, in part from the last-level cache) and 4.6 for the
// join.  Windows: 1 x 16384 x 16 on 4 x 128, window 4096, 4 sinks 503 us, 957 TFLOP/s of the pairs needed; 64 tokens over up
// to 8192 x 12 x 64, window 1024, 39.5 us (188 MB, 4.8 TB/s).  Trees: 16 sequences of up to 8192 x 4 x 128, 32 nodes of 16
// heads, 38 us and 7.5 for the join (138 MB; one token over the same caches 40 us in all); 65536 x 2 x 128, 61 nodes of 16
// heads, 53 us and 7.4 (620 TFLOP/s: bound by the products).
#pragma once

#include <algorithm>
#include <cfloat>

#include "attention_device.h"

namespace lwl {
namespace {

constexpr float kLift = 6.0f, kSlack = 8.0f;
constexpr int kKeys = kTileRows;  // keys of a tile
constexpr int kWaveRows = 32;
constexpr int kWaves = 4;
constexpr int kRows = kWaves * kWaveRows;
constexpr int kHalvedRows = kRows / 2;  // of a tree, up to which waves halve the tiles

// LDS row lengths in (16-bit) elements.  Keys are read 16 bytes a lane, 16 lanes at a time from 16 rows: 16
// bytes of padding put these on distinct banks.  Values are read by columns: rows of 16 dwords more than a
// multiple of 32, so that a transposing read's four rows of 64 bytes fall on distinct banks.
template <int DP>
using KeyRows = Padded<DP>;
template <int DP>
using ValueRows = Strided<DP + ((DP / 32) % 2 ? 0 : 32)>;

// The nodes of a tree in the line of ancestors that ends in each, as bits, by doubling: after a round a node's bits go
// twice as far up.  All threads of the workgroup call it; lds: kMostNodes of both.
constexpr int kMostNodes = 128;
struct Line {
  uint64_t low, high;
};
__device__ __forceinline__ void tree_lines(const AttnArgs& a, int64_t b, Line* lines, int* above) {
  const int n = threadIdx.x;
  Line line = {n < 64 ? 1ull << (n & 63) : 0, n >= 64 ? 1ull << (n & 63) : 0};
  int up = n < (int)a.queries ? a.parents[b * a.parents_stride + n] : -1;
  if (up >= n) up = -1;
  if (n < kMostNodes) {
    lines[n] = line;
    above[n] = up;
  }
  for (int steps = 1; steps < (int)a.queries; steps *= 2) {
    __syncthreads();  // all have written
    if (up >= 0) {
      line.low |= lines[up].low;
      line.high |= lines[up].high;
      up = above[up];
    }
    __syncthreads();  // all have read
    if (n < kMostNodes) {
      lines[n] = line;
      above[n] = up;
    }
  }
  __syncthreads();
}
// Which of the 64 keys from the node's number `from` on (negative: keys before the tree) a line holds.
__device__ __forceinline__ uint64_t line_from(const Line& line, int from) {
  if (from <= -64) return ~0ull;
  if (from < 0) return line.low << -from | ((1ull << -from) - 1);
  if (from == 0) return line.low;
  if (from < 64) return line.low >> from | line.high << (64 - from);
  return from < 128 ? line.high >> (from - 64) : 0;
}

// How the sequences' caches are cut into a tree's ranges.  Only the device knows lengths, so the host gives a number of
// ranges for all sequences together, one for each and `spare` more, and these go to the sequences by their lengths: ranges
// of `per` tiles, the least number with which `spare` of them hold all tiles.  Lane b gets sequence b's first range
// and how many it has.
struct TreeShare {
  int first, count, per;
};
constexpr int kLeastTiles = 4;  // of a range
__device__ __forceinline__ TreeShare tree_share(const AttnArgs& a) {
  const int lane = threadIdx.x & 63, keys = (int)a.keys;
  int len = lane < (int)a.batch ? a.lengths[lane] : 0;
  len = len < 0 ? 0 : len < keys ? len : keys;
  const int tiles = (len + kKeys - 1) / kKeys;
  int total = tiles;
#pragma unroll
  for (int k = 1; k < 64; k *= 2) total += __shfl_xor(total, k, 64);
  total = uniform(total);
  TreeShare s;
  s.per = (int)(((uint32_t)total + a.spare - 1) / (uint32_t)a.spare);
  if (s.per < kLeastTiles) s.per = kLeastTiles;
  s.count = lane < (int)a.batch ? (int)((uint32_t)(tiles + s.per - 1) / (uint32_t)s.per) : 0;
  if (lane < (int)a.batch && s.count == 0) s.count = 1;  // writes zeros
  int last = s.count;
#pragma unroll
  for (int k = 1; k < 64; k *= 2) {
    const int before = __shfl_up(last, k, 64);
    if (lane >= k) last += before;
  }
  s.first = last - s.count;
  return s;
}

// A tree's work: range `slot`, keys begin .. end of sequence b.  Without lengths, and for batches of more than 64, every
// sequence has a.splits ranges of split_len keys.
struct TreeRange {
  bool any;
  int64_t b;
  int slot, begin, end;  // end: as far as the sequence goes
};
__device__ __forceinline__ TreeRange tree_range(const AttnArgs& a, int number) {
  TreeRange r = {false, 0, number, 0, 0};
  if (a.spare > 0) {
    const TreeShare s = tree_share(a);
    const uint64_t hit = __ballot(number >= s.first && number < s.first + s.count);
    if (hit == 0) return r;
    const int b = (int)__builtin_ctzll(hit), split = number - uniform(__shfl(s.first, b, 64));
    r.any = true;
    r.b = b;
    r.begin = split * s.per * kKeys;
    r.end = r.begin + s.per * kKeys;
  } else {
    const int rank = (int)((uint32_t)number / (uint32_t)a.splits), split = number - rank * a.splits;
    r.any = rank < (int)a.batch;
    if (!r.any) return r;
    r.b = ranked_sequence(a, rank);
    r.slot = (int)r.b * a.splits + split;
    r.begin = split * (int)a.split_len;
    r.end = r.begin + (int)a.split_len;
  }
  return r;
}
// A tree's rows are those of every query head that shares a key head, so that a workgroup reads the cache for all of
// them.  Where rows fill more than one block of 128, the blocks of a range go to the same die, one after the other.
struct TreeWork {
  TreeRange range;
  int hk, block;
};
__device__ __forceinline__ TreeWork tree_work(const AttnArgs& a) {
  const uint32_t kvh = (uint32_t)a.kv_heads;
  const uint32_t blocks = ((uint32_t)(a.heads / a.kv_heads) * (uint32_t)a.queries + kRows - 1) / kRows;
  uint32_t unit = blockIdx.x, block = 0;
  if (blocks > 1) {
    const uint32_t eight = unit / (8 * blocks), in = unit - eight * 8 * blocks;
    unit = eight * 8 + in % 8;
    block = in / 8;
  }
  const uint32_t slot = unit / kvh;
  TreeWork w;
  w.hk = uniform((int)(unit - slot * kvh));
  w.block = uniform((int)block);
  w.range = tree_range(a, uniform((int)slot));
  return w;
}
// Where range `slot` of key head hk leaves row r of it for the join: log sums follow all the outputs.
__host__ __device__ inline int64_t tree_rows(const AttnArgs& a) { return a.heads / a.kv_heads * a.queries; }
__device__ __forceinline__ int64_t tree_partial(const AttnArgs& a, int slot, int64_t hk, int64_t r) {
  return ((int64_t)slot * a.kv_heads + hk) * tree_rows(a) + r;
}

// HALVES of 2, for a tree's calls of at most 64 rows, which would leave half the waves without any: two waves hold the same
// 32 rows and take 32 keys of every tile each; their sums meet in LDS at the end.  us with the join, 1 and 2: float32
// 85810 tokens, 60 nodes, 12 heads of size 128 447 and 337, 16 sequences of up to 1024 x 12 x 64, 20 nodes 34.6 and 29.5; bfloat16,
// which memory bounds, 8 sequences of up to 8192 x 8 x 128, 32 nodes 44.1 and 42.5, 64 of up to 1024 x 12 x 64 27 and 26.6.
//
// Size 128 of 16-bit types takes all 256 registers that two waves a SIMD leave.  A tree's then keeps 52 to 68 bytes a thread in
// scratch, a window's 12 to 36, a call's without either 24 to 28 where rows are not FAST: what is set before the loop, of which
// masked tiles read some back, behind the next tile's loads.
template <class T, int DP, bool FAST, int MASK, int HALVES = 1>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void attention_rows(const AttnArgs a) {
  using KL = KeyRows<DP>;
  using VL = ValueRows<DP>;
  constexpr int KK = DP / 16, DT = DP / 32, KP = kKeys * KL::S, VP = kKeys * VL::S;  // sizes of a plane
  constexpr int MINE = kKeys / HALVES, TS = MINE / 32;                                // a wave's keys of a tile
  __shared__ __attribute__((aligned(16))) Elem<T> lds_k[kBufs<T>][kPlanes<T> * KP];
  __shared__ __attribute__((aligned(16))) Elem<T> lds_v[kBufs<T>][kPlanes<T> * VP];
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = uniform((int)threadIdx.x >> 6);
  int64_t b, hk, h;
  int block, split, tree_begin = 0, tree_end = 0;
  if constexpr (MASK == kTree) {
    const TreeWork w = tree_work(a);
    if (!w.range.any) return;
    b = w.range.b, hk = w.hk, h = 0, block = w.block, split = w.range.slot;
    tree_begin = w.range.begin, tree_end = w.range.end;
  } else {
    const RowsWork w = rows_work(a);
    b = w.b, hk = w.hk, h = w.h, block = w.block, split = w.split;
  }
  const int q0 = block * kRows;
  const int dim = (int)a.dim;
  const Allowed allow = allowed_keys(a, b);
  // a tree's rows: the nodes of the first of the heads that share the key head, then of the next
  const int queries = (int)a.queries, rows_here = MASK == kTree ? queries * (int)(a.heads / a.kv_heads) : queries;
  const int team = HALVES == 1 ? wave : wave & 1, first = HALVES == 1 ? 0 : (wave >> 1) * MINE;  // of a tile's keys
  const int wq0 = q0 + team * kWaveRows, wave_row = wq0 + (lane & 31);
  const bool live = wave_row < rows_here;
  int q = wave_row;
  if constexpr (MASK == kTree) {
    const int g = live ? wave_row / queries : 0;
    q = live ? wave_row - g * queries : 0;
    h = hk * (a.heads / a.kv_heads) + g;
  }
  const int q_end = live ? (MASK == kTree ? allow.len : key_end(allow, q)) : 0;  // this lane's query sees keys below
  const int q_begin = MASK == kWindow && live ? window_begin(allow, q) : 0;      // and, but for sinks, from here on
  const int base = allow.len - queries;                                          // of a tree's keys
  Walk<MASK, kKeys> at;
  if constexpr (MASK == kWindow) {
    at = window_walk<kKeys>(a, allow, q0, std::min(q0 + kRows, queries) - 1, split, 0);
  } else if constexpr (MASK == kTree) {
    at.j = std::min(tree_begin, allow.len);
    at.end = std::min(tree_end, allow.len);
  } else {
    at.j = std::min(split * (int)a.split_len, allow.len);
    at.end = std::min(key_end(allow, std::min(q0 + kRows, queries) - 1), at.j + (int)a.split_len);
  }
  const int end = at.end;
  // keys below free_end are seen by every query of the wave, keys from wave_end on by none; within a window also, but
  // for sinks, none below wave_begin, and not by every one those below free_begin
  int free_end = 0, wave_end = 0, wave_begin = 0, free_begin = 0;
  if (wq0 < rows_here) {
    if constexpr (MASK == kTree) {
      free_end = std::min(std::max(base, 0), end);
      wave_end = end;
    } else {
      free_end = std::min(key_end(allow, wq0), end);
      wave_end = std::min(key_end(allow, std::min(wq0 + kWaveRows, queries) - 1), end);
    }
    if constexpr (MASK == kWindow) {
      wave_begin = window_begin(allow, wq0);
      free_begin = window_begin(allow, std::min(wq0 + kWaveRows, queries) - 1);
    }
  }

  const T* qp = (const T*)a.q + b * a.qs[0] + h * a.qs[1];
  const T* kp = (const T*)a.k + b * a.ks[0] + hk * a.ks[1];
  const T* vp = (const T*)a.v + b * a.vs[0] + hk * a.vs[1];
  Opd<T> qf[KK];
  load_operand<T, DP, FAST>(qf, qp + (int64_t)q * a.qs[2], dim, live);
  f32x16 o[DT] = {};
  float top = -FLT_MAX, sum = 0.0f;  // subtracted, in units of log2; sum of this lane's half of the keys
  const float c = a.scale * kLog2E;

  // one tile's products in LDS while the next one's loads are under way, a barrier a tile
  TileLoader<T, DP, FAST> kt, vt;
  kt.init(kp, a.ks[2], dim, (int)a.keys);
  vt.init(vp, a.vs[2], dim, (int)a.keys);
  if (at.live()) {
    kt.fetch(at.j, at.stop());
    vt.fetch(at.j, at.stop());
  }
  Line line = {};
  if constexpr (MASK == kTree) {
    __shared__ Line lds_lines[kMostNodes];
    __shared__ int lds_above[kMostNodes];
    if (end > std::max(base, 0)) {  // this range holds nodes' keys
      tree_lines(a, b, lds_lines, lds_above);
      line = lds_lines[q];
    }
  }
  if (at.live()) {
    if constexpr (kBufs<T> == 2) {
      kt.template put<KL>(lds_k[0]);
      vt.template put<VL>(lds_v[0]);
    }
  }
  wait_operands<T, FAST>(qf);
  int buf = 0;
  for (; at.live(); at.step(), buf ^= kBufs<T> - 1) {
    const int j0 = at.j;
    __syncthreads();  // this tile is there, the one before has been read
    if constexpr (kBufs<T> == 1) {
      kt.template put<KL>(lds_k[0]);
      vt.template put<VL>(lds_v[0]);
      __syncthreads();
    }
    const bool more = at.more();
    if (more) {
      kt.fetch(at.next(), at.next_stop());
      vt.fetch(at.next(), at.next_stop());
    }
    if (j0 < wave_end && (MASK != kWindow || j0 + kKeys > wave_begin || j0 < allow.sinks)) {
      const Elem<T>* lk = lds_k[buf] + KL::at(first + (lane & 31), half * 8);
      const Elem<T>* lv = lds_v[buf];
      f32x16 s[TS] = {};
      {
        Opd<T> kf[TS][KK];
        if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int t = 0; t < TS; ++t) kf[t][kk] = lds_operand<T>(lk + t * 32 * KL::S + kk * 16, KP);
          fence_schedule<T>();
        }
        if constexpr (DP > 64) __builtin_amdgcn_s_setprio(1);  // 1 x 8192 x 16 x 128: 548 -> 529 us; slower at 64
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
#pragma unroll
          for (int t = 0; t < TS; ++t) {
            if constexpr (sizeof(T) == 4) kf[t][kk] = lds_operand<T>(lk + t * 32 * KL::S + kk * 16, KP);
            s[t] = mma32(kf[t][kk], qf[kk], s[t]);
          }
          fence_operands<T>();
        }
        if constexpr (DP > 64) __builtin_amdgcn_s_setprio(0);
      }
      Opd<T> vf[TS * 2][DT];
      const auto load_v = [&](int u, int d) {
        const int key = first + u * 16 + half * 4;
        vf[u][d] = lds_column_operand<T, VL>(lv, VP, key, key + 8, d * 32 + (lane & 16));
      };
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int u = 0; u < TS * 2; ++u)
#pragma unroll
          for (int d = 0; d < DT; ++d) load_v(u, d);
        fence_schedule<T>();
      }
      if constexpr (MASK == kWindow) {
        if (j0 + kKeys > std::min(free_end, at.stop()) || (j0 < free_begin && std::min(j0 + kKeys, at.stop()) > allow.sinks)) {
          const Seen seen = seen_keys(j0, std::min(q_end, at.stop()), q_begin, allow.sinks);
#pragma unroll
          for (int t = 0; t < TS; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[t][r] = masked_score(s[t][r], bit_mask(seen.w[t], (r >> 2) * 8 + (r & 3)));
        }
      } else if (j0 + kKeys > free_end) {
        const int lim = std::min(q_end, end) - j0 - first - half * 4;
        uint64_t bits = 0;
        if constexpr (MASK == kTree) bits = line_from(line, j0 + first - base);
#pragma unroll
        for (int t = 0; t < TS; ++t) {
          const uint32_t seen = (uint32_t)(bits >> (t * 32)) >> (half * 4);
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int n = t * 32 + (r >> 2) * 8 + (r & 3);
            const bool ok = n < lim && (MASK != kTree || (seen >> (n & 31) & 1));
            s[t][r] = ok ? s[t][r] : -INFINITY;
          }
        }
      }
      float most = s[0][0];
#pragma unroll
      for (int t = 0; t < TS; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) most = max_nan(most, s[t][r]);
      most = max_halves(most) * c;
      if (__any(most > top + (kLift + kSlack))) {
        const float next = fmaxf(top, most - kLift), shrink = exp2_hw(top - next);
        top = next;
        sum *= shrink;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] *= shrink;
      }
#pragma unroll
      for (int u = 0; u < TS * 2; ++u) {
        float e[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          e[r] = exp2_hw(fmaf(s[u >> 1][(u & 1) * 8 + r], c, -top));
          sum += e[r];
        }
        const Opd<T> p = operand_of<T>(e);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          if constexpr (sizeof(T) == 4) load_v(u, d);
          o[d] = mma32(vf[u][d], p, o[d]);
        }
        fence_operands<T>();
      }
    }
    if (kBufs<T> == 2 && more) {
      kt.template put<KL>(lds_k[buf ^ (kBufs<T> - 1)]);
      vt.template put<VL>(lds_v[buf ^ (kBufs<T> - 1)]);
    }
  }
  if constexpr (HALVES == 2) {
    // The second half's waves leave theirs where keys and values were.
    __syncthreads();
    float* theirs = (float*)&lds_k[0][0] + team * DT * 16 * 64 + lane;
    float* stat = (float*)&lds_v[0][0] + team * 2 * 64 + lane;
    static_assert(sizeof(lds_k) >= 2 * DT * 16 * 64 * sizeof(float) && sizeof(lds_v) >= 4 * 64 * sizeof(float), "");
    if (first > 0) {
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) theirs[(d * 16 + r) * 64] = o[d][r];
      stat[0] = top;
      stat[64] = sum;
    }
    __syncthreads();
    if (first > 0) return;
    const float next = fmaxf(top, stat[0]), mine = exp2_hw(top - next), other = exp2_hw(stat[0] - next);
    top = next;
    sum = sum * mine + stat[64] * other;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = o[d][r] * mine + theirs[(d * 16 + r) * 64] * other;
  }
  sum += other_half(sum);
  if (!live) return;
  const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
  const float lse = sum > 0.0f ? top + log2_hw(sum) : (sum == 0.0f ? -INFINITY : sum);
  const int64_t row = (b * a.heads + h) * a.queries + q;
  const int64_t rows = MASK == kTree ? a.kv_heads * tree_rows(a) : a.batch * a.heads * a.queries;
  const bool ranges = MASK == kTree ? a.slots > a.batch : a.splits > 1;
  if (ranges) {
    const int64_t part = MASK == kTree ? tree_partial(a, split, hk, wave_row) : row * a.splits + split;
    if (half == 0) a.work[rows * (MASK == kTree ? a.slots : a.splits) * dim + part] = lse;
    if (MASK != kAll && lse == -INFINITY) return;  // the join does not read it
    store_result<float, DP, FAST>(a.work + part * dim, o, inv, dim);
    return;
  }
  if (a.lse && half == 0) a.lse[row] = lse * kLn2;
  store_result<T, DP, FAST>((T*)a.out + b * a.os[0] + h * a.os[1] + (int64_t)q * a.os[2], o, inv, dim);
}

// ---------------------------------------------------------------- few queries
// Queries times heads that share a key head: the columns of one product.  More of them take attention_rows, where a
// workgroup holds one query head and each reads the cache for itself: bfloat16 8 sequences of 8192 tokens of size 128, 16
// heads on one 10.8 us and 3.9 for the join, 32 heads on one 146 us; 8 heads on one with 4 tokens each 34 and 4.6 us.
constexpr int kTokenRows = 16;
constexpr int kStep = 32;       // keys of a wave's step

template <class T, int DP, bool WHOLE, int MASK>
__global__ __launch_bounds__(256) void attention_token(const AttnArgs a) {
  constexpr int KK = DP / 32, DT = DP / 16, CPR = DP / 8, PER = kStep * CPR / 64;
  // values' rows: 16-bit 8 dwords more than a multiple of 16 (a transposing read's eight rows of 32
  // bytes on distinct banks), float32 4 more
  constexpr int VS = sizeof(T) == 2 ? DP + 16 : DP + 4;
  constexpr int kTileBytes = kStep * VS * (int)sizeof(T);
  constexpr int kJoinBytes = kTokenRows * (DP + 4) * 4;
  constexpr int kWaveBytes = kTileBytes > kJoinBytes ? kTileBytes : kJoinBytes;
  __shared__ __attribute__((aligned(16))) unsigned char lds[kWaves * kWaveBytes];
  __shared__ float lds_stat[kWaves][2][kTokenRows];
  const int lane = threadIdx.x & 63, quad = lane >> 4, wave = uniform((int)threadIdx.x >> 6);
  T* lds_v = reinterpret_cast<T*>(lds + wave * kWaveBytes);
  const uint32_t kvh = (uint32_t)a.kv_heads, batch = (uint32_t)a.batch;
  const uint32_t id = a.lengths ? work_order(blockIdx.x, gridDim.x, (uint32_t)a.cus) : blockIdx.x;
  const int group = uniform((int)((uint32_t)a.heads / kvh));
  const int64_t hk = uniform((int)(id % kvh));
  int64_t b;
  int split, tree_begin = 0, tree_end = 0;
  if constexpr (MASK == kTree) {
    const TreeRange r = tree_range(a, uniform((int)(id / kvh)));
    if (!r.any) return;
    b = r.b, split = r.slot, tree_begin = r.begin, tree_end = r.end;
  } else {
    b = ranked_sequence(a, uniform((int)(id / kvh % batch)));
    split = uniform((int)(id / kvh / batch));
  }
  const int dim = (int)a.dim, queries = (int)a.queries, rows_here = group * queries;
  const Allowed allow = allowed_keys(a, b);
  const int row = lane & 15;  // this lane's column of the products: query row % queries of head row / queries
  const bool live = row < rows_here;
  const int g = live ? row / queries : 0, qi = live ? row % queries : 0;
  const int64_t h = hk * group + g;
  const int q_end = live ? (MASK == kTree ? allow.len : key_end(allow, qi)) : 0;
  const int q_begin = MASK == kWindow && live ? window_begin(allow, qi) : 0;
  const int base = allow.len - queries;
  Walk<MASK, kStep, kWaves> at;
  if constexpr (MASK == kWindow) {
    at = window_walk<kStep, kWaves>(a, allow, 0, queries - 1, split, wave);
  } else if constexpr (MASK == kTree) {
    at.j = std::min(tree_begin, allow.len) + wave * kStep;
    at.end = std::min(tree_end, allow.len);
  } else {
    const int begin = std::min(split * (int)a.split_len, allow.len);
    at.j = begin + wave * kStep;
    at.end = std::min(key_end(allow, queries - 1), begin + (int)a.split_len);
  }
  const T* kp = (const T*)a.k + b * a.ks[0] + hk * a.ks[1];
  const T* vp = (const T*)a.v + b * a.vs[0] + hk * a.vs[1];
  const T* qp = (const T*)a.q + b * a.qs[0] + h * a.qs[1] + qi * a.qs[2];
  Frag<T> qf[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) {
    const int col = kk * 32 + quad * 8;
    Raw8<T> r;
    load_raw8(r, qp + col, live ? dim - col : 0);
    qf[kk] = frag_of(r);
  }
  // of key j; zeros where not ok.  What a key's row reads past it is cleared before the product, a value's
  // makes columns that are not stored.
  const int keys = (int)a.keys;
  auto load8_or = [&](Raw8<T>& r, const T* p, int64_t stride, int j, bool ok, int left) {
    if constexpr (WHOLE) load_whole8(r, p, ok && left > 0);
    else load_ahead8(r, p, ok ? left : 0, stride >= 8 && j + 1 < keys);
  };
  Raw8<T> kr[2][KK], vr[PER];
  auto fetch = [&](int j0, int end) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const int j = j0 + t * 16 + row, col = kk * 32 + quad * 8;
        load8_or(kr[t][kk], kp + (int64_t)j * a.ks[2] + col, a.ks[2], j, j < end, dim - col);
      }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int cc = lane + i * 64, j = j0 + cc / CPR, col = (cc % CPR) * 8;
      load8_or(vr[i], vp + (int64_t)j * a.vs[2] + col, a.vs[2], j, j < end, dim - col);
    }
  };
  f32x4 o[DT] = {};
  float top = -FLT_MAX, sum = 0.0f;
  const float c = a.scale * kLog2E;
  if (at.live()) fetch(at.j, at.stop());
  uint32_t line = 0;  // of a tree (of 16 nodes at most): the nodes that this column's sees, found as in tree_lines
  if constexpr (MASK == kTree) {
    line = 1u << row;
    int up = row < queries ? a.parents[b * a.parents_stride + row] : -1;
    if (up >= row) up = -1;
#pragma unroll
    for (int n = 1; n < kTokenRows; n *= 2) {
      const int from = up < 0 ? row : up;
      const uint32_t theirs = __shfl(line, from, 64);
      const int next = __shfl(up, from, 64);
      line |= theirs;
      up = up < 0 ? -1 : next;
    }
    line = __shfl(line, qi, 64);
  }
  for (; at.live(); at.step()) {
    const int j0 = at.j;
    f32x4 s[2] = {};
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        if constexpr (!WHOLE) keep8(kr[t][kk], dim - kk * 32 - quad * 8);
        s[t] = mma16(frag_of(kr[t][kk]), qf[kk], s[t]);
      }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int cc = lane + i * 64;
      lds_put(lds_v + (cc / CPR) * VS + (cc % CPR) * 8, vr[i]);
    }
    if (at.more()) fetch(at.next(), at.next_stop());
    const int lim = std::min(q_end, at.stop()) - j0 - quad * 4;
    const int from = q_begin - j0 - quad * 4, sinks = allow.sinks - j0 - quad * 4;
    uint32_t seen = ~0u;
    if constexpr (MASK == kTree) seen = (uint32_t)line_from({line, 0}, j0 - base) >> (quad * 4);
    float most = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int n = t * 16 + r;
        bool ok = n < lim;
        if constexpr (MASK == kWindow) ok = ok && (n >= from || n < sinks);
        if constexpr (MASK == kTree) ok = ok && (seen >> n & 1);
        if (!ok) s[t][r] = -INFINITY;
        most = fmaxf(most, s[t][r]);
      }
    most = fmaxf(most, __shfl_xor(most, 16, 64));
    most = fmaxf(most, __shfl_xor(most, 32, 64)) * c;
    if (__any(most > top + (kLift + kSlack))) {
      const float next = fmaxf(top, most - kLift), shrink = exp2_hw(top - next);
      top = next;
      sum *= shrink;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= shrink;
    }
    Frag<T> p;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float e = exp2_hw(fmaf(s[t][r], c, -top));
        sum += e;
        p[t * 4 + r] = (T)e;
      }
    // the wave's own writes: its LDS accesses are performed in order
    asm volatile("" ::: "memory");
#pragma unroll
    for (int d = 0; d < DT; ++d)
      o[d] = mma16(lds_column_frag<Strided<VS>>(lds_v, quad * 4, quad * 4 + 16, d * 16), p, o[d]);
    asm volatile("" ::: "memory");
  }
  sum += __shfl_xor(sum, 16, 64);
  sum += __shfl_xor(sum, 32, 64);
  // join the four waves
  __syncthreads();
  float* mine = reinterpret_cast<float*>(lds + wave * kWaveBytes);
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r) mine[row * (DP + 4) + d * 16 + quad * 4 + r] = o[d][r];
  if (quad == 0) {
    lds_stat[wave][0][row] = top;
    lds_stat[wave][1][row] = sum;
  }
  __syncthreads();
  const int64_t rows = MASK == kTree ? a.kv_heads * tree_rows(a) : a.batch * a.heads * a.queries;
  const bool ranges = MASK == kTree ? a.slots > a.batch : a.splits > 1;
  for (int i = threadIdx.x; i < rows_here * DP; i += 256) {
    const int rr = i / DP, col = i % DP;
    float m = lds_stat[0][0][rr];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) m = fmaxf(m, lds_stat[w][0][rr]);
    float total = 0.0f, v = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = exp2_hw(lds_stat[w][0][rr] - m);
      total += f * lds_stat[w][1][rr];
      v += f * reinterpret_cast<const float*>(lds + w * kWaveBytes)[rr * (DP + 4) + col];
    }
    v = total > 0.0f ? v / total : (total == 0.0f ? 0.0f : total);
    const float lse = total > 0.0f ? m + log2_hw(total) : (total == 0.0f ? -INFINITY : total);
    const int64_t hh = hk * group + rr / queries, qq = rr % queries, out_row = (b * a.heads + hh) * queries + qq;
    if (col >= dim) continue;
    if (ranges) {
      const int64_t part = MASK == kTree ? tree_partial(a, split, hk, rr) : out_row * a.splits + split;
      if (MASK == kAll || lse != -INFINITY) a.work[part * dim + col] = v;
      if (col == 0) a.work[rows * (MASK == kTree ? a.slots : a.splits) * dim + part] = lse;
    } else {
      ((T*)a.out)[b * a.os[0] + hh * a.os[1] + qq * a.os[2] + col] = (T)v;
      if (a.lse && col == 0) a.lse[out_row] = lse * kLn2;
    }
  }
}

// The ranges' outputs weighed by their sums: a thread joins eight values of a row, its chunk, and computes the
// weights for itself.  Where there are few ranges every thread of a workgroup has another chunk (kSplitsAlone);
// where there are many the workgroup has 16 chunks or fewer, one row's, and its SHARE = 16 threads of a chunk take every
// 16th range each and add up through LDS in their order.
constexpr int kMaxSplits = 512, kSplitsAlone = 16;
template <class T, int SHARE, int MASK>
__global__ __launch_bounds__(256) void attention_join(const AttnArgs a) {
  constexpr int CHUNKS = 256 / SHARE;
  static_assert(CHUNKS * 8 >= kAttnMaxDim);
  __shared__ float lds_v[SHARE][CHUNKS][8], lds_m[SHARE][CHUNKS], lds_t[SHARE][CHUNKS];
  const int dim = (int)a.dim, per_row = (dim + 7) / 8;
  const uint32_t rows_wg = CHUNKS / per_row, rows = (uint32_t)(a.batch * a.heads * a.queries);
  const int part_no = threadIdx.x / CHUNKS, chunk = threadIdx.x % CHUNKS, r = chunk / per_row;
  const int col = (chunk - r * per_row) * 8;
  const uint32_t row = blockIdx.x * rows_wg + r;
  const bool live = (uint32_t)r < rows_wg && row < rows;
  int splits = a.splits;
  int64_t first = (int64_t)(live ? row : 0) * splits, step = 1, all = (int64_t)rows * splits;  // partial rows
  if constexpr (MASK == kTree) {
    const uint32_t head_row = live ? row : 0, q = head_row % (uint32_t)a.queries, head = head_row / (uint32_t)a.queries;
    const uint32_t group = (uint32_t)(a.heads / a.kv_heads), b = head / (uint32_t)a.heads, h = head - b * (uint32_t)a.heads;
    int slot = (int)b * splits;
    if (a.spare > 0) {
      const TreeShare s = tree_share(a);
      slot = __shfl(s.first, (int)b, 64);
      splits = __shfl(s.count, (int)b, 64);
    }
    first = tree_partial(a, slot, h / group, (int64_t)(h % group) * a.queries + q);
    step = a.kv_heads * tree_rows(a);
    all = step * a.slots;
  }
  const float* lses = a.work + all * dim + first;
  const float* part = a.work + first * dim + col;
  float m = -FLT_MAX, total = 0.0f, v[8] = {};
#pragma unroll 8  // one after the other, 130 ranges took 30 us, so 18
  for (int s = part_no; s < splits; s += SHARE) m = max_nan(m, lses[s * step]);
  if constexpr (SHARE > 1) {
    lds_m[part_no][chunk] = m;
    __syncthreads();
#pragma unroll
    for (int g = 0; g < SHARE; ++g) m = max_nan(m, lds_m[g][chunk]);
  }
  if (live) {
#pragma unroll 4
    for (int s = part_no; s < splits; s += SHARE) {
      float x[8];
      load8(x, part + s * step * dim, dim - col);
      const float w = exp2_hw(lses[s * step] - m);  // 0 for a range that holds nothing
      if constexpr (MASK != kAll) {                 // whose output is not written
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = w > 0.0f ? x[i] : 0.0f;
      }
      total += w;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += w * x[i];
    }
  }
  if constexpr (SHARE > 1) {
    lds_t[part_no][chunk] = total;
#pragma unroll
    for (int i = 0; i < 8; ++i) lds_v[part_no][chunk][i] = v[i];
    __syncthreads();
    total = 0.0f;
#pragma unroll
    for (int g = 0; g < SHARE; ++g) total += lds_t[g][chunk];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = 0.0f;
#pragma unroll
      for (int g = 0; g < SHARE; ++g) v[i] += lds_v[g][chunk][i];
    }
  }
  if (!live || part_no != 0) return;
  const uint32_t queries = (uint32_t)a.queries, heads = (uint32_t)a.heads, bh = row / queries, q = row - bh * queries;
  const int64_t b = bh / heads, h = bh % heads;
  const float inv = total > 0.0f ? 1.0f / total : (total == 0.0f ? 0.0f : total);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= inv;
  store8((T*)a.out + b * a.os[0] + h * a.os[1] + (int64_t)q * a.os[2] + col, v, dim - col);
  if (a.lse && col == 0)
    a.lse[row] = total > 0.0f ? (m + log2_hw(total)) * kLn2 : (total == 0.0f ? -INFINITY : total);
}


inline bool by_token(const AttnArgs& a) { return a.heads / a.kv_heads * a.queries <= kTokenRows; }
inline int64_t tree_blocks(const AttnArgs& a) { return (a.heads / a.kv_heads * a.queries + kRows - 1) / kRows; }

// Ranges of keys.  Single tokens: as many as make two workgroups for each compute unit, none shorter than
// 256 keys.  Otherwise what an estimate of the time makes shortest, in us: the larger of a workgroup's
// own walk (`alone` a tile, and as much as a tile before its first) and all work spread over the compute units
// (`spread` a tile), and with more than one range the join.  The rates are measured on MI355X: bfloat16 of head
// size 64, 0.7 us a tile when a compute unit has three workgroups and 1 us alone; float32 2.9 and 3.3 us.
// 4 x 512 x 12 x 64 in float32: 1, 2, 3, 4 ranges 31.8, 27.2, 30.4, 31.0 us with the join, 2 are taken;
// float16 6 x 515 over up to 1531 keys x 12 x 80: 34.4, 37.4, 44.0, 47.7 us, 1 is taken.
template <int MASK>
void plan_splits(AttnArgs& a) {
  const int64_t cus = device_cus();
  int64_t splits = 1;
  // keys of the longest walk
  const int64_t keys = MASK == kWindow ? window_tiles(a, kRows) * kKeys : a.keys;
  if (by_token(a)) {
    const int64_t wgs = std::max<int64_t>(1, a.batch * a.kv_heads);
    splits = std::min({2 * cus / wgs, keys / 256, (int64_t)kMaxSplits});
  } else {
    const double unit = (double)((a.dim + 31) / 32 * 32) / 64;
    const double alone = a.dtype == kF32 ? 3.3 * unit : 0.5 + 0.5 * unit, spread = (a.dtype == kF32 ? 2.9 : 0.7) * unit;
    const int64_t tiles = (keys + kKeys - 1) / kKeys;
    const double wgs = (double)(a.batch * a.heads) * (double)((a.queries + kRows - 1) / kRows);
    // about half of a square causal call's tiles are walked
    // (also of ragged sequences' tiles, whose lengths only the device knows)
    // but not of a window's
    const bool half = MASK != kWindow || keys >= a.keys;
    const double walked = (double)tiles * (half && ((a.causal && a.queries * 2 > a.keys) || a.lengths) ? 0.55 : 1.0);
    const double bytes = 8.0 * (double)(a.batch * a.heads) * (double)a.queries * (double)a.dim;  // of a range
    double best = 0.0;
    for (int64_t n = 1; n <= std::min<int64_t>(tiles / 4 + 1, kMaxSplits); n = n < 4 ? n + 1 : n + n / 4) {
      const double walk = (double)((tiles + n - 1) / n + 1) * alone;
      const double all = wgs * ((double)n + walked) * spread / (double)cus;
      const double t = std::max(walk, all) + (n > 1 ? 2.5 + (double)n * bytes / 9e6 : 0.0);
      // several only where they gain more than the estimate may be off by
      if (n == 1 || t < best * (splits == 1 ? 0.85 : 1.0)) {
        best = t;
        splits = n;
      }
    }
  }
  splits = std::max<int64_t>(1, splits);
  a.split_len = splits > 1 ? ((keys + splits - 1) / splits + kKeys - 1) / kKeys * kKeys : std::max<int64_t>(keys, 1);
  a.splits = splits > 1 ? (int)((keys + a.split_len - 1) / a.split_len) : 1;
}

// A tree's ranges (tree_share): as many as make one workgroup for each compute unit, for a workgroup leaves up to 128 rows
// of float32 outputs however short its range.  Two where one would leave sequences whole, for single tokens' kernel, and
// where rows are short or at most 64 and ranges still long; no more than 256 of a sequence on average, for the join (one that
// is longer than the others may have more: to hold that, too, took 0.3 us of every call).  Where sequences alone are as many,
// none is cut.  us with the join, one and two workgroups; bfloat16: 16 sequences of up to 8192 tokens, 32
// nodes, 16 heads on 4 of size 128 51 and 55 (uncut 161), of size 64 31 and 30; 8 of up to 8192 x 8 x 128, 32 nodes 42 and 38;
// 2 of 8192 x 12 x 64, 60 nodes, ranges of 6 tiles 17.4 and 18.4; 64 x 12 sequences and heads of up to 1024 tokens of size 64, 20
// nodes, uncut 27, cut 34.  Float16: 65536 tokens, 61 nodes, 16 heads on 2 of size 128 60 and 60; 2 x 64208, 67 nodes, 32 heads
// on 8 of size 32 146 and 101 to 117.  Float32: 2 x 16384 x 8 x 96, 40 nodes, ranges of 8 tiles 73 and 66.  131072 tokens, 32
// nodes, 4 heads on 1 of size 64, 256 ranges 23, 512 31.
inline void plan_tree(AttnArgs& a) {
  const int64_t cus = device_cus(), units = std::max<int64_t>(1, a.kv_heads * tree_blocks(a)), batch = a.batch;
  const int64_t tiles = (a.keys + kKeys - 1) / kKeys;
  a.splits = 1;
  a.spare = 0;
  a.split_len = std::max<int64_t>(a.keys, 1);
  const bool few = a.dim <= 64 || tree_rows(a) <= kHalvedRows;
  const bool lasting = tiles * batch * units >= (a.dtype == kF32 ? 8 : 12) * 2 * cus;  // a float32 tile takes longer
  int64_t ranges = (by_token(a) || (few && lasting) ? 2 : 1) * cus / units;
  if (ranges < 2 * batch) ranges = 2 * cus / units;
  if (!by_token(a)) ranges = std::min(ranges, 256 * batch);
  if (batch > 0 && ranges >= 2 * batch && tiles >= 2 * kLeastTiles) {
    if (a.lengths && batch <= kMostRanked) {
      // no more than there are tiles for; sequences' own come on top
      a.spare = (int)std::min(ranges - batch, batch * ((tiles + kLeastTiles - 1) / kLeastTiles));
    } else {
      const int64_t per = std::max<int64_t>(kLeastTiles, (tiles + ranges / batch - 1) / (ranges / batch));
      a.splits = (int)((tiles + per - 1) / per);
      a.split_len = per * kKeys;
    }
  }
  a.slots = (int)(a.spare > 0 ? batch + a.spare : batch * a.splits);
}
// The most ranges that one of a tree's sequences can have.
inline int64_t tree_most(const AttnArgs& a) {
  if (a.spare == 0) return a.splits;
  const int64_t tiles = (a.keys + kKeys - 1) / kKeys;
  return std::min<int64_t>(a.spare + 1, (tiles + kLeastTiles - 1) / kLeastTiles);
}
template <int MASK>
void plan(AttnArgs& a) {
  if constexpr (MASK == kTree) plan_tree(a);
  else plan_splits<MASK>(a);
}

// Workgroups of a planned call.  (The join has fewer: ranges are only where these are few.)
template <int MASK>
int64_t workgroups(const AttnArgs& a) {
  if (by_token(a)) return a.kv_heads * (MASK == kTree ? (int64_t)a.slots : a.batch * a.splits);
  if (MASK != kTree) return a.batch * a.heads * a.splits * ((a.queries + kRows - 1) / kRows);
  const int64_t units = a.kv_heads * a.slots, blocks = tree_blocks(a);
  return blocks == 1 ? units : (units + 7) / 8 * 8 * blocks;
}
template <int MASK>
bool fwd_fits(AttnArgs a) {
  // a block of queries has no more than kMaxSplits ranges
  if (a.batch * a.heads * ((a.queries + kRows - 1) / kRows) <= kMostWorkgroups / 1024) return true;
  plan<MASK>(a);
  return workgroups<MASK>(a) <= kMostWorkgroups;
}

template <class T, int DP, int MASK>
hipError_t run(const AttnArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)workgroups<MASK>(a));
  if (by_token(a)) {
    if (a.dim % 8 == 0) hipLaunchKernelGGL((attention_token<T, DP, true, MASK>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((attention_token<T, DP, false, MASK>), grid, dim3(256), 0, s, a);
  } else {
    const bool fast = a.dim % 8 == 0 && fast_rows(a.k, a.ks, sizeof(T)) && fast_rows(a.v, a.vs, sizeof(T));
    const auto launch = [&](auto halves) {
      constexpr int H = decltype(halves)::value;
      if (fast) hipLaunchKernelGGL((attention_rows<T, DP, true, MASK, H>), grid, dim3(256), 0, s, a);
      else hipLaunchKernelGGL((attention_rows<T, DP, false, MASK, H>), grid, dim3(256), 0, s, a);
    };
    if constexpr (MASK == kTree) {
      if (tree_rows(a) <= kHalvedRows) launch(std::integral_constant<int, 2>{});
      else launch(std::integral_constant<int, 1>{});
    } else {
      launch(std::integral_constant<int, 1>{});
    }
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !(MASK == kTree ? a.slots > a.batch : a.splits > 1)) return e;
  const int64_t rows = a.batch * a.heads * a.queries;
  const int64_t per_row = (a.dim + 7) / 8, ranges = MASK == kTree ? a.slots / a.batch : a.splits;
  const auto joins = [&](int64_t chunks) { return dim3((unsigned)((rows + chunks / per_row - 1) / (chunks / per_row))); };
  // Threads for a chunk of a row.  A tree's ranges of 4 for each, where 1024 workgroups hold them: 4096 rows of size 128 with
  // 8 ranges 7.1, 5.6 and 15 us with 1, 4 and 16, 976 rows with 64 ranges 29, 12 and 11, 8192 rows with 4 ranges 7.6, 9.2 and 37.
  // With lengths a sequence may have many more than the average: 16 where some may have more than 32 and as many
  // workgroups hold them.  bfloat16, us by the average and by the most: 64 sequences of 32 rows, one of 65536 tokens, the others
  // 60, 17.6 and 8.2; 4 of 256 rows, one of 131072, 15 and 10; all four of 131072 8.5 and 10.7; 16 of 32, all of 30000, 7.9 and 5.6.
  if constexpr (MASK == kTree) {
    if (tree_most(a) > 2 * kSplitsAlone && joins(16).x <= 1024) {
      hipLaunchKernelGGL((attention_join<T, 16, MASK>), joins(16), dim3(256), 0, s, a);
      return hipGetLastError();
    }
    if (ranges >= 4 && ranges <= 2 * kSplitsAlone && joins(64).x <= 1024) {
      hipLaunchKernelGGL((attention_join<T, 4, MASK>), joins(64), dim3(256), 0, s, a);
      return hipGetLastError();
    }
  }
  if (ranges > kSplitsAlone)
    hipLaunchKernelGGL((attention_join<T, 16, MASK>), joins(16), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((attention_join<T, 1, MASK>), joins(256), dim3(256), 0, s, a);
  return hipGetLastError();
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

template <int MASK>
int64_t fwd_work(AttnArgs a) {
  plan<MASK>(a);
  if (MASK == kTree) return a.slots > a.batch ? (int64_t)a.slots * a.kv_heads * tree_rows(a) * (a.dim + 1) : 0;
  return a.splits > 1 ? (int64_t)a.splits * a.batch * a.heads * a.queries * (a.dim + 1) : 0;
}
template <int MASK>
hipError_t launch_fwd(AttnArgs a, hipStream_t s) {
  plan<MASK>(a);
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
