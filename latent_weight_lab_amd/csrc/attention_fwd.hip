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
// What is subtracted from the scores is the maximum less kLift when it was last raised, and it is raised
// only for a score more than kSlack above that maximum: probabilities then stay below 2^(kLift +
// kSlack) = 2^14, the accumulators are rarely rescaled, and of float16's range the upper part is used, so
// that a probability 2^-20 of the largest keeps its digits.  The first value is -FLT_MAX, not -infinity, so
// that a row with no allowed key sums zeros: exp2(-inf + FLT_MAX) is 0 and nothing is NaN.
//
// Measured on MI355X: prompts are bound by the matrix cores and by what stands between their instructions, the
// exponentials (a quarter of the vector rate) and LDS reads: bfloat16 1 x 8192 x 16 on 4 x 128, causal, 297 us, 925
// TFLOP/s of the pairs needed, where a library product of 8192^3 runs at 1030; 8 x 1024 x 12 x 64 23 us, 560 TFLOP/s,
// two rounds of walks of unequal lengths.  Float32 4 x 512 x 12 x 64 22.6 us and 5.7 for the join.  Tokens are bound
// by memory: bfloat16 64 sequences of up to 1024 tokens x 12 x 64 19.6 us (101 MB, 5.2 TB/s), float32 38.3 us (202 MB,
// 5.3 TB/s); float16 2 x 65536 x 4 x 128 42.6 us (268 MB, 6.3 TB/s, in part from the last-level cache) and 4.6 for the
// join.
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

// LDS row lengths in (16-bit) elements.  Keys are read 16 bytes a lane, 16 lanes at a time from 16 rows: 16
// bytes of padding put these on distinct banks.  Values are read by columns: rows of 16 dwords more than a
// multiple of 32, so that a transposing read's four rows of 64 bytes fall on distinct banks.
template <int DP>
using KeyRows = Padded<DP>;
template <int DP>
using ValueRows = Strided<DP + ((DP / 32) % 2 ? 0 : 32)>;

template <class T, int DP, bool FAST>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void attention_rows(const AttnArgs a) {
  using KL = KeyRows<DP>;
  using VL = ValueRows<DP>;
  constexpr int KK = DP / 16, DT = DP / 32, KP = kKeys * KL::S, VP = kKeys * VL::S;  // sizes of a plane
  __shared__ __attribute__((aligned(16))) Elem<T> lds_k[kBufs<T>][kPlanes<T> * KP];
  __shared__ __attribute__((aligned(16))) Elem<T> lds_v[kBufs<T>][kPlanes<T> * VP];
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = uniform((int)threadIdx.x >> 6);
  const RowsWork w = rows_work(a);
  const int64_t b = w.b, hk = w.hk, h = w.h;
  const int q0 = w.block * kRows, split = w.split;
  const int dim = (int)a.dim;
  const Allowed allow = allowed_keys(a, b);
  const int queries = (int)a.queries, wq0 = q0 + wave * kWaveRows, q = wq0 + (lane & 31);
  const int q_end = q < queries ? key_end(allow, q) : 0;  // this lane's query sees keys below
  const int begin = std::min(split * (int)a.split_len, allow.len);
  const int end = std::min(key_end(allow, std::min(q0 + kRows, queries) - 1), begin + (int)a.split_len);
  // keys below free_end are seen by every query of the wave, keys from wave_end on by none
  const int free_end = wq0 < queries ? std::min(key_end(allow, wq0), end) : 0;
  const int wave_end = wq0 < queries ? std::min(key_end(allow, std::min(wq0 + kWaveRows, queries) - 1), end) : 0;

  const T* qp = (const T*)a.q + b * a.qs[0] + h * a.qs[1];
  const T* kp = (const T*)a.k + b * a.ks[0] + hk * a.ks[1];
  const T* vp = (const T*)a.v + b * a.vs[0] + hk * a.vs[1];
  Opd<T> qf[KK];
  load_operand<T, DP, FAST>(qf, qp + (int64_t)q * a.qs[2], dim, q < queries);
  f32x16 o[DT] = {};
  float top = -FLT_MAX, sum = 0.0f;  // subtracted, in units of log2; sum of this lane's half of the keys
  const float c = a.scale * kLog2E;

  // one tile's products in LDS while the next one's loads are under way, a barrier a tile
  TileLoader<T, DP, FAST> kt, vt;
  kt.init(kp, a.ks[2], dim, (int)a.keys);
  vt.init(vp, a.vs[2], dim, (int)a.keys);
  if (begin < end) {
    kt.fetch(begin, end);
    vt.fetch(begin, end);
    if constexpr (kBufs<T> == 2) {
      kt.template put<KL>(lds_k[0]);
      vt.template put<VL>(lds_v[0]);
    }
  }
  int buf = 0;
  for (int j0 = begin; j0 < end; j0 += kKeys, buf ^= kBufs<T> - 1) {
    __syncthreads();  // this tile is there, the one before has been read
    if constexpr (kBufs<T> == 1) {
      kt.template put<KL>(lds_k[0]);
      vt.template put<VL>(lds_v[0]);
      __syncthreads();
    }
    const bool more = j0 + kKeys < end;
    if (more) {
      kt.fetch(j0 + kKeys, end);
      vt.fetch(j0 + kKeys, end);
    }
    if (j0 < wave_end) {
      const Elem<T>* lk = lds_k[buf] + KL::at(lane & 31, half * 8);
      const Elem<T>* lv = lds_v[buf];
      f32x16 s[2] = {};
      {
        Opd<T> kf[2][KK];
        if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int t = 0; t < 2; ++t) kf[t][kk] = lds_operand<T>(lk + t * 32 * KL::S + kk * 16, KP);
          fence_schedule<T>();
        }
        if constexpr (DP > 64) __builtin_amdgcn_s_setprio(1);  // 1 x 8192 x 16 x 128: 548 -> 529 us; slower at 64
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if constexpr (sizeof(T) == 4) kf[t][kk] = lds_operand<T>(lk + t * 32 * KL::S + kk * 16, KP);
            s[t] = mma32(kf[t][kk], qf[kk], s[t]);
          }
          fence_operands<T>();
        }
        if constexpr (DP > 64) __builtin_amdgcn_s_setprio(0);
      }
      Opd<T> vf[4][DT];
      const auto load_v = [&](int u, int d) {
        vf[u][d] = lds_column_operand<T, VL>(lv, VP, u * 16 + half * 4, u * 16 + half * 4 + 8, d * 32 + (lane & 16));
      };
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int d = 0; d < DT; ++d) load_v(u, d);
        fence_schedule<T>();
      }
      if (j0 + kKeys > free_end) {
        const int lim = std::min(q_end, end) - j0 - half * 4;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[t][r] = t * 32 + (r >> 2) * 8 + (r & 3) < lim ? s[t][r] : -INFINITY;
      }
      float most = s[0][0];
#pragma unroll
      for (int t = 0; t < 2; ++t)
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
      for (int u = 0; u < 4; ++u) {
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
  sum += other_half(sum);
  if (q >= queries) return;
  const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
  const float lse = sum > 0.0f ? top + log2_hw(sum) : (sum == 0.0f ? -INFINITY : sum);
  const int64_t rows = a.batch * a.heads * a.queries, row = (b * a.heads + h) * a.queries + q;
  if (a.splits > 1) {
    if (half == 0) a.work[rows * a.splits * dim + row * a.splits + split] = lse;
    store_result<float, DP, FAST>(a.work + (row * a.splits + split) * dim, o, inv, dim);
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

template <class T, int DP, bool WHOLE>
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
  const int64_t hk = uniform((int)(id % kvh)), b = ranked_sequence(a, uniform((int)(id / kvh % batch)));
  const int split = uniform((int)(id / kvh / batch));
  const int dim = (int)a.dim, queries = (int)a.queries, rows_here = group * queries;
  const Allowed allow = allowed_keys(a, b);
  const int row = lane & 15;  // this lane's column of the products: query row % queries of head row / queries
  const bool live = row < rows_here;
  const int g = live ? row / queries : 0, qi = live ? row % queries : 0;
  const int64_t h = hk * group + g;
  const int q_end = live ? key_end(allow, qi) : 0;
  const int begin = std::min(split * (int)a.split_len, allow.len);
  const int end = std::min(key_end(allow, queries - 1), begin + (int)a.split_len);
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
  auto fetch = [&](int j0) {
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
  int j0 = begin + wave * kStep;
  if (j0 < end) fetch(j0);
  for (; j0 < end; j0 += kWaves * kStep) {
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
    if (j0 + kWaves * kStep < end) fetch(j0 + kWaves * kStep);
    const int lim = std::min(q_end, end) - j0 - quad * 4;
    float most = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (t * 16 + r >= lim) s[t][r] = -INFINITY;
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
  const int64_t rows = a.batch * a.heads * a.queries;
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
    if (a.splits > 1) {
      a.work[(out_row * a.splits + split) * dim + col] = v;
      if (col == 0) a.work[rows * a.splits * dim + out_row * a.splits + split] = lse;
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
template <class T, int SHARE>
__global__ __launch_bounds__(256) void attention_join(const AttnArgs a) {
  constexpr int CHUNKS = 256 / SHARE;
  static_assert(SHARE == 1 || CHUNKS * 8 == kAttnMaxDim);
  __shared__ float lds_v[SHARE][CHUNKS][8], lds_m[SHARE], lds_t[SHARE];
  const int dim = (int)a.dim, splits = a.splits, per_row = (dim + 7) / 8;
  const uint32_t rows_wg = SHARE == 1 ? 256 / per_row : 1, rows = (uint32_t)(a.batch * a.heads * a.queries);
  const int part_no = threadIdx.x / CHUNKS, chunk = threadIdx.x % CHUNKS, r = chunk / per_row;
  const int col = (chunk - r * per_row) * 8;
  const uint32_t row = blockIdx.x * rows_wg + r;
  const bool live = (uint32_t)r < rows_wg && row < rows;
  const int64_t first = (int64_t)(live ? row : 0) * splits;
  const float* lses = a.work + (int64_t)rows * splits * dim + first;
  const float* part = a.work + first * dim + col;
  float m = -FLT_MAX, total = 0.0f, v[8] = {};
  for (int s = part_no; s < splits; s += SHARE) m = max_nan(m, lses[s]);
  if constexpr (SHARE > 1) {
    if (chunk == 0) lds_m[part_no] = m;
    __syncthreads();
#pragma unroll
    for (int g = 0; g < SHARE; ++g) m = max_nan(m, lds_m[g]);
  }
  if (live) {
#pragma unroll 4
    for (int s = part_no; s < splits; s += SHARE) {
      float x[8];
      load8(x, part + (int64_t)s * dim, dim - col);  // written, zeros where nothing is held
      const float w = exp2_hw(lses[s] - m);          // 0 for a range that holds nothing
      total += w;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += w * x[i];
    }
  }
  if constexpr (SHARE > 1) {
    if (chunk == 0) lds_t[part_no] = total;
#pragma unroll
    for (int i = 0; i < 8; ++i) lds_v[part_no][chunk][i] = v[i];
    __syncthreads();
    total = 0.0f;
#pragma unroll
    for (int g = 0; g < SHARE; ++g) total += lds_t[g];
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

bool by_token(const AttnArgs& a) { return a.heads / a.kv_heads * a.queries <= kTokenRows; }

// Ranges of keys.  Single tokens: as many as make two workgroups for each compute unit, none shorter than
// 256 keys.  Otherwise what an estimate of the time makes shortest, in us: the larger of a workgroup's
// own walk (`alone` a tile, and as much as a tile before its first) and all work spread over the compute units
// (`spread` a tile), and with more than one range the join.  The rates are measured on MI355X: bfloat16 of head
// size 64, 0.7 us a tile when a compute unit has three workgroups and 1 us alone; float32 2.9 and 3.3 us.
// 4 x 512 x 12 x 64 in float32: 1, 2, 3, 4 ranges 31.8, 27.2, 30.4, 31.0 us with the join, 2 are taken;
// float16 6 x 515 over up to 1531 keys x 12 x 80: 34.4, 37.4, 44.0, 47.7 us, 1 is taken.
void plan_splits(AttnArgs& a) {
  const int64_t cus = device_cus();
  int64_t splits = 1;
  if (by_token(a)) {
    const int64_t wgs = std::max<int64_t>(1, a.batch * a.kv_heads);
    splits = std::min({2 * cus / wgs, a.keys / 256, (int64_t)kMaxSplits});
  } else {
    const double unit = (double)((a.dim + 31) / 32 * 32) / 64;
    const double alone = a.dtype == kF32 ? 3.3 * unit : 0.5 + 0.5 * unit, spread = (a.dtype == kF32 ? 2.9 : 0.7) * unit;
    const int64_t tiles = (a.keys + kKeys - 1) / kKeys;
    const double wgs = (double)(a.batch * a.heads) * (double)((a.queries + kRows - 1) / kRows);
    // about half of a square causal call's tiles are walked
    // (also of ragged sequences' tiles, whose lengths only the device knows)
    const double walked = (double)tiles * ((a.causal && a.queries * 2 > a.keys) || a.lengths ? 0.55 : 1.0);
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
  a.split_len = splits > 1 ? ((a.keys + splits - 1) / splits + kKeys - 1) / kKeys * kKeys : std::max<int64_t>(a.keys, 1);
  a.splits = splits > 1 ? (int)((a.keys + a.split_len - 1) / a.split_len) : 1;
}

template <class T, int DP>
hipError_t run(const AttnArgs& a, hipStream_t s) {
  if (by_token(a)) {
    const int64_t grid = a.batch * a.kv_heads * a.splits;
    if (a.dim % 8 == 0) hipLaunchKernelGGL((attention_token<T, DP, true>), dim3((unsigned)grid), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((attention_token<T, DP, false>), dim3((unsigned)grid), dim3(256), 0, s, a);
  } else {
    const dim3 grid((unsigned)(a.batch * a.heads * a.splits * ((a.queries + kRows - 1) / kRows)));
    if (a.dim % 8 == 0 && fast_rows(a.k, a.ks, sizeof(T)) && fast_rows(a.v, a.vs, sizeof(T)))
      hipLaunchKernelGGL((attention_rows<T, DP, true>), grid, dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((attention_rows<T, DP, false>), grid, dim3(256), 0, s, a);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  const int64_t rows = a.batch * a.heads * a.queries;
  const int64_t rows_wg = 256 / ((a.dim + 7) / 8);
  if (a.splits > kSplitsAlone)
    hipLaunchKernelGGL((attention_join<T, 16>), dim3((unsigned)rows), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((attention_join<T, 1>), dim3((unsigned)((rows + rows_wg - 1) / rows_wg)), dim3(256), 0, s, a);
  return hipGetLastError();
}

template <class T>
hipError_t run_dim(const AttnArgs& a, hipStream_t s) {
  switch ((a.dim + 31) / 32) {
    case 1: return run<T, 32>(a, s);
    case 2: return run<T, 64>(a, s);
    case 3: return run<T, 96>(a, s);
    case 4: return run<T, 128>(a, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace

int64_t attention_fwd_work(const AttnArgs& args) {
  AttnArgs a = args;
  plan_splits(a);
  return a.splits > 1 ? (int64_t)a.splits * a.batch * a.heads * a.queries * (a.dim + 1) : 0;
}

hipError_t launch_attention_fwd(AttnArgs a, hipStream_t s) {
  plan_splits(a);
  a.cus = (int)device_cus();
  switch (a.dtype) {
    case kF32: return run_dim<float>(a, s);
    case kF16: return run_dim<f16>(a, s);
    case kBF16: return run_dim<bf16>(a, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace lwl
