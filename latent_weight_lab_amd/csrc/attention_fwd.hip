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
#include <algorithm>
#include <cfloat>

#include "attention_device.h"

namespace lwl {
namespace {

constexpr float kLift = 6.0f, kSlack = 8.0f;
constexpr int kKeys = 64;   // keys of a tile
constexpr int kWaveRows = 32;
constexpr int kWaves = 4;
constexpr int kRows = kWaves * kWaveRows;

// LDS row lengths in elements.  Keys are read 16 bytes a lane, 16 lanes at a time from 16 rows: 16
// bytes of padding put these on distinct banks.  Values are read by columns: 16-bit rows of 16 dwords
// more than a multiple of 32, so that a transposing read's four rows of 64 bytes fall on distinct
// banks; float32 rows of 8 more than a multiple of 16.
template <class T, int DP>
struct RowsTile {
  static constexpr int KS = DP + 16 / (int)sizeof(T);
  static constexpr int VS = sizeof(T) == 2 ? DP + ((DP / 32) % 2 ? 0 : 32) : DP + 8;
  static constexpr int CPR = DP / 8;                     // chunks of eight a row
  static constexpr int PER = kKeys * CPR / 256;          // chunks a thread brings of a tile
};

template <class T, int DP>
__device__ __forceinline__ void fetch_tile(Raw8<T>* r, const T* base, int64_t stride, int j0,
                                           int end, int dim) {
  using Tile = RowsTile<T, DP>;
#pragma unroll
  for (int i = 0; i < Tile::PER; ++i) {
    const int c = threadIdx.x + i * 256, row = c / Tile::CPR, col = (c % Tile::CPR) * 8;
    // keys past the end are zeros: nothing past a sequence's length is multiplied in
    load_raw8(r[i], base + (int64_t)(j0 + row) * stride + col, j0 + row < end ? dim - col : 0);
  }
}
template <class T, int DP, int STRIDE>
__device__ __forceinline__ void stage_tile(T* lds, const Raw8<T>* r) {
  using Tile = RowsTile<T, DP>;
#pragma unroll
  for (int i = 0; i < Tile::PER; ++i) {
    const int c = threadIdx.x + i * 256;
    lds_put(lds + (c / Tile::CPR) * STRIDE + (c % Tile::CPR) * 8, r[i]);
  }
}

template <class T, int DP>
__global__ __launch_bounds__(256) void attention_rows(const AttnArgs a) {
  using Tile = RowsTile<T, DP>;
  constexpr int KK = DP / 16, DT = DP / 32;
  __shared__ __attribute__((aligned(16))) T lds_k[kKeys * Tile::KS];
  __shared__ __attribute__((aligned(16))) T lds_v[kKeys * Tile::VS];
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6;
  // Heads vary fastest, those that share a key head a multiple of the key heads apart; queries with
  // the most keys first (causal: the last ones).
  const int64_t kvb = a.batch * a.kv_heads, group = a.heads / a.kv_heads, nbh = kvb * group;
  int64_t id = blockIdx.x;
  const int64_t bh = id % nbh;
  id /= nbh;
  const int split = (int)(id % a.splits);
  id /= a.splits;
  const int64_t qblocks = (a.queries + kRows - 1) / kRows;
  const int64_t q0 = (qblocks - 1 - id) * kRows;
  const int64_t b = (bh % kvb) / a.kv_heads, hk = (bh % kvb) % a.kv_heads, h = hk * group + bh / kvb;
  const int dim = (int)a.dim;
  const Allowed allow = allowed_keys(a, b);
  const int64_t q = q0 + wave * kWaveRows + (lane & 31);
  const int q_end = q < a.queries ? key_end(allow, q) : 0;  // this lane's query sees keys below
  const int64_t last = std::min<int64_t>(q0 + kRows, a.queries) - 1;
  const int begin = (int)std::min<int64_t>((int64_t)split * a.split_len, allow.len);
  const int end = (int)std::min<int64_t>(key_end(allow, last), (int64_t)begin + a.split_len);
  // keys below which every query of the wave sees: no mask
  const int64_t wq0 = q0 + wave * kWaveRows;
  const int free_end = wq0 < a.queries ? key_end(allow, wq0) : 0;

  const T* qp = (const T*)a.q + b * a.qs[0] + h * a.qs[1];
  const T* kp = (const T*)a.k + b * a.ks[0] + hk * a.ks[1];
  const T* vp = (const T*)a.v + b * a.vs[0] + hk * a.vs[1];
  Frag<T> qf[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) {
    const int col = kk * 16 + half * 8;
    Raw8<T> r;
    load_raw8(r, qp + q * a.qs[2] + col, q < a.queries ? dim - col : 0);
    qf[kk] = frag_of(r);
  }
  f32x16 o[DT] = {};
  float top = -FLT_MAX, sum = 0.0f;  // subtracted, in units of log2; sum of this lane's half of the keys
  const float c = a.scale * kLog2E;

  Raw8<T> kr[Tile::PER], vr[Tile::PER];
  if (begin < end) {
    fetch_tile<T, DP>(kr, kp, a.ks[2], begin, end, dim);
    fetch_tile<T, DP>(vr, vp, a.vs[2], begin, end, dim);
  }
  for (int j0 = begin; j0 < end; j0 += kKeys) {
    __syncthreads();  // the previous tile has been read
    stage_tile<T, DP, Tile::KS>(lds_k, kr);
    stage_tile<T, DP, Tile::VS>(lds_v, vr);
    __syncthreads();
    if (j0 + kKeys < end) {
      fetch_tile<T, DP>(kr, kp, a.ks[2], j0 + kKeys, end, dim);
      fetch_tile<T, DP>(vr, vp, a.vs[2], j0 + kKeys, end, dim);
    }
    f32x16 s[2] = {};
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        s[t] = mma32(lds_frag(lds_k + (t * 32 + (lane & 31)) * Tile::KS + kk * 16 + half * 8), qf[kk], s[t]);
    if (j0 + kKeys > free_end || j0 + kKeys > end) {
      const int lim = std::min(q_end, end) - j0 - half * 4;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (t * 32 + (r >> 2) * 8 + (r & 3) >= lim) s[t][r] = -INFINITY;
    }
    float most = s[0][0];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) most = fmaxf(most, s[t][r]);
    most = fmaxf(most, other_half(most)) * c;
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
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[t][r] = exp2_hw(fmaf(s[t][r], c, -top));
        sum += s[t][r];
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        Frag<T> p;
#pragma unroll
        for (int r = 0; r < 8; ++r) p[r] = (T)s[t][u * 8 + r];
        const int row = t * 32 + u * 16 + half * 4;
#pragma unroll
        for (int d = 0; d < DT; ++d)
          o[d] = mma32(lds_column_frag(lds_v, Tile::VS, row, row + 8, d * 32 + (lane & 16)), p, o[d]);
      }
    }
  }
  sum += other_half(sum);
  if (q >= a.queries) return;
  const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
  const float lse = sum > 0.0f ? top + log2_hw(sum) : (sum == 0.0f ? -INFINITY : sum);
  const int64_t rows = a.batch * a.heads * a.queries, row = (b * a.heads + h) * a.queries + q;
  if (a.splits > 1) {
    float* part = a.work + (int64_t)split * rows * dim + row * dim;
    if (half == 0) a.work[(int64_t)a.splits * rows * dim + split * rows + row] = lse;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int col = d * 32 + (r >> 2) * 8 + half * 4 + (r & 3);
        if (col < dim) part[col] = o[d][r] * inv;
      }
    return;
  }
  if (a.lse && half == 0) a.lse[row] = lse * kLn2;
  T* op = (T*)a.out + b * a.os[0] + h * a.os[1] + q * a.os[2];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      const int col = d * 32 + r4 * 8 + half * 4;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (col + r < dim) op[col + r] = (T)(o[d][r4 * 4 + r] * inv);
    }
}

// ---------------------------------------------------------------- few queries
constexpr int kTokenRows = 16;  // queries times heads that share a key head
constexpr int kStep = 32;       // keys of a wave's step

template <class T, int DP>
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
  const int lane = threadIdx.x & 63, quad = lane >> 4, wave = threadIdx.x >> 6;
  T* lds_v = reinterpret_cast<T*>(lds + wave * kWaveBytes);
  const int64_t group = a.heads / a.kv_heads;
  int64_t id = blockIdx.x;
  const int64_t hk = id % a.kv_heads;
  id /= a.kv_heads;
  const int64_t b = id % a.batch;
  const int split = (int)(id / a.batch);
  const int dim = (int)a.dim, queries = (int)a.queries, rows_here = (int)group * queries;
  const Allowed allow = allowed_keys(a, b);
  const int row = lane & 15;  // this lane's column of the products: query row % queries of head row / queries
  const bool live = row < rows_here;
  const int g = live ? row / queries : 0, qi = live ? row % queries : 0;
  const int64_t h = hk * group + g;
  const int q_end = live ? key_end(allow, qi) : 0;
  const int begin = (int)std::min<int64_t>((int64_t)split * a.split_len, allow.len);
  const int end = (int)std::min<int64_t>(key_end(allow, queries - 1), (int64_t)begin + a.split_len);
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
  Raw8<T> kr[2][KK], vr[PER];
  auto fetch = [&](int j0) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const int j = j0 + t * 16 + row, col = kk * 32 + quad * 8;
        load_raw8(kr[t][kk], kp + (int64_t)j * a.ks[2] + col, j < end ? dim - col : 0);
      }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int cc = lane + i * 64, j = j0 + cc / CPR, col = (cc % CPR) * 8;
      load_raw8(vr[i], vp + (int64_t)j * a.vs[2] + col, j < end ? dim - col : 0);
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
      for (int kk = 0; kk < KK; ++kk) s[t] = mma16(frag_of(kr[t][kk]), qf[kk], s[t]);
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
      o[d] = mma16(lds_column_frag(lds_v, VS, quad * 4, quad * 4 + 16, d * 16), p, o[d]);
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
      a.work[(int64_t)split * rows * dim + out_row * dim + col] = v;
      if (col == 0) a.work[(int64_t)a.splits * rows * dim + split * rows + out_row] = lse;
    } else {
      ((T*)a.out)[b * a.os[0] + hh * a.os[1] + qq * a.os[2] + col] = (T)v;
      if (a.lse && col == 0) a.lse[out_row] = lse * kLn2;
    }
  }
}

// The ranges' outputs weighed by their sums: a wave for each row.
template <class T>
__global__ __launch_bounds__(256) void attention_join(const AttnArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t rows = a.batch * a.heads * a.queries;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int dim = (int)a.dim, splits = a.splits;
  const float* lses = a.work + (int64_t)splits * rows * dim + row;
  float m = -FLT_MAX;
  for (int s = lane; s < splits; s += 64) m = fmaxf(m, lses[s * rows]);
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) m = fmaxf(m, __shfl_xor(m, k, 64));
  float total = 0.0f, v[2] = {0.0f, 0.0f};
  for (int s = 0; s < splits; ++s) {
    const float l = lses[s * rows];
    if (l == -INFINITY) continue;
    const float w = exp2_hw(l - m);
    total += w;
    const float* part = a.work + (int64_t)s * rows * dim + row * dim;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (lane + 64 * i < dim) v[i] += w * part[lane + 64 * i];
  }
  const int64_t b = row / (a.heads * a.queries), h = row / a.queries % a.heads, q = row % a.queries;
  const float inv = total > 0.0f ? 1.0f / total : (total == 0.0f ? 0.0f : total);
  T* op = (T*)a.out + b * a.os[0] + h * a.os[1] + q * a.os[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (lane + 64 * i < dim) op[lane + 64 * i] = (T)(v[i] * inv);
  if (a.lse && lane == 0)
    a.lse[row] = total > 0.0f ? (m + log2_hw(total)) * kLn2 : (total == 0.0f ? -INFINITY : total);
}

bool by_token(const AttnArgs& a) { return a.heads / a.kv_heads * a.queries <= kTokenRows; }

// Ranges of keys: enough that the workgroups fill the chip, none shorter than 256 keys.
void plan_splits(AttnArgs& a) {
  const bool token = by_token(a);
  const int64_t wgs = token ? a.batch * a.kv_heads : a.batch * a.heads * ((a.queries + kRows - 1) / kRows);
  const int64_t want = (token ? 4 : 1) * device_cus();
  int64_t splits = wgs > 0 ? (want + wgs - 1) / wgs : 1;
  splits = std::max<int64_t>(1, std::min(splits, a.keys / 256));
  a.split_len = splits > 1 ? ((a.keys + splits - 1) / splits + kKeys - 1) / kKeys * kKeys : std::max<int64_t>(a.keys, 1);
  a.splits = splits > 1 ? (int)((a.keys + a.split_len - 1) / a.split_len) : 1;
}

template <class T, int DP>
hipError_t run(const AttnArgs& a, hipStream_t s) {
  if (by_token(a)) {
    const int64_t grid = a.batch * a.kv_heads * a.splits;
    hipLaunchKernelGGL((attention_token<T, DP>), dim3((unsigned)grid), dim3(256), 0, s, a);
  } else {
    const int64_t grid = a.batch * a.heads * a.splits * ((a.queries + kRows - 1) / kRows);
    hipLaunchKernelGGL((attention_rows<T, DP>), dim3((unsigned)grid), dim3(256), 0, s, a);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  const int64_t rows = a.batch * a.heads * a.queries;
  hipLaunchKernelGGL((attention_join<T>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a);
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
  switch (a.dtype) {
    case kF32: return run_dim<float>(a, s);
    case kF16: return run_dim<f16>(a, s);
    case kBF16: return run_dim<bf16>(a, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace lwl
