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
// attention_bwd_rows prepares for each query lse in units of log2 (+infinity for a query without
// keys, whose probabilities are then zero) and D.
#include <algorithm>

#include "attention_device.h"

namespace lwl {
namespace {

constexpr int kBlock = 128;  // keys (queries) of a workgroup: 32 for each of four waves
constexpr int kTile = 64;    // queries (keys) of a tile

// In dV's product the probabilities are 2^kLift times too large (exact, and taken back at the end): dV sums
// a key's probabilities over the queries, all of which may be small, and small ones are subnormal in
// float16 and flushed by the exponential in float32.
constexpr float kLift = 14.0f, kLower = 0x1p-14f;

template <class T, int DP>
struct BwdTile {
  static constexpr int S = DP + 16 / (int)sizeof(T);  // LDS row: 16-byte reads of 16 rows on distinct banks
  static constexpr int CPR = DP / 8;
  static constexpr int PER = kTile * CPR / 256;
};

// Rows row0 .. + 63 of base that ok() allows, else zeros.
template <class T, int DP, class Ok>
__device__ __forceinline__ void fetch_rows(Raw8<T>* r, const T* base, int64_t stride, int64_t row0, int dim, Ok ok) {
  using Tile = BwdTile<T, DP>;
#pragma unroll
  for (int i = 0; i < Tile::PER; ++i) {
    const int c = threadIdx.x + i * 256, row = c / Tile::CPR, col = (c % Tile::CPR) * 8;
    load_raw8(r[i], base + (row0 + row) * stride + col, ok(row0 + row) ? dim - col : 0);
  }
}
template <class T, int DP>
__device__ __forceinline__ void stage_rows(T* lds, const Raw8<T>* r) {
  using Tile = BwdTile<T, DP>;
#pragma unroll
  for (int i = 0; i < Tile::PER; ++i) {
    const int c = threadIdx.x + i * 256;
    lds_put(lds + (c / Tile::CPR) * Tile::S + (c % Tile::CPR) * 8, r[i]);
  }
}
template <class T, int DP>
__device__ __forceinline__ void load_operand(Frag<T> (&f)[DP / 16], const T* row, int dim, bool ok) {
  const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk) {
    const int col = kk * 16 + half * 8;
    Raw8<T> r;
    load_raw8(r, row + col, ok ? dim - col : 0);
    f[kk] = frag_of(r);
  }
}
// A result whose columns are rows of a tensor: lane's row, values 8 r4 + 4 half .. + 3 of each 32.
template <class T, int DP>
__device__ __forceinline__ void store_rows(T* row, const f32x16 (&v)[DP / 32], float scale, int dim) {
  const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      const int col = d * 32 + r4 * 8 + half * 4;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (col + r < dim) row[col + r] = (T)(v[d][r4 * 4 + r] * scale);
    }
}

// work: [rows] log2 units of lse, [rows] D
template <class T>
__global__ __launch_bounds__(256) void attention_bwd_rows(const AttnArgs a) {
  const int lane = threadIdx.x & 15;
  const int64_t rows = a.batch * a.heads * a.queries;
  const int64_t row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const bool live = row < rows;
  const int64_t rr = live ? row : 0;
  const int64_t b = rr / (a.heads * a.queries), h = rr / a.queries % a.heads, q = rr % a.queries;
  const int col = lane * 8, n = live ? (int)a.dim - col : 0;
  float o[8], g[8], s = 0.0f;
  load8(o, (const T*)a.out + b * a.os[0] + h * a.os[1] + q * a.os[2] + col, n);
  load8(g, (const T*)a.dout + b * a.dos[0] + h * a.dos[1] + q * a.dos[2] + col, n);
#pragma unroll
  for (int i = 0; i < 8; ++i) s += o[i] * g[i];
  s = lanes_sum<16>(s);
  if (!live || lane != 0) return;
  const bool none = key_end(allowed_keys(a, b), q) == 0;
  a.work[row] = none ? INFINITY : a.lse[row] * kLog2E;
  a.work[rows + row] = none ? 0.0f : s;
}

template <class T, int DP>
__global__ __launch_bounds__(256) void attention_bwd_keys(const AttnArgs a) {
  using Tile = BwdTile<T, DP>;
  constexpr int KK = DP / 16, DT = DP / 32;
  __shared__ __attribute__((aligned(16))) T lds_q[kTile * Tile::S];
  __shared__ __attribute__((aligned(16))) T lds_g[kTile * Tile::S];
  __shared__ __attribute__((aligned(16))) float lds_stat[2][kTile];
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6;
  const int64_t kvb = a.batch * a.kv_heads, group = a.heads / a.kv_heads;
  const int64_t bk = (int64_t)blockIdx.x % kvb, b = bk / a.kv_heads, hk = bk % a.kv_heads;
  const int64_t k0 = (int64_t)blockIdx.x / kvb * kBlock;  // causal: the first keys have the most queries
  const int dim = (int)a.dim;
  const Allowed allow = allowed_keys(a, b);
  const int seen = key_end(allow, a.queries - 1);  // keys that some query sees
  const int64_t key = k0 + wave * 32 + (lane & 31);
  Frag<T> kf[KK], vf[KK];
  load_operand<T, DP>(kf, (const T*)a.k + b * a.ks[0] + hk * a.ks[1] + key * a.ks[2], dim, key < seen);
  load_operand<T, DP>(vf, (const T*)a.v + b * a.vs[0] + hk * a.vs[1] + key * a.vs[2], dim, key < seen);
  f32x16 dk[DT] = {}, dv[DT] = {};
  const float c = a.scale * kLog2E;
  // queries before k0 - off see none of the block's keys
  const int64_t first = k0 >= seen ? a.queries : std::max<int64_t>(0, k0 - allow.off) / kTile * kTile;
  const int64_t rows = a.batch * a.heads * a.queries;
  auto ok = [&](int64_t q) { return q < a.queries && key_end(allow, q) > 0; };
  for (int64_t g = 0; g < group; ++g) {
    const int64_t h = hk * group + g;
    const T* qp = (const T*)a.q + b * a.qs[0] + h * a.qs[1];
    const T* gp = (const T*)a.dout + b * a.dos[0] + h * a.dos[1];
    const float* stat = a.work + (b * a.heads + h) * a.queries;
    Raw8<T> qr[Tile::PER], gr[Tile::PER];
    float sr = 0.0f;
    auto fetch = [&](int64_t q0) {
      fetch_rows<T, DP>(qr, qp, a.qs[2], q0, dim, ok);
      fetch_rows<T, DP>(gr, gp, a.dos[2], q0, dim, ok);
      if (threadIdx.x < 2 * kTile) {
        const int64_t q = q0 + (threadIdx.x & (kTile - 1));
        const bool is_d = threadIdx.x >= kTile;
        sr = q < a.queries ? stat[(is_d ? rows : 0) + q] : (is_d ? 0.0f : INFINITY);
        sr = is_d ? sr * kLower : sr - kLift;
      }
    };
    if (first < a.queries) fetch(first);
    for (int64_t q0 = first; q0 < a.queries; q0 += kTile) {
      __syncthreads();  // the previous tile has been read
      stage_rows<T, DP>(lds_q, qr);
      stage_rows<T, DP>(lds_g, gr);
      if (threadIdx.x < 2 * kTile) lds_stat[threadIdx.x / kTile][threadIdx.x & (kTile - 1)] = sr;
      __syncthreads();
      if (q0 + kTile < a.queries) fetch(q0 + kTile);
      const bool masked = key_end(allow, q0) < k0 + kBlock;  // some pair of the tile is not allowed
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        f32x16 s = {}, dp = {};
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          const int at = (t * 32 + (lane & 31)) * Tile::S + kk * 16 + half * 8;
          s = mma32(lds_frag(lds_q + at), kf[kk], s);
          dp = mma32(lds_frag(lds_g + at), vf[kk], dp);
        }
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const f32x4 l = *(const f32x4*)&lds_stat[0][t * 32 + r4 * 8 + half * 4];
          const f32x4 d = *(const f32x4*)&lds_stat[1][t * 32 + r4 * 8 + half * 4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int i = r4 * 4 + r;
            s[i] = exp2_hw(fmaf(s[i], c, -l[r]));
            dp[i] = s[i] * fmaf(dp[i], kLower, -d[r]);
          }
        }
        if (masked) {
          // key < key_end(q), that is q >= key - off
          const int64_t from = key < allow.len ? key - allow.off - q0 - t * 32 - half * 4 : kTile;
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if ((r >> 2) * 8 + (r & 3) < from) s[r] = dp[r] = 0.0f;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          Frag<T> p, ds;
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            p[r] = (T)s[u * 8 + r];
            ds[r] = (T)dp[u * 8 + r];
          }
          const int row = t * 32 + u * 16 + half * 4;
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            dv[d] = mma32(lds_column_frag(lds_g, Tile::S, row, row + 8, d * 32 + (lane & 16)), p, dv[d]);
            dk[d] = mma32(lds_column_frag(lds_q, Tile::S, row, row + 8, d * 32 + (lane & 16)), ds, dk[d]);
          }
        }
      }
    }
  }
  if (key >= a.keys) return;
  store_rows<T, DP>((T*)a.dk + b * a.dks[0] + hk * a.dks[1] + key * a.dks[2], dk, a.scale, dim);
  store_rows<T, DP>((T*)a.dv + b * a.dvs[0] + hk * a.dvs[1] + key * a.dvs[2], dv, kLower, dim);
}

template <class T, int DP>
__global__ __launch_bounds__(256) void attention_bwd_queries(const AttnArgs a) {
  using Tile = BwdTile<T, DP>;
  constexpr int KK = DP / 16, DT = DP / 32;
  __shared__ __attribute__((aligned(16))) T lds_k[kTile * Tile::S];
  __shared__ __attribute__((aligned(16))) T lds_v[kTile * Tile::S];
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6;
  const int64_t kvb = a.batch * a.kv_heads, group = a.heads / a.kv_heads, nbh = kvb * group;
  const int64_t bh = (int64_t)blockIdx.x % nbh, id = (int64_t)blockIdx.x / nbh;
  const int64_t qblocks = (a.queries + kBlock - 1) / kBlock;
  const int64_t q0 = (qblocks - 1 - id) * kBlock;
  const int64_t b = (bh % kvb) / a.kv_heads, hk = (bh % kvb) % a.kv_heads, h = hk * group + bh / kvb;
  const int dim = (int)a.dim;
  const Allowed allow = allowed_keys(a, b);
  const int64_t q = q0 + wave * 32 + (lane & 31);
  const int q_end = q < a.queries ? key_end(allow, q) : 0;
  const int end = key_end(allow, std::min<int64_t>(q0 + kBlock, a.queries) - 1);
  const int64_t wq0 = q0 + wave * 32;
  const int free_end = wq0 < a.queries ? key_end(allow, wq0) : 0;
  const T* kp = (const T*)a.k + b * a.ks[0] + hk * a.ks[1];
  const T* vp = (const T*)a.v + b * a.vs[0] + hk * a.vs[1];
  Frag<T> qf[KK], gf[KK];
  load_operand<T, DP>(qf, (const T*)a.q + b * a.qs[0] + h * a.qs[1] + q * a.qs[2], dim, q_end > 0);
  load_operand<T, DP>(gf, (const T*)a.dout + b * a.dos[0] + h * a.dos[1] + q * a.dos[2], dim, q_end > 0);
  const int64_t rows = a.batch * a.heads * a.queries, row = (b * a.heads + h) * a.queries + q;
  const float lse = q < a.queries ? a.work[row] : INFINITY, delta = q < a.queries ? a.work[rows + row] : 0.0f;
  f32x16 dq[DT] = {};
  const float c = a.scale * kLog2E;
  auto ok = [&](int64_t j) { return j < end; };
  Raw8<T> kr[Tile::PER], vr[Tile::PER];
  auto fetch = [&](int j0) {
    fetch_rows<T, DP>(kr, kp, a.ks[2], j0, dim, ok);
    fetch_rows<T, DP>(vr, vp, a.vs[2], j0, dim, ok);
  };
  if (end > 0) fetch(0);
  for (int j0 = 0; j0 < end; j0 += kTile) {
    __syncthreads();
    stage_rows<T, DP>(lds_k, kr);
    stage_rows<T, DP>(lds_v, vr);
    __syncthreads();
    if (j0 + kTile < end) fetch(j0 + kTile);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x16 s = {}, dp = {};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const int at = (t * 32 + (lane & 31)) * Tile::S + kk * 16 + half * 8;
        s = mma32(lds_frag(lds_k + at), qf[kk], s);
        dp = mma32(lds_frag(lds_v + at), gf[kk], dp);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = exp2_hw(fmaf(s[r], c, -lse)) * (dp[r] - delta);
      if (j0 + kTile > free_end) {
        const int lim = q_end - j0 - t * 32 - half * 4;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if ((r >> 2) * 8 + (r & 3) >= lim) s[r] = 0.0f;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        Frag<T> ds;
#pragma unroll
        for (int r = 0; r < 8; ++r) ds[r] = (T)s[u * 8 + r];
        const int krow = t * 32 + u * 16 + half * 4;
#pragma unroll
        for (int d = 0; d < DT; ++d)
          dq[d] = mma32(lds_column_frag(lds_k, Tile::S, krow, krow + 8, d * 32 + (lane & 16)), ds, dq[d]);
      }
    }
  }
  if (q >= a.queries) return;
  store_rows<T, DP>((T*)a.dq + b * a.dqs[0] + h * a.dqs[1] + q * a.dqs[2], dq, a.scale, dim);
}

template <class T, int DP>
hipError_t run(const AttnArgs& a, hipStream_t s) {
  const int64_t kgrid = a.batch * a.kv_heads * ((a.keys + kBlock - 1) / kBlock);
  const int64_t qgrid = a.batch * a.heads * ((a.queries + kBlock - 1) / kBlock);
  if (kgrid > 0) {
    hipLaunchKernelGGL((attention_bwd_keys<T, DP>), dim3((unsigned)kgrid), dim3(256), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (qgrid > 0) hipLaunchKernelGGL((attention_bwd_queries<T, DP>), dim3((unsigned)qgrid), dim3(256), 0, s, a);
  return hipGetLastError();
}

template <class T>
hipError_t run_dim(const AttnArgs& a, hipStream_t s) {
  const int64_t rows = a.batch * a.heads * a.queries;
  if (rows > 0) {
    hipLaunchKernelGGL((attention_bwd_rows<T>), dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  switch ((a.dim + 31) / 32) {
    case 1: return run<T, 32>(a, s);
    case 2: return run<T, 64>(a, s);
    case 3: return run<T, 96>(a, s);
    case 4: return run<T, 128>(a, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace

int64_t attention_bwd_work(const AttnArgs& a) { return 2 * a.batch * a.heads * a.queries; }

hipError_t launch_attention_bwd(AttnArgs a, hipStream_t s) {
  switch (a.dtype) {
    case kF32: return run_dim<float>(a, s);
    case kF16: return run_dim<f16>(a, s);
    case kBF16: return run_dim<bf16>(a, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace lwl
