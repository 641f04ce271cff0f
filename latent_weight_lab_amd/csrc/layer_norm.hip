// Layer norm over rows of F values, with the residual stream's addition in front:
//
//   h = round(x + r),  mu = mean(h),  s = 1 / sqrt(mean((h - mu)^2) + eps),  y = (h - mu) s w + b
//
// and its backward pass, n = (h - mu) s, a = dy w:
//
//   dh = s (a - mean(a) - n mean(a n)) + dh_out,  dw = sum over rows of dy n,  db = sum over rows of dy
//
// Both directions are bound by memory: about ten float32 operations for each value moved, and every
// stream is read or written once.  A row is held in registers by LANES lanes (eight consecutive
// values each, times CH), so that mean and squared deviations take two passes over registers and
// none over memory; the variance is that of the deviations, not a difference of squares.  All sums
// are float32.
//
// The backward's workgroups walk over the rows with the weight's and the bias's sums in registers:
// a lane holds the same columns of every row, so the sums need no exchange until the end, when a
// workgroup adds its row groups up through LDS and leaves one partial row.  launch_column_sum adds
// the partial rows in a fixed order (the result does not depend on which workgroup ends first).
//
// Measured on MI355X (a copy of as many bytes, which lie in the last-level cache, runs at 8 TB/s, one from memory at
// 4.8-5.2): bfloat16 8192 x 768 with residual, forward 13.1 us (50 MB, 3.8 TB/s), backward 16.6 us (50 MB, 3.0 TB/s,
// and two partial rows a workgroup) and 5.4 us for the sums; float32 1021 x 3072 without, forward 8.2 us (25 MB),
// backward 12.6 (38 MB) and 5.3 us; one to a few rows 3.6 us, a launch and a round trip to memory.
#include <algorithm>

#include "layer_device.h"
#include "layer_launch.h"

namespace lwl {
namespace {

// LANES lanes hold a row, WG / LANES rows at a time in a workgroup.
constexpr int kNormWG = 512;
template <int LANES>
struct NormGeo {
  static constexpr int WG = LANES > kNormWG ? LANES : kNormWG;
  static constexpr int G = WG / LANES;
  static constexpr int WAVES = LANES > 64 ? LANES / 64 : 1;  // waves of a row
};

// Sums of N values over a row's lanes.  Rows of more than one wave go through LDS (`red`: one slot
// of N per wave of the workgroup), where every thread of the workgroup has to come along.
template <int LANES, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float* red) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lanes_sum<(LANES < 64 ? LANES : 64)>(v[i]);
  if constexpr (LANES > 64) {
    const int wave = threadIdx.x >> 6, first = wave & ~(NormGeo<LANES>::WAVES - 1);
    __syncthreads();  // the previous sums have been read
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) red[wave * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < NormGeo<LANES>::WAVES; ++w) s += red[(first + w) * N + i];
      v[i] = s;
    }
  }
}

template <class T, class W, int LANES, int CH>
__global__ __launch_bounds__(NormGeo<LANES>::WG) void norm_fwd(const NormArgs a) {
  using Geo = NormGeo<LANES>;
  __shared__ float red[Geo::WG / 64 + 1];
  const int lane = threadIdx.x & (LANES - 1), group = threadIdx.x / LANES;
  const int64_t F = a.features;
  const T* x = (const T*)a.x;
  const T* res = (const T*)a.residual;
  T* out = (T*)a.out;
  T* sum = (T*)a.sum;
  float w[CH][8], b[CH][8];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int64_t col = (int64_t)(c * LANES + lane) * 8;
    load8(w[c], (const W*)a.weight + col, F - col);
    if (a.bias) {
      load8(b[c], (const W*)a.bias + col, F - col);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) b[c][i] = 0.0f;
    }
  }
  const float count = (float)F;  // divided by, so that a constant row's mean is exact
  for (int64_t row0 = (int64_t)blockIdx.x * Geo::G; row0 < a.rows; row0 += (int64_t)gridDim.x * Geo::G) {
    const int64_t row = row0 + group;
    const bool live = row < a.rows;
    const int64_t base = (live ? row : 0) * F;
    Raw8<T> xr[CH], rr[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int64_t col = (int64_t)(c * LANES + lane) * 8;
      load_raw8(xr[c], x + base + col, F - col);
    }
    if (res) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int64_t col = (int64_t)(c * LANES + lane) * 8;
        load_raw8(rr[c], res + base + col, F - col);
      }
    }
    float h[CH][8];
    float total[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      unpack8(h[c], xr[c]);
      if (res) {
        float r[8];
        unpack8(r, rr[c]);
        // rounded to the stored type first: the backward pass norms what is stored
#pragma unroll
        for (int i = 0; i < 8; ++i) h[c][i] = rounded<T>(h[c][i] + r[i]);
        const int64_t col = (int64_t)(c * LANES + lane) * 8;
        if (live) store8(sum + base + col, h[c], F - col);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) total[0] += h[c][i];
    }
    row_sums<LANES>(total, red);
    const float mean = total[0] / count;
    float dev[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int64_t col = (int64_t)(c * LANES + lane) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        h[c][i] = col + i < F ? h[c][i] - mean : 0.0f;
        dev[0] += h[c][i] * h[c][i];
      }
    }
    row_sums<LANES>(dev, red);
    const float rstd = 1.0f / sqrtf(dev[0] / count + a.eps);
    if (!live) continue;
    if (a.stats && lane == 0) {
      a.stats[row] = mean;
      a.stats[a.rows + row] = rstd;
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int64_t col = (int64_t)(c * LANES + lane) * 8;
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = h[c][i] * rstd * w[c][i] + b[c][i];
      store8(out + base + col, y, F - col);
    }
  }
}

template <class T, class W, int LANES, int CH>
__global__ __launch_bounds__(NormGeo<LANES>::WG) void norm_bwd(const NormArgs a) {
  using Geo = NormGeo<LANES>;
  __shared__ float red[2 * (Geo::WG / 64) + 1];
  __shared__ float acc[Geo::G > 1 ? Geo::WG * 8 : 1];
  const int lane = threadIdx.x & (LANES - 1), group = threadIdx.x / LANES;
  const int64_t F = a.features;
  const T* x = (const T*)a.x;
  const T* dy = (const T*)a.grad_out;
  const T* ds = (const T*)a.grad_sum;
  T* dx = (T*)a.grad_x;
  float w[CH][8], dw[CH][8], db[CH][8];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int64_t col = (int64_t)(c * LANES + lane) * 8;
    load8(w[c], (const W*)a.weight + col, F - col);
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[c][i] = db[c][i] = 0.0f;
  }
  const float count = (float)F;  // divided by, so that a constant row's mean is exact
  for (int64_t row0 = (int64_t)blockIdx.x * Geo::G; row0 < a.rows; row0 += (int64_t)gridDim.x * Geo::G) {
    const int64_t row = row0 + group;
    const bool live = row < a.rows;
    const int64_t base = (live ? row : 0) * F;
    Raw8<T> hr[CH], gr[CH], sr[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int64_t col = (int64_t)(c * LANES + lane) * 8;
      load_raw8(hr[c], x + base + col, live ? F - col : 0);
      load_raw8(gr[c], dy + base + col, live ? F - col : 0);
    }
    if (ds && dx) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int64_t col = (int64_t)(c * LANES + lane) * 8;
        load_raw8(sr[c], ds + base + col, live ? F - col : 0);
      }
    }
    const float mean = live ? a.stats[row] : 0.0f, rstd = live ? a.stats[a.rows + row] : 0.0f;
    float n[CH][8], g[CH][8];
    float m[2] = {0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      unpack8(n[c], hr[c]);
      unpack8(g[c], gr[c]);  // zero past the row's end and for rows past the last
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        n[c][i] = (n[c][i] - mean) * rstd;
        const float av = g[c][i] * w[c][i];
        m[0] += av;
        m[1] += av * n[c][i];
        dw[c][i] += g[c][i] * n[c][i];
        db[c][i] += g[c][i];
      }
    }
    if (dx) {  // the same for every thread
      row_sums<LANES>(m, red);
      m[0] /= count;
      m[1] /= count;
      if (live) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          const int64_t col = (int64_t)(c * LANES + lane) * 8;
          float d[8];
          if (ds) {
            unpack8(d, sr[c]);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = 0.0f;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) d[i] += rstd * (g[c][i] * w[c][i] - m[0] - n[c][i] * m[1]);
          store8(dx + base + col, d, F - col);
        }
      }
    }
  }
  if (!a.grad_weight && !a.grad_bias) return;
  const bool direct = gridDim.x == 1;
  auto put = [&](int which, int64_t col, float v) {
    if (col >= F) return;
    if (direct) {
      W* dst = (W*)(which ? a.grad_bias : a.grad_weight);
      if (dst) dst[col] = (W)v;
    } else {
      a.work[((int64_t)blockIdx.x * 2 + which) * F + col] = v;
    }
  };
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (which == 1 && !a.grad_bias) break;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const float(&v)[8] = which ? db[c] : dw[c];
      if constexpr (Geo::G == 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) put(which, (int64_t)(c * LANES + lane) * 8 + i, v[i]);
      } else {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[threadIdx.x * 8 + i] = v[i];
        __syncthreads();
        for (int j = threadIdx.x; j < LANES * 8; j += Geo::WG) {
          float s = 0.0f;
#pragma unroll
          for (int q = 0; q < Geo::G; ++q) s += acc[q * LANES * 8 + j];
          put(which, (int64_t)c * LANES * 8 + j, s);
        }
      }
    }
  }
}

// Rows longer than the registers of one workgroup hold: a workgroup per row, the row read again in
// each pass (from the second-level cache).
constexpr int kLongWG = 1024;

template <class T, class W>
__global__ __launch_bounds__(kLongWG) void norm_fwd_long(const NormArgs a) {
  __shared__ float red[kLongWG / 64 + 1];
  const int64_t F = a.features;
  const T* x = (const T*)a.x;
  const T* res = (const T*)a.residual;
  const float count = (float)F;  // divided by, so that a constant row's mean is exact
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* hr = (res ? (const T*)a.sum : x) + row * F;
    float total[1] = {0.0f}, dev[1] = {0.0f};
    for (int64_t col = (int64_t)threadIdx.x * 8; col < F; col += kLongWG * 8) {
      float h[8];
      load8(h, x + row * F + col, F - col);
      if (res) {  // a thread reads back only what it has stored itself
        float r[8];
        load8(r, res + row * F + col, F - col);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = rounded<T>(h[i] + r[i]);
        store8((T*)a.sum + row * F + col, h, F - col);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) total[0] += h[i];
    }
    row_sums<kLongWG>(total, red);
    const float mean = total[0] / count;
    for (int64_t col = (int64_t)threadIdx.x * 8; col < F; col += kLongWG * 8) {
      float h[8];
      load8(h, hr + col, F - col);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = col + i < F ? h[i] - mean : 0.0f;
        dev[0] += d * d;
      }
    }
    row_sums<kLongWG>(dev, red);
    const float rstd = 1.0f / sqrtf(dev[0] / count + a.eps);
    if (a.stats && threadIdx.x == 0) {
      a.stats[row] = mean;
      a.stats[a.rows + row] = rstd;
    }
    for (int64_t col = (int64_t)threadIdx.x * 8; col < F; col += kLongWG * 8) {
      float h[8], w[8], b[8] = {};
      load8(h, hr + col, F - col);
      load8(w, (const W*)a.weight + col, F - col);
      if (a.bias) load8(b, (const W*)a.bias + col, F - col);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = (h[i] - mean) * rstd * w[i] + b[i];
      store8((T*)a.out + row * F + col, h, F - col);
    }
  }
}

template <class T, class W>
__global__ __launch_bounds__(kLongWG) void norm_bwd_long_x(const NormArgs a) {
  __shared__ float red[2 * (kLongWG / 64) + 1];
  const int64_t F = a.features;
  const float count = (float)F;  // divided by, so that a constant row's mean is exact
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* h = (const T*)a.x + row * F;
    const T* dy = (const T*)a.grad_out + row * F;
    const float mean = a.stats[row], rstd = a.stats[a.rows + row];
    float m[2] = {0.0f, 0.0f};
    for (int64_t col = (int64_t)threadIdx.x * 8; col < F; col += kLongWG * 8) {
      float n[8], g[8], w[8];
      load8(n, h + col, F - col);
      load8(g, dy + col, F - col);
      load8(w, (const W*)a.weight + col, F - col);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        m[0] += g[i] * w[i];
        m[1] += g[i] * w[i] * ((n[i] - mean) * rstd);
      }
    }
    row_sums<kLongWG>(m, red);
    m[0] /= count;
    m[1] /= count;
    for (int64_t col = (int64_t)threadIdx.x * 8; col < F; col += kLongWG * 8) {
      float n[8], g[8], w[8], d[8] = {};
      load8(n, h + col, F - col);
      load8(g, dy + col, F - col);
      load8(w, (const W*)a.weight + col, F - col);
      if (a.grad_sum) load8(d, (const T*)a.grad_sum + row * F + col, F - col);
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] += rstd * (g[i] * w[i] - m[0] - (n[i] - mean) * rstd * m[1]);
      store8((T*)a.grad_x + row * F + col, d, F - col);
    }
  }
}

// Partial sums of dw and db: grid.x panels of 2048 columns, grid.y ranges of rows.
template <class T, class W>
__global__ __launch_bounds__(256) void norm_bwd_long_w(const NormArgs a) {
  const int64_t F = a.features, col = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (col >= F) return;
  float dw[8] = {}, db[8] = {};
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float mean = a.stats[row], rstd = a.stats[a.rows + row];
    float n[8], g[8];
    load8(n, (const T*)a.x + row * F + col, F - col);
    load8(g, (const T*)a.grad_out + row * F + col, F - col);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      dw[i] += g[i] * ((n[i] - mean) * rstd);
      db[i] += g[i];
    }
  }
  float* part = a.work + (int64_t)blockIdx.y * 2 * F;
  store8(part + col, dw, F - col);
  store8(part + F + col, db, F - col);
}

// Column sums: 8 lanes of four columns each, 64 row groups, joined through LDS in row order.
constexpr int kSumCols = 32, kSumGroups = 64;

template <class W>
__global__ __launch_bounds__(8 * kSumGroups) void column_sum(const float* __restrict__ part, int64_t rows,
                                                             int64_t stride, int64_t n0, W* dst0, int64_t n1,
                                                             W* dst1) {
  __shared__ float acc[kSumGroups][kSumCols + 1];
  const int cl = (threadIdx.x & 7) * 4, group = threadIdx.x >> 3;
  const int64_t n = n0 + n1, col = (int64_t)blockIdx.x * kSumCols + cl;
  float s[4] = {};
  for (int64_t r0 = group; r0 < rows; r0 += 8 * kSumGroups) {
    float v[8][4];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int64_t r = r0 + u * kSumGroups;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[u][i] = r < rows && col + i < n ? part[r * stride + col + i] : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] += v[u][i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[group][cl + i] = s[i];
  __syncthreads();
  // 16 threads a column, four row groups each, then over the 16 lanes
  const int c = threadIdx.x >> 4, q = threadIdx.x & 15;
  float t = (acc[4 * q][c] + acc[4 * q + 1][c]) + (acc[4 * q + 2][c] + acc[4 * q + 3][c]);
  t = lanes_sum<16>(t);
  const int64_t oc = (int64_t)blockIdx.x * kSumCols + c;
  if (q == 0 && oc < n) {
    W* dst = oc < n0 ? dst0 : dst1;
    if (dst) dst[oc < n0 ? oc : oc - n0] = (W)t;
  }
}

// How many lanes hold a row and how many times eight values each.  At most twice: with four times,
// the backward's row, its gradients and the column sums no longer fit 256 registers.
struct NormShape {
  int lanes, ch;  // 0: the row is longer than a workgroup's registers hold
};
NormShape norm_shape(int64_t features) {
  if (features <= 16 * 8) return {16, 1};
  if (features <= 64 * 8) return {64, 1};
  if (features <= 64 * 16) return {64, 2};
  if (features <= 256 * 8) return {256, 1};
  if (features <= 256 * 16) return {256, 2};
  if (features <= 512 * 16) return {512, 2};
  return {0, 0};
}

template <class T, class W, int LANES, int CH>
hipError_t run_norm(const NormArgs& a, bool fwd, hipStream_t s) {
  using Geo = NormGeo<LANES>;
  const int64_t groups = (a.rows + Geo::G - 1) / Geo::G;
  if (fwd) {
    const unsigned grid = (unsigned)even_ranges(groups, 4 * device_cus());
    hipLaunchKernelGGL((norm_fwd<T, W, LANES, CH>), dim3(grid), dim3(Geo::WG), 0, s, a);
  } else {
    const int64_t part = norm_bwd_partial_rows(a.rows, a.features);
    hipLaunchKernelGGL((norm_bwd<T, W, LANES, CH>), dim3((unsigned)(part ? part : 1)), dim3(Geo::WG), 0, s, a);
  }
  return hipGetLastError();
}

template <class T, class W>
hipError_t run_norm_long(const NormArgs& a, bool fwd, hipStream_t s) {
  const unsigned grid = (unsigned)std::min<int64_t>(a.rows, 2 * device_cus());
  if (fwd) {
    hipLaunchKernelGGL((norm_fwd_long<T, W>), dim3(grid), dim3(kLongWG), 0, s, a);
    return hipGetLastError();
  }
  if (a.grad_x) {
    hipLaunchKernelGGL((norm_bwd_long_x<T, W>), dim3(grid), dim3(kLongWG), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (a.grad_weight || a.grad_bias) {
    const dim3 g((unsigned)((a.features + 2047) / 2048), (unsigned)norm_bwd_partial_rows(a.rows, a.features));
    hipLaunchKernelGGL((norm_bwd_long_w<T, W>), g, dim3(256), 0, s, a);
  }
  return hipGetLastError();
}

template <class T, class W>
hipError_t dispatch_norm(const NormArgs& a, bool fwd, hipStream_t s) {
  const NormShape sh = norm_shape(a.features);
  switch (sh.lanes * 8 + sh.ch) {
    case 16 * 8 + 1: return run_norm<T, W, 16, 1>(a, fwd, s);
    case 64 * 8 + 1: return run_norm<T, W, 64, 1>(a, fwd, s);
    case 64 * 8 + 2: return run_norm<T, W, 64, 2>(a, fwd, s);
    case 256 * 8 + 1: return run_norm<T, W, 256, 1>(a, fwd, s);
    case 256 * 8 + 2: return run_norm<T, W, 256, 2>(a, fwd, s);
    case 512 * 8 + 2: return run_norm<T, W, 512, 2>(a, fwd, s);
  }
  return run_norm_long<T, W>(a, fwd, s);
}

hipError_t dispatch_norm_types(const NormArgs& a, bool fwd, hipStream_t s) {
  switch (a.dtype) {
    case kF32: return dispatch_norm<float, float>(a, fwd, s);
    case kF16:
      return a.weight_dtype == kF32 ? dispatch_norm<f16, float>(a, fwd, s) : dispatch_norm<f16, f16>(a, fwd, s);
    case kBF16:
      return a.weight_dtype == kF32 ? dispatch_norm<bf16, float>(a, fwd, s) : dispatch_norm<bf16, bf16>(a, fwd, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace

int64_t norm_bwd_partial_rows(int64_t rows, int64_t features) {
  const NormShape sh = norm_shape(features);
  if (sh.lanes == 0) {
    const int64_t panels = (features + 2047) / 2048;
    return std::max<int64_t>(1, std::min<int64_t>(rows, 4 * device_cus() / panels));
  }
  const int64_t g = kNormWG / sh.lanes, groups = (rows + g - 1) / g;
  if (groups <= 1) return 0;
  return even_ranges(groups, 2 * device_cus());
}

hipError_t launch_column_sum(const float* part, int64_t rows, int64_t stride, int64_t n0, void* dst0, int64_t n1,
                             void* dst1, int dtype, hipStream_t s) {
  const dim3 grid((unsigned)((n0 + n1 + kSumCols - 1) / kSumCols)), block(8 * kSumGroups);
  switch (dtype) {
    case kF32:
      hipLaunchKernelGGL((column_sum<float>), grid, block, 0, s, part, rows, stride, n0, (float*)dst0, n1, (float*)dst1);
      break;
    case kF16:
      hipLaunchKernelGGL((column_sum<f16>), grid, block, 0, s, part, rows, stride, n0, (f16*)dst0, n1, (f16*)dst1);
      break;
    case kBF16:
      hipLaunchKernelGGL((column_sum<bf16>), grid, block, 0, s, part, rows, stride, n0, (bf16*)dst0, n1, (bf16*)dst1);
      break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t launch_norm_fwd(const NormArgs& a, hipStream_t s) { return dispatch_norm_types(a, true, s); }

hipError_t launch_norm_bwd(const NormArgs& a, hipStream_t s) {
  if (a.rows > 0) {
    const hipError_t e = dispatch_norm_types(a, false, s);
    if (e != hipSuccess) return e;
  }
  const bool weights = a.grad_weight || a.grad_bias;
  const int64_t part = a.rows > 0 ? norm_bwd_partial_rows(a.rows, a.features) : 0;
  // no rows: the sums over none of them are written as zeros
  if (!weights || (part == 0 && a.rows > 0)) return hipSuccess;
  return launch_column_sum(a.work, part, 2 * a.features, a.features, a.grad_weight, a.grad_bias ? a.features : 0,
                           a.grad_bias, a.weight_dtype, s);
}

}  // namespace lwl
