// GELU of z = x + bias whose input is kept for the backward pass in 8 bits.
//
// Forward: y = gelu(z).  Kept: for each row and each group of 128 features one float32 scale
// s = max|z| / 127 and the integers c = rint(z / s), which stand for c s.  Use: the activation again,
// gelu(c s) (the next linear's input, for its weight gradient), and dx = dy gelu'(c s), db = column
// sums of dx.
//
// All three directions are bound by memory: the forward moves two values and 1.03 bytes for each
// element, the activation one value and 1.03 bytes, the backward two and 1.03.  What they compute is
// kept below that: Phi and its density share one exp and one reciprocal (phi_pair).  A lane holds
// eight consecutive features, so a group of 128 is 16 lanes: its maximum takes four exchanges among
// them.  A lane keeps its columns and walks over the rows, with the bias (and, backward, its
// gradient's sum) in registers, four rows in flight.
//
// Float32 throughout; the codes are what float32 gives: s = max|z| * (1/127), c = rint(z * (1/s)).
// A group of zeros, or of values below 2^-100, has s = 0 and stands for zeros.  A group that holds an
// infinity or a NaN has s = NaN and stands for NaN, so that what went wrong in the forward pass
// shows in the gradients.
//
// Measured on MI355X, bfloat16 8192 x 3072 with a bias: forward 27.6 us (126 MB, 4.6 TB/s), activation 19.8 us (76 MB,
// 3.8 TB/s), backward 30.2 us (126 MB, 4.2 TB/s) and 3.9 us for the bias's sums, where a copy runs at 4.8-5.2 TB/s
// from memory; float16 27.6, 18.4 and 28.6 us; float32 4096 x 3072 (113, 63 and 113 MB) 26.5, 21.0 and 27.0 us.  The two uses read what the forward left in the last-level cache; the instructions to unpack, evaluate
// and pack again fill what is left of their time.
#include <algorithm>

#include "layer_device.h"
#include "layer_launch.h"

namespace lwl {
namespace {

constexpr float kTiny = 0x1p-100f;

// h = 1 - Phi(|z|) and e = exp(-z^2/2).  h = e Q(t), t = 1/(1 + p|z|): Q is a polynomial fitted for
// the least relative error on |z| <= 14.5, beyond which e underflows in float32.  16-bit outputs take
// degree 6 (relative error 4.7e-6), float32 degree 9 (2e-8 before rounding) and the squared argument's
// rounding error carried along, which at |z| = 8 is worth 2e-6 of e.
template <class T>
__device__ __forceinline__ void phi_pair(float z, float& h, float& e) {
  const float az = fabsf(z);
  if constexpr (sizeof(T) == 4) {
    const float t = 1.0f / fmaf(0.21f, az, 1.0f);
    float q = -0.07129447907209396f;
    q = fmaf(q, t, 0.28180304169654846f);
    q = fmaf(q, t, -0.3264901340007782f);
    q = fmaf(q, t, 0.34498316049575806f);
    q = fmaf(q, t, -0.09077020734548569f);
    q = fmaf(q, t, 0.12347108870744705f);
    q = fmaf(q, t, 0.06957000494003296f);
    q = fmaf(q, t, 0.08501239866018295f);
    q = fmaf(q, t, 0.08371514827013016f);
    const float zc = fminf(az, 16.0f);  // past it e is 0 either way
    const float z2 = zc * zc, rest = fmaf(zc, zc, -z2);
    e = expf(-0.5f * z2);
    e = fmaf(e, -0.5f * rest, e);
    h = e * (q * t);
  } else {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.31f, az, 1.0f));
    float q = -0.07392901927232742f;
    q = fmaf(q, t, 0.18044999241828918f);
    q = fmaf(q, t, 0.01574508100748062f);
    q = fmaf(q, t, 0.1334296017885208f);
    q = fmaf(q, t, 0.12044131755828857f);
    q = fmaf(q, t, 0.12386070191860199f);
    e = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);  // log2(e) / 2
    h = e * (q * t);
  }
}

// The tanh form is z s with s = 1 / (1 + exp(-2u)), u = sqrt(2/pi) (z + 0.044715 z^3); slope = s (1 - s).
// Computed from e = exp(-2|u|), s = e / (1 + e) below zero, so that neither overflows and the tail keeps
// its digits (16-bit: the exponential 2^64 times too large and scaled back, for the same reason).
constexpr float kTanhC = 1.5957691216057308f;  // 2 sqrt(2/pi)
template <class T>
__device__ __forceinline__ void logistic_2u(float z, float& s, float& slope) {
  const float u2 = kTanhC * z * fmaf(0.044715f * z, z, 1.0f);
  float e, r;
  if constexpr (sizeof(T) == 4) {
    e = expf(-fabsf(u2));
    r = 1.0f / (1.0f + e);
  } else {
    e = __builtin_amdgcn_exp2f(fmaf(-1.4426950408889634f, fabsf(u2), 64.0f)) * 0x1p-64f;
    r = __builtin_amdgcn_rcpf(1.0f + e);
  }
  s = u2 < 0.0f ? e * r : r;
  slope = e * r * r;
}

// max(z, 0) - |z| h = z Phi(z); |z| is held to 16 in the second term, where h is 0, so that an
// infinite z does not meet a zero h.  A NaN comes through h.
template <class T, bool TANH>
__device__ __forceinline__ float gelu(float z) {
  if constexpr (TANH) {
    float s, slope;
    logistic_2u<T>(z, s, slope);
    return z < -16.0f ? 0.0f : z * s;  // -infinity too
  } else {
    float h, e;
    phi_pair<T>(z, h, e);
    return fmaf(-__builtin_elementwise_minimum(fabsf(z), 16.0f), h, __builtin_elementwise_maximum(z, 0.0f));
  }
}

// d gelu / dz; the terms with z hold it to +-16, where they are 0
template <class T, bool TANH>
__device__ __forceinline__ float gelu_slope(float z) {
  if constexpr (TANH) {
    float s, slope;
    logistic_2u<T>(z, s, slope);
    const float zc = __builtin_amdgcn_fmed3f(z, -16.0f, 16.0f);
    return fmaf(zc * slope, kTanhC * fmaf(0.134145f * zc, zc, 1.0f), s);
  } else {
    float h, e;
    phi_pair<T>(z, h, e);
    const float zc = __builtin_amdgcn_fmed3f(z, -16.0f, 16.0f);
    return fmaf(zc * 0.3989422804014327f, e, z >= 0.0f ? 1.0f - h : h);
  }
}

// Columns and rows of a workgroup: CL lanes of eight columns each, 64 / CL rows in a wave, four waves.
template <int CL>
struct Gelu8Geo {
  static constexpr int COLS = CL * 8;
  static constexpr int ROWS = 256 / CL;
};

// The codes rint(z inv) of eight values as one 8-byte store.  1.5 * 2^23 added to a float32 of up to 2^22
// rounds it to an integer (to even, as rint) and leaves that integer's low byte as the sum's.
__device__ __forceinline__ void store_codes(int8_t* p, const float (&z)[8], float inv) {
  uint32_t b[8], w[2];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float v;
    {
#pragma clang fp contract(off)
      v = z[i] * inv;  // rounded before it is rounded to an integer
      v = v + 12582912.0f;
    }
    b[i] = __float_as_uint(v);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {  // bytes 0 of four registers
    const uint32_t lo = __builtin_amdgcn_perm(b[4 * j + 1], b[4 * j], 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(b[4 * j + 3], b[4 * j + 2], 0x04000c0cu);
    w[j] = lo | hi;
  }
  *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
}
// c * scale from the codes: bytes made unsigned (c + 128) convert in one instruction, and (c + 128) scale - 128
// scale with one rounding is c * scale rounded once (128 scale is exact).
__device__ __forceinline__ void decode8(float (&z)[8], uint2 w, float scale) {
  const uint32_t u[2] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u};
  const float less = -128.0f * scale;
#pragma unroll
  for (int i = 0; i < 8; ++i) z[i] = fmaf((float)((u[i >> 2] >> (8 * (i & 3))) & 0xffu), scale, less);
}
// The largest over 16 lanes (a row of the vector unit's lanes), by rotations within them.
__device__ __forceinline__ uint32_t max_of_16(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));  // rotated by 8
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, false));
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, false));
}

template <class T, bool TANH, int CL, int U>
__global__ __launch_bounds__(256) void gelu8_fwd(const Gelu8Args a) {
  using Geo = Gelu8Geo<CL>;
  const int lane = threadIdx.x & (CL - 1), sub = threadIdx.x / CL;
  const int64_t F = a.features, col = (int64_t)blockIdx.x * Geo::COLS + lane * 8;
  const int64_t pitch = gelu8_pitch(F), groups = gelu8_groups(F);
  const int64_t n = F - col;  // may be negative: the lane then holds nothing
  float b[8] = {};
  if (a.bias) load8(b, (const T*)a.bias + col, n);
  for (int64_t r0 = (int64_t)blockIdx.y * Geo::ROWS * U; r0 < a.rows; r0 += (int64_t)gridDim.y * Geo::ROWS * U) {
    Raw8<T> xr[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = r0 + u * Geo::ROWS + sub;
      load_raw8(xr[u], (const T*)a.x + row * F + col, row < a.rows ? n : 0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = r0 + u * Geo::ROWS + sub;
      const bool live = row < a.rows;
      float z[8], y[8];
      unpack8(z, xr[u]);
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] += b[i];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = gelu<T, TANH>(z[i]);
      if (live) store8((T*)a.out + row * F + col, y, n);
      if (a.codes) {
        // |z| as integers order as the floats do, with infinities and then NaN above them
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(z[i]) & 0x7fffffffu);
        top = max_of_16(top);
        const float most = __uint_as_float(top);
        const bool fine = top < 0x7f800000u && most >= kTiny;
        const float scale = top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : fine ? most * (1.0f / 127.0f) : 0.0f;
        const float inv = fine ? 1.0f / scale : 0.0f;  // not fine: codes of 0, or any under a NaN
        if (live && n > 0) {
          store_codes(a.codes + row * pitch + col, z, inv);
          if ((lane & 15) == 0) a.scales[row * groups + col / kGelu8Group] = scale;
        }
      }
    }
  }
}

// BWD: dx and, with WORK or one row range, the bias's gradient; otherwise the activation again.
template <class T, bool TANH, int CL, int U, bool BWD>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 4 : 1) void gelu8_use(const Gelu8Args a) {
  using Geo = Gelu8Geo<CL>;
  __shared__ float acc[BWD ? 256 * 8 : 1];
  const int lane = threadIdx.x & (CL - 1), sub = threadIdx.x / CL;
  const int64_t F = a.features, col = (int64_t)blockIdx.x * Geo::COLS + lane * 8;
  const int64_t pitch = gelu8_pitch(F), groups = gelu8_groups(F);
  const int64_t n = F - col;
  float db[8] = {};
  for (int64_t r0 = (int64_t)blockIdx.y * Geo::ROWS * U; r0 < a.rows; r0 += (int64_t)gridDim.y * Geo::ROWS * U) {
    uint2 w[U];
    float scale[U];
    Raw8<T> gr[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = r0 + u * Geo::ROWS + sub;
      const bool live = row < a.rows && n > 0;
      const int64_t rr = live ? row : 0, cc = n > 0 ? col : 0;
      w[u] = *reinterpret_cast<const uint2*>(a.codes + rr * pitch + cc);
      scale[u] = a.scales[rr * groups + cc / kGelu8Group];
      if constexpr (BWD) load_raw8(gr[u], (const T*)a.grad_out + row * F + col, live ? n : 0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = r0 + u * Geo::ROWS + sub;
      const bool live = row < a.rows && n > 0;
      float z[8], v[8];
      decode8(z, w[u], scale[u]);
      if constexpr (BWD) {
        float g[8];
        unpack8(g, gr[u]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          v[i] = g[i] * gelu_slope<T, TANH>(z[i]);
          db[i] += live ? v[i] : 0.0f;  // a row past the last decodes another row's codes
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = gelu<T, TANH>(z[i]);
      }
      if (live) store8((T*)a.out + row * F + col, v, n);
    }
  }
  if constexpr (BWD) {
    if (!a.grad_bias) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[threadIdx.x * 8 + i] = db[i];
    __syncthreads();
    for (int j = threadIdx.x; j < Geo::COLS; j += 256) {
      float s = 0.0f;
#pragma unroll
      for (int q = 0; q < Geo::ROWS; ++q) s += acc[q * Geo::COLS + j];
      const int64_t c = (int64_t)blockIdx.x * Geo::COLS + j;
      if (c < F) {
        if (gridDim.y == 1) ((T*)a.grad_bias)[c] = (T)s;
        else a.work[(int64_t)blockIdx.y * F + c] = s;
      }
    }
  }
}

// Lanes that hold a row's panel of columns, rows in flight, ranges of rows.  Rows of up to 128
// features take 16 lanes; four rows in flight where that still leaves two workgroups a CU.
struct Gelu8Shape {
  int cl, u;
  int64_t panels, ranges;
};
Gelu8Shape gelu8_shape(int64_t rows, int64_t features, int64_t wgs_per_cu) {
  Gelu8Shape s;
  s.cl = features <= kGelu8Group ? 16 : 64;
  s.panels = (features + s.cl * 8 - 1) / (s.cl * 8);
  const int64_t per = 256 / s.cl;
  s.u = s.panels * ((rows + per * 4 - 1) / (per * 4)) >= 2 * device_cus() ? 4 : 1;
  const int64_t need = (rows + per * s.u - 1) / (per * s.u);
  s.ranges = even_ranges(need, std::min<int64_t>((wgs_per_cu * device_cus() + s.panels - 1) / s.panels, 65535));
  return s;
}
constexpr int64_t kFwdPerCu = 16, kBwdPerCu = 4;

enum { kGeluFwd, kGeluAgain, kGeluBwd };

template <class T, bool TANH, int CL, int U>
hipError_t run_gelu8(const Gelu8Args& a, int what, const Gelu8Shape& sh, hipStream_t s) {
  const dim3 grid((unsigned)sh.panels, (unsigned)sh.ranges), block(256);
  if (what == kGeluFwd) hipLaunchKernelGGL((gelu8_fwd<T, TANH, CL, U>), grid, block, 0, s, a);
  else if (what == kGeluAgain) hipLaunchKernelGGL((gelu8_use<T, TANH, CL, U, false>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((gelu8_use<T, TANH, CL, U, true>), grid, block, 0, s, a);
  return hipGetLastError();
}

template <class T, bool TANH>
hipError_t shape_gelu8(const Gelu8Args& a, int what, hipStream_t s) {
  const Gelu8Shape sh = gelu8_shape(a.rows, a.features, what == kGeluBwd ? kBwdPerCu : kFwdPerCu);
  if (sh.cl == 16)
    return sh.u == 4 ? run_gelu8<T, TANH, 16, 4>(a, what, sh, s) : run_gelu8<T, TANH, 16, 1>(a, what, sh, s);
  return sh.u == 4 ? run_gelu8<T, TANH, 64, 4>(a, what, sh, s) : run_gelu8<T, TANH, 64, 1>(a, what, sh, s);
}

hipError_t dispatch_gelu8(const Gelu8Args& a, int what, hipStream_t s) {
  if (a.rows == 0) return hipSuccess;
  switch (a.dtype) {
    case kF32: return a.tanh_form ? shape_gelu8<float, true>(a, what, s) : shape_gelu8<float, false>(a, what, s);
    case kF16: return a.tanh_form ? shape_gelu8<f16, true>(a, what, s) : shape_gelu8<f16, false>(a, what, s);
    case kBF16: return a.tanh_form ? shape_gelu8<bf16, true>(a, what, s) : shape_gelu8<bf16, false>(a, what, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace

int64_t gelu8_bwd_partial_rows(int64_t rows, int64_t features) {
  if (rows == 0) return 0;
  const Gelu8Shape sh = gelu8_shape(rows, features, kBwdPerCu);
  return sh.ranges > 1 ? sh.ranges : 0;
}

hipError_t launch_gelu8_fwd(const Gelu8Args& a, hipStream_t s) { return dispatch_gelu8(a, kGeluFwd, s); }
hipError_t launch_gelu8_activation(const Gelu8Args& a, hipStream_t s) { return dispatch_gelu8(a, kGeluAgain, s); }
hipError_t launch_gelu8_bwd(const Gelu8Args& a, hipStream_t s) {
  const hipError_t e = dispatch_gelu8(a, kGeluBwd, s);
  const int64_t part = gelu8_bwd_partial_rows(a.rows, a.features);
  if (e != hipSuccess || !a.grad_bias || (part == 0 && a.rows > 0)) return e;
  return launch_column_sum(a.work, part, a.features, a.features, a.grad_bias, 0, nullptr, a.dtype, s);
}

}  // namespace lwl
