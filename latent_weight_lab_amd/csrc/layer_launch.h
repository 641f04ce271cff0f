// Internal interface between the C ABI of the layer operators (layer_abi.cpp) and their kernel
// files: layer norm (layer_norm.hip), GELU with an 8-bit checkpoint (gelu8.hip), attention
// (attention_fwd.hip, attention_bwd.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "bfht_launch.h"

namespace lwl {

// Status of a C entry with its message (bfht_abi.cpp): what lwl_last_error() returns.
int status_fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int status_ok();
int status_hip(hipError_t e, const char* what);
int status_workspace(size_t need, const void* ws, size_t have);

// At most `most` ranges of `works` equal works, as equal as they can be: with one more round for some than for
// others the last round leaves most of the chip idle.
inline int64_t even_ranges(int64_t works, int64_t most) {
  if (works <= 0 || most <= 0) return 1;
  const int64_t rounds = (works + most - 1) / most;
  return (works + rounds - 1) / rounds;
}

// ---------------------------------------------------------------- layer norm
struct NormArgs {
  int dtype, weight_dtype;
  int64_t rows, features;
  const void *x, *residual, *weight, *bias;  // residual and bias may be null
  void *out, *sum;                           // sum: null without a residual
  float* stats;                              // [2][rows]: mean, 1/sqrt(var + eps); may be null
  float eps;
  // backward
  const void *grad_out, *grad_sum;  // grad_sum may be null
  void *grad_x, *grad_weight, *grad_bias;  // each may be null
  float* work;
};
hipError_t launch_norm_fwd(const NormArgs& a, hipStream_t s);
hipError_t launch_norm_bwd(const NormArgs& a, hipStream_t s);
// float32 rows of 2 * features (weight's, then bias's partial sums) in the backward's workspace;
// 0: one workgroup writes the gradients itself.
int64_t norm_bwd_partial_rows(int64_t rows, int64_t features);

// ---------------------------------------------------------------- GELU, input kept in 8 bits
constexpr int kGelu8Group = 128;  // features under one scale
__host__ __device__ inline int64_t gelu8_pitch(int64_t features) { return (features + 7) / 8 * 8; }
__host__ __device__ inline int64_t gelu8_groups(int64_t features) { return (features + kGelu8Group - 1) / kGelu8Group; }
struct Gelu8Args {
  int dtype, tanh_form;
  int64_t rows, features;
  const void *x, *bias;  // bias may be null
  void* out;             // forward and recomputation: the activation; backward: grad_x
  int8_t* codes;         // [rows][gelu8_pitch]; forward: null keeps nothing
  float* scales;         // [rows][gelu8_groups]
  const void* grad_out;
  void* grad_bias;  // may be null
  float* work;
};
hipError_t launch_gelu8_fwd(const Gelu8Args& a, hipStream_t s);
hipError_t launch_gelu8_activation(const Gelu8Args& a, hipStream_t s);
hipError_t launch_gelu8_bwd(const Gelu8Args& a, hipStream_t s);
int64_t gelu8_bwd_partial_rows(int64_t rows, int64_t features);  // float32 rows of `features`

// ---------------------------------------------------------------- attention
constexpr int kAttnMaxDim = 128;
struct AttnArgs {
  int dtype, causal, bottom_right;
  int64_t causal_offset;
  int64_t batch, heads, kv_heads, queries, keys, dim;
  float scale;
  const void *q, *k, *v;
  void* out;
  float* lse;  // may be null in the forward
  const int32_t* lengths;
  int64_t qs[3], ks[3], vs[3], os[3];  // strides of batch, head, token
  const void* dout;
  void *dq, *dk, *dv;
  int64_t dos[3], dqs[3], dks[3], dvs[3];
  float* work;
  // filled in by the launchers
  int splits;         // ranges of what is walked over that different workgroups take
  int64_t split_len;  // keys of a range
  int cus;            // compute units
};
constexpr int kTileRows = 64;  // tokens of a tile
// Whether a tensor of values of `size` bytes can be read in tiles by 32-bit offsets from a tile's first row:
// addresses and strides are multiples of 16 bytes, rows lie in ascending order (the offsets are unsigned),
// and a tile spans less than 2 GiB.
inline bool fast_rows(const void* p, const int64_t (&stride)[3], int64_t size) {
  const int64_t unit = 16 / size;
  return (uintptr_t)p % 16 == 0 && stride[0] % unit == 0 && stride[1] % unit == 0 && stride[2] % unit == 0 &&
         stride[2] >= 0 && stride[2] < ((int64_t)1 << 31) / (size * kTileRows);
}
// float32 values in the workspace
int64_t attention_fwd_work(const AttnArgs& a);
int64_t attention_bwd_work(const AttnArgs& a);
hipError_t launch_attention_fwd(AttnArgs a, hipStream_t s);
hipError_t launch_attention_bwd(AttnArgs a, hipStream_t s);

// Column sums of `rows` float32 rows of `stride` values, in a fixed order: columns [0, n0) to dst0,
// [n0, n0 + n1) to dst1, in `dtype` (layer_norm.hip).  A null destination is skipped.
hipError_t launch_column_sum(const float* part, int64_t rows, int64_t stride, int64_t n0, void* dst0, int64_t n1,
                             void* dst1, int dtype, hipStream_t s);

}  // namespace lwl
