// Device building blocks of the attention kernels: matrix-core operands and products over the three
// element types, tiles in LDS.
#pragma once

#include "layer_device.h"
#include "layer_launch.h"

namespace lwl {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// One lane's part of a product operand: eight consecutive k.
//
// 32-wide product (32 x 32 x 16): lane l holds row (column) l % 32, k = 8 (l / 32) .. + 7.  16-wide
// product (16 x 16 x 32): row l % 16, k = 8 (l / 16) .. + 7.  For 16-bit types these are the operands of
// one matrix instruction.  float32 has none of that depth; the same eight values feed eight
// instructions of depth 2 (or 4), instruction i taking value i of every lane: each covers k = i, 8 + i
// (.., 24 + i), and all eight every k once, in both operands alike.
//
// Results: lane l holds column l % 32, rows 8 (r / 4) + 4 (l / 32) + r % 4 for r < 16 (32-wide), or
// column l % 16, rows 4 (l / 16) + r for r < 4 (16-wide).
template <class T>
using Frag = typename Vec8<T>::type;

__device__ __forceinline__ f32x16 mma32(Frag<bf16> a, Frag<bf16> b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32(Frag<f16> a, Frag<f16> b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32(Frag<float> a, Frag<float> b, f32x16 c) {
#pragma unroll
  for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
  return c;
}
__device__ __forceinline__ f32x4 mma16(Frag<bf16> a, Frag<bf16> b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(Frag<f16> a, Frag<f16> b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(Frag<float> a, Frag<float> b, f32x4 c) {
#pragma unroll
  for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
  return c;
}

template <class T>
__device__ __forceinline__ Frag<T> frag_of(const Raw8<T>& v) {
  Frag<T> f;
  __builtin_memcpy(&f, &v, sizeof(f));
  return f;
}
// Eight consecutive values of LDS (16-byte aligned).
template <class T>
__device__ __forceinline__ Frag<T> lds_frag(const T* p) {
  return *reinterpret_cast<const Frag<T>*>(p);
}
template <class T>
__device__ __forceinline__ void lds_put(T* p, const Raw8<T>& v) {
  *reinterpret_cast<Frag<T>*>(p) = frag_of(v);
}

// Four values of one column from four consecutive rows of an LDS tile, for each of the 16 columns that
// 16 consecutive lanes ask for: lane i of the 16 gets column col0 + i, rows row0 .. + 3.  16-bit types
// use the transposing read: lane i names the address of row row0 + i / 4, columns col0 + 4 (i % 4) .. + 3.
template <class T>
__device__ __forceinline__ void lds_column4(T (&v)[4], const T* tile, int stride, int row0, int col0) {
  const int i = threadIdx.x & 15;
  if constexpr (sizeof(T) == 2) {
    const T* p = tile + (row0 + (i >> 2)) * stride + col0 + (i & 3) * 4;
    const s16x4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)p);
    __builtin_memcpy(v, &t, sizeof(t));
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = tile[(row0 + r) * stride + col0 + i];
  }
}
// The operand whose eight k are rows a .. a + 3 and b .. b + 3 of a tile, at column col0 + (lane % 16).
template <class T>
__device__ __forceinline__ Frag<T> lds_column_frag(const T* tile, int stride, int a, int b, int col0) {
  T lo[4], hi[4];
  lds_column4(lo, tile, stride, a, col0);
  lds_column4(hi, tile, stride, b, col0);
  Frag<T> f;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    f[r] = lo[r];
    f[4 + r] = hi[r];
  }
  return f;
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_hw(float x) { return __builtin_amdgcn_logf(x); }
constexpr float kLog2E = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// The other half's value: lane l gets lane l ^ 32's.
__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, 64); }

// Which keys a sequence's queries may see: j < len, and with causal j <= i + off.
struct Allowed {
  int len;      // keys of this sequence
  int64_t off;  // keys - 1 when not causal
};
__device__ __forceinline__ Allowed allowed_keys(const AttnArgs& a, int64_t b) {
  Allowed w;
  int64_t len = a.keys;
  if (a.lengths) {
    const int64_t l = a.lengths[b];
    len = l < 0 ? 0 : l < a.keys ? l : a.keys;  // a length past the tensor would read past it
  }
  w.len = (int)len;
  w.off = !a.causal ? a.keys : a.bottom_right ? len - a.queries : a.causal_offset;
  return w;
}
// First key that query i may not see.
__device__ __forceinline__ int key_end(const Allowed& w, int64_t i) {
  const int64_t e = i + w.off + 1;
  return e < 0 ? 0 : e < w.len ? (int)e : w.len;
}

}  // namespace lwl
