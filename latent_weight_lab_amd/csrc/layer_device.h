// Device building blocks of the layer operators (layer norm, GELU checkpoint, attention).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "bfht_device.h"

namespace lwl {

// Eight consecutive values are the unit of every access to memory: 16 bytes of a 16-bit type, two
// times 16 bytes of float32.  The address need only be aligned to an element: gfx950's global loads
// and stores take any element alignment at their full width, so rows of odd lengths and offsets go
// through the same wide accesses as aligned ones.
template <class T>
struct Vec8 {
  typedef T type __attribute__((ext_vector_type(8)));
};
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));

template <class T>
struct Raw8 {
  static constexpr int N = (int)sizeof(T) / 2;  // 16-byte pieces
  u32x4_any q[N];
};

// The n (0 .. 8) values at p; the rest of v is zero.
template <class T>
__device__ __forceinline__ void load_raw8(Raw8<T>& v, const T* p, int64_t n) {
  if (n >= 8) {
#pragma unroll
    for (int i = 0; i < Raw8<T>::N; ++i) v.q[i] = reinterpret_cast<const u32x4_any*>(p)[i];
  } else {
    // the last of the n again in place of those past it, so that the loads need no branch each
    typename Vec8<T>::type e = {};
    if (n > 0) {
      const int last = (int)n - 1;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const T t = p[i < last ? i : last];
        e[i] = i <= last ? t : (T)0.0f;
      }
    }
    __builtin_memcpy(&v, &e, sizeof(v));
  }
}
// The same where n is known to be 8 or none.
template <class T>
__device__ __forceinline__ void load_whole8(Raw8<T>& v, const T* p, bool ok) {
#pragma unroll
  for (int i = 0; i < Raw8<T>::N; ++i) v.q[i] = u32x4_any{0, 0, 0, 0};
  if (ok) {
#pragma unroll
    for (int i = 0; i < Raw8<T>::N; ++i) v.q[i] = reinterpret_cast<const u32x4_any*>(p)[i];
  }
}
// v[0 .. 4) as one store.
template <class T>
__device__ __forceinline__ void store4(T* p, float v0, float v1, float v2, float v3) {
  typedef T vec __attribute__((ext_vector_type(4)));
  const vec e = {(T)v0, (T)v1, (T)v2, (T)v3};
  if constexpr (sizeof(T) == 2) {
    u32x2_any w;
    __builtin_memcpy(&w, &e, sizeof(w));
    *reinterpret_cast<u32x2_any*>(p) = w;
  } else {
    u32x4_any w;
    __builtin_memcpy(&w, &e, sizeof(w));
    *reinterpret_cast<u32x4_any*>(p) = w;
  }
}
template <class T>
__device__ __forceinline__ void unpack8(float (&f)[8], const Raw8<T>& v) {
  typename Vec8<T>::type e;
  __builtin_memcpy(&e, &v, sizeof(v));
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (float)e[i];
}
template <class T>
__device__ __forceinline__ void load8(float (&f)[8], const T* p, int64_t n) {
  Raw8<T> v;
  load_raw8(v, p, n);
  unpack8(f, v);
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8], int64_t n) {
  typename Vec8<T>::type e;
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = (T)f[i];
  if (n >= 8) {
    Raw8<T> v;
    __builtin_memcpy(&v, &e, sizeof(v));
#pragma unroll
    for (int i = 0; i < Raw8<T>::N; ++i) reinterpret_cast<u32x4_any*>(p)[i] = v.q[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = e[i];
  }
}

// v rounded to T and back: what a stored v will be read as.
template <class T>
__device__ __forceinline__ float rounded(float v) {
  return (float)(T)v;
}

// Sum over the LANES consecutive lanes (a power of two up to 64) that this lane belongs to; every
// lane of them gets it.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int m = LANES / 2; m > 0; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
}

}  // namespace lwl
