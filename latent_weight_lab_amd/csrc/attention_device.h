// Device building blocks of the attention kernels: matrix-core operands and products over the three
// element types, tiles in LDS.
#pragma once

#include <algorithm>

#include "layer_device.h"
#include "layer_launch.h"

namespace lwl {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// One lane's part of a product operand: eight consecutive k.
//
// 32-wide product (32 x 32 x 16): lane l holds row (column) l % 32, k = 8 (l / 32) .. + 7.  16-wide
// product (16 x 16 x 32): row l % 16, k = 8 (l / 16) .. + 7.  Results: lane l holds column l % 32, rows
// 8 (r / 4) + 4 (l / 32) + r % 4 for r < 16 (32-wide), or column l % 16, rows 4 (l / 16) + r for r < 4.
template <class T>
using Frag = typename Vec8<T>::type;

// What a 32-wide product takes.  For a 16-bit type, one matrix instruction's operand.  A float32 value goes in
// as a sum of three bfloat16 ones, x = x0 + x1 + x2, each the rounding of what the ones before leave: 24
// bits, of float32's range.  Of the nine products of two such sums the six largest are taken; the others
// are below 2^-24 of x y, and the sum is float32 as ever.  Six bfloat16 instructions take 192 cycles
// where float32's own, of depth 2, take 512 for the same k (4 x 512 x 12 x 64 training step: 161 us with
// those, 108 with these).  An infinite float32 value leaves NaN (infinity less infinity).
template <class T>
struct MatrixType {
  using Elem = T;
  using Opd = Frag<T>;
  static constexpr int PLANES = 1;
};
struct Frag3 {
  Frag<bf16> p[3];
};
template <>
struct MatrixType<float> {
  using Elem = bf16;
  using Opd = Frag3;
  static constexpr int PLANES = 3;  // of a tile in LDS
};
template <class T>
using Elem = typename MatrixType<T>::Elem;
template <class T>
using Opd = typename MatrixType<T>::Opd;
template <class T>
constexpr int kPlanes = MatrixType<T>::PLANES;

__device__ __forceinline__ f32x16 mma32(Frag<bf16> a, Frag<bf16> b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32(Frag<f16> a, Frag<f16> b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32(const Frag3& a, const Frag3& b, f32x16 c) {
  // the smallest first
  c = mma32(a.p[2], b.p[0], c);
  c = mma32(a.p[0], b.p[2], c);
  c = mma32(a.p[1], b.p[1], c);
  c = mma32(a.p[1], b.p[0], c);
  c = mma32(a.p[0], b.p[1], c);
  return mma32(a.p[0], b.p[0], c);
}
// Eight float32 values as an operand.
template <class T>
__device__ __forceinline__ Opd<T> operand_of(const float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    Frag<T> f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (T)v[i];
    return f;
  } else {
    Frag3 f;
    float rest[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) rest[i] = v[i];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f.p[k][i] = (bf16)rest[i];
#pragma unroll
      for (int i = 0; i < 8; ++i) rest[i] -= (float)f.p[k][i];
    }
    return f;
  }
}
template <class T>
__device__ __forceinline__ Opd<T> operand_of(const Raw8<T>& r) {
  if constexpr (sizeof(T) == 2) {
    Frag<T> f;
    __builtin_memcpy(&f, &r, sizeof(f));
    return f;
  } else {
    float v[8];
    unpack8(v, r);
    return operand_of<T>(v);
  }
}

// 16-wide products (single tokens, whose time is the memory's): float32's own instructions, of depth 4.  The same
// eight values feed eight of them, instruction i taking value i of every lane: each covers k = i, 8 + i, 16
// + i and 24 + i, and all eight every k once, in both operands alike.
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
template <class Layout, class T>
__device__ __forceinline__ void lds_column4(T (&v)[4], const T* tile, int row0, int col0) {
  const int i = threadIdx.x & 15;
  if constexpr (sizeof(T) == 2) {
    const T* p = tile + Layout::at(row0 + (i >> 2), col0 + (i & 3) * 4);
    const s16x4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)p);
    __builtin_memcpy(v, &t, sizeof(t));
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = tile[Layout::at(row0 + r, col0 + i)];
  }
}
// Eight k as rows a .. a + 3 and b .. b + 3 of a tile, at column col0 + (lane % 16).
template <class Layout, class T>
__device__ __forceinline__ Frag<T> lds_column_frag(const T* tile, int a, int b, int col0) {
  T lo[4], hi[4];
  lds_column4<Layout>(lo, tile, a, col0);
  lds_column4<Layout>(hi, tile, b, col0);
  Frag<T> f;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    f[r] = lo[r];
    f[4 + r] = hi[r];
  }
  return f;
}
// The same as operands of 32-wide products, from a tile of kPlanes planes `plane` apart: eight values in a row
// at p, or of a column.
template <class T>
__device__ __forceinline__ Opd<T> lds_operand(const Elem<T>* p, int plane) {
  if constexpr (sizeof(T) == 2) {
    return lds_frag(p);
  } else {
    Frag3 f;
#pragma unroll
    for (int k = 0; k < 3; ++k) f.p[k] = lds_frag(p + k * plane);
    return f;
  }
}
template <class T, class Layout>
__device__ __forceinline__ Opd<T> lds_column_operand(const Elem<T>* tile, int plane, int a, int b, int col0) {
  if constexpr (sizeof(T) == 2) {
    return lds_column_frag<Layout>(tile, a, b, col0);
  } else {
    Frag3 f;
#pragma unroll
    for (int k = 0; k < 3; ++k) f.p[k] = lds_column_frag<Layout>(tile + k * plane, a, b, col0);
    return f;
  }
}

// Where value (row, col) of a tile (of 16-bit values) lies in LDS when the tile is read both by rows (16 bytes a
// lane, 16 rows at a time) and by columns (lds_column4: 4 rows of 64 bytes at a time).  A row's chunks of 16
// bytes are exchanged by an exclusive or with a number made of the row's, so that either read finds its 16
// chunks on distinct banks: rows 0 .. 15 have distinct numbers (of those that share banks), and four
// consecutive rows from a multiple of four differ in the bits that tell blocks of 64 bytes apart.  Rows of
// 96 are laid out as 128.
template <int DP>
struct BothWays {
  static constexpr int S = DP == 96 ? 128 : DP;
  static __device__ __forceinline__ int at(int row, int col) {
    const int f = S == 128 ? ((row & 3) << 2) | ((row >> 2) & 3)
                  : S == 64 ? ((row & 2) << 1) | ((row >> 2) & 3) : (row >> 2) & 3;
    return row * S + ((((col >> 3) ^ f) << 3) | (col & 7));
  }
};
// Rows of a fixed stride.
template <int STRIDE>
struct Strided {
  static constexpr int S = STRIDE;
  static __device__ __forceinline__ int at(int row, int col) { return row * STRIDE + col; }
};
// Rows padded by 16 bytes: 16-byte reads of 16 rows fall on distinct banks.
template <int DP>
using Padded = Strided<DP + 8>;

// Tiles of 64 rows that a workgroup of 256 threads brings from memory through registers into LDS: fetch()
// starts the loads, put() stores what came.  Rows from `end` on and columns past the head size are zeros.
//
// FAST: the head size is a multiple of eight and fast_rows() holds of the tensor.  A
// thread's byte offsets within a tile are then the same for every tile, the tile's address is scalar,
// and the buffer's range check makes the zeros: no vector arithmetic for a tile.  Otherwise 16-bit types read ahead
// (kReadAhead), float32 takes load_ahead8 with 64-bit addresses for every row, and keep8 when it goes to LDS.

// Eight values of a row of a tensor whose first n belong to it, without waiting for them: all eight are read where
// that is in the tensor (`inside`: a row follows, and rows are at least eight values apart), and keep8 clears
// the others later.  Reading a head's last values one by one instead, which their use waits for at once, took
// 38 us in place of 17.6 (5 x 269 queries over up to 1043 keys, 12 heads on 4, size 86 in place of 88).
template <class T>
__device__ __forceinline__ void load_ahead8(Raw8<T>& r, const T* p, int n, bool inside) {
  if (n >= 8 || (n > 0 && inside)) {
    load_whole8(r, p, true);
  } else {
    load_raw8(r, p, n);
  }
}
template <class T>
__device__ __forceinline__ void keep8(Raw8<T>& r, int n) {
#pragma unroll
  for (int i = 0; i < Raw8<T>::N; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      constexpr int per = 4 / (int)sizeof(T);  // values of a register
      const int first = (i * 4 + j) * per;
      const uint32_t part = per == 2 && n == first + 1 ? 0xffffu : 0u;
      r.q[i][j] &= n >= first + per ? 0xffffffffu : part;
    }
}
// Whether rows that are not FAST are read ahead without a branch a chunk, whose loads are waited for where the branches
// meet.  Every lane reads eight values of its tensor (TileLoader: those of the last row that would end past it end with
// it; load_chunks: those of a row's last chunk end with the row), and what does not belong is cleared on the way to LDS.
// Not so float32, whose tiles are short of vector instructions, not of loads.
// us, with a branch a chunk and without: 8 x 1024 x 12 x 81, window 256, a step 207 and 183; 2 x 2048 x 8 x 115, causal,
// forward 80.5 and 61, backward 208 and 190; a tree of 64 nodes, 24 heads on 8 of size 97 over 68762 tokens 342 and 166;
// float32 2 x 1024 x 8 x 81 forward 63.8 and 67.1, backward 167 and 179.
template <class T, bool FAST>
constexpr bool kReadAhead = !FAST && sizeof(T) == 2;
// All eight values one place down.
template <class T>
__device__ __forceinline__ void drop_first(Raw8<T>& r) {
  uint32_t w[Raw8<T>::N * 4 + 1] = {};
  __builtin_memcpy(w, &r, sizeof(r));
#pragma unroll
  for (int k = 0; k < Raw8<T>::N * 4; ++k) w[k] = sizeof(T) == 4 ? w[k + 1] : w[k] >> 16 | w[k + 1] << 16;
  __builtin_memcpy(&r, w, sizeof(r));
}
// Of global memory: loads whose address space is open are waited for with the LDS reads.
typedef const __attribute__((address_space(1))) char* GlobalBytes;
template <bool AHEAD>
struct TileUnderWay {};
template <>
struct TileUnderWay<true> {
  int from, till;
  bool near;  // its rows are read ahead
};
template <class T, int DP, bool FAST>
struct TileLoader : TileUnderWay<kReadAhead<T, FAST>> {
  static constexpr bool AHEAD = kReadAhead<T, FAST>;
  static constexpr int CPR = DP / 8;                    // chunks of eight values a row
  static constexpr int PER = kTileRows * CPR / 256;     // chunks a thread brings
  static constexpr bool EVEN = 256 % CPR == 0;          // all of the same columns
  const T* base;
  int64_t stride;
  int dim, rows;  // rows: of the tensor
  uint32_t offset[PER];
  Raw8<T> r[PER];

  __device__ __forceinline__ void init(const T* b, int64_t s, int d, int n) {
    base = b;
    stride = s;
    dim = d;
    rows = n;
    if constexpr (FAST) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int c = threadIdx.x + i * 256, row = c / CPR, col = (c % CPR) * 8;
        offset[i] = col < dim ? (uint32_t)(row * (int)stride + col) * (uint32_t)sizeof(T) : 0x80000000u;
      }
    } else if constexpr (AHEAD) {
      this->near = stride >= 8 && stride < ((int64_t)1 << 31) / ((int)sizeof(T) * kTileRows) &&
             (int64_t)(rows - 1) * stride + dim >= 8;
#pragma unroll
      for (int i = 0; i < (EVEN ? 1 : PER); ++i) {
        const int c = threadIdx.x + i * 256, row = c / CPR, col = (c % CPR) * 8;
        offset[i] = this->near ? (uint32_t)(row * (int)stride + (col < dim ? col : 0)) * (uint32_t)sizeof(T) : 0u;
      }
    }
  }
  // row0 and end are the same in all lanes
  __device__ __forceinline__ void fetch(int row0, int end) {
    if constexpr (FAST) {
      const int left = end - row0 < kTileRows ? end - row0 : kTileRows;
      const uint32_t bytes = left > 0 ? (uint32_t)((left - 1) * (int)stride + dim) * (uint32_t)sizeof(T) : 0u;
      const auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base + (int64_t)row0 * stride), (short)0,
                                                        (int)bytes, 0x00020000);
#pragma unroll
      for (int i = 0; i < PER; ++i)
#pragma unroll
        for (int j = 0; j < Raw8<T>::N; ++j)
          r[i].q[j] = __builtin_amdgcn_raw_buffer_load_b128(rs, (int)offset[i] + 16 * j, 0, 0);
    } else if constexpr (AHEAD) {
      this->from = row0;
      this->till = end;
      uintptr_t tile = (uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
      int64_t last = 0;
      if (this->near) {
        tile = (uintptr_t)(base + (int64_t)row0 * stride);
        last = ((int64_t)(rows - 1 - row0) * stride + dim - 8) * (int)sizeof(T);
        if (last < 0) tile += last;
      }
      const uint32_t next = this->near ? 256 / CPR * (uint32_t)stride * (uint32_t)sizeof(T) : 0;  // EVEN
      const uint32_t most = (uint32_t)(last < 0 ? 0 : last < 0x7fffffff ? last : 0x7fffffff);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const uint32_t at = EVEN ? offset[0] + i * next : offset[i];
        const GlobalBytes p = (GlobalBytes)tile + (at < most ? at : most);
#pragma unroll
        for (int j = 0; j < Raw8<T>::N; ++j) r[i].q[j] = ((const __attribute__((address_space(1))) u32x4_any*)p)[j];
      }
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int c = threadIdx.x + i * 256, row = c / CPR, col = (c % CPR) * 8;
        load_ahead8(r[i], base + (int64_t)(row0 + row) * stride + col, row0 + row < end ? dim - col : 0,
                    stride >= 8 && row0 + row + 1 < rows);
      }
    }
  }
  // into a tile of kPlanes planes of kTileRows rows
  template <class Layout>
  __device__ __forceinline__ void put(Elem<T>* lds) {
    int thread = threadIdx.x;
    if constexpr (AHEAD) {
      // What follows from it is not held from tile to tile: 2 x 2048 x 8 x 115 would spill, 8 x 1024 x 12 x 50 run at two
      // waves a SIMD, 31 and 34 us.  At 32 there are registers for it: a tree of size 18 237 and 217 us.
      if constexpr (DP > 32) asm volatile("" : "+v"(thread));
      if (!this->near) {
#pragma unroll 1
        for (int c = thread; c < PER * 256; c += 256) {
          const int row = this->from + c / CPR, col = (c % CPR) * 8;
          Raw8<T> values;
          load_raw8(values, base + (int64_t)row * stride + col, row < this->till ? dim - col : 0);
          *reinterpret_cast<Frag<T>*>(lds + Layout::at(c / CPR, (c % CPR) * 8)) = operand_of<T>(values);
        }
        return;
      }
      if (this->from + kTileRows >= rows) {  // the last row's last values were read as the last of eight
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int c = thread + i * 256, col = (c % CPR) * 8;
          if (this->from + c / CPR == rows - 1 && col < dim)
            for (int n = dim - col; n < 8; ++n) drop_first(r[i]);
        }
      }
      if (this->from + kTileRows > this->till) {
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if (this->from + (thread + i * 256) / CPR >= this->till) keep8(r[i], 0);
      }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = threadIdx.x + i * 256;
      Elem<T>* p = lds + Layout::at(c / CPR, (c % CPR) * 8);
      Raw8<T> kept = r[i];
      if constexpr (AHEAD) keep8(kept, dim - (thread + (EVEN ? 0 : i * 256)) % CPR * 8);
      else if constexpr (!FAST) keep8(kept, dim - (c % CPR) * 8);
      const Opd<T> v = operand_of<T>(kept);
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<Frag<T>*>(p) = v;
      } else {
#pragma unroll
        for (int k = 0; k < 3; ++k) *reinterpret_cast<Frag<bf16>*>(p + k * kTileRows * Layout::S) = v.p[k];
      }
    }
  }
};
// Tiles in LDS: two, one being read while the other is filled, where they fit.
template <class T>
constexpr int kBufs = sizeof(T) == 2 ? 2 : 1;

// A row of a tensor in the order of operands: lane l holds chunks of eight values, 8 (l / 32) + 16 kk (32-wide products).
// WHOLE: the head size is a multiple of eight.  Otherwise the last chunk is read as the row's last eight values, and
// those that belong to the chunk before are dropped when all loads are under way.
template <class T, bool WHOLE>
__device__ __forceinline__ void load_chunk(Raw8<T>& r, const T* row, int kk, int dim, bool ok) {
  const int col = kk * 16 + ((threadIdx.x & 63) >> 5) * 8;
  if constexpr (WHOLE) load_whole8(r, row + col, ok && col < dim);
  else load_raw8(r, row + col, ok ? dim - col : 0);
}
template <class T, int N>
__device__ __forceinline__ void load_chunks(Raw8<T> (&r)[N], const T* row, int dim, bool ok) {
  const int col = ((threadIdx.x & 63) >> 5) * 8;
  if (dim < 8) {
#pragma unroll
    for (int kk = 0; kk < N; ++kk) load_raw8(r[kk], row + col + kk * 16, ok ? dim - col - kk * 16 : 0);
    return;
  }
#pragma unroll
  for (int kk = 0; kk < N; ++kk) load_whole8(r[kk], row + (col + kk * 16 < dim - 8 ? col + kk * 16 : dim - 8), ok);
#pragma unroll
  for (int kk = 0; kk < N; ++kk) {
    if (kk * 16 + 16 > dim)
      for (int n = col + kk * 16 - (dim - 8) < 8 ? col + kk * 16 - (dim - 8) : 8; n > 0; --n) drop_first(r[kk]);
  }
}
template <class T, int DP, bool WHOLE>
__device__ __forceinline__ void load_operand(Opd<T> (&f)[DP / 16], const T* row, int dim, bool ok) {
  if constexpr (!kReadAhead<T, WHOLE>) {
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      Raw8<T> r;
      load_chunk<T, WHOLE>(r, row, kk, dim, ok);
      f[kk] = operand_of<T>(r);
    }
  } else {
    Raw8<T> r[DP / 16];
    load_chunks(r, row, dim, ok);
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) f[kk] = operand_of<T>(r[kk]);
  }
}
// Waits for operands.  Without WHOLE they come through branches, and a loop that uses them would wait at their first use
// for all loads, its own next tile's too.
template <class T, bool WHOLE, int N>
__device__ __forceinline__ void wait_operands(Opd<T> (&f)[N]) {
  if constexpr (kReadAhead<T, WHOLE>) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      u32x4_any w;
      __builtin_memcpy(&w, &f[k], sizeof(w));
      asm volatile("" : "+v"(w));
      __builtin_memcpy(&f[k], &w, sizeof(w));
    }
  }
}
// A result whose columns are rows of a tensor: the lane's row, values 8 r4 + 4 (l / 32) .. + 3 of each 32.
template <class T, int DP, bool WHOLE>
__device__ __forceinline__ void store_result(T* row, const f32x16 (&v)[DP / 32], float scale, int dim) {
  const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      const int col = d * 32 + r4 * 8 + half * 4;
      const float x0 = v[d][r4 * 4] * scale, x1 = v[d][r4 * 4 + 1] * scale, x2 = v[d][r4 * 4 + 2] * scale,
                  x3 = v[d][r4 * 4 + 3] * scale;
      if (WHOLE || col + 4 <= dim) {
        if (col < dim) store4(row + col, x0, x1, x2, x3);
      } else {
        const float x[4] = {x0, x1, x2, x3};
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (col + r < dim) row[col + r] = (T)x[r];
      }
    }
}

// The larger of the two; a NaN stays a NaN (one instruction for three operands).
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Nothing is moved across these points by the instruction scheduler.  16-bit types: loads from LDS issued before
// one are under way together, where the scheduler would issue each just before its use to save registers.
// float32, whose operands are three times as large and feed six instructions each: few are held at a time,
// where it would load all of them at once.
template <class T>
__device__ __forceinline__ void fence_schedule() {
  if constexpr (sizeof(T) == 2) __builtin_amdgcn_sched_barrier(0);
}
template <class T>
__device__ __forceinline__ void fence_operands() {
  if constexpr (sizeof(T) == 4) __builtin_amdgcn_sched_barrier(0);
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_hw(float x) { return __builtin_amdgcn_logf(x); }
constexpr float kLog2E = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// The other half's value: lane l gets lane l ^ 32's.
__device__ __forceinline__ float other_half(float v) {
  const uint32_t u = __float_as_uint(v);
  // the first result has the lower half's value in both halves, the second the upper half's
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}
// Over both halves, without choosing.
__device__ __forceinline__ float max_halves(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return max_nan(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// A value that is the same in all lanes of the wave, as a scalar: branches on it are then scalar branches and
// addresses from it scalar addresses.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
  return (int64_t)(((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32) | (uint32_t)uniform((int)v));
}

// The work of workgroup `block` when works are numbered heaviest first.  Every other `cus` of them (one for
// each compute unit) are taken in reverse, so that where several workgroups share a compute unit from
// the start, the one that got the heaviest first gets the lightest next.  In units of eight, so that a
// work stays with its die (workgroups go to the eight dies in turn, and heads vary fastest).
__device__ __forceinline__ uint32_t work_order(uint32_t block, uint32_t blocks, uint32_t cus) {
  const uint32_t round = block / cus, first = round * cus;
  if (!(round & 1) || first + cus > blocks || cus % 8) return block;
  const uint32_t r = block - first;
  return first + (cus / 8 - 1 - r / 8) * 8 + r % 8;
}

// The sequence with the `rank`-th most keys (ties: the lower number), so that workgroups can be numbered longest
// sequence first although only the device knows the lengths.  Batches of up to 64 (a lane each); others, and
// those without lengths, in their own order.  Every lane of the wave calls it with the same rank.
//
// The rank-th largest of the lanes' numbers length * 64 + 63 - lane, one bit after the other from the top:
// it is among those with the bit set if they are more than rank, else among the others.
constexpr int kMostRanked = 64;
__device__ __forceinline__ int ranked_sequence(const AttnArgs& a, int rank) {
  if (!a.lengths || a.batch > kMostRanked) return rank;
  const int lane = threadIdx.x & 63, batch = (int)a.batch, keys = (int)a.keys;
  int len = lane < batch ? a.lengths[lane] : 0;
  len = len < 0 ? 0 : len < keys ? len : keys;
  const uint64_t number = lane < batch ? (uint64_t)len * 64 + (63 - lane) : 0;
  uint64_t left = batch == 64 ? ~0ull : (1ull << batch) - 1;
  for (int bit = 37 - __builtin_clz((uint32_t)keys | 1u); bit >= 0; --bit) {
    const uint64_t set = __ballot((number >> bit) & 1) & left;
    const int count = __popcll(set);
    if (rank < count) {
      left = set;
    } else {
      rank -= count;
      left &= ~set;
    }
  }
  return uniform((int)__builtin_ctzll(left));
}

// Which keys a sequence's queries may see: j < len, and with causal j <= i + off.  Token numbers are 32 bits
// (the C entry refuses more than 2^30), so that comparisons of wave-uniform ones are scalar.
constexpr int kFar = (1 << 30) - 1;  // i + kFar + 1 does not overflow and is past every key
//
// Within a window (kWindow) a query at position p = i + off sees of these the last `window` and the first
// `sinks`.  Of a tree (kTree) query i is node i, the key base + i is its own; it sees the keys below base, and of the
// nodes those in its line of ancestors.
enum Mask { kAll, kWindow, kTree };
struct Allowed {
  int len;  // keys of this sequence
  int off;
  int window, sinks;
};
// For the sequence b that a whole wave works on.
__device__ __forceinline__ Allowed allowed_keys(const AttnArgs& a, int64_t b) {
  Allowed w;
  const int keys = (int)a.keys;
  int len = keys;
  if (a.lengths) {
    const int l = uniform(a.lengths[b]);
    len = l < 0 ? 0 : l < keys ? l : keys;  // a length past the tensor would read past it
  }
  w.len = len;
  const int given = a.causal_offset > kFar ? kFar : (int)a.causal_offset;
  w.off = !a.causal ? kFar : a.bottom_right ? len - (int)a.queries : given;
  w.window = (int)a.window;
  w.sinks = (int)a.sinks;
  return w;
}
// First key that query i may not see.
__device__ __forceinline__ int key_end(const Allowed& w, int i) {
  const int e = i + w.off + 1;
  return e < 0 ? 0 : e < w.len ? e : w.len;
}

// First key of query i's window.
__device__ __forceinline__ int window_begin(const Allowed& w, int i) {
  const int p = i + w.off;
  return p < w.window ? 0 : p - w.window + 1;
}

// Which keys of a tile from j0 on a query sees that sees those below `end`, of these from `begin` on or below `sinks`; as
// bits, of the half's values: bit 8 (r / 4) + r % 4 of word t is value r of 32 t's (the products' rows, above).
//
// Two instructions a value then hide what is not seen; a comparison for each value and limit takes up to six, and in a
// window of few tiles most tiles have some hidden: bfloat16 8 x 1024 x 12 x 64 with a window of 256 and 4 sinks, us:
// forward 21.7 -> 19.9, query pass 33.7 -> 28.7, key pass 41.3 -> 38.1.  (Branches for tiles with one limit only, with
// comparisons: 24.5, 29.9, 40.1; the compiler keeps their results in scalar registers and spills.)
struct Seen {
  uint32_t w[2];
};
__device__ __forceinline__ uint64_t bits_below(int n) { return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1; }
__device__ __forceinline__ Seen seen_keys(int j0, int end, int begin, int sinks) {
  const uint64_t bits = bits_below(end - j0) & (~bits_below(begin - j0) | bits_below(sinks - j0));
  const int shift = (threadIdx.x & 32) >> 3;
  return {{(uint32_t)bits >> shift, (uint32_t)(bits >> 32) >> shift}};
}
// All ones where bit n is set.
__device__ __forceinline__ uint32_t bit_mask(uint32_t w, int n) { return (uint32_t)__builtin_amdgcn_sbfe((int)w, n, 1); }
__device__ __forceinline__ float masked_score(float s, uint32_t mask) {
  return __uint_as_float((__float_as_uint(s) & mask) | (~mask & 0xff800000u));  // minus infinity
}
__device__ __forceinline__ float masked_term(float s, uint32_t mask) { return __uint_as_float(__float_as_uint(s) & mask); }

// The keys that a block of queries walks over, STEP at a time, every STRIDE-th step: begin .. end; within a
// window 0 .. head, the sinks before it, and then from the first query's window on.  j is a step's first
// key, and keys from stop() on are not of it.
template <int MASK, int STEP, int STRIDE = 1>
struct Walk {
  int j, end;
  __device__ __forceinline__ bool live() const { return j < end; }
  __device__ __forceinline__ bool more() const { return j + STEP * STRIDE < end; }
  __device__ __forceinline__ int stop() const { return end; }
  __device__ __forceinline__ int next() const { return j + STEP * STRIDE; }
  __device__ __forceinline__ int next_stop() const { return end; }
  __device__ __forceinline__ void step() { j += STEP * STRIDE; }
};
template <int STEP, int STRIDE>
struct Walk<kWindow, STEP, STRIDE> {
  int t, t_end, head_steps, head, lo, end, j;
  __device__ __forceinline__ bool live() const { return t < t_end; }
  __device__ __forceinline__ bool more() const { return t + STRIDE < t_end; }
  __device__ __forceinline__ int at(int n) const { return n < head_steps ? n * STEP : lo + (n - head_steps) * STEP; }
  __device__ __forceinline__ int stop_at(int n) const { return n < head_steps ? head : end; }
  __device__ __forceinline__ int stop() const { return stop_at(t); }
  __device__ __forceinline__ int next() const { return at(t + STRIDE); }
  __device__ __forceinline__ int next_stop() const { return stop_at(t + STRIDE); }
  __device__ __forceinline__ void step() { j = at(t += STRIDE); }
};
// Range `split` of split_len keys (a multiple of 64, or all) of the walk of queries first .. last, step `at` of it.
template <int STEP, int STRIDE = 1>
__device__ __forceinline__ Walk<kWindow, STEP, STRIDE> window_walk(const AttnArgs& a, const Allowed& w, int first, int last,
                                                                   int split, int at) {
  Walk<kWindow, STEP, STRIDE> k;
  k.end = key_end(w, last);
  k.lo = window_begin(w, first);
  k.head = w.sinks < k.lo ? w.sinks : k.lo;
  if (k.head > k.end) k.head = k.end;
  if (w.sinks >= k.lo) k.lo = k.head = 0;  // nothing between sinks and window
  k.head_steps = (k.head + STEP - 1) / STEP;
  const int steps = k.head_steps + (k.end > k.lo ? (k.end - k.lo + STEP - 1) / STEP : 0);
  const int per_range = a.splits > 1 ? (int)(a.split_len / STEP) : steps, begin = split * per_range;
  k.t_end = begin + per_range < steps ? begin + per_range : steps;
  k.t = begin + at;
  k.j = k.at(k.t);
  return k;
}
// Tiles that the longest walk of a block of `block` queries takes (host).
inline int64_t window_tiles(const AttnArgs& a, int64_t block) {
  const int64_t most = a.window + std::min(a.queries, block) - 1;
  return (std::min(most, a.keys) + kTileRows - 1) / kTileRows + (std::min(a.sinks, a.keys) + kTileRows - 1) / kTileRows;
}

// Which block of queries (of 128) of which head a workgroup takes, and which range of keys.  Heads vary fastest,
// those that share a key head a multiple of the key heads apart, then ranges, then blocks, the last queries
// (causal: those with the most keys) first.  With lengths the longest sequence's work comes first instead.
struct RowsWork {
  int64_t b, hk, h;
  int block, split;
};
__device__ __forceinline__ RowsWork rows_work(const AttnArgs& a) {
  const uint32_t kvh = (uint32_t)a.kv_heads, group = (uint32_t)a.heads / kvh, splits = (uint32_t)a.splits;
  const uint32_t blocks = (uint32_t)((a.queries + 127) / 128);
  const uint32_t id = work_order(blockIdx.x, gridDim.x, (uint32_t)a.cus);
  const bool ranked = a.lengths && a.batch <= kMostRanked;
  const uint32_t kvb = ranked ? kvh : (uint32_t)a.batch * kvh, nh = kvb * group;
  const uint32_t head = id % nh, kv = head % kvb;
  uint32_t rest = id / nh;
  RowsWork w;
  w.split = uniform((int)(rest % splits));
  rest /= splits;
  w.block = uniform((int)(blocks - 1 - rest % blocks));
  w.b = ranked ? ranked_sequence(a, uniform((int)(rest / blocks))) : uniform((int)(kv / kvh));
  w.hk = uniform((int)(kv % kvh));
  w.h = w.hk * group + uniform((int)(head / kvb));
  return w;
}

}  // namespace lwl
