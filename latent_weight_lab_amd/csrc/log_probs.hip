// Log probabilities of given tokens, the entropy and the most probable alternatives, and their gradient.
//
// Forward: one pass over a row with a running maximum m, S = sum exp(z - m) and A = sum exp(z - m) (z - m) a thread,
// joined at the end in a fixed order:
//
//   log p_t = (z_t - m) - log S,  H = log S - A / S
//
// m starts at -FLT_MAX, so that a row of minus infinities sums zeros and nothing is NaN.
//
// Without the entropy m is raised lazily (kSlack), and to the largest value at the end.  With it, m is the largest value
// so far: every term of A, and what a raise adds to it, is then 0 or below, and nothing cancels.  (Raised lazily, a
// thread that met 0 after -8 held A = 8 e^8 and took 8 (1 + e^8) from it: entropies of some 5e-3 were off by up to 2.5e-4 of
// themselves, where 2e-5 are left.)
//
// The alternatives need no second pass over the row.  Each thread also keeps the largest of its values and the chunk of
// eight that it first met it in; groups of threads keep the largest of these pairs.  The top-th largest group's bounds the
// answer from below.  The chunks of the few threads that reach it are looked at again, by all threads, and what reaches it
// there is ranked by counting.  Pairs are ordered by value, then by the lower index, so that of equal values no more than
// the first few pass.  (Each such thread reading its own part again: 16 x 50304 with five alternatives 37 us, so 10.)
//
// Bound by memory where rows are many: bfloat16 8192 x 50257 in rows of 50304 139 us (5.9 TB/s), float32 264 us (6.2);
// 512 x 50304 with one alternative 14.0 us (3.7 TB/s, two rows for a compute unit at once).  Few rows are bound by one
// compute unit: 16 x 50304 with the entropy and five alternatives 9.8 us, some 4 of them after the row has been read.
//
// Backward: one pass that reads the logits and writes their gradient; tokens that are asked about are written once more
// afterwards by the workgroup whose range they lie in, with all gradients given for them in the order given.  8192 x 50257
// bfloat16 285 us (5.8 TB/s of reading and writing), float32 584 (5.6).
#include <algorithm>
#include <cfloat>

#include "layer_device.h"
#include "layer_launch.h"

namespace lwl {
namespace {

constexpr float kLog2E = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Workgroups along a grid's first axis; more go on along the second.  A launch holds an axis' threads in 32 bits and drops,
// without an error, what is above.
constexpr uint32_t kGridX = 1u << 21;
inline dim3 grid_of(int64_t blocks) {
  return dim3((unsigned)std::min<int64_t>(blocks, kGridX), (unsigned)((blocks + kGridX - 1) / kGridX));
}
__device__ __forceinline__ uint32_t block_number() { return blockIdx.y * kGridX + blockIdx.x; }

template <class T>
__device__ __forceinline__ const T* row_of(const LogProbArgs& a, int64_t r) {
  return (const T*)a.logits + r / a.inner * a.outer_stride + r % a.inner * a.inner_stride;
}

// Numbers in the order of the values, all above 0: NaN is the largest, both zeros are one.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  return v != v ? 0xffffffffu : u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) {
  return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
// A value and where it lies, in the order wanted: larger values, then lower places, are larger numbers.
__device__ __forceinline__ uint64_t pair_of(uint32_t order, uint32_t place) {
  return (uint64_t)order << 32 | (uint32_t)~place;
}

// Eight values of a row, minus infinity past its end.  Chunks begin with the row, at any alignment, so that a row's results
// have the same bits wherever it lies.  Dense rows of odd length cost that a sixth of the time: bfloat16 8192 x 50257, dense,
// 166 us, in rows of 50304 142; with chunks at multiples of 16 bytes 141 both.
template <class T>
__device__ __forceinline__ void chunk_values(float (&v)[8], const Raw8<T>& raw, int64_t left) {
  unpack8(v, raw);
  if (left < 8) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? v[i] : -INFINITY;
  }
}

struct Sums {
  float m, s, a;
};
template <bool ENTROPY>
__device__ __forceinline__ void raise(Sums& t, float next) {
  const float shrink = exp2_hw((t.m - next) * kLog2E);
  if constexpr (ENTROPY) t.a = shrink > 0.0f ? (t.a + t.s * (t.m - next)) * shrink : 0.0f;
  t.s *= shrink;
  t.m = next;
}
// Over LANES consecutive lanes; all of them get it.
template <bool ENTROPY, int LANES>
__device__ __forceinline__ void join_lanes(Sums& t) {
  float m = t.m;
#pragma unroll
  for (int k = 1; k < LANES; k *= 2) m = fmaxf(m, __shfl_xor(m, k, 64));
  raise<ENTROPY>(t, m);
  t.s = lanes_sum<LANES>(t.s);
  if constexpr (ENTROPY) t.a = lanes_sum<LANES>(t.a);
}

// Without the entropy a thread's sums are taken relative to its largest value when that was last raised, which happens where
// one lies more than this above it, and to the largest at the end.
constexpr float kSlack = 8.0f;
constexpr int kCandidates = 1024;
constexpr int kGroups = 128;  // of threads, whose largest values bound the alternatives: more than of these

template <class T, int THREADS, int U, bool ENTROPY, bool TOP>
__global__ __launch_bounds__(THREADS) void log_probs_forward(const LogProbArgs a) {
  constexpr int WAVES = THREADS / 64;
  __shared__ float lds_sums[3][WAVES];
  __shared__ uint64_t lds_best[TOP ? THREADS : 1], lds_cand[TOP ? kCandidates : 1], lds_bound;
  __shared__ int lds_count, lds_hot[TOP ? THREADS : 1], lds_hot_count;
  const int64_t row = block_number();
  if (row >= a.outer * a.inner) return;
  const T* x = row_of<T>(a, row);
  const int vocab = (int)a.vocab, chunks = (vocab + 7) / 8;
  Raw8<T> raw[U];
  const auto load = [&](int base) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = base + u * THREADS + (int)threadIdx.x;
      load_raw8(raw[u], x + (int64_t)c * 8, c < chunks ? vocab - c * 8 : 0);
    }
  };
  load(0);
  int64_t token = -1;
  float asked = 0.0f;
  if ((int)threadIdx.x < a.each) {
    token = a.tokens[row * a.each + threadIdx.x];
    if (token >= 0 && token < vocab) asked = (float)x[token];
  }
  Sums t = {-FLT_MAX, 0.0f, 0.0f};
  float best = -INFINITY;
  uint32_t best_chunk = threadIdx.x;
  // A chunk's values, and the largest of them.
  const auto look = [&](float (&v)[8], int u, int c) {
    chunk_values(v, raw[u], vocab - c * 8);
    const float most = max_nan(max_nan(max_nan(v[0], v[1]), max_nan(v[2], v[3])),
                               max_nan(max_nan(v[4], v[5]), max_nan(v[6], v[7])));
    if constexpr (TOP) {
      if (!(most <= best) && best == best) {  // the first of equal ones; a NaN stays
        best = most;
        best_chunk = (uint32_t)c;
      }
    } else {
      best = max_nan(best, most);
    }
    return most;
  };
  const auto add = [&](const float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = v[i] - t.m, e = exp2_hw(d * kLog2E);
      t.s += e;
      if constexpr (ENTROPY) t.a = fmaf(e, max_nan(d, -FLT_MAX), t.a);
    }
  };
  for (int base = 0; base < chunks; base += THREADS * U) {
    if (base > 0) load(base);
    const int c = base + (int)threadIdx.x;
    if constexpr (ENTROPY) {  // raised once for all chunks of a step: 16 x 50304 9.8 us, for each 10.2
      if (c >= chunks) break;
      float v[U][8], most = -INFINITY;
#pragma unroll
      for (int u = 0; u < U; ++u) most = fmaxf(most, look(v[u], u, c + u * THREADS));
      if (__any(most > t.m)) raise<true>(t, fmaxf(t.m, most));
#pragma unroll
      for (int u = 0; u < U; ++u) add(v[u]);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (c + u * THREADS >= chunks) break;
        float v[8];
        const float most = look(v, u, c + u * THREADS);
        if (__any(most > t.m + kSlack)) raise<false>(t, fmaxf(t.m, most));
        add(v);
      }
    }
  }
  raise<ENTROPY>(t, fmaxf(t.m, best));
  join_lanes<ENTROPY, 64>(t);
  if ((threadIdx.x & 63) == 0) {
    lds_sums[0][threadIdx.x >> 6] = t.m;
    lds_sums[1][threadIdx.x >> 6] = t.s;
    lds_sums[2][threadIdx.x >> 6] = t.a;
  }
  uint64_t mine = 0;
  if constexpr (TOP) {
    // threads without a value come last, each with a number of its own
    mine = (int)threadIdx.x < chunks ? pair_of(order_of(best), best_chunk) : (uint64_t)threadIdx.x;
    uint64_t group = mine;
#pragma unroll
    for (int k = 1; k < THREADS / kGroups; k *= 2) {
      const uint64_t other = (uint64_t)__shfl_xor((unsigned long long)group, k, 64);
      group = other > group ? other : group;
    }
    lds_best[threadIdx.x] = mine;
    if (threadIdx.x % (THREADS / kGroups) == 0) lds_cand[threadIdx.x / (THREADS / kGroups)] = group;
    if (threadIdx.x == 0) lds_count = lds_hot_count = 0;
  }
  __syncthreads();
  {
    const int w = threadIdx.x % WAVES;
    t = {lds_sums[0][w], lds_sums[1][w], lds_sums[2][w]};
    join_lanes<ENTROPY, WAVES>(t);
    // The first lane's for all: a lane's own term may enter its sum unrounded (a fused multiply and add), so lanes may
    // differ in the last bit, and which thread writes an alternative varies.
    const auto first = [](float v) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v))); };
    t = {first(t.m), first(t.s), first(t.a)};
  }
  const bool empty = t.s == 0.0f;  // nothing but minus infinities
  const float log_s = __logf(t.s);
  if ((int)threadIdx.x < a.each) {
    const float lp = token >= vocab ? NAN : empty ? -INFINITY : (asked - t.m) - log_s;
    a.log_probs[row * a.each + threadIdx.x] = token < 0 ? 0.0f : lp;
  }
  if (threadIdx.x == 0) {
    if (ENTROPY && a.entropy) a.entropy[row] = empty ? 0.0f : log_s - t.a / t.s;
    if (a.stats) {
      a.stats[row * 2] = t.m;
      a.stats[row * 2 + 1] = log_s;
    }
  }
  if constexpr (TOP) {
    const int top = a.top;
    {
      // the groups' ranks, each counted by a few lanes
      constexpr int LANES = THREADS / kGroups, PER = kGroups / LANES;
      const int part = threadIdx.x % LANES;
      const uint64_t group = lds_cand[threadIdx.x / LANES];
      int rank = 0;
#pragma unroll 16
      for (int i = 0; i < PER; ++i) rank += lds_cand[i * LANES + part] > group;
#pragma unroll
      for (int k = 1; k < LANES; k *= 2) rank += __shfl_xor(rank, k, 64);
      if (rank == top - 1 && part == 0) lds_bound = group;
    }
    __syncthreads();
    uint64_t bound = lds_bound;
    // lds_cand held the groups
    const auto candidates = [&](int c, const Raw8<T>& chunk) {
      float v[8];
      chunk_values(v, chunk, vocab - c * 8);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t order = order_of(v[i]);
        if (c * 8 + i < vocab && pair_of(order, (uint32_t)c) >= bound) {
          const int at = atomicAdd(&lds_count, 1);
          if (at < kCandidates) lds_cand[at] = pair_of(order, (uint32_t)(c * 8 + i));
        }
      }
    };
    // The chunks of the threads that pass are looked at by all threads: their own would read them one after the other.
    if (mine >= bound && (int)threadIdx.x < chunks) lds_hot[atomicAdd(&lds_hot_count, 1)] = (int)threadIdx.x;
    __syncthreads();
    const int hot = lds_hot_count, looks = hot * ((chunks + THREADS - 1) / THREADS);
    for (int i = threadIdx.x; i < looks; i += THREADS) {
      const int n = i / hot, c = n * THREADS + lds_hot[i - n * hot];
      if (c < chunks) {
        Raw8<T> chunk;
        load_raw8(chunk, x + (int64_t)c * 8, vocab - c * 8);
        candidates(c, chunk);
      }
    }
    __syncthreads();
    int count = lds_count;
    if (count > kCandidates) {
      // Few threads hold many of the largest values (sorted rows).  With the bound of single threads no more than `top` of
      // them pass; they go chunk by chunk in step, and whenever the next chunks may not fit, all but the `top` largest
      // so far are dropped.
      int rank = 0;
      for (int i = 0; i < THREADS; ++i) rank += lds_best[i] > mine;
      __syncthreads();  // all have read count
      if (threadIdx.x == 0) lds_count = 0;
      if (rank == top - 1) lds_bound = mine;
      __syncthreads();
      bound = lds_bound;
      for (int base = 0; base < chunks; base += THREADS) {
        const int c = base + (int)threadIdx.x;
        if (c < chunks && mine >= bound) {
          Raw8<T> chunk;
          load_raw8(chunk, x + (int64_t)c * 8, vocab - c * 8);
          candidates(c, chunk);
        }
        __syncthreads();
        count = lds_count;
        __syncthreads();  // all have read it
        if (count + top * 8 > kCandidates) {
          constexpr int PER = (kCandidates + THREADS - 1) / THREADS;
          uint64_t keep[PER];
          int at[PER];
#pragma unroll
          for (int k = 0; k < PER; ++k) {
            const int i = threadIdx.x + k * THREADS;
            keep[k] = i < count ? lds_cand[i] : 0;
            at[k] = 0;
            if (i < count)
              for (int j = 0; j < count; ++j) at[k] += lds_cand[j] > keep[k];
          }
          __syncthreads();
#pragma unroll
          for (int k = 0; k < PER; ++k)
            if ((int)threadIdx.x + k * THREADS < count && at[k] < top) lds_cand[at[k]] = keep[k];
          if (threadIdx.x == 0) lds_count = top;
          __syncthreads();
          count = top;
        }
      }
    }
    for (int i = threadIdx.x; i < count; i += THREADS) {
      const uint64_t one = lds_cand[i];
      int place = 0;
#pragma unroll 4
      for (int j = 0; j < count; ++j) place += lds_cand[j] > one;
      if (place < top) {
        a.top_log_probs[row * top + place] = empty ? -INFINITY : (value_of((uint32_t)(one >> 32)) - t.m) - log_s;
        a.top_tokens[row * top + place] = (int64_t)(uint32_t)~(uint32_t)one;
      }
    }
  }
}

constexpr int kListed = 128;     // tokens that a row's gradients are given for
// Chunks of a thread: with 2, 4 and 8, us: 8192 x 50257 bfloat16 285, 301, 320, float32 584, 611, 680; 1021 x 32003 34, 34, 41
// and 45, 47, 51.  Stores past the caches: 280 and 641 with 2, so a gradient that fits stays for its next reader.
constexpr int kBwdChunks = 2;
constexpr int kBwdRange = 256 * 8 * kBwdChunks;  // logits of a workgroup

template <class T, bool ENTROPY>
__global__ __launch_bounds__(256) void log_probs_backward(const LogProbArgs a, uint32_t ranges) {
  __shared__ int lds_token[kListed];
  __shared__ float lds_grad[kListed];
  const int64_t row = block_number() / ranges;
  if (row >= a.outer * a.inner) return;
  const int begin = (int)(block_number() % ranges) * kBwdRange;
  const T* x = row_of<T>(a, row);
  T* dz = (T*)a.grad_logits + row * a.vocab;
  const int vocab = (int)a.vocab, end = vocab - begin < kBwdRange ? vocab : begin + kBwdRange;
  const int listed = a.each + a.top;
  if ((int)threadIdx.x < listed) {
    const int i = threadIdx.x;
    const bool is_top = i >= a.each;
    const float* g = is_top ? a.grad_top : a.grad_log_probs;
    int64_t token = -1;
    if (g) token = is_top ? a.top_tokens[row * a.top + i - a.each] : a.tokens[row * a.each + i];
    const bool ok = token >= 0 && token < vocab;
    lds_token[i] = ok ? (int)token : -1;
    lds_grad[i] = ok ? g[is_top ? row * a.top + i - a.each : row * a.each + i] : 0.0f;
  }
  const float m = a.stats[row * 2], log_s = a.stats[row * 2 + 1];
  const bool empty = log_s == -INFINITY;
  const float gh = ENTROPY ? a.grad_entropy[row] : 0.0f, entropy = ENTROPY ? a.entropy[row] : 0.0f;
  __syncthreads();
  float total = 0.0f;
  for (int i = 0; i < listed; ++i) total += lds_grad[i];
  // what a logit's gradient is without those given for its token
  const auto spread = [&](float z) {
    const float lp = (z - m) - log_s, p = exp2_hw(lp * kLog2E);
    float f = -total;
    if constexpr (ENTROPY) f -= gh * (fmaxf(lp, -200.0f) + entropy);  // below that p is 0
    return empty ? 0.0f : p * f;
  };
  Raw8<T> raw[kBwdChunks];
#pragma unroll
  for (int u = 0; u < kBwdChunks; ++u) {
    const int at = begin + (u * 256 + (int)threadIdx.x) * 8;
    load_raw8(raw[u], x + at, end - at);
  }
#pragma unroll
  for (int u = 0; u < kBwdChunks; ++u) {
    const int at = begin + (u * 256 + (int)threadIdx.x) * 8;
    float v[8];
    unpack8(v, raw[u]);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = spread(v[i]);
    store8(dz + at, v, end - at);
  }
  __syncthreads();
  if ((int)threadIdx.x < listed && !empty) {
    const int token = lds_token[threadIdx.x];
    if (token >= begin && token < end) {
      float g = 0.0f;
      int first = -1;
      for (int j = 0; j < listed; ++j)
        if (lds_token[j] == token) {
          g += lds_grad[j];
          if (first < 0) first = j;
        }
      if (first == (int)threadIdx.x) dz[token] = (T)(spread((float)x[token]) + g);
    }
  }
}

template <class T, int THREADS, int U>
void forward(const LogProbArgs& a, hipStream_t s) {
  const dim3 grid = grid_of(a.outer * a.inner), block(THREADS);
  if (a.top > 0) {
    if (a.entropy) hipLaunchKernelGGL((log_probs_forward<T, THREADS, U, true, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((log_probs_forward<T, THREADS, U, false, true>), grid, block, 0, s, a);
  } else {
    if (a.entropy) hipLaunchKernelGGL((log_probs_forward<T, THREADS, U, true, false>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((log_probs_forward<T, THREADS, U, false, false>), grid, block, 0, s, a);
  }
}
// Threads of a row: few lose less at the ends of short rows, many bring more of a long row at a time.  bfloat16, us with 256,
// 512 and 1024: 2048 x 4000 with the entropy and five alternatives 12.3, 18, 29; 2048 x 16000 19.2, 22, 31; 8192 x 50257 in
// rows of 50304, neither, 141, 137, 139; 16 x 50304 12.7, 9.8, 9.8; 1 x 200000 33, 22.5, 20.
template <class T>
hipError_t run_forward(const LogProbArgs& a, hipStream_t s) {
  if (a.vocab > 65536 && a.outer * a.inner <= device_cus()) forward<T, 1024, 2>(a, s);
  else if (a.vocab > 16384) forward<T, 512, 2>(a, s);
  else forward<T, 256, 2>(a, s);
  return hipGetLastError();
}

template <class T>
hipError_t run_backward(const LogProbArgs& a, hipStream_t s) {
  const int64_t ranges = log_probs_bwd_ranges(a.vocab);
  const dim3 grid = grid_of(a.outer * a.inner * ranges);
  if (a.grad_entropy)
    hipLaunchKernelGGL((log_probs_backward<T, true>), grid, dim3(256), 0, s, a, (uint32_t)ranges);
  else
    hipLaunchKernelGGL((log_probs_backward<T, false>), grid, dim3(256), 0, s, a, (uint32_t)ranges);
  return hipGetLastError();
}

}  // namespace

int64_t log_probs_bwd_ranges(int64_t vocab) { return (vocab + kBwdRange - 1) / kBwdRange; }

hipError_t launch_log_probs_fwd(const LogProbArgs& a, hipStream_t s) {
  switch (a.dtype) {
    case kF32: return run_forward<float>(a, s);
    case kF16: return run_forward<f16>(a, s);
    case kBF16: return run_forward<bf16>(a, s);
  }
  return hipErrorInvalidValue;
}

hipError_t launch_log_probs_bwd(const LogProbArgs& a, hipStream_t s) {
  switch (a.dtype) {
    case kF32: return run_backward<float>(a, s);
    case kF16: return run_backward<f16>(a, s);
    case kBF16: return run_backward<bf16>(a, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace lwl
