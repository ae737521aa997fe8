// What the sequence operators share: element types, 4-wide loads, packed chains and their pieces, and the sums
// of partial results.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

namespace cufkb_seq {

constexpr unsigned kAll = 0xffffffffu;

// Dependent launches: the next kernel may start once all blocks of this one have said so, and waits for this one's results
// where it needs them.  Every block of a dependent kernel waits before it ends, so that its end implies this one's.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename T>
__device__ __forceinline__ float to_float(T v) {
  if constexpr (std::is_same_v<T, __half>) {
    return __half2float(v);
  } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    return __bfloat162float(v);
  } else {
    return static_cast<float>(v);
  }
}

template <typename T>
__device__ __forceinline__ T from_float(float v) {
  if constexpr (std::is_same_v<T, __half>) {
    return __float2half_rn(v);
  } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    return __float2bfloat16_rn(v);
  } else {
    return static_cast<T>(v);
  }
}

// N consecutive elements as one register block; VEC says that the address is aligned to the whole block.
template <typename T, int N>
struct alignas(sizeof(T) * N) Block {
  T v[N];
};

template <typename T, int N, bool VEC>
__device__ __forceinline__ Block<T, N> load_block(const T* p, int valid) {
  Block<T, N> out;
  if constexpr (VEC) {
    if (valid >= N) {
      out = *reinterpret_cast<const Block<T, N>*>(p);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) out.v[i] = from_float<T>(0.0f);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) out.v[i] = i < valid ? p[i] : from_float<T>(0.0f);
  }
  return out;
}

template <typename T, int N, bool VEC>
__device__ __forceinline__ void store_block(T* p, const Block<T, N>& b, int valid) {
  if constexpr (VEC) {
    if (valid >= N) *reinterpret_cast<Block<T, N>*>(p) = b;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i < valid) p[i] = b.v[i];
    }
  }
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp_fast(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Two floats in one 64-bit register: sm_100 multiplies and adds both in one instruction.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float a, float b) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 halves(Pair v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair exp2_pair(Pair v) {
  const float2 f = halves(v);
  return pair(exp2_fast(f.x), exp2_fast(f.y));
}
// A decay, exp(dt A) = 2^(dt A2) with A2 = A log2(e).  The exponential unit's results are low in the mean, by 0.5e-8 for exponents of -2^-8 and
// nearer to 0, by 1.8e-8 to 2.7e-8 from -2^-7 to -2^-4 (about an rms of 3e-8 to 4e-8; correct rounding would have 1.7e-8 and no mean), and a recurrence
// multiplies one decay per row: rounding averages out, a mean adds up.  2^-26 in the exponent raises the result by 1.03e-8: half of
// the mean where it is large, and no more off above than below where it is small.  It costs nothing, the product becomes an fma, and
// exponents of 0 still give 1.  Against 64 bits, relative: the gradient of A at 8192 x 2048 x 16 (bfloat16) 1.35e-6 without it and 0.77e-6
// with it, the last state at 16384 x 1024 x 16 5.3e-7 and 3.0e-7.  A correctly rounded exponential, made in 64 bits,
// gives 0.26e-6 and 1.5e-7, at four times the time.
constexpr float kDecayMean = 1.4901161e-8f;
__device__ __forceinline__ float decay(float dt, float A2) { return exp2_fast(fmaf(dt, A2, kDecayMean)); }
__device__ __forceinline__ Pair decay2(Pair dt, Pair A2) { return exp2_pair(fma2(dt, A2, pair(kDecayMean, kDecayMean))); }

__device__ __forceinline__ float sum_pair(Pair v) {
  const float2 f = halves(v);
  return f.x + f.y;
}
// Four floats of shared memory as two pairs.
__device__ __forceinline__ void load_pairs(Pair (&dst)[2], const float* p) {
  const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(p);
  dst[0] = v.x;
  dst[1] = v.y;
}

// 1 / (1 + exp(-v)): exp(-v) may overflow to inf, whose reciprocal is the right 0
__device__ __forceinline__ float sigmoid(float v) { return rcp_fast(1.0f + exp2_fast(-kLog2e * v)); }

__device__ __forceinline__ Pair sigmoid2(Pair v) {
  const float2 e = halves(mul2(v, pair(-kLog2e, -kLog2e)));
  const float2 d = halves(add2(pair(exp2_fast(e.x), exp2_fast(e.y)), pair(1.0f, 1.0f)));
  return pair(rcp_fast(d.x), rcp_fast(d.y));
}

// softplus(v) = max(v, 0) + log(1 + e), e = exp(-|v|), with log(1 + e) = 2 atanh(s), s = e / (2 + e) <= 1/3: small e (small steps) keep their
// relative accuracy.  The polynomial is atanh(s) / s in s^2, fitted over [0, 1/9] by exchange; it is off by at most 8e-9.
__device__ __forceinline__ float softplus(float v) {
  const float e = exp2_fast(-kLog2e * fabsf(v));
  const float s = e * rcp_fast(2.0f + e), q = s * s;
  float p = 0.14089165f;
  p = fmaf(p, q, 0.13980304f);
  p = fmaf(p, q, 0.20012455f);
  p = fmaf(p, q, 0.33333158f);
  p = fmaf(p, q, 1.0f);
  return fmaf(2.0f * s, p, fmaxf(v, 0.0f));
}

// ------------------------------------------------------------------------------------------
// packed chains
// ------------------------------------------------------------------------------------------
// Chains of one call.  With offsets, the rows past the last one are one more "chain" (index `count`), whose
// results are zero.  Offsets are clamped to [0, rows].
struct Chains {
  const int64_t* points;  // count + 1 offsets, or nullptr: equal lengths
  int64_t rows;
  int64_t uniform;  // rows of each chain when points is nullptr
  int64_t count;

  __device__ __forceinline__ int64_t first(int64_t s) const {
    if (points == nullptr) return s * uniform;
    if (s == 0) return 0;
    if (s > count) return rows;
    const int64_t p = points[s];
    return p < 0 ? 0 : (p > rows ? rows : p);
  }
  // The chain of a row, for one thread on its own.
  __device__ __forceinline__ int64_t of_row(int64_t row) const {
    if (points == nullptr) return row / uniform;
    int64_t lo = 0, hi = count;
    while (hi > lo) {
      const int64_t mid = (lo + hi + 1) >> 1;
      if (first(mid) <= row) {
        lo = mid;
      } else {
        hi = mid - 1;
      }
    }
    return lo;
  }
  __device__ __forceinline__ int64_t end(int64_t s) const {
    const int64_t a = first(s), b = first(s + 1);
    return b < a ? a : b;
  }
};

// A piece of at most `length` rows of one chain.  Chain s has the item numbers from key(s) = first(s) / length + s on:
// ceil(rows of s / length) (one for an empty chain) never reach key(s + 1), so the items of a call number at most
// rows / length + count + 1, a bound that the host knows without the offsets.  Numbers in between have no piece.
struct Piece {
  int64_t chain;
  int64_t first, end;              // the piece's rows
  int64_t chain_first, chain_end;  // the chain's rows
  int64_t index;                   // piece number within the chain
  bool valid;
  bool padding;  // the rows past the last offset
};

__host__ __device__ inline int64_t pieces_of(int64_t rows, int64_t length) { return rows > 0 ? (rows - 1) / length + 1 : 1; }

__host__ __device__ inline int64_t item_count(bool packed, int64_t rows, int64_t uniform, int64_t count, int64_t length) {
  if (packed) return rows / length + count + 1;
  return pieces_of(uniform, length) * count;
}

// All 32 lanes of a warp call this together.
__device__ __forceinline__ Piece find_piece(const Chains& c, int64_t item, int length) {
  Piece p;
  p.padding = false;
  if (c.points == nullptr) {
    const int64_t per = pieces_of(c.uniform, length);
    p.chain = item / per;
    p.index = item - p.chain * per;
  } else {
    // the last chain whose key is <= item, 32 probes at a time
    int64_t lo = 0, hi = c.count;
    const int lane = threadIdx.x & 31;
    while (hi > lo) {
      const int64_t step = (hi - lo + 31) >> 5;
      const int64_t probe = lo + (lane + 1) * step;
      const bool below = probe <= hi && c.first(probe) / length + probe <= item;
      const int n = __popc(__ballot_sync(kAll, below));
      lo += n * step;
      const int64_t top = lo + step - 1;
      hi = top < hi ? top : hi;
    }
    p.chain = lo;
    p.index = item - (c.first(lo) / length + lo);
    p.padding = lo == c.count;
  }
  p.chain_first = c.first(p.chain);
  p.chain_end = c.end(p.chain);
  p.first = p.chain_first + p.index * length;
  p.valid = p.index >= 0 && (p.first < p.chain_end || p.index == 0);
  const int64_t e = p.first + length;
  p.end = e < p.chain_end ? e : p.chain_end;
  if (p.first > p.end) p.first = p.end;
  return p;
}

// ------------------------------------------------------------------------------------------
// sums of partial results: out[m] = sum_p part[p][m], in the order of p
// ------------------------------------------------------------------------------------------
// A block takes 32 columns; its 8 warps take every eighth partial and are summed in order at the end, so the
// result does not depend on timing.  The columns from `split` on go to `out1`.
__device__ __forceinline__ void sum_partials(const float* __restrict__ part, int64_t count, int64_t columns, int64_t block, int64_t split, float* __restrict__ out0,
                                             float* __restrict__ out1) {
  __shared__ float s[8][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t m = block * 32 + lane;
  float sum = 0.0f;
  if (m < columns) {
#pragma unroll 8
    for (int64_t p = w; p < count; p += 8) sum += part[p * columns + m];
  }
  s[w][lane] = sum;
  __syncthreads();
  if (w == 0 && m < columns) {
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) total += s[i][lane];
    float* out = m < split ? out0 : out1;
    if (out != nullptr) out[m < split ? m : m - split] = total;
  }
}

static __global__ __launch_bounds__(256) void sum_partials_kernel(const float* __restrict__ part, int64_t count, int64_t columns, int64_t split,
                                                                float* __restrict__ out0, float* __restrict__ out1) {
  sum_partials(part, count, columns, blockIdx.x, split, out0, out1);
}

}  // namespace cufkb_seq
