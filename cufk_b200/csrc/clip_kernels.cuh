// Gradient clipping by the global norm over many arrays.
//
//   norm = sqrt(sum g^2)      out = g min(1, max_norm / (norm + eps))
//
// Two launches and no host: the first leaves one double per block, the second adds them (every block for itself, in the same order) and
// scales.  Reading twice and writing once bounds it; the second launch takes the chunks from the last to the first, so that what
// the first one read last is still in the L2 cache.  The squares of a 16-byte block are added in float and the
// blocks in double; a block whose float sum left the range (overflow, or too small for its squares) is taken again in double.
// 160 million float32 elements in 242 arrays: 93 us and 198 us, 6.9 and 6.5 TB/s.  Small lists are bound by the two launches; one cluster
// of eight blocks with a single launch was slower from 100,000 elements on (14 us against 11).
#pragma once

#include "seq_common.cuh"

namespace cufkb_seq {

constexpr int kClipThreads = 256;
constexpr int kClipChunk = 8192;  // elements of one array that a block takes at a time

enum ClipType : uint8_t { kClipFloat, kClipDouble, kClipHalf, kClipBfloat16 };

// The arrays of one launch, passed by value.  first[i] is array i's first chunk; first[arrays] the number of chunks.
template <int MOST>
struct ClipTable {
  const void* grad[MOST];
  void* out[MOST];
  int64_t count[MOST];
  int first[MOST + 1];
  uint8_t type[MOST];
  int arrays;
};

template <typename T>
__device__ __forceinline__ double to_double(T v) {
  if constexpr (std::is_same_v<T, double>) {
    return v;
  } else {
    return static_cast<double>(to_float(v));
  }
}

// Calls f.template operator()<T>(grad, out, elements) for the chunk.
template <int MOST, typename F>
__device__ __forceinline__ void with_chunk(const ClipTable<MOST>& t, int chunk, F&& f) {
  int lo = 0, hi = t.arrays - 1;
  while (hi > lo) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= chunk) {
      lo = mid;
    } else {
      hi = mid - 1;
    }
  }
  const int64_t at = static_cast<int64_t>(chunk - t.first[lo]) * kClipChunk;
  const int64_t left = t.count[lo] - at;
  const int n = static_cast<int>(left < kClipChunk ? left : kClipChunk);
  switch (t.type[lo]) {
    case kClipFloat:
      f(static_cast<const float*>(t.grad[lo]) + at, static_cast<float*>(t.out[lo]) + at, n);
      break;
    case kClipDouble:
      f(static_cast<const double*>(t.grad[lo]) + at, static_cast<double*>(t.out[lo]) + at, n);
      break;
    case kClipHalf:
      f(static_cast<const __half*>(t.grad[lo]) + at, static_cast<__half*>(t.out[lo]) + at, n);
      break;
    default:
      f(static_cast<const __nv_bfloat16*>(t.grad[lo]) + at, static_cast<__nv_bfloat16*>(t.out[lo]) + at, n);
  }
}

template <typename T>
__device__ __forceinline__ int head_of(const T* p, int n) {
  constexpr int N = 16 / sizeof(T);
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
  const int head = off ? N - off : 0;
  return head < n ? head : n;
}

template <typename T>
__device__ __forceinline__ double square_sum(const T* g, int n) {
  constexpr int N = 16 / sizeof(T);
  const int head = head_of(g, n), blocks = (n - head) / N, tail = head + blocks * N;
  double sum = 0.0;
  if (static_cast<int>(threadIdx.x) < head) {
    const double v = to_double(g[threadIdx.x]);
    sum = fma(v, v, sum);
  }
  const Block<T, N>* body = reinterpret_cast<const Block<T, N>*>(g + head);
#pragma unroll 4
  for (int i = threadIdx.x; i < blocks; i += kClipThreads) {
    const Block<T, N> b = body[i];
    if constexpr (std::is_same_v<T, double>) {
#pragma unroll
      for (int j = 0; j < N; ++j) sum = fma(b.v[j], b.v[j], sum);
    } else {
      float q = 0.0f;
#pragma unroll
      for (int j = 0; j < N; ++j) q = fmaf(to_float(b.v[j]), to_float(b.v[j]), q);
      if (q > 1.0e-26f && q < 1.0e37f) {
        sum += static_cast<double>(q);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) sum = fma(to_double(b.v[j]), to_double(b.v[j]), sum);
      }
    }
  }
  if (tail + static_cast<int>(threadIdx.x) < n) {
    const double v = to_double(g[tail + threadIdx.x]);
    sum = fma(v, v, sum);
  }
  return sum;
}

// The sum over a block, in every thread.
__device__ __forceinline__ double block_sum(double v, double* s) {
#pragma unroll
  for (int half = 16; half > 0; half /= 2) v += __shfl_xor_sync(kAll, v, half);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  double total = 0.0;
#pragma unroll
  for (int i = 0; i < kClipThreads / 32; ++i) total += s[i];
  return total;
}

template <int MOST>
__global__ __launch_bounds__(kClipThreads) void clip_norm_kernel(const __grid_constant__ ClipTable<MOST> t, double* __restrict__ partial) {
  __shared__ double s[kClipThreads / 32];
  const int chunks = t.first[t.arrays];
  double sum = 0.0;
  for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    with_chunk(t, chunk, [&](const auto* g, auto*, int n) { sum += square_sum(g, n); });
  }
  sum = block_sum(sum, s);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// f = high * low.  Below float's normal range (a norm beyond 1e38 max_norm) a float factor would keep few bits or none, though what it
// scales may well end in range; there, high = 2^-100 takes the values down first.  Elsewhere high = 1, which changes no bit.
struct ClipFactor {
  double f;
  float high, low;
  __device__ __forceinline__ explicit ClipFactor(double factor) : f(factor), high(factor < 0x1p-100 ? 0x1p-100f : 1.0f) {
    low = static_cast<float>(factor < 0x1p-100 ? factor * 0x1p100 : factor);
  }
};

template <typename T>
__device__ __forceinline__ void scale_chunk(const T* g, T* out, int n, const ClipFactor& c) {
  constexpr int N = 16 / sizeof(T);
  auto scaled = [&](T v) {
    if constexpr (std::is_same_v<T, double>) {
      return v * c.f;
    } else {
      return from_float<T>(to_float(v) * c.high * c.low);
    }
  };
  if (((reinterpret_cast<uintptr_t>(g) ^ reinterpret_cast<uintptr_t>(out)) & 15) != 0) {
    for (int i = threadIdx.x; i < n; i += kClipThreads) out[i] = scaled(g[i]);
    return;
  }
  const int head = head_of(g, n), blocks = (n - head) / N, tail = head + blocks * N;
  if (static_cast<int>(threadIdx.x) < head) out[threadIdx.x] = scaled(g[threadIdx.x]);
  const Block<T, N>* body = reinterpret_cast<const Block<T, N>*>(g + head);
  Block<T, N>* to = reinterpret_cast<Block<T, N>*>(out + head);
#pragma unroll 4
  for (int i = threadIdx.x; i < blocks; i += kClipThreads) {
    Block<T, N> b = body[i];
#pragma unroll
    for (int j = 0; j < N; ++j) b.v[j] = scaled(b.v[j]);
    to[i] = b;
  }
  if (tail + static_cast<int>(threadIdx.x) < n) out[tail + threadIdx.x] = scaled(g[tail + threadIdx.x]);
}

// partials: of all launches of the first kernel.  norm is written by the first block of the launch that is given it.
template <int MOST>
__global__ __launch_bounds__(kClipThreads) void clip_scale_kernel(const __grid_constant__ ClipTable<MOST> t, const double* __restrict__ partial, int partials,
                                                                double max_norm, double eps, void* norm, int norm_double) {
  __shared__ double s[kClipThreads / 32];
  double sum = 0.0;
  for (int i = threadIdx.x; i < partials; i += kClipThreads) sum += partial[i];
  const double total = sqrt(block_sum(sum, s));
  if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) {
    if (norm_double) {
      *static_cast<double*>(norm) = total;
    } else {
      *static_cast<float*>(norm) = static_cast<float>(total);
    }
  }
  // max_norm = inf only measures: 1 for any norm.  Compared before dividing: of inf / inf and 0 / 0 nothing is to be clipped either.
  const double most = total + eps;
  const double f = max_norm == INFINITY ? 1.0 : most > max_norm ? max_norm / most : most == most ? 1.0 : most;
  const ClipFactor c(f);
  const int chunks = t.first[t.arrays];
  for (int chunk = chunks - 1 - static_cast<int>(blockIdx.x); chunk >= 0; chunk -= static_cast<int>(gridDim.x)) {
    with_chunk(t, chunk, [&](const auto* g, auto* out, int n) {
      if (f == 1.0 && static_cast<const void*>(g) == static_cast<const void*>(out)) return;  // in place and nothing to change
      scale_chunk(g, out, n, c);
    });
  }
}

}  // namespace cufkb_seq
