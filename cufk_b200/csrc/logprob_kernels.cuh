// Log probabilities of given tokens with entropy and the largest alternatives, and their gradient.
//
// One pass over a row of logits keeps, per thread, the running maximum m, s = sum exp(l - m) and w = sum exp(l - m)(l - m); then
//   logp = (l[token] - m) - log s      entropy = log s - w / s
// m and log s are kept apart: their sum would lose log s next to a maximum of large size (a row of nothing but masks of the type's
// lowest value is uniform).
//
// The k largest: a value that the maxima of k threads reach is a lower bound of the k-th largest logit, so only the parts of threads whose
// maximum reaches it are looked at again, by all threads together; what reaches the bound goes to a list in shared memory, where
// each entry's place is the number of entries before it (larger, or equal with a lower id).  If the list overflows (many equal
// logits), k rounds over the row take one entry each.
//
// The forward reads the row once and the backward reads it and writes the gradient once: memory bounds both, as long as little is done per
// logit: packed maxima of 16-bit logits, packed (f32x2) sums, and no care for -inf until a sum shows that there is one.  At 4096 x 32768
// (bfloat16, the 8 largest) the forward takes 78 us (3.4 TB/s; its exponentials alone 30), the backward 80 us (6.7 TB/s).
#pragma once

#include "seq_common.cuh"

namespace cufkb_seq {

constexpr float kFloor = -1.0e4f;  // exp of it is 0; keeps 0 * (-inf) out of the sums

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Order of the logits as unsigned numbers: NaN above +inf, -0 equal to 0; 0 is below all of them.
__device__ __forceinline__ uint32_t order_of(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t b = v == 0.0f ? 0u : __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) {
  if (order == 0xffffffffu) return __uint_as_float(0x7fffffffu);
  return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}

// The threads that share a row: one warp, or the whole block.
template <int THREADS>
struct Team {
  static constexpr bool kWarp = THREADS == 32;
  static __device__ __forceinline__ int rank() { return kWarp ? threadIdx.x & 31 : threadIdx.x; }
  static __device__ __forceinline__ void sync() {
    if constexpr (kWarp) {
      __syncwarp();
    } else {
      __syncthreads();
    }
  }
};

// The largest of a block's logits, NaN if there is one.
template <typename T, int N>
__device__ __forceinline__ float max_of(const Block<T, N>& b) {
  if constexpr (sizeof(T) == 2) {
    using Two = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    const Two* v = reinterpret_cast<const Two*>(&b);
    Two m = v[0];
#pragma unroll
    for (int j = 1; j < N / 2; ++j) m = __hmax2_nan(m, v[j]);
    return max_nan(to_float(m.x), to_float(m.y));
  } else {
    float m = b.v[0];
#pragma unroll
    for (int j = 1; j < N; ++j) m = max_nan(m, b.v[j]);
    return m;
  }
}

struct Running {
  float m, s, w;
  __device__ __forceinline__ void to_max(float top) {
    // a maximum that rises by d scales both sums by exp(-d) and takes d off every (l - m)
    const float d = fmaxf(m - top, kFloor);  // m = -inf: both sums are 0
    const float f = exp2_fast(d * kLog2e);
    w = f * fmaf(d, s, w);
    s *= f;
    m = top;
  }
  __device__ __forceinline__ void add(float l) {
    if (!(l <= m)) to_max(max_nan(l, m));
    const float d = fmaxf(l - m, kFloor), e = exp2_fast(d * kLog2e);
    s += e;
    w = fmaf(e, d, w);
  }
  template <typename T, int N>
  __device__ __forceinline__ void add(const Block<T, N>& b) {
    const float top = max_of(b);
    if (!(top <= m)) to_max(max_nan(top, m));
    if (!block<false>(b)) block<true>(b);  // some l - m is -inf (or NaN): once more, with care
  }
  template <bool CARE, typename T, int N>
  __device__ __forceinline__ bool block(const Block<T, N>& b) {
    const Pair less = pair(-m, -m), scale = pair(kLog2e, kLog2e);
    Pair s2 = pair(s, 0.0f), w2 = pair(w, 0.0f);
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      Pair d = add2(pair(to_float(b.v[j]), to_float(b.v[j + 1])), less);
      if (CARE) {
        const float2 f = halves(d);
        d = pair(fmaxf(f.x, kFloor), fmaxf(f.y, kFloor));
      }
      const Pair e = exp2_pair(mul2(d, scale));
      s2 = add2(s2, e);
      w2 = fma2(e, d, w2);
    }
    const float sum = sum_pair(w2);
    if (!CARE && !(sum == sum)) return false;
    s = sum_pair(s2);
    w = sum;
    return true;
  }
  // the sums over the lanes of a warp, in every lane
  __device__ __forceinline__ void over_warp() {
    float top = m;
#pragma unroll
    for (int half = 16; half > 0; half /= 2) top = max_nan(top, __shfl_xor_sync(kAll, top, half));
    to_max(top);
#pragma unroll
    for (int half = 16; half > 0; half /= 2) {
      s += __shfl_xor_sync(kAll, s, half);
      w += __shfl_xor_sync(kAll, w, half);
    }
  }
};

// How a row's elements fall to the threads that share it: single ones up to the first 16-byte boundary, 16-byte blocks, single ones at
// the end.
template <typename T, int THREADS>
struct RowParts {
  static constexpr int N = 16 / sizeof(T);
  const T* row;
  const Block<T, N>* body;
  int rank, head, blocks, n;
  __device__ __forceinline__ RowParts(const T* r, int count) : row(r), rank(Team<THREADS>::rank()), n(count) {
    const int off = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    head = off ? N - off : 0;
    if (head > n) head = n;
    blocks = (n - head) / N;
    body = reinterpret_cast<const Block<T, N>*>(row + head);
  }
  static constexpr int kDeep = THREADS == 32 ? 2 : 4;  // blocks on their way together
  __device__ __forceinline__ bool any() const { return rank < head || rank < blocks || head + blocks * N + rank < n; }
  __device__ __forceinline__ int rounds() const { return (blocks + THREADS - 1) / THREADS; }  // blocks of a thread
  // one(value, id) for a thread's single elements
  template <typename One>
  __device__ __forceinline__ void singles(int of, One&& one) const {
    if (of < head) one(to_float(row[of]), of);
    const int tail = head + blocks * N + of;
    if (tail < n) one(to_float(row[tail]), tail);
  }
  // many(block, first id) for this thread's blocks
  template <typename Many>
  __device__ __forceinline__ void each_block(Many&& many) const {
    int i = rank;
    for (; i + (kDeep - 1) * THREADS < blocks; i += kDeep * THREADS) {
      Block<T, N> b[kDeep];
#pragma unroll
      for (int d = 0; d < kDeep; ++d) b[d] = body[i + d * THREADS];
#pragma unroll
      for (int d = 0; d < kDeep; ++d) many(b[d], head + (i + d * THREADS) * N);
    }
    for (; i < blocks; i += THREADS) many(body[i], head + i * N);
  }
};

__device__ __forceinline__ uint64_t key_of(uint32_t order, int id) { return (static_cast<uint64_t>(order) << 32) | (0xffffffffu - static_cast<uint32_t>(id)); }

// The largest value that at least `top` of a warp's lanes reach.
__device__ __forceinline__ uint32_t warp_bound(uint32_t own, int top) {
  for (;;) {
    const uint32_t most = __reduce_max_sync(kAll, own);
    const int count = __popc(__ballot_sync(kAll, own == most));
    if (count >= top || most == 0u) return most;
    top -= count;
    if (own == most) own = 0u;
  }
}

// A value that at least `top` threads of a block reach: the `top`-th largest of the warps' maxima, or, where there are fewer warps, the lowest
// of the values that `top` / warps lanes of each warp reach.  It need not be the largest such value: a few more parts are looked
// at, for fewer rounds.
template <int WARPS>
__device__ __forceinline__ uint32_t block_bound(uint32_t own, int top, uint32_t* of_warp) {
  const int lane = threadIdx.x & 31, each = (top + WARPS - 1) / WARPS;
  const uint32_t mine = warp_bound(own, each);
  if (lane == 0) of_warp[threadIdx.x >> 5] = mine;
  __syncthreads();
  const uint32_t v = of_warp[lane < WARPS ? lane : 0];
  return each > 1 ? __reduce_min_sync(kAll, v) : warp_bound(lane < WARPS ? v : 0u, top);
}

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS == 32 ? 128 : THREADS, THREADS == 128 ? 12 : 1) void logprobs_kernel(const T* __restrict__ logits, int64_t stride, const int64_t* __restrict__ tokens,
                                                                               float* __restrict__ logp, float* __restrict__ entropy, float* __restrict__ log_sum,
                                                                               float* __restrict__ top_logp, int64_t* __restrict__ top_tokens, int64_t rows,
                                                                               int n, int top) {
  using G = Team<THREADS>;
  constexpr int kTeams = G::kWarp ? 4 : 1;
  constexpr int kList = G::kWarp ? 256 : 1024;
  constexpr int kWarps = THREADS / 32;
  __shared__ uint64_t s_list[kTeams][kList];
  __shared__ int s_count[kTeams];
  __shared__ Running s_run[kWarps];
  __shared__ uint64_t s_best[kWarps];
  __shared__ uint32_t s_bound[kWarps];
  __shared__ uint16_t s_reach[kTeams][THREADS];  // threads whose maximum reaches the bound
  __shared__ int s_reached[kTeams];
  const int team = G::kWarp ? threadIdx.x >> 5 : 0, rank = G::rank(), lane = threadIdx.x & 31;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * kTeams + team;
  if (r >= rows) return;
  const T* row = logits + r * stride;

  const RowParts<T, THREADS> parts(row, n);
  constexpr int N = RowParts<T, THREADS>::N;
  Running run{-INFINITY, 0.0f, 0.0f};
  parts.singles(rank, [&](float v, int) { run.add(v); });
  parts.each_block([&](const Block<T, N>& b, int) { run.add(b); });
  const uint32_t own = parts.any() ? order_of(run.m) : 0u;
  run.over_warp();
  if constexpr (!G::kWarp) {
    if (lane == 0) s_run[threadIdx.x >> 5] = run;
    __syncthreads();
    run = lane < kWarps ? s_run[lane] : Running{-INFINITY, 0.0f, 0.0f};
    run.over_warp();
  }
  const bool none = run.m == -INFINITY;  // no token is possible
  const float log_s = none ? 0.0f : logf(run.s);
  if (rank == 0) {
    const int64_t token = tokens[r];
    float lp = 0.0f;
    if (token >= n) {
      lp = __uint_as_float(0x7fffffffu);
    } else if (token >= 0) {
      lp = none ? -INFINITY : (to_float(row[token]) - run.m) - log_s;
    }
    logp[r] = lp;
    entropy[r] = none ? 0.0f : log_s - __fdividef(run.w, run.s);
    log_sum[2 * r] = run.m;
    log_sum[2 * r + 1] = log_s;
  }
  if (top == 0) return;

  if (rank == 0) s_count[team] = s_reached[team] = 0;
  uint32_t bound;
  if constexpr (G::kWarp) {
    bound = warp_bound(own, top);
    __syncwarp();
  } else {
    bound = block_bound<kWarps>(own, top, s_bound);
  }
  if (own >= bound) s_reach[team][atomicAdd(&s_reached[team], 1)] = static_cast<uint16_t>(rank);
  G::sync();
  {
    auto look = [&](float v, int id) {
      const uint32_t o = order_of(v);
      if (o >= bound) {
        const int at = atomicAdd(&s_count[team], 1);
        if (at < kList) s_list[team][at] = key_of(o, id);
      }
    };
    // a thread's blocks and, as one more, its single elements
    const int per = parts.rounds() + 1, tasks = s_reached[team] * per;
    for (int t = rank; t < tasks; t += THREADS) {
      const int which = t / per, k = t - which * per, of = s_reach[team][which];
      if (k == per - 1) {
        parts.singles(of, look);
      } else if (of + k * THREADS < parts.blocks) {
        const Block<T, N> b = parts.body[of + k * THREADS];
        if (!(order_of(max_of(b)) < bound)) {
#pragma unroll
          for (int j = 0; j < N; ++j) look(to_float(b.v[j]), parts.head + (of + k * THREADS) * N + j);
        }
      }
    }
  }
  G::sync();
  const int found = s_count[team];
  auto put = [&](int place, uint64_t key) {
    const float v = value_of(static_cast<uint32_t>(key >> 32));
    top_logp[r * top + place] = none ? -INFINITY : (v - run.m) - log_s;
    top_tokens[r * top + place] = static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(key));
  };
  if (found <= kList) {
    for (int i = rank; i < found; i += THREADS) {
      const uint64_t key = s_list[team][i];
      int place = 0;
      for (int j = 0; j < found; ++j) place += s_list[team][j] > key;
      if (place < top) put(place, key);
    }
    return;
  }
  uint64_t before = ~0ull;
  for (int k = 0; k < top; ++k) {
    uint64_t best = 0;
    auto look = [&](float v, int id) {
      const uint64_t key = key_of(order_of(v), id);
      if (key < before && key > best) best = key;
    };
    parts.singles(rank, look);
    parts.each_block([&](const Block<T, N>& b, int id) {
#pragma unroll
      for (int j = 0; j < N; ++j) look(to_float(b.v[j]), id + j);
    });
#pragma unroll
    for (int half = 16; half > 0; half /= 2) {
      const uint64_t o = __shfl_xor_sync(kAll, best, half);
      best = o > best ? o : best;
    }
    if constexpr (!G::kWarp) {
      __syncthreads();
      if (lane == 0) s_best[threadIdx.x >> 5] = best;
      __syncthreads();
      best = s_best[0];
      for (int i = 1; i < kWarps; ++i) best = s_best[i] > best ? s_best[i] : best;
    }
    if (rank == 0) put(k, best);
    before = best;
  }
}

// d logits = g (1[token] - p) - h p (log p + entropy)
struct RowGrad {
  float g, h, c, m, log_s;  // c = g + h entropy
  int token;
  __device__ __forceinline__ RowGrad(int64_t r, int n, const int64_t* tokens, const float* entropy, const float* log_sum, const float* grad_logp,
                                     const float* grad_entropy) {
    const int64_t t = tokens[r];
    g = (grad_logp != nullptr && t >= 0) ? grad_logp[r] : 0.0f;
    if (t >= n) g = __uint_as_float(0x7fffffffu);
    token = t < 0 || t >= n ? -1 : static_cast<int>(t);
    h = grad_entropy != nullptr ? grad_entropy[r] : 0.0f;
    m = log_sum[2 * r];
    log_s = log_sum[2 * r + 1];
    c = fmaf(h, entropy[r], g);
    if (m == -INFINITY) {
      // no token is possible: p = 0 everywhere, and no gradient, whatever comes back (NaN from p log p, say)
      m = INFINITY;
      g = h = c = 0.0f;
    }
  }
  // a block from id `first` on
  template <typename T, int N>
  __device__ __forceinline__ void apply(Block<T, N>& b, int first) const {
    if constexpr (N > 1) {
      const Pair less = pair(-m, -m), rest = pair(-log_s, -log_s), scale = pair(kLog2e, kLog2e), h2 = pair(-h, -h), c2 = pair(-c, -c);
      Block<T, N> out;
#pragma unroll
      for (int j = 0; j < N; j += 2) {
        const float2 f = halves(add2(pair(to_float(b.v[j]), to_float(b.v[j + 1])), less));
        const Pair lp = add2(pair(max_nan(f.x, kFloor), max_nan(f.y, kFloor)), rest);
        const float2 d = halves(mul2(exp2_pair(mul2(lp, scale)), fma2(h2, lp, c2)));
        out.v[j] = from_float<T>(d.x);
        out.v[j + 1] = from_float<T>(d.y);
      }
      if (static_cast<unsigned>(token - first) < static_cast<unsigned>(N)) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          if (first + j == token) out.v[j] = from_float<T>(one(to_float(b.v[j])) + g);
        }
      }
      b = out;
    } else {
      const float d = one(to_float(b.v[0]));
      b.v[0] = from_float<T>(first == token ? d + g : d);
    }
  }
  __device__ __forceinline__ float one(float logit) const {
    const float lp = max_nan(logit - m, kFloor) - log_s;
    return exp2_fast(lp * kLog2e) * fmaf(-h, lp, -c);
  }
};

constexpr int kGradBlocks = 4;  // 16-byte blocks of a thread in a long row

// Long rows of 16-byte blocks: a block of threads stays within one row.
template <typename T>
__global__ __launch_bounds__(256) void logprobs_backward_rows_kernel(const T* __restrict__ logits, int64_t stride, const int64_t* __restrict__ tokens,
                                                                   const float* __restrict__ entropy, const float* __restrict__ log_sum,
                                                                   const float* __restrict__ grad_logp, const float* __restrict__ grad_entropy,
                                                                   T* __restrict__ grad, int n, int parts) {
  constexpr int N = 16 / sizeof(T);
  const int64_t r = blockIdx.x / parts;
  const int blocks = n / N, first = static_cast<int>(blockIdx.x - r * parts) * (256 * kGradBlocks) + threadIdx.x;
  const RowGrad row(r, n, tokens, entropy, log_sum, grad_logp, grad_entropy);
  const Block<T, N>* from = reinterpret_cast<const Block<T, N>*>(logits + r * stride);
  Block<T, N>* to = reinterpret_cast<Block<T, N>*>(grad + r * n);
  Block<T, N> b[kGradBlocks];
#pragma unroll
  for (int k = 0; k < kGradBlocks; ++k) {
    if (first + k * 256 < blocks) b[k] = from[first + k * 256];
  }
#pragma unroll
  for (int k = 0; k < kGradBlocks; ++k) {
    const int at = first + k * 256;
    if (at >= blocks) break;
    row.apply(b[k], at * N);
    to[at] = b[k];
  }
}

// Any rows: a block of N elements per thread.
template <typename T, int N>
__global__ __launch_bounds__(256) void logprobs_backward_kernel(const T* __restrict__ logits, int64_t stride, const int64_t* __restrict__ tokens,
                                                              const float* __restrict__ entropy, const float* __restrict__ log_sum,
                                                              const float* __restrict__ grad_logp, const float* __restrict__ grad_entropy,
                                                              T* __restrict__ grad, int64_t rows, int n, int blocks) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t r = id / blocks;
  if (r >= rows) return;
  const int at = static_cast<int>(id - r * blocks) * N;
  const RowGrad row(r, n, tokens, entropy, log_sum, grad_logp, grad_entropy);
  Block<T, N> b = *reinterpret_cast<const Block<T, N>*>(logits + r * stride + at);
  row.apply(b, at);
  *reinterpret_cast<Block<T, N>*>(grad + r * n + at) = b;
}

}  // namespace cufkb_seq
