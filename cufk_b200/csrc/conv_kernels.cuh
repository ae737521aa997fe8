// Short causal convolution along packed chains, with its gradients and its single-row step.
//
//   pre[t] = bias + sum_k w[k] x[t - (W-1) + k],  y = pre sigmoid(pre)
//
// Every output needs W rows of its own channel, so a thread owns kWide consecutive channels and walks the rows of a tile, kAhead at a
// time, with the W - 1 rows around them in registers: x is read once, but for W - 1 rows at each tile's start.  The next batches
// are on their way to shared memory while these rows are worked on, and arithmetic is on pairs of channels (f32x2): reading and
// writing should bound it, and the instructions per element (about 16 forward, 27 backward) still share in that.  Tiles are as
// long as one wave of blocks allows.
#pragma once

#include "seq_common.cuh"

namespace cufkb_seq {

constexpr int kWide = 4;   // channels a thread owns
constexpr int kAhead = 4;  // rows of a batch

template <typename T>
struct ConvArgs {
  Chains chains;
  int64_t width, columns;  // columns: ceil(width / kWide)
  int64_t tiles;
  int tile_rows;
  const T* x;
  int64_t x_stride;
  const float *weight, *bias;
  const T* initial;
  T* y;
  T* final_state;
  const T* grad_y;
  int64_t grad_y_stride;
  const T* grad_final;
  T* grad_x;
  T* grad_initial;
  float* partial;  // (tiles, width * (W + 1)): weight sums, then bias sums; nullptr when not wanted
};

// A row of a thread's channels.
struct Row {
  Pair v[kWide / 2];
};

template <typename T>
__device__ __forceinline__ Row widen(const Block<T, kWide>& b) {
  Row r;
#pragma unroll
  for (int i = 0; i < kWide / 2; ++i) r.v[i] = pair(to_float(b.v[2 * i]), to_float(b.v[2 * i + 1]));
  return r;
}
template <typename T>
__device__ __forceinline__ Block<T, kWide> narrow(const Row& r) {
  Block<T, kWide> b;
#pragma unroll
  for (int i = 0; i < kWide / 2; ++i) {
    const float2 f = halves(r.v[i]);
    b.v[2 * i] = from_float<T>(f.x);
    b.v[2 * i + 1] = from_float<T>(f.y);
  }
  return b;
}

template <int W>
struct Taps {
  Row w[W], b;
  __device__ __forceinline__ void load(const float* weight, const float* bias, int64_t c, int valid) {
#pragma unroll
    for (int k = 0; k <= W; ++k) {
      float f[kWide];
#pragma unroll
      for (int i = 0; i < kWide; ++i) {
        f[i] = 0.0f;
        if (i < valid && k < W) f[i] = weight[(c + i) * W + k];
        if (i < valid && k == W && bias != nullptr) f[i] = bias[c + i];
      }
#pragma unroll
      for (int i = 0; i < kWide / 2; ++i) (k < W ? w[k < W ? k : 0] : b).v[i] = pair(f[2 * i], f[2 * i + 1]);
    }
  }
  // bias + sum_k w[k] rows[k]
  __device__ __forceinline__ Row apply(const Row* rows) const {
    Row r;
#pragma unroll
    for (int i = 0; i < kWide / 2; ++i) {
      r.v[i] = b.v[i];
#pragma unroll
      for (int k = 0; k < W; ++k) r.v[i] = fma2(w[k].v[i], rows[k].v[i], r.v[i]);
    }
    return r;
  }
};

// A thread's rows on their way to shared memory, batch by batch.  Each thread copies and reads its own columns only, so no block-wide
// sync is needed: its own wait for its own copies is enough.  One batch's place is idle at any time, the one read last.
template <typename T, int STAGES>
struct Stream {
  static constexpr int kBytes = kWide * sizeof(T);
  Block<T, kWide> (*place)[128];  // [STAGES * kAhead][128]
  template <bool VEC>
  __device__ __forceinline__ void copy(int slot, const T* from, int valid) const {
    Block<T, kWide>* to = &place[slot][threadIdx.x];
    if constexpr (VEC) {
      // zero-fills what is not there
      asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from), "n"(kBytes),
                   "r"(valid >= kWide ? kBytes : 0)
                   : "memory");
    } else {
      *to = load_block<T, kWide, false>(from, valid);
    }
  }
  __device__ __forceinline__ void put(int slot, const Block<T, kWide>& b) const { place[slot][threadIdx.x] = b; }
  __device__ __forceinline__ Block<T, kWide> get(int slot) const { return place[slot][threadIdx.x]; }
};
__device__ __forceinline__ void close_batch() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void wait_batches() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}
template <typename T>
__host__ __device__ constexpr int conv_stages() {
  return sizeof(T) == 2 ? 4 : 3;
}

// The row `place` of a chain counted from its start; negative ones are the initial state's.
template <typename T, int W, bool VEC>
__device__ __forceinline__ Block<T, kWide> row_at(const ConvArgs<T>& p, int64_t s, int64_t chain_first, int64_t place, int64_t c, int valid) {
  if (place >= 0) return load_block<T, kWide, VEC>(p.x + (chain_first + place) * p.x_stride + c, valid);
  if (p.initial != nullptr && s < p.chains.count) return load_block<T, kWide, VEC>(p.initial + (s * (W - 1) + (W - 1 + place)) * p.width + c, valid);
  return load_block<T, kWide, VEC>(p.x, 0);
}

// Resident blocks per SM.  Measured on B200 at 32768 x 2048 (bfloat16, four taps): forward 62 us (4.3 TB/s) and backward 122 us with 5 and 3;
// 62 and 144 us with 6 and 4, whose registers spill; 72 and 171 us with two channels per thread; 81 and 173 us with
// the next rows in registers instead of shared memory.
constexpr int kConvForwardBlocks = 5, kConvBackwardBlocks = 3;

template <typename T, int W, bool SILU, bool VEC>
__global__ __launch_bounds__(128, kConvForwardBlocks) void conv_forward_kernel(ConvArgs<T> p) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t tile = id / p.columns, c = (id - tile * p.columns) * kWide;
  const int valid = static_cast<int>(p.width - c < kWide ? p.width - c : kWide);
  if (tile >= p.tiles) {
    // the states left behind, one row of one chain per thread
    const int64_t job = tile - p.tiles, s = job / (W - 1), k = job - s * (W - 1);
    if (p.final_state == nullptr || s >= p.chains.count) return;
    const int64_t a = p.chains.first(s), n = p.chains.end(s) - a;
    store_block<T, kWide, VEC>(p.final_state + job * p.width + c, row_at<T, W, VEC>(p, s, a, n - (W - 1) + k, c, valid), valid);
    return;
  }
  Taps<W> taps;
  taps.load(p.weight, p.bias, c, valid);
  const int64_t r0 = tile * p.tile_rows;
  const int n = static_cast<int>(r0 + p.tile_rows < p.chains.rows ? p.tile_rows : p.chains.rows - r0);
  const T* px = p.x + r0 * p.x_stride + c;
  T* py = p.y + r0 * p.width + c;
  constexpr int kStages = conv_stages<T>();
  __shared__ Block<T, kWide> s_x[kStages * kAhead][128];
  const Stream<T, kStages> xs{s_x};
  auto load = [&](int r, int stage) {
    if (r < n) {
      const T* from = px + r * p.x_stride;
#pragma unroll
      for (int i = 0; i < kAhead; ++i, from += p.x_stride) xs.template copy<VEC>(stage * kAhead + i, r + i < n ? from : px, r + i < n ? valid : 0);
    }
    close_batch();
  };
#pragma unroll
  for (int d = 0; d < kStages - 1; ++d) load(d * kAhead, d);
  int stage = 0;
  Row rows[W - 1 + kAhead];  // the W - 1 rows before, then these
  int end = 0;               // of the chain, from the tile's start
  bool padding = false;
  auto output = [&](int i) {
    Row out = taps.apply(rows + i);
    if (SILU) {
#pragma unroll
      for (int v = 0; v < kWide / 2; ++v) out.v[v] = mul2(out.v[v], sigmoid2(out.v[v]));
    }
    return out;
  };
  for (int r = 0; r < n; r += kAhead, py += kAhead * p.width) {
    Row now[kAhead];
    wait_batches<kStages - 2>();
#pragma unroll
    for (int i = 0; i < kAhead; ++i) now[i] = widen(xs.get(stage * kAhead + i));
    load(r + (kStages - 1) * kAhead, stage == 0 ? kStages - 1 : stage - 1);  // the place read in the round before
    stage = stage == kStages - 1 ? 0 : stage + 1;
    if (r + kAhead <= end && !padding) {
      // the rows of one chain
      T* to = py;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) rows[W - 1 + i] = now[i];
#pragma unroll
      for (int i = 0; i < kAhead; ++i, to += p.width) store_block<T, kWide, VEC>(to, narrow<T>(output(i)), valid);
    } else {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (r + i >= end && r + i < n) {
          // a chain's first row here: the rows before it
          const int64_t row = r0 + r + i, s = p.chains.of_row(row), a = p.chains.first(s), e = p.chains.end(s) - r0;
          end = e > r + i && e < n ? static_cast<int>(e) : n;
          padding = s == p.chains.count;
#pragma unroll
          for (int k = 0; k < W - 1; ++k) rows[i + k] = widen(row_at<T, W, VEC>(p, s, a, row - a - (W - 1) + k, c, valid));
        }
        rows[W - 1 + i] = now[i];
        const Row out = output(i);
        if (r + i < n) store_block<T, kWide, VEC>(py + i * p.width, narrow<T>(padding ? Row{} : out), valid);
      }
    }
#pragma unroll
    for (int k = 0; k < W - 1; ++k) rows[k] = rows[k + kAhead];
  }
}

// dy silu'(pre)
template <bool SILU>
__device__ __forceinline__ Row dpre_of(const Row& pre, const Row& dy) {
  Row r = dy;
  if constexpr (SILU) {
#pragma unroll
    for (int v = 0; v < kWide / 2; ++v) {
      const Pair one = pair(1.0f, 1.0f), s = sigmoid2(pre.v[v]);
      const Pair rest = fma2(s, pair(-1.0f, -1.0f), one);
      r.v[v] = mul2(mul2(dy.v[v], s), fma2(pre.v[v], rest, one));
    }
  }
  return r;
}

// Backward: the rows of a tile from the last to the first.  With dpre = dy silu'(pre), dx[t] = sum_j w[W-1-j] dpre[t+j]
// over the chain's rows, so the walk starts W - 1 rows behind the tile's end and keeps the dpre of the W - 1 rows
// it has passed; pre is computed again from x.  The sums for the taps are kept per tile and added in a second kernel.
template <typename T, int W, bool SILU, bool VEC>
__global__ __launch_bounds__(128, kConvBackwardBlocks) void conv_backward_kernel(ConvArgs<T> p) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t tile = id / p.columns, c = (id - tile * p.columns) * kWide;
  const int valid = static_cast<int>(p.width - c < kWide ? p.width - c : kWide);
  Taps<W> taps;
  const Row none{};
  if (tile >= p.tiles) {
    // the initial state's gradient, one row of one chain per thread: tap k = i - t of row t meets row i of the state
    const int64_t job = tile - p.tiles, s = job / (W - 1);
    const int i = static_cast<int>(job - s * (W - 1));
    if (p.grad_initial == nullptr || s >= p.chains.count) return;
    taps.load(p.weight, p.bias, c, valid);
    const int64_t a = p.chains.first(s), n = p.chains.end(s) - a;
    Row sum = none;
#pragma unroll
    for (int t = 0; t < W - 1; ++t) {
      if (t > i || t >= n) break;
      Row rows[W];
#pragma unroll
      for (int k = 0; k < W; ++k) rows[k] = widen(row_at<T, W, VEC>(p, s, a, t - (W - 1) + k, c, valid));
      const Row d = dpre_of<SILU>(taps.apply(rows), widen(load_block<T, kWide, VEC>(p.grad_y + (a + t) * p.grad_y_stride + c, valid)));
#pragma unroll
      for (int v = 0; v < kWide / 2; ++v) {
        Pair w = 0;
#pragma unroll
        for (int k = 0; k < W; ++k) w = k == i - t ? taps.w[k].v[v] : w;
        sum.v[v] = fma2(w, d.v[v], sum.v[v]);
      }
    }
    if (i >= n && p.grad_final != nullptr) {
      const Row g = widen(load_block<T, kWide, VEC>(p.grad_final + (s * (W - 1) + (i - n)) * p.width + c, valid));
#pragma unroll
      for (int v = 0; v < kWide / 2; ++v) sum.v[v] = add2(sum.v[v], g.v[v]);
    }
    store_block<T, kWide, VEC>(p.grad_initial + job * p.width + c, narrow<T>(sum), valid);
    return;
  }
  taps.load(p.weight, p.bias, c, valid);
  const int64_t r0 = tile * p.tile_rows;
  const int n = static_cast<int>(r0 + p.tile_rows < p.chains.rows ? p.tile_rows : p.chains.rows - r0);
  Row dw[W] = {}, db{};
  constexpr int kStages = conv_stages<T>();
  __shared__ Block<T, kWide> s_x[kStages * kAhead][128], s_g[kStages * kAhead][128];
  const Stream<T, kStages> xs{s_x}, gs{s_g};
  int t = n - 1;
  while (t >= 0) {
    // one chain's rows of the tile: low .. high
    const int64_t row = r0 + t, s = p.chains.of_row(row), a = p.chains.first(s);
    int64_t e = p.chains.end(s);
    if (e <= row) e = row + 1;  // offsets that decrease
    const int low = a > r0 && a <= row ? static_cast<int>(a - r0) : 0, high = t;
    if (s == p.chains.count) {
      // padding rows
      for (; t >= low; --t) {
        if (p.grad_x != nullptr) store_block<T, kWide, VEC>(p.grad_x + (r0 + t) * p.width + c, narrow<T>(none), valid);
      }
      continue;
    }
    t = high + (e - row < W ? static_cast<int>(e - row) : W) - 1;
    const T* px = p.x + r0 * p.x_stride + c;
    const T* pg = p.grad_y + r0 * p.grad_y_stride + c;
    const int64_t before = r0 - a;  // rows of the chain before the tile; negative when it starts inside
    const int inner = before >= W - 1 ? low : low + W - 1 - static_cast<int>(before + low);  // from here on the rows a row needs are x's own
    // in a batch of rows t, t-1, .. t-kAhead+1:  x[i] is the row t - i,  dp[W-1+i] the dpre of the row t - i
    Row x[kAhead + W - 1], dp[W - 1 + kAhead];
    auto load = [&](int from, int stage) {
      if (from < low) {
        close_batch();
        return;
      }
      const T *g = pg + static_cast<int64_t>(from) * p.grad_y_stride, *f = px + static_cast<int64_t>(from - (W - 1)) * p.x_stride;
      if (from - (kAhead - 1) >= inner) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i, g -= p.grad_y_stride, f -= p.x_stride) {
          gs.template copy<VEC>(stage * kAhead + i, g, valid);
          xs.template copy<VEC>(stage * kAhead + i, f, valid);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kAhead; ++i, g -= p.grad_y_stride) {
          const bool real = from - i >= low;
          gs.template copy<VEC>(stage * kAhead + i, real ? g : pg, real ? valid : 0);
          xs.put(stage * kAhead + i, row_at<T, W, VEC>(p, s, a, real ? before + from - i - (W - 1) : 0, c, real ? valid : 0));
        }
      }
      close_batch();
    };
    wait_batches<0>();  // the chain before may have left a copy on its way
#pragma unroll
    for (int d = 0; d < kStages - 1; ++d) load(t - d * kAhead, d);
    int stage = 0;
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
      x[k] = widen(row_at<T, W, VEC>(p, s, a, before + t - k, c, valid));
      dp[k] = none;
    }
    // dp, dw and db of row t - i, whose dpre goes on to dx
    auto step = [&](int i, const Row& dy, bool counts) {
      Row rows[W], out;
#pragma unroll
      for (int k = 0; k < W; ++k) rows[k] = x[i + W - 1 - k];
      dp[W - 1 + i] = dpre_of<SILU>(taps.apply(rows), dy);
#pragma unroll
      for (int v = 0; v < kWide / 2; ++v) {
        const Pair d = counts ? dp[W - 1 + i].v[v] : 0;
        db.v[v] = add2(db.v[v], d);
        out.v[v] = 0;
#pragma unroll
        for (int k = 0; k < W; ++k) {
          dw[k].v[v] = fma2(d, rows[k].v[v], dw[k].v[v]);
          out.v[v] = k ? fma2(taps.w[k].v[v], dp[i + k].v[v], out.v[v]) : mul2(taps.w[0].v[v], dp[i].v[v]);  // dp[i + k]: row t - i + W - 1 - k
        }
      }
      return out;
    };
    for (; t >= low; t -= kAhead) {
      Row dy[kAhead];
      wait_batches<kStages - 2>();
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        x[W - 1 + i] = widen(xs.get(stage * kAhead + i));
        dy[i] = widen(gs.get(stage * kAhead + i));
      }
      load(t - (kStages - 1) * kAhead, stage == 0 ? kStages - 1 : stage - 1);
      stage = stage == kStages - 1 ? 0 : stage + 1;
      T* to = p.grad_x + (r0 + t) * p.width + c;
      if (t <= high && t - (kAhead - 1) >= low && (p.grad_final == nullptr || e - (r0 + t) >= W) && p.grad_x != nullptr) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i, to -= p.width) store_block<T, kWide, VEC>(to, narrow<T>(step(i, dy[i], true)), valid);
      } else {
#pragma unroll
        for (int i = 0; i < kAhead; ++i, to -= p.width) {
          const int at = t - i;
          const bool counts = at <= high && at >= low;
          Row out = step(i, dy[i], counts);  // dy is 0 below `low`
          const int64_t behind = e - (r0 + at);  // rows of the chain from here on
          if (counts && p.grad_final != nullptr && behind <= W - 1) {
            const Row g = widen(load_block<T, kWide, VEC>(p.grad_final + (s * (W - 1) + (W - 1) - behind) * p.width + c, valid));
#pragma unroll
            for (int v = 0; v < kWide / 2; ++v) out.v[v] = add2(out.v[v], g.v[v]);
          }
          if (counts && p.grad_x != nullptr) store_block<T, kWide, VEC>(to, narrow<T>(out), valid);
        }
      }
#pragma unroll
      for (int k = 0; k < W - 1; ++k) {
        x[k] = x[k + kAhead];
        dp[k] = dp[k + kAhead];
      }
    }
    t = low - 1;
  }
  if (p.partial == nullptr) return;
  float* part = p.partial + tile * p.width * (W + 1);
#pragma unroll
  for (int v = 0; v < kWide; ++v) {
    if (v < valid) {
#pragma unroll
      for (int k = 0; k < W; ++k) part[(c + v) * W + k] = v & 1 ? halves(dw[k].v[v / 2]).y : halves(dw[k].v[v / 2]).x;
      part[p.width * W + c + v] = v & 1 ? halves(db.v[v / 2]).y : halves(db.v[v / 2]).x;
    }
  }
}

// One row per chain; the state moves up by one row.  The kernel in front may still be writing x, the taps or the state while this one starts, so no
// pointer is restrict: that would let the compiler read them before the wait.
template <typename T, int W, bool SILU, bool VEC>
__global__ __launch_bounds__(128) void conv_step_kernel(const T* x, int64_t x_stride, T* state, const float* weight, const float* bias, T* y, int64_t chains,
                                                        int64_t width, int64_t columns) {
  let_next_start();
  wait_for_previous();
  const int64_t id = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t s = id / columns, c = (id - s * columns) * kWide;
  if (s >= chains) return;
  const int valid = static_cast<int>(width - c < kWide ? width - c : kWide);
  Taps<W> taps;
  taps.load(weight, bias, c, valid);
  T* st = state + s * (W - 1) * width + c;
  Block<T, kWide> rows[W];
#pragma unroll
  for (int k = 0; k < W - 1; ++k) rows[k] = load_block<T, kWide, VEC>(st + k * width, valid);
  rows[W - 1] = load_block<T, kWide, VEC>(x + s * x_stride + c, valid);
  Row wide[W];
#pragma unroll
  for (int k = 0; k < W; ++k) wide[k] = widen(rows[k]);
  Row out = taps.apply(wide);
#pragma unroll
  for (int v = 0; v < kWide / 2; ++v) {
    if (SILU) out.v[v] = mul2(out.v[v], sigmoid2(out.v[v]));
  }
  store_block<T, kWide, VEC>(y + s * width + c, narrow<T>(out), valid);
#pragma unroll
  for (int k = 0; k < W - 1; ++k) store_block<T, kWide, VEC>(st + k * width, rows[k + 1], valid);
}

}  // namespace cufkb_seq
