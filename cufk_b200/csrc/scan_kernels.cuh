// Selective scan along packed chains: forward, backward and the single-row step.
//
//   dt = softplus(delta + bias)     a_t = exp(dt A[d,n])     h_t = a_t h_{t-1} + dt x B_t[n]
//   y  = (sum_n C_t[n] h_t[n] + D x) z sigmoid(z)
//
// Each (channel, state) pair is its own affine recurrence.  A group of LPC lanes holds two neighbouring channels, KN states of each
// per lane, and walks the rows; B_t and C_t are shared by all channels of a group and come from shared memory, two
// channels per read.  Multiplies and adds take two states at once (f32x2).  Per row and state the forward needs one
// exponential, of which an SM does 16 per clock, and two packed instructions' worth of arithmetic, so exponentials bound it: 72 us
// at 16384 x 1024 x 16, where memory would take 21.
// Between two lanes' states and the rows' scalars the work is turned around: for LPC / 2 rows at a time each lane owns one (row,
// channel) of its group.  It loads x, delta and z there, one element each (any stride and alignment will do), makes dt
// and dt x for the group, and after LPC - 1 shuffles holds that row's sum over the states, which it gates and stores.
//
// Long chains are cut into pieces that run in parallel.  A first launch takes each piece from a zero state and keeps its
// last state and its sum of dt; the decay over a whole piece is exp(A sum dt), so the second launch finds the state
// that a piece starts from with one multiply-add per earlier piece.  The backward does the same from the chain's end.
#pragma once

#include <cfloat>

#include "seq_common.cuh"

namespace cufkb_seq {

constexpr int kScanThreads = 128;
constexpr int kScanWarps = kScanThreads / 32;
constexpr int kChunk = 8;      // rows between checkpoints, and rows that a warp takes at a time
constexpr int kTile = 32;      // rows of B and C in the forward's shared memory
constexpr int kForwardBlocks = 4, kBackwardBlocks = 3;  // resident per SM: what the registers allow

// How many states (KN) and channels (KC) a thread holds and how many lanes share them, by the padded states of a channel.  Measured on
// B200 at 8192 x 2048 x 16 and 16384 x 1024 x 16 (bfloat16): the forward takes 267 us and 241 us with (8, 1), 271 and 271 with
// (8, 2), 300 and 276 with (4, 2), 292 and 286 with (4, 1); the backward 712 us with (4, 2), whose B and C are read once
// for two channels, and 888 us with (4, 1).  With 64 states (4096 x 2048 x 64) the forward takes 426 us with (8, 2) and 502 us with
// (8, 1), the backward 1544 us with (4, 2) and 1994 us with (8, 1).
template <int NP>
struct ForwardShape {
  static constexpr int KN = 8, KC = NP == 64 ? 2 : 1, LPC = NP / KN;
};
template <int NP>
struct BackwardShape {
  static constexpr int KN = 4, KC = 2, LPC = NP / KN;
};

template <typename T>
struct ScanArgs {
  Chains chains;
  int64_t items;
  int length;  // most rows of a piece, a multiple of kChunk
  int softplus;
  int width, group_width, states, blocks_per_group, blocks;  // blocks: of channels, over all groups
  const T *x, *delta, *z;
  int x_stride, delta_stride, z_stride;  // at most 2^24, but for a step: the rows of a tile are addressed with 32 bits from its first
  const float* A;
  const T *B, *C;
  int B_stride, C_stride;
  int64_t B_group_stride, C_group_stride;
  const float *D, *bias, *initial;
  T* y;
  float* final_state;
  float* checkpoints;  // [chunk id][width][padded states]
  float* piece_state;  // [slot][width][padded states]
  float* piece_dt;     // [slot][width]
  // backward
  int walkers;  // blocks that share the items of one channel block
  const T* grad_y;
  int grad_y_stride;
  const float* grad_final;
  T *grad_x, *grad_delta, *grad_z;
  float* grad_initial;
  float* partial_bc;  // [channel block][row][2][padded states]
  float* partial_A;   // [walker][width][states]
  float* partial_d;   // [walker][2][width]: D, then delta_bias
};

// Where a thread works: KC channels, KN of their states, and in turned-around phases one (row, channel) of its group.
template <int LPC, int KN, int KC>
struct Place {
  static constexpr int kGroups = 32 / LPC;
  static constexpr int kWarpChannels = KC * kGroups;
  static constexpr int kChannels = kScanWarps * kWarpChannels;  // of a block
  static constexpr int kStates = LPC * KN;                      // padded
  static constexpr int kBatch = LPC / KC;                       // rows that are turned around together
  static constexpr int kItems = kChunk / kBatch;                // (row, channel)s of a lane in a chunk
  static constexpr int kPairs = KN / 2;
  static_assert(kBatch <= kChunk && KN % 4 == 0, "a chunk holds whole batches");
  int group, first, count;  // the block's group, first channel and channels
  int lane, warp, g, q;     // q: the thread's place in its lane group
  int c0;                   // the thread's first channel in the block
  int n0;                   // the thread's first state
  int row, own, slot;       // of the turned-around phases: row of the batch, channel in the block and in the warp
  __device__ __forceinline__ Place(int block, int blocks_per_group, int group_width) {
    group = block / blocks_per_group;
    const int at = (block - group * blocks_per_group) * kChannels;
    first = group * group_width + at;
    count = group_width - at < kChannels ? group_width - at : kChannels;
    lane = threadIdx.x & 31;
    warp = threadIdx.x >> 5;
    g = lane / LPC;
    q = lane % LPC;
    c0 = warp * kWarpChannels + KC * g;
    n0 = q * KN;
    row = q / KC;
    slot = KC * g + q % KC;
    own = warp * kWarpChannels + slot;
  }
  __device__ __forceinline__ bool whole() const { return count == kChannels; }
  __device__ __forceinline__ bool idle() const { return warp * kWarpChannels >= count; }  // the whole warp
};

// The thread's states of its channels, out of (width, states) floats.
template <int KN, int KC>
__device__ __forceinline__ void load_states(Pair (&h)[KC][KN / 2], const float* base, int64_t channel, int left, int states, int n0) {
#pragma unroll
  for (int c = 0; c < KC; ++c) {
#pragma unroll
    for (int i = 0; i < KN / 2; ++i) {
      float v[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int n = n0 + 2 * i + k;
        v[k] = (base != nullptr && c < left && n < states) ? base[(channel + c) * states + n] : 0.0f;
      }
      h[c][i] = pair(v[0], v[1]);
    }
  }
}
// A log2(e), so that exp(dt A) is 2 to the power of dt times it.  -inf (of A, or of the product) becomes the lowest finite number: its
// exponential is 0 for any dt a row has, and 1 for the dt = 0 of the places behind a chain's end, where -inf would make NaN.
__device__ __forceinline__ float decay_of(float a) {
  const float v = a * kLog2e;
  return v < -FLT_MAX ? -FLT_MAX : v;
}
template <int KN, int KC>
__device__ __forceinline__ void load_decays(Pair (&A2)[KC][KN / 2], const float* A, int64_t channel, int left, int states, int n0) {
  load_states<KN, KC>(A2, A, channel, left, states, n0);
#pragma unroll
  for (int c = 0; c < KC; ++c) {
#pragma unroll
    for (int i = 0; i < KN / 2; ++i) {
      const float2 v = halves(A2[c][i]);
      A2[c][i] = pair(decay_of(v.x), decay_of(v.y));
    }
  }
}
template <int KN, int KC>
__device__ __forceinline__ void store_states(float* base, const Pair (&h)[KC][KN / 2], int64_t channel, int left, int states, int n0) {
#pragma unroll
  for (int c = 0; c < KC; ++c) {
#pragma unroll
    for (int i = 0; i < KN / 2; ++i) {
      const float2 v = halves(h[c][i]);
      if (c < left && n0 + 2 * i < states) base[(channel + c) * states + n0 + 2 * i] = v.x;
      if (c < left && n0 + 2 * i + 1 < states) base[(channel + c) * states + n0 + 2 * i + 1] = v.y;
    }
  }
}
// The same with padded states: 16-byte accesses.
template <int KN, int KC, int NP>
__device__ __forceinline__ void load_padded(Pair (&h)[KC][KN / 2], const float* base, int64_t channel, int left, int n0) {
#pragma unroll
  for (int c = 0; c < KC; ++c) {
#pragma unroll
    for (int i = 0; i < KN / 4; ++i) {
      ulonglong2 v = make_ulonglong2(0, 0);
      if (c < left) v = *reinterpret_cast<const ulonglong2*>(base + (channel + c) * NP + n0 + 4 * i);
      h[c][2 * i] = v.x;
      h[c][2 * i + 1] = v.y;
    }
  }
}
template <int KN, int KC, int NP>
__device__ __forceinline__ void store_padded(float* base, const Pair (&h)[KC][KN / 2], int64_t channel, int left, int n0) {
#pragma unroll
  for (int c = 0; c < KC; ++c) {
#pragma unroll
    for (int i = 0; i < KN / 4; ++i) {
      if (c < left) *reinterpret_cast<ulonglong2*>(base + (channel + c) * NP + n0 + 4 * i) = make_ulonglong2(h[c][2 * i], h[c][2 * i + 1]);
    }
  }
}

template <int PAIRS>
__device__ __forceinline__ void load_pairs(Pair (&dst)[PAIRS], const float* p) {
#pragma unroll
  for (int i = 0; i < PAIRS / 2; ++i) {
    const ulonglong2 v = reinterpret_cast<const ulonglong2*>(p)[i];
    dst[2 * i] = v.x;
    dst[2 * i + 1] = v.y;
  }
}

// What a group's lanes staged for one row of its channels.
template <int KC>
struct Staged {
  float2 v[KC];
  __device__ __forceinline__ explicit Staged(const float2* p) {
    if constexpr (KC == 2) {
      const float4 f = *reinterpret_cast<const float4*>(p);
      v[0] = make_float2(f.x, f.y);
      v[1] = make_float2(f.z, f.w);
    } else {
      v[0] = *p;
    }
  }
};
template <int KC>
struct StagedOne {
  float v[KC];
  __device__ __forceinline__ explicit StagedOne(const float* p) {
    if constexpr (KC == 2) {
      const float2 f = *reinterpret_cast<const float2*>(p);
      v[0] = f.x;
      v[1] = f.y;
    } else {
      v[0] = *p;
    }
  }
};

// Sums v[0..N) over the N lanes with equal lane / N; lane l % N ends with the sum of v[l % N].
template <int N>
__device__ __forceinline__ float sum_transposed(float (&v)[N], int q) {
#pragma unroll
  for (int half = N / 2; half > 0; half /= 2) {
    const bool upper = q & half;
#pragma unroll
    for (int i = 0; i < half; ++i) {
      const float keep = upper ? v[i + half] : v[i];
      const float send = upper ? v[i] : v[i + half];
      v[i] = keep + __shfl_xor_sync(kAll, send, half);
    }
  }
  return v[0];
}

// Rows of B or C on their way to shared memory.
template <typename T, int ROWS, int NP>
struct StageBc {
  static constexpr int kCount = (ROWS * NP + kScanThreads - 1) / kScanThreads;
  T v[kCount];
  // src: the first row; zero past the rows that are left and past the states
  __device__ __forceinline__ void load(const T* src, int rows, int stride, int states) {
#pragma unroll
    for (int k = 0; k < kCount; ++k) {
      const int i = threadIdx.x + k * kScanThreads, r = i / NP, n = i % NP;
      v[k] = (r < rows && n < states) ? src[r * stride + n] : from_float<T>(0.0f);
    }
  }
  __device__ __forceinline__ void store(float (*dst)[NP]) const {
#pragma unroll
    for (int k = 0; k < kCount; ++k) {
      const int i = threadIdx.x + k * kScanThreads;
      if (ROWS * NP % kScanThreads == 0 || i < ROWS * NP) dst[i / NP][i % NP] = to_float(v[k]);
    }
  }
};

// A lane's elements of a chunk of a (rows, width) activation: src is its first one, left the rows from there on.
template <typename T, int ITEMS, int BATCH>
struct OwnRows {
  T v[ITEMS];
  // full: no lane of the block is short of rows
  __device__ __forceinline__ void load(const T* src, int left, int stride, bool full) {
    if (full) {
#pragma unroll
      for (int k = 0; k < ITEMS; ++k) v[k] = src[k * BATCH * stride];
    } else {
#pragma unroll
      for (int k = 0; k < ITEMS; ++k) v[k] = k * BATCH < left ? src[k * BATCH * stride] : from_float<T>(0.0f);
    }
  }
};

// Where the first launch leaves what a piece hands over.  Only whole pieces hand over in the forward, and in the backward only pieces
// behind a whole one, which gives the slot: whole pieces never share one.
__device__ __forceinline__ int64_t slot_of(int64_t whole_piece_row, int length) { return whole_piece_row / length; }

// The chunks of a chain are numbered from first / kChunk + chain on, as pieces are.
__device__ __forceinline__ int64_t chunk_of(const Piece& p, int64_t row) { return p.chain_first / kChunk + p.chain + (row - p.chain_first) / kChunk; }

// Takes a state, or what a state's gradient hands back, over `count` whole pieces from the one at row `row` on, `step` rows apart.  What four of
// them hand over is on its way together.
template <typename T, int KN, int KC, int NP>
__device__ __forceinline__ void over_pieces(Pair (&h)[KC][KN / 2], const ScanArgs<T>& p, int64_t row, int64_t step, int64_t count, int channel, int left, int n0,
                                            const Pair (&A2)[KC][KN / 2]) {
  constexpr int kDeep = 4;
  for (int64_t j0 = 0; j0 < count; j0 += kDeep) {
    Pair e[kDeep][KC][KN / 2];
    float sum[kDeep][KC];
#pragma unroll
    for (int j = 0; j < kDeep; ++j) {
      const bool real = j0 + j < count;
      const int64_t slot = slot_of(row + (real ? j0 + j : 0) * step, p.length);
      load_padded<KN, KC, NP>(e[j], p.piece_state + slot * p.width * NP, channel, real ? left : 0, n0);
#pragma unroll
      for (int c = 0; c < KC; ++c) sum[j][c] = real && c < left ? p.piece_dt[slot * p.width + channel + c] : 0.0f;  // 0: the state stays
    }
#pragma unroll
    for (int j = 0; j < kDeep; ++j) {
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const Pair s = pair(sum[j][c], sum[j][c]);
#pragma unroll
        for (int i = 0; i < KN / 2; ++i) h[c][i] = fma2(decay2(s, A2[c][i]), h[c][i], e[j][c][i]);
      }
    }
  }
}

// LOCAL: the first launch for chains in several pieces; it runs every piece that another one follows, from a zero state, and
// keeps the last state and the sum of dt.  At 16384 x 1024 x 16 (bfloat16) the first launch takes 94 us, with the exponential unit 70%
// busy, and the second 135 us, with it 56% busy and an instruction issued in 56% of the clocks.
// What a chunk needs is loaded while the chunk before it is worked on.
template <typename T, int LPC, int KN, int KC, bool LOCAL>
__global__ __launch_bounds__(kScanThreads, kForwardBlocks) void scan_forward_kernel(ScanArgs<T> p) {
  using P = Place<LPC, KN, KC>;
  constexpr int NP = P::kStates, kBatch = P::kBatch, kItems = P::kItems, kPairs = P::kPairs;
  __shared__ __align__(16) float s_b[kTile][NP];
  __shared__ __align__(16) float s_c[LOCAL ? 1 : kTile][NP];
  __shared__ __align__(16) float2 s_du[kScanWarps][kChunk][P::kWarpChannels];  // dt, dt x

  if (LOCAL) let_next_start();
  const int64_t item = blockIdx.x / p.blocks;
  const P at(static_cast<int>(blockIdx.x - item * p.blocks), p.blocks_per_group, p.group_width);
  const Piece piece = find_piece(p.chains, item, p.length);
  const bool last = piece.end == piece.chain_end;
  if (LOCAL && (!piece.valid || last || piece.padding)) return;
  if (!piece.valid) {
    wait_for_previous();
    return;
  }
  if (piece.padding) {
    wait_for_previous();
    for (int64_t r = piece.first + at.warp; r < piece.end; r += kScanWarps) {
      for (int c = at.lane; c < at.count; c += 32) p.y[r * p.width + at.first + c] = from_float<T>(0.0f);
    }
    return;
  }
  const int channel = at.first + at.c0, left = at.count - at.c0;
  const bool mine = at.own < at.count;
  const int own = at.first + (mine ? at.own : 0);
  const int n = static_cast<int>(piece.end - piece.first);
  const int lane_end = mine ? n - at.row : 0;  // a lane without a channel has no rows
  // the lane's first element of each activation
  const int64_t first_row = piece.first + at.row;
  const T* px = p.x + first_row * p.x_stride + own;
  const T* pd = p.delta + first_row * p.delta_stride + own;
  const T* pz = p.z != nullptr ? p.z + first_row * p.z_stride + own : nullptr;
  T* py = p.y + first_row * p.width + own;

  StageBc<T, kTile, NP> bs, cs;
  const T* bp = p.B + at.group * p.B_group_stride + piece.first * p.B_stride;
  const T* cp = p.C + at.group * p.C_group_stride + piece.first * p.C_stride;
  auto load_tile = [&](int r0) {
    bs.load(bp + static_cast<int64_t>(r0) * p.B_stride, n - r0, p.B_stride, p.states);
    if constexpr (!LOCAL) cs.load(cp + static_cast<int64_t>(r0) * p.C_stride, n - r0, p.C_stride, p.states);
  };
  OwnRows<T, kItems, kBatch> xs, ds;
  auto load_chunk = [&](int r0) {
    const bool full = at.whole() && r0 + kChunk <= n;
    ds.load(pd + static_cast<int64_t>(r0) * p.delta_stride, lane_end - r0, p.delta_stride, full);
    xs.load(px + static_cast<int64_t>(r0) * p.x_stride, lane_end - r0, p.x_stride, full);
  };
  load_tile(0);
  load_chunk(0);
  const float bias = p.bias != nullptr ? p.bias[own] : 0.0f, D = !LOCAL && p.D != nullptr ? p.D[own] : 0.0f;

  Pair A2[KC][kPairs], h[KC][kPairs];
  load_decays<KN, KC>(A2, p.A, channel, left, p.states, at.n0);
  if (LOCAL) {
    load_states<KN, KC>(h, nullptr, channel, left, p.states, at.n0);
  } else {
    load_states<KN, KC>(h, p.initial != nullptr ? p.initial + piece.chain * p.width * p.states : nullptr, channel, left, p.states, at.n0);
    if (piece.index > 0) wait_for_previous();
    over_pieces<T, KN, KC, NP>(h, p, piece.chain_first, p.length, piece.index, channel, left, at.n0, A2);
  }
  float dt_sum = 0.0f;
  int64_t chunk = chunk_of(piece, piece.first);

  for (int tile = 0; tile < n; tile += kTile) {
    __syncthreads();
    bs.store(s_b);
    if constexpr (!LOCAL) cs.store(s_c);
    __syncthreads();
    if (tile + kTile < n) load_tile(tile + kTile);
    if (at.idle()) continue;
    const int stop = tile + kTile < n ? tile + kTile : n;
    for (int row0 = tile; row0 < stop; row0 += kChunk) {
      const int lane_left = lane_end - row0;
      const bool full = at.whole() && row0 + kChunk <= n;
#pragma unroll
      for (int k = 0; k < kItems; ++k) {
        float dt = to_float(ds.v[k]) + bias;
        if (p.softplus) dt = softplus(dt);
        // rows past the end count as dt = 0: they leave the state as it is
        if (!full && k * kBatch >= lane_left) dt = 0.0f;
        s_du[at.warp][k * kBatch + at.row][at.slot] = make_float2(dt, dt * to_float(xs.v[k]));
        if constexpr (LOCAL) dt_sum += dt;
      }
      if (row0 + kChunk < n) load_chunk(row0 + kChunk);
      OwnRows<T, kItems, kBatch> zs;
      if constexpr (!LOCAL) {
        if (p.z != nullptr) zs.load(pz + static_cast<int64_t>(row0) * p.z_stride, lane_left, p.z_stride, full);
      }
      __syncwarp();
      if (!LOCAL && p.checkpoints != nullptr) store_padded<KN, KC, NP>(p.checkpoints + chunk++ * p.width * NP, h, channel, left, at.n0);
      const int r0 = row0 - tile;
      float yv[LPC], y_own[kItems];
#pragma unroll
      for (int j = 0; j < kChunk; ++j) {
        const Staged<KC> du(&s_du[at.warp][j][KC * at.g]);
        Pair b[kPairs];
        load_pairs(b, &s_b[r0 + j][at.n0]);
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          const Pair dt = pair(du.v[c].x, du.v[c].x), u = pair(du.v[c].y, du.v[c].y);
#pragma unroll
          for (int i = 0; i < kPairs; ++i) h[c][i] = fma2(decay2(dt, A2[c][i]), h[c][i], mul2(u, b[i]));
        }
        if constexpr (!LOCAL) {
          Pair cc[kPairs];
          load_pairs(cc, &s_c[r0 + j][at.n0]);
#pragma unroll
          for (int c = 0; c < KC; ++c) {
            Pair y = mul2(h[c][0], cc[0]);
#pragma unroll
            for (int i = 1; i < kPairs; ++i) y = fma2(h[c][i], cc[i], y);
            yv[(j % kBatch) * KC + c] = sum_pair(y);
          }
          if (j % kBatch == kBatch - 1) y_own[j / kBatch] = sum_transposed<LPC>(yv, at.q);
        }
      }
      if constexpr (!LOCAL) {
        OwnRows<T, kItems, kBatch> x_now;  // from the cache: cheaper than registers held over the walk
        if (p.D != nullptr) {
          x_now.load(px + static_cast<int64_t>(row0) * p.x_stride, lane_left, p.x_stride, full);
#pragma unroll
          for (int k = 0; k < kItems; ++k) y_own[k] = fmaf(D, to_float(x_now.v[k]), y_own[k]);
        }
        if (p.z != nullptr) {
#pragma unroll
          for (int k = 0; k < kItems; ++k) {
            const float z = to_float(zs.v[k]);
            y_own[k] *= z * sigmoid(z);
          }
        }
        T* to = py + static_cast<int64_t>(row0) * p.width;
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
          if (full || k * kBatch < lane_left) to[k * kBatch * p.width] = from_float<T>(y_own[k]);
        }
      }
      __syncwarp();
    }
  }
  if (!LOCAL) wait_for_previous();
  if (at.idle()) return;
  if constexpr (LOCAL) {
    const int64_t slot = slot_of(piece.first, p.length);
    store_padded<KN, KC, NP>(p.piece_state + slot * p.width * NP, h, channel, left, at.n0);
#pragma unroll
    for (int half = LPC / 2; half >= KC; half /= 2) dt_sum += __shfl_xor_sync(kAll, dt_sum, half);
    if (mine && at.row == 0) p.piece_dt[slot * p.width + own] = dt_sum;
  } else if (last && p.final_state != nullptr) {
    store_states<KN, KC>(p.final_state + piece.chain * p.width * p.states, h, channel, left, p.states, at.n0);
  }
}

// ------------------------------------------------------------------------------------------
// backward
// ------------------------------------------------------------------------------------------
// With dypre = dy z sigmoid(z), g_t the gradient of h_t and R_t = a_t g_t what row t hands to row t - 1:
//   g_t = C_t dypre_t + R_{t+1}            m = g_t a_t h_{t-1}
//   dA += m dt      ddt = sum_n m A + x sum_n g B      dx = dt sum_n g B + D dypre      dB = sum_d g dt x      dC = sum_d h dypre
// A chunk of eight rows is run forward again from its checkpoint, a_t h_{t-1} staying in registers, then backward.  The sums over
// channels for dB and dC are taken over a warp's channels by shuffles, over its block's warps in shared memory, and
// over blocks in a second kernel, in an order that does not depend on timing.  At 8192 x 2048 x 16 in ragged chains (bfloat16) the
// first launch takes 94 us, the second 490: per row, eight channels and 16 states a warp issues 129 instructions in 250
// clocks with 2.8 warps per scheduler, which the registers of a_t h_{t-1} limit; eight instructions in ten are not
// exponentials, which would take 72 clocks.
// LOCAL: the first launch for chains in several pieces: R of every piece that another one comes before, from zero.

// Sums over the lanes that hold the same states of different channels (lane / LPC).  v[0..V) are V values per lane, V >= 32 / LPC a
// power of two; lane ends with the sums of the V LPC / 32 values from (lane / LPC) * (V LPC / 32) on, in v[0..).
template <int LPC, int V>
__device__ __forceinline__ void sum_channels(float (&v)[V], int lane) {
  int n = V;
#pragma unroll
  for (int half = 16; half >= LPC; half /= 2) {
    const bool upper = lane & half;
    n /= 2;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      if (i < n) {
        const float keep = upper ? v[i + n] : v[i];
        const float send = upper ? v[i] : v[i + n];
        v[i] = keep + __shfl_xor_sync(kAll, send, half);
      }
    }
  }
}

template <typename T, int LPC, int KN, int KC, bool LOCAL>
__global__ __launch_bounds__(kScanThreads, LOCAL ? 4 : kBackwardBlocks) void scan_backward_kernel(ScanArgs<T> p) {
  using P = Place<LPC, KN, KC>;
  constexpr int NP = P::kStates, kBatch = P::kBatch, kItems = P::kItems, kPairs = P::kPairs;
  __shared__ __align__(16) float s_b[LOCAL ? 1 : kChunk][NP];
  __shared__ __align__(16) float s_c[kChunk][NP];
  __shared__ __align__(16) float2 s_du[kScanWarps][kChunk][P::kWarpChannels];  // dt, dt x
  __shared__ __align__(16) float s_dyp[kScanWarps][kChunk][P::kWarpChannels];  // dypre
  constexpr int kGroupRows = P::kGroups > KN ? P::kGroups / KN : 1;  // rows whose dB or dC are summed over channels together
  constexpr int kSums = kGroupRows * KN;
  constexpr int kLeft = kSums * LPC / 32;  // sums a lane ends with
  __shared__ float s_bc[LOCAL ? 1 : kScanWarps][2][kChunk][NP];                // dB, dC of each warp's channels

  if (LOCAL) let_next_start();
  const int64_t walker = blockIdx.x / p.blocks;
  const int block = static_cast<int>(blockIdx.x - walker * p.blocks);
  const P at(block, p.blocks_per_group, p.group_width);
  const int channel = at.first + at.c0, left = at.count - at.c0;
  const bool mine = at.own < at.count;
  const int own = at.first + (mine ? at.own : 0);
  const float bias = p.bias != nullptr ? p.bias[own] : 0.0f, D = p.D != nullptr ? p.D[own] : 0.0f;

  Pair A2[KC][kPairs], dA[KC][kPairs] = {};
  load_decays<KN, KC>(A2, p.A, channel, left, p.states, at.n0);
  float dD = 0.0f, dbias = 0.0f;
  if constexpr (!LOCAL) {
    if (at.idle()) {
      for (int i = at.lane; i < 2 * kChunk * NP; i += 32) (&s_bc[at.warp][0][0][0])[i] = 0.0f;
    }
  }

  bool waited = LOCAL;
  for (int64_t item = walker; item < p.items; item += p.walkers) {
    const Piece piece = find_piece(p.chains, item, p.length);
    if (!piece.valid) continue;
    if (LOCAL && (piece.index == 0 || piece.padding)) continue;
    if (piece.padding) {
      for (int64_t r = piece.first + at.warp; r < piece.end; r += kScanWarps) {
        for (int c = at.lane; c < at.count; c += 32) {
          const int64_t w = r * p.width + at.first + c;
          p.grad_x[w] = p.grad_delta[w] = from_float<T>(0.0f);
          if (p.z != nullptr) p.grad_z[w] = from_float<T>(0.0f);
        }
        for (int i = at.lane; i < 2 * NP; i += 32) p.partial_bc[(static_cast<int64_t>(block) * p.chains.rows + r) * (2 * NP) + i] = 0.0f;
      }
      continue;
    }
    const int n = static_cast<int>(piece.end - piece.first), chunks = (n + kChunk - 1) / kChunk;
    const int lane_end = mine ? n - at.row : 0;  // a lane without a channel has no rows
    const int64_t first_row = piece.first + at.row;
    const T* px = p.x + first_row * p.x_stride + own;
    const T* pd = p.delta + first_row * p.delta_stride + own;
    const T* pz = p.z != nullptr ? p.z + first_row * p.z_stride + own : nullptr;
    const T* pg = p.grad_y + first_row * p.grad_y_stride + own;
    const int64_t out0 = first_row * p.width + own;
    const T* bp = p.B + at.group * p.B_group_stride + piece.first * p.B_stride;
    const T* cp = p.C + at.group * p.C_group_stride + piece.first * p.C_stride;
    const int64_t chunk0 = chunk_of(piece, piece.first);
    StageBc<T, kChunk, NP> bs, cs;
    OwnRows<T, kItems, kBatch> xs, ds, zs, gs;
    Pair start[KC][kPairs];
    auto load_chunk = [&](int k) {
      const int r0 = k * kChunk, lane_left = lane_end - r0;
      cs.load(cp + static_cast<int64_t>(r0) * p.C_stride, n - r0, p.C_stride, p.states);
      if constexpr (!LOCAL) bs.load(bp + static_cast<int64_t>(r0) * p.B_stride, n - r0, p.B_stride, p.states);
      const bool full = at.whole() && r0 + kChunk <= n;
      ds.load(pd + static_cast<int64_t>(r0) * p.delta_stride, lane_left, p.delta_stride, full);
      gs.load(pg + static_cast<int64_t>(r0) * p.grad_y_stride, lane_left, p.grad_y_stride, full);
      if (p.z != nullptr) zs.load(pz + static_cast<int64_t>(r0) * p.z_stride, lane_left, p.z_stride, full);
      if constexpr (!LOCAL) {
        xs.load(px + static_cast<int64_t>(r0) * p.x_stride, lane_left, p.x_stride, full);
        load_padded<KN, KC, NP>(start, p.checkpoints + (chunk0 + k) * p.width * NP, channel, left, at.n0);
      }
    };
    if (chunks > 0) load_chunk(chunks - 1);
    if (!waited) {
      wait_for_previous();
      waited = true;
    }
    Pair R[KC][kPairs];
    if (LOCAL) {
      load_states<KN, KC>(R, nullptr, channel, left, p.states, at.n0);
    } else {
      // what the chain's end hands back, through the pieces behind this one
      load_states<KN, KC>(R, p.grad_final != nullptr ? p.grad_final + piece.chain * p.width * p.states : nullptr, channel, left, p.states, at.n0);
      const int64_t behind = pieces_of(piece.chain_end - piece.chain_first, p.length) - 1 - piece.index;
      over_pieces<T, KN, KC, NP>(R, p, piece.chain_first + (piece.index + behind - 1) * p.length, -p.length, behind, channel, left, at.n0, A2);
    }
    float dt_sum = 0.0f;
    for (int k = chunks - 1; k >= 0; --k) {
      const int r0 = k * kChunk, lane_left = lane_end - r0;
      const bool full = at.whole() && r0 + kChunk <= n;
      // the last sync of the chunk before stands between its reads and these writes
      cs.store(s_c);
      if constexpr (!LOCAL) bs.store(s_b);
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        float dt = to_float(ds.v[i]) + bias;
        if (p.softplus) dt = softplus(dt);
        if (!full && i * kBatch >= lane_left) dt = 0.0f;  // leaves what is handed back as it is
        float dyp = to_float(gs.v[i]);
        if (p.z != nullptr) {
          const float z = to_float(zs.v[i]);
          dyp *= z * sigmoid(z);
        }
        const int r = i * kBatch + at.row;
        s_dyp[at.warp][r][at.slot] = dyp;
        s_du[at.warp][r][at.slot] = make_float2(dt, LOCAL ? 0.0f : dt * to_float(xs.v[i]));
        if constexpr (LOCAL) dt_sum += dt;
      }
      Pair h[KC][kPairs];
#pragma unroll
      for (int c = 0; c < KC; ++c) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) h[c][i] = LOCAL ? 0 : start[c][i];
      }
      __syncthreads();
      if constexpr (LOCAL) {
        if (k > 0) load_chunk(k - 1);
#pragma unroll
        for (int t = kChunk - 1; t >= 0; --t) {
          const Staged<KC> du(&s_du[at.warp][t][KC * at.g]);
          const StagedOne<KC> dy(&s_dyp[at.warp][t][KC * at.g]);
          Pair cc[kPairs];
          load_pairs(cc, &s_c[t][at.n0]);
#pragma unroll
          for (int c = 0; c < KC; ++c) {
            const Pair dt = pair(du.v[c].x, du.v[c].x), dyp = pair(dy.v[c], dy.v[c]);
#pragma unroll
            for (int i = 0; i < kPairs; ++i) R[c][i] = mul2(decay2(dt, A2[c][i]), fma2(cc[i], dyp, R[c][i]));
          }
        }
        __syncthreads();
      } else {
        if (!at.idle()) {
          Pair ah[kChunk][KC][kPairs];  // a_t h_(t-1)
          float y_own[kItems];
          float yv[LPC], sums[kSums];
#pragma unroll
          for (int t = 0; t < kChunk; ++t) {
            const Staged<KC> du(&s_du[at.warp][t][KC * at.g]);
            const StagedOne<KC> dy(&s_dyp[at.warp][t][KC * at.g]);
            Pair b[kPairs], cc[kPairs], dC[kPairs];
            load_pairs(b, &s_b[t][at.n0]);
            load_pairs(cc, &s_c[t][at.n0]);
#pragma unroll
            for (int c = 0; c < KC; ++c) {
              const Pair dt = pair(du.v[c].x, du.v[c].x), u = pair(du.v[c].y, du.v[c].y);
              const Pair dyp = pair(dy.v[c], dy.v[c]);
              Pair y = 0;
#pragma unroll
              for (int i = 0; i < kPairs; ++i) {
                ah[t][c][i] = mul2(decay2(dt, A2[c][i]), h[c][i]);
                h[c][i] = fma2(u, b[i], ah[t][c][i]);
                dC[i] = c ? fma2(h[c][i], dyp, dC[i]) : mul2(h[c][i], dyp);
                y = i ? fma2(h[c][i], cc[i], y) : mul2(h[c][i], cc[i]);
              }
              yv[(t % kBatch) * KC + c] = sum_pair(y);
            }
#pragma unroll
            for (int i = 0; i < kPairs; ++i) {
              const float2 v = halves(dC[i]);
              sums[(t % kGroupRows) * KN + 2 * i] = v.x;
              sums[(t % kGroupRows) * KN + 2 * i + 1] = v.y;
            }
            if (t % kGroupRows == kGroupRows - 1) {
              sum_channels<LPC, kSums>(sums, at.lane);
#pragma unroll
              for (int i = 0; i < kLeft; ++i) {
                const int e = at.g * kLeft + i;
                s_bc[at.warp][1][t - (kGroupRows - 1) + e / KN][at.n0 + e % KN] = sums[i];
              }
            }
            if (t % kBatch == kBatch - 1) y_own[t / kBatch] = sum_transposed<LPC>(yv, at.q);
          }
          asm volatile("" ::: "memory");  // read the staged rows again: what the first walk read would fill the registers
          float sa[LPC], sb[LPC], ma_own[kItems], gb_own[kItems];
          Pair dA_now[KC][kPairs] = {};  // of this chunk: a long sum of small terms keeps its accuracy in two levels
#pragma unroll
          for (int t = kChunk - 1; t >= 0; --t) {
            // the next chunk's loads go out once half of a_t h_(t-1) has left its registers to them
            if (t == kChunk / 2 - 1 && k > 0) load_chunk(k - 1);
            const Staged<KC> du(&s_du[at.warp][t][KC * at.g]);
            const StagedOne<KC> dy(&s_dyp[at.warp][t][KC * at.g]);
            Pair b[kPairs], cc[kPairs], dB[kPairs];
            load_pairs(b, &s_b[t][at.n0]);
            load_pairs(cc, &s_c[t][at.n0]);
#pragma unroll
            for (int c = 0; c < KC; ++c) {
              const Pair dt = pair(du.v[c].x, du.v[c].x), u = pair(du.v[c].y, du.v[c].y);
              const Pair dyp = pair(dy.v[c], dy.v[c]);
              Pair ma = 0, gb = 0;
#pragma unroll
              for (int i = 0; i < kPairs; ++i) {
                const Pair gr = fma2(cc[i], dyp, R[c][i]);
                const Pair m = mul2(gr, ah[t][c][i]);
                dA_now[c][i] = fma2(m, dt, dA_now[c][i]);
                ma = i ? fma2(m, A2[c][i], ma) : mul2(m, A2[c][i]);
                gb = i ? fma2(gr, b[i], gb) : mul2(gr, b[i]);
                dB[i] = c ? fma2(gr, u, dB[i]) : mul2(gr, u);
                R[c][i] = mul2(decay2(dt, A2[c][i]), gr);  // a_t once more: cheaper than its registers
              }
              sa[(t % kBatch) * KC + c] = sum_pair(ma);
              sb[(t % kBatch) * KC + c] = sum_pair(gb);
            }
#pragma unroll
            for (int i = 0; i < kPairs; ++i) {
              const float2 v = halves(dB[i]);
              sums[(t % kGroupRows) * KN + 2 * i] = v.x;
              sums[(t % kGroupRows) * KN + 2 * i + 1] = v.y;
            }
            if (t % kGroupRows == 0) {
              sum_channels<LPC, kSums>(sums, at.lane);
#pragma unroll
              for (int i = 0; i < kLeft; ++i) {
                const int e = at.g * kLeft + i;
                s_bc[at.warp][0][t + e / KN][at.n0 + e % KN] = sums[i];
              }
            }
            if (t % kBatch == 0) {
              ma_own[t / kBatch] = sum_transposed<LPC>(sa, at.q);
              gb_own[t / kBatch] = sum_transposed<LPC>(sb, at.q);
            }
          }
#pragma unroll
          for (int c = 0; c < KC; ++c) {
#pragma unroll
            for (int i = 0; i < kPairs; ++i) dA[c][i] = add2(dA[c][i], dA_now[c][i]);
          }
          // this lane's rows and channel once more, from the cache: cheaper than registers held over both walks
          OwnRows<T, kItems, kBatch> x_now, d_now;
          x_now.load(px + static_cast<int64_t>(r0) * p.x_stride, lane_left, p.x_stride, full);
          if (p.softplus) d_now.load(pd + static_cast<int64_t>(r0) * p.delta_stride, lane_left, p.delta_stride, full);
          const int64_t out = out0 + static_cast<int64_t>(r0) * p.width;
          T *to_x = p.grad_x + out, *to_d = p.grad_delta + out;
#pragma unroll
          for (int i = 0; i < kItems; ++i) {
            const int r = i * kBatch + at.row;
            const float x = to_float(x_now.v[i]), dyp = s_dyp[at.warp][r][at.slot], dt = s_du[at.warp][r][at.slot].x;
            float dd = fmaf(gb_own[i], x, ma_own[i] * kLn2);
            if (p.softplus) dd *= sigmoid(to_float(d_now.v[i]) + bias);
            if (full || i * kBatch < lane_left) {
              dD = fmaf(dyp, x, dD);
              dbias += dd;
              to_x[i * kBatch * p.width] = from_float<T>(fmaf(gb_own[i], dt, D * dyp));
              to_d[i * kBatch * p.width] = from_float<T>(dd);
            }
          }
          if (p.z != nullptr) {
            OwnRows<T, kItems, kBatch> z_now, g_now;
            z_now.load(pz + static_cast<int64_t>(r0) * p.z_stride, lane_left, p.z_stride, full);
            g_now.load(pg + static_cast<int64_t>(r0) * p.grad_y_stride, lane_left, p.grad_y_stride, full);
            T* to_z = p.grad_z + out;
#pragma unroll
            for (int i = 0; i < kItems; ++i) {
              const float z = to_float(z_now.v[i]), sg = sigmoid(z);
              const float dz = to_float(g_now.v[i]) * fmaf(D, to_float(x_now.v[i]), y_own[i]) * sg * fmaf(z, 1.0f - sg, 1.0f);
              if (full || i * kBatch < lane_left) to_z[i * kBatch * p.width] = from_float<T>(dz);
            }
          }
        } else if (k > 0) {
          load_chunk(k - 1);
        }
        __syncthreads();
#pragma unroll
        for (int i = threadIdx.x; i < 2 * kChunk * NP; i += kScanThreads) {
          const int r = i / (2 * NP), w = i % (2 * NP);
          if (r0 + r < n) {
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < kScanWarps; ++j) sum += s_bc[j][w / NP][r][w % NP];
            p.partial_bc[(static_cast<int64_t>(block) * p.chains.rows + piece.first + r0 + r) * (2 * NP) + w] = sum;
          }
        }
      }
    }
    if constexpr (LOCAL) {
      const int64_t slot = slot_of(piece.first - p.length, p.length);
      store_padded<KN, KC, NP>(p.piece_state + slot * p.width * NP, R, channel, left, at.n0);
#pragma unroll
      for (int half = LPC / 2; half >= KC; half /= 2) dt_sum += __shfl_xor_sync(kAll, dt_sum, half);
      if (mine && at.row == 0) p.piece_dt[slot * p.width + own] = dt_sum;
    } else if (piece.index == 0 && p.grad_initial != nullptr) {
      store_states<KN, KC>(p.grad_initial + piece.chain * p.width * p.states, R, channel, left, p.states, at.n0);
    }
  }
  if (!waited) wait_for_previous();
  if constexpr (!LOCAL) {
    store_states<KN, KC>(p.partial_A + walker * p.width * p.states, dA, channel, left, p.states, at.n0);
#pragma unroll
    for (int half = LPC / 2; half >= KC; half /= 2) {
      dD += __shfl_xor_sync(kAll, dD, half);
      dbias += __shfl_xor_sync(kAll, dbias, half);
    }
    if (mine && at.row == 0) {
      p.partial_d[walker * 2 * p.width + own] = dD;
      p.partial_d[(walker * 2 + 1) * p.width + own] = dbias;
    }
  }
}

// What the backward's blocks left, added in order: dB and dC over the channel blocks of a group (bc_blocks blocks of this kernel), then dA, dD
// and d delta_bias over the walkers (32 columns to a block, as sum_partials_kernel does).
template <typename T, int NP>
__global__ __launch_bounds__(256) void scan_finish_kernel(ScanArgs<T> p, int groups, T* __restrict__ grad_B, T* __restrict__ grad_C, float* __restrict__ grad_A,
                                                        float* __restrict__ grad_D, float* __restrict__ grad_bias, int bc_blocks, int A_blocks) {
  if (static_cast<int>(blockIdx.x) < bc_blocks) {
    const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int64_t per = p.chains.rows * (2 * NP);
    if (id >= per * groups) return;
    const int64_t g = id / per, in = id - g * per, t = in / (2 * NP);
    const int w = static_cast<int>(in % (2 * NP)), n = w % NP;
    if (n >= p.states) return;
    const float* part = p.partial_bc + g * p.blocks_per_group * per + in;
    float sum = 0.0f;
#pragma unroll 8
    for (int b = 0; b < p.blocks_per_group; ++b) sum += part[b * per];
    T* out = w < NP ? grad_B : grad_C;
    out[(t * groups + g) * p.states + n] = from_float<T>(sum);
    return;
  }
  const int block = static_cast<int>(blockIdx.x) - bc_blocks;
  if (block < A_blocks) {
    const int64_t columns = static_cast<int64_t>(p.width) * p.states;
    sum_partials(p.partial_A, p.walkers, columns, block, columns, grad_A, nullptr);
  } else {
    sum_partials(p.partial_d, p.walkers, 2 * static_cast<int64_t>(p.width), block - A_blocks, p.width, grad_D, grad_bias);
  }
}

// One row per chain: LPC lanes hold the states of a channel, four each, and the state is updated in place.  Reading and writing the states
// bounds it, as long as little else is done: a thread takes its channel in four chains, so that A is read once for them, and lane q
// makes dt and the gate of chain q % 4 only, for the group, and stores that chain's y.  256 chains of 2048 x 16 (67 MB of states read and
// written) take 16 us; one chain per thread, with every lane making its own dt, took 27.
constexpr int kStepChains = 4;

template <typename T, int LPC, bool VEC>
__global__ __launch_bounds__(kScanThreads) void scan_step_kernel(ScanArgs<T> p) {
  constexpr int kPer = 4;
  let_next_start();
  wait_for_previous();
  const int d = (blockIdx.x * kScanThreads + threadIdx.x) / LPC, q = threadIdx.x % LPC, n0 = q * kPer;
  if (static_cast<int>(blockIdx.x * (kScanThreads / LPC) + (threadIdx.x & ~31) / LPC) >= p.width) return;  // the whole warp
  const bool mine = d < p.width;
  const int g = p.group_width == p.width || !mine ? 0 : d / p.group_width;
  const int left = mine ? p.states - n0 : 0;
  const int own = mine ? d : 0;
  Block<float, kPer> A = load_block<float, kPer, VEC>(p.A + static_cast<int64_t>(own) * p.states + n0, left);
#pragma unroll
  for (int i = 0; i < kPer; ++i) A.v[i] = decay_of(A.v[i]);
  const float bias = p.bias != nullptr ? p.bias[own] : 0.0f, D = p.D != nullptr ? p.D[own] : 0.0f;
  const T *bp = p.B + g * p.B_group_stride + n0, *cp = p.C + g * p.C_group_stride + n0;
  const int64_t next = static_cast<int64_t>(p.width) * p.states;
  const int64_t set = static_cast<int64_t>(gridDim.y) * kStepChains;
  for (int64_t s0 = static_cast<int64_t>(blockIdx.y) * kStepChains; s0 < p.chains.count; s0 += set) {
    // spare places read the first chain once more and store nothing
    const int real = static_cast<int>(p.chains.count - s0 < kStepChains ? p.chains.count - s0 : kStepChains);
    const int64_t s = s0 + ((q & 3) < real ? q & 3 : 0);
    const float raw = to_float(p.delta[s * p.delta_stride + own]) + bias, x = to_float(p.x[s * p.x_stride + own]);
    const float z = p.z != nullptr ? to_float(p.z[s * p.z_stride + own]) : 0.0f;
    float* state = p.final_state + s0 * next + static_cast<int64_t>(own) * p.states + n0;
    Block<float, kPer> h[kStepChains];
    Block<T, kPer> b[kStepChains], c[kStepChains];
#pragma unroll
    for (int k = 0; k < kStepChains; ++k) {
      const int j = k < real ? k : 0;
      h[k] = load_block<float, kPer, VEC>(state + j * next, left);
      b[k] = load_block<T, kPer, VEC>(bp + (s0 + j) * p.B_stride, left);
      c[k] = load_block<T, kPer, VEC>(cp + (s0 + j) * p.C_stride, left);
    }
    const float dt = p.softplus ? softplus(raw) : raw, u = dt * x;
    float y[kStepChains];
#pragma unroll
    for (int k = 0; k < kStepChains; ++k) {
      const float dk = __shfl_sync(kAll, dt, k, 4), uk = __shfl_sync(kAll, u, k, 4);
      y[k] = 0.0f;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        h[k].v[i] = fmaf(decay(dk, A.v[i]), h[k].v[i], uk * to_float(b[k].v[i]));
        y[k] = i < left ? fmaf(h[k].v[i], to_float(c[k].v[i]), y[k]) : y[k];
      }
      if (k < real) store_block<float, kPer, VEC>(state + k * next, h[k], left);
#pragma unroll
      for (int half = LPC / 2; half >= 4; half /= 2) y[k] += __shfl_xor_sync(kAll, y[k], half);
    }
    float sum = fmaf(D, x, sum_transposed<4>(y, q & 3));
    if (p.z != nullptr) sum *= z * sigmoid(z);
    if (mine && q < real) p.y[s * p.width + own] = from_float<T>(sum);
  }
}

}  // namespace cufkb_seq
