// Plan and argument block of a scan call, shared by its forward and backward entry points.
#pragma once

#include "scan_kernels.cuh"
#include "seq_api.cuh"

namespace cufkb_seq {

template <template <int> class Shape>
int64_t block_channels(int64_t padded) {
  switch (padded) {
    case 8:
      return kScanThreads / Shape<8>::LPC * Shape<8>::KC;
    case 16:
      return kScanThreads / Shape<16>::LPC * Shape<16>::KC;
    case 32:
      return kScanThreads / Shape<32>::LPC * Shape<32>::KC;
    default:
      return kScanThreads / Shape<64>::LPC * Shape<64>::KC;
  }
}

struct ScanPlan {
  int64_t padded;  // states of a channel, rounded up to 8, 16, 32 or 64
  int64_t blocks_per_group, blocks;
  int length;
  bool pieces;  // some chain may have several
  int64_t items, slots, walkers;
};

// Rows of a piece: so that the pieces give the SMs their resident blocks, but at least a few chunks, and equal ones where all chains are
// equal.  Ragged chains leave pieces of any length, so three times as many: the SMs that get short ones take more.  Measured on
// B200 at 8192 x 2048 x 16 in 16 ragged chains with one, two, three and four times: forward 248, 225, 221, 231 us, backward 703,
// 608, 582, 592 us; one chain of 16384 x 1024 x 16: forward 236, 252, 287, 332 us.
inline ScanPlan scan_plan(const cufkb_scan_params& q, bool backward) {
  ScanPlan p;
  p.padded = q.states <= 8 ? 8 : q.states <= 16 ? 16 : q.states <= 32 ? 32 : 64;
  const int64_t group_width = q.width / q.groups, channels = backward ? block_channels<BackwardShape>(p.padded) : block_channels<ForwardShape>(p.padded);
  p.blocks_per_group = ceil_div(group_width, channels);
  p.blocks = p.blocks_per_group * q.groups;
  const bool packed = q.chain_points != nullptr;
  const int64_t resident = kSms * (backward ? kBackwardBlocks : kForwardBlocks) * (packed && q.chains > 1 ? 3 : 1);
  const int64_t uniform = packed || q.chains == 0 ? 0 : q.rows / q.chains;
  int64_t length = ceil_div(q.rows * p.blocks, resident);
  // A chain's last piece takes the state over all pieces before it and walks its own rows twice, at about 2.5 times as many clocks a row
  // as a piece before it costs: with few channels, where more pieces would still find room, 2 L^2 rows of a chain in pieces of L
  // are best (8192 x 64 x 16, one chain: 58 us; 62 and 73 us with 3 and 6 in the place of 2, 155 us with pieces of 16 rows).
  const int64_t average = q.chains > 0 ? ceil_div(q.rows, q.chains) : 0;
  const int64_t longest = packed ? (4 * average < q.rows ? 4 * average : q.rows) : uniform;
  int64_t least = 2 * kChunk;
  while (least < (1 << 15) && 2 * least * least < longest) least += kChunk;
  if (length < least) length = least;
  if (!packed && uniform > 0) length = ceil_div(uniform, pieces_of(uniform, length));
  if (length > (1 << 30)) length = 1 << 30;
  p.length = static_cast<int>(ceil_div(length, kChunk) * kChunk);
  p.pieces = (packed ? q.rows : uniform) > p.length;
  p.items = item_count(packed, q.rows, uniform, q.chains, p.length);
  p.slots = q.rows / p.length + 1;
  // partial sums of A, D and the bias are kept per walker
  const int64_t most = ceil_div(kSms * 16, p.blocks) > 16 ? ceil_div(kSms * 16, p.blocks) : 16;
  p.walkers = p.items < most ? p.items : most;
  return p;
}

struct ScanSpace {
  size_t piece_state, piece_dt, partial_bc, partial_A, partial_d, total;
};

inline ScanSpace scan_space(const cufkb_scan_params& q, const ScanPlan& p, bool backward) {
  ScanSpace s{};
  size_t at = 0;
  auto take = [&](int64_t floats) {
    const size_t here = at;
    at += round16(static_cast<size_t>(floats) * sizeof(float));
    return here;
  };
  s.piece_state = take(p.pieces ? p.slots * q.width * p.padded : 0);
  s.piece_dt = take(p.pieces ? p.slots * q.width : 0);
  if (backward) {
    s.partial_bc = take(p.blocks * q.rows * 2 * p.padded);
    s.partial_A = take(p.walkers * q.width * q.states);
    s.partial_d = take(p.walkers * 2 * q.width);
  }
  s.total = at;
  return s;
}

inline int scan_check(const cufkb_scan_params& q, int64_t most_stride = CUFKB_MAX_SCAN_STRIDE) {
  if (int st = check_activation_dtype(q.dtype)) return st;
  if (int st = check_rows(q.rows, q.chains, q.width, q.chain_points)) return st;
  if (q.states < 1 || q.states > CUFKB_MAX_STATES || q.groups < 1 || q.width % q.groups != 0) return CUFKB_ERROR_INVALID_VALUE;
  int64_t const strides1[] = {q.x_stride, q.delta_stride, q.z_stride, q.B_stride, q.B_group_stride, q.C_stride, q.C_group_stride, q.grad_y_stride};
  for (int64_t stride : strides1) {
    if (stride < 0) return CUFKB_ERROR_BAD_STRIDE;
  }
  const int64_t row_strides[] = {q.x_stride, q.delta_stride, q.z_stride, q.B_stride, q.C_stride, q.grad_y_stride};
  for (int64_t stride : row_strides) {
    if (stride > most_stride) return CUFKB_ERROR_BAD_STRIDE;
  }
  const size_t e = element_size(q.dtype);
  const void* const ptrs2[] = {q.x, q.delta, q.z, q.B, q.C, static_cast<const void*>(q.y), q.grad_y, static_cast<const void*>(q.grad_x),
                          static_cast<const void*>(q.grad_delta), static_cast<const void*>(q.grad_z), static_cast<const void*>(q.grad_B),
                          static_cast<const void*>(q.grad_C)};
  for (const void* ptr : ptrs2) {
    if (!aligned_to(ptr, e)) return CUFKB_ERROR_MISALIGNED;
  }
  const float* const ptrs3[] = {q.A, q.D, q.delta_bias, q.initial_state, static_cast<const float*>(q.final_state), q.grad_final_state,
                           static_cast<const float*>(q.grad_A), static_cast<const float*>(q.grad_D), static_cast<const float*>(q.grad_delta_bias),
                           static_cast<const float*>(q.grad_initial_state)};
  for (const float* ptr : ptrs3) {
    if (!aligned_to(ptr, 4)) return CUFKB_ERROR_MISALIGNED;
  }
  if (!aligned_to(q.checkpoints, 16) || !aligned_to(q.workspace, 16)) return CUFKB_ERROR_MISALIGNED;
  return CUFKB_SUCCESS;
}

inline int scan_check_inputs(const cufkb_scan_params& q) {
  if (q.A == nullptr || (q.rows > 0 && (q.x == nullptr || q.delta == nullptr || q.B == nullptr || q.C == nullptr))) return CUFKB_ERROR_NULL_POINTER;
  return CUFKB_SUCCESS;
}

template <typename T>
ScanArgs<T> scan_args(const cufkb_scan_params& q, const ScanPlan& p, const ScanSpace& s) {
  ScanArgs<T> a{};
  a.chains = chains_of(q.chain_points, q.rows, q.chains);
  a.items = p.items;
  a.length = p.length;
  a.softplus = q.softplus;
  a.width = static_cast<int>(q.width);
  a.group_width = static_cast<int>(q.width / q.groups);
  a.states = static_cast<int>(q.states);
  a.blocks_per_group = static_cast<int>(p.blocks_per_group);
  a.blocks = static_cast<int>(p.blocks);
  a.x = static_cast<const T*>(q.x);
  a.delta = static_cast<const T*>(q.delta);
  a.z = static_cast<const T*>(q.z);
  a.x_stride = static_cast<int>(q.x_stride);
  a.delta_stride = static_cast<int>(q.delta_stride);
  a.z_stride = static_cast<int>(q.z_stride);
  a.A = q.A;
  a.B = static_cast<const T*>(q.B);
  a.C = static_cast<const T*>(q.C);
  a.B_stride = static_cast<int>(q.B_stride);
  a.B_group_stride = q.B_group_stride;
  a.C_stride = static_cast<int>(q.C_stride);
  a.C_group_stride = q.C_group_stride;
  a.D = q.D;
  a.bias = q.delta_bias;
  a.initial = q.initial_state;
  a.y = static_cast<T*>(q.y);
  a.final_state = q.final_state;
  a.checkpoints = q.checkpoints;
  a.walkers = static_cast<int>(p.walkers);
  a.grad_y = static_cast<const T*>(q.grad_y);
  a.grad_y_stride = static_cast<int>(q.grad_y_stride);
  a.grad_final = q.grad_final_state;
  a.grad_x = static_cast<T*>(q.grad_x);
  a.grad_delta = static_cast<T*>(q.grad_delta);
  a.grad_z = static_cast<T*>(q.grad_z);
  a.grad_initial = q.grad_initial_state;
  char* w = static_cast<char*>(q.workspace);
  if (w != nullptr) {
    a.piece_state = reinterpret_cast<float*>(w + s.piece_state);
    a.piece_dt = reinterpret_cast<float*>(w + s.piece_dt);
    a.partial_bc = reinterpret_cast<float*>(w + s.partial_bc);
    a.partial_A = reinterpret_cast<float*>(w + s.partial_A);
    a.partial_d = reinterpret_cast<float*>(w + s.partial_d);
  }
  return a;
}

}  // namespace cufkb_seq
