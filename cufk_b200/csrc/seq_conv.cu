// C entry points of the short causal convolution.
#include "conv_kernels.cuh"
#include "seq_api.cuh"

namespace cufkb_seq {
namespace {

struct ConvPlan {
  int64_t columns, tiles;
  int tile_rows;
};

// Rows per tile: one wave of blocks, but at least 8 rows (a tile reads W - 1 rows more than its own).
ConvPlan plan_of(int64_t rows, int64_t width, bool backward) {
  ConvPlan p;
  p.columns = ceil_div(width, kWide);
  const int64_t threads = kSms * (backward ? kConvBackwardBlocks : kConvForwardBlocks) * 128;
  int64_t tile_rows = ceil_div(rows * p.columns, threads);
  tile_rows = tile_rows < 8 ? 8 : tile_rows > (1 << 20) ? 1 << 20 : tile_rows;
  p.tile_rows = static_cast<int>(ceil_div(tile_rows, kAhead) * kAhead);
  p.tiles = ceil_div(rows, p.tile_rows);
  return p;
}

int check(const cufkb_conv_params& q) {
  if (int st = check_activation_dtype(q.dtype)) return st;
  if (int st = check_rows(q.rows, q.chains, q.width, q.chain_points)) return st;
  if (q.taps < CUFKB_MIN_TAPS || q.taps > CUFKB_MAX_TAPS) return CUFKB_ERROR_INVALID_VALUE;
  if (q.x_stride < 0 || q.grad_y_stride < 0) return CUFKB_ERROR_BAD_STRIDE;
  const size_t e = element_size(q.dtype);
  const void* const ptrs1[] = {q.x, q.initial_state, static_cast<const void*>(q.y), static_cast<const void*>(q.final_state), q.grad_y, q.grad_final_state,
                          static_cast<const void*>(q.grad_x), static_cast<const void*>(q.grad_initial_state)};
  for (const void* ptr : ptrs1) {
    if (!aligned_to(ptr, e)) return CUFKB_ERROR_MISALIGNED;
  }
  const float* const ptrs2[] = {q.weight, q.bias, static_cast<const float*>(q.grad_weight), static_cast<const float*>(q.grad_bias)};
  for (const float* ptr : ptrs2) {
    if (!aligned_to(ptr, 4)) return CUFKB_ERROR_MISALIGNED;
  }
  return CUFKB_SUCCESS;
}

template <typename T>
ConvArgs<T> args_of(const cufkb_conv_params& q, const ConvPlan& plan) {
  ConvArgs<T> a{};
  a.chains = chains_of(q.chain_points, q.rows, q.chains);
  a.width = q.width;
  a.columns = plan.columns;
  a.tiles = plan.tiles;
  a.tile_rows = plan.tile_rows;
  a.x = static_cast<const T*>(q.x);
  a.x_stride = q.x_stride;
  a.weight = q.weight;
  a.bias = q.bias;
  a.initial = static_cast<const T*>(q.initial_state);
  a.y = static_cast<T*>(q.y);
  a.final_state = static_cast<T*>(q.final_state);
  a.grad_y = static_cast<const T*>(q.grad_y);
  a.grad_y_stride = q.grad_y_stride;
  a.grad_final = static_cast<const T*>(q.grad_final_state);
  a.grad_x = static_cast<T*>(q.grad_x);
  a.grad_initial = static_cast<T*>(q.grad_initial_state);
  a.partial = q.grad_weight != nullptr ? static_cast<float*>(q.workspace) : nullptr;
  return a;
}

// four channels at once need every row to start on a four-element boundary
template <typename T>
bool wide_ok(const ConvArgs<T>& a) {
  const size_t block = kWide * sizeof(T);
  if (a.width % kWide != 0 || a.x_stride % kWide != 0 || a.grad_y_stride % kWide != 0) return false;
  const T* const ptrs3[] = {a.x, a.initial, static_cast<const T*>(a.y), static_cast<const T*>(a.final_state), a.grad_y, a.grad_final,
                       static_cast<const T*>(a.grad_x), static_cast<const T*>(a.grad_initial)};
  for (const T* ptr : ptrs3) {
    if (!aligned_to(ptr, block)) return false;
  }
  return true;
}

template <typename T, int W, bool SILU>
int launch(const ConvArgs<T>& a, bool backward, cudaStream_t stream) {
  const bool states = backward ? a.grad_initial != nullptr : a.final_state != nullptr;
  const int64_t threads = (a.tiles + (states ? a.chains.count * (W - 1) : 0)) * a.columns;
  const int64_t blocks = ceil_div(threads, 128);
  if (blocks == 0) return CUFKB_SUCCESS;
  if (blocks > INT32_MAX) return CUFKB_ERROR_SHAPE_LIMITS;
  const unsigned grid = static_cast<unsigned>(blocks);
  const bool wide = wide_ok(a);
  if (backward) {
    if (wide) {
      conv_backward_kernel<T, W, SILU, true><<<grid, 128, 0, stream>>>(a);
    } else {
      conv_backward_kernel<T, W, SILU, false><<<grid, 128, 0, stream>>>(a);
    }
  } else {
    if (wide) {
      conv_forward_kernel<T, W, SILU, true><<<grid, 128, 0, stream>>>(a);
    } else {
      conv_forward_kernel<T, W, SILU, false><<<grid, 128, 0, stream>>>(a);
    }
  }
  return launch_status();
}

template <typename T>
struct Run {
  static int run(const cufkb_conv_params& q, const ConvPlan& plan, bool backward, cudaStream_t stream) {
    const ConvArgs<T> a = args_of<T>(q, plan);
    switch (q.taps * 2 + (q.silu != 0)) {
      case 4:
        return launch<T, 2, false>(a, backward, stream);
      case 5:
        return launch<T, 2, true>(a, backward, stream);
      case 6:
        return launch<T, 3, false>(a, backward, stream);
      case 7:
        return launch<T, 3, true>(a, backward, stream);
      case 8:
        return launch<T, 4, false>(a, backward, stream);
      default:
        return launch<T, 4, true>(a, backward, stream);
    }
  }
};

template <typename T, int W>
int launch_step(const T* x, int64_t x_stride, T* state, const float* weight, const float* bias, T* y, int64_t chains, int64_t width, bool silu,
                cudaStream_t stream) {
  const int64_t columns = ceil_div(width, kWide), blocks = ceil_div(chains * columns, 128);
  if (blocks > INT32_MAX) return CUFKB_ERROR_SHAPE_LIMITS;
  const unsigned grid = static_cast<unsigned>(blocks);
  const size_t block = kWide * sizeof(T);
  const bool wide = width % kWide == 0 && x_stride % kWide == 0 && aligned_to(x, block) && aligned_to(state, block) && aligned_to(y, block);
  auto* kernel = silu ? (wide ? conv_step_kernel<T, W, true, true> : conv_step_kernel<T, W, true, false>)
                      : (wide ? conv_step_kernel<T, W, false, true> : conv_step_kernel<T, W, false, false>);
  return launch_dependent(kernel, dim3(grid), 128, stream, x, x_stride, state, weight, bias, y, chains, width, columns);
}

template <typename T>
struct Step {
  static int run(const void* x, int64_t x_stride, void* state, const float* weight, const float* bias, void* y, int64_t chains, int64_t width, int taps,
                 bool silu, cudaStream_t stream) {
    const T* xt = static_cast<const T*>(x);
    T *st = static_cast<T*>(state), *yt = static_cast<T*>(y);
    if (taps == 2) return launch_step<T, 2>(xt, x_stride, st, weight, bias, yt, chains, width, silu, stream);
    if (taps == 3) return launch_step<T, 3>(xt, x_stride, st, weight, bias, yt, chains, width, silu, stream);
    return launch_step<T, 4>(xt, x_stride, st, weight, bias, yt, chains, width, silu, stream);
  }
};

}  // namespace
}  // namespace cufkb_seq

using namespace cufkb_seq;

extern "C" {

int cufkb_conv_forward(const cufkb_conv_params* params, cufkb_stream_t stream) {
  if (params == nullptr) return CUFKB_ERROR_NULL_POINTER;
  const cufkb_conv_params& q = *params;
  if (int st = check(q)) return st;
  if (q.width == 0) return CUFKB_SUCCESS;
  if (q.weight == nullptr || (q.rows > 0 && (q.x == nullptr || q.y == nullptr))) return CUFKB_ERROR_NULL_POINTER;
  if (q.rows > 1 && q.x_stride < 0) return CUFKB_ERROR_BAD_STRIDE;
  return for_activation<Run>(q.dtype, q, plan_of(q.rows, q.width, false), false, reinterpret_cast<cudaStream_t>(stream));
}

int cufkb_conv_backward_workspace_bytes(const cufkb_conv_params* params, size_t* bytes) {
  if (params == nullptr || bytes == nullptr) return CUFKB_ERROR_NULL_POINTER;
  if (int st = check(*params)) return st;
  const ConvPlan plan = plan_of(params->rows, params->width, true);
  *bytes = static_cast<size_t>(plan.tiles) * params->width * (params->taps + 1) * sizeof(float);
  return CUFKB_SUCCESS;
}

int cufkb_conv_backward(const cufkb_conv_params* params, cufkb_stream_t stream) {
  if (params == nullptr) return CUFKB_ERROR_NULL_POINTER;
  const cufkb_conv_params& q = *params;
  if (int st = check(q)) return st;
  if (q.width == 0) return CUFKB_SUCCESS;
  if (q.weight == nullptr || (q.rows > 0 && (q.x == nullptr || q.grad_y == nullptr))) return CUFKB_ERROR_NULL_POINTER;
  if ((q.grad_weight == nullptr) != (q.grad_bias == nullptr)) return CUFKB_ERROR_NULL_POINTER;
  const ConvPlan plan = plan_of(q.rows, q.width, true);
  const int64_t columns = q.width * (q.taps + 1);
  if (q.grad_weight != nullptr && plan.tiles > 0) {
    if (q.workspace == nullptr || q.workspace_bytes < static_cast<size_t>(plan.tiles) * columns * sizeof(float)) return CUFKB_ERROR_WORKSPACE;
    if (!aligned_to(q.workspace, 16)) return CUFKB_ERROR_MISALIGNED;
  }
  const auto s = reinterpret_cast<cudaStream_t>(stream);
  if (int st = for_activation<Run>(q.dtype, q, plan, true, s)) return st;
  if (q.grad_weight == nullptr) return CUFKB_SUCCESS;
  sum_partials_kernel<<<static_cast<unsigned>(ceil_div(columns, 32)), 256, 0, s>>>(static_cast<const float*>(q.workspace), plan.tiles, columns, q.width * q.taps,
                                                                                q.grad_weight, q.grad_bias);
  return launch_status();
}

int cufkb_conv_step(int dtype, const void* x, int64_t x_stride, void* state, const float* weight, const float* bias, void* y, int64_t chains,
                    int64_t width, int taps, int silu, cufkb_stream_t stream) {
  if (int st = check_activation_dtype(dtype)) return st;
  if (int st = check_rows(chains, chains, width, nullptr)) return st;
  if (taps < CUFKB_MIN_TAPS || taps > CUFKB_MAX_TAPS) return CUFKB_ERROR_INVALID_VALUE;
  if (x_stride < 0) return CUFKB_ERROR_BAD_STRIDE;
  if (chains == 0 || width == 0) return CUFKB_SUCCESS;
  if (x == nullptr || state == nullptr || weight == nullptr || y == nullptr) return CUFKB_ERROR_NULL_POINTER;
  const size_t e = element_size(dtype);
  if (!aligned_to(x, e) || !aligned_to(state, e) || !aligned_to(y, e) || !aligned_to(weight, 4) || !aligned_to(bias, 4)) return CUFKB_ERROR_MISALIGNED;
  return for_activation<Step>(dtype, x, x_stride, state, weight, bias, y, chains, width, taps, silu != 0, reinterpret_cast<cudaStream_t>(stream));
}

const char* cufkb_seq_status_string(int status) {
  switch (status) {
    case CUFKB_ERROR_SHAPE_LIMITS:
      return "a size is negative or too large, or rows do not split into equal chains";
    case CUFKB_ERROR_BAD_STRIDE:
      return "strides must not be negative, nor the row strides of a scan over 2^24 elements (of its step 2^31 - 1)";
    case CUFKB_ERROR_INVALID_VALUE:
      return "a count is out of its range (taps 2 to 4, states 1 to 64, groups that divide the width, top 0 to 32), or arrays of a clipping share memory that one of "
             "them is written to";
    case CUFKB_ERROR_WORKSPACE:
      return "workspace or checkpoints are missing or too small";
    case CUFKB_ERROR_UNSUPPORTED_DTYPE:
      return "activations are float32, float16 or bfloat16";
    default:
      return cufkb_status_string(status);
  }
}

}  // extern "C"

namespace cufkb_seq {
namespace {
thread_local int g_last_cuda_error = 0;
}
int cuda_status(cudaError_t e) {
  if (e == cudaSuccess) return CUFKB_SUCCESS;
  g_last_cuda_error = static_cast<int>(e);
  return CUFKB_ERROR_CUDA;
}
}  // namespace cufkb_seq

extern "C" int cufkb_seq_last_cuda_error(void) { return cufkb_seq::g_last_cuda_error; }
