// C entry points of the token log probabilities.
#include "logprob_kernels.cuh"
#include "seq_api.cuh"

namespace cufkb_seq {
namespace {

template <typename T>
struct Forward {
  static int run(const void* logits, int64_t stride, const int64_t* tokens, float* logp, float* entropy, float* log_sum, float* top_logp, int64_t* top_tokens,
                 int64_t rows, int64_t n, int top, cudaStream_t stream) {
    const T* l = static_cast<const T*>(logits);
    const int count = static_cast<int>(n);
    // Threads that share a row: a warp up to 1024 tokens, 128 up to 4096 and wherever rows fill the SMs, else 1024.  Measured (a call in us, bfloat16, the 8
    // largest): with a warp, 128 and 1024 threads 33, 53 and 3196 at 16384 rows of 1024, 47, 61 and 559 at 2048, 70, 70 and 555 at 4096; at 64 rows 10, 10 and
    // 35, then 12, 10 and 10, then 16, 10 and 10.  With 128 and 1024 threads 12 and 10, 14 and 16, 14 and 23 at 148, 296 and 444 rows of 8192, 23 and 12, 25
    // and 21, 26 and 27 at 32768.  A warp would still be faster at many rows of up to 2048, and 1024 threads at some hundred rows of 131072 (592: 80 and 57).
    if (n <= 1024) {
      const int64_t blocks = ceil_div(rows, 4);
      if (blocks > INT32_MAX) return CUFKB_ERROR_SHAPE_LIMITS;
      logprobs_kernel<T, 32><<<static_cast<unsigned>(blocks), 128, 0, stream>>>(l, stride, tokens, logp, entropy, log_sum, top_logp, top_tokens, rows, count, top);
    } else if (rows > INT32_MAX) {
      return CUFKB_ERROR_SHAPE_LIMITS;
    } else if (rows >= kSms * 2 || n <= 4096) {
      // 256 threads instead of 128 took 147 us for 86 at 4096 x 32768 (bfloat16)
      logprobs_kernel<T, 128><<<static_cast<unsigned>(rows), 128, 0, stream>>>(l, stride, tokens, logp, entropy, log_sum, top_logp, top_tokens, rows, count, top);
    } else {
      logprobs_kernel<T, 1024><<<static_cast<unsigned>(rows), 1024, 0, stream>>>(l, stride, tokens, logp, entropy, log_sum, top_logp, top_tokens, rows, count, top);
    }
    return launch_status();
  }
};

template <typename T>
struct Backward {
  static int run(const void* logits, int64_t stride, const int64_t* tokens, const float* entropy, const float* log_sum, const float* grad_logp,
                 const float* grad_entropy, void* grad, int64_t rows, int64_t n, cudaStream_t stream) {
    constexpr int N = 16 / sizeof(T);
    const T* l = static_cast<const T*>(logits);
    T* g = static_cast<T*>(grad);
    const bool wide = n % N == 0 && stride % N == 0 && aligned_to(l, 16) && aligned_to(g, 16);
    const int count = static_cast<int>(n);
    if (wide && n / N >= 256) {
      const int64_t parts = ceil_div(n / N, 256 * kGradBlocks);
      if (rows * parts > INT32_MAX) return CUFKB_ERROR_SHAPE_LIMITS;
      logprobs_backward_rows_kernel<T><<<static_cast<unsigned>(rows * parts), 256, 0, stream>>>(l, stride, tokens, entropy, log_sum, grad_logp, grad_entropy, g, count,
                                                                                               static_cast<int>(parts));
      return launch_status();
    }
    const int64_t per = wide ? n / N : n, blocks = ceil_div(rows * per, 256);
    if (blocks > INT32_MAX) return CUFKB_ERROR_SHAPE_LIMITS;
    const unsigned grid = static_cast<unsigned>(blocks);
    if (wide) {
      logprobs_backward_kernel<T, N><<<grid, 256, 0, stream>>>(l, stride, tokens, entropy, log_sum, grad_logp, grad_entropy, g, rows, count, static_cast<int>(per));
    } else {
      logprobs_backward_kernel<T, 1><<<grid, 256, 0, stream>>>(l, stride, tokens, entropy, log_sum, grad_logp, grad_entropy, g, rows, count, static_cast<int>(per));
    }
    return launch_status();
  }
};

int check(int dtype, const void* logits, int64_t stride, int64_t rows, int64_t n) {
  if (int st = check_activation_dtype(dtype)) return st;
  if (rows < 0 || n < 1 || n > INT32_MAX || rows > (int64_t{1} << 40)) return CUFKB_ERROR_SHAPE_LIMITS;
  if (stride < 0) return CUFKB_ERROR_BAD_STRIDE;
  if (!aligned_to(logits, element_size(dtype))) return CUFKB_ERROR_MISALIGNED;
  return CUFKB_SUCCESS;
}

}  // namespace
}  // namespace cufkb_seq

using namespace cufkb_seq;

extern "C" {

int cufkb_token_logprobs(int dtype, const void* logits, int64_t logits_stride, const int64_t* tokens, float* logp, float* entropy, float* log_sum,
                         float* top_logp, int64_t* top_tokens, int64_t rows, int64_t tokens_count, int top, cufkb_stream_t stream) {
  if (int st = check(dtype, logits, logits_stride, rows, tokens_count)) return st;
  if (top < 0 || top > CUFKB_MAX_TOP || top > tokens_count) return CUFKB_ERROR_INVALID_VALUE;
  if (rows == 0) return CUFKB_SUCCESS;
  if (logits == nullptr || tokens == nullptr || logp == nullptr || entropy == nullptr || log_sum == nullptr) return CUFKB_ERROR_NULL_POINTER;
  if (top > 0 && (top_logp == nullptr || top_tokens == nullptr)) return CUFKB_ERROR_NULL_POINTER;
  if (!aligned_to(tokens, 8) || !aligned_to(top_tokens, 8) || !aligned_to(logp, 4) || !aligned_to(entropy, 4) || !aligned_to(log_sum, 4) ||
      !aligned_to(top_logp, 4)) {
    return CUFKB_ERROR_MISALIGNED;
  }
  return for_activation<Forward>(dtype, logits, logits_stride, tokens, logp, entropy, log_sum, top_logp, top_tokens, rows, tokens_count, top,
                                 reinterpret_cast<cudaStream_t>(stream));
}

int cufkb_token_logprobs_backward(int dtype, const void* logits, int64_t logits_stride, const int64_t* tokens, const float* entropy, const float* log_sum,
                                  const float* grad_logp, const float* grad_entropy, void* grad_logits, int64_t rows, int64_t tokens_count,
                                  cufkb_stream_t stream) {
  if (int st = check(dtype, logits, logits_stride, rows, tokens_count)) return st;
  if (rows == 0) return CUFKB_SUCCESS;
  if (logits == nullptr || tokens == nullptr || entropy == nullptr || log_sum == nullptr || grad_logits == nullptr) return CUFKB_ERROR_NULL_POINTER;
  if (!aligned_to(tokens, 8) || !aligned_to(grad_logits, element_size(dtype)) || !aligned_to(entropy, 4) || !aligned_to(log_sum, 4) ||
      !aligned_to(grad_logp, 4) || !aligned_to(grad_entropy, 4)) {
    return CUFKB_ERROR_MISALIGNED;
  }
  return for_activation<Backward>(dtype, logits, logits_stride, tokens, entropy, log_sum, grad_logp, grad_entropy, grad_logits, rows, tokens_count,
                                  reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
