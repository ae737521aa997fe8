/*
 * cufkb_seq.h — C ABI of the sequence operators along packed chains (libcufkb.so).
 *
 * The operators of a model that reads and writes chains next to their reconstruction: a short causal
 * convolution and a selective scan (prompts, training, single tokens), log probabilities of given
 * tokens, and gradient clipping by the global norm.  No counterpart in the reference, whose path
 * ends at xyz.  Conventions are those of cufkb.h: plain device pointers, sizes, a dtype code and a
 * stream; asynchronous launches; status codes; no allocation and no synchronisation.
 *
 * Packed rows.  Row-major activations of `rows` rows hold `chains` chains.  chain_points is a device
 * array of chains+1 int64 offsets, chain_points[0] = 0, nondecreasing: chain s owns the rows
 * [chain_points[s], chain_points[s+1]) and may be empty.  Rows past chain_points[chains] are padding:
 * their results and gradients are zero.  chain_points NULL means chains of equal length, rows =
 * chains * length.  Offsets stay on the device; the kernels clamp them to [0, rows], so that wrong
 * ones give wrong rows but no access outside the arrays.
 *
 * Activations are float32, float16 or bfloat16 (CUFKB_ERROR_UNSUPPORTED_DTYPE otherwise), computed in
 * float and rounded once on output; parameters (taps, bias, A, D, delta_bias), scan states and
 * parameter gradients are float32.  Row strides count elements; columns are contiguous.
 */
#ifndef CUFKB_SEQ_H_
#define CUFKB_SEQ_H_

#include "cufkb.h"

#ifdef __cplusplus
extern "C" {
#endif

#define CUFKB_MAX_STATES 64
#define CUFKB_MIN_TAPS 2
#define CUFKB_MAX_TAPS 4
#define CUFKB_MAX_TOP 32
#define CUFKB_MAX_SCAN_STRIDE (1 << 24) /* elements between the rows of a scan */
#define CUFKB_MAX_STEP_STRIDE 0x7fffffff /* and of its single-row step */

/* Short causal convolution, one filter per channel: pre[t] = bias + sum_k weight[:, k] x[t-taps+1+k],
 * y = pre sigmoid(pre) (silu != 0) or pre.  Rows before a chain's start are initial_state's taps-1 rows,
 * oldest first, or zero; final_state gets the last taps-1 rows.  States are in the activations' dtype.
 * The backward takes grad_y and (optionally) grad_final_state and writes every gradient whose pointer
 * is not NULL. */
typedef struct cufkb_conv_params {
  int dtype, taps, silu;
  int64_t rows, chains, width;
  const int64_t* chain_points;  /* (chains+1) or NULL */
  const void* x;                /* (rows, width), row stride x_stride */
  int64_t x_stride;
  const float* weight;          /* (width, taps) */
  const float* bias;            /* (width) or NULL */
  const void* initial_state;    /* (chains, taps-1, width) or NULL */
  void* y;                      /* (rows, width) contiguous */
  void* final_state;            /* (chains, taps-1, width) or NULL */
  const void* grad_y;           /* (rows, width), row stride grad_y_stride */
  int64_t grad_y_stride;
  const void* grad_final_state; /* (chains, taps-1, width) or NULL */
  void* grad_x;                 /* (rows, width) contiguous or NULL */
  float* grad_weight;           /* (width, taps); both or neither of grad_weight, grad_bias may be NULL */
  float* grad_bias;             /* (width) */
  void* grad_initial_state;     /* (chains, taps-1, width) or NULL */
  void* workspace;              /* backward with grad_weight: cufkb_conv_backward_workspace_bytes, 16-byte aligned */
  size_t workspace_bytes;
} cufkb_conv_params;

CUFKB_API int cufkb_conv_forward(const cufkb_conv_params* params, cufkb_stream_t stream);
CUFKB_API int cufkb_conv_backward_workspace_bytes(const cufkb_conv_params* params, size_t* bytes);
CUFKB_API int cufkb_conv_backward(const cufkb_conv_params* params, cufkb_stream_t stream);

/* One row per chain: y from x (chains, width) and state (chains, taps-1, width), which then drops its oldest
 * row and takes x as its newest. */
CUFKB_API int cufkb_conv_step(int dtype, const void* x, int64_t x_stride, void* state, const float* weight, const float* bias, void* y,
                              int64_t chains, int64_t width, int taps, int silu, cufkb_stream_t stream);

/* Selective scan: dt = softplus(delta + delta_bias) (softplus != 0) or delta + delta_bias; per channel d and
 * state n  h_t = exp(dt A[d,n]) h_{t-1} + dt x B_t[g,n];  y = (sum_n C_t[g,n] h_t + D x) z sigmoid(z), with
 * g the group of width/groups consecutive channels that d lies in.  h starts from initial_state or zero;
 * final_state gets the last h.  D, z and delta_bias may be NULL (0, no gate, 0).
 * Training: the forward also fills `checkpoints` (h every 8 rows), which the backward reads. */
typedef struct cufkb_scan_params {
  int dtype, softplus;
  int64_t rows, chains, width, groups, states;
  const int64_t* chain_points; /* (chains+1) or NULL */
  const void *x, *delta, *z;   /* (rows, width), row strides below (all row strides at most CUFKB_MAX_SCAN_STRIDE); z may be NULL */
  int64_t x_stride, delta_stride, z_stride;
  const float* A;              /* (width, states) */
  const void *B, *C;           /* (rows, groups, states): row and group strides, states contiguous */
  int64_t B_stride, B_group_stride, C_stride, C_group_stride;
  const float *D, *delta_bias; /* (width) or NULL */
  const float* initial_state;  /* (chains, width, states) or NULL */
  void* y;                     /* (rows, width) contiguous */
  float* final_state;          /* (chains, width, states) or NULL */
  float* checkpoints;          /* cufkb_scan_checkpoint_bytes, 16-byte aligned; NULL when no backward follows */
  const void* grad_y;          /* (rows, width), row stride grad_y_stride */
  int64_t grad_y_stride;
  const float* grad_final_state; /* (chains, width, states) or NULL */
  /* the gradients, contiguous in the shapes above; grad_z NULL when z is, grad_D, grad_delta_bias and
   * grad_initial_state optional */
  void *grad_x, *grad_delta, *grad_z, *grad_B, *grad_C;
  float *grad_A, *grad_D, *grad_delta_bias, *grad_initial_state;
  void* workspace;             /* cufkb_scan_workspace_bytes, 16-byte aligned; NULL when that is 0 */
  size_t workspace_bytes;
} cufkb_scan_params;

CUFKB_API int cufkb_scan_checkpoint_bytes(const cufkb_scan_params* params, size_t* bytes);
CUFKB_API int cufkb_scan_workspace_bytes(const cufkb_scan_params* params, int backward, size_t* bytes);
CUFKB_API int cufkb_scan_forward(const cufkb_scan_params* params, cufkb_stream_t stream);
CUFKB_API int cufkb_scan_backward(const cufkb_scan_params* params, cufkb_stream_t stream);

/* One row per chain (rows = chains, chain_points, checkpoints and workspace ignored): `final_state`
 * (chains, width, states) is read and updated in place.  Row strides are at most CUFKB_MAX_STEP_STRIDE. */
CUFKB_API int cufkb_scan_step(const cufkb_scan_params* params, cufkb_stream_t stream);

/* Per row of logits (rows, tokens_count), row stride logits_stride: logp of the given token, the entropy
 * -sum p log p, and the `top` largest logits' log probabilities and ids, largest first, ties to the lowest id
 * (NaN above +inf).  Results are float32; log_sum (rows, 2) gets the row's largest logit and the log of the sum of
 * exp(logit - largest), for the backward.  A negative
 * token means "none": logp 0; one >= tokens_count gives NaN.  A row of -inf only has logp -inf (none: 0),
 * entropy 0 and a zero gradient. */
CUFKB_API int cufkb_token_logprobs(int dtype, const void* logits, int64_t logits_stride, const int64_t* tokens, float* logp, float* entropy,
                                   float* log_sum, float* top_logp, int64_t* top_tokens, int64_t rows, int64_t tokens_count, int top,
                                   cufkb_stream_t stream);

/* grad_logits (rows, tokens_count) contiguous from grad_logp and grad_entropy (either may be NULL: zero). */
CUFKB_API int cufkb_token_logprobs_backward(int dtype, const void* logits, int64_t logits_stride, const int64_t* tokens, const float* entropy,
                                            const float* log_sum, const float* grad_logp, const float* grad_entropy, void* grad_logits,
                                            int64_t rows, int64_t tokens_count, cufkb_stream_t stream);

/* One flat array of a gradient list: its elements and where the clipped ones go (may be the same). */
typedef struct cufkb_grad_array {
  const void* grad;
  void* out;
  int64_t count;
  int dtype;
} cufkb_grad_array;

/* norm = sqrt(sum of squares over all arrays) (double accumulation, stored as float32 or, norm_dtype =
 * CUFKB_FLOAT64, as float64); out = grad * min(1, max_norm / (norm + eps)), where max_norm = inf is a factor of 1
 * for any norm.  All four dtypes.  `arrays` is a host array, read before the call returns; the workspace is device
 * memory.  An array that is named again (equal grad, out, count and dtype) counts again in the norm and is scaled once; any other memory
 * that is written for one array and read or written for another is refused with CUFKB_ERROR_INVALID_VALUE. */
CUFKB_API int cufkb_clip_workspace_bytes(const cufkb_grad_array* arrays, int64_t count, size_t* bytes);
CUFKB_API int cufkb_clip_gradients(const cufkb_grad_array* arrays, int64_t count, double max_norm, double eps, void* norm, int norm_dtype,
                                   void* workspace, size_t workspace_bytes, cufkb_stream_t stream);

/* Static text for a status code of these entry points. */
CUFKB_API const char* cufkb_seq_status_string(int status);

/* cudaError_t value of the last CUFKB_ERROR_CUDA that an entry point of this header returned on the calling
 * thread (0 if none). */
CUFKB_API int cufkb_seq_last_cuda_error(void);

#ifdef __cplusplus
}
#endif

#endif /* CUFKB_SEQ_H_ */
