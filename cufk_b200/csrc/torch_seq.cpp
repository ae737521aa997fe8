// PyTorch boundary of the sequence operators (cufkb_seq.h): checks, autograd and outputs.
//
// As for the reconstruction path: outputs come from the caching allocator on the input's device, launches go to the current
// stream under a device guard, nothing synchronises with the host, and refusals are RuntimeErrors that name the argument.
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/autograd.h>
#include <torch/extension.h>

#include <optional>
#include <string>
#include <vector>

#include "cufkb_seq.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;
using OptTensor = std::optional<Tensor>;

int dtype_code(torch::ScalarType t) {
  switch (t) {
    case torch::kFloat32:
      return CUFKB_FLOAT32;
    case torch::kFloat64:
      return CUFKB_FLOAT64;
    case torch::kFloat16:
      return CUFKB_FLOAT16;
    case torch::kBFloat16:
      return CUFKB_BFLOAT16;
    default:
      return -1;
  }
}

void check_status(int status, const char* op) {
  if (status == CUFKB_SUCCESS) return;
  if (status == CUFKB_ERROR_CUDA) {
    TORCH_CHECK(false, op, ": CUDA error: ", cudaGetErrorString(static_cast<cudaError_t>(cufkb_seq_last_cuda_error())));
  }
  TORCH_CHECK(false, op, ": ", cufkb_seq_status_string(status));
}

cufkb_stream_t current_stream() { return reinterpret_cast<cufkb_stream_t>(at::cuda::getCurrentCUDAStream().stream()); }

Tensor get(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
const void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* out(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* floats(const Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; }

// The kernels write through pointers, which autograd does not see: a tensor that a call has written in place says so here, and a backward that
// saved it refuses.  Tensors of inference mode have no version.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void check_activation(const Tensor& x, const char* name) {
  TORCH_CHECK(x.is_cuda(), name, " must be CUDA");
  const auto t = x.scalar_type();
  TORCH_CHECK(t == torch::kFloat32 || t == torch::kFloat16 || t == torch::kBFloat16, name, " must be float32, float16, or bfloat16");
}

bool asks_gradient(const Tensor& t) { return t.defined() && t.requires_grad(); }

void refuse_gradients(std::initializer_list<Tensor> inputs, const char* op) {
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor& t : inputs) TORCH_CHECK(!asks_gradient(t), op, " takes no gradients");
}

void check_like(const Tensor& x, const Tensor& ref, const char* name, const char* ref_name) {
  TORCH_CHECK(x.is_cuda() && x.device() == ref.device(), name, " must be CUDA, on the device of ", ref_name);
  TORCH_CHECK(x.scalar_type() == ref.scalar_type(), name, " must have the dtype of ", ref_name);
}

// a float32 parameter or state of the given shape
Tensor check_float(const Tensor& x, at::IntArrayRef shape, const Tensor& ref, const char* name) {
  if (!x.defined()) return x;
  TORCH_CHECK(x.is_cuda() && x.device() == ref.device(), name, " must be CUDA, on the device of x");
  TORCH_CHECK(x.scalar_type() == torch::kFloat32, name, " must be float32");
  TORCH_CHECK(x.sizes() == shape, name, " must have shape ", shape);
  return x.contiguous();
}

// The widest row strides that a scan and its step walk (cufkb_scan_params); rows further apart are copied.
constexpr int64_t kScanStride = CUFKB_MAX_SCAN_STRIDE, kStepStride = CUFKB_MAX_STEP_STRIDE;

// Rows of a (..., width) activation as (rows, width) with one row stride of at most `most`; a copy only where there is none.
struct Rows {
  Tensor kept;
  const void* ptr = nullptr;
  int64_t stride = 0;
};

Rows rows_of(const Tensor& x, int64_t most = INT64_MAX) {
  Rows r;
  const int64_t d = x.dim(), width = x.size(d - 1), rows = d == 3 ? x.size(0) * x.size(1) : x.size(0);
  bool flat = x.numel() == 0 || width <= 1 || x.stride(d - 1) == 1;
  if (flat && d == 3 && x.size(0) > 1 && x.size(1) > 1) flat = x.stride(0) == x.size(1) * x.stride(1);
  auto stride_of = [&](const Tensor& t) {
    if (rows <= 1 || width == 0) return width;  // never used
    return (d == 3 && t.size(1) <= 1) ? t.stride(0) : t.stride(d - 2);
  };
  r.kept = flat && stride_of(x) <= most ? x : x.contiguous();
  r.ptr = r.kept.data_ptr();
  r.stride = stride_of(r.kept);
  return r;
}

// How the rows of an activation belong to chains: packed (rows, width) with offsets, (rows, width) as one chain, or (chains,
// length, width).
struct Layout {
  int64_t rows = 0, chains = 0, width = 0;
  const int64_t* points = nullptr;
};

Layout layout_of(const Tensor& x, const Tensor& points) {
  TORCH_CHECK(x.dim() == 2 || x.dim() == 3, "x must have shape (rows, width) or (chains, length, width)");
  Layout l;
  l.width = x.size(-1);
  l.rows = x.dim() == 3 ? x.size(0) * x.size(1) : x.size(0);
  l.chains = x.dim() == 3 ? x.size(0) : 1;
  if (points.defined()) {
    TORCH_CHECK(x.dim() == 2, "chain_points needs packed rows: x must have shape (rows, width)");
    TORCH_CHECK(points.is_cuda() && points.device() == x.device(), "chain_points must be CUDA, on the device of x");
    TORCH_CHECK(points.scalar_type() == torch::kInt64 && points.dim() == 1 && points.is_contiguous() && points.size(0) >= 1,
                "chain_points must be a contiguous 1-D int64 tensor of chains+1 offsets");
    l.chains = points.size(0) - 1;
    l.points = points.data_ptr<int64_t>();
  }
  return l;
}

// An uninitialised CUDA tensor from the caching allocator, past the dispatcher: a call allocates up to ten of them.
Tensor fresh(at::IntArrayRef shape, torch::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(shape, type, like.device(), std::nullopt);
}
Tensor fresh(const Tensor& like) { return fresh(like.sizes(), like.scalar_type(), like); }

Tensor workspace(size_t bytes, const Tensor& like) {
  return bytes == 0 ? Tensor() : fresh({static_cast<int64_t>(bytes)}, torch::kUInt8, like);
}

// Gradients that were asked for with a graph of their own (create_graph) come from kernels, which leave none.  They pass through here, so that
// differentiating them again is an error instead of a zero.
class OnceAutograd : public torch::autograd::Function<OnceAutograd> {
 public:
  // `through`: the gradients, then what they depend on
  static tensor_list forward(AutogradContext* ctx, at::TensorList through, int64_t gradients, std::string op) {
    ctx->saved_data["op"] = op;
    tensor_list out;
    for (int64_t i = 0; i < gradients; ++i) out.push_back(through[i].tensor_data());
    return out;
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list) {
    TORCH_CHECK(false, ctx->saved_data["op"].toStringRef(), " can be differentiated only once");
  }
};

tensor_list differentiated_once(tensor_list grads, const tensor_list& outputs, const tensor_list& inputs, const char* op) {
  if (!at::GradMode::is_enabled()) return grads;
  tensor_list through;
  for (const Tensor& t : grads) {
    if (t.defined()) through.push_back(t);
  }
  const int64_t count = static_cast<int64_t>(through.size());
  for (const tensor_list* list : {&outputs, &inputs}) {
    for (const Tensor& t : *list) {
      if (t.defined()) through.push_back(t);
    }
  }
  const tensor_list marked = OnceAutograd::apply(at::TensorList(through), count, std::string(op));
  size_t next = 0;
  for (Tensor& t : grads) {
    if (t.defined()) t = marked[next++];
  }
  return grads;
}

// ---------------------------------------------------------------------------------------------
// short causal convolution
// ---------------------------------------------------------------------------------------------
struct ConvCall {
  cufkb_conv_params p{};
  Rows x;
  Tensor weight, bias, initial;
};

ConvCall conv_call(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& points, const Tensor& initial, bool silu) {
  check_activation(x, "x");
  const Layout l = layout_of(x, points);
  ConvCall c;
  TORCH_CHECK(weight.defined() && weight.dim() == 2, "weight must have shape (width, taps)");
  const int64_t taps = weight.size(1);
  TORCH_CHECK(taps >= CUFKB_MIN_TAPS && taps <= CUFKB_MAX_TAPS, "weight must have ", CUFKB_MIN_TAPS, " to ", CUFKB_MAX_TAPS, " taps");
  c.weight = check_float(weight, {l.width, taps}, x, "weight");
  c.bias = check_float(bias, {l.width}, x, "bias");
  if (initial.defined()) {
    check_like(initial, x, "initial_state", "x");
    TORCH_CHECK(initial.sizes() == at::IntArrayRef({l.chains, taps - 1, l.width}), "initial_state must have shape (chains, taps - 1, width)");
    c.initial = initial.contiguous();
  }
  c.x = rows_of(x);
  c.p.dtype = dtype_code(x.scalar_type());
  c.p.taps = static_cast<int>(taps);
  c.p.silu = silu;
  c.p.rows = l.rows;
  c.p.chains = l.chains;
  c.p.width = l.width;
  c.p.chain_points = l.points;
  c.p.x = c.x.ptr;
  c.p.x_stride = c.x.stride;
  c.p.weight = floats(c.weight);
  c.p.bias = floats(c.bias);
  c.p.initial_state = data(c.initial);
  return c;
}

class ConvAutograd : public torch::autograd::Function<ConvAutograd> {
 public:
  static tensor_list forward(AutogradContext* ctx, Tensor x, Tensor weight, OptTensor bias, OptTensor points, OptTensor initial, bool silu, bool keep) {
    ConvCall c = conv_call(x, weight, get(bias), get(points), get(initial), silu);
    const c10::cuda::CUDAGuard guard(x.device());
    Tensor y = fresh(x);
    Tensor state = keep ? fresh({c.p.chains, c.p.taps - 1, c.p.width}, x.scalar_type(), x) : Tensor();
    c.p.y = y.data_ptr();
    c.p.final_state = out(state);
    check_status(cufkb_conv_forward(&c.p, current_stream()), "short_conv");
    ctx->save_for_backward({x, weight, get(bias), get(points), get(initial)});
    ctx->saved_data["silu"] = silu;
    const Tensor b = get(bias), i = get(initial);
    ctx->saved_data["needs_x"] = x.requires_grad();
    ctx->saved_data["needs_taps"] = weight.requires_grad() || (b.defined() && b.requires_grad());
    ctx->saved_data["needs_initial"] = i.defined() && i.requires_grad();
    return keep ? tensor_list{y, state} : tensor_list{y};
  }

  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &initial = saved[4];
    ConvCall c = conv_call(x, weight, bias, saved[3], initial, ctx->saved_data["silu"].toBool());
    const c10::cuda::CUDAGuard guard(x.device());
    const bool want_x = ctx->saved_data["needs_x"].toBool(), want_w = ctx->saved_data["needs_taps"].toBool();
    const Tensor gy = grads[0].defined() ? grads[0] : torch::zeros(x.sizes(), x.options());
    check_like(gy, x, "grad_y", "x");
    const Rows g = rows_of(gy);
    c.p.grad_y = g.ptr;
    c.p.grad_y_stride = g.stride;
    Tensor gs;
    if (grads.size() > 1 && grads[1].defined()) {
      check_like(grads[1], x, "grad_state", "x");
      gs = grads[1].contiguous();
      c.p.grad_final_state = gs.data_ptr();
    }
    Tensor gx, gw, gb, gi, ws;
    if (want_x) gx = fresh(x);
    if (want_w) {
      gw = fresh(c.weight);
      gb = fresh({c.p.width}, torch::kFloat32, x);
      size_t bytes = 0;
      check_status(cufkb_conv_backward_workspace_bytes(&c.p, &bytes), "short_conv backward");
      ws = workspace(bytes, x);
      c.p.workspace = out(ws);
      c.p.workspace_bytes = bytes;
    }
    if (ctx->saved_data["needs_initial"].toBool()) gi = fresh(initial);
    c.p.grad_x = out(gx);
    c.p.grad_weight = floats(gw);
    c.p.grad_bias = floats(gb);
    c.p.grad_initial_state = out(gi);
    check_status(cufkb_conv_backward(&c.p, current_stream()), "short_conv backward");
    return differentiated_once({gx, gw, bias.defined() ? gb : Tensor(), Tensor(), gi, Tensor(), Tensor()}, grads, saved, "short_conv");
  }
};

tensor_list short_conv(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& points, const OptTensor& initial, bool silu, bool keep) {
  return ConvAutograd::apply(x, weight, bias, points, initial, silu, keep);
}

Tensor short_conv_step(const Tensor& x, const Tensor& state, const Tensor& weight, const OptTensor& bias, bool silu) {
  check_activation(x, "x");
  TORCH_CHECK(x.dim() == 2, "x must have shape (chains, width)");
  check_like(state, x, "state", "x");
  TORCH_CHECK(weight.dim() == 2, "weight must have shape (width, taps)");
  const int64_t taps = weight.size(1);
  TORCH_CHECK(taps >= CUFKB_MIN_TAPS && taps <= CUFKB_MAX_TAPS, "weight must have ", CUFKB_MIN_TAPS, " to ", CUFKB_MAX_TAPS, " taps");
  TORCH_CHECK(state.sizes() == at::IntArrayRef({x.size(0), taps - 1, x.size(1)}) && state.is_contiguous(),
              "state must be contiguous, of shape (chains, taps - 1, width)");
  refuse_gradients({x, state, weight, get(bias)}, "short_conv_step");
  const Tensor w = check_float(weight, {x.size(1), taps}, x, "weight"), b = check_float(get(bias), {x.size(1)}, x, "bias");
  const c10::cuda::CUDAGuard guard(x.device());
  const Rows r = rows_of(x);
  Tensor y = fresh(x);
  check_status(cufkb_conv_step(dtype_code(x.scalar_type()), r.ptr, r.stride, state.data_ptr(), floats(w), floats(b), y.data_ptr(), x.size(0), x.size(1),
                               static_cast<int>(taps), silu, current_stream()),
               "short_conv_step");
  written(state);
  return y;
}

// ---------------------------------------------------------------------------------------------
// selective scan
// ---------------------------------------------------------------------------------------------
struct ScanCall {
  cufkb_scan_params p{};
  Rows x, delta, z;
  Tensor A, B, C, D, bias, initial;
};

// (rows, states), (rows, groups, states), or the same with (chains, length) in the place of rows: pointer and strides
Tensor bc_rows(const Tensor& t, const Tensor& x, const Layout& l, int64_t states, int64_t most, int64_t& groups, int64_t& stride, int64_t& group_stride,
               const char* name) {
  check_like(t, x, name, "x");
  const int64_t lead = x.dim() - 1;
  TORCH_CHECK(t.dim() == lead + 1 || t.dim() == lead + 2, name, " must have shape (rows, states) or (rows, groups, states), rows as in x");
  for (int64_t i = 0; i < lead; ++i) TORCH_CHECK(t.size(i) == x.size(i), name, " must have the rows of x");
  TORCH_CHECK(t.size(-1) == states, name, " must have as many states as A");
  groups = t.dim() == lead + 2 ? t.size(lead) : 1;
  TORCH_CHECK(groups >= 1 && l.width % groups == 0, name, ": the groups must divide the width");
  bool flat = states <= 1 || t.stride(-1) == 1;
  if (flat && lead == 2 && t.size(0) > 1 && t.size(1) > 1) flat = t.stride(0) == t.size(1) * t.stride(1);
  auto stride_of = [&](const Tensor& v) {
    if (l.rows <= 1) return states * groups;  // never used
    return (lead == 2 && v.size(1) <= 1) ? v.stride(0) : v.stride(lead - 1);
  };
  const Tensor kept = flat && stride_of(t) <= most ? t : t.contiguous();
  stride = stride_of(kept);
  group_stride = kept.dim() == lead + 2 ? kept.stride(lead) : 0;
  return kept;
}

ScanCall scan_call(const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C, const Tensor& D, const Tensor& z,
                   const Tensor& bias, const Tensor& points, const Tensor& initial, bool softplus, const Layout& l, int64_t most = kScanStride) {
  ScanCall c;
  check_like(delta, x, "delta", "x");
  TORCH_CHECK(delta.sizes() == x.sizes(), "delta must have the shape of x");
  if (z.defined()) {
    check_like(z, x, "z", "x");
    TORCH_CHECK(z.sizes() == x.sizes(), "z must have the shape of x");
  }
  TORCH_CHECK(A.dim() == 2, "A must have shape (width, states)");
  const int64_t states = A.size(1);
  TORCH_CHECK(states >= 1 && states <= CUFKB_MAX_STATES, "A must have 1 to ", CUFKB_MAX_STATES, " states");
  c.A = check_float(A, {l.width, states}, x, "A");
  c.D = check_float(D, {l.width}, x, "D");
  c.bias = check_float(bias, {l.width}, x, "delta_bias");
  int64_t groups = 1, groups_c = 1;
  c.B = bc_rows(B, x, l, states, most, groups, c.p.B_stride, c.p.B_group_stride, "B");
  c.C = bc_rows(C, x, l, states, most, groups_c, c.p.C_stride, c.p.C_group_stride, "C");
  TORCH_CHECK(groups == groups_c, "B and C must have the same groups");
  c.initial = check_float(initial, {l.chains, l.width, states}, x, "initial_state");
  c.x = rows_of(x, most);
  c.delta = rows_of(delta, most);
  if (z.defined()) c.z = rows_of(z, most);
  c.p.dtype = dtype_code(x.scalar_type());
  c.p.softplus = softplus;
  c.p.rows = l.rows;
  c.p.chains = l.chains;
  c.p.width = l.width;
  c.p.groups = groups;
  c.p.states = states;
  c.p.chain_points = l.points;
  c.p.x = c.x.ptr;
  c.p.x_stride = c.x.stride;
  c.p.delta = c.delta.ptr;
  c.p.delta_stride = c.delta.stride;
  c.p.z = c.z.ptr;
  c.p.z_stride = c.z.stride;
  c.p.A = floats(c.A);
  c.p.B = c.B.data_ptr();
  c.p.C = c.C.data_ptr();
  c.p.D = floats(c.D);
  c.p.delta_bias = floats(c.bias);
  c.p.initial_state = floats(c.initial);
  return c;
}

class ScanAutograd : public torch::autograd::Function<ScanAutograd> {
 public:
  static tensor_list forward(AutogradContext* ctx, Tensor x, Tensor delta, Tensor A, Tensor B, Tensor C, OptTensor D, OptTensor z, OptTensor bias,
                             OptTensor points, OptTensor initial, bool softplus, bool keep, bool train) {
    check_activation(x, "x");
    const Layout l = layout_of(x, get(points));
    ScanCall c = scan_call(x, delta, A, B, C, get(D), get(z), get(bias), get(points), get(initial), softplus, l);
    const c10::cuda::CUDAGuard guard(x.device());
    Tensor y = fresh(x);
    Tensor state = keep ? fresh({l.chains, l.width, c.p.states}, torch::kFloat32, x) : Tensor();
    size_t bytes = 0;
    check_status(cufkb_scan_workspace_bytes(&c.p, 0, &bytes), "selective_scan");
    Tensor ws = workspace(bytes, x), checkpoints;
    c.p.workspace = out(ws);
    c.p.workspace_bytes = bytes;
    if (train) {
      check_status(cufkb_scan_checkpoint_bytes(&c.p, &bytes), "selective_scan");
      checkpoints = workspace(bytes, x);
      c.p.checkpoints = floats(checkpoints);
    }
    c.p.y = y.data_ptr();
    c.p.final_state = floats(state);
    check_status(cufkb_scan_forward(&c.p, current_stream()), "selective_scan");
    if (train) {
      ctx->save_for_backward({x, delta, A, B, C, get(D), get(z), get(bias), get(points), get(initial), checkpoints});
      ctx->saved_data["softplus"] = softplus;
    }
    return keep ? tensor_list{y, state} : tensor_list{y};
  }

  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &D = saved[5], &z = saved[6], &bias = saved[7], &initial = saved[9], &checkpoints = saved[10];
    const Layout l = layout_of(x, saved[8]);
    ScanCall c = scan_call(x, saved[1], saved[2], saved[3], saved[4], D, z, bias, saved[8], initial, ctx->saved_data["softplus"].toBool(), l);
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor gy = grads[0].defined() ? grads[0] : torch::zeros(x.sizes(), x.options());
    check_like(gy, x, "grad_y", "x");
    const Rows g = rows_of(gy, kScanStride);
    c.p.grad_y = g.ptr;
    c.p.grad_y_stride = g.stride;
    Tensor gs;
    if (grads.size() > 1 && grads[1].defined()) {
      gs = check_float(grads[1], {l.chains, l.width, c.p.states}, x, "grad_state");
      c.p.grad_final_state = floats(gs);
    }
    c.p.checkpoints = floats(checkpoints);
    Tensor gx = fresh(x), gd = fresh(x);
    Tensor gB = fresh(saved[3]), gC = fresh(saved[4]);
    Tensor gA = fresh(c.A), gz, gD, gbias, gi;
    if (z.defined()) gz = fresh(x);
    if (D.defined()) gD = fresh({l.width}, torch::kFloat32, x);
    if (bias.defined()) gbias = fresh({l.width}, torch::kFloat32, x);
    if (initial.defined()) gi = fresh(c.initial);
    size_t bytes = 0;
    check_status(cufkb_scan_workspace_bytes(&c.p, 1, &bytes), "selective_scan backward");
    Tensor ws = workspace(bytes, x);
    c.p.workspace = out(ws);
    c.p.workspace_bytes = bytes;
    c.p.grad_x = gx.data_ptr();
    c.p.grad_delta = gd.data_ptr();
    c.p.grad_z = out(gz);
    c.p.grad_A = floats(gA);
    c.p.grad_B = gB.data_ptr();
    c.p.grad_C = gC.data_ptr();
    c.p.grad_D = floats(gD);
    c.p.grad_delta_bias = floats(gbias);
    c.p.grad_initial_state = floats(gi);
    check_status(cufkb_scan_backward(&c.p, current_stream()), "selective_scan backward");
    return differentiated_once({gx, gd, gA, gB, gC, gD, gz, gbias, Tensor(), gi, Tensor(), Tensor(), Tensor()}, grads, saved, "selective_scan");
  }
};

tensor_list selective_scan(const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C, const OptTensor& D, const OptTensor& z,
                           const OptTensor& bias, const OptTensor& points, const OptTensor& initial, bool softplus, bool keep) {
  const bool train = at::GradMode::is_enabled() && (x.requires_grad() || delta.requires_grad() || A.requires_grad() || B.requires_grad() ||
                                                    C.requires_grad() || asks_gradient(get(D)) || asks_gradient(get(z)) ||
                                                    asks_gradient(get(bias)) || asks_gradient(get(initial)));
  return ScanAutograd::apply(x, delta, A, B, C, D, z, bias, points, initial, softplus, keep, train);
}

Tensor selective_scan_step(const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C, const Tensor& state, const OptTensor& D,
                           const OptTensor& z, const OptTensor& bias, bool softplus) {
  check_activation(x, "x");
  TORCH_CHECK(x.dim() == 2, "x must have shape (chains, width)");
  refuse_gradients({x, delta, A, B, C, state, get(D), get(z), get(bias)}, "selective_scan_step");
  Layout l;
  l.rows = l.chains = x.size(0);
  l.width = x.size(1);
  ScanCall c = scan_call(x, delta, A, B, C, get(D), get(z), get(bias), Tensor(), Tensor(), softplus, l, kStepStride);
  TORCH_CHECK(state.is_cuda() && state.device() == x.device() && state.scalar_type() == torch::kFloat32 && state.is_contiguous() &&
                  state.sizes() == at::IntArrayRef({l.chains, l.width, c.p.states}),
              "state must be contiguous float32 of shape (chains, width, states), on the device of x");
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor y = fresh(x);
  c.p.y = y.data_ptr();
  c.p.final_state = floats(state);
  check_status(cufkb_scan_step(&c.p, current_stream()), "selective_scan_step");
  written(state);
  return y;
}

// ---------------------------------------------------------------------------------------------
// token log probabilities
// ---------------------------------------------------------------------------------------------
Rows logit_rows(const Tensor& logits, int64_t& rows) {
  TORCH_CHECK(logits.dim() >= 1 && logits.size(-1) >= 1, "logits must have shape (..., tokens) with at least one token");
  const int64_t n = logits.size(-1);
  rows = 1;
  for (int64_t i = 0; i + 1 < logits.dim(); ++i) rows *= logits.size(i);
  Rows r;
  if (logits.dim() == 2 && (n == 1 || logits.stride(1) == 1) && logits.stride(0) >= 0) {
    r.kept = logits;
    r.stride = logits.stride(0);
  } else {
    r.kept = logits.contiguous();
    r.stride = n;
  }
  r.ptr = r.kept.data_ptr();
  return r;
}

class LogprobsAutograd : public torch::autograd::Function<LogprobsAutograd> {
 public:
  static tensor_list forward(AutogradContext* ctx, Tensor logits, Tensor tokens, int64_t top) {
    check_activation(logits, "logits");
    int64_t rows = 0;
    const Rows l = logit_rows(logits, rows);
    const auto lead = logits.sizes().slice(0, logits.dim() - 1);
    TORCH_CHECK(tokens.is_cuda() && tokens.device() == logits.device() && tokens.scalar_type() == torch::kInt64, "tokens must be CUDA int64, on the device of logits");
    TORCH_CHECK(tokens.sizes() == lead, "tokens must have the shape of logits without its last dimension");
    const int64_t n = logits.size(-1);
    TORCH_CHECK(top >= 0 && top <= CUFKB_MAX_TOP && top <= n, "top must be 0 to ", CUFKB_MAX_TOP, ", and at most the number of tokens");
    const c10::cuda::CUDAGuard guard(logits.device());
    const Tensor t = tokens.contiguous();
    Tensor logp = fresh(lead, torch::kFloat32, logits), entropy = fresh(lead, torch::kFloat32, logits), log_sum = fresh({rows, 2}, torch::kFloat32, logits);
    std::vector<int64_t> shape = lead.vec();
    shape.push_back(top);
    Tensor top_logp = fresh(shape, torch::kFloat32, logits), top_tokens = fresh(shape, torch::kInt64, logits);
    check_status(cufkb_token_logprobs(dtype_code(logits.scalar_type()), l.ptr, l.stride, t.data_ptr<int64_t>(), floats(logp), floats(entropy), floats(log_sum),
                                      floats(top_logp), top_tokens.data_ptr<int64_t>(), rows, n, static_cast<int>(top), current_stream()),
                 "token_logprobs");
    ctx->mark_non_differentiable({top_logp, top_tokens});
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, t, entropy, log_sum});
    return {logp, entropy, top_logp, top_tokens};
  }

  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    if (!grads[0].defined() && !grads[1].defined()) return {Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const Tensor& logits = saved[0];
    int64_t rows = 0;
    const Rows l = logit_rows(logits, rows);
    const c10::cuda::CUDAGuard guard(logits.device());
    const Tensor gl = grads[0].defined() ? grads[0].contiguous() : Tensor(), gh = grads[1].defined() ? grads[1].contiguous() : Tensor();
    Tensor g = fresh(logits);
    check_status(cufkb_token_logprobs_backward(dtype_code(logits.scalar_type()), l.ptr, l.stride, saved[1].data_ptr<int64_t>(), floats(saved[2]), floats(saved[3]),
                                               floats(gl), floats(gh), g.data_ptr(), rows, logits.size(-1), current_stream()),
                 "token_logprobs backward");
    return differentiated_once({g, Tensor(), Tensor()}, grads, saved, "token_logprobs");
  }
};

tensor_list token_logprobs(const Tensor& logits, const Tensor& tokens, int64_t top) { return LogprobsAutograd::apply(logits, tokens, top); }

// ---------------------------------------------------------------------------------------------
// gradient clipping
// ---------------------------------------------------------------------------------------------
Tensor clip_gradients(const std::vector<Tensor>& grads, double max_norm, double eps, const std::vector<Tensor>& outs) {
  TORCH_CHECK(!grads.empty(), "clip_gradients needs at least one gradient");
  TORCH_CHECK(grads.size() == outs.size(), "out must hold one tensor per gradient");
  TORCH_CHECK(max_norm >= 0.0, "max_norm must not be negative");
  TORCH_CHECK(eps >= 0.0, "eps must not be negative");
  const Tensor& first = grads[0];
  std::vector<cufkb_grad_array> arrays;
  std::vector<Tensor> kept;
  std::vector<std::pair<Tensor, Tensor>> back;  // results that go to a tensor with other strides
  arrays.reserve(grads.size());
  bool wide = false;
  for (size_t i = 0; i < grads.size(); ++i) {
    const Tensor &g = grads[i], &o = outs[i];
    TORCH_CHECK(g.is_cuda() && o.is_cuda() && g.device() == first.device() && o.device() == first.device(), "gradients and outputs must be CUDA, on one device");
    const int code = dtype_code(g.scalar_type());
    TORCH_CHECK(code >= 0, "gradients must be float32, float64, float16, or bfloat16");
    TORCH_CHECK(o.sizes() == g.sizes() && o.scalar_type() == g.scalar_type(), "each output must have the shape and dtype of its gradient");
    TORCH_CHECK(!(at::GradMode::is_enabled() && (g.requires_grad() || o.requires_grad())), "clip_gradients takes no gradients of gradients");
    wide = wide || code == CUFKB_FLOAT64;
    Tensor from = g, to = o;
    // elements in memory order: any dense layout will do as long as both have the same
    const bool same = g.is_contiguous() ? o.is_contiguous() : (g.is_non_overlapping_and_dense() && g.strides() == o.strides());
    if (!same) {
      TORCH_CHECK(at::has_internal_overlap(o) != at::MemOverlap::Yes, "an expanded gradient cannot be clipped in place: give it an output of its own");
      from = g.contiguous();
      to = o.is_contiguous() ? o : fresh(g);
      if (!o.is_contiguous()) back.emplace_back(o, to);
      kept.push_back(from);
    }
    arrays.push_back({from.data_ptr(), to.data_ptr(), g.numel(), code});
  }
  const c10::cuda::CUDAGuard guard(first.device());
  const int64_t count = static_cast<int64_t>(arrays.size());
  size_t bytes = 0;
  check_status(cufkb_clip_workspace_bytes(arrays.data(), count, &bytes), "clip_gradients");
  Tensor ws = workspace(bytes, first);
  Tensor norm = fresh({}, wide ? torch::kFloat64 : torch::kFloat32, first);
  check_status(cufkb_clip_gradients(arrays.data(), count, max_norm, eps, norm.data_ptr(), wide ? CUFKB_FLOAT64 : CUFKB_FLOAT32, ws.data_ptr(), bytes, current_stream()),
               "clip_gradients");
  for (const Tensor& o : outs) written(o);
  for (auto& b : back) b.first.copy_(b.second);
  return norm;
}

}  // namespace

void register_seq(pybind11::module_& m) {
  m.def("short_conv", &short_conv);
  m.def("short_conv_step", &short_conv_step);
  m.def("selective_scan", &selective_scan);
  m.def("selective_scan_step", &selective_scan_step);
  m.def("token_logprobs", &token_logprobs);
  m.def("clip_gradients", &clip_gradients);
}
