// C entry points of the selective scan's forward and step.
#include "seq_scan.cuh"

namespace cufkb_seq {
namespace {

template <typename T, int NP>
int launch(const ScanArgs<T>& a, bool pieces, cudaStream_t stream) {
  using S = ForwardShape<NP>;
  const int64_t blocks = a.items * a.blocks;
  if (blocks > INT32_MAX) return CUFKB_ERROR_SHAPE_LIMITS;
  if (blocks == 0) return CUFKB_SUCCESS;
  const unsigned grid = static_cast<unsigned>(blocks);
  if (pieces) {
    scan_forward_kernel<T, S::LPC, S::KN, S::KC, true><<<grid, kScanThreads, 0, stream>>>(a);
    if (int st = launch_status()) return st;
    return launch_dependent(scan_forward_kernel<T, S::LPC, S::KN, S::KC, false>, dim3(grid), kScanThreads, stream, a);
  }
  scan_forward_kernel<T, S::LPC, S::KN, S::KC, false><<<grid, kScanThreads, 0, stream>>>(a);
  return launch_status();
}

template <typename T>
struct Forward {
  static int run(const cufkb_scan_params& q, const ScanPlan& p, const ScanSpace& s, cudaStream_t stream) {
    const ScanArgs<T> a = scan_args<T>(q, p, s);
    switch (p.padded) {
      case 8:
        return launch<T, 8>(a, p.pieces, stream);
      case 16:
        return launch<T, 16>(a, p.pieces, stream);
      case 32:
        return launch<T, 32>(a, p.pieces, stream);
      default:
        return launch<T, 64>(a, p.pieces, stream);
    }
  }
};

template <typename T, int LPC>
int launch_step(const ScanArgs<T>& a, cudaStream_t stream) {
  const int64_t sets = ceil_div(a.chains.count, kStepChains);
  const dim3 grid(static_cast<unsigned>(ceil_div(static_cast<int64_t>(a.width) * LPC, kScanThreads)), static_cast<unsigned>(sets < 65535 ? sets : 65535));
  // four states at once
  const bool wide = a.states % 4 == 0 && aligned_to(a.A, 16) && aligned_to(a.final_state, 16) && aligned_to(a.B, 4 * sizeof(T)) &&
                    aligned_to(a.C, 4 * sizeof(T)) && a.B_stride % 4 == 0 && a.C_stride % 4 == 0 && a.B_group_stride % 4 == 0 && a.C_group_stride % 4 == 0;
  if (wide) {
    return launch_dependent(scan_step_kernel<T, LPC, true>, grid, kScanThreads, stream, a);
  }
  return launch_dependent(scan_step_kernel<T, LPC, false>, grid, kScanThreads, stream, a);
}

template <typename T>
struct Step {
  static int run(const cufkb_scan_params& q, const ScanPlan& p, cudaStream_t stream) {
    const ScanArgs<T> a = scan_args<T>(q, p, ScanSpace{});
    switch (p.padded) {
      case 8:
      case 16:
        return launch_step<T, 4>(a, stream);
      case 32:
        return launch_step<T, 8>(a, stream);
      default:
        return launch_step<T, 16>(a, stream);
    }
  }
};

}  // namespace
}  // namespace cufkb_seq

using namespace cufkb_seq;

extern "C" {

int cufkb_scan_checkpoint_bytes(const cufkb_scan_params* params, size_t* bytes) {
  if (params == nullptr || bytes == nullptr) return CUFKB_ERROR_NULL_POINTER;
  if (int st = scan_check(*params)) return st;
  if (params->width == 0) {
    *bytes = 0;
    return CUFKB_SUCCESS;
  }
  const ScanPlan p = scan_plan(*params, false);
  *bytes = static_cast<size_t>(params->rows / kChunk + params->chains + 1) * params->width * p.padded * sizeof(float);
  return CUFKB_SUCCESS;
}

int cufkb_scan_workspace_bytes(const cufkb_scan_params* params, int backward, size_t* bytes) {
  if (params == nullptr || bytes == nullptr) return CUFKB_ERROR_NULL_POINTER;
  if (int st = scan_check(*params)) return st;
  *bytes = params->width == 0 ? 0 : scan_space(*params, scan_plan(*params, backward != 0), backward != 0).total;
  return CUFKB_SUCCESS;
}

int cufkb_scan_forward(const cufkb_scan_params* params, cufkb_stream_t stream) {
  if (params == nullptr) return CUFKB_ERROR_NULL_POINTER;
  const cufkb_scan_params& q = *params;
  if (int st = scan_check(q)) return st;
  if (q.width == 0) return CUFKB_SUCCESS;
  if (int st = scan_check_inputs(q)) return st;
  if (q.rows > 0 && q.y == nullptr) return CUFKB_ERROR_NULL_POINTER;
  const ScanPlan p = scan_plan(q, false);
  const ScanSpace s = scan_space(q, p, false);
  if (s.total > 0 && (q.workspace == nullptr || q.workspace_bytes < s.total)) return CUFKB_ERROR_WORKSPACE;
  return for_activation<Forward>(q.dtype, q, p, s, reinterpret_cast<cudaStream_t>(stream));
}

int cufkb_scan_step(const cufkb_scan_params* params, cufkb_stream_t stream) {
  if (params == nullptr) return CUFKB_ERROR_NULL_POINTER;
  cufkb_scan_params q = *params;
  q.rows = q.chains;
  q.chain_points = nullptr;
  q.workspace = nullptr;
  if (int st = scan_check(q, CUFKB_MAX_STEP_STRIDE)) return st;
  if (q.width == 0 || q.chains == 0) return CUFKB_SUCCESS;
  if (int st = scan_check_inputs(q)) return st;
  if (q.y == nullptr || q.final_state == nullptr) return CUFKB_ERROR_NULL_POINTER;
  return for_activation<Step>(q.dtype, q, scan_plan(q, false), reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
