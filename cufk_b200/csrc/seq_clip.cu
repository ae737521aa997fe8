// C entry points of gradient clipping.
#include <algorithm>
#include <memory>
#include <new>

#include "clip_kernels.cuh"
#include "seq_api.cuh"

namespace cufkb_seq {
namespace {

constexpr int kSmall = 64, kLarge = 512;       // arrays of one launch
constexpr int64_t kClipBlocks = kSms * 8;      // of one launch: all resident

int check(const cufkb_grad_array* arrays, int64_t count) {
  if (count < 0 || count > (1 << 20)) return CUFKB_ERROR_SHAPE_LIMITS;
  if (count > 0 && arrays == nullptr) return CUFKB_ERROR_NULL_POINTER;
  for (int64_t i = 0; i < count; ++i) {
    const cufkb_grad_array& a = arrays[i];
    if (a.dtype < CUFKB_FLOAT32 || a.dtype > CUFKB_BFLOAT16) return CUFKB_ERROR_INVALID_DTYPE;
    // the chunks of a launch are counted in 32 bits
    if (a.count < 0 || a.count > int64_t{1} << 34) return CUFKB_ERROR_SHAPE_LIMITS;
    if (a.count > 0 && (a.grad == nullptr || a.out == nullptr)) return CUFKB_ERROR_NULL_POINTER;
    const size_t e = element_size(a.dtype);
    if (!aligned_to(a.grad, e) || !aligned_to(a.out, e)) return CUFKB_ERROR_MISALIGNED;
  }
  return CUFKB_SUCCESS;
}

uintptr_t address(const void* p) { return reinterpret_cast<uintptr_t>(p); }

// Blocks scale arrays in no order, so what one writes no other may read or write.  The common lists say so in one pass: results one behind
// the other, and all gradients that are not scaled in place apart from all results.
bool plainly_apart(const cufkb_grad_array* arrays, int64_t count) {
  uintptr_t end = 0, result_first = UINTPTR_MAX, grad_first = UINTPTR_MAX, grad_end = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (arrays[i].count == 0) continue;
    const uintptr_t grad = address(arrays[i].grad), out = address(arrays[i].out), bytes = arrays[i].count * element_size(arrays[i].dtype);
    if (out < end) return false;
    result_first = std::min(result_first, out);
    end = out + bytes;
    if (grad != out) {
      grad_first = std::min(grad_first, grad);
      grad_end = std::max(grad_end, grad + bytes);
    }
  }
  return grad_end <= result_first || grad_first >= end;
}

struct Span {
  uintptr_t first, end;
  int64_t array;
  bool written;
};

// The same for any list, by its spans of memory in order.  An array that is named again, with the same gradient and result, is no
// fault: it counts again in the norm and is scaled once.  `repeated` marks such arrays; it stays empty when there are none.
int check_shared(const cufkb_grad_array* arrays, int64_t count, std::unique_ptr<bool[]>& repeated) {
  if (plainly_apart(arrays, count)) return CUFKB_SUCCESS;
  const std::unique_ptr<Span[]> spans(new (std::nothrow) Span[2 * count]);
  if (spans == nullptr) return CUFKB_ERROR_SHAPE_LIMITS;
  int64_t n = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (arrays[i].count == 0) continue;
    const uintptr_t grad = address(arrays[i].grad), out = address(arrays[i].out), bytes = arrays[i].count * element_size(arrays[i].dtype);
    spans[n++] = {out, out + bytes, i, true};
    if (grad != out) spans[n++] = {grad, grad + bytes, i, false};
  }
  std::sort(spans.get(), spans.get() + n, [](const Span& a, const Span& b) {
    if (a.first != b.first) return a.first < b.first;
    if (a.written != b.written) return a.written;
    return a.array < b.array;
  });
  uintptr_t written_end = 0, read_end = 0;
  int64_t last = -1;  // the last array whose result was met
  for (int64_t k = 0; k < n; ++k) {
    const Span& s = spans[k];
    if (s.first < written_end) {
      const cufkb_grad_array &a = arrays[s.array], &b = arrays[last];
      if (!s.written || a.grad != b.grad || a.out != b.out || a.count != b.count || a.dtype != b.dtype) return CUFKB_ERROR_INVALID_VALUE;
      if (repeated == nullptr) {
        repeated.reset(new (std::nothrow) bool[count]());
        if (repeated == nullptr) return CUFKB_ERROR_SHAPE_LIMITS;
      }
      repeated[s.array] = true;
    } else if (s.written) {
      if (s.first < read_end) return CUFKB_ERROR_INVALID_VALUE;
      written_end = s.end;
      last = s.array;
    } else {
      read_end = std::max(read_end, s.end);
    }
  }
  return CUFKB_SUCCESS;
}

// skip: arrays to leave out, or nullptr
template <int MOST>
int64_t fill(ClipTable<MOST>& t, const cufkb_grad_array* arrays, int64_t count, const bool* skip) {
  int64_t chunks = 0;
  int n = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (arrays[i].count == 0 || (skip != nullptr && skip[i])) continue;
    t.grad[n] = arrays[i].grad;
    t.out[n] = arrays[i].out;
    t.count[n] = arrays[i].count;
    t.type[n] = static_cast<uint8_t>(arrays[i].dtype);
    t.first[n] = static_cast<int>(chunks);
    chunks += ceil_div(arrays[i].count, kClipChunk);
    ++n;
  }
  t.first[n] = static_cast<int>(chunks);
  t.arrays = n;
  return chunks;
}

unsigned grid_of(int64_t chunks) { return static_cast<unsigned>(chunks < 1 ? 1 : chunks < kClipBlocks ? chunks : kClipBlocks); }

template <int MOST>
int run(const cufkb_grad_array* arrays, int64_t count, const bool* repeated, double max_norm, double eps, void* norm, bool norm_double, double* partial,
        cudaStream_t stream) {
  ClipTable<MOST> table;  // of one launch at a time; 15 KB for the large one
  int partials = 0;
  for (int64_t at = 0; at == 0 || at < count; at += MOST) {
    const unsigned grid = grid_of(fill(table, arrays + at, count - at < MOST ? count - at : MOST, nullptr));
    clip_norm_kernel<MOST><<<grid, kClipThreads, 0, stream>>>(table, partial + partials);
    if (int st = launch_status()) return st;
    partials += static_cast<int>(grid);
  }
  const int64_t last = count > 0 ? (count - 1) / MOST * MOST : 0;
  for (int64_t at = last; at >= 0; at -= MOST) {
    if (last > 0 || repeated != nullptr) {
      fill(table, arrays + at, count - at < MOST ? count - at : MOST, repeated != nullptr ? repeated + at : nullptr);
    }
    clip_scale_kernel<MOST><<<grid_of(table.first[table.arrays]), kClipThreads, 0, stream>>>(table, partial, partials, max_norm, eps, at == 0 ? norm : nullptr, norm_double);
    if (int st = launch_status()) return st;
  }
  return CUFKB_SUCCESS;
}

}  // namespace
}  // namespace cufkb_seq

using namespace cufkb_seq;

extern "C" {

int cufkb_clip_workspace_bytes(const cufkb_grad_array* arrays, int64_t count, size_t* bytes) {
  if (bytes == nullptr) return CUFKB_ERROR_NULL_POINTER;
  if (int st = check(arrays, count)) return st;
  const int64_t launches = count <= kSmall ? 1 : ceil_div(count, kLarge);
  *bytes = static_cast<size_t>(launches * kClipBlocks) * sizeof(double);
  return CUFKB_SUCCESS;
}

int cufkb_clip_gradients(const cufkb_grad_array* arrays, int64_t count, double max_norm, double eps, void* norm, int norm_dtype, void* workspace,
                         size_t workspace_bytes, cufkb_stream_t stream) {
  size_t wanted = 0;
  if (int st = cufkb_clip_workspace_bytes(arrays, count, &wanted)) return st;
  if (norm_dtype != CUFKB_FLOAT32 && norm_dtype != CUFKB_FLOAT64) return CUFKB_ERROR_UNSUPPORTED_DTYPE;
  if (!(max_norm >= 0.0) || !(eps >= 0.0)) return CUFKB_ERROR_INVALID_VALUE;
  if (norm == nullptr) return CUFKB_ERROR_NULL_POINTER;
  if (workspace == nullptr || workspace_bytes < wanted) return CUFKB_ERROR_WORKSPACE;
  if (!aligned_to(workspace, 8) || !aligned_to(norm, element_size(norm_dtype))) return CUFKB_ERROR_MISALIGNED;
  std::unique_ptr<bool[]> repeated;
  if (int st = check_shared(arrays, count, repeated)) return st;
  const auto s = reinterpret_cast<cudaStream_t>(stream);
  double* partial = static_cast<double*>(workspace);
  if (count <= kSmall) return run<kSmall>(arrays, count, repeated.get(), max_norm, eps, norm, norm_dtype == CUFKB_FLOAT64, partial, s);
  return run<kLarge>(arrays, count, repeated.get(), max_norm, eps, norm, norm_dtype == CUFKB_FLOAT64, partial, s);
}

}  // extern "C"
