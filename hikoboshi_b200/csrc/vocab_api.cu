// C entry points of the operators on vocabulary rows: argument checks, the
// device guard and the launch.  No workspace, no state, no synchronisation.
#include <atomic>
#include <cmath>

#include "hkb_mpnn.h"
#include "vocab.hpp"

namespace hkb {
namespace {

hkb_status invalid(const char* why) { return {HKB_INVALID_ARGUMENT, why}; }

// Whether a device can run this build; the answer is asked for once a device.
hkb_status usable(int device) {
  constexpr int kKnown = 64;
  static std::atomic<int> known[kKnown];  // 0: not asked yet, 1: it can
  if (device >= 0 && device < kKnown && known[device].load(std::memory_order_relaxed) == 1)
    return {HKB_OK, ""};
  int count = 0;
  if (cudaGetDeviceCount(&count) != cudaSuccess || count == 0) {
    cudaGetLastError();
    return {HKB_UNAVAILABLE, "no CUDA device is available"};
  }
  if (device < 0 || device >= count) return invalid("device ordinal out of range");
  int major = 0;
  if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device) != cudaSuccess) {
    cudaGetLastError();
    return {HKB_UNAVAILABLE, "the CUDA device cannot be used"};
  }
  if (major != 10) return {HKB_UNAVAILABLE, "this build targets sm_100a (B200) only"};
  if (device < kKnown) known[device].store(1, std::memory_order_relaxed);
  return {HKB_OK, ""};
}

// Makes `device` current for the call and puts the caller's device back.
class DeviceGuard {
 public:
  explicit DeviceGuard(int device) : status_(usable(device)) {
    if (status_.code != HKB_OK) return;
    if (cudaGetDevice(&previous_) != cudaSuccess ||
        (previous_ != device && cudaSetDevice(device) != cudaSuccess)) {
      cudaGetLastError();
      status_ = {HKB_UNAVAILABLE, "the CUDA device cannot be used"};
      return;
    }
    restore_ = previous_ != device;
  }
  ~DeviceGuard() {
    if (restore_) cudaSetDevice(previous_);
  }
  DeviceGuard(const DeviceGuard&) = delete;
  DeviceGuard& operator=(const DeviceGuard&) = delete;
  const hkb_status& status() const { return status_; }

 private:
  hkb_status status_;
  int previous_ = 0;
  bool restore_ = false;
};

hkb_status launched(cudaError_t e) {
  if (e == cudaSuccess) return {HKB_OK, ""};
  cudaGetLastError();
  return {HKB_INTERNAL_ERROR, cudaGetErrorString(e)};
}

constexpr double kLog2e = 1.4426950408889634074;

bool real_dtype(int d) { return d == HKB_F32 || d == HKB_F16 || d == HKB_BF16; }
uintptr_t elem_bytes(int d) { return d == HKB_F32 ? 4 : 2; }

hkb_status check_rows(const hkb_vocab_rows* v) {
  if (v == nullptr) return invalid("vocabulary rows are null");
  if (v->rows < 0 || v->rows > HKB_VOCAB_ROWS_MAX)
    return invalid("the number of rows must be 0 to HKB_VOCAB_ROWS_MAX");
  if (v->vocab < 1 || v->vocab > HKB_VOCAB_MAX)
    return invalid("vocab must be 1 to HKB_VOCAB_MAX");
  if (!real_dtype(v->dtype)) return invalid("logits must be F32, F16 or BF16");
  if (v->row_stride < 0) return invalid("the row stride must not be negative");
  if (v->rows > 0 && v->logits == nullptr) return invalid("logits pointer is null");
  if (reinterpret_cast<uintptr_t>(v->logits) % elem_bytes(v->dtype) != 0)
    return invalid("logits pointer is not aligned to its type");
  return {HKB_OK, ""};
}

VocabRows internal_rows(const hkb_vocab_rows& v) {
  return {v.rows, v.vocab, v.dtype, v.logits, v.row_stride};
}

// Whether `n` rows of `width` elements, `stride` elements apart, share bytes with
// the memory from `lo` to `hi`.
bool meets(const void* p, int64_t n, int64_t stride, int64_t width, uintptr_t bytes, uintptr_t lo,
           uintptr_t hi) {
  const uintptr_t first = reinterpret_cast<uintptr_t>(p);
  const uintptr_t end = first + (uintptr_t)((n - 1) * stride + width) * bytes;
  return p != nullptr && first < hi && lo < end;
}

hkb_status check_distill(const hkb_vocab_rows* rows, const hkb_distill_teacher* t,
                         const hkb_distill_out* out) {
  const hkb_status st = check_rows(rows);
  if (st.code != HKB_OK) return st;
  if (t == nullptr || out == nullptr) return invalid("teacher and output must be non-null");
  if (t->k < 1 || t->k > HKB_LISTING_MAX)
    return invalid("a row's listing must have 1 to HKB_LISTING_MAX entries");
  if (!real_dtype(t->dtype)) return invalid("teacher values must be F32, F16 or BF16");
  if (!(t->temperature >= HKB_TEMPERATURE_MIN &&
        t->temperature <= HKB_DISTILL_TEMPERATURE_MAX))
    return invalid("temperature must be 1e-30 to 1e4");
  if (out->row_weight_stride < 0) return invalid("the row weight stride must not be negative");
  if (out->grad != nullptr) {
    if (out->grad_row_stride < rows->vocab)
      return invalid("the gradient's rows must not overlap");
    const uintptr_t b = elem_bytes(rows->dtype);
    const uintptr_t x0 = reinterpret_cast<uintptr_t>(rows->logits);
    const uintptr_t g0 = reinterpret_cast<uintptr_t>(out->grad);
    if (g0 % b != 0) return invalid("gradient pointer is not aligned to its type");
    if (rows->rows > 0) {
      const uintptr_t n = (uintptr_t)rows->rows - 1;
      const uintptr_t x1 = x0 + (n * (uintptr_t)rows->row_stride + rows->vocab) * b;
      const uintptr_t g1 = g0 + (n * (uintptr_t)out->grad_row_stride + rows->vocab) * b;
      const bool same = x0 == g0 && (n == 0 || rows->row_stride == out->grad_row_stride);
      if (!same && x0 < g1 && g0 < x1)
        return invalid("grad must be the logits' own buffer or lie apart from it");
    }
  }
  return {HKB_OK, ""};
}

// The gradient is written while the rest is read, so they must not meet.
hkb_status check_apart(const hkb_vocab_rows& rows, const hkb_distill_teacher& t,
                       const hkb_distill_out& out) {
  if (out.grad == nullptr) return {HKB_OK, ""};
  const int64_t n = rows.rows;
  const uintptr_t g0 = reinterpret_cast<uintptr_t>(out.grad);
  const uintptr_t g1 =
      g0 + (uintptr_t)((n - 1) * out.grad_row_stride + rows.vocab) * elem_bytes(rows.dtype);
  if (meets(t.values, n, t.k, t.k, elem_bytes(t.dtype), g0, g1) ||
      meets(t.tokens, n, t.k, t.k, 4, g0, g1) || meets(t.log_norm, n, 1, 1, 4, g0, g1) ||
      meets(out.row_weights, n, out.row_weight_stride, 1, 4, g0, g1) ||
      meets(out.loss, n, 1, 1, 4, g0, g1) ||
      meets(out.stats, n, HKB_DISTILL_STATS, HKB_DISTILL_STATS, 8, g0, g1))
    return invalid("grad must lie apart from the teacher, the weights, the loss and the stats");
  return {HKB_OK, ""};
}

DistillArgs internal_distill(const hkb_distill_teacher& t, const hkb_distill_out& out) {
  DistillArgs a{};
  a.k = t.k;
  a.teacher_dtype = t.dtype;
  a.values = t.values;
  a.tokens = t.tokens;
  a.log_norm = t.log_norm;
  a.temperature = (double)t.temperature;
  a.inv_temperature = 1.0 / a.temperature;
  a.c = (float)(kLog2e * a.inv_temperature);
  a.loss = out.loss;
  a.grad = out.grad;
  a.grad_row_stride = out.grad_row_stride;
  a.row_weights = out.row_weights;
  a.row_weight_stride = out.row_weight_stride;
  a.stats = out.stats;
  return a;
}

}  // namespace
}  // namespace hkb

using namespace hkb;

extern "C" {

hkb_status hkb_sample_tokens(int device, const hkb_vocab_rows* rows,
                             const hkb_sample_settings* s, const hkb_sample_out* out,
                             void* stream) {
  const hkb_status st = check_rows(rows);
  if (st.code != HKB_OK) return st;
  if (s == nullptr || out == nullptr) return invalid("settings and output must be non-null");
  if (s->temperatures == nullptr && !(std::isfinite(s->temperature) && s->temperature >= 0.0f))
    return invalid("temperature must be finite and >= 0");
  if (s->top_ks == nullptr && s->top_k < 0) return invalid("top_k must be >= 0");
  if (s->top_ps == nullptr && !(s->top_p >= 0.0f && s->top_p <= 1.0f))
    return invalid("top_p must be 0 to 1");
  if (s->min_ps == nullptr && !(s->min_p >= 0.0f && s->min_p <= 1.0f))
    return invalid("min_p must be 0 to 1");
  if (s->uniforms_dtype != HKB_F32 && s->uniforms_dtype != HKB_F64)
    return invalid("uniforms must be F32 or F64");
  if (rows->rows == 0) return {HKB_OK, ""};
  if (s->uniforms == nullptr) return invalid("uniforms pointer is null");
  if (out->tokens == nullptr || out->log_probs == nullptr || out->kept == nullptr)
    return invalid("tokens, log_probs and kept must be non-null");
  DeviceGuard guard(device);
  if (guard.status().code != HKB_OK) return guard.status();
  SampleArgs a{};
  a.temperatures = s->temperatures;
  a.top_ks = s->top_ks;
  a.top_ps = s->top_ps;
  a.min_ps = s->min_ps;
  a.temperature = s->temperature;
  a.top_k = s->top_k;
  a.top_p = s->top_p;
  a.min_p = s->min_p;
  a.uniforms = s->uniforms;
  a.uniforms_f64 = s->uniforms_dtype == HKB_F64;
  a.tokens = out->tokens;
  a.log_probs = out->log_probs;
  a.kept = out->kept;
  return launched(launch_sample_tokens(static_cast<cudaStream_t>(stream), internal_rows(*rows), a));
}

hkb_status hkb_top_logits(int device, const hkb_vocab_rows* rows, int32_t k, float temperature,
                          const hkb_top_out* out, void* stream) {
  const hkb_status st = check_rows(rows);
  if (st.code != HKB_OK) return st;
  if (out == nullptr) return invalid("output must be non-null");
  if (k < 1 || k > HKB_LISTING_MAX) return invalid("k must be 1 to HKB_LISTING_MAX");
  if (!(temperature >= HKB_TEMPERATURE_MIN && temperature <= HKB_TEMPERATURE_MAX))
    return invalid("temperature must be 1e-30 to 1e30");
  if (rows->rows == 0) return {HKB_OK, ""};
  if (out->values == nullptr || out->tokens == nullptr)
    return invalid("values and tokens must be non-null");
  DeviceGuard guard(device);
  if (guard.status().code != HKB_OK) return guard.status();
  TopArgs a{};
  a.k = k;
  a.inv_temperature = 1.0 / (double)temperature;
  a.c = (float)(kLog2e * a.inv_temperature);
  a.values = out->values;
  a.tokens = out->tokens;
  a.log_norm = out->log_norm;
  return launched(launch_top_logits(static_cast<cudaStream_t>(stream), internal_rows(*rows), a));
}

hkb_status hkb_distill(int device, const hkb_vocab_rows* rows, const hkb_distill_teacher* t,
                       const hkb_distill_out* out, void* stream) {
  const hkb_status st = check_distill(rows, t, out);
  if (st.code != HKB_OK || rows->rows == 0) return st;
  if (out->loss == nullptr && out->grad == nullptr)
    return invalid("loss or grad must be non-null");
  if (t->values == nullptr || t->tokens == nullptr)
    return invalid("teacher values and tokens must be non-null");
  const hkb_status apart = check_apart(*rows, *t, *out);
  if (apart.code != HKB_OK) return apart;
  DeviceGuard guard(device);
  if (guard.status().code != HKB_OK) return guard.status();
  return launched(launch_distill(static_cast<cudaStream_t>(stream), internal_rows(*rows),
                                 internal_distill(*t, *out)));
}

hkb_status hkb_distill_backward(int device, const hkb_vocab_rows* rows,
                                const hkb_distill_teacher* t, const hkb_distill_out* out,
                                void* stream) {
  const hkb_status st = check_distill(rows, t, out);
  if (st.code != HKB_OK || rows->rows == 0) return st;
  if (out->loss != nullptr) return invalid("a backward pass has no loss");
  if (out->grad == nullptr || out->stats == nullptr)
    return invalid("a backward pass needs grad and stats");
  if (t->values == nullptr || t->tokens == nullptr)
    return invalid("teacher values and tokens must be non-null");
  const hkb_status apart = check_apart(*rows, *t, *out);
  if (apart.code != HKB_OK) return apart;
  DeviceGuard guard(device);
  if (guard.status().code != HKB_OK) return guard.status();
  return launched(launch_distill_backward(static_cast<cudaStream_t>(stream), internal_rows(*rows),
                                          internal_distill(*t, *out)));
}

}  // extern "C"
