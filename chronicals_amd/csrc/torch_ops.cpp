// The torch operators of chronicals_hip over the C ABI of libchronicals_cce
// (include/chronicals_cce.h): operand checks, output and workspace allocation,
// the current stream and one C call each.  In C++ because the same steps in
// Python take longer than the kernels of a small call: 16 rows of fp32 logits,
// V 151936, forward and backward (43 us of kernels) took 179 us with Python
// operators over ctypes and take 87 us with these; 64 rows of d 896 against
// V 32000 went from 222 to 143 us.  Layer norm and the distillation losses have
// their autograd functions here too: a backward in Python waits for the
// interpreter's lock in the autograd thread.  Forward and backward with a Python
// function / so: layer norm of 16384 x 896 106 / 76 us, the fused distillation of
// 64 rows against V 32000 154 / 119 us.
//
// ops.py defines the schemas and the fake (meta) implementations; the kernels
// are registered here.  The C functions come from the library that the Python
// loader opens (chronicals_torch_bind), so that CHRONICALS_CCE_LIB and the
// loader's checks hold for both.  The first call of an operator asks for it, and
// a failing call raises what the package's Python code raises: both through two
// Python callables that ops.py hands over (chronicals_torch_hooks).
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/library.h>

#include <algorithm>
#include <atomic>

#include "../../include/chronicals_cce.h"

namespace {

using at::Tensor;
using std::optional;

struct Api {
  decltype(&cce_last_error) last_error;
  decltype(&cce_forward_workspace_bytes) forward_workspace_bytes;
  decltype(&cce_backward_workspace_bytes) backward_workspace_bytes;
  decltype(&cce_forward) forward;
  decltype(&cce_backward) backward;
  decltype(&cce_logits_forward_workspace_bytes) logits_forward_workspace_bytes;
  decltype(&cce_logits_forward) logits_forward;
  decltype(&cce_logits_backward) logits_backward;
  decltype(&cce_logits_forward_backward) logits_forward_backward;
  decltype(&cce_distill_logits_workspace_bytes) distill_logits_workspace_bytes;
  decltype(&cce_distill_logits_forward) distill_logits_forward;
  decltype(&cce_distill_logits_backward) distill_logits_backward;
  decltype(&cce_distill_forward_workspace_bytes) distill_forward_workspace_bytes;
  decltype(&cce_distill_forward) distill_forward;
  decltype(&cce_distill_backward_workspace_bytes) distill_backward_workspace_bytes;
  decltype(&cce_distill_backward) distill_backward;
  decltype(&cce_top_logits_workspace_bytes) top_logits_workspace_bytes;
  decltype(&cce_top_logits) top_logits;
  decltype(&cce_layer_norm_forward) layer_norm_forward;
  decltype(&cce_layer_norm_backward_workspace_bytes_for) layer_norm_backward_workspace_bytes_for;
  decltype(&cce_layer_norm_backward) layer_norm_backward;
  decltype(&cce_token_logprobs_workspace_bytes) token_logprobs_workspace_bytes;
  decltype(&cce_token_logprobs_forward) token_logprobs_forward;
  decltype(&cce_token_logprobs_backward) token_logprobs_backward;
  decltype(&cce_linear_token_logprobs_workspace_bytes) linear_token_logprobs_workspace_bytes;
  decltype(&cce_linear_token_logprobs_forward) linear_token_logprobs_forward;
  decltype(&cce_linear_token_logprobs_backward_workspace_bytes) linear_token_logprobs_backward_workspace_bytes;
  decltype(&cce_linear_token_logprobs_backward) linear_token_logprobs_backward;
  decltype(&cce_rms_norm_forward) rms_norm_forward;
  decltype(&cce_rms_norm_quantized) rms_norm_quantized;
  decltype(&cce_rms_norm_backward_workspace_bytes) rms_norm_backward_workspace_bytes;
  decltype(&cce_rms_norm_backward) rms_norm_backward;
};

Api g_api;
std::atomic<bool> g_bound{false};

PyObject* g_load = nullptr;   // load(): opens the library and binds it here, or raises
PyObject* g_check = nullptr;  // check(rc): raises for a failing rc, with cce_last_error()'s text

// Calls a hook with its argument, if any; what it raises goes on as a Python
// exception.  Operators run without the interpreter's lock.
void call_hook(PyObject* hook, const long* arg) {
  TORCH_CHECK(hook != nullptr, "chronicals_amd.ops is not imported");
  struct Gil {
    PyGILState_STATE state = PyGILState_Ensure();
    ~Gil() { PyGILState_Release(state); }
  } gil;
  PyObject* const res = arg ? PyObject_CallFunction(hook, "l", *arg) : PyObject_CallObject(hook, nullptr);
  if (!res) {
    python_error e;
    e.persist();
    throw e;
  }
  Py_DECREF(res);
}

const Api& api() {
  if (!g_bound.load(std::memory_order_acquire)) call_hook(g_load, nullptr);
  TORCH_CHECK(g_bound.load(std::memory_order_acquire), "libchronicals_cce.so is not bound");
  return g_api;
}

// cce_last_error() is the calling thread's, and the hook runs in this thread.
void check(const Api& a, int rc) {
  if (rc == CCE_OK) return;
  const long code = rc;
  call_hook(g_check, &code);
  TORCH_CHECK(false, "libchronicals_cce error ", rc, ": ", a.last_error());
}

void* stream(const at::Device& device) {
  return c10::hip::getCurrentHIPStream(device.index()).stream();
}

// The kernels need 16-byte aligned rows: a view at an unaligned storage offset
// is copied to fresh storage.
Tensor aligned(const Tensor& t) {
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 ? t : t.clone();
}

bool is_label(const Tensor& t) { return t.scalar_type() == at::kLong || t.scalar_type() == at::kInt; }

void check_head(const Tensor& hidden, const Tensor& weight, const optional<Tensor>& bias) {
  TORCH_CHECK(hidden.scalar_type() == at::kBFloat16 && weight.scalar_type() == at::kBFloat16,
              "cce ops take bf16 hidden and weight, got ", hidden.scalar_type(), " and ", weight.scalar_type());
  TORCH_CHECK(hidden.dim() == 2 && weight.dim() == 2 && hidden.size(1) == weight.size(1),
              "cce ops take hidden [N, d] and weight [V, d], got ", hidden.sizes(), " and ", weight.sizes());
  TORCH_CHECK(hidden.is_contiguous(), "hidden must be contiguous");
  TORCH_CHECK(weight.is_contiguous(), "weight must be contiguous");
  TORCH_CHECK(hidden.device() == weight.device(), "hidden and weight must be on the same device");
  if (bias.has_value())
    TORCH_CHECK(bias->scalar_type() == at::kFloat && bias->dim() == 1 && bias->size(0) == weight.size(0) &&
                    bias->is_contiguous() && bias->device() == hidden.device(),
                "bias must be a contiguous fp32 [V] tensor");
}

void check_operands(const Tensor& hidden, const Tensor& weight, const Tensor& labels, const optional<Tensor>& bias) {
  check_head(hidden, weight, bias);
  TORCH_CHECK(labels.dim() == 1 && labels.size(0) == hidden.size(0) && is_label(labels),
              "cce ops take int64/int32 labels [N], got ", labels.scalar_type(), " ", labels.sizes());
  TORCH_CHECK(hidden.device() == labels.device(), "hidden, weight and labels must be on the same device");
}

const float* bias_ptr(const optional<Tensor>& bias) {
  return bias.has_value() ? static_cast<const float*>(bias->data_ptr()) : nullptr;
}

// A per-row or scalar gradient as contiguous fp32 (most are: four calls of torch's less).
Tensor grad_rows(const Tensor& g) {
  if (g.dim() == 1 && g.scalar_type() == at::kFloat && g.is_contiguous()) return g;
  return g.detach().to(at::kFloat).reshape({-1}).contiguous();
}

std::tuple<Tensor, Tensor, Tensor, Tensor> cce_fwd(const Tensor& hidden_, const Tensor& weight_, const Tensor& labels_,
                                                   const optional<Tensor>& bias, int64_t ignore_index,
                                                   double label_smoothing, double z_loss_weight,
                                                   int64_t smoothing_form, int64_t reduction, int64_t lse_rows) {
  check_operands(hidden_, weight_, labels_, bias);
  const Api& a = api();
  const c10::DeviceGuard guard(hidden_.device());
  const Tensor hidden = aligned(hidden_), weight = aligned(weight_), labels = labels_.contiguous();
  const int64_t N = hidden.size(0), d = hidden.size(1), V = weight.size(0);
  size_t bytes = 0;
  check(a, a.forward_workspace_bytes(N, d, V, (int)reduction, (int)lse_rows, &bytes));
  const auto f32 = hidden.options().dtype(at::kFloat);
  const Tensor ws = at::empty({(int64_t)bytes}, hidden.options().dtype(at::kByte));
  Tensor loss = at::empty({reduction == CCE_REDUCTION_NONE ? N : 1}, f32);
  Tensor lse = at::empty({N}, f32), target = at::empty({N}, f32);
  Tensor n_valid = at::empty({1}, hidden.options().dtype(at::kInt));
  check(a, a.forward(hidden.data_ptr(), weight.data_ptr(), labels.data_ptr(), labels.scalar_type() == at::kLong,
                     bias_ptr(bias), N, d, V, ignore_index, (float)label_smoothing, (float)z_loss_weight,
                     (int)smoothing_form, (int)reduction, (int)lse_rows, static_cast<float*>(loss.data_ptr()),
                     static_cast<float*>(lse.data_ptr()), static_cast<float*>(target.data_ptr()),
                     static_cast<int32_t*>(n_valid.data_ptr()), ws.data_ptr(), bytes, stream(hidden.device())));
  return {loss, lse, n_valid, target};
}

std::tuple<Tensor, Tensor, Tensor> cce_bwd(const Tensor& grad_out, const Tensor& hidden_, const Tensor& weight_,
                                           const Tensor& labels_, const Tensor& lse, const Tensor& n_valid,
                                           const optional<Tensor>& bias, int64_t ignore_index, double label_smoothing,
                                           double z_loss_weight, int64_t reduction, int64_t chunk_size, bool need_dh,
                                           bool need_dw, bool need_db, bool dh_f32, bool dw_f32) {
  check_operands(hidden_, weight_, labels_, bias);
  TORCH_CHECK(!need_db || bias.has_value(), "need_db requires a bias");
  const Api& a = api();
  const c10::DeviceGuard guard(hidden_.device());
  const Tensor hidden = aligned(hidden_), weight = aligned(weight_), labels = labels_.contiguous();
  const int64_t N = hidden.size(0), d = hidden.size(1), V = weight.size(0);
  const Tensor g = grad_rows(grad_out);
  const auto f32 = hidden.options().dtype(at::kFloat);
  auto empty = [&](bool need, at::IntArrayRef size, bool f) {
    return need ? at::empty(size, f ? f32 : hidden.options()) : at::empty({0}, f ? f32 : hidden.options());
  };
  Tensor dh = empty(need_dh, {N, d}, dh_f32), dw = empty(need_dw, {V, d}, dw_f32), db = empty(need_db, {V}, true);
  if (need_dh || need_dw || need_db) {
    const int hdt = dh_f32 ? CCE_DTYPE_F32 : CCE_DTYPE_BF16, wdt = dw_f32 ? CCE_DTYPE_F32 : CCE_DTYPE_BF16;
    size_t bytes = 0;
    check(a, a.backward_workspace_bytes(N, d, V, chunk_size, need_dh, hdt, need_dw, wdt, &bytes));
    const Tensor ws = at::empty({(int64_t)bytes}, hidden.options().dtype(at::kByte));
    check(a, a.backward(static_cast<const float*>(g.data_ptr()), hidden.data_ptr(), weight.data_ptr(),
                        labels.data_ptr(), labels.scalar_type() == at::kLong, bias_ptr(bias),
                        static_cast<const float*>(lse.data_ptr()), static_cast<const int32_t*>(n_valid.data_ptr()), N,
                        d, V, ignore_index, (float)label_smoothing, (float)z_loss_weight, (int)reduction, chunk_size,
                        need_dh ? dh.data_ptr() : nullptr, hdt, need_dw ? dw.data_ptr() : nullptr, wdt,
                        need_db ? static_cast<float*>(db.data_ptr()) : nullptr, ws.data_ptr(), bytes,
                        stream(hidden.device())));
  }
  return {dh, dw, db};
}

int logits_dtype(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return CCE_DTYPE_BF16;
    case at::kHalf: return CCE_DTYPE_F16;
    case at::kFloat: return CCE_DTYPE_F32;
    default: TORCH_CHECK(false, "logits dtype ", t.scalar_type(), " not supported (bf16, fp16, fp32)");
  }
}

void check_logits(const Tensor& logits, const Tensor& labels) {
  logits_dtype(logits);
  TORCH_CHECK(logits.dim() == 2 && (logits.size(1) <= 1 || logits.stride(1) == 1),
              "ce_logits ops take [N, V] logits with a contiguous last dimension, got shape ", logits.sizes(),
              " strides ", logits.strides());
  TORCH_CHECK(labels.dim() == 1 && labels.size(0) == logits.size(0) && is_label(labels),
              "ce_logits ops take int64/int32 labels [N], got ", labels.scalar_type(), " ", labels.sizes());
  TORCH_CHECK(labels.is_contiguous(), "labels must be contiguous");
  TORCH_CHECK(labels.device() == logits.device(), "logits and labels must be on the same device");
}

int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

struct LogitsOut {
  Tensor ws, loss, lse, n_valid;
  size_t bytes = 0;
  LogitsOut(const Api& a, const Tensor& logits, int64_t reduction) {
    const int64_t N = logits.size(0), V = logits.size(1);
    check(a, a.logits_forward_workspace_bytes(N, V, (int)reduction, &bytes));
    const auto f32 = logits.options().dtype(at::kFloat);
    ws = at::empty({(int64_t)bytes}, logits.options().dtype(at::kByte));
    loss = at::empty({reduction == CCE_REDUCTION_NONE ? N : 1}, f32);
    lse = at::empty({N}, f32);
    n_valid = at::empty({1}, logits.options().dtype(at::kInt));
  }
};

std::tuple<Tensor, Tensor, Tensor> ce_logits_fwd(const Tensor& logits, const Tensor& labels, int64_t ignore_index,
                                                 double label_smoothing, double z_loss_weight, int64_t smoothing_form,
                                                 int64_t reduction) {
  check_logits(logits, labels);
  const Api& a = api();
  const c10::DeviceGuard guard(logits.device());
  LogitsOut o(a, logits, reduction);
  check(a, a.logits_forward(logits.data_ptr(), logits_dtype(logits), row_stride(logits), labels.data_ptr(),
                            labels.scalar_type() == at::kLong, logits.size(0), logits.size(1), ignore_index,
                            (float)label_smoothing, (float)z_loss_weight, (int)smoothing_form, (int)reduction,
                            static_cast<float*>(o.loss.data_ptr()), static_cast<float*>(o.lse.data_ptr()),
                            static_cast<int32_t*>(o.n_valid.data_ptr()), o.ws.data_ptr(), o.bytes,
                            stream(logits.device())));
  return {o.loss, o.lse, o.n_valid};
}

Tensor gradient_like(const Tensor& logits, bool f32_grad) {
  return at::empty(logits.sizes(), f32_grad ? logits.options().dtype(at::kFloat) : logits.options());
}

Tensor ce_logits_bwd(const Tensor& grad_out, const Tensor& logits, const Tensor& labels, const Tensor& lse,
                     const Tensor& n_valid, int64_t ignore_index, double label_smoothing, double z_loss_weight,
                     int64_t smoothing_form, int64_t reduction, bool f32_grad) {
  check_logits(logits, labels);
  const Api& a = api();
  const c10::DeviceGuard guard(logits.device());
  Tensor dx = gradient_like(logits, f32_grad);
  if (logits.size(0) == 0) return dx;
  const Tensor g = grad_rows(grad_out);
  check(a, a.logits_backward(static_cast<const float*>(g.data_ptr()), logits.data_ptr(), logits_dtype(logits),
                             row_stride(logits), labels.data_ptr(), labels.scalar_type() == at::kLong,
                             static_cast<const float*>(lse.data_ptr()),
                             static_cast<const int32_t*>(n_valid.data_ptr()), logits.size(0), logits.size(1),
                             ignore_index, (float)label_smoothing, (float)z_loss_weight, (int)smoothing_form,
                             (int)reduction, dx.data_ptr(), logits_dtype(dx), row_stride(dx),
                             stream(logits.device())));
  return dx;
}

std::tuple<Tensor, Tensor, Tensor, Tensor> ce_logits_fwd_bwd(const Tensor& logits, const Tensor& labels,
                                                             int64_t ignore_index, double label_smoothing,
                                                             double z_loss_weight, int64_t smoothing_form,
                                                             int64_t reduction, bool grad_mean, bool f32_grad) {
  check_logits(logits, labels);
  const Api& a = api();
  const c10::DeviceGuard guard(logits.device());
  LogitsOut o(a, logits, reduction);
  Tensor dx = gradient_like(logits, f32_grad);
  check(a, a.logits_forward_backward(
               logits.data_ptr(), logits_dtype(logits), row_stride(logits), labels.data_ptr(),
               labels.scalar_type() == at::kLong, logits.size(0), logits.size(1), ignore_index,
               (float)label_smoothing, (float)z_loss_weight, (int)smoothing_form, (int)reduction, grad_mean,
               static_cast<float*>(o.loss.data_ptr()), static_cast<float*>(o.lse.data_ptr()),
               static_cast<int32_t*>(o.n_valid.data_ptr()), dx.data_ptr(), logits_dtype(dx), row_stride(dx),
               o.ws.data_ptr(), o.bytes, stream(logits.device())));
  return {o.loss, o.lse, o.n_valid, dx};
}

// ---------------------------------------------------------------------------
// Distillation, the teacher's top logits, layer norm
// ---------------------------------------------------------------------------

float* f32(const Tensor& t) { return static_cast<float*>(t.data_ptr()); }

bool is_logits(const Tensor& t) {
  return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf || t.scalar_type() == at::kFloat;
}

// What a forward kept, as it came.
void check_kept(const Tensor& t, const char* name, at::ScalarType type, int64_t numel, const Tensor& student) {
  TORCH_CHECK(t.scalar_type() == type && t.numel() == numel && t.is_contiguous() && t.device() == student.device(), name,
              " must be the forward's output (", numel, " contiguous ", type, " values), got ", t.scalar_type(), " ",
              t.sizes());
}

// A teacher's entries with what they need checked against N student rows.
struct TeacherArgs {
  cce_teacher t;
  TeacherArgs(const Tensor& logits, const Tensor& indices, const Tensor& student, int64_t N, double temperature,
              double distill_weight, double ce_weight) {
    TORCH_CHECK(is_logits(logits), "teacher logits dtype ", logits.scalar_type(), " not supported (bf16, fp16, fp32)");
    TORCH_CHECK(logits.dim() == 2 && logits.size(0) == N && indices.sizes() == logits.sizes() && is_label(indices),
                "distill ops take teacher logits [N = ", N, ", K] and int64/int32 indices of the same shape, got ",
                logits.sizes(), " and ", indices.scalar_type(), " ", indices.sizes());
    TORCH_CHECK(logits.is_contiguous() && indices.is_contiguous(), "teacher logits and indices must be contiguous");
    TORCH_CHECK(logits.device() == student.device() && indices.device() == student.device(),
                "teacher logits and indices must be on the student's device");
    t.logits = logits.data_ptr();
    t.indices = indices.data_ptr();
    t.entries = logits.size(1);
    t.logits_dtype = logits_dtype(logits);
    t.indices_int64 = indices.scalar_type() == at::kLong;
    t.temperature = (float)temperature;
    t.distill_weight = (float)distill_weight;
    t.ce_weight = (float)ce_weight;
  }
};

void check_row_labels(const optional<Tensor>& labels, const Tensor& student, int64_t N) {
  if (!labels.has_value()) return;
  TORCH_CHECK(labels->dim() == 1 && labels->size(0) == N && is_label(*labels) && labels->is_contiguous(),
              "distill ops take contiguous int64/int32 labels [N = ", N, "], got ", labels->scalar_type(), " ",
              labels->sizes());
  TORCH_CHECK(labels->device() == student.device(), "labels must be on the student's device");
}

const void* label_ptr(const optional<Tensor>& labels) { return labels.has_value() ? labels->data_ptr() : nullptr; }
int label_int64(const optional<Tensor>& labels) { return labels.has_value() && labels->scalar_type() == at::kLong; }

void check_student_logits(const Tensor& logits) {
  logits_dtype(logits);
  TORCH_CHECK(logits.dim() == 2 && (logits.size(1) <= 1 || logits.stride(1) == 1),
              "distill ops take [N, V] logits with a contiguous last dimension, got shape ", logits.sizes(),
              " strides ", logits.strides());
}

std::tuple<Tensor, Tensor, Tensor> distill_logits_fwd(const Tensor& logits, const Tensor& teacher_logits,
                                                      const Tensor& teacher_indices, const optional<Tensor>& labels,
                                                      double temperature, double distill_weight, double ce_weight,
                                                      int64_t ignore_index, int64_t reduction) {
  check_student_logits(logits);
  const int64_t N = logits.size(0), V = logits.size(1);
  check_row_labels(labels, logits, N);
  const TeacherArgs teacher(teacher_logits, teacher_indices, logits, N, temperature, distill_weight, ce_weight);
  const Api& a = api();
  const c10::DeviceGuard guard(logits.device());
  size_t bytes = 0;
  check(a, a.distill_logits_workspace_bytes(N, V, (int)reduction, &bytes));
  const auto opt = logits.options().dtype(at::kFloat);
  const Tensor ws = at::empty({(int64_t)bytes}, logits.options().dtype(at::kByte));
  Tensor loss = at::empty({reduction == CCE_REDUCTION_NONE ? N : 1}, opt), stats = at::empty({N, 4}, opt);
  Tensor n_valid = at::empty({1}, logits.options().dtype(at::kInt));
  check(a, a.distill_logits_forward(logits.data_ptr(), logits_dtype(logits), row_stride(logits), &teacher.t,
                                    label_ptr(labels), label_int64(labels), N, V, ignore_index, (int)reduction,
                                    f32(loss), f32(stats), static_cast<int32_t*>(n_valid.data_ptr()), ws.data_ptr(),
                                    bytes, stream(logits.device())));
  return {loss, stats, n_valid};
}

Tensor distill_logits_bwd(const Tensor& grad_out, const Tensor& logits, const Tensor& teacher_logits,
                          const Tensor& teacher_indices, const optional<Tensor>& labels, const Tensor& stats,
                          const Tensor& n_valid, double temperature, double distill_weight, double ce_weight,
                          int64_t ignore_index, int64_t reduction) {
  check_student_logits(logits);
  const int64_t N = logits.size(0), V = logits.size(1);
  check_row_labels(labels, logits, N);
  const TeacherArgs teacher(teacher_logits, teacher_indices, logits, N, temperature, distill_weight, ce_weight);
  const Api& a = api();
  const c10::DeviceGuard guard(logits.device());
  Tensor dx = at::empty(logits.sizes(), logits.options());
  const Tensor g = grad_rows(grad_out);
  check_kept(g, "grad_out", at::kFloat, reduction == CCE_REDUCTION_NONE ? N : 1, logits);
  check_kept(stats, "stats", at::kFloat, 4 * N, logits);
  check_kept(n_valid, "n_valid", at::kInt, 1, logits);
  check(a, a.distill_logits_backward(f32(g), logits.data_ptr(), logits_dtype(logits), row_stride(logits), &teacher.t,
                                     label_ptr(labels), label_int64(labels), f32(stats),
                                     static_cast<const int32_t*>(n_valid.data_ptr()), N, V, ignore_index,
                                     (int)reduction, dx.data_ptr(), row_stride(dx), stream(logits.device())));
  return dx;
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> distill_fwd(
    const Tensor& hidden_, const Tensor& weight_, const optional<Tensor>& bias, const Tensor& teacher_logits,
    const Tensor& teacher_indices, const optional<Tensor>& labels, double temperature, double distill_weight,
    double ce_weight, int64_t ignore_index, int64_t reduction) {
  check_head(hidden_, weight_, bias);
  const int64_t N = hidden_.size(0), d = hidden_.size(1), V = weight_.size(0);
  check_row_labels(labels, hidden_, N);
  const TeacherArgs teacher(teacher_logits, teacher_indices, hidden_, N, temperature, distill_weight, ce_weight);
  const Api& a = api();
  const c10::DeviceGuard guard(hidden_.device());
  const Tensor hidden = aligned(hidden_), weight = aligned(weight_);
  size_t bytes = 0;
  check(a, a.distill_forward_workspace_bytes(N, d, V, (int)reduction, &bytes));
  const auto opt = hidden.options().dtype(at::kFloat), i32 = hidden.options().dtype(at::kInt);
  const Tensor ws = at::empty({(int64_t)bytes}, hidden.options().dtype(at::kByte));
  Tensor loss = at::empty({reduction == CCE_REDUCTION_NONE ? N : 1}, opt), stats = at::empty({N, 2}, opt);
  Tensor entry_logits = at::empty({N, teacher.t.entries + 1}, opt), rows = at::empty({N}, i32);
  Tensor n_valid = at::empty({1}, i32);
  check(a, a.distill_forward(hidden.data_ptr(), weight.data_ptr(), bias_ptr(bias), &teacher.t, label_ptr(labels),
                             label_int64(labels), N, d, V, ignore_index, (int)reduction, f32(loss), f32(stats),
                             f32(entry_logits), static_cast<int32_t*>(rows.data_ptr()),
                             static_cast<int32_t*>(n_valid.data_ptr()), ws.data_ptr(), bytes,
                             stream(hidden.device())));
  return {loss, stats, entry_logits, rows, n_valid};
}

std::tuple<Tensor, Tensor, Tensor> distill_bwd(const Tensor& grad_out, const Tensor& hidden_, const Tensor& weight_,
                                               const optional<Tensor>& bias, const Tensor& teacher_logits,
                                               const Tensor& teacher_indices, const Tensor& stats,
                                               const Tensor& entry_logits, const Tensor& rows, const Tensor& n_valid,
                                               double temperature, double distill_weight, double ce_weight,
                                               int64_t reduction, int64_t chunk_size, bool need_dh, bool need_dw,
                                               bool need_db, bool dh_f32, bool dw_f32) {
  check_head(hidden_, weight_, bias);
  TORCH_CHECK(!need_db || bias.has_value(), "need_db requires a bias");
  const int64_t N = hidden_.size(0), d = hidden_.size(1), V = weight_.size(0);
  const TeacherArgs teacher(teacher_logits, teacher_indices, hidden_, N, temperature, distill_weight, ce_weight);
  const Api& a = api();
  const c10::DeviceGuard guard(hidden_.device());
  const Tensor hidden = aligned(hidden_), weight = aligned(weight_);
  const Tensor g = grad_rows(grad_out);
  check_kept(g, "grad_out", at::kFloat, reduction == CCE_REDUCTION_NONE ? N : 1, hidden);
  check_kept(stats, "stats", at::kFloat, 2 * N, hidden);
  check_kept(entry_logits, "entry_logits", at::kFloat, N * (teacher.t.entries + 1), hidden);
  check_kept(rows, "rows", at::kInt, N, hidden);
  check_kept(n_valid, "n_valid", at::kInt, 1, hidden);
  const auto opt = hidden.options().dtype(at::kFloat);
  auto empty = [&](bool need, at::IntArrayRef size, bool f) {
    return at::empty(need ? size : at::IntArrayRef{0}, f ? opt : hidden.options());
  };
  Tensor dh = empty(need_dh, {N, d}, dh_f32), dw = empty(need_dw, {V, d}, dw_f32), db = empty(need_db, {V}, true);
  if (need_dh || need_dw || need_db) {
    const int hdt = dh_f32 ? CCE_DTYPE_F32 : CCE_DTYPE_BF16, wdt = dw_f32 ? CCE_DTYPE_F32 : CCE_DTYPE_BF16;
    size_t bytes = 0;
    check(a, a.distill_backward_workspace_bytes(N, d, V, teacher.t.entries, chunk_size, need_dh, hdt, need_dw, wdt,
                                                &bytes));
    const Tensor ws = at::empty({(int64_t)bytes}, hidden.options().dtype(at::kByte));
    check(a, a.distill_backward(f32(g), hidden.data_ptr(), weight.data_ptr(), bias_ptr(bias), &teacher.t, f32(stats),
                                f32(entry_logits), static_cast<const int32_t*>(rows.data_ptr()),
                                static_cast<const int32_t*>(n_valid.data_ptr()), N, d, V, (int)reduction, chunk_size,
                                need_dh ? dh.data_ptr() : nullptr, hdt, need_dw ? dw.data_ptr() : nullptr, wdt,
                                need_db ? f32(db) : nullptr, ws.data_ptr(), bytes, stream(hidden.device())));
  }
  return {dh, dw, db};
}

std::tuple<Tensor, Tensor> top_logits(const Tensor& logits, int64_t k) {
  logits_dtype(logits);
  TORCH_CHECK(logits.dim() == 2 && (logits.size(1) <= 1 || logits.stride(1) == 1),
              "top_logits takes [N, V] logits with a contiguous last dimension, got shape ", logits.sizes(),
              " strides ", logits.strides());
  const Api& a = api();
  const c10::DeviceGuard guard(logits.device());
  const int64_t N = logits.size(0), V = logits.size(1);
  TORCH_CHECK(k >= 1 && k <= std::min<int64_t>(V, CCE_MAX_TEACHER_ENTRIES), "k must be in [1, min(",
              CCE_MAX_TEACHER_ENTRIES, ", V = ", V, ")], got ", k);
  Tensor values = at::empty({N, k}, logits.options()), indices = at::empty({N, k}, logits.options().dtype(at::kLong));
  size_t bytes = 0;
  check(a, a.top_logits_workspace_bytes(N, V, k, &bytes));
  const Tensor ws = at::empty({(int64_t)bytes}, logits.options().dtype(at::kByte));
  check(a, a.top_logits(logits.data_ptr(), logits_dtype(logits), row_stride(logits), N, V, k, values.data_ptr(),
                        static_cast<int64_t*>(indices.data_ptr()), ws.data_ptr(), bytes, stream(logits.device())));
  return {values, indices};
}

void check_norm_rows(const Tensor& x, const char* what) {
  TORCH_CHECK(is_logits(x), what, " dtype ", x.scalar_type(), " not supported (bf16, fp16, fp32)");
  TORCH_CHECK(x.dim() == 2 && (x.size(0) == 0 || x.size(1) <= 1 || x.stride(1) == 1), what,
              " ops take [N, D] rows with a contiguous last dimension, got shape ", x.sizes(), " strides ", x.strides());
}

// The parameters' type: that of the weight or, without one, of the bias.
int check_norm(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias) {
  check_norm_rows(x, "layer_norm");
  at::ScalarType type = x.scalar_type();
  for (const optional<Tensor>* p : {&bias, &weight}) {
    if (!p->has_value()) continue;
    const Tensor& t = **p;
    TORCH_CHECK(t.dim() == 1 && t.size(0) == x.size(1) && t.is_contiguous() && t.device() == x.device(),
                "weight and bias must be contiguous [D] tensors on the input's device, got ", t.sizes());
    type = t.scalar_type();
    TORCH_CHECK(type == x.scalar_type() || type == at::kFloat, "weight and bias must have the input's dtype or fp32, got ",
                type);
  }
  TORCH_CHECK(!weight.has_value() || !bias.has_value() || weight->scalar_type() == bias->scalar_type(),
              "weight and bias must have the same dtype");
  return type == at::kFloat ? CCE_DTYPE_F32 : logits_dtype(x);
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_fwd(const Tensor& x, const optional<Tensor>& weight,
                                                  const optional<Tensor>& bias, double eps) {
  const int pdt = check_norm(x, weight, bias);
  const Api& a = api();
  const c10::DeviceGuard guard(x.device());
  const int64_t N = x.size(0), D = x.size(1);
  const auto opt = x.options().dtype(at::kFloat);
  Tensor y = at::empty({N, D}, x.options()), mean = at::empty({N}, opt), rstd = at::empty({N}, opt);
  check(a, a.layer_norm_forward(x.data_ptr(), logits_dtype(x), row_stride(x), label_ptr(weight), label_ptr(bias), pdt,
                                N, D, (float)eps, y.data_ptr(), f32(mean), f32(rstd), stream(x.device())));
  return {y, mean, rstd};
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_bwd(const Tensor& grad_y, const Tensor& x, const optional<Tensor>& weight,
                                                  const Tensor& mean, const Tensor& rstd, bool param_f32, bool need_dx,
                                                  bool need_dw, bool need_db) {
  const int wdt = check_norm(x, weight, std::nullopt);
  const int pdt = param_f32 ? CCE_DTYPE_F32 : logits_dtype(x);
  TORCH_CHECK(!weight.has_value() || wdt == pdt, "param_f32 does not fit the weight's dtype");
  TORCH_CHECK(grad_y.sizes() == x.sizes() && grad_y.scalar_type() == x.scalar_type() && grad_y.is_contiguous() &&
                  grad_y.device() == x.device(),
              "grad_y must be a contiguous tensor of the input's shape, dtype and device");
  const int64_t N = x.size(0), D = x.size(1);
  check_kept(mean, "mean", at::kFloat, N, x);
  check_kept(rstd, "rstd", at::kFloat, N, x);
  const Api& a = api();
  const c10::DeviceGuard guard(x.device());
  const auto popt = x.options().dtype(param_f32 ? at::kFloat : x.scalar_type());
  Tensor dx = at::empty(need_dx ? x.sizes() : at::IntArrayRef{0}, x.options());
  Tensor dw = at::empty({need_dw ? D : 0}, popt), db = at::empty({need_db ? D : 0}, popt);
  size_t bytes = 0;
  check(a, a.layer_norm_backward_workspace_bytes_for(N, D, logits_dtype(x), need_dw || need_db, &bytes));
  const Tensor ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
  check(a, a.layer_norm_backward(grad_y.data_ptr(), x.data_ptr(), logits_dtype(x), row_stride(x), label_ptr(weight),
                                 pdt, f32(mean), f32(rstd), N, D, need_dx ? dx.data_ptr() : nullptr,
                                 need_dw ? dw.data_ptr() : nullptr, need_db ? db.data_ptr() : nullptr, ws.data_ptr(),
                                 bytes, stream(x.device())));
  return {dx, dw, db};
}

// ---------------------------------------------------------------------------
// Token log-probabilities, RMS norm
// ---------------------------------------------------------------------------

void check_tokens(const Tensor& tokens, const Tensor& x) {
  TORCH_CHECK(tokens.dim() == 1 && tokens.size(0) == x.size(0) && is_label(tokens) && tokens.is_contiguous(),
              "token_logprobs ops take contiguous int64/int32 tokens [N = ", x.size(0), "], got ", tokens.scalar_type(),
              " ", tokens.sizes());
  TORCH_CHECK(tokens.device() == x.device(), "tokens must be on the device of the logits or hidden states");
}

struct LogprobsOut {
  Tensor logprobs, entropy, stats, top_logprobs, top_indices;
  LogprobsOut(const Tensor& x, int64_t top_k, int64_t V) {
    TORCH_CHECK(top_k >= 0 && top_k <= std::min<int64_t>(V, CCE_MAX_TEACHER_ENTRIES), "top_k must be in [0, min(",
                CCE_MAX_TEACHER_ENTRIES, ", V = ", V, ")], got ", top_k);
    const int64_t N = x.size(0);
    const auto opt = x.options().dtype(at::kFloat);
    logprobs = at::empty({N}, opt);
    entropy = at::empty({N}, opt);
    stats = at::empty({N, 4}, opt);
    top_logprobs = at::empty({N, top_k}, opt);
    top_indices = at::empty({N, top_k}, x.options().dtype(at::kLong));
  }
  std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> all() const {
    return {logprobs, entropy, stats, top_logprobs, top_indices};
  }
  int64_t* indices() const { return static_cast<int64_t*>(top_indices.data_ptr()); }
};

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> token_logprobs_fwd(const Tensor& logits, const Tensor& tokens,
                                                                      double temperature, int64_t top_k,
                                                                      int64_t ignore_index) {
  check_student_logits(logits);
  check_tokens(tokens, logits);
  const Api& a = api();
  const c10::DeviceGuard guard(logits.device());
  const int64_t N = logits.size(0), V = logits.size(1);
  const LogprobsOut o(logits, top_k, V);
  size_t bytes = 0;
  check(a, a.token_logprobs_workspace_bytes(N, V, top_k, &bytes));
  const Tensor ws = at::empty({(int64_t)bytes}, logits.options().dtype(at::kByte));
  check(a, a.token_logprobs_forward(logits.data_ptr(), logits_dtype(logits), row_stride(logits), tokens.data_ptr(),
                                    tokens.scalar_type() == at::kLong, N, V, ignore_index, (float)temperature, top_k,
                                    f32(o.logprobs), f32(o.entropy), f32(o.stats), f32(o.top_logprobs), o.indices(),
                                    ws.data_ptr(), bytes, stream(logits.device())));
  return o.all();
}

// A gradient per row that may be absent, as contiguous fp32.
struct RowGrad {
  Tensor t;
  RowGrad(const optional<Tensor>& g, const char* name, const Tensor& x) {
    if (!g.has_value()) return;
    t = grad_rows(*g);
    check_kept(t, name, at::kFloat, x.size(0), x);
  }
  const float* ptr() const { return t.defined() ? f32(t) : nullptr; }
};

Tensor token_logprobs_bwd(const optional<Tensor>& grad_logprobs, const optional<Tensor>& grad_entropy,
                          const Tensor& logits, const Tensor& tokens, const Tensor& stats, double temperature,
                          int64_t ignore_index) {
  check_student_logits(logits);
  check_tokens(tokens, logits);
  check_kept(stats, "stats", at::kFloat, 4 * logits.size(0), logits);
  const Api& a = api();
  const c10::DeviceGuard guard(logits.device());
  const RowGrad g(grad_logprobs, "grad_logprobs", logits), h(grad_entropy, "grad_entropy", logits);
  Tensor dx = at::empty(logits.sizes(), logits.options());
  check(a, a.token_logprobs_backward(g.ptr(), h.ptr(), logits.data_ptr(), logits_dtype(logits), row_stride(logits),
                                     tokens.data_ptr(), tokens.scalar_type() == at::kLong, f32(stats), logits.size(0),
                                     logits.size(1), ignore_index, (float)temperature, dx.data_ptr(), row_stride(dx),
                                     stream(logits.device())));
  return dx;
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> linear_token_logprobs_fwd(
    const Tensor& hidden_, const Tensor& weight_, const optional<Tensor>& bias, const Tensor& tokens, double temperature,
    int64_t top_k, int64_t ignore_index) {
  check_head(hidden_, weight_, bias);
  check_tokens(tokens, hidden_);
  const Api& a = api();
  const c10::DeviceGuard guard(hidden_.device());
  const Tensor hidden = aligned(hidden_), weight = aligned(weight_);
  const int64_t N = hidden.size(0), d = hidden.size(1), V = weight.size(0);
  const LogprobsOut o(hidden, top_k, V);
  size_t bytes = 0;
  check(a, a.linear_token_logprobs_workspace_bytes(N, d, V, top_k, &bytes));
  const Tensor ws = at::empty({(int64_t)bytes}, hidden.options().dtype(at::kByte));
  check(a, a.linear_token_logprobs_forward(hidden.data_ptr(), weight.data_ptr(), bias_ptr(bias), tokens.data_ptr(),
                                           tokens.scalar_type() == at::kLong, N, d, V, ignore_index, (float)temperature,
                                           top_k, f32(o.logprobs), f32(o.entropy), f32(o.stats), f32(o.top_logprobs),
                                           o.indices(), ws.data_ptr(), bytes, stream(hidden.device())));
  return o.all();
}

std::tuple<Tensor, Tensor, Tensor> linear_token_logprobs_bwd(
    const optional<Tensor>& grad_logprobs, const optional<Tensor>& grad_entropy, const Tensor& hidden_,
    const Tensor& weight_, const optional<Tensor>& bias, const Tensor& tokens, const Tensor& stats, double temperature,
    int64_t ignore_index, int64_t chunk_size, bool need_dh, bool need_dw, bool need_db, bool dh_f32, bool dw_f32) {
  check_head(hidden_, weight_, bias);
  check_tokens(tokens, hidden_);
  TORCH_CHECK(!need_db || bias.has_value(), "need_db requires a bias");
  const Api& a = api();
  const c10::DeviceGuard guard(hidden_.device());
  const Tensor hidden = aligned(hidden_), weight = aligned(weight_);
  const int64_t N = hidden.size(0), d = hidden.size(1), V = weight.size(0);
  check_kept(stats, "stats", at::kFloat, 4 * N, hidden);
  const RowGrad g(grad_logprobs, "grad_logprobs", hidden), h(grad_entropy, "grad_entropy", hidden);
  const auto opt = hidden.options().dtype(at::kFloat);
  auto empty = [&](bool need, at::IntArrayRef size, bool f) {
    return at::empty(need ? size : at::IntArrayRef{0}, f ? opt : hidden.options());
  };
  Tensor dh = empty(need_dh, {N, d}, dh_f32), dw = empty(need_dw, {V, d}, dw_f32), db = empty(need_db, {V}, true);
  if (need_dh || need_dw || need_db) {
    const int hdt = dh_f32 ? CCE_DTYPE_F32 : CCE_DTYPE_BF16, wdt = dw_f32 ? CCE_DTYPE_F32 : CCE_DTYPE_BF16;
    size_t bytes = 0;
    check(a, a.linear_token_logprobs_backward_workspace_bytes(N, d, V, chunk_size, need_dh, hdt, need_dw, wdt, &bytes));
    const Tensor ws = at::empty({(int64_t)bytes}, hidden.options().dtype(at::kByte));
    check(a, a.linear_token_logprobs_backward(
                 g.ptr(), h.ptr(), hidden.data_ptr(), weight.data_ptr(), bias_ptr(bias), tokens.data_ptr(),
                 tokens.scalar_type() == at::kLong, f32(stats), N, d, V, ignore_index, (float)temperature, chunk_size,
                 need_dh ? dh.data_ptr() : nullptr, hdt, need_dw ? dw.data_ptr() : nullptr, wdt,
                 need_db ? f32(db) : nullptr, ws.data_ptr(), bytes, stream(hidden.device())));
  }
  return {dh, dw, db};
}

// Operands of an RMS norm: the weight's type, and the residual's as the C functions take it.
struct RmsArgs {
  int param, dtype;
  const void* residual = nullptr;
  int residual_dtype;
  int64_t ldr;
  RmsArgs(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& r) {
    check_norm_rows(x, "rms_norm");
    dtype = residual_dtype = logits_dtype(x);
    ldr = x.size(1);
    param = check_norm(x, weight, std::nullopt);
    if (!r.has_value()) return;
    check_norm_rows(*r, "rms_norm residual");
    TORCH_CHECK(r->sizes() == x.sizes() && r->device() == x.device() &&
                    (r->scalar_type() == x.scalar_type() || r->scalar_type() == at::kFloat),
                "residual must have the input's shape and device, and its dtype or fp32, got ", r->scalar_type(), " ",
                r->sizes());
    residual = r->data_ptr();
    residual_dtype = logits_dtype(*r);
    ldr = row_stride(*r);
  }
};

Tensor sum_like(const Tensor& x, const optional<Tensor>& residual) {
  return residual.has_value() ? at::empty(x.sizes(), residual->options()) : at::empty({0}, x.options());
}

std::tuple<Tensor, Tensor, Tensor> rms_norm_fwd(const Tensor& x, const optional<Tensor>& weight,
                                                const optional<Tensor>& residual, double eps) {
  const RmsArgs r(x, weight, residual);
  const Api& a = api();
  const c10::DeviceGuard guard(x.device());
  const int64_t N = x.size(0), D = x.size(1);
  Tensor y = at::empty({N, D}, x.options()), sum = sum_like(x, residual);
  Tensor rstd = at::empty({N}, x.options().dtype(at::kFloat));
  check(a, a.rms_norm_forward(x.data_ptr(), r.dtype, row_stride(x), r.residual, r.residual_dtype, r.ldr,
                              label_ptr(weight), r.param, N, D, (float)eps, y.data_ptr(),
                              r.residual ? sum.data_ptr() : nullptr, f32(rstd), stream(x.device())));
  return {y, sum, rstd};
}

std::tuple<Tensor, Tensor, Tensor> rms_norm_quantized(const Tensor& x, const optional<Tensor>& weight,
                                                      const optional<Tensor>& residual, double eps, bool int8,
                                                      int64_t group) {
  const RmsArgs r(x, weight, residual);
  TORCH_CHECK(group == 0 || group == 32 || group == 64 || group == 128 || group == 256,
              "group must be 0 (a row), 32, 64, 128 or 256, got ", group);
  const Api& a = api();
  const c10::DeviceGuard guard(x.device());
  const int64_t N = x.size(0), D = x.size(1);
  Tensor q = at::empty({N, D}, x.options().dtype(int8 ? at::kChar : at::kFloat8_e4m3fn));
  const auto opt = x.options().dtype(at::kFloat);
  Tensor scales = group ? at::empty({N, (D + group - 1) / group}, opt) : at::empty({N}, opt);
  Tensor sum = sum_like(x, residual);
  check(a, a.rms_norm_quantized(x.data_ptr(), r.dtype, row_stride(x), r.residual, r.residual_dtype, r.ldr,
                                label_ptr(weight), r.param, N, D, (float)eps, int8 ? CCE_DTYPE_INT8 : CCE_DTYPE_E4M3,
                                group, q.data_ptr(), f32(scales), r.residual ? sum.data_ptr() : nullptr,
                                stream(x.device())));
  return {q, scales, sum};
}

std::tuple<Tensor, Tensor, Tensor> rms_norm_bwd(const Tensor& grad_y, const optional<Tensor>& grad_sum, const Tensor& sum,
                                                const optional<Tensor>& weight, const Tensor& rstd, bool param_f32,
                                                bool need_dx, bool need_dr, bool need_dw) {
  const RmsArgs r(grad_y, weight, sum);
  const int pdt = param_f32 ? CCE_DTYPE_F32 : r.dtype;
  TORCH_CHECK(!weight.has_value() || r.param == pdt, "param_f32 does not fit the weight's dtype");
  TORCH_CHECK(grad_y.is_contiguous(), "grad_y must be contiguous");
  TORCH_CHECK(!grad_sum.has_value() || (grad_sum->sizes() == sum.sizes() && grad_sum->is_contiguous() &&
                                        grad_sum->scalar_type() == sum.scalar_type() && grad_sum->device() == sum.device()),
              "grad_sum must be a contiguous tensor of the sum's shape, dtype and device");
  const int64_t N = grad_y.size(0), D = grad_y.size(1);
  check_kept(rstd, "rstd", at::kFloat, N, grad_y);
  const Api& a = api();
  const c10::DeviceGuard guard(grad_y.device());
  Tensor dx = at::empty(need_dx ? grad_y.sizes() : at::IntArrayRef{0}, grad_y.options());
  Tensor dr = at::empty(need_dr ? grad_y.sizes() : at::IntArrayRef{0}, sum.options());
  Tensor dw = at::empty({need_dw ? D : 0}, grad_y.options().dtype(param_f32 ? at::kFloat : grad_y.scalar_type()));
  size_t bytes = 0;
  check(a, a.rms_norm_backward_workspace_bytes(N, D, r.dtype, need_dw, &bytes));
  const Tensor ws = at::empty({(int64_t)bytes}, grad_y.options().dtype(at::kByte));
  check(a, a.rms_norm_backward(grad_y.data_ptr(), label_ptr(grad_sum), sum.data_ptr(), r.dtype, r.residual_dtype, r.ldr,
                               label_ptr(weight), pdt, f32(rstd), N, D, need_dx ? dx.data_ptr() : nullptr,
                               need_dr ? dr.data_ptr() : nullptr, need_dw ? dw.data_ptr() : nullptr, ws.data_ptr(), bytes,
                               stream(grad_y.device())));
  return {dx, dr, dw};
}

// ---------------------------------------------------------------------------
// Differentiable operators: autograd functions over the ones above, which they
// call through the dispatcher, so that a trace sees those.  The gradients are
// kernels' results and have none of their own (gradients()).
// ---------------------------------------------------------------------------
using c10::SymInt;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

template <typename Sig>
c10::TypedOperatorHandle<Sig> find(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Sig>();
}

// [..., D] as [N, D] with a contiguous last dimension and rows that do not overlap.
Tensor as_rows(const Tensor& t) {
  const Tensor r = t.dim() == 2 ? t : t.reshape_symint({SymInt(-1), t.sym_size(-1)});
  if ((r.sym_size(1) > 1 && r.sym_stride(1) != 1) || (r.sym_size(0) > 1 && r.sym_stride(0) < r.sym_size(1)))
    return r.contiguous();
  return r;
}

optional<Tensor> given(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : std::nullopt; }
optional<Tensor> contiguous(const optional<Tensor>& t) { return t.has_value() ? optional<Tensor>(t->contiguous()) : t; }

// The one element of a fresh tensor.  Autograd forbids its user to change a result
// of a function in place that is a view made inside the function; this one, as
// _unsafe_view elsewhere, counts as none, and nothing else holds its storage.
Tensor scalar(const Tensor& t) { return at::_unsafe_view(t, at::IntArrayRef()); }

// An operator's call without the dispatcher's autograd step, whose boxed "no derivative"
// kernel costs a few microseconds: an autograd function's forward and backward run
// with gradients off as they are.
template <typename F>
auto below_autograd(F&& call) {
  const at::AutoDispatchBelowAutograd guard;
  return call();
}

// Refuses a backward pass that is captured into a HIP graph where a gradient goes on to
// a node of the default stream: a leaf's, made before the capture and kept by another
// graph of the same leaves.  The engine would make the default stream wait for
// the capturing one, which a capture does not survive: its end ends the process.
void check_capture(at::ArrayRef<Tensor> grads) {
  for (const Tensor& grad : grads) {
    if (!grad.defined() || !grad.is_cuda()) continue;
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    const auto node = torch::autograd::get_current_node();
    if (!node) return;
    const c10::StreamId other = c10::hip::getDefaultHIPStream(grad.device().index()).id();
    for (size_t i = 0; i < node->num_outputs(); ++i) {
      if (!node->task_should_compute_output(i)) continue;  // not asked for: nothing goes there
      const auto at = node->next_edge(i).function->stream();
      TORCH_CHECK(!at.has_value() || at->id() != other,
                  "a backward pass cannot be captured into a graph while another graph of the same leaves lives: drop "
                  "the results of earlier steps, or make them on the stream that is captured");
    }
    return;
  }
}

// The body of a backward: the gradients are computed without a graph of their own.
// Where one is asked for (create_graph), they lead to what the function's inputs
// and its incoming gradients came from, through a node that raises.  Without it
// they would be constants where the operands saved are copies (of another type,
// of strided rows), and a penalty on them would be left out without a word.
template <typename F>
variable_list gradients(at::ArrayRef<Tensor> grads, F&& compute) {
  check_capture(grads);
  const bool twice = at::GradMode::is_enabled();
  variable_list out;
  {
    at::AutoGradMode off(false);
    out = compute();
  }
  if (!twice) return out;
  torch::autograd::edge_list edges;
  if (const auto node = torch::autograd::get_current_node()) edges = node->next_edges();
  for (const Tensor& grad : grads)
    if (grad.defined() && grad.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(grad));
  const auto error = std::make_shared<torch::autograd::Error>(
      "the gradients of chronicals_hip operators cannot be differentiated again", std::move(edges));
  const variable_list plain = out;
  for (size_t i = 0; i < out.size(); ++i) {
    if (!out[i].defined()) continue;
    size_t first = 0;
    while (!plain[first].is_same(plain[i])) ++first;
    if (first < i) {  // what was one tensor stays one
      out[i] = out[first];
      continue;
    }
    out[i] = plain[i].tensor_data();  // no view: it gets a graph
    torch::autograd::set_history(out[i], error);
  }
  return out;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& weight,
                        const optional<Tensor>& bias, double eps) {
    static const auto fwd =
        find<std::tuple<Tensor, Tensor, Tensor>(const Tensor&, const optional<Tensor>&, const optional<Tensor>&, double)>(
            "chronicals_hip::layer_norm_fwd");
    const Tensor rows = as_rows(x);
    const auto [y, mean, rstd] = fwd.call(rows, weight, bias, eps);
    ctx->save_for_backward({rows, weight.value_or(Tensor()), mean, rstd});
    const optional<Tensor>& p = weight.has_value() ? weight : bias;
    ctx->saved_data["param_f32"] = p.has_value() && p->scalar_type() == at::kFloat;
    ctx->saved_data["bias"] = bias.has_value();
    return x.dim() == 2 ? y : at::_unsafe_view_symint(y, x.sym_sizes());
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    static const auto bwd =
        find<std::tuple<Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const optional<Tensor>&, const Tensor&,
                                                const Tensor&, bool, bool, bool, bool)>("chronicals_hip::layer_norm_bwd");
    const auto saved = ctx->get_saved_variables();
    // absent inputs have no edge
    const bool has_w = saved[1].defined(), need_dx = ctx->needs_input_grad(0),
               need_dw = has_w && ctx->needs_input_grad(1),
               need_db = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(has_w ? 2 : 1);
    if (!need_dx && !need_dw && !need_db) return variable_list(4);
    return gradients(grads[0], [&]() -> variable_list {
      const Tensor g = grads[0].reshape_symint(saved[0].sym_sizes()).contiguous();
      const auto [dx, dw, db] = bwd.call(g, saved[0], given(saved[1]), saved[2], saved[3],
                                         ctx->saved_data["param_f32"].toBool(), need_dx, need_dw, need_db);
      return {need_dx ? dx.view_symint(grads[0].sym_sizes()) : Tensor(), need_dw ? dw : Tensor(),
              need_db ? db : Tensor(), Tensor()};
    });
  }
};

Tensor layer_norm(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias, double eps) {
  return LayerNorm::apply(x, contiguous(weight), contiguous(bias), eps);
}

// The teacher's tensors are contiguous [N, K], labels contiguous [N] or undefined.
struct DistillLogits : torch::autograd::Function<DistillLogits> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& t, const Tensor& index,
                        const optional<Tensor>& labels, double temperature, double distill_weight, double ce_weight,
                        int64_t ignore_index, int64_t reduction) {
    static const auto fwd =
        find<std::tuple<Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const optional<Tensor>&, double,
                                                double, double, SymInt, SymInt)>("chronicals_hip::distill_logits_fwd");
    const Tensor x = as_rows(logits);
    const auto [loss, stats, n_valid] =
        fwd.call(x, t, index, labels, temperature, distill_weight, ce_weight, ignore_index, reduction);
    ctx->save_for_backward({x, t, index, labels.value_or(Tensor()), stats, n_valid});
    ctx->saved_data["how"] = std::vector<double>{temperature, distill_weight, ce_weight};
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->saved_data["reduction"] = reduction;
    ctx->saved_data["dim"] = logits.dim();
    if (logits.dim() != 2) ctx->saved_data["shape"] = logits.sym_sizes();
    return reduction == CCE_REDUCTION_NONE ? loss : scalar(loss);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    static const auto bwd =
        find<Tensor(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const optional<Tensor>&, const Tensor&,
                    const Tensor&, double, double, double, SymInt, SymInt)>("chronicals_hip::distill_logits_bwd");
    if (!ctx->needs_input_grad(0)) return variable_list(9);
    return gradients(grads[0], [&] {
      variable_list out(9);
      const auto s = ctx->get_saved_variables();
      const auto how = ctx->saved_data["how"].toDoubleVector();
      out[0] = bwd.call(grads[0], s[0], s[1], s[2], given(s[3]), s[4], s[5], how[0], how[1], how[2],
                        ctx->saved_data["ignore_index"].toInt(), ctx->saved_data["reduction"].toInt());
      if (ctx->saved_data["dim"].toInt() != 2) out[0] = out[0].view_symint(ctx->saved_data["shape"].toSymIntVector());
      return out;
    });
  }
};

Tensor distill_logits(const Tensor& logits, const Tensor& t, const Tensor& index, const optional<Tensor>& labels,
                      double temperature, double distill_weight, double ce_weight, int64_t ignore_index,
                      int64_t reduction) {
  return DistillLogits::apply(logits, t, index, labels, temperature, distill_weight, ce_weight,
                              ignore_index, reduction);
}

struct DistillLinear : torch::autograd::Function<DistillLinear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const optional<Tensor>& bias,
                        const Tensor& t, const Tensor& index, const optional<Tensor>& labels, int64_t chunk_size,
                        double temperature, double distill_weight, double ce_weight, int64_t ignore_index,
                        int64_t reduction) {
    static const auto fwd = find<std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>(
        const Tensor&, const Tensor&, const optional<Tensor>&, const Tensor&, const Tensor&, const optional<Tensor>&, double,
        double, double, SymInt, SymInt)>("chronicals_hip::distill_fwd");
    // fp16 and fp32 operands are rounded to bf16, the GEMMs' type
    const Tensor h = as_rows(hidden).to(at::kBFloat16).contiguous(), w = weight.to(at::kBFloat16).contiguous();
    const Tensor b = bias.has_value() ? bias->to(at::kFloat).contiguous() : Tensor();
    const auto [loss, stats, entry_logits, rows, n_valid] = fwd.call(
        h, w, given(b), t, index, labels, temperature, distill_weight, ce_weight, ignore_index, reduction);
    ctx->save_for_backward({h, w, b, t, index, stats, entry_logits, rows, n_valid});
    ctx->saved_data["how"] = std::vector<double>{temperature, distill_weight, ce_weight};
    ctx->saved_data["reduction"] = reduction;
    ctx->saved_data["chunk_size"] = chunk_size;
    ctx->saved_data["shape"] = hidden.sym_sizes();
    ctx->saved_data["hidden"] = (int64_t)hidden.scalar_type();
    ctx->saved_data["weight"] = (int64_t)weight.scalar_type();
    if (bias.has_value()) ctx->saved_data["bias"] = (int64_t)bias->scalar_type();
    return reduction == CCE_REDUCTION_NONE ? loss : scalar(loss);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    static const auto bwd = find<std::tuple<Tensor, Tensor, Tensor>(
        const Tensor&, const Tensor&, const Tensor&, const optional<Tensor>&, const Tensor&, const Tensor&, const Tensor&,
        const Tensor&, const Tensor&, const Tensor&, double, double, double, SymInt, SymInt, bool, bool, bool, bool,
        bool)>("chronicals_hip::distill_bwd");
    const auto s = ctx->get_saved_variables();
    const bool need_dh = ctx->needs_input_grad(0), need_dw = ctx->needs_input_grad(1),
               need_db = s[2].defined() && ctx->needs_input_grad(2);
    if (!need_dh && !need_dw && !need_db) return variable_list(12);
    return gradients(grads[0], [&] {
      variable_list out(12);
      auto& kept = ctx->saved_data;
      const auto how = kept["how"].toDoubleVector();
      const auto htype = (at::ScalarType)kept["hidden"].toInt(), wtype = (at::ScalarType)kept["weight"].toInt();
      // bf16 inputs get bf16 gradients, fp16 and fp32 inputs get them from fp32
      const auto [dh, dw, db] =
          bwd.call(grads[0], s[0], s[1], given(s[2]), s[3], s[4], s[5], s[6], s[7], s[8], how[0], how[1], how[2],
                   kept["reduction"].toInt(), kept["chunk_size"].toInt(), need_dh, need_dw, need_db,
                   htype != at::kBFloat16, wtype != at::kBFloat16);
      if (need_dh) out[0] = dh.view_symint(kept["shape"].toSymIntVector()).to(htype);
      if (need_dw) out[1] = dw.to(wtype);
      if (need_db) out[2] = db.to((at::ScalarType)kept["bias"].toInt());
      return out;
    });
  }
};

Tensor distill_linear(const Tensor& hidden, const Tensor& weight, const optional<Tensor>& bias, const Tensor& t,
                      const Tensor& index, const optional<Tensor>& labels, int64_t chunk_size, double temperature,
                      double distill_weight, double ce_weight, int64_t ignore_index, int64_t reduction) {
  return DistillLinear::apply(hidden, weight, bias, t, index, labels, chunk_size, temperature, distill_weight, ce_weight, ignore_index, reduction);
}

// A result of N rows in the shape of the rows of x, whose last dimension is left out,
// followed by the result's own last one, if it has one.
Tensor shaped_rows(const Tensor& t, const Tensor& x) {
  if (x.dim() == 2) return t;
  auto shape = x.sym_sizes().vec();
  shape.pop_back();
  for (int64_t i = 1; i < t.dim(); ++i) shape.push_back(t.sym_size(i));
  return at::_unsafe_view_symint(t, shape);
}

typedef std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> FiveTensors;
typedef std::tuple<Tensor, Tensor, Tensor, Tensor> FourTensors;

// What the two functions below return: the alternatives carry no gradient, and the
// gradient that is not asked for stays undefined.
variable_list logprobs_results(AutogradContext* ctx, const FiveTensors& r, const Tensor& x) {
  const auto& [logprobs, entropy, stats, top_logprobs, top_indices] = r;
  variable_list out = {shaped_rows(logprobs, x), shaped_rows(entropy, x), shaped_rows(top_logprobs, x),
                       shaped_rows(top_indices, x)};
  ctx->mark_non_differentiable({out[2], out[3]});
  ctx->set_materialize_grads(false);
  return out;
}

// Tokens are contiguous [N].
struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  static const auto& op() {
    static const auto fwd =
        find<FiveTensors(const Tensor&, const Tensor&, double, SymInt, SymInt)>("chronicals_hip::token_logprobs_fwd");
    return fwd;
  }
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, double temperature,
                               int64_t top_k, int64_t ignore_index) {
    const Tensor x = as_rows(logits);
    const FiveTensors r = below_autograd([&] { return op().call(x, tokens, temperature, top_k, ignore_index); });
    ctx->save_for_backward({x, tokens, std::get<2>(r)});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->saved_data["dim"] = logits.dim();
    if (logits.dim() != 2) ctx->saved_data["shape"] = logits.sym_sizes();
    return logprobs_results(ctx, r, logits);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    static const auto bwd =
        find<Tensor(const optional<Tensor>&, const optional<Tensor>&, const Tensor&, const Tensor&, const Tensor&, double,
                    SymInt)>("chronicals_hip::token_logprobs_bwd");
    if (!ctx->needs_input_grad(0) || (!grads[0].defined() && !grads[1].defined())) return variable_list(5);
    return gradients({grads[0], grads[1]}, [&] {
      variable_list out(5);
      const auto s = ctx->get_saved_variables();
      out[0] = below_autograd([&] {
        return bwd.call(given(grads[0]), given(grads[1]), s[0], s[1], s[2], ctx->saved_data["temperature"].toDouble(),
                        ctx->saved_data["ignore_index"].toInt());
      });
      if (ctx->saved_data["dim"].toInt() != 2) out[0] = out[0].view_symint(ctx->saved_data["shape"].toSymIntVector());
      return out;
    });
  }
};

// t of another type; a call of torch's less where it has that one.
Tensor as_type(const Tensor& t, at::ScalarType type) { return t.scalar_type() == type ? t : t.to(type); }

// Whether a call is recorded for a backward.  One that is not goes to its operator as
// it is, without an autograd function's node (1 us of 7); the dispatcher's autograd
// step then refuses what the function would (forward-mode tensors).
bool recorded(const Tensor& a, const optional<Tensor>& b = std::nullopt, const optional<Tensor>& c = std::nullopt) {
  auto one = [](const optional<Tensor>& t) { return t.has_value() && t->requires_grad(); };
  return at::GradMode::is_enabled() && (a.requires_grad() || one(b) || one(c));
}

// The results of a forward that is not recorded.
FourTensors plain_results(const FiveTensors& r, const Tensor& x) {
  return {shaped_rows(std::get<0>(r), x), shaped_rows(std::get<1>(r), x), shaped_rows(std::get<3>(r), x),
          shaped_rows(std::get<4>(r), x)};
}

FourTensors token_logprobs(const Tensor& logits, const Tensor& tokens, double temperature, int64_t top_k,
                           int64_t ignore_index) {
  if (!recorded(logits))
    return plain_results(TokenLogprobs::op().call(as_rows(logits), tokens, temperature, top_k, ignore_index), logits);
  const auto r = TokenLogprobs::apply(logits, tokens, temperature, top_k, ignore_index);
  return {r[0], r[1], r[2], r[3]};
}

// fp16 and fp32 operands of the head are rounded to bf16, the GEMMs' type.
Tensor head_rows(const Tensor& hidden) { return as_type(as_rows(hidden), at::kBFloat16).contiguous(); }
Tensor head_weight(const Tensor& weight) { return as_type(weight, at::kBFloat16).contiguous(); }
Tensor head_bias(const optional<Tensor>& bias) {
  return bias.has_value() ? as_type(*bias, at::kFloat).contiguous() : Tensor();
}

struct LinearTokenLogprobs : torch::autograd::Function<LinearTokenLogprobs> {
  static const auto& op() {
    static const auto fwd = find<FiveTensors(const Tensor&, const Tensor&, const optional<Tensor>&, const Tensor&, double,
                                             SymInt, SymInt)>("chronicals_hip::linear_token_logprobs_fwd");
    return fwd;
  }
  static variable_list forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight,
                               const optional<Tensor>& bias, const Tensor& tokens, int64_t chunk_size, double temperature,
                               int64_t top_k, int64_t ignore_index) {
    const Tensor h = head_rows(hidden), w = head_weight(weight), b = head_bias(bias);
    const FiveTensors r =
        below_autograd([&] { return op().call(h, w, given(b), tokens, temperature, top_k, ignore_index); });
    ctx->save_for_backward({h, w, b, tokens, std::get<2>(r)});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->saved_data["chunk_size"] = chunk_size;
    if (hidden.dim() != 2) ctx->saved_data["shape"] = hidden.sym_sizes();
    ctx->saved_data["dim"] = hidden.dim();
    ctx->saved_data["hidden"] = (int64_t)hidden.scalar_type();
    ctx->saved_data["weight"] = (int64_t)weight.scalar_type();
    if (bias.has_value()) ctx->saved_data["bias"] = (int64_t)bias->scalar_type();
    return logprobs_results(ctx, r, hidden);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    static const auto bwd = find<std::tuple<Tensor, Tensor, Tensor>(
        const optional<Tensor>&, const optional<Tensor>&, const Tensor&, const Tensor&, const optional<Tensor>&,
        const Tensor&, const Tensor&, double, SymInt, SymInt, bool, bool, bool, bool, bool)>(
        "chronicals_hip::linear_token_logprobs_bwd");
    const auto s = ctx->get_saved_variables();
    const bool need_dh = ctx->needs_input_grad(0), need_dw = ctx->needs_input_grad(1),
               need_db = s[2].defined() && ctx->needs_input_grad(2);
    if ((!need_dh && !need_dw && !need_db) || (!grads[0].defined() && !grads[1].defined())) return variable_list(8);
    return gradients({grads[0], grads[1]}, [&] {
      variable_list out(8);
      auto& kept = ctx->saved_data;
      const auto htype = (at::ScalarType)kept["hidden"].toInt(), wtype = (at::ScalarType)kept["weight"].toInt();
      // bf16 inputs get bf16 gradients, fp16 and fp32 inputs get them from fp32
      const auto [dh, dw, db] = below_autograd([&] {
        return bwd.call(given(grads[0]), given(grads[1]), s[0], s[1], given(s[2]), s[3], s[4],
                        kept["temperature"].toDouble(), kept["ignore_index"].toInt(), kept["chunk_size"].toInt(), need_dh,
                        need_dw, need_db, htype != at::kBFloat16, wtype != at::kBFloat16);
      });
      if (need_dh)
        out[0] = as_type(kept["dim"].toInt() == 2 ? dh : dh.view_symint(kept["shape"].toSymIntVector()), htype);
      if (need_dw) out[1] = as_type(dw, wtype);
      if (need_db) out[2] = as_type(db, (at::ScalarType)kept["bias"].toInt());
      return out;
    });
  }
};

FourTensors linear_token_logprobs(const Tensor& hidden, const Tensor& weight, const optional<Tensor>& bias,
                                  const Tensor& tokens, int64_t chunk_size, double temperature, int64_t top_k,
                                  int64_t ignore_index) {
  if (!recorded(hidden, weight, bias))
    return plain_results(LinearTokenLogprobs::op().call(head_rows(hidden), head_weight(weight), given(head_bias(bias)),
                                                        tokens, temperature, top_k, ignore_index),
                         hidden);
  const auto r =
      LinearTokenLogprobs::apply(hidden, weight, bias, tokens, chunk_size, temperature, top_k, ignore_index);
  return {r[0], r[1], r[2], r[3]};
}

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static const auto& op() {
    static const auto fwd = find<std::tuple<Tensor, Tensor, Tensor>(const Tensor&, const optional<Tensor>&,
                                                                    const optional<Tensor>&, double)>(
        "chronicals_hip::rms_norm_fwd");
    return fwd;
  }
  static Tensor shaped(const Tensor& t, const Tensor& x) {
    return x.dim() == 2 ? t : at::_unsafe_view_symint(t, x.sym_sizes());
  }
  // y and the sum, which is empty without a residual
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& weight,
                               const optional<Tensor>& residual, double eps) {
    const Tensor rows = as_rows(x);
    const bool has_r = residual.has_value();
    const optional<Tensor> r = has_r ? optional<Tensor>(as_rows(*residual)) : residual;
    const auto [y, sum, rstd] = below_autograd([&] { return op().call(rows, weight, r, eps); });
    variable_list out = {shaped(y, x), has_r ? shaped(sum, x) : sum};
    ctx->save_for_backward({has_r ? out[1] : rows, weight.value_or(Tensor()), rstd});
    ctx->saved_data["residual"] = has_r;
    ctx->saved_data["same"] = has_r && residual->scalar_type() == x.scalar_type();
    ctx->saved_data["x"] = (int64_t)x.scalar_type();
    if (!has_r) ctx->mark_non_differentiable({out[1]});
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    static const auto bwd = find<std::tuple<Tensor, Tensor, Tensor>(
        const Tensor&, const optional<Tensor>&, const Tensor&, const optional<Tensor>&, const Tensor&, bool, bool, bool,
        bool)>("chronicals_hip::rms_norm_bwd");
    const auto saved = ctx->get_saved_variables();
    auto& kept = ctx->saved_data;
    // absent inputs have no edge
    const bool has_w = saved[1].defined(), has_r = kept["residual"].toBool(), same = kept["same"].toBool(),
               need_x = ctx->needs_input_grad(0), need_dw = has_w && ctx->needs_input_grad(1),
               need_r = has_r && ctx->needs_input_grad(has_w ? 2 : 1);
    if ((!need_x && !need_dw && !need_r) || (!grads[0].defined() && !grads[1].defined())) return variable_list(4);
    return gradients({grads[0], grads[1]}, [&]() -> variable_list {
      const Tensor& like = grads[0].defined() ? grads[0] : grads[1];
      const Tensor sum = as_rows(saved[0]);
      auto rows = [&](const Tensor& t) {
        return (t.dim() == 2 ? t : t.reshape_symint(sum.sym_sizes())).contiguous();
      };
      const Tensor g = grads[0].defined()
                           ? rows(grads[0])
                           : at::zeros_symint(sum.sym_sizes(), sum.options().dtype((at::ScalarType)kept["x"].toInt()));
      const optional<Tensor> gs = grads[1].defined() ? optional<Tensor>(rows(grads[1])) : std::nullopt;
      const auto [dx, dr, dw] = below_autograd([&] {
        return bwd.call(g, gs, sum, given(saved[1]), saved[2], has_w && saved[1].scalar_type() == at::kFloat,
                        need_x || (need_r && same), need_r && !same, need_dw);
      });
      auto out = [&](const Tensor& t) { return like.dim() == 2 ? t : t.view_symint(like.sym_sizes()); };
      // Of one type the two gradients are one tensor, as an addition's are.  It has to be one
      // object: its two owners are how the engine knows that a leaf's .grad needs a copy (two
      // views of one storage would each pass for a tensor that nobody else has).
      const Tensor gx = need_x || (need_r && same) ? out(dx) : Tensor();
      return {need_x ? gx : Tensor(), need_dw ? dw : Tensor(), need_r ? (same ? gx : out(dr)) : Tensor(), Tensor()};
    });
  }
};

std::tuple<Tensor, Tensor> rms_norm(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& residual,
                                    double eps) {
  if (!recorded(x, weight, residual)) {
    const auto [y, sum, rstd] = RmsNorm::op().call(
        as_rows(x), contiguous(weight), residual.has_value() ? optional<Tensor>(as_rows(*residual)) : residual, eps);
    return {RmsNorm::shaped(y, x), residual.has_value() ? RmsNorm::shaped(sum, x) : sum};
  }
  const auto r = RmsNorm::apply(x, contiguous(weight), residual, eps);
  return {r[0], r[1]};
}

}  // namespace

extern "C" {

// Takes the C functions from an open libchronicals_cce; 0 when it has them all.
int chronicals_torch_bind(void* handle) {
  Api a;
  bool ok = true;
  auto get = [&](auto& fn, const char* name) {
    fn = reinterpret_cast<std::decay_t<decltype(fn)>>(dlsym(handle, name));
    ok = ok && fn != nullptr;
  };
  get(a.last_error, "cce_last_error");
  get(a.forward_workspace_bytes, "cce_forward_workspace_bytes");
  get(a.backward_workspace_bytes, "cce_backward_workspace_bytes");
  get(a.forward, "cce_forward");
  get(a.backward, "cce_backward");
  get(a.logits_forward_workspace_bytes, "cce_logits_forward_workspace_bytes");
  get(a.logits_forward, "cce_logits_forward");
  get(a.logits_backward, "cce_logits_backward");
  get(a.logits_forward_backward, "cce_logits_forward_backward");
  get(a.distill_logits_workspace_bytes, "cce_distill_logits_workspace_bytes");
  get(a.distill_logits_forward, "cce_distill_logits_forward");
  get(a.distill_logits_backward, "cce_distill_logits_backward");
  get(a.distill_forward_workspace_bytes, "cce_distill_forward_workspace_bytes");
  get(a.distill_forward, "cce_distill_forward");
  get(a.distill_backward_workspace_bytes, "cce_distill_backward_workspace_bytes");
  get(a.distill_backward, "cce_distill_backward");
  get(a.top_logits_workspace_bytes, "cce_top_logits_workspace_bytes");
  get(a.top_logits, "cce_top_logits");
  get(a.layer_norm_forward, "cce_layer_norm_forward");
  get(a.layer_norm_backward_workspace_bytes_for, "cce_layer_norm_backward_workspace_bytes_for");
  get(a.layer_norm_backward, "cce_layer_norm_backward");
  get(a.token_logprobs_workspace_bytes, "cce_token_logprobs_workspace_bytes");
  get(a.token_logprobs_forward, "cce_token_logprobs_forward");
  get(a.token_logprobs_backward, "cce_token_logprobs_backward");
  get(a.linear_token_logprobs_workspace_bytes, "cce_linear_token_logprobs_workspace_bytes");
  get(a.linear_token_logprobs_forward, "cce_linear_token_logprobs_forward");
  get(a.linear_token_logprobs_backward_workspace_bytes, "cce_linear_token_logprobs_backward_workspace_bytes");
  get(a.linear_token_logprobs_backward, "cce_linear_token_logprobs_backward");
  get(a.rms_norm_forward, "cce_rms_norm_forward");
  get(a.rms_norm_quantized, "cce_rms_norm_quantized");
  get(a.rms_norm_backward_workspace_bytes, "cce_rms_norm_backward_workspace_bytes");
  get(a.rms_norm_backward, "cce_rms_norm_backward");
  if (!ok) return 1;
  if (!g_bound.load(std::memory_order_acquire)) {
    g_api = a;
    g_bound.store(true, std::memory_order_release);
  }
  return 0;
}

// The Python callables of api() and check(); called with the interpreter's lock.
void chronicals_torch_hooks(PyObject* load, PyObject* check) {
  Py_XINCREF(load);
  Py_XINCREF(check);
  Py_XSETREF(g_load, load);
  Py_XSETREF(g_check, check);
}

}  // extern "C"

// HIP tensors carry the CUDA dispatch key in torch.
TORCH_LIBRARY_IMPL(chronicals_hip, CUDA, m) {
  m.impl("cce_fwd", cce_fwd);
  m.impl("cce_bwd", cce_bwd);
  m.impl("ce_logits_fwd", ce_logits_fwd);
  m.impl("ce_logits_bwd", ce_logits_bwd);
  m.impl("ce_logits_fwd_bwd", ce_logits_fwd_bwd);
  m.impl("distill_logits_fwd", distill_logits_fwd);
  m.impl("distill_logits_bwd", distill_logits_bwd);
  m.impl("distill_fwd", distill_fwd);
  m.impl("distill_bwd", distill_bwd);
  m.impl("top_logits", top_logits);
  m.impl("layer_norm_fwd", layer_norm_fwd);
  m.impl("layer_norm_bwd", layer_norm_bwd);
  m.impl("token_logprobs_fwd", token_logprobs_fwd);
  m.impl("token_logprobs_bwd", token_logprobs_bwd);
  m.impl("linear_token_logprobs_fwd", linear_token_logprobs_fwd);
  m.impl("linear_token_logprobs_bwd", linear_token_logprobs_bwd);
  m.impl("rms_norm_fwd", rms_norm_fwd);
  m.impl("rms_norm_quantized", rms_norm_quantized);
  m.impl("rms_norm_bwd", rms_norm_bwd);
}

TORCH_LIBRARY_IMPL(chronicals_hip, CompositeImplicitAutograd, m) {
  m.impl("layer_norm", layer_norm);
  m.impl("distill_logits", distill_logits);
  m.impl("distill_linear", distill_linear);
  m.impl("token_logprobs", token_logprobs);
  m.impl("linear_token_logprobs", linear_token_logprobs);
  m.impl("rms_norm", rms_norm);
}

// The operators on HIP tensors have no derivative of their own (the autograd functions call
// them): a backward through one raises.
TORCH_LIBRARY_IMPL(chronicals_hip, Autograd, m) {
  for (const char* op : {"cce_fwd", "cce_bwd", "ce_logits_fwd", "ce_logits_bwd", "ce_logits_fwd_bwd",
                         "distill_logits_fwd", "distill_logits_bwd", "distill_fwd", "distill_bwd", "top_logits",
                         "layer_norm_fwd", "layer_norm_bwd", "token_logprobs_fwd", "token_logprobs_bwd",
                         "linear_token_logprobs_fwd", "linear_token_logprobs_bwd", "rms_norm_fwd", "rms_norm_quantized",
                         "rms_norm_bwd"})
    m.impl(op, torch::autograd::autogradNotImplementedFallback());
}
