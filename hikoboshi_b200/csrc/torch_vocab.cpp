// Python module hikoboshi_b200._vocab: torch tensors to the C entry points of
// the operators on vocabulary rows (vocab.py documents the calls).
//
// A call of these operators takes a few microseconds on the device, so what
// counts as much is the work on the host: the checks, the outputs' allocation
// and autograd's nodes are here in C++ (a sampling call: 7 us; through ctypes
// and Python checks it was 21 us).  Errors are raised as the package's HkbError.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <optional>
#include <string>

#include "hkb_mpnn.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

PyObject* g_error = nullptr;  // hikoboshi_b200.HkbError

struct Refusal {
  int code;
  std::string detail;
};

[[noreturn]] void refuse(std::string why, int code = HKB_INVALID_ARGUMENT) {
  throw Refusal{code, std::move(why)};
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return HKB_F32;
    case at::kHalf: return HKB_F16;
    case at::kBFloat16: return HKB_BF16;
    default: return -1;
  }
}

// Number and common stride of the dimensions taken as one; false if they have
// none.
bool flatten(at::IntArrayRef size, at::IntArrayRef stride, int64_t* n, int64_t* step) {
  int64_t count = 1, st = 0;
  bool one = true;
  for (size_t d = size.size(); d-- > 0;) {
    if (size[d] == 1) continue;
    if (count == 1) st = stride[d];
    else if (stride[d] != st * count) one = false;
    count *= size[d];
  }
  *n = count;
  *step = count ? st : 0;
  return one || count == 0;
}

// [.., V] logits as the library takes them; never a copy.
hkb_vocab_rows rows_of(const Tensor& x, const char* name) {
  const int code = dtype_code(x.scalar_type());
  const std::string n = name;
  if (code < 0) refuse(n + " must be float32, float16 or bfloat16");
  if (x.dim() == 0 || x.size(-1) == 0)
    refuse(n + " must have a last dimension of at least one token");
  if (x.layout() != at::kStrided || x.is_neg()) refuse(n + " must be a plain strided tensor");
  const int64_t v = x.size(-1);
  if (v > 1 && x.stride(-1) != 1) refuse(n + " must have a last dimension of stride 1");
  const size_t lead = (size_t)x.dim() - 1;
  int64_t count, step;
  if (!flatten(x.sizes().slice(0, lead), x.strides().slice(0, lead), &count, &step))
    refuse(n + ": the leading dimensions must flatten to rows of one stride");
  hkb_vocab_rows r{};
  r.rows = count;
  r.vocab = (int32_t)std::min<int64_t>(v, INT32_MAX);
  r.dtype = code;
  r.logits = x.const_data_ptr();
  r.row_stride = count > 1 ? step : v;
  return r;
}

at::IntArrayRef lead_of(const Tensor& x) { return x.sizes().slice(0, (size_t)x.dim() - 1); }

// A dense per-row tensor.
const void* per_row(const Tensor& x, const Tensor& like, std::initializer_list<at::ScalarType> types,
                    const char* type_text, const char* name) {
  const std::string n = name;
  if (x.device() != like.device()) refuse(n + " must be on the logits' device");
  if (std::find(types.begin(), types.end(), x.scalar_type()) == types.end())
    refuse(n + " must be " + type_text);
  if (x.sizes() != lead_of(like)) refuse(n + " must have one number per row");
  if (!x.is_contiguous() || x.is_neg()) refuse(n + " must be contiguous");
  return x.const_data_ptr();
}

hkb_distill_teacher teacher_of(const Tensor& x, const Tensor& values, const Tensor& tokens,
                               const std::optional<Tensor>& log_norm, double temperature) {
  hkb_distill_teacher t{};
  t.dtype = dtype_code(values.scalar_type());
  if (t.dtype < 0) refuse("teacher_values must be float32, float16 or bfloat16");
  if (tokens.scalar_type() != at::kInt) refuse("teacher_tokens must be int32");
  if (values.dim() == 0 || lead_of(values) != lead_of(x) || tokens.sizes() != values.sizes())
    refuse("teacher_values and teacher_tokens must be [.., k] with the logits' rows");
  if (values.device() != x.device()) refuse("teacher_values must be on the logits' device");
  if (tokens.device() != x.device()) refuse("teacher_tokens must be on the logits' device");
  if (!values.is_contiguous() || !tokens.is_contiguous() || values.is_neg())
    refuse("teacher_values and teacher_tokens must be contiguous");
  t.k = (int32_t)std::min<int64_t>(values.size(-1), INT32_MAX);
  t.values = values.const_data_ptr();
  t.tokens = tokens.const_data_ptr<int32_t>();
  if (log_norm)
    t.log_norm = static_cast<const float*>(
        per_row(*log_norm, x, {at::kFloat}, "float32", "teacher_log_norm"));
  t.temperature = (float)temperature;
  return t;
}

void set_weights(hkb_distill_out* o, const Tensor& w, const Tensor& x) {
  if (w.device() != x.device()) refuse("row_weights must be on the logits' device");
  if (w.scalar_type() != at::kFloat) refuse("row_weights must be float32");
  if (w.sizes() != lead_of(x)) refuse("row_weights must have one number per row");
  int64_t n;
  if (!flatten(w.sizes(), w.strides(), &n, &o->row_weight_stride) || w.is_neg())
    refuse("row_weights must flatten to one stride");
  o->row_weights = w.const_data_ptr<float>();
}

// call(device, stream) on the logits' device and its current stream.
template <typename F>
void run(const Tensor& x, F call) {
  const bool cuda = x.is_cuda();
  // without a device the library checks the other arguments, then refuses it
  const int device = cuda ? x.get_device() : -1;
  void* stream = cuda ? (void*)c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream()
                      : nullptr;
  hkb_status s;
  {
    // autograd's threads come here without the interpreter's lock
    std::optional<pybind11::gil_scoped_release> open;
    if (PyGILState_Check()) open.emplace();
    s = call(device, stream);
  }
  if (s.code == HKB_OK) return;
  if (!cuda && s.code == HKB_INVALID_ARGUMENT &&
      std::string(s.detail) == "device ordinal out of range")
    refuse("logits must be on a CUDA device");
  refuse(s.detail, s.code);
}

bool capturing(const Tensor& x) {
  return x.is_cuda() &&
         c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None;
}

// The loss; `stats`, if given, receives what a backward pass needs.
Tensor loss_only(const Tensor& x, const Tensor& values, const Tensor& tokens,
                 const std::optional<Tensor>& log_norm, double temperature, Tensor* stats) {
  const hkb_vocab_rows rows = rows_of(x, "logits");
  const hkb_distill_teacher t = teacher_of(x, values, tokens, log_norm, temperature);
  Tensor loss = at::empty(lead_of(x), x.options().dtype(at::kFloat));
  hkb_distill_out o{};
  o.loss = loss.data_ptr<float>();
  if (stats) {
    *stats = at::empty({rows.rows, HKB_DISTILL_STATS}, x.options().dtype(at::kDouble));
    o.stats = stats->data_ptr<double>();
  }
  run(x, [&](int d, void* st) { return hkb_distill(d, &rows, &t, &o, st); });
  return loss;
}

// Autograd's threads take the refusal of a backward pass as a C++ exception.
struct DistillLoss : torch::autograd::Function<DistillLoss> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& values,
                        const Tensor& tokens, const std::optional<Tensor>& log_norm,
                        double temperature) {
    Tensor stats, loss;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      loss = loss_only(x, values, tokens, log_norm, temperature, &stats);
    }
    ctx->save_for_backward({x, values, tokens, log_norm ? *log_norm : Tensor(), stats});
    ctx->saved_data["temperature"] = temperature;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor& x = saved[0];
    const std::optional<Tensor> norm =
        saved[3].defined() ? std::optional<Tensor>(saved[3]) : std::nullopt;
    Tensor w = grads[0];
    if (!w.defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    TORCH_CHECK(!(at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad())),
                "distill_loss is differentiable once: its gradient has none");
    // the forward pass was not captured, so an eager graph of the same leaves
    // lives: to accumulate their gradients would break the capture
    TORCH_CHECK(!capturing(x), "distill_loss backward: autograd through distill_loss cannot be "
                               "captured; capture distill_loss_and_grad");
    int64_t n, step;
    if (w.is_neg() || !flatten(w.sizes(), w.strides(), &n, &step))
      w = w.resolve_neg().contiguous();
    try {
      const hkb_vocab_rows rows = rows_of(x, "logits");
      const hkb_distill_teacher t =
          teacher_of(x, saved[1], saved[2], norm, ctx->saved_data["temperature"].toDouble());
      Tensor grad = at::empty(x.sizes(), x.options());
      hkb_distill_out o{};
      set_weights(&o, w, x);
      o.grad = grad.data_ptr();
      o.grad_row_stride = x.size(-1);
      Tensor stats = saved[4];
      o.stats = stats.data_ptr<double>();
      run(x, [&](int d, void* st) { return hkb_distill_backward(d, &rows, &t, &o, st); });
      return {grad, Tensor(), Tensor(), Tensor(), Tensor()};
    } catch (const Refusal& r) {
      TORCH_CHECK(false, "distill_loss backward: ", r.detail);
    }
  }
};

// ---- arguments -----------------------------------------------------------------

const Tensor& tensor_arg(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}

std::optional<Tensor> optional_arg(PyObject* o, const char* name) {
  if (o == Py_None) return std::nullopt;
  return tensor_arg(o, name);
}

double number_arg(PyObject* o, const char* name) {
  if (PyFloat_Check(o)) return PyFloat_AS_DOUBLE(o);
  if (PyLong_Check(o) && !PyBool_Check(o)) {
    const double v = PyLong_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      refuse(std::string(name) + " is out of range");
    }
    return v;
  }
  refuse(std::string(name) + " must be a number or a tensor of one number per row");
}

// A whole number, cut to the range of 32 bits (what lies outside is refused).
int32_t whole_arg(PyObject* o, const char* what) {
  if (!PyLong_Check(o) || PyBool_Check(o)) refuse(what);
  int overflow = 0;
  const long long v = PyLong_AsLongLongAndOverflow(o, &overflow);
  if (overflow > 0 || v > INT32_MAX) return INT32_MAX;
  if (overflow < 0 || v < -1) return -1;
  return (int32_t)v;
}

// Runs f and hands its refusal, or what torch throws, to Python.
template <typename F>
PyObject* guarded(F f) {
  HANDLE_TH_ERRORS
  try {
    return f();
  } catch (const Refusal& r) {
    PyObject* args = Py_BuildValue("(is)", r.code, r.detail.c_str());
    if (args) {
      PyObject* e = PyObject_CallObject(g_error, args);
      Py_DECREF(args);
      if (e) {
        PyErr_SetObject(g_error, e);
        Py_DECREF(e);
      }
    }
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

bool arity(Py_ssize_t got, Py_ssize_t want) {
  if (got == want) return true;
  PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, got);
  return false;
}

PyObject* tuple_of(std::initializer_list<Tensor> ts) {
  PyObject* t = PyTuple_New((Py_ssize_t)ts.size());
  if (!t) return nullptr;
  Py_ssize_t i = 0;
  for (const Tensor& x : ts) PyTuple_SET_ITEM(t, i++, THPVariable_Wrap(x));
  return t;
}

// sample(logits, uniforms, temperature, top_k, top_p, min_p)
PyObject* sample(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!arity(n, 6)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Tensor& x = tensor_arg(args[0], "logits");
    const hkb_vocab_rows rows = rows_of(x, "logits");
    const Tensor& u = tensor_arg(args[1], "uniforms");
    hkb_sample_settings s{};
    s.uniforms = per_row(u, x, {at::kFloat, at::kDouble}, "float32 or float64", "uniforms");
    s.uniforms_dtype = u.scalar_type() == at::kDouble ? HKB_F64 : HKB_F32;
    auto setting = [&](PyObject* o, const char* name, const float** array, float* number) {
      if (THPVariable_Check(o))
        *array = static_cast<const float*>(
            per_row(THPVariable_Unpack(o), x, {at::kFloat}, "float32", name));
      else
        *number = (float)number_arg(o, name);
    };
    setting(args[2], "temperature", &s.temperatures, &s.temperature);
    if (THPVariable_Check(args[3]))
      s.top_ks = static_cast<const int32_t*>(
          per_row(THPVariable_Unpack(args[3]), x, {at::kInt}, "int32", "top_k"));
    else
      s.top_k = whole_arg(args[3], "top_k must be a whole number or a tensor of one per row");
    setting(args[4], "top_p", &s.top_ps, &s.top_p);
    setting(args[5], "min_p", &s.min_ps, &s.min_p);
    const auto lead = lead_of(x);
    Tensor tokens = at::empty(lead, x.options().dtype(at::kInt));
    Tensor log_probs = at::empty(lead, x.options().dtype(at::kFloat));
    Tensor kept = at::empty(lead, x.options().dtype(at::kInt));
    const hkb_sample_out o{tokens.data_ptr<int32_t>(), log_probs.data_ptr<float>(),
                           kept.data_ptr<int32_t>()};
    run(x, [&](int d, void* st) { return hkb_sample_tokens(d, &rows, &s, &o, st); });
    return tuple_of({tokens, log_probs, kept});
  });
}

// top(logits, k, temperature)
PyObject* top(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!arity(n, 3)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Tensor& x = tensor_arg(args[0], "logits");
    const hkb_vocab_rows rows = rows_of(x, "logits");
    const int32_t k = whole_arg(args[1], "k must be a whole number");
    const double temperature = number_arg(args[2], "temperature");
    std::vector<int64_t> shape = lead_of(x).vec();
    shape.push_back(std::clamp<int64_t>(k, 0, HKB_LISTING_MAX));
    Tensor values = at::empty(shape, x.options());
    Tensor tokens = at::empty(shape, x.options().dtype(at::kInt));
    Tensor norm = at::empty(lead_of(x), x.options().dtype(at::kFloat));
    const hkb_top_out o{values.data_ptr(), tokens.data_ptr<int32_t>(), norm.data_ptr<float>()};
    run(x, [&](int d, void* st) {
      return hkb_top_logits(d, &rows, k, (float)temperature, &o, st);
    });
    return tuple_of({values, tokens, norm});
  });
}

// loss(logits, values, tokens, log_norm, temperature)
PyObject* loss(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!arity(n, 5)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Tensor& x = tensor_arg(args[0], "logits");
    const Tensor& values = tensor_arg(args[1], "teacher_values");
    const Tensor& tokens = tensor_arg(args[2], "teacher_tokens");
    const std::optional<Tensor> norm = optional_arg(args[3], "teacher_log_norm");
    const double temperature = number_arg(args[4], "temperature");
    // without this a tangent would be dropped
    if (x._fw_grad(0).defined()) refuse("distill_loss has no forward-mode derivative");
    if (!(x.requires_grad() && at::GradMode::is_enabled()))
      return THPVariable_Wrap(loss_only(x, values, tokens, norm, temperature, nullptr));
    if (capturing(x))
      refuse("autograd through distill_loss cannot be captured; capture distill_loss_and_grad",
             HKB_FAILED_PRECONDITION);
    return THPVariable_Wrap(DistillLoss::apply(x, values, tokens, norm, temperature));
  });
}

// loss_and_grad(logits, values, tokens, log_norm, temperature, row_weights, grad_out)
PyObject* loss_and_grad(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (!arity(n, 7)) return nullptr;
  return guarded([&]() -> PyObject* {
    at::NoGradGuard no_grad;
    const Tensor& x = tensor_arg(args[0], "logits");
    const hkb_vocab_rows rows = rows_of(x, "logits");
    const hkb_distill_teacher t =
        teacher_of(x, tensor_arg(args[1], "teacher_values"), tensor_arg(args[2], "teacher_tokens"),
                   optional_arg(args[3], "teacher_log_norm"), number_arg(args[4], "temperature"));
    hkb_distill_out o{};
    const std::optional<Tensor> w = optional_arg(args[5], "row_weights");
    if (w) set_weights(&o, *w, x);
    std::optional<Tensor> grad = optional_arg(args[6], "grad_out");
    if (grad) {
      if (grad->device() != x.device()) refuse("grad_out must be on the logits' device");
      if (grad->scalar_type() != x.scalar_type() || grad->sizes() != x.sizes())
        refuse("grad_out must have the logits' type and shape");
      o.grad_row_stride = rows_of(*grad, "grad_out").row_stride;
    } else {
      grad = at::empty(x.sizes(), x.options());
      o.grad_row_stride = x.size(-1);
    }
    Tensor loss = at::empty(lead_of(x), x.options().dtype(at::kFloat));
    o.loss = loss.data_ptr<float>();
    o.grad = grad->data_ptr();
    run(x, [&](int d, void* st) { return hkb_distill(d, &rows, &t, &o, st); });
    // autograd refuses a backward pass that needs what was here before
    if (args[6] != Py_None && !grad->is_inference())
      grad->unsafeGetTensorImpl()->bump_version();
    return tuple_of({loss, *grad});
  });
}

PyMethodDef g_methods[] = {
    {"sample", (PyCFunction)(void (*)())sample, METH_FASTCALL, nullptr},
    {"top", (PyCFunction)(void (*)())top, METH_FASTCALL, nullptr},
    {"loss", (PyCFunction)(void (*)())loss, METH_FASTCALL, nullptr},
    {"loss_and_grad", (PyCFunction)(void (*)())loss_and_grad, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_vocab", nullptr, -1, g_methods};

}  // namespace

PyMODINIT_FUNC PyInit__vocab() {
  PyObject* lib = PyImport_ImportModule("hikoboshi_b200._lib");
  if (!lib) return nullptr;
  g_error = PyObject_GetAttrString(lib, "HkbError");
  Py_DECREF(lib);
  if (!g_error) return nullptr;
  return PyModule_Create(&g_module);
}
