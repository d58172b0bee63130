// host.cpp — liftreg_amd._host: the host side of the ops whose calls are shorter than a microsecond-by-microsecond Python front end
// (liftreg_amd/optim.py over lists of tensors, ops.layer_norm on a few rows): argument checks, outputs and workspaces, the call of
// the C entry.  In Python the checks alone cost 0.3 us a tensor, and 18 tensors' AdamW step 32 us around 9 us of kernels.
// Plain C++ against torch's headers, no GPU code; the C entries come from the loaded libliftreg_hip (bind()).
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>

#include <algorithm>
#include <deque>
#include <string>
#include <utility>
#include <vector>

#include "../../include/liftreg_hip.h"

namespace {

struct Set {};      // a Python error has been set

// the library's entries, by the addresses that bind() was given (in this order)
struct Entries {
  decltype(&lr_strerror) strerror_;
  decltype(&lr_layer_norm_resident_cols) resident;
  decltype(&lr_layer_norm_workspace) workspace;
  decltype(&lr_layer_norm) norm;
  decltype(&lr_layer_norm_bwd) norm_bwd;
  decltype(&lr_grad_norm_partials) partials;
  decltype(&lr_grad_norm) grad_norm;
  decltype(&lr_adamw_step) adamw;
} lr;
PyObject* hip_error = nullptr;      // liftreg_amd._hip.LiftRegHipError
PyObject* raw_stream = nullptr;     // torch._C._cuda_getCurrentRawStream

[[noreturn]] void fail(PyObject* kind, const std::string& text) {
  PyErr_SetString(kind, text.c_str());
  throw Set();
}
void check(int rc, const char* what) {
  if (rc != LR_OK) fail(hip_error, std::string(what) + ": " + lr.strerror_(rc) + " (" + std::to_string(rc) + ")");
}
int64_t count(int64_t n, const char* what) {
  if (n < 0) check(static_cast<int>(n), what);
  return n;
}

std::string shape_of(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + (t.dim() == 1 ? ",)" : ")");
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) fail(PyExc_TypeError, std::string(name) + ": expected a torch.Tensor, got " + Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
void on_gpu(const at::Tensor& t, const char* name) {
  if (!t.is_cuda() || t.layout() != at::kStrided)
    fail(hip_error, std::string(name) + ": tensor is on " + t.device().str() + "; liftreg_amd ops run on the GPU only (no CPU fallback)");
}
void of_type(const at::Tensor& t, at::ScalarType want, const char* name) {
  if (t.scalar_type() != want)
    fail(PyExc_TypeError, std::string(name) + ": expected " + c10::toString(want) + ", got " + c10::toString(t.scalar_type()));
}
void float_or_bf16(const at::Tensor& t, const char* name) {
  if (t.scalar_type() != at::kFloat && t.scalar_type() != at::kBFloat16)
    fail(PyExc_TypeError, std::string(name) + ": expected float32 or bfloat16, got " + c10::toString(t.scalar_type()));
}

double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Set();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Set();
  return v;
}
void* stream_of(c10::DeviceIndex device) {
  PyObject* index = PyLong_FromLong(device);
  PyObject* s = index ? PyObject_CallOneArg(raw_stream, index) : nullptr;
  Py_XDECREF(index);
  if (!s) throw Set();
  void* p = PyLong_AsVoidPtr(s);
  Py_DECREF(s);
  if (!p && PyErr_Occurred()) throw Set();
  return p;
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, const at::Device& device) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(device));
}
void* data(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// an entry's frame: no C++ exception leaves it, and nothing in it is recorded by autograd
template <class F>
PyObject* entry(F f) {
  HANDLE_TH_ERRORS
  try {
    at::AutoDispatchBelowADInplaceOrView below;
    return f();
  } catch (const Set&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}
void arguments(Py_ssize_t got, Py_ssize_t want) {
  if (got != want) fail(PyExc_TypeError, "expected " + std::to_string(want) + " arguments, got " + std::to_string(got));
  if (!raw_stream) fail(hip_error ? hip_error : PyExc_RuntimeError, "liftreg_amd._host is not bound to the library");
}

PyObject* wrap(const at::Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}
PyObject* tuple(std::initializer_list<at::Tensor> ts) {
  PyObject* r = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
  if (!r) throw Set();
  Py_ssize_t i = 0;
  for (const at::Tensor& t : ts) {
    PyObject* o = wrap(t);
    if (!o) {
      Py_DECREF(r);
      throw Set();
    }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

// ---------------------------------------------------------------- layer norm
struct Norm {
  at::Tensor x, w, b;
  int64_t rows, cols;
  double eps, slope;
  bool bf16;
};
at::Tensor norm_param(PyObject* o, const char* name, const at::Tensor& x) {
  if (o == Py_None) return {};
  const at::Tensor& t = tensor(o, name);
  on_gpu(t, name);
  of_type(t, at::kFloat, name);
  if (t.dim() != 1 || t.size(0) != x.size(-1) || t.device() != x.device())
    fail(PyExc_ValueError, std::string(name) + " must have shape (" + std::to_string(x.size(-1)) + ",) on " + x.device().str() + ", got " +
                               shape_of(t) + " on " + t.device().str());
  return t.contiguous();
}
Norm norm_arguments(PyObject* x, PyObject* w, PyObject* b, PyObject* eps, PyObject* slope) {
  Norm n;
  n.x = tensor(x, "x");
  float_or_bf16(n.x, "x");
  if (n.x.dim() < 1 || n.x.size(-1) < 1) fail(PyExc_ValueError, "x must have a last axis to normalise, got shape " + shape_of(n.x));
  n.eps = number(eps);
  n.slope = number(slope);
  if (!(n.eps >= 0.0) || (n.eps > 0.0 && static_cast<float>(n.eps) == 0.f))
    fail(PyExc_ValueError, "eps must be 0 or a positive fp32 number");
  on_gpu(n.x, "x");
  n.x = n.x.contiguous();
  n.w = norm_param(w, "weight", n.x);
  n.b = norm_param(b, "bias", n.x);
  n.cols = n.x.size(-1);
  n.rows = n.x.numel() / n.cols;
  n.bf16 = n.x.scalar_type() == at::kBFloat16;
  return n;
}

// (x, weight, bias, eps, negative_slope, return_stats) -> y or (y, stats)
PyObject* layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry([&]() -> PyObject* {
    arguments(n, 6);
    const Norm q = norm_arguments(a[0], a[1], a[2], a[3], a[4]);
    const bool want = truth(a[5]);
    const c10::DeviceGuard guard(q.x.device());
    const at::Tensor y = at::empty_like(q.x, at::MemoryFormat::Contiguous);
    at::Tensor stats, ws;
    if (q.cols > lr.resident()) {
      ws = empty({std::max<int64_t>(16, count(lr.workspace(q.rows, q.cols, 0), "lr_layer_norm_workspace"))}, at::kByte, q.x.device());
      if (want) stats = empty({q.rows, 2}, at::kFloat, q.x.device());
    }
    check(lr.norm(data(q.x), static_cast<const float*>(data(q.w)), static_cast<const float*>(data(q.b)), data(y),
                  static_cast<float*>(data(stats)), data(ws), q.rows, q.cols, q.bf16, static_cast<float>(q.eps), static_cast<float>(q.slope),
                  stream_of(q.x.device().index())),
          "lr_layer_norm");
    return want ? tuple({y, stats}) : wrap(y);
  });
}

// (x, weight, bias, gy, eps, negative_slope, stats, need_gx, need_gwb) -> (gx, gw, gb)
PyObject* layer_norm_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry([&]() -> PyObject* {
    arguments(n, 9);
    const Norm q = norm_arguments(a[0], a[1], a[2], a[4], a[5]);
    at::Tensor gy = tensor(a[3], "gy"), stats, gx, gw, gb, ws;
    on_gpu(gy, "gy");
    of_type(gy, q.x.scalar_type(), "gy");
    if (gy.sizes() != q.x.sizes() || gy.device() != q.x.device())
      fail(PyExc_ValueError, "gy must have x's shape " + shape_of(q.x) + " and device, got " + shape_of(gy) + " on " + gy.device().str());
    gy = gy.contiguous();
    if (a[6] != Py_None) {
      stats = tensor(a[6], "stats");
      on_gpu(stats, "stats");
      of_type(stats, at::kFloat, "stats");
      if (stats.dim() != 2 || stats.size(0) != q.rows || stats.size(1) != 2 || stats.device() != q.x.device())
        fail(PyExc_ValueError, "stats must be a (" + std::to_string(q.rows) + ", 2) tensor on " + q.x.device().str() + ", got " +
                                   shape_of(stats) + " on " + stats.device().str());
      stats = stats.contiguous();
    }
    const bool need_gx = truth(a[7]), need_gwb = truth(a[8]);
    const c10::DeviceGuard guard(q.x.device());
    if (need_gx) gx = at::empty_like(q.x, at::MemoryFormat::Contiguous);
    if (need_gwb && q.w.defined()) gw = empty({q.cols}, at::kFloat, q.x.device());
    if (need_gwb && q.b.defined()) gb = empty({q.cols}, at::kFloat, q.x.device());
    const int64_t need = count(lr.workspace(q.rows, q.cols, 1), "lr_layer_norm_workspace");
    if (need) ws = empty({need}, at::kByte, q.x.device());
    check(lr.norm_bwd(data(q.x), static_cast<const float*>(data(q.w)), static_cast<const float*>(data(q.b)), data(gy),
                      static_cast<const float*>(data(stats)), data(gx), static_cast<float*>(data(gw)), static_cast<float*>(data(gb)),
                      data(ws), q.rows, q.cols, q.bf16, static_cast<float>(q.eps), static_cast<float>(q.slope),
                      stream_of(q.x.device().index())),
          "lr_layer_norm_bwd");
    return tuple({gx, gw, gb});
  });
}

// ---------------------------------------------------------------- lists of tensors
// The columns of a call: lists of n tensors each, checked against the first list's sizes, type and device.
struct Columns {
  int64_t n = 0;
  at::ScalarType type = at::kFloat;
  at::Device device = at::kCPU;
  std::vector<int64_t> numel;
  std::vector<std::pair<uint64_t, uint64_t>> written;      // what the call writes: first byte, end
  std::vector<std::vector<void*>> at;
  std::vector<at::Tensor> keep;       // the first list's tensors
  std::vector<PyObject*> lists;       // held until the launches: of a generator's tensors nothing else does, and what they free the call's own
                                      // workspace would take

  Columns() { lists.reserve(6); }
  Columns(const Columns&) = delete;
  ~Columns() {
    for (PyObject* o : lists) Py_DECREF(o);
  }

  // blocks: one element for each 32 of the first list's tensor
  void add(PyObject* list, const char* name, at::ScalarType want, bool blocks, bool writes) {
    PyObject* fast = PySequence_Fast(list, "expected a list of tensors");
    if (!fast) throw Set();
    lists.push_back(fast);
    const int64_t size = PySequence_Fast_GET_SIZE(fast);
    PyObject** items = PySequence_Fast_ITEMS(fast);
    const bool first = at.empty();
    if (first) {
      if (!size) fail(PyExc_ValueError, std::string(name) + ": no tensors");
      const at::Tensor& t = tensor(items[0], name);
      on_gpu(t, name);
      float_or_bf16(t, name);
      n = size;
      type = t.scalar_type();
      device = t.device();
      want = type;
      numel.reserve(n);
    } else if (size != n) {
      fail(PyExc_ValueError, std::string(name) + ": " + std::to_string(size) + " tensors for " + std::to_string(n) + " parameters");
    }
    std::vector<void*> column(n);
    for (int64_t i = 0; i < n; ++i) {
      const at::Tensor& t = tensor(items[i], name);
      on_gpu(t, name);
      if (t.device() != device)
        fail(PyExc_ValueError, std::string(name) + ": all tensors must be on the parameters' device, " + device.str() + ", got " + t.device().str());
      of_type(t, want, name);
      if (first) numel.push_back(t.numel());
      if (t.numel() != (blocks ? (numel[i] + 31) / 32 : numel[i])) fail(PyExc_ValueError, std::string(name) + ": the tensors' sizes do not match the parameters'");
      if (!t.is_contiguous()) fail(PyExc_ValueError, std::string(name) + ": tensors must be contiguous");
      column[i] = t.data_ptr();
      if (writes && t.numel()) {
        const uint64_t from = reinterpret_cast<uint64_t>(column[i]);
        written.emplace_back(from, from + t.nbytes());
      }
      if (first) keep.push_back(t);
    }
    at.push_back(std::move(column));
  }
  void no_overlap() {
    std::sort(written.begin(), written.end());
    for (size_t i = 1; i < written.size(); ++i)
      if (written[i].first < written[i - 1].second) fail(PyExc_ValueError, "parameters or states of the call share memory (is one there twice?)");
  }
  at::Tensor partial() const {
    return empty({std::max<int64_t>(1, count(lr.partials(numel.data(), static_cast<int>(n)), "lr_grad_norm_partials"))}, at::kDouble, device);
  }
};

// (grads) -> norm
PyObject* grad_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry([&]() -> PyObject* {
    arguments(n, 1);
    Columns c;
    c.add(a[0], "grads", at::kFloat, false, false);
    const c10::DeviceGuard guard(c.device);
    const at::Tensor partial = c.partial(), norm = empty({}, at::kFloat, c.device);
    check(lr.grad_norm(c.at[0].data(), c.numel.data(), static_cast<int>(c.n), c.type == at::kBFloat16, partial.data_ptr<double>(),
                       norm.data_ptr<float>(), stream_of(c.device.index())),
          "lr_grad_norm");
    return wrap(norm);
  });
}

// a one-element tensor that stays on the device
const at::Tensor& on_device(PyObject* o, const char* name, at::ScalarType type, const at::Device& device) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != type || t.numel() != 1 || t.device() != device)
    fail(PyExc_ValueError, std::string(name) + ": a tensor must be one " + c10::toString(type) + " on " + device.str() + ", got " +
                               c10::toString(t.scalar_type()) + " " + shape_of(t) + " on " + t.device().str());
  return t;
}

// One AdamW step: the constructor checks the arguments and allocates, run() launches.
// a: (params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, step, lr, beta1, beta2, eps, weight_decay, max_norm,
//     grad_norm, seed)
struct Step {
  Columns c;
  double b1, b2, eps, wd, max_norm, rate = 0.0;
  bool eight, clip;
  const float* rate_dev = nullptr;
  const int64_t* step_dev = nullptr;
  int64_t step = 1;
  uint64_t seed;
  at::Tensor norm, partial;

  explicit Step(PyObject* const* a) : b1(number(a[8])), b2(number(a[9])), eps(number(a[10])), wd(number(a[11])) {
    if (!(b1 >= 0.0 && b1 < 1.0 && b2 >= 0.0 && b2 < 1.0 && (eps == 0.0 || eps >= 0x1p-126) && wd >= 0.0))
      fail(PyExc_ValueError, "betas must be in [0, 1), eps 0 or at least 2^-126, weight_decay not negative; got " + std::to_string(b1) + ", " + std::to_string(b2) +
                                 ", " + std::to_string(eps) + ", " + std::to_string(wd));
    eight = a[4] != Py_None;
    clip = a[12] != Py_None;
    if (eight != (a[5] != Py_None)) fail(PyExc_ValueError, "8-bit states need both exp_avg_scales and exp_avg_sq_scales");
    if (!clip && a[13] != Py_None) fail(PyExc_ValueError, "grad_norm is for max_norm");
    max_norm = clip ? number(a[12]) : 0.0;
    if (clip && !(max_norm > 0.0)) fail(PyExc_ValueError, "max_norm must be positive, got " + std::to_string(max_norm));
    c.add(a[0], "params", at::kFloat, false, true);
    c.add(a[2], "exp_avgs", eight ? at::kFloat8_e4m3fn : at::kFloat, false, true);
    c.add(a[3], "exp_avg_sqs", eight ? at::kFloat8_e5m2 : at::kFloat, false, true);
    if (eight) {
      c.add(a[4], "exp_avg_scales", at::kFloat8_e8m0fnu, true, true);
      c.add(a[5], "exp_avg_sq_scales", at::kFloat8_e8m0fnu, true, true);
    }
    c.add(a[1], "grads", c.type, false, false);
    c.no_overlap();
    if (THPVariable_Check(a[7])) rate_dev = on_device(a[7], "lr", at::kFloat, c.device).data_ptr<float>();
    else rate = number(a[7]);
    if (THPVariable_Check(a[6])) step_dev = on_device(a[6], "step", at::kLong, c.device).data_ptr<int64_t>();
    else step = PyLong_AsLongLong(a[6]);
    if (step == -1 && PyErr_Occurred()) throw Set();
    if (!(rate >= 0.0) || step < 1) fail(PyExc_ValueError, "lr must not be negative and step starts at 1; got " + std::to_string(rate) + ", " + std::to_string(step));
    seed = PyLong_AsUnsignedLongLongMask(a[14]);
    if (PyErr_Occurred()) throw Set();
    const c10::DeviceGuard guard(c.device);
    if (clip && a[13] != Py_None) {
      norm = on_device(a[13], "grad_norm", at::kFloat, c.device);
    } else if (clip) {
      partial = c.partial();
      norm = empty({}, at::kFloat, c.device);
    }
  }
  void run() {
    const c10::DeviceGuard guard(c.device);
    const bool own = partial.defined();
    check(lr.adamw(c.at[0].data(), c.at.back().data(), c.at[1].data(), c.at[2].data(), eight ? c.at[3].data() : nullptr,
                   eight ? c.at[4].data() : nullptr, c.numel.data(), static_cast<int>(c.n), c.type == at::kBFloat16, rate, b1, b2, eps, wd, step,
                   rate_dev, step_dev, static_cast<float>(max_norm), clip && !own ? norm.data_ptr<float>() : nullptr,
                   own ? partial.data_ptr<double>() : nullptr, own ? norm.data_ptr<float>() : nullptr, seed, stream_of(c.device.index())),
          "lr_adamw_step");
    // written behind autograd's back: what is kept by a parameter's version sees it
    for (const at::Tensor& t : c.keep)
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  }
};

// (Step's arguments) -> norm or None
PyObject* adamw_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry([&]() -> PyObject* {
    arguments(n, 15);
    Step s(a);
    s.run();
    return wrap(s.norm);
  });
}

// (a tuple of Step's arguments, ...) -> the last one's norm or None.  All are checked before the first is launched: a call that is refused has
// written nothing.
PyObject* adamw_steps(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry([&]() -> PyObject* {
    std::deque<Step> steps;
    for (Py_ssize_t i = 0; i < n; ++i) {
      if (!PyTuple_Check(a[i])) fail(PyExc_TypeError, "expected tuples of arguments");
      arguments(PyTuple_GET_SIZE(a[i]), 15);
      steps.emplace_back(&PyTuple_GET_ITEM(a[i], 0));
    }
    for (Step& s : steps) s.run();
    return wrap(steps.empty() ? at::Tensor() : steps.back().norm);
  });
}

// (LiftRegHipError, torch._C._cuda_getCurrentRawStream, the addresses of Entries)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void** to = reinterpret_cast<void**>(&lr);
  constexpr Py_ssize_t entries = sizeof(Entries) / sizeof(void*);
  if (n != entries + 2) {
    PyErr_SetString(PyExc_TypeError, "bind: wrong number of entries");
    return nullptr;
  }
  for (Py_ssize_t i = 0; i < entries; ++i) {
    to[i] = PyLong_AsVoidPtr(a[i + 2]);
    if (!to[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: an entry is missing");
      return nullptr;
    }
  }
  Py_INCREF(a[0]);
  hip_error = a[0];
  Py_INCREF(a[1]);
  raw_stream = a[1];
  Py_RETURN_NONE;
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind), METHOD(layer_norm), METHOD(layer_norm_bwd), METHOD(grad_norm), METHOD(adamw_step), METHOD(adamw_steps), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "Host side of liftreg_amd.optim and ops.layer_norm (csrc/host.cpp).", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

#define TEXT_OF(x) #x
#define TEXT(x) TEXT_OF(x)

PyMODINIT_FUNC PyInit__host() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", TEXT(LR_TORCH)) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
