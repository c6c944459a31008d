// The tensor-level front ends of sirius_b200.ops whose calls take microseconds on the device: checks of arguments, outputs,
// workspaces and the C entry point in one native call. As Python over ctypes the same took 13 us for a norm and 0.4 us per
// gradient of a list, most of what a short call costs; here 4.6 us and 0.02.
//
// Module sirius_b200._ops_native. bind(path, error, no_memory) opens libsirius_b200.so (the one that ctypes has open already)
// and keeps the exceptions. Wrong operands raise ValueError or TypeError and name the operand.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/python_variable.h>

#include <stdexcept>
#include <string>
#include <vector>

#include "../../../include/sirius_b200.h"

namespace {

using at::Tensor;

// ---- the library -----------------------------------------------------------------------------------------
#define ENTRY(name) decltype(&::name) name = nullptr
struct Library {
  ENTRY(srt_last_error);
  ENTRY(srt_rmsnorm_fwd);
  ENTRY(srt_rmsnorm_fwd_e4m3);
  ENTRY(srt_quantize_rows_e4m3);
  ENTRY(srt_rmsnorm_bwd_scratch_bytes);
  ENTRY(srt_rmsnorm_bwd);
  ENTRY(srt_gated_ffn_fwd_scratch_bytes);
  ENTRY(srt_gated_ffn_fwd);
  ENTRY(srt_gated_ffn_fwd_e4m3);
  ENTRY(srt_gated_ffn_bwd_scratch_bytes);
  ENTRY(srt_gated_ffn_bwd);
  ENTRY(srt_grad_norm_scratch_bytes);
  ENTRY(srt_grad_norm);
  ENTRY(srt_clip_grad_norm);
  ENTRY(srt_adamw_clipped);
  ENTRY(srt_sgd_momentum_clipped);
} lib;
#undef ENTRY
PyObject *call_error = nullptr, *memory_error = nullptr;

// ---- errors ----------------------------------------------------------------------------------------------
struct Raise {  // thrown with the Python error to set
  PyObject* type;
  std::string text;
};
struct PySet {};  // a Python error is set already
[[noreturn]] void value_error(const std::string& t) { throw Raise{PyExc_ValueError, t}; }
[[noreturn]] void type_error(const std::string& t) { throw Raise{PyExc_TypeError, t}; }
void check(int status, const char* what) {
  if (status == SRT_OK) return;
  throw Raise{call_error, std::string(what) + " failed with status " + std::to_string(status) + ": " + lib.srt_last_error()};
}
// Every function of the module: C++ exceptions end here.
template <typename F>
PyObject* guarded(F&& f) {
  try {
    if (!call_error) throw Raise{PyExc_RuntimeError, "sirius_b200._ops_native is not bound"};
    return f();
  } catch (const Raise& e) {
    PyErr_SetString(e.type, e.text.c_str());
  } catch (const PySet&) {
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(memory_error, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

// The interpreter's lock is given up around allocations and entry points: both may wait, for memory or for a full launch queue,
// and other threads go on meanwhile.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  Unlocked() = default;
  Unlocked(const Unlocked&) = delete;
  ~Unlocked() { PyEval_RestoreThread(state); }
};
template <typename F>
auto unlocked(F&& f) {
  Unlocked u;
  return f();
}

// ---- arguments -------------------------------------------------------------------------------------------
std::string text(at::IntArrayRef s) {
  std::string t = "(";
  for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
  return t + (s.size() == 1 ? ",)" : ")");
}
struct Call {
  const char* what;
  int device;
  explicit Call(const char* w) : what(w), device(-1) {}
  std::string at(const char* name) const { return std::string(what) + ": " + name; }
  // A contiguous CUDA tensor on the current device, whose stream the call goes to.
  const Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) value_error(at(name) + " must be a contiguous CUDA tensor");
    const Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda() || !t.is_contiguous()) value_error(at(name) + " must be a contiguous CUDA tensor");
    if (device < 0) device = c10::cuda::current_device();
    if (t.device().index() != device)
      value_error(at(name) + " is on " + t.device().str() + "; operands are on the current device, cuda:" + std::to_string(device));
    return t;
  }
  const Tensor& tensor(PyObject* o, const char* name, at::ScalarType type) {
    const Tensor& t = tensor(o, name);
    if (t.scalar_type() != type) type_error(at(name) + " is " + c10::toString(t.scalar_type()) + ", not " + c10::toString(type));
    return t;
  }
  const Tensor& tensor(PyObject* o, const char* name, at::ScalarType type, at::IntArrayRef shape) {
    const Tensor& t = tensor(o, name, type);
    if (t.sizes() != shape) value_error(at(name) + " has shape " + text(t.sizes()) + ", not " + text(shape));
    return t;
  }
  void* optional(PyObject* o, const char* name, at::ScalarType type, at::IntArrayRef shape) {
    return o == Py_None ? nullptr : tensor(o, name, type, shape).data_ptr();
  }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(device).stream(); }
};
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PySet{};
  return v;
}
void count(Py_ssize_t got, Py_ssize_t want, const char* what) {
  if (got != want) type_error(std::string(what) + ": " + std::to_string(want) + " arguments");
}
// Straight from the caching allocator: through the dispatcher each of a call's three or four tensors took 0.3 us longer.
Tensor make(at::IntArrayRef shape, at::ScalarType type, int device) {
  return at::detail::empty_cuda(shape, type, at::Device(at::kCUDA, (c10::DeviceIndex)device), std::nullopt);
}
Tensor like(const Tensor& t, at::ScalarType type) { return make(t.sizes(), type, t.device().index()); }
Tensor like(const Tensor& t) { return like(t, t.scalar_type()); }
Tensor bytes(size_t n, int device) { return make({(int64_t)n}, at::kByte, device); }
PyObject* wrap(const Tensor& t) { return THPVariable_Wrap(t); }
// A tuple of new references.
template <typename... T>
PyObject* tuple(T... items) {
  PyObject* r = PyTuple_New(sizeof...(T));
  if (!r) throw PySet{};
  Py_ssize_t i = 0;
  (PyTuple_SET_ITEM(r, i++, items), ...);
  return r;
}
PyObject* same(PyObject* o) {
  Py_INCREF(o);
  return o;
}

int row_kind(const Call& c, const Tensor& x, const char* name) {
  if (x.dim() < 1) value_error(c.at(name) + " has no rows");
  if (x.scalar_type() == at::kBFloat16) return SRT_BF16;
  if (x.scalar_type() == at::kFloat) return SRT_F32;
  type_error(c.at(name) + " is " + c10::toString(x.scalar_type()) + "; rows are float32 or bfloat16");
}
int columns(const Call& c, const Tensor& x, const char* name) {
  const int64_t n = x.size(-1);
  if (n > INT32_MAX) value_error(c.at(name) + " has rows of more than 2^31 elements");
  return (int)n;
}
int64_t rows_of(at::IntArrayRef lead) {
  int64_t n = 1;
  for (int64_t v : lead) n *= v;
  return n;
}

// ---- norms -----------------------------------------------------------------------------------------------
// (x, gamma, eps, residual) -> (y, h, rstd)
PyObject* rmsnorm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] {
    Call c("rmsnorm");
    count(n, 4, c.what);
    const Tensor& x = c.tensor(a[0], "x");
    const int kind = row_kind(c, x, "x"), C = columns(c, x, "x");
    const Tensor& gamma = c.tensor(a[1], "gamma", at::kFloat, {x.size(-1)});
    const float eps = (float)number(a[2]);
    const void* residual = c.optional(a[3], "residual", x.scalar_type(), x.sizes());
    const at::IntArrayRef lead = x.sizes().slice(0, x.dim() - 1);
    Tensor y, h, rstd;
    check(unlocked([&] {
            y = like(x), rstd = make(lead, at::kFloat, c.device);
            if (residual) h = like(x);
            return lib.srt_rmsnorm_fwd(kind, x.data_ptr(), residual, gamma.data_ptr<float>(), residual ? h.data_ptr() : nullptr, y.data_ptr(),
                                       rstd.data_ptr<float>(), rows_of(lead), C, eps, c.stream());
          }),
          "srt_rmsnorm_fwd");
    return tuple(wrap(y), residual ? wrap(h) : same(a[0]), wrap(rstd));
  });
}
// (x, gamma, eps, residual) -> (q, scale, h, rstd)
PyObject* rmsnorm_e4m3(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] {
    Call c("rmsnorm_e4m3");
    count(n, 4, c.what);
    const Tensor& x = c.tensor(a[0], "x");
    const int kind = row_kind(c, x, "x"), C = columns(c, x, "x");
    const Tensor& gamma = c.tensor(a[1], "gamma", at::kFloat, {x.size(-1)});
    const float eps = (float)number(a[2]);
    const void* residual = c.optional(a[3], "residual", x.scalar_type(), x.sizes());
    const at::IntArrayRef lead = x.sizes().slice(0, x.dim() - 1);
    Tensor q, h, scale, rstd;
    check(unlocked([&] {
            q = like(x, at::kFloat8_e4m3fn), scale = make(lead, at::kFloat, c.device), rstd = make(lead, at::kFloat, c.device);
            if (residual) h = like(x);
            return lib.srt_rmsnorm_fwd_e4m3(kind, x.data_ptr(), residual, gamma.data_ptr<float>(), residual ? h.data_ptr() : nullptr, q.data_ptr(),
                                            scale.data_ptr<float>(), rstd.data_ptr<float>(), rows_of(lead), C, eps, c.stream());
          }),
          "srt_rmsnorm_fwd_e4m3");
    return tuple(wrap(q), wrap(scale), residual ? wrap(h) : same(a[0]), wrap(rstd));
  });
}
// (x) -> (q, scale)
PyObject* quantize_rows_e4m3(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] {
    Call c("quantize_rows_e4m3");
    count(n, 1, c.what);
    const Tensor& x = c.tensor(a[0], "x");
    const int kind = row_kind(c, x, "x"), C = columns(c, x, "x");
    const at::IntArrayRef lead = x.sizes().slice(0, x.dim() - 1);
    Tensor q, scale;
    check(unlocked([&] {
            q = like(x, at::kFloat8_e4m3fn), scale = make(lead, at::kFloat, c.device);
            return lib.srt_quantize_rows_e4m3(kind, x.data_ptr(), q.data_ptr(), scale.data_ptr<float>(), rows_of(lead), C, c.stream());
          }),
          "srt_quantize_rows_e4m3");
    return tuple(wrap(q), wrap(scale));
  });
}
// (dy, h, gamma, rstd, dh) -> (dx, dgamma)
PyObject* rmsnorm_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] {
    Call c("rmsnorm_backward");
    count(n, 5, c.what);
    const Tensor& h = c.tensor(a[1], "h");
    const int kind = row_kind(c, h, "h"), C = columns(c, h, "h");
    const at::IntArrayRef lead = h.sizes().slice(0, h.dim() - 1);
    const Tensor& dy = c.tensor(a[0], "dy", h.scalar_type(), h.sizes());
    const Tensor& gamma = c.tensor(a[2], "gamma", at::kFloat, {h.size(-1)});
    const Tensor& rstd = c.tensor(a[3], "rstd", at::kFloat, lead);
    const void* dh = c.optional(a[4], "dh", h.scalar_type(), h.sizes());
    const size_t need = lib.srt_rmsnorm_bwd_scratch_bytes(C);
    Tensor dx, dgamma;
    check(unlocked([&] {
            dx = like(h), dgamma = like(gamma);
            const Tensor scratch = bytes(need, c.device);
            return lib.srt_rmsnorm_bwd(kind, dy.data_ptr(), h.data_ptr(), gamma.data_ptr<float>(), rstd.data_ptr<float>(), dh, dx.data_ptr(),
                                       dgamma.data_ptr<float>(), rows_of(lead), C, scratch.data_ptr(), need, c.stream());
          }),
          "srt_rmsnorm_bwd");
    return tuple(wrap(dx), wrap(dgamma));
  });
}

// ---- feed-forward block ----------------------------------------------------------------------------------
struct Ffn {
  const Tensor &x, &w_gate_up, &w_down;
  srt_gated_ffn_desc d;
};
Ffn ffn(Call& c, PyObject* x, PyObject* w_gate_up, PyObject* w_down, at::ScalarType type) {
  Ffn f{c.tensor(x, "x", type), c.tensor(w_gate_up, "w_gate_up", type), c.tensor(w_down, "w_down", at::kBFloat16), {}};
  if (f.x.dim() != 2 || f.w_gate_up.dim() != 2 || f.w_down.dim() != 2 || f.w_gate_up.size(0) != 2 * f.w_down.size(1) ||
      f.w_gate_up.size(1) != f.x.size(1) || f.w_down.size(0) != f.x.size(1))
    value_error(std::string(c.what) + ": x [tokens, width], w_gate_up [2 hidden, width] and w_down [width, hidden] are wanted, not " +
                text(f.x.sizes()) + ", " + text(f.w_gate_up.sizes()) + " and " + text(f.w_down.sizes()));
  if (f.x.size(0) > INT32_MAX || f.x.size(1) > INT32_MAX || f.w_down.size(1) > INT32_MAX) value_error(std::string(c.what) + ": a size beyond 2^31");
  f.d = {(int)f.x.size(0), (int)f.x.size(1), (int)f.w_down.size(1)};
  return f;
}
// (x, w_gate_up, w_down, residual) -> y
PyObject* gated_ffn(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] {
    Call c("gated_ffn");
    count(n, 4, c.what);
    const Ffn f = ffn(c, a[0], a[1], a[2], at::kBFloat16);
    const void* residual = c.optional(a[3], "residual", at::kBFloat16, f.x.sizes());
    const size_t need = lib.srt_gated_ffn_fwd_scratch_bytes(&f.d);
    Tensor y;
    check(unlocked([&] {
            y = like(f.x);
            const Tensor scratch = bytes(need, c.device);
            return lib.srt_gated_ffn_fwd(&f.d, f.x.data_ptr(), f.w_gate_up.data_ptr(), f.w_down.data_ptr(), residual, y.data_ptr(),
                                         scratch.data_ptr(), need, c.stream());
          }),
          "srt_gated_ffn_fwd");
    return wrap(y);
  });
}
// (x, x_scale, w_gate_up, w_scale, w_down, residual) -> y
PyObject* gated_ffn_e4m3(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] {
    Call c("gated_ffn_e4m3");
    count(n, 6, c.what);
    const Ffn f = ffn(c, a[0], a[2], a[4], at::kFloat8_e4m3fn);
    const Tensor& x_scale = c.tensor(a[1], "x_scale", at::kFloat, {f.d.tokens});
    const Tensor& w_scale = c.tensor(a[3], "w_scale", at::kFloat, {2 * (int64_t)f.d.hidden});
    const void* residual = c.optional(a[5], "residual", at::kBFloat16, f.x.sizes());
    const size_t need = lib.srt_gated_ffn_fwd_scratch_bytes(&f.d);
    Tensor y;
    check(unlocked([&] {
            y = like(f.x, at::kBFloat16);
            const Tensor scratch = bytes(need, c.device);
            return lib.srt_gated_ffn_fwd_e4m3(&f.d, f.x.data_ptr(), x_scale.data_ptr<float>(), f.w_gate_up.data_ptr(), w_scale.data_ptr<float>(),
                                              f.w_down.data_ptr(), residual, y.data_ptr(), scratch.data_ptr(), need, c.stream());
          }),
          "srt_gated_ffn_fwd_e4m3");
    return wrap(y);
  });
}
// (dy, x, w_gate_up, w_down, fp32) -> (dx, dw_gate_up, dw_down)
PyObject* gated_ffn_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] {
    Call c("gated_ffn_backward");
    count(n, 5, c.what);
    const Ffn f = ffn(c, a[1], a[2], a[3], at::kBFloat16);
    const Tensor& dy = c.tensor(a[0], "dy", at::kBFloat16, f.x.sizes());
    const bool wide = PyObject_IsTrue(a[4]) == 1;
    const int kind = wide ? SRT_F32 : SRT_BF16;
    const at::ScalarType type = wide ? at::kFloat : at::kBFloat16;
    const size_t need = lib.srt_gated_ffn_bwd_scratch_bytes(&f.d, kind);
    Tensor dx, dw_gate_up, dw_down;
    check(unlocked([&] {
            dx = like(f.x), dw_gate_up = like(f.w_gate_up, type), dw_down = like(f.w_down, type);
            const Tensor scratch = bytes(need, c.device);
            return lib.srt_gated_ffn_bwd(&f.d, dy.data_ptr(), f.x.data_ptr(), f.w_gate_up.data_ptr(), f.w_down.data_ptr(), kind, dx.data_ptr(),
                                         dw_gate_up.data_ptr(), dw_down.data_ptr(), scratch.data_ptr(), need, c.stream());
          }),
          "srt_gated_ffn_bwd");
    return tuple(wrap(dx), wrap(dw_gate_up), wrap(dw_down));
  });
}

// ---- clipping --------------------------------------------------------------------------------------------
// (grads, max_norm, in_place) -> tensor of the norm and the coefficient
PyObject* grad_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] {
    const bool in_place = n == 3 && PyObject_IsTrue(a[2]) == 1;
    Call c(in_place ? "clip_grad_norm" : "grad_norm");
    count(n, 3, c.what);
    const float max_norm = (float)number(a[1]);
    if (!(max_norm > 0.f)) value_error(std::string(c.what) + ": max_norm (" + std::to_string(max_norm) + ") must be positive");
    struct Release {
      PyObject* o;
      ~Release() { Py_XDECREF(o); }
    } given{PySequence_Fast(a[0], "the gradients are a list of tensors")};
    if (!given.o) throw PySet{};
    // The call's own references: a caller's list may change in another thread while the lock is given up, and its tensors go.
    const Release held{PySequence_Tuple(given.o)};
    PyObject* list = held.o;
    if (!list) throw PySet{};
    const Py_ssize_t tensors = PySequence_Fast_GET_SIZE(list);
    if (tensors > INT32_MAX) value_error(std::string(c.what) + ": too many tensors");
    std::vector<void*> ptr((size_t)tensors);
    std::vector<int64_t> numel((size_t)tensors);
    at::ScalarType type = at::kFloat;
    for (Py_ssize_t i = 0; i < tensors; ++i) {
      PyObject* o = PySequence_Fast_GET_ITEM(list, i);
      if (i == 0) {
        type = c.tensor(o, "a gradient").scalar_type();
        if (type != at::kFloat && type != at::kBFloat16) type_error(c.at("gradients are ") + c10::toString(type) + ", not float32 or bfloat16");
      }
      const Tensor& t = c.tensor(o, "a gradient", type);
      ptr[(size_t)i] = t.data_ptr();
      numel[(size_t)i] = t.numel();
    }
    if (c.device < 0) c.device = c10::cuda::current_device();
    const size_t need = lib.srt_grad_norm_scratch_bytes((int)tensors);
    Tensor work;  // the results first, the partial sums behind them
    const int kind = type == at::kFloat ? SRT_F32 : SRT_BF16;
    const int status = unlocked([&] {
      work = bytes(256 + need, c.device);
      char* base = (char*)work.data_ptr();
      return in_place ? lib.srt_clip_grad_norm(kind, (int)tensors, ptr.data(), numel.data(), max_norm, (float*)base, base + 256, need, c.stream())
                      : lib.srt_grad_norm(kind, (int)tensors, ptr.data(), numel.data(), max_norm, (float*)base, base + 256, need, c.stream());
    });
    check(status, in_place ? "srt_clip_grad_norm" : "srt_grad_norm");
    return wrap(work.slice(0, 0, 8).view(at::kFloat));
  });
}
struct State {
  float *p, *g, *m, *v;
  void* p_bf16;
  const float* clip;
  int64_t n;
};
State state(Call& c, PyObject* p, PyObject* g, PyObject* m, PyObject* v, PyObject* p_bf16, PyObject* clip) {
  const Tensor& t = c.tensor(p, "p", at::kFloat);
  auto f = [&](PyObject* o, const char* name) { return c.tensor(o, name, at::kFloat, t.sizes()).data_ptr<float>(); };
  return {t.data_ptr<float>(), f(g, "g"), f(m, "m"), v ? f(v, "v") : nullptr, c.optional(p_bf16, "p_bf16", at::kBFloat16, t.sizes()),
          c.tensor(clip, "clip", at::kFloat, {2}).data_ptr<float>(), t.numel()};
}
// (p, g, m, v, lr, b1, b2, eps, wd, step, p_bf16, clip)
PyObject* adamw_clipped(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] {
    Call c("adamw");
    count(n, 12, c.what);
    const State s = state(c, a[0], a[1], a[2], a[3], a[10], a[11]);
    const long step = PyLong_AsLong(a[9]);
    if (step == -1 && PyErr_Occurred()) throw PySet{};
    const double lr = number(a[4]), b1 = number(a[5]), b2 = number(a[6]), eps = number(a[7]), wd = number(a[8]);
    check(unlocked([&] {
            return lib.srt_adamw_clipped(s.p, s.g, s.m, s.v, s.p_bf16, s.n, lr, b1, b2, eps, wd, step > INT32_MAX ? INT32_MAX : (int)step, s.clip,
                                         c.stream());
          }),
          "srt_adamw_clipped");
    Py_RETURN_NONE;
  });
}
// (p, g, m, lr, mu, wd, first_step, p_bf16, clip)
PyObject* sgd_momentum_clipped(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] {
    Call c("sgd_momentum");
    count(n, 9, c.what);
    const State s = state(c, a[0], a[1], a[2], nullptr, a[7], a[8]);
    const float lr = (float)number(a[3]), mu = (float)number(a[4]), wd = (float)number(a[5]);
    const int first_step = PyObject_IsTrue(a[6]) == 1;
    check(unlocked([&] { return lib.srt_sgd_momentum_clipped(s.p, s.g, s.m, s.p_bf16, s.n, lr, mu, wd, first_step, s.clip, c.stream()); }),
          "srt_sgd_momentum_clipped");
    Py_RETURN_NONE;
  });
}

// (path of the library, exceptions of failing calls and of device memory that ran out)
PyObject* bind(PyObject*, PyObject* args) {
  const char* path;
  PyObject *error, *no_memory;
  if (!PyArg_ParseTuple(args, "sOO", &path, &error, &no_memory)) return nullptr;
  void* handle = dlopen(path, RTLD_NOW | RTLD_LOCAL);
  if (!handle) return PyErr_Format(PyExc_OSError, "%s", dlerror());
  bool all = true;
  std::string missing;
#define FIND(name)                                                        \
  lib.name = (decltype(lib.name))dlsym(handle, #name);                    \
  if (!lib.name) { all = false; missing += std::string(" ") + #name; }
  FIND(srt_last_error)
  FIND(srt_rmsnorm_fwd)
  FIND(srt_rmsnorm_fwd_e4m3)
  FIND(srt_quantize_rows_e4m3)
  FIND(srt_rmsnorm_bwd_scratch_bytes)
  FIND(srt_rmsnorm_bwd)
  FIND(srt_gated_ffn_fwd_scratch_bytes)
  FIND(srt_gated_ffn_fwd)
  FIND(srt_gated_ffn_fwd_e4m3)
  FIND(srt_gated_ffn_bwd_scratch_bytes)
  FIND(srt_gated_ffn_bwd)
  FIND(srt_grad_norm_scratch_bytes)
  FIND(srt_grad_norm)
  FIND(srt_clip_grad_norm)
  FIND(srt_adamw_clipped)
  FIND(srt_sgd_momentum_clipped)
#undef FIND
  if (!all) return PyErr_Format(PyExc_OSError, "%s lacks%s", path, missing.c_str());
  Py_INCREF(no_memory);
  Py_XSETREF(memory_error, no_memory);
  Py_INCREF(error);
  Py_XSETREF(call_error, error);
  Py_RETURN_NONE;
}

#define FAST(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(rmsnorm),        FAST(rmsnorm_e4m3),       FAST(quantize_rows_e4m3), FAST(rmsnorm_backward),
                         FAST(gated_ffn),      FAST(gated_ffn_e4m3),     FAST(gated_ffn_backward), FAST(grad_norm),
                         FAST(adamw_clipped),  FAST(sgd_momentum_clipped), {"bind", bind, METH_VARARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops_native() { return PyModule_Create(&module); }
