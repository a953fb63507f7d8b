// Host path of the operators around the experts for the calls that need nothing but checks: contiguous tensors on the current device.
//
// A decode call is a kernel of a few microseconds; checked and allocated from Python it took 9 to 12 us of host time, from here 4 to 6.
// Every function returns None for a call that is not one of these (another layout, another device, anything to refuse): the Python layer then
// takes it, says what is wrong with it, copies what has to be copied.  Nothing is kept between calls.  Allocation and launch may wait (for
// memory, for room in the stream's queue) and so run without the interpreter's lock, as they do from Python.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include "../../include/b200moe.h"

namespace {

decltype(&b200moe_block_norm) g_norm;
decltype(&b200moe_gated_activation) g_act;
decltype(&b200moe_fp8_linear) g_linear;
decltype(&b200moe_fp8_linear_workspace_bytes) g_linear_ws;
decltype(&b200moe_env_set) g_env_set;

constexpr auto kFp8 = at::kFloat8_e4m3fn;

int code_of(at::ScalarType t) {
  return t == at::kBFloat16 ? B200MOE_DTYPE_BF16 : t == at::kHalf ? B200MOE_DTYPE_FP16 : t == at::kFloat ? B200MOE_DTYPE_FP32 : -2;
}

// A tensor argument: missing (None), or a plain contiguous one.
struct Arg {
  const at::Tensor* t = nullptr;
  bool ok = true;
  explicit Arg(PyObject* o) {
    if (o == Py_None) return;
    if (!THPVariable_CheckExact(o)) {       // (a subclass may mean something else by its operations)
      ok = false;
      return;
    }
    t = &THPVariable_Unpack(o);
  }
  bool on(const at::Tensor& x) const { return t == nullptr || (t->device() == x.device() && t->is_contiguous()); }
  void* data() const { return t == nullptr ? nullptr : t->data_ptr(); }
  int code() const { return t == nullptr ? 0 : code_of(t->scalar_type()); }
};

bool number(PyObject* o, float* f) {
  if (!PyFloat_CheckExact(o) && !PyLong_CheckExact(o)) return false;
  const double d = PyFloat_AsDouble(o);
  if (d == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  *f = static_cast<float>(d);
  return true;
}

// x: contiguous rows on the current device, in a type the kernels know
bool plain_rows(const Arg& a) {
  return a.ok && a.t != nullptr && a.t->is_cuda() && a.t->dim() >= 1 && a.t->layout() == at::kStrided && a.t->size(-1) > 0 &&
         a.t->is_contiguous() && a.t->numel() > 0 && a.t->device().index() == c10::cuda::current_device();
}
// [n] of x's type or fp32
bool plain_vector(const Arg& v, const at::Tensor& x, int64_t n) {
  return v.ok && (v.t == nullptr || (v.on(x) && v.t->dim() == 1 && v.t->size(0) == n &&
                                     (v.t->scalar_type() == x.scalar_type() || v.t->scalar_type() == at::kFloat)));
}

at::Tensor rows_like(const at::Tensor& x, int64_t last, at::ScalarType type) {
  c10::SmallVector<int64_t, 4> sizes(x.sizes().begin(), x.sizes().end());
  sizes.back() = last;
  return at::empty(sizes, x.options().dtype(type).requires_grad(false));
}

void* stream_of(const at::Tensor& x) { return c10::cuda::getCurrentCUDAStream(x.device().index()).stream(); }

PyObject* none() { Py_RETURN_NONE; }

PyObject* failed(int rc) { return PyLong_FromLong(rc); }

// (a, b), which are taken over
PyObject* tuple_of(PyObject* a, PyObject* b) {
  PyObject* r = a != nullptr && b != nullptr ? PyTuple_New(2) : nullptr;
  if (r == nullptr) {
    Py_XDECREF(a);
    Py_XDECREF(b);
    return nullptr;
  }
  PyTuple_SET_ITEM(r, 0, a);
  PyTuple_SET_ITEM(r, 1, b);
  return r;
}

// init(block_norm, gated_activation, fp8_linear, fp8_linear_workspace_bytes, env_set): addresses in the loaded library
PyObject* init(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "five addresses");
    return nullptr;
  }
  void* p[5];
  for (int i = 0; i < 5; ++i) {
    p[i] = PyLong_AsVoidPtr(args[i]);
    if (p[i] == nullptr && PyErr_Occurred()) return nullptr;
  }
  g_norm = reinterpret_cast<decltype(g_norm)>(p[0]);
  g_act = reinterpret_cast<decltype(g_act)>(p[1]);
  g_linear = reinterpret_cast<decltype(g_linear)>(p[2]);
  g_linear_ws = reinterpret_cast<decltype(g_linear_ws)>(p[3]);
  g_env_set = reinterpret_cast<decltype(g_env_set)>(p[4]);
  Py_RETURN_NONE;
}

// norm(post, pre, layer, quantize, inplace, residual_scale, eps, weight_offset, x, residual, gate, w_post, b_post, w_pre, b_pre)
// -> (y or (q, scale) or None, hidden), None: not this path's, an int: the library's error
PyObject* norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 15) return none();
  const bool post = args[0] == Py_True, pre = args[1] == Py_True, layer = args[2] == Py_True, quant = args[3] == Py_True,
             inplace = args[4] == Py_True;
  float f[3];
  for (int i = 0; i < 3; ++i)
    if (!number(args[5 + i], &f[i])) return none();
  const Arg x(args[8]), residual(args[9]), gate(args[10]), w_post(args[11]), b_post(args[12]), w_pre(args[13]), b_pre(args[14]);
  if (!plain_rows(x) || !residual.ok || !gate.ok || !(f[1] >= 0.f) || g_env_set()) return none();
  const at::Tensor& t = *x.t;
  const int64_t h = t.size(-1), m = t.numel() / h;
  const int dt = code_of(t.scalar_type());
  if (dt < 0 || h > B200MOE_NORM_MAX_H || m > B200MOE_NORM_MAX_ROWS) return none();
  if (residual.t != nullptr && (!residual.on(t) || residual.t->sizes() != t.sizes() ||
                                (residual.t->scalar_type() != t.scalar_type() && residual.t->scalar_type() != at::kFloat)))
    return none();
  if (inplace && residual.t == nullptr) return none();
  if (!plain_vector(w_post, t, h) || !plain_vector(b_post, t, h) || !plain_vector(w_pre, t, h) || !plain_vector(b_pre, t, h)) return none();
  b200moe_norm p = {};
  p.struct_bytes = sizeof(p);
  if (gate.t != nullptr) {
    const at::Tensor& g = *gate.t;
    if (!gate.on(t) || (g.scalar_type() != t.scalar_type() && g.scalar_type() != at::kFloat)) return none();
    if (g.dim() == 1 && g.size(0) == h) {
      p.gate_mode = B200MOE_GATE_CHANNEL;
    } else if (g.sizes() == t.sizes() && h > 1) {
      p.gate_mode = B200MOE_GATE_FULL;
      p.ldg = h;
    } else if (g.dim() == t.dim() && g.size(-1) == 1 && g.sizes().slice(0, g.dim() - 1) == t.sizes().slice(0, t.dim() - 1)) {
      p.gate_mode = B200MOE_GATE_TOKEN;
      p.ldg = 1;
    } else {
      return none();
    }
  }
  p.M = static_cast<int32_t>(m);
  p.H = static_cast<int32_t>(h);
  p.kind = layer ? B200MOE_NORM_LAYER : B200MOE_NORM_RMS;
  p.dtype = dt;
  p.residual_dtype = residual.t != nullptr ? residual.code() : dt;
  p.post = post;
  p.pre = pre;
  p.gate_dtype = gate.code();
  p.w_post_dtype = w_post.code();
  p.b_post_dtype = b_post.code();
  p.w_pre_dtype = w_pre.code();
  p.b_pre_dtype = b_pre.code();
  p.residual_scale = f[0];
  p.eps = f[1];
  p.weight_offset = f[2];
  p.ldx = p.ldr = p.ldh = h;
  const bool same = !post && residual.t == nullptr && gate.t == nullptr && f[0] == 1.f;      // hidden is x itself
  at::Tensor hidden, y, scale;
  int rc;
  {
    pybind11::gil_scoped_release unlocked;
    if (!inplace && !same) hidden = at::empty(t.sizes(), (residual.t != nullptr ? *residual.t : t).options().requires_grad(false));
    if (pre) y = rows_like(t, h, quant ? kFp8 : t.scalar_type());
    if (pre && quant) scale = rows_like(t, (h + 127) / 128, at::kFloat);
    rc = g_norm(&p, t.data_ptr(), residual.data(), gate.data(), w_post.data(), b_post.data(), w_pre.data(), b_pre.data(),
                same ? nullptr : inplace ? residual.data() : hidden.data_ptr(), pre ? y.data_ptr() : nullptr,
                pre && quant ? static_cast<float*>(scale.data_ptr()) : nullptr, stream_of(t));
  }
  if (rc != B200MOE_OK) return failed(rc);
  PyObject* out = !pre    ? none()
                  : quant ? tuple_of(THPVariable_Wrap(std::move(y)), THPVariable_Wrap(std::move(scale)))
                          : THPVariable_Wrap(std::move(y));
  PyObject* hid = inplace ? args[9] : same ? args[8] : nullptr;
  if (hid != nullptr) Py_INCREF(hid);
  else hid = THPVariable_Wrap(std::move(hidden));
  return tuple_of(out, hid);
  END_HANDLE_TH_ERRORS
}

// activation(kind, alpha, limit, quantize, x) -> y or (q, scale); None and int as above
PyObject* activation(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  float alpha, limit;
  if (n != 5 || !PyLong_CheckExact(args[0]) || !number(args[1], &alpha) || !number(args[2], &limit)) return none();
  const Arg x(args[4]);
  const bool quant = args[3] == Py_True;
  if (!plain_rows(x) || g_env_set()) return none();
  const at::Tensor& t = *x.t;
  const int64_t w = t.size(-1), m = t.numel() / w, i = w / 2;
  const int dt = code_of(t.scalar_type());
  if (dt < 0 || w % 2 != 0 || m > B200MOE_MAX_ROWS || i > B200MOE_ACT_MAX_I) return none();
  const int kind = static_cast<int>(PyLong_AsLong(args[0]));
  at::Tensor y, scale;
  int rc;
  {
    pybind11::gil_scoped_release unlocked;
    y = rows_like(t, i, quant ? kFp8 : t.scalar_type());
    if (quant) scale = rows_like(t, (i + 127) / 128, at::kFloat);
    rc = g_act(t.data_ptr(), w, dt, static_cast<int>(m), static_cast<int>(i), kind, alpha, limit, y.data_ptr(),
               quant ? static_cast<float*>(scale.data_ptr()) : nullptr, 0, stream_of(t));
  }
  if (rc != B200MOE_OK) return failed(rc);
  return quant ? tuple_of(THPVariable_Wrap(std::move(y)), THPVariable_Wrap(std::move(scale))) : THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// linear(x, weight, weight_scale, bias, x_scale, status) -> out in x's type (e4m3 x: bfloat16); None and int as above
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) return none();
  const Arg x(args[0]), weight(args[1]), weight_scale(args[2]), bias(args[3]), x_scale(args[4]), status(args[5]);
  if (!plain_rows(x) || !weight.ok || !weight_scale.ok || !bias.ok || !x_scale.ok || !status.ok || weight.t == nullptr || weight_scale.t == nullptr ||
      status.t == nullptr || g_env_set())
    return none();
  const at::Tensor &t = *x.t, &w = *weight.t, &ws = *weight_scale.t;
  if (w.dim() != 2 || w.scalar_type() != kFp8 || w.device() != t.device() || w.size(0) <= 0 || w.size(1) != t.size(-1)) return none();
  const int64_t rows = w.size(0), k = w.size(1), m = t.numel() / k, g = (k + 127) / 128;
  if (k % 16 != 0 || k > B200MOE_LINEAR_MAX_K || rows > B200MOE_MAX_ROWS || m > B200MOE_MAX_ROWS) return none();
  if (w.stride(1) != 1 || (rows > 1 && (w.stride(0) < k || w.stride(0) % 16 != 0))) return none();
  if (!weight_scale.on(t) || ws.scalar_type() != at::kFloat || ws.dim() != 2 || ws.size(0) != (rows + 127) / 128 || ws.size(1) != g) return none();
  const bool fp8 = t.scalar_type() == kFp8;
  const int dt = fp8 ? B200MOE_X_E4M3 : code_of(t.scalar_type());
  if (!fp8 && dt != B200MOE_DTYPE_BF16 && dt != B200MOE_DTYPE_FP16) return none();
  if (fp8 != (x_scale.t != nullptr)) return none();
  if (fp8) {
    const at::Tensor& s = *x_scale.t;
    if (!x_scale.on(t) || s.scalar_type() != at::kFloat || s.dim() != t.dim() || s.size(-1) != g ||
        s.sizes().slice(0, s.dim() - 1) != t.sizes().slice(0, t.dim() - 1))
      return none();
  }
  if (bias.t != nullptr && (!bias.on(t) || bias.t->dim() != 1 || bias.t->size(0) != rows || bias.code() < 0)) return none();
  if (((reinterpret_cast<uintptr_t>(t.data_ptr()) | reinterpret_cast<uintptr_t>(w.data_ptr())) & 15) != 0) return none();
  b200moe_linear p = {};
  p.struct_bytes = sizeof(p);
  p.M = static_cast<int32_t>(m);
  p.N = static_cast<int32_t>(rows);
  p.K = static_cast<int32_t>(k);
  p.x_dtype = dt;
  p.out_dtype = fp8 ? B200MOE_DTYPE_BF16 : dt;
  p.bias_dtype = bias.code();
  p.ldx = k;
  p.ldw = rows > 1 ? w.stride(0) : k;
  at::Tensor out, work;
  int rc;
  {
    pybind11::gil_scoped_release unlocked;
    out = rows_like(t, rows, fp8 ? at::kBFloat16 : t.scalar_type());
    // (the workspace is torch's: kept for this stream by its allocator, or for the graph under capture, so that no two share it)
    const size_t bytes = g_linear_ws(&p);
    if (bytes > 0) work = at::empty({static_cast<int64_t>(bytes)}, t.options().dtype(at::kByte).requires_grad(false));
    rc = g_linear(&p, t.data_ptr(), static_cast<const float*>(x_scale.data()), w.data_ptr(), static_cast<const float*>(ws.data_ptr()),
                  bias.data(), bytes > 0 ? work.data_ptr() : nullptr, bytes, out.data_ptr(), static_cast<int32_t*>(status.t->data_ptr()),
                  stream_of(t));
  }
  if (rc != B200MOE_OK) return failed(rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"init", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(init)), METH_FASTCALL, nullptr},
                         {"norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(norm)), METH_FASTCALL, nullptr},
                         {"activation", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(activation)), METH_FASTCALL, nullptr},
                         {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(linear)), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fastcall", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fastcall() {
  PyObject* m = PyModule_Create(&module);
  if (m != nullptr && (PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) != 0 ||
                       PyModule_AddIntConstant(m, "version", B200MOE_VERSION) != 0)) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
