// The call around a quantized linear layer (mlx-rs/src/nn/quantized.rs:363-386) on torch tensors without the interpreter: the same
// checks, result, workspace and stream as ops.quantized_linear's own lines, which stay the general path.  One token's layer is 5 us of
// kernel; its call took 10 us in Python (checks 3, two allocations 2, the foreign call's conversions 3) and takes the kernel's time with this.
//
// quantized_linear(x, w, scales, biases, linear_bias, transpose, group_size, bits) returns the result, None for whatever is not a
// plain device tensor of the expected type, shape, layout and alignment (the caller then goes the general way, which takes it or words
// the refusal), or the library's status where that is not zero.  Nothing is kept between calls.  The interpreter is let go around the
// allocations and the launch, any of which may wait (for memory, for room in a queue, for a kernel to load).
//
// So with the operators around a layer, in ops' argument order: add_rms_norm, add_rms_norm_rows8, add_rms_norm_grad, quantized_linear_rows8, select_experts
// and select_experts_grad, whose kernels take 4 us for a few tokens and whose calls took 9 in Python and
// take 5 with this.
#include <ATen/ATen.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/api/include/torch/version.h>

#include "../../include/mi_moe.h"
#include "../../include/mi_moe_layer.h"

namespace {

decltype(&mi_moe_quantized_linear_typed) g_linear;
decltype(&mi_moe_quantized_matmul_typed) g_matmul;
decltype(&mi_moe_quantized_matmul_workspace_size) g_workspace;
struct {
  decltype(&mi_moe_add_rms_norm) norm;
  decltype(&mi_moe_add_rms_norm_rows8) norm_rows8;
  decltype(&mi_moe_add_rms_norm_grad_workspace_size) norm_grad_workspace;
  decltype(&mi_moe_add_rms_norm_grad) norm_grad;
  decltype(&mi_moe_quantized_linear_rows8_workspace_size) rows8_workspace;
  decltype(&mi_moe_quantized_linear_rows8) rows8;
  decltype(&mi_moe_select_experts) select;
  decltype(&mi_moe_select_experts_grad) select_grad;
} g_layer;

// a tensor itself (no subclass), dense, on a GPU, contiguous, seen through no transform (vmap, functionalisation, a Python key)
const at::Tensor *plain(PyObject *o, at::ScalarType type) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor &t = THPVariable_Unpack(o);
  if (!t.defined() || t.scalar_type() != type || !t.is_cuda() || t.layout() != at::kStrided || !t.has_storage() || !t.is_contiguous()) return nullptr;
  constexpr c10::DispatchKeySet other({c10::DispatchKey::Python, c10::DispatchKey::Functionalize, c10::DispatchKey::FuncTorchBatched,
                                       c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Conjugate, c10::DispatchKey::Negative});
  return t.key_set().has_any(other) ? nullptr : &t;
}

PyObject *quantized_linear(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != 8) {
    PyErr_SetString(PyExc_TypeError, "quantized_linear: eight arguments");
    return nullptr;
  }
  try {
    if (!THPVariable_CheckExact(args[0]) || !PyLong_Check(args[6]) || !PyLong_Check(args[7])) Py_RETURN_NONE;
    const at::ScalarType type = THPVariable_Unpack(args[0]).scalar_type();
    const int dt = type == at::kBFloat16 ? MI_MOE_DTYPE_BF16 : type == at::kHalf ? MI_MOE_DTYPE_F16 : type == at::kFloat ? MI_MOE_DTYPE_F32 : -1;
    const int transpose = PyObject_IsTrue(args[5]);
    const long group = PyLong_AsLong(args[6]), bits = PyLong_AsLong(args[7]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    if (dt < 0 || transpose < 0 || (group != 32 && group != 64 && group != 128) || (bits != 2 && bits != 4 && bits != 8)) Py_RETURN_NONE;
    const at::Tensor *const x = plain(args[0], type), *const w = plain(args[1], at::kInt), *const s = plain(args[2], type), *const b = plain(args[3], type);
    if (!x || !w || !s || !b || x->dim() < 1 || w->dim() != 2 || s->dim() != 2 || b->dim() != 2) Py_RETURN_NONE;
    const int64_t K = x->size(-1), per = 32 / bits;
    const int64_t N = transpose ? w->size(0) : w->size(1) * per, kw = transpose ? w->size(1) * per : w->size(0);
    const int64_t rows = transpose ? N : K, q_axis = transpose ? K : N;
    if (kw != K || x->numel() == 0 || N == 0 || q_axis % group || K > INT32_MAX || N > INT32_MAX) Py_RETURN_NONE;
    for (const at::Tensor *t : {s, b})
      if (t->size(0) != rows || t->size(1) != q_axis / group) Py_RETURN_NONE;
    const at::Tensor *lb = nullptr;
    if (args[4] != Py_None) {
      lb = plain(args[4], type);
      if (!lb || !transpose || lb->numel() != N) Py_RETURN_NONE;
    }
    for (const at::Tensor *t : {x, w, s, b})
      if (reinterpret_cast<uintptr_t>(t->const_data_ptr()) & 15u) Py_RETURN_NONE;
    const int64_t M = x->numel() / K;
    if (M > (int64_t)1 << 30) Py_RETURN_NONE;
    size_t need = 0;
    if (g_workspace(M, (int32_t)K, (int32_t)bits, &need)) Py_RETURN_NONE;
    at::DimVector shape(x->sizes().begin(), x->sizes().end());
    shape.back() = N;
    // (the operands' own references: another thread may drop the caller's while the interpreter is let go)
    const at::Tensor xk = *x, wk = *w, sk = *s, bk = *b, lk = lb ? *lb : at::Tensor();
    at::Tensor y;
    int status = 0;
    {
      pybind11::gil_scoped_release let_go;
      const at::TensorOptions on = at::TensorOptions().device(xk.device());
      y = at::empty(shape, on.dtype(type));
      at::Tensor ws = at::empty({(int64_t)need + 256}, on.dtype(at::kByte));
      void *const st = c10::hip::getCurrentHIPStream(c10::hip::current_device()).stream();
      status = lk.defined()
                   ? g_linear(xk.const_data_ptr(), static_cast<const uint32_t *>(wk.const_data_ptr()), sk.const_data_ptr(), bk.const_data_ptr(), lk.const_data_ptr(),
                              M, (int32_t)N, (int32_t)K, (int32_t)group, (int32_t)bits, dt, y.data_ptr(), ws.data_ptr(), need + 256, st)
                   : g_matmul(xk.const_data_ptr(), static_cast<const uint32_t *>(wk.const_data_ptr()), sk.const_data_ptr(), bk.const_data_ptr(), M, (int32_t)N,
                              (int32_t)K, transpose, (int32_t)group, (int32_t)bits, dt, y.data_ptr(), ws.data_ptr(), need + 256, st);
    }
    if (status) return PyLong_FromLong(status);
    return THPVariable_Wrap(std::move(y));
  } catch (python_error &e) {  // what a mode written in Python raised from an allocation: the caller's
    e.restore();
  } catch (pybind11::error_already_set &e) {
    e.restore();
  } catch (const std::exception &) {  // (out of memory: the general path meets it again and words it)
  }
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

int dtype_code(at::ScalarType type) {
  return type == at::kBFloat16 ? MI_MOE_DTYPE_BF16 : type == at::kHalf ? MI_MOE_DTYPE_F16 : type == at::kFloat ? MI_MOE_DTYPE_F32 : -1;
}

// The operands of a call, kept alive across it (another thread may drop the caller's references while the interpreter is let go): plain tensors on the current device.
struct Operands {
  at::Tensor t[6];
  int n = 0;
  bool good = true;
  const at::Tensor &add(PyObject *o, at::ScalarType type) {
    const at::Tensor *const p = plain(o, type);
    if (p && p->device().index() == c10::hip::current_device()) t[n] = *p;
    else good = false;
    return t[n++];
  }
  const at::Tensor &add_or_none(PyObject *o, at::ScalarType type) { return o == Py_None ? t[n++] : add(o, type); }
};

const void *data_of(const at::Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }
at::ScalarType type_of(PyObject *o) { return THPVariable_CheckExact(o) ? THPVariable_Unpack(o).scalar_type() : at::ScalarType::Undefined; }
void *stream_here() { return c10::hip::getCurrentHIPStream(c10::hip::current_device()).stream(); }

// numbers of the call; `good` turns false for what is none
struct Numbers {
  bool good = true;
  int64_t whole(PyObject *o) {
    const long long v = PyLong_CheckExact(o) ? PyLong_AsLongLong(o) : -1;
    if (v < 0 || v > INT32_MAX) good = false;
    return v;
  }
  float real(PyObject *o) {
    if (!PyFloat_CheckExact(o) && !PyLong_CheckExact(o)) return good = false, 0.f;
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) good = false;
    return (float)v;
  }
  bool truth(PyObject *o) {
    if (!PyBool_Check(o)) good = false;
    return o == Py_True;
  }
  int word(PyObject *o, const char *first, int code, const char *second, int other) {
    if (PyUnicode_CheckExact(o)) {
      if (PyUnicode_CompareWithASCIIString(o, first) == 0) return code;
      if (PyUnicode_CompareWithASCIIString(o, second) == 0) return other;
    }
    return good = false, 0;
  }
  ~Numbers() {
    if (!good) PyErr_Clear();  // (of an integer too large)
  }
};

// what the entries below end in: `f` fills `out` and returns the library's status, or -1 for the general way; results as a tuple, an undefined one as `same`
template <int RESULTS, class F>
PyObject *call(F f, PyObject *same = nullptr) {
  at::Tensor out[RESULTS];
  int status;
  {
    pybind11::gil_scoped_release let_go;
    status = f(out);
  }
  if (status == -1) Py_RETURN_NONE;
  if (status) return PyLong_FromLong(status);
  if (RESULTS == 1) return THPVariable_Wrap(std::move(out[0]));
  PyObject *const all = PyTuple_New(RESULTS);
  if (!all) return nullptr;
  for (int i = 0; i < RESULTS; ++i) {
    PyObject *one = same;
    if (out[i].defined()) one = THPVariable_Wrap(std::move(out[i]));
    else Py_XINCREF(same);
    if (!one) {
      Py_DECREF(all);
      return nullptr;
    }
    PyTuple_SET_ITEM(all, i, one);
  }
  return all;
}

bool count_is(Py_ssize_t n, Py_ssize_t want, const char *who) {
  if (n != want) PyErr_Format(PyExc_TypeError, "%s: %zd arguments", who, want);
  return n == want;
}

// x, residual, weight, eps: what the two forward calls of the norm share
struct NormCall {
  Operands in;
  int dt, good;
  float eps;
  int64_t T = 0, H = 0;
  explicit NormCall(PyObject *const *args) {
    Numbers num;
    const at::ScalarType type = type_of(args[0]);
    dt = dtype_code(type);
    eps = num.real(args[3]);
    good = 0;
    if (dt < 0 || !num.good) return;
    const at::Tensor &x = in.add(args[0], type), &r = in.add_or_none(args[1], type), &w = in.add(args[2], type);
    if (!in.good || x.dim() < 1 || x.numel() == 0 || x.size(-1) > INT32_MAX || w.numel() != x.size(-1) || (r.defined() && r.sizes() != x.sizes())) return;
    H = x.size(-1);
    T = x.numel() / H;
    good = 1;
  }
};

PyObject *add_rms_norm(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (!count_is(n, 4, "add_rms_norm")) return nullptr;
  const NormCall c(args);
  if (!c.good) Py_RETURN_NONE;
  return call<2>([&](at::Tensor *out) {
    const at::Tensor &x = c.in.t[0];
    out[0] = at::empty(x.sizes(), x.options());
    if (c.in.t[1].defined()) out[1] = at::empty(x.sizes(), x.options());
    return g_layer.norm(data_of(x), data_of(c.in.t[1]), data_of(c.in.t[2]), c.eps, c.T, (int32_t)c.H, c.dt, out[1].defined() ? out[1].data_ptr() : nullptr, out[0].data_ptr(),
                        stream_here());
  }, args[0]);
}

PyObject *add_rms_norm_rows8(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (!count_is(n, 4, "add_rms_norm_rows8")) return nullptr;
  const NormCall c(args);
  if (!c.good) Py_RETURN_NONE;
  return call<3>([&](at::Tensor *out) {
    const at::Tensor &x = c.in.t[0];
    out[0] = at::empty(x.sizes(), x.options().dtype(at::kChar));
    out[1] = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
    if (c.in.t[1].defined()) out[2] = at::empty(x.sizes(), x.options());
    return g_layer.norm_rows8(data_of(x), data_of(c.in.t[1]), data_of(c.in.t[2]), c.eps, c.T, (int32_t)c.H, c.dt, out[2].defined() ? out[2].data_ptr() : nullptr,
                              out[0].data_ptr(), static_cast<float *>(out[1].data_ptr()), stream_here());
  }, args[0]);
}

// dy, h, weight, eps, dh
PyObject *add_rms_norm_grad(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (!count_is(n, 5, "add_rms_norm_grad")) return nullptr;
  PyObject *const own[4] = {args[1], args[0], args[2], args[3]};
  if (args[0] == Py_None) Py_RETURN_NONE;
  NormCall c(own);
  if (!c.good) Py_RETURN_NONE;
  const at::Tensor &dh = c.in.add_or_none(args[4], c.in.t[0].scalar_type());
  if (!c.in.good || (dh.defined() && dh.sizes() != c.in.t[0].sizes())) Py_RETURN_NONE;
  return call<2>([&](at::Tensor *out) {
    const at::Tensor &h = c.in.t[0], &w = c.in.t[2];
    size_t need = 0;
    if (g_layer.norm_grad_workspace(c.T, (int32_t)c.H, &need)) return -1;
    out[0] = at::empty(h.sizes(), h.options());
    out[1] = at::empty(w.sizes(), w.options());
    const at::Tensor ws = at::empty({(int64_t)need}, h.options().dtype(at::kByte));
    return g_layer.norm_grad(data_of(c.in.t[1]), data_of(h), data_of(dh), data_of(w), c.eps, c.T, (int32_t)c.H, c.dt, out[0].data_ptr(), out[1].data_ptr(), ws.data_ptr(), need,
                             stream_here());
  });
}

// x, row_scales, w, scales, biases, linear_bias, group_size, bits
PyObject *quantized_linear_rows8(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (!count_is(n, 8, "quantized_linear_rows8")) return nullptr;
  Numbers num;
  Operands in;
  const int64_t group = num.whole(args[6]), bits = num.whole(args[7]);
  const at::ScalarType type = type_of(args[3]);
  const int dt = dtype_code(type);
  if (dt < 0 || !num.good || (group != 32 && group != 64 && group != 128) || (bits != 4 && bits != 8)) Py_RETURN_NONE;
  const at::Tensor &x = in.add(args[0], at::kChar), &rs = in.add(args[1], at::kFloat), &w = in.add(args[2], at::kInt), &s = in.add(args[3], type),
                   &b = in.add(args[4], type), &lb = in.add_or_none(args[5], type);
  if (!in.good || x.dim() < 1 || x.numel() == 0 || w.dim() != 2 || s.dim() != 2 || b.dim() != 2 || rs.sizes() != x.sizes().slice(0, x.dim() - 1)) Py_RETURN_NONE;
  const int64_t K = x.size(-1), N = w.size(0), M = rs.numel();
  if (N == 0 || K > INT32_MAX || N > INT32_MAX || K % group || w.size(1) * (32 / bits) != K || (lb.defined() && lb.numel() != N)) Py_RETURN_NONE;
  for (const at::Tensor *t : {&s, &b})
    if (t->size(0) != N || t->size(1) != K / group) Py_RETURN_NONE;
  return call<1>([&](at::Tensor *out) {
    size_t need = 0;
    if (g_layer.rows8_workspace(M, (int32_t)K, &need)) return -1;
    at::DimVector shape(x.sizes().begin(), x.sizes().end());
    shape.back() = N;
    out[0] = at::empty(shape, s.options());
    at::Tensor ws;
    if (need) ws = at::empty({(int64_t)need}, x.options().dtype(at::kByte));
    return g_layer.rows8(data_of(x), static_cast<const float *>(data_of(rs)), static_cast<const uint32_t *>(data_of(w)), data_of(s), data_of(b), data_of(lb), M, (int32_t)N,
                         (int32_t)K, (int32_t)group, (int32_t)bits, dt, out[0].data_ptr(), need ? ws.data_ptr() : nullptr, need, stream_here());
  });
}

// logits, top_k, scoring, bias, n_groups, top_groups, group_score, renormalize, scale, dtype
PyObject *select_experts(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (!count_is(n, 10, "select_experts")) return nullptr;
  Numbers num;
  Operands in;
  const int64_t k = num.whole(args[1]), groups = num.whole(args[4]), top_groups = num.whole(args[5]);
  const int scoring = num.word(args[2], "softmax", MI_MOE_SCORING_SOFTMAX, "sigmoid", MI_MOE_SCORING_SIGMOID);
  const int group_score = num.word(args[6], "max", MI_MOE_GROUP_SCORE_MAX, "top2", MI_MOE_GROUP_SCORE_TOP2);
  const bool renormalize = num.truth(args[7]);
  const float scale = num.real(args[8]);
  const at::ScalarType type = type_of(args[0]);
  const int dt = dtype_code(type);
  if (dt < 0 || !num.good || !THPDtype_Check(args[9])) Py_RETURN_NONE;
  const at::ScalarType w_type = reinterpret_cast<THPDtype *>(args[9])->scalar_type;
  const int wt = dtype_code(w_type);
  const at::Tensor &l = in.add(args[0], type), &b = in.add_or_none(args[3], at::kFloat);
  if (wt < 0 || !in.good || l.dim() < 1 || l.numel() == 0) Py_RETURN_NONE;
  const int64_t E = l.size(-1);
  if (E > INT32_MAX || k < 1 || k > E || (b.defined() && b.numel() != E)) Py_RETURN_NONE;
  return call<2>([&](at::Tensor *out) {
    at::DimVector shape(l.sizes().begin(), l.sizes().end());
    shape.back() = k;
    out[0] = at::empty(shape, l.options().dtype(at::kInt));
    out[1] = at::empty(shape, l.options().dtype(w_type));
    return g_layer.select(data_of(l), dt, static_cast<const float *>(data_of(b)), l.numel() / E, (int32_t)E, (int32_t)k, scoring, (int32_t)groups, (int32_t)top_groups, group_score,
                          renormalize, scale, static_cast<uint32_t *>(out[0].data_ptr()), out[1].data_ptr(), wt, stream_here());
  });
}

// dweights, logits, inds, scoring, renormalize, scale
PyObject *select_experts_grad(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (!count_is(n, 6, "select_experts_grad")) return nullptr;
  Numbers num;
  Operands in;
  const int scoring = num.word(args[3], "softmax", MI_MOE_SCORING_SOFTMAX, "sigmoid", MI_MOE_SCORING_SIGMOID);
  const bool renormalize = num.truth(args[4]);
  const float scale = num.real(args[5]);
  const at::ScalarType type = type_of(args[1]), w_type = type_of(args[0]);
  const int dt = dtype_code(type), wt = dtype_code(w_type);
  if (dt < 0 || wt < 0 || !num.good) Py_RETURN_NONE;
  const at::Tensor &dw = in.add(args[0], w_type), &l = in.add(args[1], type), &id = in.add(args[2], at::kInt);
  if (!in.good || l.dim() < 1 || l.numel() == 0 || id.dim() != l.dim() || id.numel() == 0 || dw.sizes() != id.sizes() ||
      id.sizes().slice(0, id.dim() - 1) != l.sizes().slice(0, l.dim() - 1) || l.size(-1) > INT32_MAX || id.size(-1) > INT32_MAX)
    Py_RETURN_NONE;
  return call<1>([&](at::Tensor *out) {
    const int64_t E = l.size(-1);
    out[0] = at::empty(l.sizes(), l.options());
    return g_layer.select_grad(data_of(dw), wt, data_of(l), dt, static_cast<const uint32_t *>(data_of(id)), l.numel() / E, (int32_t)E, (int32_t)id.size(-1), scoring, renormalize,
                               scale, out[0].data_ptr(), stream_here());
  });
}

// bind_layer(addresses of the eight functions of g_layer, in its order)
PyObject *bind_layer(PyObject *, PyObject *args) {
  unsigned long long a[8];
  if (!PyArg_ParseTuple(args, "KKKKKKKK", a, a + 1, a + 2, a + 3, a + 4, a + 5, a + 6, a + 7)) return nullptr;
  g_layer = {reinterpret_cast<decltype(g_layer.norm)>(a[0]), reinterpret_cast<decltype(g_layer.norm_rows8)>(a[1]),
             reinterpret_cast<decltype(g_layer.norm_grad_workspace)>(a[2]), reinterpret_cast<decltype(g_layer.norm_grad)>(a[3]),
             reinterpret_cast<decltype(g_layer.rows8_workspace)>(a[4]), reinterpret_cast<decltype(g_layer.rows8)>(a[5]),
             reinterpret_cast<decltype(g_layer.select)>(a[6]), reinterpret_cast<decltype(g_layer.select_grad)>(a[7])};
  Py_RETURN_NONE;
}

// bind(addresses of the library's quantized_linear_typed, quantized_matmul_typed and quantized_matmul_workspace_size)
PyObject *bind(PyObject *, PyObject *args) {
  unsigned long long l = 0, m = 0, ws = 0;
  if (!PyArg_ParseTuple(args, "KKK", &l, &m, &ws)) return nullptr;
  g_linear = reinterpret_cast<decltype(g_linear)>(l);
  g_matmul = reinterpret_cast<decltype(g_matmul)>(m);
  g_workspace = reinterpret_cast<decltype(g_workspace)>(ws);
  Py_RETURN_NONE;
}

using Fast = PyObject *(PyObject *, PyObject *const *, Py_ssize_t);
PyCFunction fast(Fast *f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)); }

// an entry whose exceptions end in the interpreter's: a mode's own (written in Python) is the caller's; after any other (out of memory) the general path meets it again and words it
template <Fast *F>
PyObject *caught(PyObject *self, PyObject *const *args, Py_ssize_t n) {
  try {
    return F(self, args, n);
  } catch (python_error &e) {
    e.restore();
  } catch (pybind11::error_already_set &e) {
    e.restore();
  } catch (const std::exception &) {
  }
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"quantized_linear", fast(quantized_linear), METH_FASTCALL, nullptr},
    {"add_rms_norm", fast(caught<add_rms_norm>), METH_FASTCALL, nullptr},
    {"add_rms_norm_rows8", fast(caught<add_rms_norm_rows8>), METH_FASTCALL, nullptr},
    {"add_rms_norm_grad", fast(caught<add_rms_norm_grad>), METH_FASTCALL, nullptr},
    {"quantized_linear_rows8", fast(caught<quantized_linear_rows8>), METH_FASTCALL, nullptr},
    {"select_experts", fast(caught<select_experts>), METH_FASTCALL, nullptr},
    {"select_experts_grad", fast(caught<select_experts_grad>), METH_FASTCALL, nullptr},
    {"bind", bind, METH_VARARGS, nullptr},
    {"bind_layer", bind_layer, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_linear_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__linear_call() {
  PyObject *const m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "built_with", TORCH_VERSION)) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
