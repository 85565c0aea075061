// Python calls of the mixture-of-experts layer's operators (dense, moe_route,
// moe_combine and their gradients) on torch tensors: checks of arguments,
// outputs from torch's allocator, the current stream, one call of the C ABI.
//
// The C ABI itself is reached as everywhere in the package: the library is
// loaded by ctypes (cutile_b200/_lib.py), which hands the entry points'
// addresses to bind(). What this file replaces is the Python between the user
// and the library: 11 us a call, against 2.5 us for a kernel launch, which is
// what the smallest calls (one token) consist of.
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "../../include/cutile_b200.h"

namespace {

// ---- the library's entry points, set by bind() ---------------------------------------
#define CTB_FUNCTIONS(F) \
  F(ctb_last_error)      \
  F(ctb_dense_fwd_workspace_bytes) F(ctb_dense_fwd) F(ctb_dense_bwd_workspace_bytes) \
  F(ctb_dense_bwd) F(ctb_moe_route) F(ctb_moe_route_bwd) F(ctb_moe_combine)          \
  F(ctb_moe_combine_bwd)
struct Library {
#define CTB_DECLARE(name) decltype(&::name) name = nullptr;
  CTB_FUNCTIONS(CTB_DECLARE)
#undef CTB_DECLARE
} lib;
PyObject* g_error = nullptr;  // cutile_b200.B200Error

// ---- errors: B200Error(code, message), raised as a C++ exception until the boundary ------
struct Refused {
  int code;
  std::string message;
};
[[noreturn]] void refuse(int code, const std::string& message) { throw Refused{code, message}; }

void raise_refused(const Refused& r) {
  PyObject* e = PyObject_CallFunction(g_error, "is", r.code, r.message.c_str());
  if (e) {
    PyErr_SetObject(g_error, e);
    Py_DECREF(e);
  }
}
void check(int rc) {
  if (rc != CTB_OK) refuse(rc, lib.ctb_last_error());
}

// ---- arguments -----------------------------------------------------------------------------
using at::Tensor;

std::string text(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}
int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return CTB_F16;
    case at::kBFloat16: return CTB_BF16;
    case at::kFloat: return CTB_F32;
    case at::kDouble: return CTB_F64;
    case at::kInt: return CTB_I32;
    default: return 0;
  }
}
bool given(PyObject* o) { return o != Py_None; }

const Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) refuse(CTB_ERR_ARG, std::string(what) + ": expected a CUDA tensor");
  return THPVariable_Unpack(o);
}
int64_t integer(PyObject* o, const char* what) {
  if (!PyLong_Check(o)) refuse(CTB_ERR_ARG, std::string(what) + ": expected an integer");
  int over = 0;
  const int64_t v = PyLong_AsLongLongAndOverflow(o, &over);
  if (over) refuse(CTB_ERR_SHAPE, std::string(what) + ": out of range");
  return v;
}
int int32(int64_t v, const char* what) {
  if (v < INT32_MIN || v > INT32_MAX) refuse(CTB_ERR_SHAPE, std::string(what) + ": out of range");
  return (int)v;
}
float real(PyObject* o, const char* what) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(CTB_ERR_ARG, std::string(what) + ": expected a number");
  }
  return (float)v;
}
bool truth(PyObject* o, const char* what) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) {
    PyErr_Clear();
    refuse(CTB_ERR_ARG, std::string(what) + ": expected a truth value");
  }
  return v == 1;
}

// A call's first matrix, whose shape, dtype and device the others are held to.
const Tensor& rows(PyObject* o, const char* what) {
  const Tensor& t = tensor(o, what);
  if (!t.is_cuda()) refuse(CTB_ERR_ARG, std::string(what) + ": expected CUDA tensors");
  if (t.dim() != 2)
    refuse(CTB_ERR_SHAPE, std::string(what) + ": expected a matrix, got shape " + text(t));
  if (t.size(1) > 1 && t.stride(1) != 1)
    refuse(CTB_ERR_LAYOUT, std::string(what) + ": rows must be contiguous");
  int32(t.size(0), what);
  int32(t.size(1), what);
  return t;
}
void same(const Tensor& t, at::ScalarType dtype, at::Device device, const char* what) {
  if (t.device() != device)
    refuse(CTB_ERR_ARG, std::string(what) + ": expected a CUDA tensor on " + device.str() +
                            ", got " + t.device().str());
  if (t.scalar_type() != dtype)
    refuse(CTB_ERR_DTYPE, std::string(what) + ": expected " + c10::toString(dtype) + ", got " +
                              c10::toString(t.scalar_type()));
}
const Tensor& matrix(PyObject* o, int64_t r, int64_t c, at::ScalarType dtype, at::Device device,
                     const char* what) {
  const Tensor& t = tensor(o, what);
  same(t, dtype, device, what);
  if (t.dim() != 2 || t.size(0) != r || t.size(1) != c)
    refuse(CTB_ERR_SHAPE, std::string(what) + ": expected shape (" + std::to_string(r) + ", " +
                              std::to_string(c) + "), got " + text(t));
  if (c > 1 && t.stride(1) != 1)
    refuse(CTB_ERR_LAYOUT, std::string(what) + ": rows must be contiguous");
  return t;
}
const Tensor& packed(PyObject* o, int64_t r, int64_t c, at::ScalarType dtype, at::Device device,
                     const char* what) {
  const Tensor& t = matrix(o, r, c, dtype, device, what);
  if (!t.is_contiguous()) refuse(CTB_ERR_LAYOUT, std::string(what) + ": must be contiguous");
  return t;
}
const Tensor& vector(PyObject* o, int64_t n, at::ScalarType dtype, at::Device device,
                     const char* what) {
  const Tensor& t = tensor(o, what);
  same(t, dtype, device, what);
  if (t.dim() != 1 || t.size(0) != n)
    refuse(CTB_ERR_SHAPE, std::string(what) + ": expected shape (" + std::to_string(n) +
                              "), got " + text(t));
  if (!t.is_contiguous()) refuse(CTB_ERR_LAYOUT, std::string(what) + ": must be contiguous");
  return t;
}
Tensor new_matrix(int64_t r, int64_t c, at::ScalarType dtype, at::Device device) {
  return Tensor(at::detail::empty_strided_cuda({r, c}, {c > 0 ? c : 1, 1}, dtype, device));
}
Tensor new_vector(int64_t n, at::ScalarType dtype, at::Device device) {
  return Tensor(at::detail::empty_strided_cuda({n}, {1}, dtype, device));
}
// Row stride for the C ABI. A single row has none that matters (torch gives any
// number for it): its length does.
int64_t ld(const Tensor& t) {
  return t.size(0) > 1 ? t.stride(0) : std::max<int64_t>(t.size(1), 1);
}
void* ptr(const Tensor& t) { return t.data_ptr(); }

PyObject* pair_of(Tensor a, Tensor b) {
  PyObject* r = PyTuple_New(2);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, a.defined() ? THPVariable_Wrap(std::move(a)) : Py_NewRef(Py_None));
  PyTuple_SET_ITEM(r, 1, b.defined() ? THPVariable_Wrap(std::move(b)) : Py_NewRef(Py_None));
  return r;
}

// Runs on the tensors' device, which need not be the current one.
struct On {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit On(at::Device d)
      : guard(d), stream(c10::cuda::getCurrentCUDAStream(d.index()).stream()) {}
};

void count(Py_ssize_t got, Py_ssize_t want, const char* what) {
  if (got != want) refuse(CTB_ERR_ARG, std::string(what) + ": wrong number of arguments");
}

// ---- dense layer -------------------------------------------------------------------------------
struct Layer {
  const Tensor &A, &B;
  int M, N, K;
  at::ScalarType dt;
  at::Device dev;
};
Layer layer(PyObject* a, PyObject* b, const char* k) {
  const Tensor &A = rows(a, k), &B = rows(b, k);
  const auto dt = A.scalar_type();
  if ((dt != at::kHalf && dt != at::kBFloat16) || B.scalar_type() != dt)
    refuse(CTB_ERR_DTYPE, std::string(k) + ": A_t and B_t must both be float16 or both bfloat16");
  if (A.size(0) != B.size(1))
    refuse(CTB_ERR_SHAPE, std::string(k) + ": A_t must be (K, M), B_t (N, K); got " + text(A) +
                              " and " + text(B));
  if (A.device() != B.device())
    refuse(CTB_ERR_ARG, std::string(k) + ": A_t and B_t are on different devices");
  return {A, B, (int)A.size(1), (int)B.size(0), (int)A.size(0), dt, A.device()};
}
bool lines16(const Tensor& t, int64_t stride) {
  return (reinterpret_cast<uintptr_t>(ptr(t)) & 15) == 0 && (stride & 7) == 0;
}
// Scratch of one call: from torch's allocator, which keeps it to this stream's
// order and, in a capture, to the graph.
Tensor scratch(int64_t bytes, at::Device dev) {
  return bytes > 0 ? new_vector(bytes, at::kByte, dev) : Tensor();
}

PyObject* dense(PyObject* const* v) {
  const Layer l = layer(v[0], v[1], "dense");
  const void *bias = nullptr, *res = nullptr;
  void* pre = nullptr;
  int bias_dt = 0;
  int64_t ldr = 0, ldz = 0;
  if (given(v[2])) {
    const Tensor& b = tensor(v[2], "dense: bias");
    vector(v[2], l.M, b.scalar_type() == at::kFloat ? at::kFloat : l.dt, l.dev, "dense: bias");
    bias = ptr(b);
    bias_dt = dtype_code(b.scalar_type());
  }
  const int act = (int)integer(v[3], "dense: act");
  if (given(v[4])) {
    const Tensor& r = matrix(v[4], l.N, l.M, l.dt, l.dev, "dense: residual");
    res = ptr(r);
    ldr = ld(r);
  }
  if (given(v[6])) {
    const Tensor& z = matrix(v[6], l.N, l.M, l.dt, l.dev, "dense: preact");
    pre = ptr(z);
    ldz = ld(z);
  }
  if (given(v[5])) matrix(v[5], l.N, l.M, l.dt, l.dev, "dense: out");
  On on(l.dev);
  Tensor out = given(v[5]) ? THPVariable_Unpack(v[5]) : new_matrix(l.N, l.M, l.dt, l.dev);
  const int64_t lda = ld(l.A), ldb = ld(l.B);
  int64_t bytes = 0;
  if (!lines16(l.A, lda) || !lines16(l.B, ldb))
    bytes = lib.ctb_dense_fwd_workspace_bytes(ptr(l.A), ptr(l.B), l.M, l.N, l.K, lda, ldb);
  const Tensor ws = scratch(bytes, l.dev);
  check(lib.ctb_dense_fwd(dtype_code(l.dt), ptr(l.A), ptr(l.B), bias, bias_dt, res, pre, ptr(out),
                          l.M, l.N, l.K, lda, ldb, ldr, ldz, ld(out), act,
                          bytes > 0 ? ptr(ws) : nullptr, bytes, on.stream));
  return THPVariable_Wrap(std::move(out));
}

PyObject* dense_bwd(PyObject* const* v) {
  const Layer l = layer(v[1], v[2], "dense_bwd");
  const Tensor& dC = matrix(v[0], l.N, l.M, l.dt, l.dev, "dense_bwd: dC_t");
  const int act = (int)integer(v[3], "dense_bwd: act");
  const void* pre = nullptr;
  int64_t ldz = 0;
  if (act != CTB_ACT_NONE) {
    if (!given(v[4])) refuse(CTB_ERR_ARG, "dense_bwd: an activation's gradient needs preact");
    const Tensor& z = matrix(v[4], l.N, l.M, l.dt, l.dev, "dense_bwd: preact");
    pre = ptr(z);
    ldz = ld(z);
  }
  const bool need[3] = {truth(v[8], "dense_bwd: need_dA"), truth(v[9], "dense_bwd: need_dB"),
                        truth(v[10], "dense_bwd: need_dbias")};
  if (need[0] && given(v[5])) matrix(v[5], l.K, l.M, l.dt, l.dev, "dense_bwd: dA_t");
  if (need[1] && given(v[6])) matrix(v[6], l.N, l.K, l.dt, l.dev, "dense_bwd: dB_t");
  if (need[2] && given(v[7])) vector(v[7], l.M, at::kFloat, l.dev, "dense_bwd: dbias");
  On on(l.dev);
  Tensor out[3];
  for (int i = 0; i < 3; ++i) {
    if (!need[i]) continue;
    if (given(v[5 + i])) out[i] = THPVariable_Unpack(v[5 + i]);
    else if (i == 0) out[i] = new_matrix(l.K, l.M, l.dt, l.dev);
    else if (i == 1) out[i] = new_matrix(l.N, l.K, l.dt, l.dev);
    else out[i] = new_vector(l.M, at::kFloat, l.dev);
  }
  const int64_t lddc = ld(dC), lda = ld(l.A), ldb = ld(l.B);
  const int64_t bytes = lib.ctb_dense_bwd_workspace_bytes(
      ptr(dC), ptr(l.A), ptr(l.B), l.M, l.N, l.K, lddc, lda, ldb, act, need[2] ? 1 : 0);
  const Tensor ws = scratch(bytes, l.dev);
  check(lib.ctb_dense_bwd(dtype_code(l.dt), ptr(dC), ptr(l.A), ptr(l.B), pre,
                          need[0] ? ptr(out[0]) : nullptr, need[1] ? ptr(out[1]) : nullptr,
                          need[2] ? static_cast<float*>(ptr(out[2])) : nullptr, l.M, l.N, l.K,
                          lddc, lda, ldb, ldz, need[0] ? ld(out[0]) : 0, need[1] ? ld(out[1]) : 0,
                          act, bytes > 0 ? ptr(ws) : nullptr, bytes, on.stream));
  PyObject* r = PyTuple_New(3);
  if (!r) return nullptr;
  for (int i = 0; i < 3; ++i)
    PyTuple_SET_ITEM(r, i, need[i] ? THPVariable_Wrap(std::move(out[i])) : Py_NewRef(Py_None));
  return r;
}

// ---- routing -------------------------------------------------------------------------------------
// (logits, topk, score, bias, groups, topk_groups, group_top, renorm, scale, weights, ids)
PyObject* moe_route(PyObject* const* v) {
  const Tensor& x = rows(v[0], "moe_route: logits");
  const int T = (int)x.size(0), E = (int)x.size(1);
  const at::Device dev = x.device();
  const int topk = int32(integer(v[1], "moe_route: topk"), "moe_route: topk");
  if (topk < 1) refuse(CTB_ERR_SHAPE, "moe_route: topk must be positive");
  const int score = (int)integer(v[2], "moe_route: score");
  const int groups = int32(integer(v[4], "moe_route: groups"), "moe_route: groups");
  const int kept = given(v[5]) ? int32(integer(v[5], "moe_route: topk_groups"),
                                       "moe_route: topk_groups") : groups;
  const int top = int32(integer(v[6], "moe_route: group_top"), "moe_route: group_top");
  const float* bias = nullptr;
  if (given(v[3]))
    bias = static_cast<const float*>(ptr(vector(v[3], E, at::kFloat, dev, "moe_route: bias")));
  if (given(v[9])) packed(v[9], T, topk, at::kFloat, dev, "moe_route: weights");
  if (given(v[10])) packed(v[10], T, topk, at::kInt, dev, "moe_route: ids");
  const float scale = real(v[8], "moe_route: scale");
  const int renorm = truth(v[7], "moe_route: renorm") ? 1 : 0;
  On on(dev);
  Tensor w = given(v[9]) ? THPVariable_Unpack(v[9]) : new_matrix(T, topk, at::kFloat, dev);
  Tensor i = given(v[10]) ? THPVariable_Unpack(v[10]) : new_matrix(T, topk, at::kInt, dev);
  check(lib.ctb_moe_route(dtype_code(x.scalar_type()), ptr(x), bias, static_cast<float*>(ptr(w)),
                          static_cast<int32_t*>(ptr(i)), T, E, topk, ld(x), score, groups, kept,
                          top, renorm, scale, on.stream));
  return pair_of(std::move(w), std::move(i));
}

// (dweights, logits, ids, score, renorm, scale, dlogits)
PyObject* moe_route_bwd(PyObject* const* v) {
  const Tensor& x = rows(v[1], "moe_route_bwd: logits");
  const Tensor& i = rows(v[2], "moe_route_bwd: ids");
  const int T = (int)x.size(0), E = (int)x.size(1), topk = (int)i.size(1);
  const at::Device dev = x.device();
  packed(v[2], T, topk, at::kInt, dev, "moe_route_bwd: ids");
  const Tensor& dw = packed(v[0], T, topk, at::kFloat, dev, "moe_route_bwd: dweights");
  if (given(v[6])) matrix(v[6], T, E, x.scalar_type(), dev, "moe_route_bwd: dlogits");
  const int score = (int)integer(v[3], "moe_route_bwd: score");
  const float scale = real(v[5], "moe_route_bwd: scale");
  const int renorm = truth(v[4], "moe_route_bwd: renorm") ? 1 : 0;
  On on(dev);
  Tensor dx = given(v[6]) ? THPVariable_Unpack(v[6]) : new_matrix(T, E, x.scalar_type(), dev);
  check(lib.ctb_moe_route_bwd(dtype_code(x.scalar_type()), static_cast<const float*>(ptr(dw)),
                              ptr(x), static_cast<const int32_t*>(ptr(i)), ptr(dx), T, E, topk,
                              ld(x), ld(dx), score, renorm, scale, on.stream));
  return THPVariable_Wrap(std::move(dx));
}

// ---- combine -------------------------------------------------------------------------------------
struct Slots {
  const float* weights = nullptr;
  const int32_t* ids = nullptr;
  int E = 0;
};
Slots slots(PyObject* w, PyObject* i, PyObject* experts, int64_t T, int topk, at::Device dev) {
  Slots s;
  if (given(w))
    s.weights = static_cast<const float*>(ptr(packed(w, T, topk, at::kFloat, dev, "weights")));
  if (given(i)) {
    s.ids = static_cast<const int32_t*>(ptr(packed(i, T, topk, at::kInt, dev, "ids")));
    if (!given(experts)) refuse(CTB_ERR_ARG, "ids need num_experts");
    s.E = int32(integer(experts, "num_experts"), "num_experts");
  }
  return s;
}

// (y, topk, weights, ids, num_experts, residual, out)
PyObject* moe_combine(PyObject* const* v) {
  const Tensor& y = rows(v[0], "moe_combine: y");
  const int topk = int32(integer(v[1], "moe_combine: topk"), "moe_combine: topk");
  if (topk < 1 || y.size(0) % topk != 0)
    refuse(CTB_ERR_SHAPE, "moe_combine: y must have T * topk rows, topk positive");
  const int T = (int)(y.size(0) / topk), N = (int)y.size(1);
  const auto dt = y.scalar_type();
  const at::Device dev = y.device();
  const Slots s = slots(v[2], v[3], v[4], T, topk, dev);
  const void* res = nullptr;
  int64_t ldr = 0;
  if (given(v[5])) {
    const Tensor& r = matrix(v[5], T, N, dt, dev, "moe_combine: residual");
    res = ptr(r);
    ldr = ld(r);
  }
  if (given(v[6])) matrix(v[6], T, N, dt, dev, "moe_combine: out");
  On on(dev);
  Tensor out = given(v[6]) ? THPVariable_Unpack(v[6]) : new_matrix(T, N, dt, dev);
  check(lib.ctb_moe_combine(dtype_code(dt), ptr(y), s.weights, s.ids, res, ptr(out), T, topk, N,
                            s.E, ld(y), ldr, ld(out), on.stream));
  return THPVariable_Wrap(std::move(out));
}

// (dout, y, topk, weights, ids, num_experts, dy, dweights)
PyObject* moe_combine_bwd(PyObject* const* v) {
  const Tensor& d = rows(v[0], "moe_combine_bwd: dout");
  const int topk = int32(integer(v[2], "moe_combine_bwd: topk"), "moe_combine_bwd: topk");
  if (topk < 1) refuse(CTB_ERR_SHAPE, "moe_combine_bwd: topk must be positive");
  const int T = (int)d.size(0), N = (int)d.size(1);
  const int64_t n = (int64_t)T * topk;
  const auto dt = d.scalar_type();
  const at::Device dev = d.device();
  const Slots s = slots(v[3], v[4], v[5], T, topk, dev);
  const void* y = nullptr;
  int64_t ldy = 0;
  if (given(v[3])) {
    const Tensor& t = matrix(v[1], n, N, dt, dev, "moe_combine_bwd: y");
    y = ptr(t);
    ldy = ld(t);
    if (given(v[7])) packed(v[7], T, topk, at::kFloat, dev, "moe_combine_bwd: dweights");
  } else if (given(v[7])) {
    refuse(CTB_ERR_ARG, "moe_combine_bwd: dweights without weights");
  }
  if (given(v[6])) matrix(v[6], n, N, dt, dev, "moe_combine_bwd: dy");
  On on(dev);
  Tensor dw;
  if (given(v[3]))
    dw = given(v[7]) ? THPVariable_Unpack(v[7]) : new_matrix(T, topk, at::kFloat, dev);
  Tensor dy = given(v[6]) ? THPVariable_Unpack(v[6]) : new_matrix(n, N, dt, dev);
  check(lib.ctb_moe_combine_bwd(dtype_code(dt), ptr(d), y, s.weights, s.ids, ptr(dy),
                                dw.defined() ? static_cast<float*>(ptr(dw)) : nullptr, T, topk, N,
                                s.E, ld(d), ldy, ld(dy), on.stream));
  return pair_of(std::move(dy), std::move(dw));
}

// ---- module ----------------------------------------------------------------------------------------
template <PyObject* (*F)(PyObject* const*), int ARGS>
PyObject* entry(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    if (!g_error) {
      PyErr_SetString(PyExc_RuntimeError, "bind() has not been called");
      return nullptr;
    }
    count(n, ARGS, "cutile_b200");
    return F(v);
  } catch (const Refused& r) {
    raise_refused(r);
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// bind(addresses: dict name -> int, error type)
PyObject* bind(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (n != 2 || !PyDict_Check(v[0])) {
    PyErr_SetString(PyExc_TypeError, "bind(addresses, error)");
    return nullptr;
  }
#define CTB_TAKE(name)                                                                   \
  {                                                                                      \
    PyObject* o = PyDict_GetItemString(v[0], #name);                                     \
    void* p = o ? PyLong_AsVoidPtr(o) : nullptr;                                         \
    if (!p) {                                                                            \
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_KeyError, #name);                     \
      return nullptr;                                                                    \
    }                                                                                    \
    lib.name = reinterpret_cast<decltype(lib.name)>(p);                                  \
  }
  CTB_FUNCTIONS(CTB_TAKE)
#undef CTB_TAKE
  Py_XSETREF(g_error, Py_NewRef(v[1]));
  Py_RETURN_NONE;
}

#define CTB_ENTRY(name, args) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<name, args>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&bind)), METH_FASTCALL,
     nullptr},
    CTB_ENTRY(dense, 7),         CTB_ENTRY(dense_bwd, 11),  CTB_ENTRY(moe_route, 11),
    CTB_ENTRY(moe_route_bwd, 7), CTB_ENTRY(moe_combine, 7), CTB_ENTRY(moe_combine_bwd, 8),
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_torch_binding", nullptr, -1, methods,
                          nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_binding() { return PyModule_Create(&module_def); }
