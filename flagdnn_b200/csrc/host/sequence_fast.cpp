// Steady-state host path of group norm and the state space operators: one native call from Python each.  The calls for
// single tokens run kernels of a few microseconds; argument checks and ctypes marshalling in Python cost 25 us a call.
//
// As in fastcall.cpp every function answers None for a call it does not take as it is; the Python implementation then runs
// (it makes what is not dense dense, differentiates, raises).  A status other than FDNN_OK is answered as an int.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Exceptions.h>

#include <cstring>

#include "host_common.h"

using namespace fdnn_host;

namespace {

using Bytes2Fn = int (*)(const fdnn_norm_desc*, int, int64_t*);
using NormFn = int (*)(const fdnn_norm_desc*, const void*, const void*, const void*, void*, float*, float*, void*, int64_t, void*);
using NormBackFn = int (*)(const fdnn_norm_desc*, const void*, const void*, const float*, const float*, const void*, const void*, void*,
                           void*, void*, void*, int64_t, void*);
using ConvFn = int (*)(const fdnn_causal_conv_desc*, const void*, const void*, const void*, const void*, const int32_t*, void*, void*,
                       void*);
using ConvStepFn = int (*)(const fdnn_causal_conv_desc*, const void*, const void*, const void*, void*, int32_t, const int32_t*, void*,
                           void*);
using BytesFn = int (*)(const fdnn_scan_desc*, int64_t*);
using ScanFn = int (*)(const fdnn_scan_desc*, const void*, const void*, const float*, const void*, const void*, const float*, const void*,
                       const float*, const float*, const int32_t*, void*, float*, void*, int64_t, void*);
using ScanStepFn = int (*)(const fdnn_scan_desc*, const void*, const void*, const float*, const void*, const void*, const float*,
                           const void*, const float*, float*, int32_t, const int32_t*, void*, void*);
Bytes2Fn g_norm_bytes = nullptr;
NormFn g_norm = nullptr;
NormBackFn g_norm_back = nullptr;
ConvFn g_conv = nullptr;
ConvStepFn g_conv_step = nullptr;
BytesFn g_scan_bytes = nullptr;
ScanFn g_scan = nullptr;
ScanStepFn g_scan_step = nullptr;

void strides4(const at::Tensor& t, int64_t* s) {
  s[0] = t.stride(0);
  s[1] = t.stride(1);
  if (t.dim() == 4) {
    s[2] = t.stride(2);
    s[3] = t.stride(3);
  } else if (t.dim() == 3) {
    s[2] = t.stride(2) * t.size(2);
    s[3] = t.stride(2);
  } else {
    s[2] = s[3] = s[1] * t.size(1);
  }
}

// A dense tensor of x's shape: channels last where x has its channels together, contiguous otherwise.
at::Tensor empty_like_layout(const at::Tensor& x) {
  const auto options = x.options().requires_grad(false);
  if (x.dim() == 2 || x.stride(1) != 1 || x.size(1) == 1) return at::empty(x.sizes(), options);
  const int64_t c = x.size(1);
  if (x.dim() == 3) return at::empty_strided(x.sizes(), {x.size(2) * c, 1, c}, options);
  return at::empty_strided(x.sizes(), {x.size(2) * x.size(3) * c, 1, x.size(3) * c, c}, options);
}

struct NormCall {
  const at::Tensor *x, *weight, *bias;
  fdnn_norm_desc d;
};
// The common part of both directions: false for calls that are left to Python.
bool norm_call(NormCall& k, PyObject* x, PyObject* groups, PyObject* weight, PyObject* bias, PyObject* act) {
  k.x = plain(x);
  if (k.x == nullptr || !optional(weight, &k.weight) || !optional(bias, &k.bias)) return false;
  if (k.x->dim() < 2 || k.x->dim() > 4 || k.x->numel() == 0 || !small(*k.x) || !PyLong_CheckExact(groups) || !PyLong_CheckExact(act))
    return false;
  const int dtype = dtype_code(k.x->scalar_type());
  const int64_t c = k.x->size(1), g = PyLong_AsLongLong(groups);
  if (dtype < 0 || g < 1 || c % g != 0) {
    PyErr_Clear();
    return false;
  }
  const at::Tensor* p = k.weight != nullptr ? k.weight : k.bias;
  const at::ScalarType type = p == nullptr ? k.x->scalar_type() : p->scalar_type();
  if (type != k.x->scalar_type() && type != at::kFloat) return false;
  if (!dense(k.weight, type, {c}, *k.x) || !dense(k.bias, type, {c}, *k.x)) return false;
  fdnn_norm_desc& d = k.d;
  std::memset(&d, 0, sizeof d);
  d.dtype = dtype;
  d.param_dtype = dtype_code(type);
  d.n = int(k.x->size(0));
  d.c = int(c);
  d.h = k.x->dim() == 4 ? int(k.x->size(2)) : 1;
  d.w = k.x->dim() == 4 ? int(k.x->size(3)) : k.x->dim() == 3 ? int(k.x->size(2)) : 1;
  d.groups = int(g);
  d.activation = int(PyLong_AsLong(act));
  strides4(*k.x, d.x_strides);
  return true;
}

// Values of 3-d tensors [N, L, C] (or 2-d [N, C], l_stride 0) in the descriptors' order.
void strides3(const at::Tensor& t, int64_t* s) {
  s[0] = t.stride(0);
  s[1] = t.dim() == 3 ? t.stride(1) : 0;
  s[2] = t.stride(t.dim() - 1);
}

bool conv_call(fdnn_causal_conv_desc& d, const at::Tensor* x, const at::Tensor* w, const at::Tensor* bias, int64_t dims, PyObject* act) {
  if (x == nullptr || w == nullptr || x->dim() != dims || w->dim() != 2 || !small(*x) || !PyLong_CheckExact(act)) return false;
  const int dtype = dtype_code(x->scalar_type());
  const int64_t c = x->size(dims - 1), width = w->size(1);
  if (dtype < 0 || width < 1 || width > FDNN_CAUSAL_CONV_MAX_WIDTH) return false;
  if (!dense(w, x->scalar_type(), {c, width}, *x) || !dense(bias, x->scalar_type(), {c}, *x)) return false;
  std::memset(&d, 0, sizeof d);
  d.dtype = dtype;
  d.n = int(x->size(0));
  d.l = dims == 3 ? int(x->size(1)) : 1;
  d.c = int(c);
  d.width = int(width);
  d.activation = int(PyLong_AsLong(act));
  strides3(*x, d.x_strides);
  return true;
}

struct ScanCall {
  const at::Tensor *u, *delta, *A, *B, *C, *D, *z, *bias;
  fdnn_scan_desc d;
};
// u, delta, A, B, C, D, z, delta_bias
bool scan_call(ScanCall& k, PyObject* const* a, PyObject* D, PyObject* z, PyObject* bias, PyObject* softplus, int64_t dims) {
  k.u = plain(a[0]);
  k.delta = plain(a[1]);
  k.A = plain(a[2]);
  k.B = plain(a[3]);
  k.C = plain(a[4]);
  if (k.u == nullptr || k.delta == nullptr || k.A == nullptr || k.B == nullptr || k.C == nullptr) return false;
  if (!optional(D, &k.D) || !optional(z, &k.z) || !optional(bias, &k.bias) || !PyBool_Check(softplus)) return false;
  const at::Tensor& u = *k.u;
  if (u.dim() != dims || k.A->dim() != 2 || !small(u)) return false;
  const int dtype = dtype_code(u.scalar_type());
  const int64_t c = u.size(dims - 1), s = k.A->size(1);
  if (dtype < 0 || s < 1 || s > FDNN_SCAN_MAX_STATES) return false;
  const int64_t groups = k.B->dim() == dims + 1 ? k.B->size(dims - 1) : 1;
  if (groups < 1 || groups > kMost || c % groups != 0) return false;
  for (const at::Tensor* t : {k.delta, k.z})
    if (t != nullptr && (t->sizes() != u.sizes() || t->scalar_type() != u.scalar_type() || t->device() != u.device())) return false;
  for (const at::Tensor* t : {k.B, k.C}) {
    if (t->scalar_type() != u.scalar_type() || t->device() != u.device() || (t->dim() != dims && t->dim() != dims + 1)) return false;
    for (int64_t i = 0; i < dims - 1; ++i)
      if (t->size(i) != u.size(i)) return false;
    if (t->size(t->dim() - 1) != s || (t->dim() == dims + 1 ? t->size(dims - 1) : 1) != groups) return false;
  }
  if (!dense(k.A, at::kFloat, {c, s}, u) || !dense(k.D, at::kFloat, {c}, u) || !dense(k.bias, at::kFloat, {c}, u)) return false;
  fdnn_scan_desc& d = k.d;
  std::memset(&d, 0, sizeof d);
  d.dtype = dtype;
  d.n = int(u.size(0));
  d.l = dims == 3 ? int(u.size(1)) : 1;
  d.c = int(c);
  d.s = int(s);
  d.groups = int(groups);
  d.delta_softplus = softplus == Py_True;
  strides3(u, d.u_strides);
  strides3(*k.delta, d.delta_strides);
  if (k.z != nullptr) strides3(*k.z, d.z_strides);
  const at::Tensor* bc[2] = {k.B, k.C};
  int64_t* to[2] = {d.b_strides, d.c_strides};
  for (int i = 0; i < 2; ++i) {
    const at::Tensor& t = *bc[i];
    to[i][0] = t.stride(0);
    to[i][1] = dims == 3 ? t.stride(1) : 0;
    to[i][2] = t.dim() == dims + 1 ? t.stride(dims - 1) : 0;
    to[i][3] = t.stride(t.dim() - 1);
  }
  return true;
}

}  // namespace

// group_norm(input, num_groups, weight, bias, eps, activation, return_stats)
PyObject* fast_group_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7 || g_norm == nullptr || !PyFloat_Check(a[4]) || !PyBool_Check(a[6])) return none();
  NormCall k;
  if (!norm_call(k, a[0], a[1], a[2], a[3], a[5]) || any_grad({k.x, k.weight, k.bias})) return none();
  k.d.eps = float(PyFloat_AsDouble(a[4]));
  c10::DeviceGuard guard(k.x->device());
  at::Tensor y, mean, rstd, scratch;
  int st;
  {
    WithoutGil free;
    y = empty_like_layout(*k.x);
    strides4(y, k.d.y_strides);
    const auto floats = k.x->options().dtype(at::kFloat).requires_grad(false);
    if (a[6] == Py_True) {
      mean = at::empty({k.d.n, k.d.groups}, floats);
      rstd = at::empty({k.d.n, k.d.groups}, floats);
    }
    int64_t bytes = 0;
    st = g_norm_bytes(&k.d, 0, &bytes);
    if (st == FDNN_OK) {
      if (bytes > 0) scratch = at::empty({bytes}, floats.dtype(at::kByte));
      st = g_norm(&k.d, k.x->const_data_ptr(), ptr(k.weight), ptr(k.bias), y.mutable_data_ptr(),
                  mean.defined() ? mean.mutable_data_ptr<float>() : nullptr, rstd.defined() ? rstd.mutable_data_ptr<float>() : nullptr,
                  bytes > 0 ? scratch.mutable_data_ptr() : nullptr, bytes, stream_of(*k.x));
    }
  }
  if (a[6] == Py_True) return answer(st, {y, mean, rstd});
  return answer(st, std::move(y));
  END_HANDLE_TH_ERRORS
}

// group_norm_backward(dy, input, mean, rstd, num_groups, weight, bias, activation)
PyObject* fast_group_norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8 || g_norm_back == nullptr) return none();
  NormCall k;
  const at::Tensor *dy = plain(a[0]), *mean = plain(a[2]), *rstd = plain(a[3]);
  if (dy == nullptr || mean == nullptr || rstd == nullptr || !norm_call(k, a[1], a[4], a[5], a[6], a[7])) return none();
  if (dy->sizes() != k.x->sizes() || dy->scalar_type() != k.x->scalar_type() || dy->device() != k.x->device()) return none();
  if (!dense(mean, at::kFloat, {k.d.n, k.d.groups}, *k.x) || !dense(rstd, at::kFloat, {k.d.n, k.d.groups}, *k.x)) return none();
  if (any_grad({dy, k.x, mean, rstd, k.weight, k.bias})) return none();
  c10::DeviceGuard guard(k.x->device());
  at::Tensor dx, dw, db, scratch;
  int st;
  {
    WithoutGil free;
    dx = empty_like_layout(*k.x);
    strides4(*dy, k.d.dy_strides);
    strides4(dx, k.d.dx_strides);
    if (k.weight != nullptr) dw = at::empty(k.weight->sizes(), k.weight->options().requires_grad(false));
    if (k.bias != nullptr) db = at::empty(k.bias->sizes(), k.bias->options().requires_grad(false));
    int64_t bytes = 0;
    st = g_norm_bytes(&k.d, 1, &bytes);
    if (st == FDNN_OK) {
      if (bytes > 0) scratch = at::empty({bytes}, k.x->options().dtype(at::kByte).requires_grad(false));
      st = g_norm_back(&k.d, dy->const_data_ptr(), k.x->const_data_ptr(), f32(mean), f32(rstd), ptr(k.weight), ptr(k.bias),
                       dx.mutable_data_ptr(), dw.defined() ? dw.mutable_data_ptr() : nullptr, db.defined() ? db.mutable_data_ptr() : nullptr,
                       bytes > 0 ? scratch.mutable_data_ptr() : nullptr, bytes, stream_of(*k.x));
    }
  }
  return answer(st, {dx, dw, db});
  END_HANDLE_TH_ERRORS
}

// causal_conv1d(x, weight, bias, activation, initial_state, lengths, return_final_state)
PyObject* fast_causal_conv1d(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7 || g_conv == nullptr || !PyBool_Check(a[6])) return none();
  const at::Tensor *x = plain(a[0]), *w = plain(a[1]), *bias, *initial, *lengths;
  if (!optional(a[2], &bias) || !optional(a[4], &initial) || !optional(a[5], &lengths)) return none();
  fdnn_causal_conv_desc d;
  if (!conv_call(d, x, w, bias, 3, a[3]) || any_grad({x, w, bias, initial})) return none();
  const std::array<int64_t, 3> state{d.n, d.width - 1, d.c};
  if (!dense(initial, x->scalar_type(), state, *x) || !dense(lengths, at::kInt, {d.n}, *x)) return none();
  c10::DeviceGuard guard(x->device());
  at::Tensor y, final;
  int st;
  {
    WithoutGil free;
    const auto options = x->options().requires_grad(false);
    y = at::empty({d.n, d.l, d.c}, options);
    strides3(y, d.y_strides);
    if (a[6] == Py_True) final = at::empty(state, options);
    st = g_conv(&d, x->const_data_ptr(), w->const_data_ptr(), ptr(bias), ptr(initial), i32(lengths), y.mutable_data_ptr(),
                final.defined() ? final.mutable_data_ptr() : nullptr, stream_of(*x));
  }
  if (a[6] == Py_True) return answer(st, {y, final});
  return answer(st, std::move(y));
  END_HANDLE_TH_ERRORS
}

// causal_conv1d_step(x, conv_state, weight, bias, activation, slots)
PyObject* fast_causal_conv1d_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || g_conv_step == nullptr) return none();
  const at::Tensor *x = plain(a[0]), *state = plain(a[1]), *w = plain(a[2]), *bias, *slots;
  if (state == nullptr || !optional(a[3], &bias) || !optional(a[5], &slots)) return none();
  fdnn_causal_conv_desc d;
  if (!conv_call(d, x, w, bias, 2, a[4]) || any_grad({x, state, w, bias}) || state->dim() != 3) return none();
  const int64_t cache = state->size(0);
  if (cache > kMost || (slots == nullptr && cache < d.n)) return none();
  if (!dense(state, x->scalar_type(), {cache, d.width - 1, d.c}, *x) || !dense(slots, at::kInt, {d.n}, *x)) return none();
  c10::DeviceGuard guard(x->device());
  at::Tensor y;
  int st;
  {
    WithoutGil free;
    y = at::empty({d.n, d.c}, x->options().requires_grad(false));
    strides3(y, d.y_strides);
    st = g_conv_step(&d, x->const_data_ptr(), w->const_data_ptr(), ptr(bias), state->mutable_data_ptr(), int32_t(cache), i32(slots),
                     y.mutable_data_ptr(), stream_of(*x));
  }
  if (st == FDNN_OK) written(*state);
  return answer(st, std::move(y));
  END_HANDLE_TH_ERRORS
}

// selective_scan(u, delta, A, B, C, D, z, delta_bias, delta_softplus, initial_state, lengths, return_final_state)
PyObject* fast_selective_scan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 12 || g_scan == nullptr || !PyBool_Check(a[11])) return none();
  ScanCall k;
  const at::Tensor *initial, *lengths;
  if (!scan_call(k, a, a[5], a[6], a[7], a[8], 3) || !optional(a[9], &initial) || !optional(a[10], &lengths)) return none();
  if (any_grad({k.u, k.delta, k.A, k.B, k.C, k.D, k.z, k.bias, initial})) return none();
  const at::Tensor& u = *k.u;
  const std::array<int64_t, 3> state{k.d.n, k.d.c, k.d.s};
  if (!dense(initial, at::kFloat, state, u) || !dense(lengths, at::kInt, {k.d.n}, u)) return none();
  c10::DeviceGuard guard(u.device());
  at::Tensor y, final, scratch;
  int st;
  {
    WithoutGil free;
    const auto options = u.options().requires_grad(false);
    y = at::empty(u.sizes(), options);
    strides3(y, k.d.y_strides);
    if (a[11] == Py_True) final = at::empty(state, options.dtype(at::kFloat));
    int64_t bytes = 0;
    st = g_scan_bytes(&k.d, &bytes);
    if (st == FDNN_OK) {
      if (bytes > 0) scratch = at::empty({bytes}, options.dtype(at::kByte));
      st = g_scan(&k.d, u.const_data_ptr(), k.delta->const_data_ptr(), f32(k.A), k.B->const_data_ptr(), k.C->const_data_ptr(), f32(k.D),
                  ptr(k.z), f32(k.bias), f32(initial), i32(lengths), y.mutable_data_ptr(),
                  final.defined() ? final.mutable_data_ptr<float>() : nullptr, bytes > 0 ? scratch.mutable_data_ptr() : nullptr, bytes,
                  stream_of(u));
    }
  }
  if (a[11] == Py_True) return answer(st, {y, final});
  return answer(st, std::move(y));
  END_HANDLE_TH_ERRORS
}

// selective_scan_step(u, delta, A, B, C, state, D, z, delta_bias, delta_softplus, slots)
PyObject* fast_selective_scan_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 11 || g_scan_step == nullptr) return none();
  ScanCall k;
  const at::Tensor *state = plain(a[5]), *slots;
  if (state == nullptr || !scan_call(k, a, a[6], a[7], a[8], a[9], 2) || !optional(a[10], &slots)) return none();
  if (any_grad({k.u, k.delta, k.A, k.B, k.C, k.D, k.z, k.bias, state}) || state->dim() != 3) return none();
  const at::Tensor& u = *k.u;
  const int64_t cache = state->size(0);
  if (cache > kMost || (slots == nullptr && cache < k.d.n)) return none();
  if (!dense(state, at::kFloat, {cache, k.d.c, k.d.s}, u) || !dense(slots, at::kInt, {k.d.n}, u)) return none();
  c10::DeviceGuard guard(u.device());
  at::Tensor y;
  int st;
  {
    WithoutGil free;
    y = at::empty(u.sizes(), u.options().requires_grad(false));
    strides3(y, k.d.y_strides);
    st = g_scan_step(&k.d, u.const_data_ptr(), k.delta->const_data_ptr(), f32(k.A), k.B->const_data_ptr(), k.C->const_data_ptr(), f32(k.D),
                     ptr(k.z), f32(k.bias), state->mutable_data_ptr<float>(), int32_t(cache), i32(slots), y.mutable_data_ptr(), stream_of(u));
  }
  if (st == FDNN_OK) written(*state);
  return answer(st, std::move(y));
  END_HANDLE_TH_ERRORS
}

// bind_sequence(addresses of the eight functions in the order above, then the sizes of the three descriptors as the caller
// knows them): refuses a caller of other structures.
PyObject* bind_sequence(PyObject*, PyObject* args) {
  unsigned long long f[8], norm_bytes, conv_bytes, scan_bytes;
  if (!PyArg_ParseTuple(args, "KKKKKKKKKKK", &f[0], &f[1], &f[2], &f[3], &f[4], &f[5], &f[6], &f[7], &norm_bytes, &conv_bytes, &scan_bytes))
    return nullptr;
  if (norm_bytes != sizeof(fdnn_norm_desc) || conv_bytes != sizeof(fdnn_causal_conv_desc) || scan_bytes != sizeof(fdnn_scan_desc)) {
    PyErr_SetString(PyExc_ImportError, "compiled for other descriptors of the C ABI");
    return nullptr;
  }
  g_norm_bytes = reinterpret_cast<Bytes2Fn>(uintptr_t(f[0]));
  g_norm = reinterpret_cast<NormFn>(uintptr_t(f[1]));
  g_norm_back = reinterpret_cast<NormBackFn>(uintptr_t(f[2]));
  g_conv = reinterpret_cast<ConvFn>(uintptr_t(f[3]));
  g_conv_step = reinterpret_cast<ConvStepFn>(uintptr_t(f[4]));
  g_scan_bytes = reinterpret_cast<BytesFn>(uintptr_t(f[5]));
  g_scan = reinterpret_cast<ScanFn>(uintptr_t(f[6]));
  g_scan_step = reinterpret_cast<ScanStepFn>(uintptr_t(f[7]));
  return none();
}
