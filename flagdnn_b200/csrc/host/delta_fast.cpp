// Steady-state host path of the gated delta rule: one native call from Python each, as in sequence_fast.cpp.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Exceptions.h>

#include <cmath>
#include <cstring>

#include "host_common.h"

using namespace fdnn_host;

namespace {

using BytesFn = int (*)(const fdnn_delta_rule_desc*, int64_t*);
using RuleFn = int (*)(const fdnn_delta_rule_desc*, const void*, const void*, const void*, const void*, const void*, const float*,
                       const float*, const float*, const int32_t*, void*, float*, void*, int64_t, void*);
using StepFn = int (*)(const fdnn_delta_rule_desc*, const void*, const void*, const void*, const void*, const void*, const float*,
                       const float*, float*, int32_t, const int32_t*, void*, void*);
BytesFn g_bytes = nullptr;
RuleFn g_rule = nullptr;
StepFn g_step = nullptr;

struct Call {
  const at::Tensor *q, *k, *v, *delta, *beta, *A, *bias;
  fdnn_delta_rule_desc d;
};

// The strides of [N, L, ...] (or [N, ...]: l stride 0) in the descriptor's order.
void strides(const at::Tensor& t, int64_t tokens, int64_t* s) {
  *s++ = t.stride(0);
  *s++ = tokens == 1 ? t.stride(1) : 0;
  for (int64_t i = 1 + tokens; i < t.dim(); ++i) *s++ = t.stride(i);
}

// q, k, v, delta, beta at `a`; A, delta_bias, softplus, sigmoid, norm, scale at `o`.  tokens: 1 with a token dimension, else 0.
bool call_of(Call& c, PyObject* const* a, PyObject* const* o, int64_t tokens) {
  const at::Tensor** five[5] = {&c.q, &c.k, &c.v, &c.delta, &c.beta};
  for (int i = 0; i < 5; ++i)
    if ((*five[i] = plain(a[i])) == nullptr) return false;
  if (!optional(o[0], &c.A) || !optional(o[1], &c.bias)) return false;
  if (!PyBool_Check(o[2]) || !PyBool_Check(o[3]) || !PyBool_Check(o[4]) || (o[5] != Py_None && !PyFloat_CheckExact(o[5]))) return false;
  const at::Tensor& v = *c.v;
  const int64_t dims = 3 + tokens;
  if (v.dim() != dims || c.q->dim() != dims || !small(v) || !small(*c.q)) return false;
  const int dtype = dtype_code(v.scalar_type());
  const int64_t heads = v.size(dims - 2), dv = v.size(dims - 1), key_heads = c.q->size(dims - 2), dk = c.q->size(dims - 1);
  if (dtype < 0 || key_heads < 1 || heads % key_heads != 0 || heads > FDNN_DELTA_RULE_MAX_HEADS) return false;
  if (dk < 1 || dk > FDNN_DELTA_RULE_MAX_DK || dv < 1 || dv > FDNN_DELTA_RULE_MAX_DV) return false;
  for (const at::Tensor* t : {c.q, c.k}) {
    if (t->sizes() != c.q->sizes() || t->scalar_type() != v.scalar_type() || t->device() != v.device()) return false;
    for (int64_t i = 0; i <= tokens; ++i)
      if (t->size(i) != v.size(i)) return false;
  }
  const at::ScalarType gates = c.delta->scalar_type();
  if (gates != v.scalar_type() && gates != at::kFloat) return false;
  for (const at::Tensor* t : {c.delta, c.beta})
    if (t->scalar_type() != gates || t->device() != v.device() || t->sizes() != v.sizes().slice(0, size_t(dims - 1))) return false;
  if (!dense(c.A, at::kFloat, {heads}, v) || !dense(c.bias, at::kFloat, {heads}, v)) return false;
  fdnn_delta_rule_desc& d = c.d;
  std::memset(&d, 0, sizeof d);
  d.dtype = dtype;
  d.gate_dtype = dtype_code(gates);
  d.n = int(v.size(0));
  d.l = tokens == 1 ? int(v.size(1)) : 1;
  d.key_heads = int(key_heads);
  d.heads = int(heads);
  d.dk = int(dk);
  d.dv = int(dv);
  d.delta_softplus = o[2] == Py_True;
  d.beta_sigmoid = o[3] == Py_True;
  d.qk_norm = o[4] == Py_True;
  d.scale = float(o[5] == Py_None ? 1.0 / std::sqrt(double(dk)) : PyFloat_AsDouble(o[5]));
  strides(*c.q, tokens, d.q_strides);
  strides(*c.k, tokens, d.k_strides);
  strides(v, tokens, d.v_strides);
  strides(*c.delta, tokens, d.delta_strides);
  strides(*c.beta, tokens, d.beta_strides);
  return true;
}

}  // namespace

// gated_delta_rule(q, k, v, delta, beta, A, delta_bias, softplus, sigmoid, norm, scale, initial_state, lengths, return_final_state)
PyObject* fast_gated_delta_rule(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 14 || g_rule == nullptr || !PyBool_Check(a[13])) return none();
  Call c;
  const at::Tensor *initial, *lengths;
  if (!call_of(c, a, a + 5, 1) || !optional(a[11], &initial) || !optional(a[12], &lengths)) return none();
  if (any_grad({c.q, c.k, c.v, c.delta, c.beta, c.A, c.bias, initial})) return none();
  const at::Tensor& v = *c.v;
  const std::array<int64_t, 4> state{c.d.n, c.d.heads, c.d.dv, c.d.dk};
  if (!dense(initial, at::kFloat, state, v) || !dense(lengths, at::kInt, {c.d.n}, v)) return none();
  c10::DeviceGuard guard(v.device());
  at::Tensor y, final, scratch;
  int st;
  {
    WithoutGil free;
    const auto options = v.options().requires_grad(false);
    y = at::empty(v.sizes(), options);
    strides(y, 1, c.d.y_strides);
    if (a[13] == Py_True) final = at::empty(state, options.dtype(at::kFloat));
    int64_t bytes = 0;
    st = g_bytes(&c.d, &bytes);
    if (st == FDNN_OK) {
      if (bytes > 0) scratch = at::empty({bytes}, options.dtype(at::kByte));
      st = g_rule(&c.d, c.q->const_data_ptr(), c.k->const_data_ptr(), v.const_data_ptr(), c.delta->const_data_ptr(), c.beta->const_data_ptr(),
                  f32(c.A), f32(c.bias), f32(initial), i32(lengths), y.mutable_data_ptr(),
                  final.defined() ? final.mutable_data_ptr<float>() : nullptr, bytes > 0 ? scratch.mutable_data_ptr() : nullptr, bytes,
                  stream_of(v));
    }
  }
  if (a[13] == Py_True) return answer(st, {y, final});
  return answer(st, std::move(y));
  END_HANDLE_TH_ERRORS
}

// gated_delta_rule_step(q, k, v, delta, beta, state, A, delta_bias, softplus, sigmoid, norm, scale, slots)
PyObject* fast_gated_delta_rule_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 13 || g_step == nullptr) return none();
  Call c;
  const at::Tensor *state = plain(a[5]), *slots;
  if (state == nullptr || !call_of(c, a, a + 6, 0) || !optional(a[12], &slots)) return none();
  if (any_grad({c.q, c.k, c.v, c.delta, c.beta, state, c.A, c.bias}) || state->dim() != 4) return none();
  const at::Tensor& v = *c.v;
  const int64_t cache = state->size(0);
  if (cache > kMost || (slots == nullptr && cache < c.d.n)) return none();
  if (!dense(state, at::kFloat, {cache, c.d.heads, c.d.dv, c.d.dk}, v) || !dense(slots, at::kInt, {c.d.n}, v)) return none();
  c10::DeviceGuard guard(v.device());
  at::Tensor y;
  int st;
  {
    WithoutGil free;
    y = at::empty(v.sizes(), v.options().requires_grad(false));
    strides(y, 0, c.d.y_strides);
    st = g_step(&c.d, c.q->const_data_ptr(), c.k->const_data_ptr(), v.const_data_ptr(), c.delta->const_data_ptr(), c.beta->const_data_ptr(),
                f32(c.A), f32(c.bias), state->mutable_data_ptr<float>(), int32_t(cache), i32(slots), y.mutable_data_ptr(), stream_of(v));
  }
  if (st == FDNN_OK) written(*state);
  return answer(st, std::move(y));
  END_HANDLE_TH_ERRORS
}

// bind_delta_rule(addresses of the three functions, the descriptor's size as the caller knows it)
PyObject* bind_delta_rule(PyObject*, PyObject* args) {
  unsigned long long f[3], bytes;
  if (!PyArg_ParseTuple(args, "KKKK", &f[0], &f[1], &f[2], &bytes)) return nullptr;
  if (bytes != sizeof(fdnn_delta_rule_desc)) {
    PyErr_SetString(PyExc_ImportError, "compiled for other descriptors of the C ABI");
    return nullptr;
  }
  g_bytes = reinterpret_cast<BytesFn>(uintptr_t(f[0]));
  g_rule = reinterpret_cast<RuleFn>(uintptr_t(f[1]));
  g_step = reinterpret_cast<StepFn>(uintptr_t(f[2]));
  return none();
}
