// What the native host paths share (fastcall.cpp, sequence_fast.cpp, delta_fast.cpp).
#pragma once
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../../include/flagdnn_b200.h"

namespace fdnn_host {

// nullptr: not a plain strided CUDA tensor (subclasses and other layouts take the Python route).  The tensors belong to
// the caller's arguments, which outlive the call.
inline const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.has_storage() || t.is_conj() || t.is_neg())
    return nullptr;   // (tensors without storage: wrappers of function transforms)
  return &t;
}

inline int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return FDNN_F16;
    case at::kBFloat16: return FDNN_BF16;
    case at::kFloat: return FDNN_F32;
    default: return -1;
  }
}

inline PyObject* none() { Py_RETURN_NONE; }

// Other Python threads may run while this one allocates and launches (an allocation can wait for the device).
struct WithoutGil {
  PyThreadState* state = PyEval_SaveThread();
  ~WithoutGil() { PyEval_RestoreThread(state); }
};

constexpr int64_t kMost = 0x7fffffff;

// An optional operand: false if it is there but not a plain tensor.
inline bool optional(PyObject* o, const at::Tensor** t) {
  *t = nullptr;
  if (o == Py_None) return true;
  *t = plain(o);
  return *t != nullptr;
}
// A dense tensor of this type and these sizes on x's device (absent ones are fine).
inline bool dense(const at::Tensor* t, at::ScalarType type, at::IntArrayRef sizes, const at::Tensor& x) {
  return t == nullptr || (t->scalar_type() == type && t->sizes() == sizes && t->device() == x.device() && t->is_contiguous());
}
inline const void* ptr(const at::Tensor* t) { return t == nullptr ? nullptr : t->const_data_ptr(); }
inline const float* f32(const at::Tensor* t) { return static_cast<const float*>(ptr(t)); }
inline const int32_t* i32(const at::Tensor* t) { return static_cast<const int32_t*>(ptr(t)); }
// Whether one of them asks for a gradient or has a tangent of forward-mode differentiation: Python differentiates or refuses.
inline bool any_grad(std::initializer_list<const at::Tensor*> ts) {
  const bool back = c10::GradMode::is_enabled(), forward = c10::AutogradState::get_tls_state().get_fw_grad_mode();
  for (const at::Tensor* t : ts)
    if (t != nullptr && ((back && t->requires_grad()) || (forward && t->_fw_grad(0).defined()))) return true;
  return false;
}
// A state that a kernel has written through its address: autograd's check of saved tensors goes by their versions.  (Tensors made in
// inference mode have none.)
inline void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
inline bool small(const at::Tensor& t) {
  for (int64_t s : t.sizes())
    if (s > kMost) return false;
  return true;
}
inline void* stream_of(const at::Tensor& x) { return c10::cuda::getCurrentCUDAStream(x.get_device()).stream(); }

inline PyObject* answer(int status, at::Tensor&& y) {
  if (status != FDNN_OK) return PyLong_FromLong(status);
  return THPVariable_Wrap(std::move(y));
}
inline PyObject* answer(int status, std::initializer_list<at::Tensor> ts) {
  if (status != FDNN_OK) return PyLong_FromLong(status);
  PyObject* tuple = PyTuple_New(Py_ssize_t(ts.size()));
  if (tuple == nullptr) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor& t : ts) {
    PyObject* o = nullptr;
    if (t.defined()) {
      o = THPVariable_Wrap(t);
      if (o == nullptr) {
        Py_DECREF(tuple);
        return nullptr;
      }
    } else {
      o = Py_None;
      Py_INCREF(o);
    }
    PyTuple_SET_ITEM(tuple, i++, o);
  }
  return tuple;
}

}  // namespace fdnn_host

// sequence_fast.cpp: group norm and the state space operators
PyObject* fast_group_norm(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* fast_group_norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* fast_causal_conv1d(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* fast_causal_conv1d_step(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* fast_selective_scan(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* fast_selective_scan_step(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* bind_sequence(PyObject*, PyObject* args);

// delta_fast.cpp: the gated delta rule
PyObject* fast_gated_delta_rule(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* fast_gated_delta_rule_step(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* bind_delta_rule(PyObject*, PyObject* args);
