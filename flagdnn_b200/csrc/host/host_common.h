// What the native host paths share (fastcall.cpp, sequence_fast.cpp).
#pragma once
#include <Python.h>

#include <ATen/ATen.h>
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

}  // namespace fdnn_host

// sequence_fast.cpp: group norm and the state space operators
PyObject* fast_group_norm(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* fast_group_norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* fast_causal_conv1d(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* fast_causal_conv1d_step(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* fast_selective_scan(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* fast_selective_scan_step(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* bind_sequence(PyObject*, PyObject* args);
