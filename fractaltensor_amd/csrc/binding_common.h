// What the native modules over the library share: checks of tensors, allocation of results, errors, and the counts of calls.
#pragma once

#include <ATen/core/Tensor.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cmath>
#include <vector>

#include "../../include/ftk.h"

namespace {

PyObject* g_counts = nullptr;   // dict: calls by name
PyObject* g_raise = nullptr;    // callable: raises for a return code of the library

bool is_tensor(PyObject* o) { return THPVariable_Check(o); }
const at::Tensor& tensor_of(PyObject* o) { return THPVariable_Unpack(o); }

// a dense tensor on the GPU of one type
bool plain(PyObject* o, at::ScalarType type) {
  if (!is_tensor(o)) return false;
  const at::Tensor& t = tensor_of(o);
  return t.is_cuda() && t.scalar_type() == type && t.is_contiguous();
}

bool count(const char* name) {
  PyObject* key = PyUnicode_InternFromString(name);
  if (!key) return false;
  PyObject* old = PyDict_GetItem(g_counts, key);
  PyObject* now = PyLong_FromLong((old ? PyLong_AsLong(old) : 0) + 1);
  const bool ok = now && PyDict_SetItem(g_counts, key, now) == 0;
  Py_XDECREF(now);
  Py_DECREF(key);
  return ok;
}

PyObject* raise(int rc) {
  PyObject* r = PyObject_CallFunction(g_raise, "i", rc);
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "libftkernels: an error code that raised nothing");
  return nullptr;
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, const at::Tensor& like) {
  return at::detail::empty_cuda(shape, type, like.device(), std::nullopt);
}

void* stream() { return c10::hip::getCurrentHIPStream().stream(); }

int dim(const at::Tensor& t, int i) { return (int)t.size(i); }

template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// Other Python threads run while one is in the library: a launch may wait for the lock that orders launches of several streams,
// or for the device.
struct WithoutGil {
  PyThreadState* state = PyEval_SaveThread();
  ~WithoutGil() { PyEval_RestoreThread(state); }
};
template <typename F>
int in_library(F&& f) {
  WithoutGil released;
  return f();
}

[[maybe_unused]] PyObject* init(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 2 || !PyDict_Check(args[0]) || !PyCallable_Check(args[1])) {
    PyErr_SetString(PyExc_TypeError, "init(counts, raise)");
    return nullptr;
  }
  Py_INCREF(args[0]);
  Py_INCREF(args[1]);
  Py_XDECREF(g_counts);
  Py_XDECREF(g_raise);
  g_counts = args[0];
  g_raise = args[1];
  Py_RETURN_NONE;
}

}  // namespace
