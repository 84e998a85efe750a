// What the compiled Python entry points share: refusals, checks, outputs, and the way back to Python.
#pragma once

#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/torch.h>

#include <string>

#include "../../include/motif_b200.h"

namespace mb_host {

struct Refusal {
  PyObject* type;
  std::string what;
};
[[noreturn]] inline void refuse(const std::string& what) { throw Refusal{PyExc_ValueError, what}; }

inline std::string shape_of(const at::Tensor& t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}
inline std::string kind_of(const at::Tensor& t) { return std::string(c10::toString(t.scalar_type())) + " " + shape_of(t); }

inline const at::Tensor& tensor(const char* name, PyObject* o) {
  if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}
inline const at::Tensor& on(const char* name, PyObject* o, c10::Device dev) {
  const at::Tensor& t = tensor(name, o);
  if (t.device() != dev) refuse(std::string(name) + " must live on " + dev.str());
  return t;
}
inline int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return MB_F32;
    case at::kHalf: return MB_F16;
    case at::kBFloat16: return MB_BF16;
    default: refuse(std::string("unsupported dtype ") + c10::toString(t) + " (only fp16 / bf16 / fp32)");
  }
}

inline int64_t whole(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Refusal{nullptr, ""};
  return v;
}
inline double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Refusal{nullptr, ""};
  return v;
}

inline void check(const char* name, int rc) {
  if (rc == MB_OK) return;
  PyObject* type = rc == MB_ERR_UNSUPPORTED ? PyExc_NotImplementedError
                   : rc == MB_ERR_CUDA      ? PyExc_RuntimeError
                                            : PyExc_ValueError;
  throw Refusal{type, std::string(name) + ": " + motif_b200_last_error()};
}

inline void* stream_of(c10::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

inline PyObject* wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }
inline PyObject* tuple(std::initializer_list<at::Tensor> ts) {
  PyObject* out = PyTuple_New((Py_ssize_t)ts.size());
  Py_ssize_t i = 0;
  for (const at::Tensor& t : ts) PyTuple_SET_ITEM(out, i++, wrap(t));
  return out;
}

// A contiguous output.  Straight from the allocator: the dispatcher would take as long again, and there
// is nothing for it to do for a tensor without a gradient on a known device.
inline at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, c10::Device dev) {
  return at::detail::empty_cuda(sizes, type, dev, c10::nullopt);
}

// Other Python threads run while a call allocates and launches (a launch waits where the queue is full).
struct NoGil {
  PyThreadState* const state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

// No C++ exception leaves a Python entry.
template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
inline PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Refusal& r) {
    if (r.type) PyErr_SetString(r.type, r.what.c_str());
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    if (type) PyErr_SetString(type, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
constexpr PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, N>)), METH_FASTCALL, nullptr};
}

}  // namespace mb_host
