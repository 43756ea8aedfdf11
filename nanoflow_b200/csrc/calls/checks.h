// Arguments of calls from Python: what the calls' modules (csrc/calls/*.cpp) check before the C ABI, and how they launch.
#pragma once
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <stdexcept>
#include <string>

#include "kernels.h"

namespace {

using at::Tensor;

[[noreturn]] void refuse(const char* what, const std::string& why) { throw std::runtime_error(std::string(what) + ": " + why); }

const char* name_of(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return "bfloat16";
    case at::kFloat: return "float32";
    case at::kInt: return "int32";
    case at::kLong: return "int64";
    case at::kByte: return "uint8";
    default: return "";
  }
}

const Tensor& tensor(const char* what, const char* name, PyObject* o) {
  if (!THPVariable_Check(o)) refuse(what, std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}
// A contiguous tensor of one type on the cache's device.
const Tensor& checked(const char* what, const char* name, PyObject* o, at::ScalarType type, c10::Device device) {
  const Tensor& t = tensor(what, name, o);
  if (t.scalar_type() != type || t.device() != device || !t.is_contiguous())
    refuse(what, std::string(name) + " must be a contiguous " + name_of(type) + " tensor on " + device.str());
  return t;
}
const Tensor* optional(const char* what, const char* name, PyObject* o, at::ScalarType type, c10::Device device) {
  return o == Py_None ? nullptr : &checked(what, name, o, type, device);
}
int whole(PyObject* o, const char* what, const char* name) {
  const long v = PyLong_AsLong(o);
  if ((v == -1 && PyErr_Occurred()) || v < INT32_MIN || v > INT32_MAX) {
    PyErr_Clear();
    refuse(what, std::string(name) + " must be an int of 32 bits");
  }
  return static_cast<int>(v);
}
float real(PyObject* o, const char* what, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(what, std::string(name) + " must be a number");
  }
  return static_cast<float>(v);
}
int count(const char* what, const Tensor& t, const char* name) {
  if (t.numel() > INT32_MAX) refuse(what, std::string(name) + " has too many entries");
  return static_cast<int>(t.numel());
}
const Tensor* status_word(const char* what, PyObject* o, c10::Device device) {
  const Tensor* t = optional(what, "status", o, at::kInt, device);
  if (t != nullptr && t->numel() < 1) refuse(what, "status must have a word");
  return t;
}
unsigned int* word(const Tensor* t) { return t == nullptr ? nullptr : static_cast<unsigned int*>(t->data_ptr()); }

// What a kernel writes must not lie over anything else that it reads or writes. (Null: a tensor that the call goes without.) Rows at the same
// distance may lie between each other: columns of one buffer.
void apart(const char* what, std::initializer_list<const Tensor*> written, std::initializer_list<const Tensor*> read) {
  struct Span {
    const char *begin, *end;
    int64_t row, distance;                       // bytes of a row, and from row to row; 0: no rows
  } spans[16];
  int n = 0, n_written = 0;
  const auto add = [&](const Tensor* t) {
    if (t == nullptr || t->numel() == 0) return;
    int64_t last = 0;
    for (int64_t d = 0; d < t->dim(); ++d) last += (t->size(d) - 1) * t->stride(d);
    const char* begin = static_cast<const char*>(t->data_ptr());
    const int64_t bytes = t->element_size();
    const bool rows = t->dim() == 2 && t->size(0) > 1 && (t->size(1) == 1 || t->stride(1) == 1) && t->stride(0) >= t->size(1);
    spans[n++] = Span{begin, begin + (last + 1) * bytes, rows ? t->size(1) * bytes : 0, rows ? t->stride(0) * bytes : 0};
  };
  const auto between = [](const Span& a, const Span& b) {        // whether b's rows lie behind a's in the same columns of bytes
    if (a.distance == 0 || a.distance != b.distance) return false;
    const int64_t off = ((b.begin - a.begin) % a.distance + a.distance) % a.distance;
    return off >= a.row && off + b.row <= a.distance;
  };
  if (written.size() + read.size() > 16) refuse(what, "too many tensors");
  for (const Tensor* t : written) add(t);
  n_written = n;
  for (const Tensor* t : read) add(t);
  for (int i = 0; i < n_written; ++i)
    for (int j = i + 1; j < n; ++j)
      if (spans[i].begin < spans[j].end && spans[j].begin < spans[i].end && !between(spans[i], spans[j])) refuse(what, "tensors overlap, and one of them is written");
}

template <class P>
void launch(const char* name, int (*entry)(const P*, cudaStream_t), const P& p, c10::Device device) {
  if (entry == nullptr) refuse(name, "the kernel library is not loaded");
  c10::cuda::OptionalCUDAGuard guard;
  if (device.index() != c10::cuda::current_device()) guard.set_device(device);       // whichever device is the current one
  const int rc = entry(&p, c10::cuda::getCurrentCUDAStream(device.index()).stream());
  if (rc == 0) return;
  refuse(name, rc == 1 ? "bad argument (shape / alignment / size limit)" : rc == 2 ? "CUDA call failed" : "unsupported configuration");
}

// Arguments as they come, and no C++ exception beyond this module.
template <class F>
PyObject* guarded(Py_ssize_t have, Py_ssize_t want, F f) {
  if (have != want) {
    PyErr_Format(PyExc_TypeError, "%zd arguments expected, %zd given", want, have);
    return nullptr;
  }
  try {
    f();
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown error");
    return nullptr;
  }
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return PyMethodDef{name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}

}  // namespace
