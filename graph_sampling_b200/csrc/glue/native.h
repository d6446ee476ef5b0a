// What the functions of the extension module share: taking operands from Python, giving results back, errors.
#pragma once
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <exception>
#include <string>
#include <vector>

#include "../../../include/gsb200.h"

namespace native {

using at::Tensor;

extern PyObject* g_error;  // graph_sampling_b200.cabi.GsbError

struct PyErrorSet : std::exception {};  // a Python exception is already set

[[noreturn]] inline void type_error(const std::string& what) {
  PyErr_SetString(PyExc_TypeError, what.c_str());
  throw PyErrorSet();
}

// An operand: the tensor a pointer was taken from, kept alive (a contiguous copy when the caller's was not contiguous).
struct Arg {
  Tensor hold;
  const Tensor* t = nullptr;
  bool given() const { return t != nullptr; }
  int64_t numel() const { return t->numel(); }
  const int64_t* ids() const { return t ? static_cast<const int64_t*>(t->const_data_ptr()) : nullptr; }
  const float* floats() const { return t ? static_cast<const float*>(t->const_data_ptr()) : nullptr; }
};

inline Arg operand(PyObject* o, const char* name, bool optional, at::ScalarType dtype, const char* dtype_name) {
  Arg a;
  if (o == Py_None) {
    if (optional) return a;
    type_error(std::string(name) + " is required");
  }
  // device memory, or page-locked host memory that the kernels read in place
  if (!THPVariable_Check(o)) type_error(std::string(name) + " must be " + dtype_name + " CUDA (or pinned host) tensor");
  const Tensor& t = THPVariable_Unpack(o);
  if (t.scalar_type() != dtype || !(t.is_cuda() || t.is_pinned()))
    type_error(std::string(name) + " must be " + dtype_name + " CUDA (or pinned host) tensor");
  if (t.is_contiguous()) {
    a.t = &t;
  } else {
    if (!t.is_cuda()) type_error(std::string(name) + ": a pinned host tensor must be contiguous");
    a.hold = t.contiguous();
    a.t = nullptr;
  }
  return a;
}
// (the address of `hold` is only stable in its final place)
inline void settle(Arg& a) {
  if (!a.t && a.hold.defined()) a.t = &a.hold;
}
// A tensor the caller provides for the results.
inline Arg destination(PyObject* o, const char* name) {
  Arg a = operand(o, name, false, at::kFloat, "a float32");
  if (!a.t) type_error(std::string(name) + " must be contiguous");
  return a;
}
#define IDS(var, obj, name) \
  Arg var = operand(obj, name, false, at::kLong, "an int64"); \
  settle(var)
#define IDS_OR_NONE(var, obj, name) \
  Arg var = operand(obj, name, true, at::kLong, "an int64"); \
  settle(var)
#define FLOATS(var, obj, name) \
  Arg var = operand(obj, name, false, at::kFloat, "a float32"); \
  settle(var)
#define FLOATS_OR_NONE(var, obj, name) \
  Arg var = operand(obj, name, true, at::kFloat, "a float32"); \
  settle(var)

inline int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw PyErrorSet();
  return v;
}
inline uint64_t unsigned_integer(PyObject* o) {
  const unsigned long long v = PyLong_AsUnsignedLongLong(o);
  if (v == (unsigned long long)-1 && PyErr_Occurred()) throw PyErrorSet();
  return v;
}
inline bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw PyErrorSet();
  return v == 1;
}
inline gsb_ctx* context(PyObject* o) { return reinterpret_cast<gsb_ctx*>(unsigned_integer(o)); }

inline void* stream() { return static_cast<void*>(c10::cuda::getCurrentCUDAStream().stream()); }

// Results live on the operand's device, or on the current one when the operand is pinned host memory.
inline c10::Device device_of(const Arg& a) {
  return a.t->is_cuda() ? a.t->device() : c10::Device(c10::kCUDA, c10::cuda::current_device());
}
// Entries of an array in device memory; 0 for one that is read from the host.
inline int64_t device_entries(const Arg& a) { return a.t->is_cuda() ? a.numel() : 0; }
inline Tensor empty(int64_t n, c10::Device dev, at::ScalarType dtype = at::kLong) {
  return at::detail::empty_cuda({n}, dtype, dev, c10::nullopt);
}
inline int64_t* mut(const Tensor& t) { return t.defined() ? static_cast<int64_t*>(t.mutable_data_ptr()) : nullptr; }
inline float* mutf(const Tensor& t) { return t.defined() ? static_cast<float*>(t.mutable_data_ptr()) : nullptr; }
// The first n elements of a fresh tensor: the tensor itself is shortened, no view is made.
inline void trim(Tensor& t, int64_t n) {
  if (t.defined() && t.numel() != n) t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
}

inline void check(gsb_ctx* ctx, int st, const char* where) {
  if (st == GSB_OK) return;
  PyObject* e = PyObject_CallFunction(g_error, "iss", st, where, gsb_last_error_message(ctx));
  if (e) {
    PyErr_SetObject(g_error, e);
    Py_DECREF(e);
  }
  throw PyErrorSet();
}

struct NoGil {
  PyThreadState* state;
  NoGil() : state(PyEval_SaveThread()) {}
  ~NoGil() { PyEval_RestoreThread(state); }
};

inline PyObject* wrap(Tensor t) {
  if (!t.defined()) Py_RETURN_NONE;
  PyObject* o = THPVariable_Wrap(std::move(t));
  if (!o) throw PyErrorSet();
  return o;
}
template <class... T>
inline PyObject* tuple_of(T&&... items) {
  PyObject* objs[] = {items...};
  PyObject* out = PyTuple_New(sizeof...(items));
  for (size_t i = 0; i < sizeof...(items); ++i) PyTuple_SET_ITEM(out, (Py_ssize_t)i, objs[i]);
  return out;
}

// Calls `body`, turning C++ exceptions into Python ones.
template <class F>
inline PyObject* guarded(Py_ssize_t got, Py_ssize_t want, F body) {
  if (got != want) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, got);
    return nullptr;
  }
  try {
    return body();
  } catch (const PyErrorSet&) {
    return nullptr;
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* cuda_oom = nullptr;
    if (PyObject* torch = PyImport_ImportModule("torch")) {
      cuda_oom = PyObject_GetAttrString(torch, "OutOfMemoryError");
      Py_DECREF(torch);
    }
    PyErr_SetString(cuda_oom ? cuda_oom : PyExc_RuntimeError, e.what_without_backtrace());
    Py_XDECREF(cuda_oom);
    return nullptr;
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}
#define FUNCTION(name, nargs) \
  PyObject* name##_body(PyObject* const* a); \
  PyObject* name(PyObject*, PyObject* const* a, Py_ssize_t n) { \
    return guarded(n, nargs, [&] { return name##_body(a); }); \
  } \
  PyObject* name##_body(PyObject* const* a)

#define ENTRY(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}

// The functions of gs_rows.cc, ended by an empty entry.
extern PyMethodDef row_methods[];

}  // namespace native
