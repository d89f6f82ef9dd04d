// bind.h — what the Python entry points share: refusing a call's tensors, and the call into
// libflashbfp.so on the tensors' device and its current stream.
#pragma once
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <cstdio>
#include <string>

#include "../../include/flashbfp.h"

namespace {

struct Refusal {
  PyObject* type;
  std::string text;
};
[[noreturn]] __attribute__((format(printf, 2, 3))) void refuse(PyObject* type, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  throw Refusal{type, buf};
}

const at::Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o) || !THPVariable_Unpack(o).is_cuda())
    refuse(PyExc_RuntimeError, "%s must be a CUDA tensor: FlashBFP-B200 runs only on the GPU (no CPU fallback)", what);
  return THPVariable_Unpack(o);
}

int dtype_code(at::ScalarType t, const char* what) {
  switch (t) {
    case at::kFloat: return FBFP_F32;
    case at::kBFloat16: return FBFP_BF16;
    case at::kHalf: return FBFP_F16;
    default: refuse(PyExc_NotImplementedError, "%s: unsupported dtype %s", what, c10::toString(t));
  }
}

// Runs f(stream) on device `index` and its current stream; raises what a status stands for.
template <typename F>
void call(int index, const char* what, F f) {
  const int before = c10::cuda::current_device();
  if (before != index) c10::cuda::set_device((c10::DeviceIndex)index);
  void* const stream = (void*)c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)index).stream();
  int status;
  Py_BEGIN_ALLOW_THREADS                // a launch waits while the device's queue is full
  status = f(stream);
  Py_END_ALLOW_THREADS
  if (before != index) c10::cuda::set_device((c10::DeviceIndex)before);
  if (status == FBFP_OK) return;
  PyObject* type = status == FBFP_ERR_ARG || status == FBFP_ERR_ALIGN ? PyExc_ValueError
                   : status == FBFP_ERR_UNSUPPORTED                   ? PyExc_NotImplementedError
                                                                      : PyExc_RuntimeError;
  refuse(type, "%s: %s: %s", what, fbfp_status_string(status), fbfp_last_error());
}

// A tensor that a call writes in place. There are no gradients, so one that requires a gradient is
// refused while they are recorded; afterwards its autograd version goes up, so that a backward pass
// which needs the old values says so.
void check_written(const at::Tensor& t, const char* what) {
  if (t.requires_grad() && at::GradMode::is_enabled())
    refuse(PyExc_RuntimeError,
           "%s is written in place and requires a gradient, which these operators do not give: detach it or "
           "call under torch.no_grad()", what);
}
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
// A reference that is given up unless it is taken.
struct Ref {
  PyObject* o;
  explicit Ref(PyObject* p) : o(p) {}
  Ref(const Ref&) = delete;
  ~Ref() { Py_XDECREF(o); }
  PyObject* take() {
    PyObject* p = o;
    o = nullptr;
    return p;
  }
};
// Per device: the word in which its kernels record what went wrong, made at its first call.
struct ErrorWords {
  PyObject* make = nullptr;             // callable(device index) -> address
  void* words[64] = {nullptr};
  bool has[64] = {false};
  void* of(int index) {
    if (index >= 64) refuse(PyExc_RuntimeError, "device index %d", index);
    if (!has[index]) {
      PyObject* r = PyObject_CallFunction(make, "i", index);
      if (!r) throw python_error();
      words[index] = PyLong_AsVoidPtr(r);
      Py_DECREF(r);
      if (PyErr_Occurred()) throw python_error();
      has[index] = true;
    }
    return words[index];
  }
};

template <typename F>
PyObject* guarded(F f) {
  HANDLE_TH_ERRORS
  try {
    return f();
  } catch (const Refusal& r) {
    PyErr_SetString(r.type, r.text.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

bool arity(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
  return n == want;
}

#define FAST(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}

}  // namespace
