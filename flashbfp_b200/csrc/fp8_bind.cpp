// fp8_bind.cpp — Python entry points of the block-scaled 8-bit path: the checks of a call's tensors
// and the call into libflashbfp.so, without Python code in between. A small call's time is its host
// side (the launch itself takes about 2 us): checked in Python and called through ctypes, a
// quantisation took 6.9 us, of which this leaves the launch and less than a microsecond.
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

PyObject* g_rows_type = nullptr;        // Fp8Rows
PyObject* g_error_word = nullptr;       // callable(device index) -> address, for a device's first product
void* g_error_words[64] = {nullptr};
bool g_has_word[64] = {false};

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

struct Plain {                          // a 2-D tensor of plain values
  const at::Tensor* t;
  int index, code;
  int64_t m, k, ld;
};
Plain plain(PyObject* o, const char* what) {
  const at::Tensor& t = tensor(o, what);
  if (t.dim() != 2) refuse(PyExc_ValueError, "%s must have two dimensions, not %lld", what, (long long)t.dim());
  Plain p{&t, t.get_device(), dtype_code(t.scalar_type(), what), t.size(0), t.size(1), t.stride(0)};
  if (t.stride(1) != 1 && p.k > 1)
    refuse(PyExc_ValueError, "%s must have contiguous rows (stride %lld between columns)", what,
           (long long)t.stride(1));
  if (p.m <= 1) p.ld = (p.k + 15) / 16 * 16;    // a single row's stride is never used
  return p;
}

struct Rows {                           // an 8-bit operand
  const at::Tensor *v, *s;
  int64_t m, k, ld;
};
// The pair (values, scales); m, k: the shape it must have (-1: any).
Rows rows(PyObject* o, const char* what, int index, int64_t m, int64_t k) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 2)
    refuse(PyExc_TypeError, "%s must be Fp8Rows (values, scales)", what);
  PyObject *vo = PyTuple_GET_ITEM(o, 0), *so = PyTuple_GET_ITEM(o, 1);
  if (!THPVariable_Check(vo) || !THPVariable_Check(so))
    refuse(PyExc_TypeError, "%s must be Fp8Rows (values, scales)", what);
  const at::Tensor &v = THPVariable_Unpack(vo), &s = THPVariable_Unpack(so);
  if (!v.is_cuda() || !s.is_cuda())
    refuse(PyExc_RuntimeError, "%s must be on a CUDA device (no CPU fallback)", what);
  if (index < 0) index = v.get_device();
  if (v.get_device() != index || s.get_device() != index)
    refuse(PyExc_ValueError, "%s is not on cuda:%d", what, index);
  if (v.scalar_type() != at::kFloat8_e4m3fn || s.scalar_type() != at::kFloat8_e8m0fnu || v.dim() != 2)
    refuse(PyExc_ValueError, "%s: values must be 2-D float8_e4m3fn and scales float8_e8m0fnu", what);
  Rows r{&v, &s, v.size(0), v.size(1), v.stride(0)};
  if ((m >= 0 && r.m != m) || (k >= 0 && r.k != k))
    refuse(PyExc_ValueError, "%s has shape (%lld, %lld), not (%s, %s)", what, (long long)r.m, (long long)r.k,
           m >= 0 ? std::to_string(m).c_str() : "*", k >= 0 ? std::to_string(k).c_str() : "*");
  if (r.k < 1) refuse(PyExc_ValueError, "rows must have at least one value");
  if (r.m <= 1) r.ld = (r.k + 15) / 16 * 16;
  if ((v.stride(1) != 1 && r.k > 1) || r.ld % 16 != 0 || r.ld < r.k)
    refuse(PyExc_ValueError, "%s: rows must be contiguous and a multiple of 16 bytes apart (strides (%lld, %lld))",
           what, (long long)v.stride(0), (long long)v.stride(1));
  const int64_t mt = (r.m + 127) / 128, kt = (r.k + 511) / 512;
  if (s.dim() != 5 || s.size(0) != mt || s.size(1) != kt || s.size(2) != 32 || s.size(3) != 4 || s.size(4) != 4 ||
      !s.is_contiguous())
    refuse(PyExc_ValueError, "%s: scales must be contiguous (%lld, %lld, 32, 4, 4)", what, (long long)mt,
           (long long)kt);
  return r;
}

// New Fp8Rows of m x k (a new reference): values whose rows are a multiple of 16 bytes apart.
PyObject* new_rows(int64_t m, int64_t k, int index) {
  if (k < 1) refuse(PyExc_ValueError, "rows must have at least one value");
  const auto dev = at::Device(at::kCUDA, (at::DeviceIndex)index);
  at::Tensor v = at::empty({m, (k + 15) / 16 * 16}, at::TensorOptions().dtype(at::kFloat8_e4m3fn).device(dev));
  if (k % 16) v = v.narrow(1, 0, k);
  at::Tensor s = at::empty({(m + 127) / 128, (k + 511) / 512, 32, 4, 4},
                           at::TensorOptions().dtype(at::kFloat8_e8m0fnu).device(dev));
  PyObject *vo = THPVariable_Wrap(v), *so = THPVariable_Wrap(s);
  PyObject* r = vo && so ? PyObject_CallFunctionObjArgs(g_rows_type, vo, so, nullptr) : nullptr;
  Py_XDECREF(vo);
  Py_XDECREF(so);
  if (!r) throw python_error();
  return r;
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
           "%s is written in place and requires a gradient, which the 8-bit operators do not give: detach it or "
           "call under torch.no_grad()", what);
}
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void written(const Rows& r) {
  written(*r.v);
  written(*r.s);
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
// `given`, or new rows where it is None (a new reference either way).
PyObject* rows_or_new(PyObject* given, int64_t m, int64_t k, int index) {
  if (given == Py_None) return new_rows(m, k, index);
  Py_INCREF(given);
  return given;
}

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

// quantize(x, out)
PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 2)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Plain x = plain(a[0], "x");
    Ref out(rows_or_new(a[1], x.m, x.k, x.index));
    const Rows r = rows(out.o, "out", x.index, x.m, x.k);
    if (x.m)
      call(x.index, "fbfp_fp8_quantize", [&](void* st) {
        return fbfp_fp8_quantize(x.t->const_data_ptr(), x.code, x.m, x.k, x.ld, r.v->data_ptr(), r.ld,
                                 r.s->data_ptr(), st);
      });
    written(r);
    return out.take();
  });
}

// geglu(gate_up, out)
PyObject* geglu(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 2)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Plain x = plain(a[0], "gate_up");
    if (x.k % 2)
      refuse(PyExc_ValueError, "gate_up must hold as many gate as up columns (got %lld)", (long long)x.k);
    Ref out(rows_or_new(a[1], x.m, x.k / 2, x.index));
    const Rows r = rows(out.o, "out", x.index, x.m, x.k / 2);
    if (x.m)
      call(x.index, "fbfp_fp8_geglu", [&](void* st) {
        return fbfp_fp8_geglu(x.t->const_data_ptr(), x.code, x.m, x.k / 2, x.ld, r.v->data_ptr(), r.ld,
                              r.s->data_ptr(), st);
      });
    written(r);
    return out.take();
  });
}

const void* norm_weight(PyObject* o, const char* what, const Plain& x) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "%s must be a tensor", what);
  const at::Tensor& w = THPVariable_Unpack(o);
  if (!w.is_cuda() || w.get_device() != x.index || w.scalar_type() != x.t->scalar_type() || w.dim() != 1 ||
      w.size(0) != x.k || !w.is_contiguous())
    refuse(PyExc_ValueError, "%s must be a contiguous %s vector of %lld on cuda:%d", what,
           c10::toString(x.t->scalar_type()), (long long)x.k, x.index);
  return w.const_data_ptr();
}

// rmsnorm(x, weight, eps, residual, post_weight, out)
PyObject* rmsnorm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 6)) return nullptr;
  const double eps = PyFloat_AsDouble(a[2]);
  if (eps == -1.0 && PyErr_Occurred()) return nullptr;
  return guarded([&]() -> PyObject* {
    const Plain x = plain(a[0], "x");
    const void* w = norm_weight(a[1], "weight", x);
    const void* post = nullptr;
    void* resid = nullptr;
    int64_t ldr = 0;
    if (a[3] != Py_None) {
      const Plain r = plain(a[3], "residual");
      if (r.code != x.code || r.index != x.index || r.m != x.m || r.k != x.k)
        refuse(PyExc_ValueError, "residual must be %s of shape (%lld, %lld) on cuda:%d",
               c10::toString(x.t->scalar_type()), (long long)x.m, (long long)x.k, x.index);
      if (r.ld < r.k) refuse(PyExc_ValueError, "residual rows overlap: each is updated in place");
      check_written(*r.t, "residual");
      resid = r.t->data_ptr();
      ldr = r.ld;
      if (a[4] != Py_None) post = norm_weight(a[4], "post_weight", x);
    } else if (a[4] != Py_None) {
      refuse(PyExc_ValueError, "post_weight needs the residual that its output is added to");
    }
    Ref out(rows_or_new(a[5], x.m, x.k, x.index));
    const Rows q = rows(out.o, "out", x.index, x.m, x.k);
    if (x.m)
      call(x.index, "fbfp_fp8_rmsnorm", [&](void* st) {
        return fbfp_fp8_rmsnorm(x.t->const_data_ptr(), x.code, x.m, x.k, x.ld, w, post, resid, ldr, (float)eps,
                                q.v->data_ptr(), q.ld, q.s->data_ptr(), st);
      });
    written(q);
    if (resid) written(THPVariable_Unpack(a[3]));
    return out.take();
  });
}

void* error_word(int index) {
  if (index >= 64) refuse(PyExc_RuntimeError, "device index %d", index);
  if (!g_has_word[index]) {
    PyObject* r = PyObject_CallFunction(g_error_word, "i", index);
    if (!r) throw python_error();
    g_error_words[index] = PyLong_AsVoidPtr(r);
    Py_DECREF(r);
    if (PyErr_Occurred()) throw python_error();
    g_has_word[index] = true;
  }
  return g_error_words[index];
}

// linear(x, w, bias, out_dtype, out)
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 5)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Rows x = rows(a[0], "x", -1, -1, -1);
    const int index = x.v->get_device();
    const Rows w = rows(a[1], "w", index, -1, x.k);
    const void* bias = nullptr;
    int bias_code = 0;
    if (a[2] != Py_None) {
      const at::Tensor& b = tensor(a[2], "bias");
      if (b.dim() != 1 || b.size(0) != w.m || b.get_device() != index || !b.is_contiguous())
        refuse(PyExc_ValueError, "bias must be a contiguous vector of %lld on cuda:%d", (long long)w.m, index);
      bias = b.const_data_ptr();
      bias_code = dtype_code(b.scalar_type(), "bias");
    }
    const bool typed = a[3] != Py_None;
    if (typed && !THPDtype_Check(a[3])) refuse(PyExc_TypeError, "out_dtype must be a torch.dtype");
    const at::ScalarType want = typed ? reinterpret_cast<THPDtype*>(a[3])->scalar_type : at::kBFloat16;
    if (a[4] == Py_None) dtype_code(want, "out");
    Ref out(nullptr);
    if (a[4] == Py_None) {
      out.o = THPVariable_Wrap(at::empty(
          {x.m, w.m}, at::TensorOptions().dtype(want).device(at::Device(at::kCUDA, (at::DeviceIndex)index))));
      if (!out.o) throw python_error();
    } else {
      Py_INCREF(a[4]);
      out.o = a[4];
    }
    const Plain y = plain(out.o, "out");
    if (y.m != x.m || y.k != w.m || y.index != index || (typed && y.t->scalar_type() != want))
      refuse(PyExc_ValueError, "out must have shape (%lld, %lld) on cuda:%d%s%s", (long long)x.m, (long long)w.m,
             index, typed ? " and dtype " : "", typed ? c10::toString(want) : "");
    if (y.ld < y.k) refuse(PyExc_ValueError, "out's rows overlap");
    check_written(*y.t, "out");
    if (x.m && w.m) {
      void* const word = error_word(index);
      call(index, "fbfp_fp8_linear", [&](void* st) {
        return fbfp_fp8_linear(x.v->const_data_ptr(), x.m, x.k, x.ld, x.s->const_data_ptr(), w.v->const_data_ptr(),
                               w.m, w.ld, w.s->const_data_ptr(), bias, bias_code, y.t->data_ptr(), y.code, y.ld,
                               word, st);
      });
      written(*y.t);
    }
    return out.take();
  });
}

// setup(rows_type, error_word)
PyObject* setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 2)) return nullptr;
  for (int i = 0; i < 2; ++i) Py_INCREF(a[i]);
  g_rows_type = a[0];
  g_error_word = a[1];
  Py_RETURN_NONE;
}

#define FAST(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(quantize), FAST(geglu), FAST(rmsnorm), FAST(linear), FAST(setup),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fp8_bind", "checks and calls of flashbfp_b200.fp8", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

// `built_for` names the torch and the Python whose headers this was compiled with.
extern "C" __attribute__((visibility("default"))) PyObject* PyInit__fp8_bind(void) {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "built_for", FBFP_BUILT_FOR) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
