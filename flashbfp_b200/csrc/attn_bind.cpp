// attn_bind.cpp — Python entry points of the prompts' attention and of the 4-bit key/value cache, beside
// those of the 8-bit path in the same module.
#include "bind.h"

#include <cmath>
#include <cstdint>

namespace {

ErrorWords g_words;

const at::Tensor& on(PyObject* o, const char* what, int index) {
  const at::Tensor& t = tensor(o, what);
  if (index >= 0 && t.get_device() != index) refuse(PyExc_ValueError, "%s is not on cuda:%d", what, index);
  return t;
}

// An int32 vector of n values (n < 0: any count from 1 on).
const int32_t* ints(PyObject* o, const char* what, int index, int64_t n, int64_t* count = nullptr) {
  const at::Tensor& t = on(o, what, index);
  if (t.scalar_type() != at::kInt || t.dim() != 1 || !t.is_contiguous() || (n >= 0 ? t.size(0) != n : t.size(0) < 1))
    refuse(PyExc_ValueError, "%s must be a contiguous int32 vector%s%s", what, n >= 0 ? " of " : "",
           n >= 0 ? std::to_string(n).c_str() : "");
  if (count) *count = t.size(0);
  return t.const_data_ptr<int32_t>();
}

struct Heads {                          // rows of heads: [rows, heads, dim]
  const at::Tensor* t;
  int index, code;
  int64_t rows, heads, dim, row, head;
};
Heads heads(PyObject* o, const char* what, int index, int64_t rows, int64_t n_heads, int64_t dim) {
  const at::Tensor& t = on(o, what, index);
  if (t.dim() != 3) refuse(PyExc_ValueError, "%s must have three dimensions, not %lld", what, (long long)t.dim());
  Heads h{&t, (int)t.get_device(), dtype_code(t.scalar_type(), what), t.size(0), t.size(1), t.size(2), t.stride(0),
          t.stride(1)};
  if ((rows >= 0 && h.rows != rows) || (n_heads >= 0 && h.heads != n_heads) || (dim >= 0 && h.dim != dim))
    refuse(PyExc_ValueError, "%s has shape (%lld, %lld, %lld), not (%s, %s, %s)", what, (long long)h.rows,
           (long long)h.heads, (long long)h.dim, rows >= 0 ? std::to_string(rows).c_str() : "*",
           n_heads >= 0 ? std::to_string(n_heads).c_str() : "*", dim >= 0 ? std::to_string(dim).c_str() : "*");
  if (h.dim > 1 && t.stride(2) != 1) refuse(PyExc_ValueError, "%s: the values of a head must be contiguous", what);
  if (h.rows <= 1) h.row = (h.heads * h.dim + 7) / 8 * 8;       // never used
  if (h.heads <= 1) h.head = (h.dim + 7) / 8 * 8;
  return h;
}

// A tensor that a call writes: no two of its elements in one place.
void check_out(const at::Tensor& t, const char* what) {
  check_written(t, what);
  int64_t size[8], stride[8];
  int n = 0;
  for (int64_t i = 0; i < t.dim(); ++i) {
    if (t.size(i) == 0) return;
    if (t.size(i) == 1) continue;
    int j = n++;
    for (; j > 0 && stride[j - 1] > t.stride(i); --j) size[j] = size[j - 1], stride[j] = stride[j - 1];
    size[j] = t.size(i), stride[j] = t.stride(i);
  }
  int64_t reach = 1;
  for (int j = 0; j < n; ++j) {
    if (stride[j] < reach) refuse(PyExc_ValueError, "%s's rows overlap", what);
    reach += (size[j] - 1) * stride[j];
  }
}

struct Cache {
  fbfp_kv4_cache c;
  int index;
  const at::Tensor* t[4];
};
// A KV4Cache: (k_values, k_scales, v_values, v_scales, head_dim).
Cache cache_of(PyObject* o) {
  static const char* const names[4] = {"k_values", "k_scales", "v_values", "v_scales"};
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 5) refuse(PyExc_TypeError, "cache must be a KV4Cache");
  const int64_t dim = PyLong_AsLongLong(PyTuple_GET_ITEM(o, 4));
  if (dim == -1 && PyErr_Occurred()) throw python_error();
  if (dim < 8 || dim > 256 || dim % 8) refuse(PyExc_ValueError, "head_dim %lld is not a multiple of 8 up to 256", (long long)dim);
  const int64_t groups = (dim + 31) / 32;
  Cache r{};
  for (int i = 0; i < 4; ++i) {
    const at::Tensor& t = on(PyTuple_GET_ITEM(o, i), names[i], i ? r.index : -1);
    if (i == 0) r.index = t.get_device();
    r.t[i] = &t;
    if (t.dim() != 4 || t.scalar_type() != (i & 1 ? at::kBFloat16 : at::kByte) || !t.is_contiguous() ||
        t.size(3) != (i & 1 ? groups : 16 * groups) ||
        (i && (t.size(0) != r.t[0]->size(0) || t.size(1) != r.t[0]->size(1) || t.size(2) != r.t[0]->size(2))))
      refuse(PyExc_ValueError, "%s must be contiguous %s [sequences, heads, positions, %lld]", names[i],
             i & 1 ? "bfloat16" : "uint8", (long long)(i & 1 ? groups : 16 * groups));
  }
  r.c = fbfp_kv4_cache{r.t[0]->data_ptr(), r.t[1]->data_ptr(), r.t[2]->data_ptr(), r.t[3]->data_ptr(),
                       r.t[0]->size(0), r.t[0]->size(1), r.t[0]->size(2), dim};
  return r;
}

// The caller's error word, or the device's.
int32_t* error_word(PyObject* o, int index) {
  if (o == Py_None) return (int32_t*)g_words.of(index);
  const at::Tensor& t = on(o, "err", index);
  if (t.scalar_type() != at::kInt || t.numel() != 1) refuse(PyExc_ValueError, "err must be one int32");
  return t.data_ptr<int32_t>();
}

int64_t window_of(PyObject* o) {
  const int64_t w = PyLong_AsLongLong(o);
  if (w == -1 && PyErr_Occurred()) throw python_error();
  if (w < 0) refuse(PyExc_ValueError, "window %lld is negative (0: none)", (long long)w);
  return w;
}

float scaling_of(PyObject* o, int64_t dim) {
  if (o == Py_None) return 1.f / std::sqrt((float)dim);
  const double s = PyFloat_AsDouble(o);
  if (s == -1.0 && PyErr_Occurred()) throw python_error();
  if (!std::isfinite(s)) refuse(PyExc_ValueError, "scaling must be finite");
  return (float)s;
}

void attention_dtype(const at::Tensor& t) {
  if (t.scalar_type() != at::kBFloat16 && t.scalar_type() != at::kHalf)
    refuse(PyExc_NotImplementedError, "attention takes bf16 or fp16, not %s", c10::toString(t.scalar_type()));
}

at::Tensor workspace(int64_t bytes, int index) {
  return at::empty({bytes}, at::TensorOptions().dtype(at::kByte).device(at::Device(at::kCUDA, (at::DeviceIndex)index)));
}

// A result like q: `given`, or new (a new reference either way).
PyObject* out_or_new(PyObject* given, const at::Tensor& q) {
  if (given != Py_None) {
    Py_INCREF(given);
    return given;
  }
  PyObject* o = THPVariable_Wrap(at::empty(q.sizes(), q.options().requires_grad(false)));
  if (!o) throw python_error();
  return o;
}

// prompt_attention(q, k, v, starts, kv_starts, window, scaling, out, err)
PyObject* prompt_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 9)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Heads q = heads(a[0], "q", -1, -1, -1, -1);
    attention_dtype(*q.t);
    const Heads k = heads(a[1], "k", q.index, -1, -1, q.dim), v = heads(a[2], "v", q.index, k.rows, k.heads, q.dim);
    if (k.code != q.code || v.code != q.code) refuse(PyExc_ValueError, "q, k and v must have one dtype");
    int64_t count;
    const int32_t* starts = ints(a[3], "starts", q.index, -1, &count);
    if (count < 2) refuse(PyExc_ValueError, "starts must hold one value more than there are sequences");
    const int32_t* kv_starts = a[4] == Py_None ? nullptr : ints(a[4], "kv_starts", q.index, count);
    const int64_t window = window_of(a[5]);
    const float scaling = scaling_of(a[6], q.dim);
    Ref out(out_or_new(a[7], *q.t));
    const Heads o = heads(out.o, "out", q.index, q.rows, q.heads, q.dim);
    if (o.code != q.code) refuse(PyExc_ValueError, "out must have q's dtype");
    check_out(*o.t, "out");
    if (q.rows && q.heads) {
      if (!k.rows) refuse(PyExc_ValueError, "no keys");
      int32_t* const err = error_word(a[8], q.index);
      const int64_t bytes = fbfp_prompt_attention_workspace_bytes(q.rows, k.rows, count - 1, q.heads, k.heads, q.dim, window);
      at::Tensor ws;
      if (bytes > 0) ws = workspace(bytes, q.index);
      call(q.index, "fbfp_prompt_attention", [&](void* st) {
        return fbfp_prompt_attention(q.t->const_data_ptr(), k.t->const_data_ptr(), v.t->const_data_ptr(), q.code, q.rows,
                                     k.rows, count - 1, q.heads, k.heads, q.dim, q.row, q.head, k.row, k.head, v.row,
                                     v.head, starts, kv_starts, window, scaling, o.t->data_ptr(), o.row, o.head,
                                     bytes > 0 ? ws.data_ptr() : nullptr, bytes, err, st);
      });
      written(*o.t);
    }
    return out.take();
  });
}

// kv4_check(cache, out): refuses a cache that is not one, and tensors that must not be written.
PyObject* kv4_check(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 2)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Cache c = cache_of(a[0]);
    for (int i = 0; i < 4; ++i) check_written(*c.t[i], "cache");
    check_out(on(a[1], "q_out", c.index), "q_out");
    Py_RETURN_NONE;
  });
}

// kv4_write(cache, k, v, pos, starts, err)
PyObject* kv4_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 6)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Cache c = cache_of(a[0]);
    const Heads k = heads(a[1], "k", c.index, -1, c.c.kv_heads, c.c.head_dim);
    const Heads v = heads(a[2], "v", c.index, k.rows, c.c.kv_heads, c.c.head_dim);
    if (k.code != v.code) refuse(PyExc_ValueError, "k and v must have one dtype");
    const int32_t* pos = ints(a[3], "pos", c.index, c.c.seqs);
    const int32_t* starts = a[4] == Py_None ? nullptr : ints(a[4], "starts", c.index, c.c.seqs + 1);
    if (!starts && k.rows != c.c.seqs)
      refuse(PyExc_ValueError, "%lld rows for %lld sequences: pass starts", (long long)k.rows, (long long)c.c.seqs);
    for (int i = 0; i < 4; ++i) check_written(*c.t[i], "cache");
    if (k.rows) {
      int32_t* const err = error_word(a[5], c.index);
      call(c.index, "fbfp_kv4_write", [&](void* st) {
        return fbfp_kv4_write(&c.c, k.t->const_data_ptr(), v.t->const_data_ptr(), k.code, k.rows, k.row, k.head, v.row,
                              v.head, pos, starts, err, st);
      });
      for (int i = 0; i < 4; ++i) written(*c.t[i]);
    }
    Py_RETURN_NONE;
  });
}

// kv4_read(cache, first, starts, k, v, err)
PyObject* kv4_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 6)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Cache c = cache_of(a[0]);
    const int32_t* first = ints(a[1], "first", c.index, c.c.seqs);
    const int32_t* starts = ints(a[2], "starts", c.index, c.c.seqs + 1);
    const Heads k = heads(a[3], "k", c.index, -1, c.c.kv_heads, c.c.head_dim);
    const Heads v = heads(a[4], "v", c.index, k.rows, c.c.kv_heads, c.c.head_dim);
    if (k.code != v.code) refuse(PyExc_ValueError, "k and v must have one dtype");
    check_out(*k.t, "k");
    check_out(*v.t, "v");
    if (k.rows && k.t->const_data_ptr() == v.t->const_data_ptr())
      refuse(PyExc_ValueError, "k and v are written to one place");
    if (k.rows) {
      int32_t* const err = error_word(a[5], c.index);
      call(c.index, "fbfp_kv4_read", [&](void* st) {
        return fbfp_kv4_read(&c.c, k.t->data_ptr(), v.t->data_ptr(), k.code, k.rows, k.row, k.head, v.row, v.head, first,
                             starts, err, st);
      });
      written(*k.t);
      written(*v.t);
    }
    Py_RETURN_NONE;
  });
}

// kv4_attention(q, cache, pos, window, scaling, out, err)
PyObject* kv4_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 7)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Cache c = cache_of(a[1]);
    const at::Tensor& q = on(a[0], "q", c.index);
    attention_dtype(q);
    const int64_t d = q.dim();
    if (d != 3 && d != 4) refuse(PyExc_ValueError, "q must have three or four dimensions, not %lld", (long long)d);
    const int64_t rows = d == 4 ? q.size(1) : 1, n_heads = q.size(d - 2);
    if (q.size(0) != c.c.seqs || q.size(d - 1) != c.c.head_dim)
      refuse(PyExc_ValueError, "q must be [%lld, (rows,) heads, %lld]", (long long)c.c.seqs, (long long)c.c.head_dim);
    const int32_t* pos = ints(a[2], "pos", c.index, c.c.seqs);
    const int64_t window = window_of(a[3]);
    const float scaling = scaling_of(a[4], c.c.head_dim);
    Ref out(out_or_new(a[5], q));
    const at::Tensor& o = on(out.o, "out", c.index);
    if (o.sizes() != q.sizes() || o.scalar_type() != q.scalar_type())
      refuse(PyExc_ValueError, "out must have q's shape and dtype");
    check_out(o, "out");
    if (q.stride(d - 1) != 1 || o.stride(d - 1) != 1)
      refuse(PyExc_ValueError, "the values of a head must be contiguous");
    const auto stride = [&](const at::Tensor& t, int64_t i) {        // 0 where it is never used
      return t.size(i) > 1 ? t.stride(i) : (int64_t)0;
    };
    if (rows && n_heads) {
      int32_t* const err = error_word(a[6], c.index);
      const int64_t bytes = fbfp_kv4_attention_workspace_bytes(&c.c, rows, n_heads);
      at::Tensor ws;
      if (bytes > 0) ws = workspace(bytes, c.index);
      call(c.index, "fbfp_kv4_attention", [&](void* st) {
        return fbfp_kv4_attention(&c.c, q.const_data_ptr(), dtype_code(q.scalar_type(), "q"), rows, n_heads, stride(q, 0),
                                  d == 4 ? stride(q, 1) : 0, stride(q, d - 2), pos, window, scaling, o.data_ptr(),
                                  stride(o, 0), d == 4 ? stride(o, 1) : 0, stride(o, d - 2),
                                  bytes > 0 ? ws.data_ptr() : nullptr, bytes, err, st);
      });
      written(o);
    }
    return out.take();
  });
}

// attn_setup(error_word)
PyObject* attn_setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity(n, 1)) return nullptr;
  Py_INCREF(a[0]);
  g_words.make = a[0];
  Py_RETURN_NONE;
}

}  // namespace

PyMethodDef attn_methods[] = {FAST(prompt_attention), FAST(kv4_write), FAST(kv4_read), FAST(kv4_attention),
                              FAST(kv4_check),
                              FAST(attn_setup), {nullptr, nullptr, 0, nullptr}};
