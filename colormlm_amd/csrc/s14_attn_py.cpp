// The attention entry points' Python call, in C++: a single token's call is a
// few us of GPU work, and reading its tensors' types, shapes, strides and
// addresses in Python and handing them over through ctypes took longer than
// that (norm and rotation of one token: 9.3 us a call in Python, 5.4 by the
// tensors' Python methods here, 3.3 by torch's own, most of it the launch).
//
// No part of libs14hip.so: colormlm_amd/attention.py loads it and gives it the
// library's entry points.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <exception>

#include "s14_hip.h"

typedef int (*norm_rope_fn)(s14_ctx *, void *, uint32_t, uint32_t, const s14_rows *, const s14_rows *, const s14_rows *,
                            const s14_rows *, s14_buffer, s14_buffer, float, const s14_rope *, s14_buffer);
typedef int (*append_fn)(s14_ctx *, void *, const s14_kv_cache *, uint32_t, uint32_t, uint32_t, const s14_rows *,
                         const s14_rows *, s14_buffer, uint32_t, s14_buffer, s14_buffer, s14_buffer, float,
                         const s14_rope *);
typedef int (*paged_fn)(s14_ctx *, void *, const s14_rows *, const s14_kv_cache *, uint32_t, uint32_t, uint32_t, uint32_t,
                        s14_buffer, uint32_t, s14_buffer, s14_buffer, const s14_rows *, s14_buffer, float, uint32_t);
typedef int (*prompt_fn)(s14_ctx *, void *, uint32_t, const s14_rows *, const s14_rows *, const s14_rows *, uint32_t,
                         uint32_t, s14_buffer, const s14_rows *, s14_buffer, float, uint32_t);

static norm_rope_fn f_norm_rope;
static append_fn f_append;
static paged_fn f_paged;
static prompt_fn f_prompt;
static PyObject *p_refuse, *p_check, *p_stream;      // attention.py's functions

// Raises S14Error(code, message); returns -1.
static int refuse(int code, const char *format, ...) {
  va_list args;
  va_start(args, format);
  PyObject *text = PyUnicode_FromFormatV(format, args);
  va_end(args);
  if (text) {
    PyObject *r = PyObject_CallFunction(p_refuse, "iN", code, text);
    Py_XDECREF(r);
  }
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "attention call refused");
  return -1;
}

// The tensor of a Python object on the device, or NULL (refused).
static const at::Tensor *tensor_of(PyObject *t, const char *label, long device) {
  if (THPVariable_Check(t)) {
    const at::Tensor &x = THPVariable_Unpack(t);
    if (x.defined() && x.layout() == at::kStrided && x.get_device() == device) return &x;
  }
  refuse(S14_ERR_INVALID, "%s must be a tensor on the context's device %ld", label, device);
  return nullptr;
}

// The s14_rows of a [tokens, heads, dim] tensor (dim 0: any).
static int rows_of(PyObject *t, const char *label, long device, long long dim, s14_rows *r, long long shape[3]) {
  const at::Tensor *x = tensor_of(t, label, device);
  if (!x) return -1;
  const bool f32 = x->scalar_type() == at::kFloat;
  if (!f32 && x->scalar_type() != at::kBFloat16) return refuse(S14_ERR_INVALID, "%s must be float32 or bfloat16", label);
  const at::IntArrayRef size = x->sizes(), stride = x->strides();
  if (size.size() != 3 || (stride[2] != 1 && size[2] > 1) || (dim && size[2] != dim))
    return refuse(S14_ERR_SHAPE, "%s must be [tokens, heads, dim] of the call's dim, its last dimension contiguous", label);
  // strides of a dimension of one are not used; what torch gives there may be anything
  const uint64_t token = size[0] < 2 ? 0 : uint64_t(stride[0]), head = size[1] < 2 ? 0 : uint64_t(stride[1]);
  if (size[0] > UINT32_MAX || size[1] > UINT32_MAX || size[2] > UINT32_MAX || head > UINT32_MAX)
    return refuse(S14_ERR_SHAPE, "%s is too large", label);
  for (int i = 0; i < 3; ++i) shape[i] = size[i];
  r->buf.ptr = x->data_ptr();
  r->buf.bytes = size[0] && size[1] ? ((size[0] - 1) * token + (size[1] - 1) * head + size[2]) * (f32 ? 4 : 2) : 0;
  r->dtype = f32 ? S14_X_F32 : S14_X_BF16;
  r->heads = uint32_t(size[1]);
  r->token_stride = token;
  r->head_stride = uint32_t(head);
  return 0;
}

// The buffer of a contiguous tensor of one 4-byte type, of `values` at least; None: no buffer.
static int flat_of(PyObject *t, const char *label, long device, at::ScalarType type, unsigned long long values, s14_buffer *b) {
  b->ptr = nullptr, b->bytes = 0;
  if (t == Py_None) return 0;
  const at::Tensor *x = tensor_of(t, label, device);
  if (!x) return -1;
  if (x->scalar_type() != type || !x->is_contiguous())
    return refuse(S14_ERR_INVALID, "%s must be a contiguous %s tensor", label, type == at::kFloat ? "float32" : "int32");
  const unsigned long long have = x->numel();
  if (have < values) return refuse(S14_ERR_CAPACITY, "%s has %llu values, %llu are required", label, have, values);
  b->ptr = x->data_ptr(), b->bytes = 4 * have;
  return 0;
}

// A [sequences, pages] page table with its cu and lengths.
typedef struct {
  s14_buffer table, cu, len;
  uint32_t seqs, width;
} index_rows;
static int index_of(PyObject *table, PyObject *cu, PyObject *len, const char *label, long device, index_rows *x) {
  if (table == Py_None || cu == Py_None || len == Py_None) return refuse(S14_ERR_INVALID, "page table, cu and %s are required", label);
  if (flat_of(table, "page table", device, at::kInt, 0, &x->table)) return -1;
  const at::IntArrayRef size = THPVariable_Unpack(table).sizes();
  if (size.size() != 2 || size[0] > UINT32_MAX || size[1] > UINT32_MAX)
    return refuse(S14_ERR_SHAPE, "a page table is [sequences, pages]");
  const long long seqs = size[0], width = size[1];
  x->seqs = (uint32_t)seqs, x->width = (uint32_t)width;
  if (flat_of(cu, "cu", device, at::kInt, (unsigned long long)seqs + 1, &x->cu)) return -1;
  return flat_of(len, label, device, at::kInt, (unsigned long long)seqs, &x->len);
}

// The stream: the caller's, or the device's current one.
static int stream_of(PyObject *stream, long device, void **out) {
  PyObject *r = stream == Py_None ? PyObject_CallFunction(p_stream, "l", device) : Py_NewRef(stream);
  if (!r) return -1;
  *out = (void *)(uintptr_t)PyLong_AsUnsignedLongLong(r);
  Py_DECREF(r);
  return PyErr_Occurred() ? -1 : 0;
}

// An unsigned 32-bit argument.
static int u32_of(PyObject *v, const char *label, uint32_t *out) {
  const long long x = PyLong_AsLongLong(v);
  if (x == -1 && PyErr_Occurred()) return -1;
  if (x < 0 || x > UINT32_MAX) return refuse(S14_ERR_INVALID, "%s is %lld", label, x);
  *out = (uint32_t)x;
  return 0;
}

static void *pointer_of(PyObject *v) { return v == Py_None ? nullptr : PyLong_AsVoidPtr(v); }

// A KvCache or Rope holds the addresses that its tensors had when it was made:
// refused where one has other memory since (resize_, set_, .data).
static int held(PyObject *tensors, const s14_buffer *const *bufs, Py_ssize_t n, const char *what) {
  if (!PyTuple_Check(tensors) || PyTuple_GET_SIZE(tensors) != n) return refuse(S14_ERR_INVALID, "%s has no tensors", what);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject *t = PyTuple_GET_ITEM(tensors, i);
    if (!THPVariable_Check(t) || THPVariable_Unpack(t).data_ptr() != bufs[i]->ptr ||
        THPVariable_Unpack(t).nbytes() < bufs[i]->bytes)
      return refuse(S14_ERR_INVALID, "%s was made of other memory than its tensors have now", what);
  }
  return 0;
}
static int cache_of(PyObject *at, PyObject *tensors, const s14_kv_cache **out) {
  const s14_kv_cache *c = *out = (const s14_kv_cache *)pointer_of(at);
  if (!c) return refuse(S14_ERR_INVALID, "a cache is required");
  const s14_buffer *const bufs[4] = {&c->k, &c->k_scale, &c->v, &c->v_scale};
  return held(tensors, bufs, 4, "the cache");
}
static int rope_of(PyObject *at, PyObject *tensors, const s14_rope **out) {
  const s14_rope *r = *out = (const s14_rope *)pointer_of(at);
  if (!r) return 0;
  const s14_buffer *const buf = &r->table;
  return held(tensors, &buf, 1, "the rotation");
}

static PyObject *done(int rc) {
  if (!rc) Py_RETURN_NONE;
  PyObject *r = PyObject_CallFunction(p_check, "i", rc);
  Py_XDECREF(r);
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

static int same(const long long a[3], const long long b[3]) { return a[0] == b[0] && a[1] == b[1] && a[2] == b[2]; }

#define ARGUMENTS(n)                                                                              \
  do {                                                                                            \
    if (argc != (n)) return PyErr_Format(PyExc_TypeError, "%d arguments, not %zd", (n), argc);    \
  } while (0)

// handle, device, stream, q, k, q_out, k_out, q_weight, k_weight, eps, rope, positions, the rotation's tensors
static PyObject *qk_norm_rope(PyObject *, PyObject *const *v, Py_ssize_t argc) {
  ARGUMENTS(13);
  s14_ctx *ctx = (s14_ctx *)pointer_of(v[0]);
  const long device = PyLong_AsLong(v[1]);
  const double eps = PyFloat_AsDouble(v[9]);
  const s14_rope *rope;
  void *stream;
  s14_rows q, qo, k, ko;
  s14_buffer qw, kw, pos;
  long long shape[3], other[3], ks[3];
  if (PyErr_Occurred() || rope_of(v[10], v[12], &rope)) return nullptr;
  if (rows_of(v[3], "q", device, 0, &q, shape) || rows_of(v[5], "q output", device, shape[2], &qo, other)) return nullptr;
  if (!same(shape, other)) return refuse(S14_ERR_SHAPE, "q output must have q's shape"), nullptr;
  if (v[4] == Py_None) {
    k = ko = s14_rows{};
  } else {
    if (rows_of(v[4], "k", device, shape[2], &k, ks) || rows_of(v[6], "k output", device, shape[2], &ko, other)) return nullptr;
    if (ks[0] != shape[0] || !same(ks, other))
      return refuse(S14_ERR_SHAPE, "k must have q's tokens, and k output k's shape"), nullptr;
  }
  if (flat_of(v[7], "q norm weight", device, at::kFloat, 0, &qw) || flat_of(v[8], "k norm weight", device, at::kFloat, 0, &kw) ||
      flat_of(v[11], "positions", device, at::kInt, 0, &pos))
    return nullptr;
  if (stream_of(v[2], device, &stream)) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f_norm_rope(ctx, stream, (uint32_t)shape[0], (uint32_t)shape[2], &q, &k, &qo, &ko, qw, kw, (float)eps, rope, pos);
  Py_END_ALLOW_THREADS
  return done(rc);
}

// handle, device, stream, cache, dim, k, v, page_table, cu, past, k_weight, eps, rope, max_new, the cache's and the rotation's tensors
static PyObject *kv_append(PyObject *, PyObject *const *v, Py_ssize_t argc) {
  ARGUMENTS(16);
  s14_ctx *ctx = (s14_ctx *)pointer_of(v[0]);
  const long device = PyLong_AsLong(v[1]);
  const s14_kv_cache *cache;
  const long long dim = PyLong_AsLongLong(v[4]);
  const double eps = PyFloat_AsDouble(v[11]);
  const s14_rope *rope;
  void *stream;
  s14_rows k, x;
  s14_buffer kw;
  index_rows at;
  long long shape[3], other[3];
  uint32_t most;
  if (PyErr_Occurred() || cache_of(v[3], v[14], &cache) || rope_of(v[12], v[15], &rope)) return nullptr;
  if (rows_of(v[5], "k", device, dim, &k, shape) || rows_of(v[6], "v", device, dim, &x, other)) return nullptr;
  if (shape[0] != other[0]) return refuse(S14_ERR_SHAPE, "k and v have different token counts"), nullptr;
  if (index_of(v[7], v[8], v[9], "past", device, &at) || flat_of(v[10], "k norm weight", device, at::kFloat, 0, &kw)) return nullptr;
  most = (uint32_t)shape[0];
  if (v[13] != Py_None && u32_of(v[13], "max_new", &most)) return nullptr;
  if (stream_of(v[2], device, &stream)) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f_append(ctx, stream, cache, (uint32_t)shape[0], at.seqs, most, &k, &x, at.table, at.width, at.cu, at.len, kw,
                (float)eps, rope);
  Py_END_ALLOW_THREADS
  return done(rc);
}

// scale: None is 1 / sqrt(dim)
static int scale_of(PyObject *v, long long dim, float *out) {
  const double s = v == Py_None ? 1.0 / std::sqrt((double)(dim ? dim : 1)) : PyFloat_AsDouble(v);
  *out = (float)s;
  return PyErr_Occurred() ? -1 : 0;
}

// handle, device, stream, q, cache, dim, page_table, cu, lens, out, lse, scale, window, max_new, max_len, tokens a page, the cache's tensors
static PyObject *paged_attention(PyObject *, PyObject *const *v, Py_ssize_t argc) {
  ARGUMENTS(17);
  s14_ctx *ctx = (s14_ctx *)pointer_of(v[0]);
  const long device = PyLong_AsLong(v[1]);
  const s14_kv_cache *cache;
  const long long dim = PyLong_AsLongLong(v[5]);
  const long long page = PyLong_AsLongLong(v[15]);
  void *stream;
  s14_rows q, out;
  s14_buffer lse;
  index_rows at;
  long long shape[3], other[3];
  uint32_t window = 0, most, length;
  float scale;
  if (PyErr_Occurred() || cache_of(v[4], v[16], &cache)) return nullptr;
  if (rows_of(v[3], "q", device, dim, &q, shape) || rows_of(v[9], "out", device, dim, &out, other)) return nullptr;
  if (!same(shape, other)) return refuse(S14_ERR_SHAPE, "out must have q's shape"), nullptr;
  if (index_of(v[6], v[7], v[8], "lens", device, &at)) return nullptr;
  if (flat_of(v[10], "lse", device, at::kFloat, (unsigned long long)shape[0] * shape[1], &lse)) return nullptr;
  if (scale_of(v[11], dim, &scale) || u32_of(v[12], "window", &window)) return nullptr;
  most = (uint32_t)shape[0];
  if (v[13] != Py_None && u32_of(v[13], "max_new", &most)) return nullptr;
  const unsigned long long reach = (unsigned long long)at.width * (unsigned long long)page;
  length = reach > INT32_MAX ? INT32_MAX : (uint32_t)reach;
  if (v[14] != Py_None && u32_of(v[14], "max_len", &length)) return nullptr;
  if (stream_of(v[2], device, &stream)) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f_paged(ctx, stream, &q, cache, (uint32_t)shape[0], at.seqs, most, length, at.table, at.width, at.cu, at.len, &out,
               lse, scale, window);
  Py_END_ALLOW_THREADS
  return done(rc);
}

// handle, device, stream, q, k, v, cu, out, lse, scale, window
static PyObject *prompt_attention(PyObject *, PyObject *const *v, Py_ssize_t argc) {
  ARGUMENTS(11);
  s14_ctx *ctx = (s14_ctx *)pointer_of(v[0]);
  const long device = PyLong_AsLong(v[1]);
  void *stream;
  s14_rows q, k, x, out;
  s14_buffer cu, lse;
  long long shape[3], ks[3], other[3];
  uint32_t window = 0;
  float scale;
  if (PyErr_Occurred()) return nullptr;
  if (rows_of(v[3], "q", device, 0, &q, shape) || rows_of(v[7], "out", device, shape[2], &out, other)) return nullptr;
  if (!same(shape, other)) return refuse(S14_ERR_SHAPE, "out must have q's shape"), nullptr;
  if (rows_of(v[4], "k", device, shape[2], &k, ks) || rows_of(v[5], "v", device, shape[2], &x, other)) return nullptr;
  if (ks[0] != shape[0] || !same(ks, other)) return refuse(S14_ERR_SHAPE, "k and v must have one shape and q's tokens"), nullptr;
  if (v[6] == Py_None) return refuse(S14_ERR_INVALID, "cu is required"), nullptr;
  if (flat_of(v[6], "cu", device, at::kInt, 1, &cu)) return nullptr;
  if (flat_of(v[8], "lse", device, at::kFloat, (unsigned long long)shape[0] * shape[1], &lse)) return nullptr;
  if (scale_of(v[9], shape[2], &scale) || u32_of(v[10], "window", &window)) return nullptr;
  if (cu.bytes / 4 - 1 > UINT32_MAX) return refuse(S14_ERR_SHAPE, "cu is too long"), nullptr;
  if (stream_of(v[2], device, &stream)) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f_prompt(ctx, stream, (uint32_t)shape[2], &q, &k, &x, (uint32_t)shape[0], (uint32_t)(cu.bytes / 4 - 1), cu, &out, lse,
                scale, window);
  Py_END_ALLOW_THREADS
  return done(rc);
}

// bind(addresses of the four entry points, refuse, check, current stream)
static PyObject *bind(PyObject *, PyObject *args) {
  unsigned long long f[4];
  PyObject *p[3];
  if (!PyArg_ParseTuple(args, "(KKKK)OOO", &f[0], &f[1], &f[2], &f[3], &p[0], &p[1], &p[2])) return nullptr;
  f_norm_rope = (norm_rope_fn)(uintptr_t)f[0];
  f_append = (append_fn)(uintptr_t)f[1];
  f_paged = (paged_fn)(uintptr_t)f[2];
  f_prompt = (prompt_fn)(uintptr_t)f[3];
  PyObject **to[3] = {&p_refuse, &p_check, &p_stream};
  for (int i = 0; i < 3; ++i) {
    Py_INCREF(p[i]);
    Py_XSETREF(*to[i], p[i]);
  }
  Py_RETURN_NONE;
}

// What torch throws (a tensor without storage, say) becomes a refusal.
template <PyObject *(*call)(PyObject *, PyObject *const *, Py_ssize_t)>
static PyObject *guarded(PyObject *self, PyObject *const *v, Py_ssize_t argc) {
  try {
    return call(self, v, argc);
  } catch (const std::exception &e) {
    refuse(S14_ERR_INVALID, "%.200s", e.what());
  }
  return nullptr;
}

static PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, NULL},
    {"qk_norm_rope", (PyCFunction)(void (*)(void))guarded<qk_norm_rope>, METH_FASTCALL, NULL},
    {"kv_append", (PyCFunction)(void (*)(void))guarded<kv_append>, METH_FASTCALL, NULL},
    {"paged_attention", (PyCFunction)(void (*)(void))guarded<paged_attention>, METH_FASTCALL, NULL},
    {"prompt_attention", (PyCFunction)(void (*)(void))guarded<prompt_attention>, METH_FASTCALL, NULL},
    {NULL, NULL, 0, NULL},
};
static PyModuleDef module = {PyModuleDef_HEAD_INIT, "_s14attn", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__s14attn(void) { return PyModule_Create(&module); }
