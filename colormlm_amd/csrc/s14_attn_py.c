/* The attention entry points' Python call, in C: a single token's call is a
 * few us of GPU work, and reading its tensors' types, shapes, strides and
 * addresses in Python and handing them over through ctypes took longer than
 * that (norm and rotation of one token: 9.3 us a call in Python, 5.4 here, of
 * which the launch is about 4).
 *
 * No part of libs14hip.so: colormlm_amd/attention.py loads it and gives it the
 * library's entry points.  It knows tensors only by their Python methods. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <math.h>
#include <string.h>

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
static PyObject *t_f32, *t_bf16, *t_i32;             /* torch's dtypes */
static PyObject *p_refuse, *p_check, *p_stream;      /* attention.py's functions */
static PyObject *n_dtype, *n_shape, *n_stride, *n_data_ptr, *n_get_device, *n_is_contiguous, *n_nbytes;

/* Raises S14Error(code, message); returns -1. */
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

static int not_here(const char *label, long device) {
  PyErr_Clear();
  return refuse(S14_ERR_INVALID, "%s must be a tensor on the context's device %ld", label, device);
}

/* An int property or method result; -1 with an exception if there is none. */
static int call_long(PyObject *t, PyObject *name, unsigned long long *out) {
  PyObject *r = PyObject_CallMethodNoArgs(t, name);
  if (!r) return -1;
  *out = PyLong_AsUnsignedLongLongMask(r);
  Py_DECREF(r);
  return PyErr_Occurred() ? -1 : 0;
}

static int on_device(PyObject *t, const char *label, long device) {
  unsigned long long d = 0;
  if (call_long(t, n_get_device, &d) || (long)d != device) return not_here(label, device);
  return 0;
}

/* The s14_rows of a [tokens, heads, dim] tensor (dim 0: any). */
static int rows_of(PyObject *t, const char *label, long device, long long dim, s14_rows *r, long long shape[3]) {
  PyObject *dtype = PyObject_GetAttr(t, n_dtype);
  if (!dtype) return not_here(label, device);
  const int f32 = dtype == t_f32, known = f32 || dtype == t_bf16;
  Py_DECREF(dtype);
  if (on_device(t, label, device)) return -1;
  if (!known) return refuse(S14_ERR_INVALID, "%s must be float32 or bfloat16", label);
  PyObject *size = PyObject_GetAttr(t, n_shape), *stride = size ? PyObject_CallMethodNoArgs(t, n_stride) : NULL;
  long long step[3] = {0, 0, 0};
  int ok = stride && PyTuple_Check(size) && PyTuple_Check(stride) && PyTuple_GET_SIZE(size) == 3 &&
           PyTuple_GET_SIZE(stride) == 3;
  for (int i = 0; ok && i < 3; ++i) {
    shape[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(size, i));
    step[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(stride, i));
  }
  Py_XDECREF(size);
  Py_XDECREF(stride);
  if (PyErr_Occurred()) return -1;
  if (!ok || (step[2] != 1 && shape[2] > 1) || (dim && shape[2] != dim))
    return refuse(S14_ERR_SHAPE, "%s must be [tokens, heads, dim] of the call's dim, its last dimension contiguous", label);
  if (shape[0] > UINT32_MAX || shape[1] > UINT32_MAX || shape[2] > UINT32_MAX || step[1] > UINT32_MAX)
    return refuse(S14_ERR_SHAPE, "%s is too large", label);
  unsigned long long at = 0;
  if (call_long(t, n_data_ptr, &at)) return -1;
  /* strides of a dimension of one are not used; what torch gives there may be anything */
  if (shape[0] < 2) step[0] = 0;
  if (shape[1] < 2) step[1] = 0;
  r->buf.ptr = (void *)(uintptr_t)at;
  r->buf.bytes = shape[0] && shape[1]
                     ? (uint64_t)((shape[0] - 1) * step[0] + (shape[1] - 1) * step[1] + shape[2]) * (f32 ? 4 : 2)
                     : 0;
  r->dtype = f32 ? S14_X_F32 : S14_X_BF16;
  r->heads = (uint32_t)shape[1];
  r->token_stride = (uint64_t)step[0];
  r->head_stride = (uint32_t)step[1];
  return 0;
}

/* The buffer of a contiguous tensor of one 4-byte dtype, of `values` at least; None: no buffer. */
static int flat_of(PyObject *t, const char *label, long device, PyObject *dtype, unsigned long long values, s14_buffer *b) {
  b->ptr = NULL, b->bytes = 0;
  if (t == Py_None) return 0;
  PyObject *have = PyObject_GetAttr(t, n_dtype);
  if (!have) return not_here(label, device);
  Py_DECREF(have);
  if (on_device(t, label, device)) return -1;
  PyObject *whole = have == dtype ? PyObject_CallMethodNoArgs(t, n_is_contiguous) : Py_NewRef(Py_False);
  if (!whole) return -1;
  Py_DECREF(whole);
  if (whole != Py_True) return refuse(S14_ERR_INVALID, "%s must be a contiguous %s tensor", label, dtype == t_f32 ? "float32" : "int32");
  PyObject *n = PyObject_GetAttr(t, n_nbytes);
  if (!n) return -1;
  const unsigned long long bytes = PyLong_AsUnsignedLongLong(n);
  Py_DECREF(n);
  if (PyErr_Occurred()) return -1;
  if (bytes < 4 * values) return refuse(S14_ERR_CAPACITY, "%s has %llu values, %llu are required", label, bytes / 4, values);
  unsigned long long at = 0;
  if (call_long(t, n_data_ptr, &at)) return -1;
  b->ptr = (void *)(uintptr_t)at, b->bytes = bytes;
  return 0;
}

/* A [sequences, pages] page table with its cu and lengths. */
typedef struct {
  s14_buffer table, cu, len;
  uint32_t seqs, width;
} index_rows;
static int index_of(PyObject *table, PyObject *cu, PyObject *len, const char *label, long device, index_rows *x) {
  if (table == Py_None || cu == Py_None || len == Py_None) return refuse(S14_ERR_INVALID, "page table, cu and %s are required", label);
  if (flat_of(table, "page table", device, t_i32, 0, &x->table)) return -1;
  PyObject *size = PyObject_GetAttr(table, n_shape);
  long long seqs = -1, width = -1;
  if (size && PyTuple_Check(size) && PyTuple_GET_SIZE(size) == 2) {
    seqs = PyLong_AsLongLong(PyTuple_GET_ITEM(size, 0));
    width = PyLong_AsLongLong(PyTuple_GET_ITEM(size, 1));
  }
  Py_XDECREF(size);
  if (PyErr_Occurred()) return -1;
  if (seqs < 0 || width < 0 || seqs > UINT32_MAX || width > UINT32_MAX)
    return refuse(S14_ERR_SHAPE, "a page table is [sequences, pages]");
  x->seqs = (uint32_t)seqs, x->width = (uint32_t)width;
  if (flat_of(cu, "cu", device, t_i32, (unsigned long long)seqs + 1, &x->cu)) return -1;
  return flat_of(len, label, device, t_i32, (unsigned long long)seqs, &x->len);
}

/* The stream: the caller's, or the device's current one. */
static int stream_of(PyObject *stream, long device, void **out) {
  PyObject *r = stream == Py_None ? PyObject_CallFunction(p_stream, "l", device) : Py_NewRef(stream);
  if (!r) return -1;
  *out = (void *)(uintptr_t)PyLong_AsUnsignedLongLong(r);
  Py_DECREF(r);
  return PyErr_Occurred() ? -1 : 0;
}

/* An unsigned 32-bit argument. */
static int u32_of(PyObject *v, const char *label, uint32_t *out) {
  const long long x = PyLong_AsLongLong(v);
  if (x == -1 && PyErr_Occurred()) return -1;
  if (x < 0 || x > UINT32_MAX) return refuse(S14_ERR_INVALID, "%s is %lld", label, x);
  *out = (uint32_t)x;
  return 0;
}

static void *pointer_of(PyObject *v) { return v == Py_None ? NULL : PyLong_AsVoidPtr(v); }

static PyObject *done(int rc) {
  if (!rc) Py_RETURN_NONE;
  PyObject *r = PyObject_CallFunction(p_check, "i", rc);
  Py_XDECREF(r);
  if (PyErr_Occurred()) return NULL;
  Py_RETURN_NONE;
}

static int same(const long long a[3], const long long b[3]) { return a[0] == b[0] && a[1] == b[1] && a[2] == b[2]; }

#define ARGUMENTS(n)                                                                              \
  do {                                                                                            \
    if (argc != (n)) return PyErr_Format(PyExc_TypeError, "%d arguments, not %zd", (n), argc);    \
  } while (0)

/* handle, device, stream, q, k, q_out, k_out, q_weight, k_weight, eps, rope, positions */
static PyObject *qk_norm_rope(PyObject *self, PyObject *const *v, Py_ssize_t argc) {
  (void)self;
  ARGUMENTS(12);
  s14_ctx *ctx = pointer_of(v[0]);
  const long device = PyLong_AsLong(v[1]);
  const double eps = PyFloat_AsDouble(v[9]);
  const s14_rope *rope = pointer_of(v[10]);
  void *stream;
  s14_rows q, qo, k, ko;
  s14_buffer qw, kw, pos;
  long long shape[3], other[3], ks[3];
  if (PyErr_Occurred()) return NULL;
  if (rows_of(v[3], "q", device, 0, &q, shape) || rows_of(v[5], "q output", device, shape[2], &qo, other)) return NULL;
  if (!same(shape, other)) return refuse(S14_ERR_SHAPE, "q output must have q's shape"), NULL;
  if (v[4] == Py_None) {
    memset(&k, 0, sizeof k);
    ko = k;
  } else {
    if (rows_of(v[4], "k", device, shape[2], &k, ks) || rows_of(v[6], "k output", device, shape[2], &ko, other)) return NULL;
    if (ks[0] != shape[0] || !same(ks, other))
      return refuse(S14_ERR_SHAPE, "k must have q's tokens, and k output k's shape"), NULL;
  }
  if (flat_of(v[7], "q norm weight", device, t_f32, 0, &qw) || flat_of(v[8], "k norm weight", device, t_f32, 0, &kw) ||
      flat_of(v[11], "positions", device, t_i32, 0, &pos))
    return NULL;
  if (stream_of(v[2], device, &stream)) return NULL;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f_norm_rope(ctx, stream, (uint32_t)shape[0], (uint32_t)shape[2], &q, &k, &qo, &ko, qw, kw, (float)eps, rope, pos);
  Py_END_ALLOW_THREADS
  return done(rc);
}

/* handle, device, stream, cache, dim, k, v, page_table, cu, past, k_weight, eps, rope, max_new */
static PyObject *kv_append(PyObject *self, PyObject *const *v, Py_ssize_t argc) {
  (void)self;
  ARGUMENTS(14);
  s14_ctx *ctx = pointer_of(v[0]);
  const long device = PyLong_AsLong(v[1]);
  const s14_kv_cache *cache = pointer_of(v[3]);
  const long long dim = PyLong_AsLongLong(v[4]);
  const double eps = PyFloat_AsDouble(v[11]);
  const s14_rope *rope = pointer_of(v[12]);
  void *stream;
  s14_rows k, x;
  s14_buffer kw;
  index_rows at;
  long long shape[3], other[3];
  uint32_t most;
  if (PyErr_Occurred()) return NULL;
  if (rows_of(v[5], "k", device, dim, &k, shape) || rows_of(v[6], "v", device, dim, &x, other)) return NULL;
  if (shape[0] != other[0]) return refuse(S14_ERR_SHAPE, "k and v have different token counts"), NULL;
  if (index_of(v[7], v[8], v[9], "past", device, &at) || flat_of(v[10], "k norm weight", device, t_f32, 0, &kw)) return NULL;
  most = (uint32_t)shape[0];
  if (v[13] != Py_None && u32_of(v[13], "max_new", &most)) return NULL;
  if (stream_of(v[2], device, &stream)) return NULL;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f_append(ctx, stream, cache, (uint32_t)shape[0], at.seqs, most, &k, &x, at.table, at.width, at.cu, at.len, kw,
                (float)eps, rope);
  Py_END_ALLOW_THREADS
  return done(rc);
}

/* scale: None is 1 / sqrt(dim) */
static int scale_of(PyObject *v, long long dim, float *out) {
  const double s = v == Py_None ? 1.0 / sqrt((double)(dim ? dim : 1)) : PyFloat_AsDouble(v);
  *out = (float)s;
  return PyErr_Occurred() ? -1 : 0;
}

/* handle, device, stream, q, cache, dim, page_table, cu, lens, out, lse, scale, window, max_new, max_len, reach of the table's pages */
static PyObject *paged_attention(PyObject *self, PyObject *const *v, Py_ssize_t argc) {
  (void)self;
  ARGUMENTS(16);
  s14_ctx *ctx = pointer_of(v[0]);
  const long device = PyLong_AsLong(v[1]);
  const s14_kv_cache *cache = pointer_of(v[4]);
  const long long dim = PyLong_AsLongLong(v[5]);
  const long long page = PyLong_AsLongLong(v[15]);
  void *stream;
  s14_rows q, out;
  s14_buffer lse;
  index_rows at;
  long long shape[3], other[3];
  uint32_t window = 0, most, length;
  float scale;
  if (PyErr_Occurred()) return NULL;
  if (rows_of(v[3], "q", device, dim, &q, shape) || rows_of(v[9], "out", device, dim, &out, other)) return NULL;
  if (!same(shape, other)) return refuse(S14_ERR_SHAPE, "out must have q's shape"), NULL;
  if (index_of(v[6], v[7], v[8], "lens", device, &at)) return NULL;
  if (flat_of(v[10], "lse", device, t_f32, (unsigned long long)shape[0] * shape[1], &lse)) return NULL;
  if (scale_of(v[11], dim, &scale) || u32_of(v[12], "window", &window)) return NULL;
  most = (uint32_t)shape[0];
  if (v[13] != Py_None && u32_of(v[13], "max_new", &most)) return NULL;
  const unsigned long long reach = (unsigned long long)at.width * (unsigned long long)page;
  length = reach > INT32_MAX ? INT32_MAX : (uint32_t)reach;
  if (v[14] != Py_None && u32_of(v[14], "max_len", &length)) return NULL;
  if (stream_of(v[2], device, &stream)) return NULL;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f_paged(ctx, stream, &q, cache, (uint32_t)shape[0], at.seqs, most, length, at.table, at.width, at.cu, at.len, &out,
               lse, scale, window);
  Py_END_ALLOW_THREADS
  return done(rc);
}

/* handle, device, stream, q, k, v, cu, out, lse, scale, window */
static PyObject *prompt_attention(PyObject *self, PyObject *const *v, Py_ssize_t argc) {
  (void)self;
  ARGUMENTS(11);
  s14_ctx *ctx = pointer_of(v[0]);
  const long device = PyLong_AsLong(v[1]);
  void *stream;
  s14_rows q, k, x, out;
  s14_buffer cu, lse;
  long long shape[3], ks[3], other[3];
  uint32_t window = 0;
  float scale;
  if (PyErr_Occurred()) return NULL;
  if (rows_of(v[3], "q", device, 0, &q, shape) || rows_of(v[7], "out", device, shape[2], &out, other)) return NULL;
  if (!same(shape, other)) return refuse(S14_ERR_SHAPE, "out must have q's shape"), NULL;
  if (rows_of(v[4], "k", device, shape[2], &k, ks) || rows_of(v[5], "v", device, shape[2], &x, other)) return NULL;
  if (ks[0] != shape[0] || !same(ks, other)) return refuse(S14_ERR_SHAPE, "k and v must have one shape and q's tokens"), NULL;
  if (v[6] == Py_None) return refuse(S14_ERR_INVALID, "cu is required"), NULL;
  if (flat_of(v[6], "cu", device, t_i32, 1, &cu)) return NULL;
  if (flat_of(v[8], "lse", device, t_f32, (unsigned long long)shape[0] * shape[1], &lse)) return NULL;
  if (scale_of(v[9], shape[2], &scale) || u32_of(v[10], "window", &window)) return NULL;
  if (cu.bytes / 4 - 1 > UINT32_MAX) return refuse(S14_ERR_SHAPE, "cu is too long"), NULL;
  if (stream_of(v[2], device, &stream)) return NULL;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f_prompt(ctx, stream, (uint32_t)shape[2], &q, &k, &x, (uint32_t)shape[0], (uint32_t)(cu.bytes / 4 - 1), cu, &out, lse,
                scale, window);
  Py_END_ALLOW_THREADS
  return done(rc);
}

/* bind(addresses of the four entry points, (f32, bf16, i32), refuse, check, current stream) */
static PyObject *bind(PyObject *self, PyObject *args) {
  (void)self;
  unsigned long long f[4];
  PyObject *d[3], *p[3];
  if (!PyArg_ParseTuple(args, "(KKKK)(OOO)OOO", &f[0], &f[1], &f[2], &f[3], &d[0], &d[1], &d[2], &p[0], &p[1], &p[2])) return NULL;
  f_norm_rope = (norm_rope_fn)(uintptr_t)f[0];
  f_append = (append_fn)(uintptr_t)f[1];
  f_paged = (paged_fn)(uintptr_t)f[2];
  f_prompt = (prompt_fn)(uintptr_t)f[3];
  PyObject **to[6] = {&t_f32, &t_bf16, &t_i32, &p_refuse, &p_check, &p_stream};
  for (int i = 0; i < 6; ++i) {
    PyObject *x = i < 3 ? d[i] : p[i - 3];
    Py_INCREF(x);
    Py_XSETREF(*to[i], x);
  }
  Py_RETURN_NONE;
}

static PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, NULL},
    {"qk_norm_rope", (PyCFunction)(void (*)(void))qk_norm_rope, METH_FASTCALL, NULL},
    {"kv_append", (PyCFunction)(void (*)(void))kv_append, METH_FASTCALL, NULL},
    {"paged_attention", (PyCFunction)(void (*)(void))paged_attention, METH_FASTCALL, NULL},
    {"prompt_attention", (PyCFunction)(void (*)(void))prompt_attention, METH_FASTCALL, NULL},
    {NULL, NULL, 0, NULL},
};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_s14attn", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__s14attn(void) {
  n_dtype = PyUnicode_InternFromString("dtype");
  n_shape = PyUnicode_InternFromString("shape");
  n_stride = PyUnicode_InternFromString("stride");
  n_data_ptr = PyUnicode_InternFromString("data_ptr");
  n_get_device = PyUnicode_InternFromString("get_device");
  n_is_contiguous = PyUnicode_InternFromString("is_contiguous");
  n_nbytes = PyUnicode_InternFromString("nbytes");
  return n_nbytes ? PyModule_Create(&module) : NULL;
}
