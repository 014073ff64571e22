/* fastcall.c -- CPython entry points of the paged-cache operators.
 *
 * A decode step's operators run for a few microseconds, less than checking a dozen tensor
 * arguments in Python and converting them through ctypes takes (12 to 19 us a call). So the
 * checks are here: each tensor's attributes are read once through its Python interface (no
 * torch headers, no torch ABI), compared, and the C ABI of include/clove/capi.h, found in
 * the loaded library by init(), is called. clove_compute_b200/paged.py documents the
 * functions and handles streams and devices other than the current ones. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <dlfcn.h>
#include <limits.h>
#include <string.h>

#include "clove/capi.h"

static int (*p_rope)(const void*, const void*, const void*, long long, long long, long long,
                     const void*, const void*, float, const float*, int, int, int, const int*,
                     const clove_paged_cache*, const int*, void*, long long, void*, long long, int,
                     int, int, int, int, void*);
static int (*p_attn)(const void*, long long, const clove_paged_cache*, const int*, long long, int,
                     const int*, void*, long long, float*, float*, int, int, int, float, int, int,
                     void*);
static int (*p_evict)(const clove_paged_cache*, float*, const int*, long long, int, const int*,
                      const int*, long long, int, int*, int*, int, int, int, void*);

/* What init() is given: torch's dtypes in the order of Code, and Python callables. */
enum Code { kF16, kBF16, kE4M3, kF32, kI32, kCodes };
static const char* const kNames[kCodes] = {"torch.float16", "torch.bfloat16", "torch.float8_e4m3fn",
                                           "torch.float32", "torch.int32"};
static PyObject* g_dtype[kCodes];
static PyObject *g_empty_like, *g_empty_like_kw, *g_contiguous, *g_device, *g_stream, *g_check, *g_cache;
static PyObject *s_dtype, *s_shape, *s_stride, *s_data_ptr, *s_get_device, *s_new_empty, *s_key;

#define MAX_DIMS 4
typedef struct {
  const char* name;
  PyObject* obj;
  void* ptr;
  int code;   /* Code, or -1 */
  int index;  /* GPU, -1: not on one */
  int nd;     /* dimensions, MAX_DIMS + 1: more */
  long long size[MAX_DIMS], stride[MAX_DIMS];
} Tensor;

static int read_dims(PyObject* tuple, long long* out, int* nd) {
  if (tuple == NULL) return 0;
  int ok = PyTuple_Check(tuple);
  if (ok) {
    const Py_ssize_t n = PyTuple_GET_SIZE(tuple);
    *nd = n > MAX_DIMS ? MAX_DIMS + 1 : (int)n;
    for (Py_ssize_t i = 0; i < n && i < MAX_DIMS && ok; ++i) {
      out[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(tuple, i));
      ok = !(out[i] == -1 && PyErr_Occurred());
    }
  }
  Py_DECREF(tuple);
  return ok;
}

/* Reads a tensor's attributes. */
static int take(Tensor* t, PyObject* o, const char* name) {
  t->name = name;
  t->obj = o;
  t->code = -1;
  PyObject* d = PyObject_GetAttr(o, s_dtype);
  PyObject* dev = d ? PyObject_CallMethodNoArgs(o, s_get_device) : NULL;
  PyObject* ptr = dev ? PyObject_CallMethodNoArgs(o, s_data_ptr) : NULL;
  int nd = 0, ok = ptr != NULL;
  if (ok) {
    for (int i = 0; i < kCodes; ++i)
      if (d == g_dtype[i]) t->code = i;
    t->index = (int)PyLong_AsLong(dev);
    t->ptr = PyLong_AsVoidPtr(ptr);
    ok = !PyErr_Occurred() && read_dims(PyObject_GetAttr(o, s_shape), t->size, &t->nd) &&
         read_dims(PyObject_CallMethodNoArgs(o, s_stride), t->stride, &nd);
  }
  Py_XDECREF(d);
  Py_XDECREF(dev);
  Py_XDECREF(ptr);
  if (!ok) {
    /* A tensor without storage, in torch's own words. */
    if (PyErr_Occurred() && PyErr_ExceptionMatches(PyExc_RuntimeError)) return 0;
    PyErr_Clear();
    PyErr_Format(PyExc_TypeError, "%s must be a torch.Tensor", name);
  }
  return ok;
}

static int type_is(const Tensor* t, int code) {
  if (t->code == code) return 1;
  PyErr_Format(PyExc_TypeError, "%s must be %s", t->name, kNames[code]);
  return 0;
}

/* ValueError with the tensor's shape, strides and place. */
static int refuse(const Tensor* t, const char* want, int index) {
  PyObject* shape = PyObject_GetAttr(t->obj, s_shape);
  PyErr_Format(PyExc_ValueError, "%s must be %s on GPU %d; it is %R on %s %d", t->name, want, index,
               shape ? shape : Py_None, t->index < 0 ? "device" : "GPU", t->index);
  Py_XDECREF(shape);
  return 0;
}

/* A contiguous tensor of nd given sizes. */
static int dense(const Tensor* t, int code, int index, int nd, const long long* size) {
  if (!type_is(t, code)) return 0;
  int ok = t->index == index && t->nd == nd;
  long long step = 1;
  int empty = 0;
  for (int i = 0; i < nd; ++i) empty |= size[i] == 0;
  for (int i = nd - 1; i >= 0 && ok; --i) {
    ok = t->size[i] == size[i] && (empty || size[i] == 1 || t->stride[i] == step);
    step *= size[i];
  }
  if (ok) return 1;
  char want[160];
  int n = snprintf(want, sizeof(want), "contiguous [");
  for (int i = 0; i < nd; ++i) n += snprintf(want + n, sizeof(want) - (size_t)n, i ? ", %lld" : "%lld", size[i]);
  snprintf(want + n, sizeof(want) - (size_t)n, "]");
  return refuse(t, want, index);
}
static int dense1(const Tensor* t, int code, int index, long long n) { return dense(t, code, index, 1, &n); }

/* [rows, heads, D] whose rows are contiguous; *row gets the stride between them. */
static int heads(const Tensor* t, int code, int index, const long long* size, long long* row) {
  if (!type_is(t, code)) return 0;
  if (t->index != index || t->nd != 3 || t->size[0] != size[0] || t->size[1] != size[1] ||
      t->size[2] != size[2] || (size[2] > 1 && t->stride[2] != 1) || (size[1] > 1 && t->stride[1] != size[2])) {
    char want[160];
    snprintf(want, sizeof(want), "[%lld, %lld, %lld] with contiguous rows", size[0], size[1], size[2]);
    return refuse(t, want, index);
  }
  *row = size[0] > 1 ? t->stride[0] : size[1] * size[2];
  return 1;
}

/* [batch, pages] with contiguous rows. */
static int table(const Tensor* t, int index, long long batch) {
  if (!type_is(t, kI32)) return 0;
  if (t->index != index || t->nd != 2 || t->size[0] != batch || (t->size[1] > 1 && t->stride[1] != 1)) {
    char want[80];
    snprintf(want, sizeof(want), "[%lld, pages] with contiguous rows", batch);
    return refuse(t, want, index);
  }
  return 1;
}

/* The call's first operand: fp16 or bf16, three dimensions, on a GPU. */
static int operand(const Tensor* t) {
  if (t->code != kF16 && t->code != kBF16)
    PyErr_Format(PyExc_TypeError, "%s must be an fp16 or bf16 tensor", t->name);
  else if (t->index < 0)
    PyErr_Format(PyExc_ValueError, "%s must be a CUDA tensor", t->name);
  else if (t->nd != 3)
    refuse(t, "3-D", t->index);
  else
    return 1;
  return 0;
}

static int fits(long long v, const char* what) {
  if (v >= INT_MIN && v <= INT_MAX) return 1;
  PyErr_Format(PyExc_ValueError, "%s does not fit in 32 bits", what);
  return 0;
}

/* What a PagedCache describes; its GPU is *index, or is put there where that is -1. (Its _key
 * is (address, GPU); no other object's numbers are followed.) */
static const clove_paged_cache* cache_of(PyObject* cache, int* index) {
  const int is = PyObject_IsInstance(cache, g_cache);
  if (is <= 0) {
    if (is == 0) PyErr_SetString(PyExc_TypeError, "cache must be a PagedCache");
    return NULL;
  }
  PyObject* key = PyObject_GetAttr(cache, s_key);
  if (key == NULL) return NULL;
  const clove_paged_cache* c = NULL;
  long at = -1;
  if (PyTuple_Check(key) && PyTuple_GET_SIZE(key) == 2) {
    c = PyLong_AsVoidPtr(PyTuple_GET_ITEM(key, 0));
    at = PyLong_AsLong(PyTuple_GET_ITEM(key, 1));
  }
  Py_DECREF(key); /* the struct lives as long as the cache */
  if (PyErr_Occurred()) return NULL;
  if (*index < 0) *index = (int)at;
  if (c == NULL || at != *index) {
    PyErr_Format(PyExc_ValueError, "the cache must be on GPU %d", *index);
    return NULL;
  }
  return c;
}

/* The stream: a handle, or None for the current one. 0: an error; -1: GPU `index` is not
 * the current device (the caller switches to it). */
static int stream_of(PyObject* stream, int index, void** out) {
  if (stream != Py_None) {
    *out = PyLong_AsVoidPtr(stream);
    return PyErr_Occurred() ? 0 : 1;
  }
  PyObject* d = PyObject_CallNoArgs(g_device);
  if (d == NULL) return 0;
  const long now = PyLong_AsLong(d);
  PyObject* s = now == index ? PyObject_CallOneArg(g_stream, d) : NULL;
  Py_DECREF(d);
  if (now != index) return -1;
  if (s == NULL) return 0;
  *out = PyLong_AsVoidPtr(s);
  Py_DECREF(s);
  return PyErr_Occurred() ? 0 : 1;
}

/* torch.empty_like(t, memory_format=torch.contiguous_format) */
static PyObject* empty_like(PyObject* t) {
  PyObject* args[2] = {t, g_contiguous};
  return PyObject_Vectorcall(g_empty_like, args, 1, g_empty_like_kw);
}

static void* address(PyObject* t) {
  PyObject* p = PyObject_CallMethodNoArgs(t, s_data_ptr);
  void* v = p ? PyLong_AsVoidPtr(p) : NULL;
  Py_XDECREF(p);
  return v;
}

static int wants(Py_ssize_t got, Py_ssize_t need) {
  if (got == need && g_check != NULL) return 1;
  if (g_check == NULL)
    PyErr_SetString(PyExc_RuntimeError, "init() has not been called");
  else
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", need, got);
  return 0;
}

/* Status of the C ABI: 1 on success, else the package's exception is set. */
static int passed(int rc) {
  if (rc == CLOVE_OK) return 1;
  PyObject* r = PyObject_CallFunction(g_check, "i", rc);
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "status %d", rc);
  return 0;
}

/* Launches may wait for room in the stream's queue: other threads run meanwhile. */
#define CALL(rc, expr)                                  \
  Py_BEGIN_ALLOW_THREADS rc = (expr);                   \
  Py_END_ALLOW_THREADS

#define GIVEN(o) ((o) != Py_None)

/* qk_norm_rope(Q, K, table, positions, q_weight, k_weight, eps, interleaved, V, cache, slots,
 *              Q_out, K_out, stream) */
static PyObject* qk_norm_rope(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  (void)self;
  if (!wants(n, 14)) return NULL;
  Tensor q, k, t, pos, qw, kw, v, slots, qo, ko;
  qw.ptr = kw.ptr = v.ptr = slots.ptr = qo.ptr = ko.ptr = NULL;
  if (!take(&q, a[0], "Q") || !operand(&q)) return NULL;
  const int code = q.code;
  int index = q.index;
  void* s = NULL;
  const int here = stream_of(a[13], index, &s);
  if (here == 0) return NULL;
  if (here < 0) Py_RETURN_NOTIMPLEMENTED;
  const long long T = q.size[0], H = q.size[1], D = q.size[2];
  if (!take(&k, a[1], "K") || !take(&t, a[2], "rope_table") || !take(&pos, a[3], "positions")) return NULL;
  const long long kv[3] = {T, k.nd == 3 ? k.size[1] : 0, D};
  long long qs, ks, vs = 0, qos = H * D, kos = 0;
  if (!heads(&q, code, index, q.size, &qs) || !heads(&k, code, index, kv, &ks)) return NULL;
  if (t.nd != 2) return refuse(&t, "[positions, rotary_dim]", index), NULL;
  if (!dense(&t, kF32, index, 2, t.size) || !dense1(&pos, kI32, index, T)) return NULL;
  if (GIVEN(a[4]) != GIVEN(a[5])) {
    PyErr_SetString(PyExc_ValueError, "q_weight and k_weight: both or neither");
    return NULL;
  }
  if (GIVEN(a[4]) && (!take(&qw, a[4], "q_weight") || !take(&kw, a[5], "k_weight") ||
                      !dense1(&qw, code, index, D) || !dense1(&kw, code, index, D)))
    return NULL;
  const double eps = PyFloat_AsDouble(a[6]);
  const int inter = PyObject_IsTrue(a[7]);
  if (PyErr_Occurred()) return NULL;
  const clove_paged_cache* cache = NULL;
  if (GIVEN(a[9])) {
    if (!GIVEN(a[8]) || !GIVEN(a[10])) {
      PyErr_SetString(PyExc_ValueError, "a cache needs V and slots");
      return NULL;
    }
    if (!(cache = cache_of(a[9], &index)) || !take(&v, a[8], "V") || !take(&slots, a[10], "slots") ||
        !heads(&v, code, index, kv, &vs) || !dense1(&slots, kI32, index, T))
      return NULL;
  } else if (GIVEN(a[8]) || GIVEN(a[10])) {
    PyErr_SetString(PyExc_ValueError, "V and slots need a cache");
    return NULL;
  }
  if (!fits(T, "Q") || !fits(H, "Q") || !fits(D, "Q") || !fits(kv[1], "K") || !fits(t.size[0], "rope_table") ||
      !fits(t.size[1], "rope_table"))
    return NULL;
  PyObject *out_q, *out_k = Py_None;
  if (GIVEN(a[11])) {
    if (!take(&qo, a[11], "Q_out") || !heads(&qo, code, index, q.size, &qos)) return NULL;
    out_q = Py_NewRef(a[11]);
  } else {
    if ((out_q = empty_like(a[0])) == NULL) return NULL;
    qo.ptr = address(out_q);
  }
  if (GIVEN(a[12])) {
    if (!take(&ko, a[12], "K_out") || !heads(&ko, code, index, kv, &kos)) goto failed;
    Py_INCREF(out_k = a[12]);
  } else if (cache == NULL) {
    if ((out_k = empty_like(a[1])) == NULL) goto failed;
    ko.ptr = address(out_k);
    kos = kv[1] * D;
  } else {
    Py_INCREF(out_k);
  }
  int rc;
  CALL(rc, p_rope(q.ptr, k.ptr, v.ptr, qs, ks, vs, qw.ptr, kw.ptr, (float)eps, t.ptr, (int)t.size[0],
                  (int)t.size[1], inter, pos.ptr, cache, slots.ptr, qo.ptr, qos, ko.ptr, kos, (int)T, (int)H,
                  (int)kv[1], (int)D, code, s));
  if (passed(rc)) {
    PyObject* r = PyTuple_Pack(2, out_q, out_k);
    Py_DECREF(out_q);
    Py_DECREF(out_k);
    return r;
  }
  Py_DECREF(out_k);
failed:
  Py_DECREF(out_q);
  return NULL;
}

/* paged_attention(Q, cache, page_table, seq_lens, scale, window, lse, key_weights, accumulate,
 *                 O, stream) */
static PyObject* paged_attention(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  (void)self;
  if (!wants(n, 11)) return NULL;
  Tensor q, pt, sl, lse, kw, o;
  lse.ptr = kw.ptr = NULL;
  if (!take(&q, a[0], "Q") || !operand(&q)) return NULL;
  const int code = q.code;
  int index = q.index;
  void* s = NULL;
  const int here = stream_of(a[10], index, &s);
  if (here == 0) return NULL;
  if (here < 0) Py_RETURN_NOTIMPLEMENTED;
  const clove_paged_cache* c = cache_of(a[1], &index);
  if (c == NULL) return NULL;
  const long long B = q.size[0], H = q.size[1], D = q.size[2];
  if (D != c->head_dim) {
    PyErr_Format(PyExc_ValueError, "Q has head_dim %lld, the cache %d", D, c->head_dim);
    return NULL;
  }
  long long qs, os = H * D;
  if (!heads(&q, code, index, q.size, &qs) || !take(&pt, a[2], "page_table") || !table(&pt, index, B) ||
      !take(&sl, a[3], "seq_lens") || !dense1(&sl, kI32, index, B))
    return NULL;
  const double scale = GIVEN(a[4]) ? PyFloat_AsDouble(a[4]) : 0.0;
  const long long window = PyLong_AsLongLong(a[5]);
  const int acc = PyObject_IsTrue(a[8]);
  if (PyErr_Occurred()) return NULL;
  const long long bh[2] = {B, H}, w[3] = {c->num_pages, c->num_kv_heads, c->page_size};
  if (GIVEN(a[6]) && (!take(&lse, a[6], "lse") || !dense(&lse, kF32, index, 2, bh))) return NULL;
  if (GIVEN(a[7])) {
    if (!take(&kw, a[7], "key_weights") || !dense(&kw, kF32, index, 3, w)) return NULL;
  } else if (acc) {
    PyErr_SetString(PyExc_ValueError, "accumulate needs key_weights");
    return NULL;
  }
  if (!fits(B, "Q") || !fits(H, "Q") || !fits(pt.size[1], "page_table") || !fits(window, "window")) return NULL;
  PyObject* out;
  if (GIVEN(a[9])) {
    if (!take(&o, a[9], "O") || !heads(&o, code, index, q.size, &os)) return NULL;
    out = Py_NewRef(a[9]);
  } else {
    if ((out = empty_like(a[0])) == NULL) return NULL;
    o.ptr = address(out);
  }
  /* 1 / sqrt(D) of the supported 64, 128 and 256; of others any number: they are refused. */
  const float usual = D == 64 ? 0.125f : D == 256 ? 0.0625f : 0.08838834764831845f;
  int rc;
  CALL(rc, p_attn(q.ptr, qs, c, pt.ptr, pt.stride[0], (int)pt.size[1], sl.ptr, o.ptr, os, lse.ptr, kw.ptr, acc,
                  (int)B, (int)H, GIVEN(a[4]) ? (float)scale : usual, (int)window, code, s));
  if (passed(rc)) return out;
  Py_DECREF(out);
  return NULL;
}

/* evict_cache(cache, key_weights, page_table, seq_lens, dst_table, budget, recent, stream) */
static PyObject* evict_cache(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  (void)self;
  if (!wants(n, 8)) return NULL;
  int index = -1;
  const clove_paged_cache* c = cache_of(a[0], &index);
  if (c == NULL) return NULL;
  void* s = NULL;
  const int here = stream_of(a[7], index, &s);
  if (here == 0) return NULL;
  if (here < 0) Py_RETURN_NOTIMPLEMENTED;
  Tensor kw, pt, sl, dst;
  const long long w[3] = {c->num_pages, c->num_kv_heads, c->page_size};
  if (!take(&sl, a[3], "seq_lens") || !type_is(&sl, kI32)) return NULL;
  const long long B = sl.nd == 1 ? sl.size[0] : -1;
  if (!dense1(&sl, kI32, index, B) || !take(&kw, a[1], "key_weights") || !dense(&kw, kF32, index, 3, w) ||
      !take(&pt, a[2], "page_table") || !table(&pt, index, B) || !take(&dst, a[4], "dst_table") ||
      !table(&dst, index, B))
    return NULL;
  const long long budget = PyLong_AsLongLong(a[5]), recent = PyLong_AsLongLong(a[6]);
  if (PyErr_Occurred()) return NULL;
  if (budget <= 0) {
    PyErr_SetString(PyExc_ValueError, "budget must be positive");
    return NULL;
  }
  if (!fits(B, "seq_lens") || !fits(pt.size[1], "page_table") || !fits(dst.size[1], "dst_table") ||
      !fits(budget, "budget") || !fits(recent, "recent"))
    return NULL;
  PyObject* shape = Py_BuildValue("(LiL)", B, c->num_kv_heads, budget);
  PyObject* kept = shape ? PyObject_CallMethodOneArg(a[3], s_new_empty, shape) : NULL;
  PyObject* lens = kept ? empty_like(a[3]) : NULL;
  Py_XDECREF(shape);
  int rc;
  if (lens != NULL) {
    int* kp = address(kept);
    int* lp = address(lens);
    CALL(rc, p_evict(c, kw.ptr, pt.ptr, pt.stride[0], (int)pt.size[1], sl.ptr, dst.ptr, dst.stride[0],
                     (int)dst.size[1], kp, lp, (int)B, (int)budget, (int)recent, s));
    if (passed(rc)) {
      PyObject* r = PyTuple_Pack(2, kept, lens);
      Py_DECREF(kept);
      Py_DECREF(lens);
      return r;
    }
  }
  Py_XDECREF(kept);
  Py_XDECREF(lens);
  return NULL;
}

/* init(library path, (dtypes), empty_like, contiguous_format, current device, current stream,
 *      check, PagedCache) */
static PyObject* init(PyObject* self, PyObject* args) {
  (void)self;
  const char* path;
  PyObject *dtypes, *like, *format, *device, *stream, *check, *cache;
  if (!PyArg_ParseTuple(args, "sO!OOOOOO", &path, &PyTuple_Type, &dtypes, &like, &format, &device, &stream, &check,
                        &cache))
    return NULL;
  if (PyTuple_GET_SIZE(dtypes) != kCodes) return PyErr_Format(PyExc_ValueError, "%d dtypes expected", kCodes);
  void* lib = dlopen(path, RTLD_NOW | RTLD_LOCAL);
  if (lib == NULL) return PyErr_Format(PyExc_ImportError, "%s", dlerror());
  *(void**)&p_rope = dlsym(lib, "clove_qk_norm_rope");
  *(void**)&p_attn = dlsym(lib, "clove_paged_attention");
  *(void**)&p_evict = dlsym(lib, "clove_evict_cache");
  if (!p_rope || !p_attn || !p_evict)
    return PyErr_Format(PyExc_ImportError, "%s lacks the paged-cache entry points", path);
  for (int i = 0; i < kCodes; ++i) g_dtype[i] = Py_NewRef(PyTuple_GET_ITEM(dtypes, i));
  g_empty_like = Py_NewRef(like);
  g_contiguous = Py_NewRef(format);
  g_device = Py_NewRef(device);
  g_stream = Py_NewRef(stream);
  g_empty_like_kw = Py_BuildValue("(s)", "memory_format");
  s_dtype = PyUnicode_InternFromString("dtype");
  s_shape = PyUnicode_InternFromString("shape");
  s_stride = PyUnicode_InternFromString("stride");
  s_data_ptr = PyUnicode_InternFromString("data_ptr");
  s_get_device = PyUnicode_InternFromString("get_device");
  s_new_empty = PyUnicode_InternFromString("new_empty");
  s_key = PyUnicode_InternFromString("_key");
  if (!g_empty_like_kw || !s_dtype || !s_shape || !s_stride || !s_data_ptr || !s_get_device || !s_new_empty ||
      !s_key)
    return NULL;
  g_cache = Py_NewRef(cache);
  g_check = Py_NewRef(check);
  Py_RETURN_NONE;
}

static PyMethodDef methods[] = {
    {"init", init, METH_VARARGS, "binds the library and torch's objects"},
    {"qk_norm_rope", (PyCFunction)(void (*)(void))qk_norm_rope, METH_FASTCALL, "see paged.py"},
    {"paged_attention", (PyCFunction)(void (*)(void))paged_attention, METH_FASTCALL, "see paged.py"},
    {"evict_cache", (PyCFunction)(void (*)(void))evict_cache, METH_FASTCALL, "see paged.py"},
    {NULL, NULL, 0, NULL}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fastcall", NULL, -1, methods,
                                    NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__fastcall(void) { return PyModule_Create(&module); }
