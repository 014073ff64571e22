/* fastcall.c -- CPython entry points of the paged-cache operators.
 *
 * The decode step's operators take 15 to 26 arguments; through ctypes their conversion
 * alone costs about 5 us a call, more than the kernels of a small step. These functions
 * take the same arguments positionally (addresses as int or None) and call the C ABI of
 * include/clove/capi.h, found in the loaded library by init(). They return its status. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <dlfcn.h>

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

static void* ptr(PyObject* o) { return o == Py_None ? NULL : PyLong_AsVoidPtr(o); }
static long long ll(PyObject* o) { return PyLong_AsLongLong(o); }
static int in(PyObject* o) {
  const long v = PyLong_AsLong(o);
  if (v != (int)v) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_OverflowError, "argument does not fit in 32 bits");
    return -1;
  }
  return (int)v;
}
static float fl(PyObject* o) { return (float)PyFloat_AsDouble(o); }

static int wants(Py_ssize_t got, Py_ssize_t need, const void* fn) {
  if (got != need)
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", need, got);
  else if (fn == NULL)
    PyErr_SetString(PyExc_RuntimeError, "init() has not been called");
  else
    return 1;
  return 0;
}

/* Launches may wait for room in the stream's queue: other threads run meanwhile. */
#define CALL(expr)            \
  int rc;                     \
  if (PyErr_Occurred()) return NULL; \
  Py_BEGIN_ALLOW_THREADS rc = (expr); \
  Py_END_ALLOW_THREADS return PyLong_FromLong(rc)

static PyObject* qk_norm_rope(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  (void)self;
  if (!wants(n, 26, (const void*)p_rope)) return NULL;
  const void *q = ptr(a[0]), *k = ptr(a[1]), *v = ptr(a[2]);
  const long long qs = ll(a[3]), ks = ll(a[4]), vs = ll(a[5]);
  const void *qw = ptr(a[6]), *kw = ptr(a[7]);
  const float eps = fl(a[8]);
  const float* table = ptr(a[9]);
  const int len = in(a[10]), rot = in(a[11]), il = in(a[12]);
  const int* pos = ptr(a[13]);
  const clove_paged_cache* cache = ptr(a[14]);
  const int* slots = ptr(a[15]);
  void* qo = ptr(a[16]);
  const long long qos = ll(a[17]);
  void* ko = ptr(a[18]);
  const long long kos = ll(a[19]);
  const int t = in(a[20]), h = in(a[21]), hkv = in(a[22]), d = in(a[23]), dt = in(a[24]);
  void* s = ptr(a[25]);
  CALL(p_rope(q, k, v, qs, ks, vs, qw, kw, eps, table, len, rot, il, pos, cache, slots, qo, qos, ko,
              kos, t, h, hkv, d, dt, s));
}

static PyObject* paged_attention(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  (void)self;
  if (!wants(n, 18, (const void*)p_attn)) return NULL;
  const void* q = ptr(a[0]);
  const long long qs = ll(a[1]);
  const clove_paged_cache* cache = ptr(a[2]);
  const int* table = ptr(a[3]);
  const long long ts = ll(a[4]);
  const int pages = in(a[5]);
  const int* lens = ptr(a[6]);
  void* o = ptr(a[7]);
  const long long os = ll(a[8]);
  float *lse = ptr(a[9]), *kw = ptr(a[10]);
  const int acc = in(a[11]), b = in(a[12]), h = in(a[13]);
  const float scale = fl(a[14]);
  const int window = in(a[15]), dt = in(a[16]);
  void* s = ptr(a[17]);
  CALL(p_attn(q, qs, cache, table, ts, pages, lens, o, os, lse, kw, acc, b, h, scale, window, dt, s));
}

static PyObject* evict_cache(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  (void)self;
  if (!wants(n, 15, (const void*)p_evict)) return NULL;
  const clove_paged_cache* cache = ptr(a[0]);
  float* w = ptr(a[1]);
  const int* table = ptr(a[2]);
  const long long ts = ll(a[3]);
  const int pages = in(a[4]);
  const int *lens = ptr(a[5]), *dst = ptr(a[6]);
  const long long ds = ll(a[7]);
  const int dp = in(a[8]);
  int *kept = ptr(a[9]), *nl = ptr(a[10]);
  const int b = in(a[11]), budget = in(a[12]), recent = in(a[13]);
  void* s = ptr(a[14]);
  CALL(p_evict(cache, w, table, ts, pages, lens, dst, ds, dp, kept, nl, b, budget, recent, s));
}

/* init(path of libclove_b200.so) */
static PyObject* init(PyObject* self, PyObject* path) {
  (void)self;
  const char* p = PyUnicode_AsUTF8(path);
  if (p == NULL) return NULL;
  void* lib = dlopen(p, RTLD_NOW | RTLD_LOCAL);
  if (lib == NULL) return PyErr_Format(PyExc_ImportError, "%s", dlerror());
  *(void**)&p_rope = dlsym(lib, "clove_qk_norm_rope");
  *(void**)&p_attn = dlsym(lib, "clove_paged_attention");
  *(void**)&p_evict = dlsym(lib, "clove_evict_cache");
  if (!p_rope || !p_attn || !p_evict)
    return PyErr_Format(PyExc_ImportError, "%s lacks the paged-cache entry points", p);
  Py_RETURN_NONE;
}

static PyMethodDef methods[] = {
    {"init", init, METH_O, "init(library path)"},
    {"qk_norm_rope", (PyCFunction)(void (*)(void))qk_norm_rope, METH_FASTCALL, "clove_qk_norm_rope"},
    {"paged_attention", (PyCFunction)(void (*)(void))paged_attention, METH_FASTCALL, "clove_paged_attention"},
    {"evict_cache", (PyCFunction)(void (*)(void))evict_cache, METH_FASTCALL, "clove_evict_cache"},
    {NULL, NULL, 0, NULL}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fastcall", NULL, -1, methods,
                                    NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__fastcall(void) { return PyModule_Create(&module); }
