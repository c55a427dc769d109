/* Argument conversion for the entry points that a decode step calls in every layer.
 *
 * ctypes takes some 90 ns an argument; these entry points have 17 to 31, and the
 * kernels behind them run for a few microseconds. This module converts the same
 * arguments at a tenth of that and calls the same functions of libqtts_b200.so by
 * address (bind). It holds nothing else: the binding works without it, through
 * ctypes (qtts_b200/_native.py).
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "../../include/qtts_b200.h"

enum { ADD_RMS_NORM_QUANT, ROPE_KV4_APPEND, KV4_ATTENTION, ENTRIES };
static void* entry[ENTRIES];

static void* ptr(PyObject* o) { return o == Py_None ? NULL : PyLong_AsVoidPtr(o); }
static int64_t i64(PyObject* o) { return PyLong_AsLongLong(o); }
static int num(PyObject* o) {
  const long v = PyLong_AsLong(o);
  if (v != (int)v && !PyErr_Occurred()) PyErr_SetString(PyExc_OverflowError, "argument does not fit an int");
  return (int)v;
}
static unsigned flags(PyObject* o) { return (unsigned)PyLong_AsUnsignedLongMask(o); }
static float real(PyObject* o) { return (float)PyFloat_AsDouble(o); }

static int ready(int which, Py_ssize_t got, Py_ssize_t want) {
  if (entry[which] == NULL) {
    PyErr_SetString(PyExc_RuntimeError, "entry point is not bound");
  } else if (got != want) {
    PyErr_Format(PyExc_TypeError, "%zd arguments, expected %zd", got, want);
  } else {
    return 1;
  }
  return 0;
}

/* The converted arguments are locals, so that a failed conversion is seen before the call and the call
 * holds no Python object: other threads run during it (a launch blocks while its queue is full). */
#define CALL(type, ...)                                    \
  do {                                                     \
    int code;                                              \
    if (PyErr_Occurred()) return NULL;                     \
    Py_BEGIN_ALLOW_THREADS;                                \
    code = ((type)entry[which])(__VA_ARGS__);              \
    Py_END_ALLOW_THREADS;                                  \
    return PyLong_FromLong(code);                          \
  } while (0)

static PyObject* add_rms_norm_quant(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  enum { which = ADD_RMS_NORM_QUANT };
  (void)self;
  if (!ready(which, n, 17)) return NULL;
  const void* x = ptr(a[0]);
  const int64_t ldx = i64(a[1]);
  const void* res = ptr(a[2]);
  const int64_t ldr = i64(a[3]);
  const void* w = ptr(a[4]);
  const float eps = real(a[5]);
  void* ro = ptr(a[6]);
  const int64_t ldro = i64(a[7]);
  const int dtype = num(a[8]);
  void* q = ptr(a[9]);
  const int64_t ldq = i64(a[10]);
  const int qt = num(a[11]);
  float* scale = (float*)ptr(a[12]);
  const int rows = num(a[13]), width = num(a[14]);
  const unsigned f = flags(a[15]);
  void* stream = ptr(a[16]);
  typedef int (*fn)(const void*, int64_t, const void*, int64_t, const void*, float, void*, int64_t, int, void*, int64_t,
                    int, float*, int, int, unsigned, void*);
  CALL(fn, x, ldx, res, ldr, w, eps, ro, ldro, dtype, q, ldq, qt, scale, rows, width, f, stream);
}

static PyObject* rope_kv4_append(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  enum { which = ROPE_KV4_APPEND };
  (void)self;
  if (!ready(which, n, 31)) return NULL;
  const void* qkv = ptr(a[0]);
  const int64_t ldqkv = i64(a[1]);
  const int dtype = num(a[2]), tokens = num(a[3]), qh = num(a[4]), kvh = num(a[5]), d = num(a[6]);
  const void *qn = ptr(a[7]), *kn = ptr(a[8]);
  const float eps = real(a[9]);
  const float *c = (const float*)ptr(a[10]), *s = (const float*)ptr(a[11]);
  const int64_t len = i64(a[12]);
  const int64_t* pos = (const int64_t*)ptr(a[13]);
  const int64_t ldpos = i64(a[14]);
  const int axes = num(a[15]);
  /* sections: a tuple of up to four counts, or None */
  int sections[4] = {0, 0, 0, 0};
  const int* sec = NULL;
  if (a[16] != Py_None) {
    if (!PyTuple_Check(a[16]) || PyTuple_GET_SIZE(a[16]) > 4) {
      PyErr_SetString(PyExc_TypeError, "sections must be a tuple of at most four");
      return NULL;
    }
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(a[16]); ++i) sections[i] = num(PyTuple_GET_ITEM(a[16], i));
    sec = sections;
  }
  const int inter = num(a[17]);
  const int64_t* slots = (const int64_t*)ptr(a[18]);
  void* q = ptr(a[19]);
  const int64_t ldq = i64(a[20]);
  uint8_t* kc = (uint8_t*)ptr(a[21]);
  void* kp = ptr(a[22]);
  uint8_t* vc = (uint8_t*)ptr(a[23]);
  void* vp = ptr(a[24]);
  const int64_t pages = i64(a[25]);
  const int page = num(a[26]);
  void *kv = ptr(a[27]), *vv = ptr(a[28]);
  const unsigned f = flags(a[29]);
  void* stream = ptr(a[30]);
  typedef int (*fn)(const void*, int64_t, int, int, int, int, int, const void*, const void*, float, const float*,
                    const float*, int64_t, const int64_t*, int64_t, int, const int*, int, const int64_t*, void*,
                    int64_t, uint8_t*, void*, uint8_t*, void*, int64_t, int, void*, void*, unsigned, void*);
  CALL(fn, qkv, ldqkv, dtype, tokens, qh, kvh, d, qn, kn, eps, c, s, len, pos, ldpos, axes, sec, inter, slots, q, ldq,
       kc, kp, vc, vp, pages, page, kv, vv, f, stream);
}

static PyObject* kv4_attention(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  enum { which = KV4_ATTENTION };
  (void)self;
  if (!ready(which, n, 28)) return NULL;
  const void* q = ptr(a[0]);
  const int64_t ts = i64(a[1]), hs = i64(a[2]);
  const int dtype = num(a[3]);
  const uint8_t* kc = (const uint8_t*)ptr(a[4]);
  const void* kp = ptr(a[5]);
  const uint8_t* vc = (const uint8_t*)ptr(a[6]);
  const void* vp = ptr(a[7]);
  const int64_t pages = i64(a[8]);
  const int page = num(a[9]);
  const int32_t* table = (const int32_t*)ptr(a[10]);
  const int64_t ldt = i64(a[11]);
  const int cols = num(a[12]);
  const int32_t *lengths = (const int32_t*)ptr(a[13]), *starts = (const int32_t*)ptr(a[14]);
  const int total = num(a[15]), max_q = num(a[16]), batch = num(a[17]), qh = num(a[18]), kvh = num(a[19]),
            d = num(a[20]);
  const float scale = real(a[21]);
  const int causal = num(a[22]);
  void* out = ptr(a[23]);
  const int64_t ots = i64(a[24]);
  void* work = ptr(a[25]);
  const unsigned f = flags(a[26]);
  void* stream = ptr(a[27]);
  typedef int (*fn)(const void*, int64_t, int64_t, int, const uint8_t*, const void*, const uint8_t*, const void*,
                    int64_t, int, const int32_t*, int64_t, int, const int32_t*, const int32_t*, int, int, int, int, int,
                    int, float, int, void*, int64_t, void*, unsigned, void*);
  CALL(fn, q, ts, hs, dtype, kc, kp, vc, vp, pages, page, table, ldt, cols, lengths, starts, total, max_q, batch, qh,
       kvh, d, scale, causal, out, ots, work, f, stream);
}

/* bind(addresses): the three functions, in the order of the table below. */
static PyObject* bind(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  (void)self;
  if (n != ENTRIES) {
    PyErr_Format(PyExc_TypeError, "%zd addresses, expected %d", n, ENTRIES);
    return NULL;
  }
  for (int i = 0; i < ENTRIES; ++i) {
    void* p = ptr(a[i]);
    if (PyErr_Occurred()) return NULL;
    entry[i] = p;
  }
  Py_RETURN_NONE;
}

static PyMethodDef methods[] = {
    {"qtts_add_rms_norm_quant", (PyCFunction)(void (*)(void))add_rms_norm_quant, METH_FASTCALL, NULL},
    {"qtts_rope_kv4_append", (PyCFunction)(void (*)(void))rope_kv4_append, METH_FASTCALL, NULL},
    {"qtts_kv4_attention", (PyCFunction)(void (*)(void))kv4_attention, METH_FASTCALL, NULL},
    {"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, NULL},
    {NULL, NULL, 0, NULL}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_qtts_fastcall", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__qtts_fastcall(void) { return PyModule_Create(&module); }
