/* calls.c -- the call path of the small serving-step operators from Python: one
 * pass over a call's tensors and one typed call of the C ABI.
 *
 * ctypes and five method calls a tensor from bytecode cost 5-9 us where the
 * launch behind them costs 3 (a step makes several such calls for every layer);
 * this module takes them in 2-4. It computes nothing and keeps nothing: what is
 * checked and what is passed stands in attention.py.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "zealot_attn.h"

static PyObject *s_dtype, *s_numel, *s_get_device, *s_is_contiguous, *s_data_ptr, *s_shape, *s_stride;

static PyObject* method(PyObject* o, PyObject* name) {
  PyObject* args[1] = {o};
  return PyObject_VectorcallMethod(name, args, 1 | PY_VECTORCALL_ARGUMENTS_OFFSET, NULL);
}

/* o.name() as a whole number; -1 with an exception set on failure. */
static long long number(PyObject* o, PyObject* name) {
  PyObject* r = method(o, name);
  if (!r) return -1;
  const long long v = PyLong_AsLongLong(r);
  Py_DECREF(r);
  return v;
}

/* 1: a contiguous tensor of `dtype` with n elements on the device, 0: not, -1: exception. */
static int fits(PyObject* t, PyObject* dtype, long long n, long long device) {
  PyObject* d = PyObject_GetAttr(t, s_dtype);
  if (!d) return -1;
  Py_DECREF(d);
  if (d != dtype) return 0;
  const long long have = number(t, s_numel);
  if (have == -1 && PyErr_Occurred()) return -1;
  const long long on = number(t, s_get_device);
  if (on == -1 && PyErr_Occurred()) return -1;
  if (have != n || on != device) return 0;
  PyObject* c = method(t, s_is_contiguous);
  if (!c) return -1;
  const int whole = PyObject_IsTrue(c);
  Py_DECREF(c);
  return whole;
}

/* addresses(device, tensor, dtype, elements, tensor, dtype, elements, ...) -> the tensors'
 * addresses as a tuple (0 for None), or the number of the first that does not fit. */
static PyObject* addresses(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs < 1 || nargs % 3 != 1) {
    PyErr_SetString(PyExc_TypeError, "addresses(device, tensor, dtype, elements, ...)");
    return NULL;
  }
  const long long device = PyLong_AsLongLong(args[0]);
  if (device == -1 && PyErr_Occurred()) return NULL;
  const Py_ssize_t count = nargs / 3;
  PyObject* out = PyTuple_New(count);
  if (!out) return NULL;
  for (Py_ssize_t i = 0; i < count; i++) {
    PyObject *t = args[1 + 3 * i], *a;
    if (t == Py_None) {
      a = PyLong_FromLong(0);
    } else {
      const long long n = PyLong_AsLongLong(args[3 + 3 * i]);
      const int ok = n == -1 && PyErr_Occurred() ? -1 : fits(t, args[2 + 3 * i], n, device);
      if (ok != 1) {
        Py_DECREF(out);
        return ok == 0 ? PyLong_FromSsize_t(i) : NULL;
      }
      a = method(t, s_data_ptr);
    }
    if (!a) {
      Py_DECREF(out);
      return NULL;
    }
    PyTuple_SET_ITEM(out, i, a);
  }
  return out;
}

/* item i of a tuple of whole numbers */
static long long item(PyObject* t, Py_ssize_t i) { return PyLong_AsLongLong(PyTuple_GET_ITEM(t, i)); }

/* head_rows(device, dtype, T, d, tensor, heads, tensor, heads, ...) -> (address, token stride, ...)
 * of tensors [T][heads][d] whose heads lie side by side, or the number of the first that is none. */
static PyObject* head_rows(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs < 4 || nargs % 2) {
    PyErr_SetString(PyExc_TypeError, "head_rows(device, dtype, T, d, tensor, heads, ...)");
    return NULL;
  }
  const long long device = PyLong_AsLongLong(args[0]), T = PyLong_AsLongLong(args[2]), d = PyLong_AsLongLong(args[3]);
  if (PyErr_Occurred()) return NULL;
  const Py_ssize_t count = (nargs - 4) / 2;
  PyObject* out = PyTuple_New(2 * count);
  if (!out) return NULL;
  for (Py_ssize_t i = 0; i < count; i++) {
    PyObject *t = args[4 + 2 * i], *kind = NULL, *shape = NULL, *stride = NULL, *a = NULL, *step = NULL;
    const long long heads = PyLong_AsLongLong(args[5 + 2 * i]);
    int ok = !PyErr_Occurred() && (kind = PyObject_GetAttr(t, s_dtype)) && (shape = PyObject_GetAttr(t, s_shape)) &&
             (stride = method(t, s_stride));
    if (ok) {
      ok = kind == args[1] && PyTuple_Check(shape) && PyTuple_Check(stride) && PyTuple_GET_SIZE(shape) == 3 &&
           PyTuple_GET_SIZE(stride) == 3 && item(shape, 0) == T && item(shape, 1) == heads && item(shape, 2) == d &&
           (item(stride, 2) == 1 || d == 1) && (item(stride, 1) == d || heads == 1) && number(t, s_get_device) == device;
      if (ok && (a = method(t, s_data_ptr))) step = Py_NewRef(PyTuple_GET_ITEM(stride, 0));
    }
    Py_XDECREF(kind);
    Py_XDECREF(shape);
    Py_XDECREF(stride);
    if (!step) {
      Py_XDECREF(a);
      Py_DECREF(out);
      return PyErr_Occurred() ? NULL : PyLong_FromSsize_t(i);
    }
    PyTuple_SET_ITEM(out, 2 * i, a);
    PyTuple_SET_ITEM(out, 2 * i + 1, step);
  }
  return out;
}

/* A call's arguments in the order of the C function. */
typedef struct {
  PyObject* const* at;
} Args;
static void* P(Args* a) {
  PyObject* o = *a->at++;
  return o == Py_None ? NULL : PyLong_AsVoidPtr(o);
}
static long long L(Args* a) { return PyLong_AsLongLong(*a->at++); }
static int I(Args* a) {
  const long long v = L(a);
  if (v != (int)v && !PyErr_Occurred()) PyErr_SetString(PyExc_OverflowError, "an argument is past 32 bits");
  return (int)v;
}
static float F(Args* a) { return (float)PyFloat_AsDouble(*a->at++); }

#define CALL(name, count)                                                                         \
  static PyObject* call_##name(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {         \
    if (nargs != count) {                                                                         \
      PyErr_SetString(PyExc_TypeError, #name " takes " #count " arguments");                      \
      return NULL;                                                                                \
    }                                                                                             \
    Args a = {args};                                                                              \
    zl_status s;

#define RUN(expr)               \
    if (PyErr_Occurred()) return NULL; \
    Py_BEGIN_ALLOW_THREADS      \
    s = expr;                   \
    Py_END_ALLOW_THREADS        \
    return PyLong_FromLong(s);  \
  }

CALL(step_tables, 20)
  void* ctx = P(&a); int32_t* seq_blocks = P(&a); const int num_rows = I(&a); const int32_t *rows = P(&a), *ctx_lens = P(&a), *q_lens = P(&a), *fresh = P(&a);
  const int64_t num_new = L(&a); int32_t *tables = P(&a), *cu = P(&a), *lens = P(&a), *pos = P(&a); int64_t* slots = P(&a); int32_t* last = P(&a);
  const int n = I(&a); const int64_t tokens = L(&a); const int max_blocks = I(&a), bs = I(&a); const int64_t num_blocks = L(&a); void* stream = P(&a);
RUN(zl_step_tables(ctx, seq_blocks, num_rows, rows, ctx_lens, q_lens, fresh, num_new, tables, cu, lens, pos, slots, last, n, tokens, max_blocks, bs, num_blocks, stream))

CALL(qk_norm_rope, 28)
  void *ctx = P(&a), *q = P(&a), *k = P(&a), *v = P(&a); const int64_t qs = L(&a), ks = L(&a), vs = L(&a); void *qw = P(&a), *kw = P(&a);
  const float eps = F(&a); const int32_t* pos = P(&a); const double* freq = P(&a); const int rot = I(&a), inter = I(&a);
  void *qo = P(&a), *ko = P(&a), *vo = P(&a), *kp = P(&a), *vp = P(&a); const int64_t* slots = P(&a); const int bs = I(&a);
  const int64_t num_blocks = L(&a), tokens = L(&a); const int H = I(&a), Hkv = I(&a), d = I(&a), dtype = I(&a); void* stream = P(&a);
RUN(zl_qk_norm_rope(ctx, q, k, v, qs, ks, vs, qw, kw, eps, pos, freq, rot, inter, qo, ko, vo, kp, vp, slots, bs, num_blocks, tokens, H, Hkv, d, (zl_dtype)dtype, stream))

CALL(block_bounds, 14)
  void *ctx = P(&a), *kp = P(&a); const int32_t *tables = P(&a), *begin = P(&a), *lens = P(&a); void* bounds = P(&a);
  const int B = I(&a), Hkv = I(&a), d = I(&a), bs = I(&a), max_blocks = I(&a); const int64_t num_blocks = L(&a); const int dtype = I(&a); void* stream = P(&a);
RUN(zl_block_bounds(ctx, kp, tables, begin, lens, bounds, B, Hkv, d, bs, max_blocks, num_blocks, (zl_dtype)dtype, stream))

CALL(block_scores, 17)
  void *ctx = P(&a), *q = P(&a), *bounds = P(&a); const int32_t *tables = P(&a), *lens = P(&a); float* scores = P(&a);
  const int B = I(&a), H = I(&a), Hkv = I(&a), d = I(&a), bs = I(&a), max_blocks = I(&a); const int64_t num_blocks = L(&a);
  const float scale = F(&a); const int map = I(&a), dtype = I(&a); void* stream = P(&a);
RUN(zl_block_scores(ctx, q, bounds, tables, lens, scores, B, H, Hkv, d, bs, max_blocks, num_blocks, scale, (zl_gqa_map)map, (zl_dtype)dtype, stream))

CALL(select_blocks, 12)
  void* ctx = P(&a); const float* scores = P(&a); const int32_t* lens = P(&a); int32_t* selected = P(&a);
  const int B = I(&a), Hkv = I(&a), bs = I(&a), max_blocks = I(&a), top = I(&a), first = I(&a), last = I(&a); void* stream = P(&a);
RUN(zl_select_blocks(ctx, scores, lens, selected, B, Hkv, bs, max_blocks, top, first, last, stream))

CALL(paged_decode_selected, 20)
  void *ctx = P(&a), *q = P(&a), *kp = P(&a), *vp = P(&a); const int32_t *tables = P(&a), *lens = P(&a), *selected = P(&a); void* o = P(&a);
  const int B = I(&a), H = I(&a), Hkv = I(&a), d = I(&a), bs = I(&a), max_blocks = I(&a); const int64_t num_blocks = L(&a); const int top = I(&a);
  const float scale = F(&a); const int map = I(&a), dtype = I(&a); void* stream = P(&a);
RUN(zl_paged_decode_selected(ctx, q, kp, vp, tables, lens, selected, o, B, H, Hkv, d, bs, max_blocks, num_blocks, top, scale, (zl_gqa_map)map, (zl_dtype)dtype, stream))

#define ENTRY(name) {#name, (PyCFunction)(void (*)(void))call_##name, METH_FASTCALL, "zl_" #name " of the C ABI, argument by argument"}
static PyMethodDef methods[] = {
    {"addresses", (PyCFunction)(void (*)(void))addresses, METH_FASTCALL,
     "addresses(device, tensor, dtype, elements, ...): a tuple, or the number of the first tensor that does not fit"},
    {"head_rows", (PyCFunction)(void (*)(void))head_rows, METH_FASTCALL,
     "head_rows(device, dtype, T, d, tensor, heads, ...): a tuple, or the number of the first tensor that does not fit"},
    ENTRY(step_tables), ENTRY(qk_norm_rope), ENTRY(block_bounds), ENTRY(block_scores), ENTRY(select_blocks),
    ENTRY(paged_decode_selected), {NULL, NULL, 0, NULL}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "calls", "Call path of the serving-step operators.", -1, methods};

PyMODINIT_FUNC PyInit_calls(void) {
  s_dtype = PyUnicode_InternFromString("dtype");
  s_numel = PyUnicode_InternFromString("numel");
  s_get_device = PyUnicode_InternFromString("get_device");
  s_is_contiguous = PyUnicode_InternFromString("is_contiguous");
  s_data_ptr = PyUnicode_InternFromString("data_ptr");
  s_shape = PyUnicode_InternFromString("shape");
  s_stride = PyUnicode_InternFromString("stride");
  if (!s_dtype || !s_numel || !s_get_device || !s_is_contiguous || !s_data_ptr || !s_shape || !s_stride) return NULL;
  return PyModule_Create(&module);
}
