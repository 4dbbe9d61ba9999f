/* calls.c -- the call path of the small serving-step operators from Python: one
 * pass over a call's tensors and one typed call of the C ABI.
 *
 * ctypes and five method calls a tensor from bytecode cost 5-9 us where the
 * launch behind them costs 3 (a step makes several such calls for every layer).
 * A tensor is read through the C exchange table that torch.Tensor offers
 * (__dlpack_c_exchange_api__), in one call without a Python object made; what
 * that does not take (a tensor that is only like one, a conjugate), and every
 * tensor of a torch that has no such table, through its methods. This module
 * computes nothing and keeps nothing: what is checked and what is passed stands
 * in attention.py.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/dlpack.h>

#include "zealot_attn.h"

static PyObject *s_dtype, *s_get_device, *s_data_ptr, *s_shape, *s_stride;

/* torch, from the first call that has a tensor on */
static struct {
  int found;
  const DLPackExchangeAPI* exchange; /* NULL where this torch has none that is known here: tensors through their methods */
  PyObject* tensor;
  struct {
    PyObject* dtype;
    uint8_t code, bits;
  } kinds[5];
} torch;

static int find_torch(void) {
  static const struct {
    const char* name;
    uint8_t code, bits;
  } kinds[5] = {{"int32", kDLInt, 32}, {"int64", kDLInt, 64}, {"float32", kDLFloat, 32}, {"float64", kDLFloat, 64}, {"bfloat16", kDLBfloat, 16}};
  PyObject *m = PyImport_ImportModule("torch"), *tensor = m ? PyObject_GetAttrString(m, "Tensor") : NULL;
  int ok = tensor != NULL;
  for (int i = 0; i < 5 && ok; i++) {
    torch.kinds[i].code = kinds[i].code;
    torch.kinds[i].bits = kinds[i].bits;
    ok = (torch.kinds[i].dtype = PyObject_GetAttrString(m, kinds[i].name)) != NULL;
  }
  if (ok) {
    PyObject* table = PyObject_GetAttrString(tensor, "__dlpack_c_exchange_api__");
    const DLPackExchangeAPI* exchange = table ? PyCapsule_GetPointer(table, "dlpack_exchange_api") : NULL;
    PyErr_Clear();
    torch.exchange = exchange && exchange->header.version.major == DLPACK_MAJOR_VERSION ? exchange : NULL;
    torch.tensor = Py_NewRef(tensor);
    torch.found = 1; /* last: it says that the rest is there */
    Py_XDECREF(table);
  }
  Py_XDECREF(tensor);
  Py_XDECREF(m);
  return ok;
}

static PyObject* method(PyObject* o, PyObject* name) {
  PyObject* args[1] = {o};
  return PyObject_VectorcallMethod(name, args, 1 | PY_VECTORCALL_ARGUMENTS_OFFSET, NULL);
}

#define MAX_DIMS 8
/* What the checks ask of a tensor. */
typedef struct {
  int is_dtype, dims;
  long long device; /* -1: the host */
  int64_t shape[MAX_DIMS], stride[MAX_DIMS];
  unsigned long long address;
} View;

/* 0: filled, with is_dtype whether `dtype` is the tensor's; -1: exception. */
static int look_slowly(PyObject* t, PyObject* dtype, View* v) {
  PyObject *kind = PyObject_GetAttr(t, s_dtype), *shape = NULL, *stride = NULL, *device = NULL, *address = NULL;
  int ok = kind && (shape = PyObject_GetAttr(t, s_shape)) && (stride = method(t, s_stride)) &&
           (device = method(t, s_get_device)) && (address = method(t, s_data_ptr));
  if (ok && !(PyTuple_Check(shape) && PyTuple_Check(stride) && PyTuple_GET_SIZE(shape) <= MAX_DIMS &&
              PyTuple_GET_SIZE(shape) == PyTuple_GET_SIZE(stride))) {
    PyErr_Format(PyExc_TypeError, "no tensor of up to %d dimensions", MAX_DIMS);
    ok = 0;
  }
  if (ok) {
    v->is_dtype = kind == dtype;
    v->dims = (int)PyTuple_GET_SIZE(shape);
    for (int i = 0; i < v->dims; i++) {
      v->shape[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, i));
      v->stride[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(stride, i));
    }
    v->device = PyLong_AsLongLong(device);
    v->address = PyLong_AsUnsignedLongLong(address);
    ok = !PyErr_Occurred();
  }
  Py_XDECREF(kind);
  Py_XDECREF(shape);
  Py_XDECREF(stride);
  Py_XDECREF(device);
  Py_XDECREF(address);
  return ok ? 0 : -1;
}

static int look(PyObject* t, PyObject* dtype, View* v) {
  if (!torch.found && !find_torch()) return -1;
  int kind = 0;
  while (kind < 5 && torch.kinds[kind].dtype != dtype) kind++;
  DLTensor d;
  if (!torch.exchange || kind == 5 || !PyObject_TypeCheck(t, (PyTypeObject*)torch.tensor)) return look_slowly(t, dtype, v);
  if (torch.exchange->dltensor_from_py_object_no_sync(t, &d) != 0) {
    PyErr_Clear();
    return look_slowly(t, dtype, v);
  }
  if (d.ndim > MAX_DIMS || !d.strides || (d.device.device_type != kDLCPU && d.device.device_type != kDLCUDA))
    return look_slowly(t, dtype, v);
  v->is_dtype = d.dtype.code == torch.kinds[kind].code && d.dtype.bits == torch.kinds[kind].bits && d.dtype.lanes == 1;
  v->dims = d.ndim;
  v->device = d.device.device_type == kDLCUDA ? d.device.device_id : -1;
  for (int i = 0; i < d.ndim; i++) {
    v->shape[i] = d.shape[i];
    v->stride[i] = d.strides[i];
  }
  v->address = (unsigned long long)((uintptr_t)d.data + d.byte_offset);
  return 0;
}

/* Whether the view is of n elements that lie in order. */
static int in_order(const View* v, long long n) {
  unsigned long long have = 1;
  int whole = 1;
  for (int i = v->dims - 1; i >= 0; i--) {
    whole &= v->shape[i] == 1 || (unsigned long long)v->stride[i] == have;
    have *= (unsigned long long)v->shape[i];
  }
  return n >= 0 && have == (unsigned long long)n && (whole || n == 0);
}

/* What a tensor is asked to have: a number of elements, or a shape (a tuple). 1: it has, with the
 * number in *n; 0: not; -1: exception. */
static int has(const View* v, PyObject* want, long long* n) {
  if (!PyTuple_Check(want)) {
    *n = PyLong_AsLongLong(want);
    return *n == -1 && PyErr_Occurred() ? -1 : 1;
  }
  int same = PyTuple_GET_SIZE(want) == v->dims;
  *n = 1;
  for (int i = 0; i < v->dims && same; i++) {
    const long long x = PyLong_AsLongLong(PyTuple_GET_ITEM(want, i));
    if (x == -1 && PyErr_Occurred()) return -1;
    same = x == v->shape[i];
    *n *= v->shape[i];
  }
  return same;
}

/* addresses(device, tensor, dtype, elements or shape, tensor, dtype, elements or shape, ...) -> the
 * tensors' addresses as a tuple (0 for None), or the number of the first that does not fit. */
static PyObject* addresses(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs < 1 || nargs % 3 != 1) {
    PyErr_SetString(PyExc_TypeError, "addresses(device, tensor, dtype, elements or shape, ...)");
    return NULL;
  }
  const long long device = PyLong_AsLongLong(args[0]);
  if (device == -1 && PyErr_Occurred()) return NULL;
  const Py_ssize_t count = nargs / 3;
  PyObject* out = PyTuple_New(count);
  if (!out) return NULL;
  for (Py_ssize_t i = 0; i < count; i++) {
    unsigned long long address = 0;
    if (args[1 + 3 * i] != Py_None) {
      View v;
      long long n = 0;
      const int fits = look(args[1 + 3 * i], args[2 + 3 * i], &v) ? -1 : has(&v, args[3 + 3 * i], &n);
      if (fits <= 0 || !v.is_dtype || v.device != device || !in_order(&v, n)) {
        Py_DECREF(out);
        return fits < 0 ? NULL : PyLong_FromSsize_t(i);
      }
      address = n ? v.address : 0;
    }
    PyObject* a = PyLong_FromUnsignedLongLong(address);
    if (!a) {
      Py_DECREF(out);
      return NULL;
    }
    PyTuple_SET_ITEM(out, i, a);
  }
  return out;
}

/* head_rows(device, dtype, T, d, tensor, heads, tensor, heads, ...) -> (address, token stride, ...)
 * of tensors [T][heads][d] whose heads lie side by side (0, 0 for None), or the number of the first that is none. */
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
    View v = {0};
    const int none = args[4 + 2 * i] == Py_None;
    const long long heads = PyLong_AsLongLong(args[5 + 2 * i]);
    const int bad = (heads == -1 && PyErr_Occurred()) || (!none && look(args[4 + 2 * i], args[1], &v));
    if (bad || (!none && (!v.is_dtype || v.device != device || v.dims != 3 || v.shape[0] != T || v.shape[1] != heads ||
        v.shape[2] != d || (v.stride[2] != 1 && d != 1) || (v.stride[1] != d && heads != 1)))) {
      Py_DECREF(out);
      return bad ? NULL : PyLong_FromSsize_t(i);
    }
    PyObject *a = PyLong_FromUnsignedLongLong(T && heads && d ? v.address : 0), *step = PyLong_FromLongLong(v.stride[0]);
    if (!a || !step) {
      Py_XDECREF(a);
      Py_XDECREF(step);
      Py_DECREF(out);
      return NULL;
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
     "addresses(device, tensor, dtype, elements or shape, ...): a tuple, or the number of the first tensor that does not fit"},
    {"head_rows", (PyCFunction)(void (*)(void))head_rows, METH_FASTCALL,
     "head_rows(device, dtype, T, d, tensor, heads, ...): a tuple, or the number of the first tensor that does not fit"},
    ENTRY(step_tables), ENTRY(qk_norm_rope), ENTRY(block_bounds), ENTRY(block_scores), ENTRY(select_blocks),
    ENTRY(paged_decode_selected), {NULL, NULL, 0, NULL}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "calls", "Call path of the serving-step operators.", -1, methods};

PyMODINIT_FUNC PyInit_calls(void) {
  s_dtype = PyUnicode_InternFromString("dtype");
  s_get_device = PyUnicode_InternFromString("get_device");
  s_data_ptr = PyUnicode_InternFromString("data_ptr");
  s_shape = PyUnicode_InternFromString("shape");
  s_stride = PyUnicode_InternFromString("stride");
  if (!s_dtype || !s_get_device || !s_data_ptr || !s_shape || !s_stride) return NULL;
  return PyModule_Create(&module);
}
