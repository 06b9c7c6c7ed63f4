/* The calls of the paged key-value cache (fbgemm_b200/paged.py) as a CPython extension over the C ABI
 * (include/fbgemm_b200/embedding_c_api.h).  Shapes, strides, types and devices are looked at here, at a tenth of a microsecond a
 * question; the same in Python took 4 us of the 13 that a call took. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <math.h>

#include "fbgemm_b200/embedding_c_api.h"

static PyObject* s_data_ptr;

/* Addresses of tensors whose strides the caller has looked at. */
static int pointers(PyObject* const* args, int first, int n, void** p) {
  for (int i = 0; i < n; ++i) {
    p[i] = NULL;
    if (args[first + i] != Py_None) {
      PyObject* a = PyObject_CallMethodNoArgs(args[first + i], s_data_ptr);
      if (!a) {
        return -1;
      }
      p[i] = PyLong_AsVoidPtr(a);
      Py_DECREF(a);
      if (p[i] == NULL && PyErr_Occurred()) {
        return -1;
      }
    }
  }
  return 0;
}

/* Contexts, caches and streams: their addresses as numbers; None = null. */
static int handles(PyObject* const* args, int first, int n, void** p) {
  for (int i = 0; i < n; ++i) {
    PyObject* x = args[first + i];
    p[i] = x == Py_None ? NULL : PyLong_AsVoidPtr(x);
    if (p[i] == NULL && PyErr_Occurred()) {
      return -1;
    }
  }
  return 0;
}

static int integers(PyObject* const* args, int first, int n, int64_t* v) {
  for (int i = 0; i < n; ++i) {
    v[i] = PyLong_AsLongLong(args[first + i]);
    if (v[i] == -1 && PyErr_Occurred()) {
      return -1;
    }
  }
  return 0;
}

static int arity(Py_ssize_t got, Py_ssize_t want) {
  if (got != want) {
    PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", want, got);
    return -1;
  }
  return 0;
}

/* Runs CALL, which gives an int, without the interpreter's lock: a launch waits when the stream's queue is full. */
#define WITHOUT_LOCK(CALL)    \
  int rc;                     \
  Py_BEGIN_ALLOW_THREADS      \
  rc = (CALL);                \
  Py_END_ALLOW_THREADS        \
  return PyLong_FromLong(rc)

static PyObject *s_shape, *s_stride, *s_dtype, *s_get_device;
static PyObject *t_int32, *t_int64, *t_float32, *t_float16, *t_bfloat16; /* torch's types; looked up at the first call */

static int torch_types(void) {
  if (t_bfloat16) {
    return 0;
  }
  PyObject* torch = PyImport_ImportModule("torch");
  if (!torch) {
    return -1;
  }
  t_int32 = PyObject_GetAttrString(torch, "int32");
  t_int64 = PyObject_GetAttrString(torch, "int64");
  t_float32 = PyObject_GetAttrString(torch, "float32");
  t_float16 = PyObject_GetAttrString(torch, "float16");
  t_bfloat16 = PyObject_GetAttrString(torch, "bfloat16");
  Py_DECREF(torch);
  return t_int32 && t_int64 && t_float32 && t_float16 && t_bfloat16 ? 0 : -1;
}

typedef struct {
  void* p;
  PyObject* dtype; /* (torch's types live as long as torch) */
  int64_t device, size[3], stride[3];
} Tensor;

/* What a tensor of `ndim` dimensions is; a null pointer for None if `optional`. */
static int look(PyObject* x, const char* name, int ndim, int optional, Tensor* t) {
  t->p = NULL;
  if (x == Py_None && optional) {
    return 0;
  }
  PyObject* shape = PyObject_GetAttr(x, s_shape);
  PyObject* stride = shape ? PyObject_CallMethodNoArgs(x, s_stride) : NULL;
  PyObject* device = stride ? PyObject_CallMethodNoArgs(x, s_get_device) : NULL;
  PyObject* address = device ? PyObject_CallMethodNoArgs(x, s_data_ptr) : NULL;
  t->dtype = address ? PyObject_GetAttr(x, s_dtype) : NULL;
  int bad = !t->dtype;
  if (!bad && (!PyTuple_Check(shape) || !PyTuple_Check(stride) || PyTuple_GET_SIZE(shape) != ndim ||
               PyTuple_GET_SIZE(stride) != ndim)) {
    PyErr_Format(PyExc_ValueError, "%s has %zd dimensions, %d expected", name,
                 PyTuple_Check(shape) ? PyTuple_GET_SIZE(shape) : (Py_ssize_t)-1, ndim);
    bad = 1;
  }
  for (int i = 0; !bad && i < ndim; ++i) {
    t->size[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, i));
    t->stride[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(stride, i));
  }
  if (!bad) {
    t->device = PyLong_AsLongLong(device);
    t->p = PyLong_AsVoidPtr(address);
    bad = PyErr_Occurred() != NULL;
  }
  Py_XDECREF(shape);
  Py_XDECREF(stride);
  Py_XDECREF(device);
  Py_XDECREF(address);
  Py_XDECREF(t->dtype);
  return bad ? -1 : 0;
}

static int value_error(const char* format, const char* name, long long a, long long b, long long c) {
  PyErr_Format(PyExc_ValueError, format, name, a, b, c);
  return -1;
}
static int type_error(const char* name, const char* wanted) {
  PyErr_Format(PyExc_TypeError, "%s is %s", name, wanted);
  return -1;
}

/* A contiguous vector of n (any number: -1) of a type. */
static int vector(PyObject* x, const char* name, PyObject* dtype, const char* type, int64_t n, Tensor* t) {
  if (look(x, name, 1, 0, t)) {
    return -1;
  }
  if (t->dtype != dtype) {
    return type_error(name, type);
  }
  if ((n >= 0 && t->size[0] != n) || (t->stride[0] != 1 && t->size[0] > 1)) {
    return value_error("%s is a contiguous vector of %lld", name, n < 0 ? t->size[0] : n, 0, 0);
  }
  return 0;
}

/* A block table of `batch` rows; *row: elements between them. */
static int block_table(PyObject* x, int64_t batch, Tensor* t, int64_t* row) {
  if (look(x, "block_tables", 2, 0, t)) {
    return -1;
  }
  if (t->dtype != t_int32) {
    return type_error("block_tables", "torch.int32");
  }
  if (t->size[0] != batch || (t->stride[1] != 1 && t->size[1] > 1)) {
    return value_error("%s is [%lld, pages of a request], its columns side by side", "block_tables", batch, 0, 0);
  }
  *row = batch > 1 ? t->stride[0] : (t->stride[0] > t->size[1] ? t->stride[0] : t->size[1]);
  return 0;
}

/* [tokens (any number: -1), heads (any number: -1), dim] of `dtype`; strides of single tokens and heads are 0. */
static int heads_of(PyObject* x, const char* name, PyObject* dtype, int64_t tokens, int64_t heads, int64_t dim, int optional,
                    Tensor* t) {
  if (look(x, name, 3, optional, t)) {
    return -1;
  }
  if (x == Py_None) {
    t->size[1] = t->stride[0] = t->stride[1] = 0;
    return 0;
  }
  if (t->dtype != dtype) {
    return type_error(name, dtype == t_bfloat16 ? "torch.bfloat16" : "torch.float16");
  }
  if ((tokens >= 0 && t->size[0] != tokens) || (heads >= 0 && t->size[1] != heads) || t->size[2] != dim || t->stride[2] != 1) {
    return value_error("%s is [%lld, %lld, %lld], a head's values side by side", name, tokens < 0 ? t->size[0] : tokens,
                       heads < 0 ? t->size[1] : heads, dim);
  }
  if (t->size[0] <= 1) {
    t->stride[0] = 0;
  }
  if (t->size[1] <= 1) {
    t->stride[1] = 0;
  }
  return 0;
}

/* Sizes that the library takes as 32-bit numbers. */
static int small(const char* name, int64_t n) {
  return n < 0 || n > INT32_MAX ? value_error("%s is %lld: out of range", name, n, 0, 0) : 0;
}

static int same_shape(PyObject* x, const char* name, const Tensor* like, Tensor* t) {
  if (look(x, name, 3, 0, t)) {
    return -1;
  }
  if (t->dtype != like->dtype || t->size[0] != like->size[0] || t->size[1] != like->size[1] || t->size[2] != like->size[2] ||
      (t->size[0] > 1 && t->stride[0] != t->size[1] * t->size[2]) || (t->size[1] > 1 && t->stride[1] != t->size[2]) ||
      (t->size[2] > 1 && t->stride[2] != 1)) {
    return value_error("%s is a contiguous tensor of q's shape and type", name, 0, 0, 0);
  }
  return 0;
}

static int on_device(const Tensor* t, const char* name, int64_t device) {
  if (t->p && t->device != device) {
    return value_error("%s does not lie on the device of the other tensors", name, 0, 0, 0);
  }
  return 0;
}

/* The type of activations beside a cache, -1 if it cannot be. */
static int activation_type(const fbgemm_b200_paged_cache* c, const Tensor* t, const char* name) {
  const int dtype = t->dtype == t_float16    ? FBGEMM_B200_OUT_F16
                    : t->dtype == t_bfloat16 ? FBGEMM_B200_OUT_BF16
                                             : -1;
  if (dtype < 0 || (c->in_dtype == FBGEMM_B200_IN_F16 && dtype != FBGEMM_B200_OUT_F16) ||
      (c->in_dtype == FBGEMM_B200_IN_BF16 && dtype != FBGEMM_B200_OUT_BF16)) {
    return type_error(name, c->in_dtype == FBGEMM_B200_IN_F16      ? "torch.float16, as the cache"
                            : c->in_dtype == FBGEMM_B200_IN_BF16 ? "torch.bfloat16, as the cache"
                                                                 : "torch.float16 or torch.bfloat16");
  }
  return dtype;
}

static int on_cuda(int64_t device) {
  if (device < 0) {
    PyErr_SetString(PyExc_ValueError, "the tensors have to lie on a CUDA device");
    return -1;
  }
  return 0;
}

/* paged_slots(ctx, lengths, new_tokens, tables, free_pages, num_free, page_size, capacity, slots, rest, slot, stream):
 * `rest` is positions, requests, offsets, lengths and num_free behind one another */
static PyObject* paged_slots(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  (void)self;
  void *ctx, *out[2], *stream;
  int64_t size[2], slot, row;
  Tensor lengths, fresh, table, pages, num;
  if (torch_types() || arity(n, 12) || handles(args, 0, 1, &ctx) || vector(args[1], "lengths", t_int32, "torch.int32", -1, &lengths) ||
      vector(args[2], "new_tokens", t_int32, "torch.int32", lengths.size[0], &fresh) ||
      block_table(args[3], lengths.size[0], &table, &row) ||
      vector(args[4], "free_pages", t_int32, "torch.int32", -1, &pages) ||
      vector(args[5], "num_free", t_int32, "torch.int32", 1, &num) || integers(args, 6, 2, size) || pointers(args, 8, 2, out) ||
      integers(args, 10, 1, &slot) || small("slot", slot) || handles(args, 11, 1, &stream) || on_device(&fresh, "new_tokens", lengths.device) ||
      on_device(&table, "block_tables", lengths.device) || on_device(&pages, "free_pages", lengths.device) ||
      on_device(&num, "num_free", lengths.device) || on_cuda(lengths.device)) {
    return NULL;
  }
  const int64_t batch = lengths.size[0], capacity = size[1];
  if (small("batch", batch) || small("block_tables' width", table.size[1]) || small("free_pages' length", pages.size[0]) ||
      small("page_size", size[0]) || small("capacity", capacity)) {
    return NULL;
  }
  int32_t* rest = out[1];
  WITHOUT_LOCK(fbgemm_b200_paged_slots(ctx, (int32_t)batch, lengths.p, fresh.p, table.p, (int32_t)table.size[1], row, pages.p,
                                       (int32_t)pages.size[0], num.p, (int32_t)size[0], (int32_t)capacity, out[0], rest,
                                       rest + capacity, rest + 2 * capacity, rest + 2 * capacity + batch + 1,
                                       rest + 2 * capacity + 2 * batch + 1, (int)slot, stream));
}

/* rotary_append(ctx, cache, device, q, k, v, q_out, slots, positions, cos_sin, interleaved, ends, slot, stream): `ends` the
 * section ends of several axes, or None */
static PyObject* rotary_append(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  (void)self;
  void *h[2], *stream;
  int64_t device, interleaved, slot;
  Tensor q, k, v, q_out, slots, positions, angles;
  if (torch_types() || arity(n, 14) || handles(args, 0, 2, h) || integers(args, 2, 1, &device) || look(args[4], "k", 3, 0, &k)) {
    return NULL;
  }
  const fbgemm_b200_paged_cache* c = h[1];
  const int dtype = activation_type(c, &k, "k");
  if (dtype < 0 || heads_of(args[4], "k", k.dtype, -1, c->kv_heads, c->head_dim, 0, &k) ||
      heads_of(args[5], "v", k.dtype, k.size[0], c->kv_heads, c->head_dim, 0, &v) ||
      heads_of(args[3], "q", k.dtype, k.size[0], -1, c->head_dim, 1, &q) ||
      vector(args[7], "slots", t_int64, "torch.int64", k.size[0], &slots) || integers(args, 10, 1, &interleaved) ||
      integers(args, 12, 1, &slot) || small("slot", slot) || handles(args, 13, 1, &stream)) {
    return NULL;
  }
  q_out.p = NULL;
  if (args[3] != Py_None && same_shape(args[6], "q_out", &q, &q_out)) {
    return NULL;
  }
  fbgemm_b200_rotary r = {0};
  int64_t positions_stride = 0;
  positions.p = angles.p = NULL;
  if (args[9] != Py_None) {
    if (look(args[9], "cos_sin", 2, 0, &angles)) {
      return NULL;
    }
    if (angles.dtype != t_float32) {
      type_error("cos_sin", "torch.float32");
      return NULL;
    }
    if (angles.stride[1] != 1 || (angles.size[0] > 1 && angles.stride[0] != angles.size[1])) {
      value_error("%s is [max_pos, rot_dim], contiguous", "cos_sin", 0, 0, 0);
      return NULL;
    }
    if (small("rot_dim", angles.size[1])) {
      return NULL;
    }
    r.cos_sin = angles.p;
    r.max_pos = angles.size[0];
    r.rot_dim = (int32_t)angles.size[1];
    r.interleaved = (int32_t)interleaved;
    if (args[11] == Py_None) {
      if (vector(args[8], "positions", t_int32, "torch.int32", k.size[0], &positions)) {
        return NULL;
      }
      r.axes = 1;
      r.section_end[0] = r.rot_dim / 2;
    } else {
      const Py_ssize_t axes = PyTuple_Check(args[11]) ? PyTuple_GET_SIZE(args[11]) : 0;
      if (axes < 1 || axes > 4) {
        value_error("%s are the pairs of 1 to 4 axes", "sections", 0, 0, 0);
        return NULL;
      }
      for (Py_ssize_t i = 0; i < axes; ++i) {
        const int64_t end = PyLong_AsLongLong(PyTuple_GET_ITEM(args[11], i));
        if ((end == -1 && PyErr_Occurred()) || small("the sum of sections", end)) {
          return NULL;
        }
        r.section_end[i] = (int32_t)end;
      }
      r.axes = (int32_t)axes;
      if (PyErr_Occurred() || look(args[8], "positions", 2, 0, &positions)) {
        return NULL;
      }
      if (positions.dtype != t_int32) {
        type_error("positions", "torch.int32");
        return NULL;
      }
      if (positions.size[0] != axes || positions.size[1] != k.size[0] || (positions.stride[1] != 1 && k.size[0] > 1)) {
        value_error("%s with sections is [%lld, %lld]", "positions", axes, k.size[0], 0);
        return NULL;
      }
      positions_stride = positions.stride[0];
    }
  }
  if (small("heads", q.size[1]) || on_device(&q, "q", device) || on_device(&k, "k", device) || on_device(&v, "v", device) ||
      on_device(&slots, "slots", device) || on_device(&positions, "positions", device) ||
      on_device(&angles, "cos_sin", device) || on_device(&q_out, "q_out", device) || on_cuda(device)) {
    return NULL;
  }
  WITHOUT_LOCK(fbgemm_b200_rotary_append(h[0], c, k.size[0], (int32_t)q.size[1], dtype, q.p, q.stride[0], q.stride[1], k.p,
                                         k.stride[0], k.stride[1], v.p, v.stride[0], v.stride[1], q_out.p, slots.p,
                                         positions.p, positions_stride, angles.p ? &r : NULL, (int)slot, stream));
}

/* paged_attention(ctx, cache, device, q, tables, lengths, scale or None, window, out, lse, workspace, workspace_bytes, slot,
 * stream) */
static PyObject* paged_attention(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  (void)self;
  void *h[2], *more[2], *stream;
  int64_t device, window, bytes, slot, row;
  Tensor q, table, lengths, out;
  if (torch_types() || arity(n, 14) || handles(args, 0, 2, h) || integers(args, 2, 1, &device) || look(args[3], "q", 3, 0, &q)) {
    return NULL;
  }
  const fbgemm_b200_paged_cache* c = h[1];
  const int dtype = activation_type(c, &q, "q");
  if (dtype < 0 || heads_of(args[3], "q", q.dtype, -1, -1, c->head_dim, 0, &q) ||
      block_table(args[4], q.size[0], &table, &row) ||
      vector(args[5], "lengths", t_int32, "torch.int32", q.size[0], &lengths) || integers(args, 7, 1, &window) ||
      same_shape(args[8], "out", &q, &out) || pointers(args, 9, 2, more) || integers(args, 11, 1, &bytes) ||
      integers(args, 12, 1, &slot) || small("slot", slot) || handles(args, 13, 1, &stream) || on_device(&q, "q", device) ||
      on_device(&table, "block_tables", device) || on_device(&lengths, "lengths", device) || on_device(&out, "out", device) ||
      on_cuda(device)) {
    return NULL;
  }
  double scale = 1.0;
  if (args[6] == Py_None) {
    scale = 1.0 / sqrt((double)c->head_dim);
  } else {
    scale = PyFloat_AsDouble(args[6]);
    if (scale == -1.0 && PyErr_Occurred()) {
      return NULL;
    }
  }
  if (small("window", window) || small("batch", q.size[0]) || small("heads", q.size[1]) ||
      small("block_tables' width", table.size[1])) {
    return NULL;
  }
  WITHOUT_LOCK(fbgemm_b200_paged_attention(h[0], c, (int32_t)q.size[0], (int32_t)q.size[1], dtype, q.p, q.stride[0], q.stride[1],
                                           table.p, (int32_t)table.size[1], row, lengths.p, (float)scale, (int32_t)window,
                                           out.p, more[0], more[1], bytes, (int)slot, stream));
}

static PyMethodDef methods[] = {
    {"paged_slots", (PyCFunction)(void (*)(void))paged_slots, METH_FASTCALL, "fbgemm_b200_paged_slots"},
    {"rotary_append", (PyCFunction)(void (*)(void))rotary_append, METH_FASTCALL, "fbgemm_b200_rotary_append"},
    {"paged_attention", (PyCFunction)(void (*)(void))paged_attention, METH_FASTCALL, "fbgemm_b200_paged_attention"},
    {NULL, NULL, 0, NULL}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged_calls", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__paged_calls(void) {
  s_data_ptr = PyUnicode_InternFromString("data_ptr");
  s_shape = PyUnicode_InternFromString("shape");
  s_stride = PyUnicode_InternFromString("stride");
  s_dtype = PyUnicode_InternFromString("dtype");
  s_get_device = PyUnicode_InternFromString("get_device");
  return s_data_ptr && s_shape && s_stride && s_dtype && s_get_device ? PyModule_Create(&module) : NULL;
}
