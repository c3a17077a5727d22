/*
 * The 4-bit operators' argument checks and launches for Python (module _kv4_native), through CPython's API.
 *
 * One call of these operators reads about thirty tensor attributes, and their kernels take a few microseconds: in
 * Python the reading, checking and the foreign call cost several times that.  Tensors are
 * taken through their public attributes (shape, stride, dtype, ...), so nothing here depends on torch's headers;
 * outputs come from torch.empty, scratch and the status word from the Python module, and the entry points are
 * the C ABI of include/b200kv_kv4.h, whose addresses setup() is given.
 *
 * Host time per call, us, this / the same checks in Python with the launch through ctypes: decode 6.8 / 13.3, append
 * 3.8 / 6.8, read-back 5.5 / 8.4; a launch takes 2.9 of them and a new output tensor 1.5.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>

#include "b200kv_kv4.h"

enum { kPageTok = 16, kDim = 128 };

/* What setup() hands over; owned references, for the life of the process. */
static struct {
  PyObject *f16, *i32, *i64, *u8;                 /* torch dtypes (one object each) */
  PyObject *empty, *empty_like;                   /* torch.empty, torch.empty_like */
  PyObject *current_device, *raw_stream;          /* torch's accessors */
  PyObject* status;                               /* kernels._status: device index -> status word */
  PyObject *status_ptr, *workspace, *on_device, *refuse_cpu, *check;   /* functions of the kernels module */
  __typeof__(b200kv_kv4_append)* append;
  __typeof__(b200kv_kv4_qk_norm_rope_append)* prologue;
  __typeof__(b200kv_kv4_gather)* gather;
  __typeof__(b200kv_kv4_paged_decode)* decode;
  __typeof__(b200kv_kv4_paged_prefill)* prefill;
  __typeof__(b200kv_stream_capture_id)* capture_id;
} st;

static PyObject *s_shape, *s_stride, *s_dtype, *s_get_device, *s_data_ptr, *s_contiguous, *s_device,
    *empty_names;

/* ---- tensors ------------------------------------------------------------------------------------- */

typedef struct {
  PyObject* t;         /* borrowed */
  PyObject* dtype;     /* compared by identity only */
  int nd;
  int64_t shape[3], stride[3];
  int64_t dev;
} Tensor;

static int64_t as_int(PyObject* o) { return PyLong_AsLongLong(o); }   /* -1 with an error set when it is none */

static int call_int(PyObject* t, PyObject* name, int64_t* out) {
  PyObject* r = PyObject_CallMethodNoArgs(t, name);
  if (r == NULL) return -1;
  *out = as_int(r);
  Py_DECREF(r);
  return *out == -1 && PyErr_Occurred() ? -1 : 0;
}
static int read_dims(PyObject* tuple, int64_t out[3], int* nd) {
  if (!PyTuple_Check(tuple)) {
    PyErr_SetString(PyExc_TypeError, "a tensor's shape and strides must be tuples");
    return -1;
  }
  *nd = (int)PyTuple_GET_SIZE(tuple);
  for (int i = 0; i < *nd && i < 3; ++i) {
    out[i] = as_int(PyTuple_GET_ITEM(tuple, i));
    if (out[i] == -1 && PyErr_Occurred()) return -1;
  }
  return 0;
}
/* Everything but the address.  Dimensions beyond the third are counted, not kept. */
static int read_tensor(PyObject* t, Tensor* x) {
  x->t = t;
  PyObject* o = PyObject_GetAttr(t, s_shape);
  if (o == NULL) return -1;
  int rc = read_dims(o, x->shape, &x->nd);
  Py_DECREF(o);
  if (rc != 0) return -1;
  if ((o = PyObject_CallMethodNoArgs(t, s_stride)) == NULL) return -1;
  int nd = 0;
  rc = read_dims(o, x->stride, &nd);
  Py_DECREF(o);
  if (rc != 0) return -1;
  if (nd != x->nd) {
    PyErr_SetString(PyExc_TypeError, "a tensor's shape and strides must agree");
    return -1;
  }
  if ((o = PyObject_GetAttr(t, s_dtype)) == NULL) return -1;
  x->dtype = o;
  Py_DECREF(o);        /* torch keeps its dtype objects */
  return call_int(t, s_get_device, &x->dev);
}
/* An address as an integer; addresses of pool tensors are below 2^63. */
static int address(PyObject* t, uintptr_t* out) {
  int64_t p = 0;
  if (call_int(t, s_data_ptr, &p) != 0) return -1;
  *out = (uintptr_t)p;
  return 0;
}
static int fail(const char* msg) {
  PyErr_SetString(PyExc_ValueError, msg);
  return -1;
}
static int off_device(const char* name, PyObject* t, int64_t dev) {
  PyObject* where = PyObject_GetAttr(t, s_device);
  if (where == NULL) return -1;
  PyErr_Format(PyExc_ValueError, "%s must be on the pool's device cuda:%lld (got %S)", name, (long long)dev, where);
  Py_DECREF(where);
  return -1;
}

/* ---- arguments of one kind -------------------------------------------------------------------------- */

typedef struct {
  int64_t dev, pages, stride, kv_heads;
  uintptr_t ptr;
} Pool;

static int read_pool(PyObject* t, Pool* p) {
  if (st.check == NULL) return fail("_kv4_native has not been set up");
  Tensor x;
  if (read_tensor(t, &x) != 0) return -1;
  if (x.dev < 0) {
    PyObject* r = PyObject_CallOneArg(st.refuse_cpu, t);   /* raises */
    Py_XDECREF(r);
    return r == NULL ? -1 : fail("KV4_Buffer must be on a CUDA device");
  }
  if (x.dtype != st.u8 || x.nd != 3 || x.shape[2] != B200KV_KV4_BLOCK_BYTES || x.shape[1] == 0 || (x.shape[1] & 1))
    return fail("KV4_Buffer must be uint8 [num_pages, 2*kv_heads, 1152]");
  if (x.stride[2] != 1 || x.stride[1] != B200KV_KV4_BLOCK_BYTES) return fail("KV4_Buffer must be contiguous inside a page");
  p->dev = x.dev;
  p->pages = x.shape[0];
  p->kv_heads = x.shape[1] / 2;
  p->stride = x.stride[0];
  const int64_t least = x.shape[1] * B200KV_KV4_BLOCK_BYTES;
  if (p->pages <= 1 && p->stride < least) p->stride = least;   /* the stride of a dimension of one may be anything */
  return address(t, &p->ptr);
}

/* slot_mapping: a new reference to a contiguous tensor in *keep */
static int read_slots(PyObject* t, int64_t dev, PyObject** keep, int64_t* n, uintptr_t* ptr) {
  Tensor x;
  if (read_tensor(t, &x) != 0) return -1;
  if (x.dtype != st.i32 || x.nd != 1) return fail("Select_Index must be a 1-D int32 tensor");
  if (x.dev != dev) return off_device("Select_Index", t, dev);
  *n = x.shape[0];
  if (x.stride[0] == 1 || x.shape[0] <= 1) {
    *keep = Py_NewRef(t);
  } else if ((*keep = PyObject_CallMethodNoArgs(t, s_contiguous)) == NULL) {
    return -1;
  }
  return address(*keep, ptr);
}

/* fp16 head rows [n or more, heads, 128], contiguous inside a token */
static int check_rows(const Tensor* x, const char* name, int64_t heads, int64_t n, int64_t dev, int64_t* stride, uintptr_t* ptr) {
  if (x->dtype != st.f16 || x->nd != 3 || x->shape[1] != heads || x->shape[2] != kDim || x->shape[0] < n) {
    PyErr_Format(PyExc_ValueError, "%s must be float16 [%lld or more, %lld, 128]", name, (long long)n, (long long)heads);
    return -1;
  }
  if (x->stride[2] != 1 || (x->stride[1] != kDim && heads > 1)) {
    PyErr_Format(PyExc_ValueError, "%s must be contiguous inside a token", name);
    return -1;
  }
  if (x->dev != dev) return off_device(name, x->t, dev);
  *stride = n > 1 ? x->stride[0] : heads * kDim;
  return address(x->t, ptr);
}
static int read_rows(PyObject* t, const char* name, int64_t heads, int64_t n, int64_t dev, int64_t* stride, uintptr_t* ptr,
                     int64_t* rows) {
  Tensor x;
  if (read_tensor(t, &x) != 0) return -1;
  if (rows != NULL) *rows = x.nd > 0 ? x.shape[0] : 0;
  return check_rows(&x, name, heads, n, dev, stride, ptr);
}

typedef struct {
  int64_t stride, rows, cols;
  int kind;
  uintptr_t ptr;
} Table;

static int read_table(PyObject* t, PyObject* kind, int64_t dev, Table* b) {
  if (PyUnicode_Check(kind) && PyUnicode_CompareWithASCIIString(kind, "block") == 0) b->kind = B200KV_TABLE_BLOCK;
  else if (PyUnicode_Check(kind) && PyUnicode_CompareWithASCIIString(kind, "token") == 0) b->kind = B200KV_TABLE_TOKEN;
  else return fail("the 4-bit operators take a 'token' or 'block' table");
  Tensor x;
  if (read_tensor(t, &x) != 0) return -1;
  if (x.dtype != st.i32 || x.nd != 2 || x.stride[1] != 1)
    return fail("the table must be a 2-D int32 tensor contiguous along its last dimension");
  if (x.dev != dev) return off_device("the table", t, dev);
  b->rows = x.shape[0];
  b->cols = x.shape[1];
  b->stride = x.shape[0] > 1 ? x.stride[0] : x.shape[1];
  if (b->rows > INT32_MAX) return fail("the table has too many rows");
  return address(t, &b->ptr);
}

/* a contiguous 1-D tensor of n int32 (or, with wide != NULL, int64) values */
static int check_ints(const Tensor* x, const char* name, int64_t n, int64_t dev, int* wide, uintptr_t* ptr) {
  const int is64 = wide != NULL && x->dtype == st.i64;
  if ((x->dtype != st.i32 && !is64) || x->nd != 1 || x->shape[0] != n || (x->stride[0] != 1 && n > 1)) {
    PyErr_Format(PyExc_ValueError, "%s must be a contiguous 1-D %s tensor of %lld values", name,
                 wide != NULL ? "int32 or int64" : "int32", (long long)n);
    return -1;
  }
  if (x->dev != dev) return off_device(name, x->t, dev);
  if (wide != NULL) *wide = is64;
  return address(x->t, ptr);
}
static int read_ints(PyObject* t, const char* name, int64_t n, int64_t dev, int* wide, uintptr_t* ptr) {
  Tensor x;
  return read_tensor(t, &x) != 0 ? -1 : check_ints(&x, name, n, dev, wide, ptr);
}

/* ---- launching --------------------------------------------------------------------------------------- */

/* torch.empty(a, b, c, dtype=float16, device=like's) */
static PyObject* new_rows(int64_t a, int64_t b, int64_t c, PyObject* like) {
  PyObject* args[5] = {PyLong_FromLongLong(a), PyLong_FromLongLong(b), PyLong_FromLongLong(c), st.f16,
                       PyObject_GetAttr(like, s_device)};
  PyObject* out = NULL;
  if (args[0] && args[1] && args[2] && args[4]) out = PyObject_Vectorcall(st.empty, args, 3, empty_names);
  Py_XDECREF(args[0]);
  Py_XDECREF(args[1]);
  Py_XDECREF(args[2]);
  Py_XDECREF(args[4]);
  return out;
}

/* rows like q's (read as x), contiguous */
static PyObject* rows_like(const Tensor* x) {
  if (x->stride[1] == x->shape[2] && x->stride[0] == x->shape[1] * x->shape[2]) return PyObject_CallOneArg(st.empty_like, x->t);
  return new_rows(x->shape[0], x->shape[1], x->shape[2], x->t);
}

/* 1: the device is current; 0: it is not; -1: error */
static int is_current(int64_t dev) {
  PyObject* r = PyObject_CallNoArgs(st.current_device);
  if (r == NULL) return -1;
  const int64_t cur = as_int(r);
  Py_DECREF(r);
  if (cur == -1 && PyErr_Occurred()) return -1;
  return cur == dev;
}
/* the call again, with the device made current (arguments as they came) */
static PyObject* again_on(int64_t dev, const char* name, PyObject* const* args, Py_ssize_t n) {
  PyObject* all = PyTuple_New(n + 2);
  if (all == NULL) return NULL;
  PyTuple_SET_ITEM(all, 0, PyLong_FromLongLong(dev));
  PyTuple_SET_ITEM(all, 1, PyUnicode_FromString(name));
  for (Py_ssize_t i = 0; i < n; ++i) PyTuple_SET_ITEM(all, i + 2, Py_NewRef(args[i]));
  PyObject* r = PyTuple_GET_ITEM(all, 0) && PyTuple_GET_ITEM(all, 1) ? PyObject_CallObject(st.on_device, all) : NULL;
  Py_DECREF(all);
  return r;
}
static int int_of(PyObject* callable, PyObject* dev, uintptr_t* out) {
  PyObject* r = PyObject_CallOneArg(callable, dev);
  if (r == NULL) return -1;
  const int64_t v = as_int(r);
  Py_DECREF(r);
  if (v == -1 && PyErr_Occurred()) return -1;
  *out = (uintptr_t)v;
  return 0;
}
typedef struct {
  uintptr_t status, stream;
} Launch;
static int read_launch(int64_t dev, Launch* l) {
  PyObject* d = PyLong_FromLongLong(dev);
  if (d == NULL) return -1;
  PyObject* word = PyDict_GetItemWithError(st.status, d);   /* borrowed */
  int rc = -1;
  if (word != NULL) rc = address(word, &l->status);
  else if (!PyErr_Occurred()) rc = int_of(st.status_ptr, d, &l->status);
  if (rc == 0) rc = int_of(st.raw_stream, d, &l->stream);
  Py_DECREF(d);
  return rc;
}
/* raises for a return code other than 0 */
static int done(int rc) {
  if (rc == 0) return 0;
  PyObject* code = PyLong_FromLong(rc);
  PyObject* r = code != NULL ? PyObject_CallOneArg(st.check, code) : NULL;
  Py_XDECREF(code);
  if (r == NULL) return -1;
  Py_DECREF(r);
  return fail("a launch was refused");
}
/* Scratch of the last few eager shapes; the Python module owns the policy, and forget() drops what is held here. */
typedef struct {
  int64_t dev, batch, rows, q_heads, kv_heads, bytes;
  uintptr_t stream, ptr;
  PyObject* ws;       /* owned; NULL: the entry is free */
} Scratch;
enum { kHeld = 4 };
static Scratch held[kHeld];
static int held_next;

/* scratch: its address and bytes, and a reference that keeps it until the launch is made (NULL for none) */
static int read_scratch(int64_t dev, uintptr_t stream, int64_t batch, int64_t rows, int64_t q_heads, int64_t kv_heads,
                        PyObject** keep, uintptr_t* ptr, int64_t* bytes) {
  uint64_t capture = 0;
  *keep = NULL;
  *ptr = 0;
  *bytes = 0;
  if (done(st.capture_id((void*)stream, &capture)) != 0) return -1;
  if (capture == 0) {
    for (int i = 0; i < kHeld; ++i) {
      const Scratch* h = &held[i];
      if (h->ws != NULL && h->dev == dev && h->stream == stream && h->batch == batch && h->rows == rows &&
          h->q_heads == q_heads && h->kv_heads == kv_heads) {
        *keep = Py_NewRef(h->ws);
        *ptr = h->ptr;
        *bytes = h->bytes;
        return 0;
      }
    }
  }
  PyObject* args = Py_BuildValue("(LKKLLLL)", (long long)dev, (unsigned long long)stream, (unsigned long long)capture,
                                 (long long)batch, (long long)rows, (long long)q_heads, (long long)kv_heads);
  if (args == NULL) return -1;
  PyObject* ws = PyObject_CallObject(st.workspace, args);
  Py_DECREF(args);
  if (ws == NULL) return -1;
  if (ws == Py_None) {
    Py_DECREF(ws);
    return 0;
  }
  *keep = ws;
  PyObject* shape = PyObject_GetAttr(ws, s_shape);
  int64_t dims[3] = {0, 0, 0};
  int nd = 0;
  if (shape == NULL || read_dims(shape, dims, &nd) != 0 || address(ws, ptr) != 0) {
    Py_XDECREF(shape);
    Py_CLEAR(*keep);
    return -1;
  }
  Py_DECREF(shape);
  *bytes = dims[0];
  if (capture == 0) {
    Scratch* h = &held[held_next];
    PyObject* old = h->ws;
    *h = (Scratch){dev, batch, rows, q_heads, kv_heads, *bytes, stream, *ptr, Py_NewRef(ws)};
    held_next = (held_next + 1) % kHeld;
    Py_XDECREF(old);
  }
  return 0;
}
static PyObject* py_forget(PyObject* self, PyObject* none) {
  for (int i = 0; i < kHeld; ++i) Py_CLEAR(held[i].ws);
  Py_RETURN_NONE;
}
static int wanted(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return 0;
  PyErr_Format(PyExc_TypeError, "%zd arguments, not %zd", want, n);
  return -1;
}
#define P(x) ((void*)(x))
#define LAUNCH(rc, call)       \
  Py_BEGIN_ALLOW_THREADS;      \
  rc = call;                   \
  Py_END_ALLOW_THREADS

/* ---- the operators ------------------------------------------------------------------------------------ */

/* append(k, v or None, slots, pool): rows [n, 2*kv_heads, 128], or K and V apart */
static PyObject* py_append(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  if (wanted(nargs, 4) != 0) return NULL;
  Pool pool;
  if (read_pool(args[3], &pool) != 0) return NULL;
  PyObject* slots = NULL;
  int64_t n = 0, ks = 0, vs = 0;
  uintptr_t sp = 0, kp = 0, vp = 0;
  if (read_slots(args[2], pool.dev, &slots, &n, &sp) != 0) goto error;
  if (args[1] == Py_None) {
    if (read_rows(args[0], "KV_Values", 2 * pool.kv_heads, n, pool.dev, &ks, &kp, NULL) != 0) goto error;
    vs = ks;
    vp = kp + (uintptr_t)pool.kv_heads * kDim * 2;
  } else if (read_rows(args[0], "xk", pool.kv_heads, n, pool.dev, &ks, &kp, NULL) != 0 ||
             read_rows(args[1], "xv", pool.kv_heads, n, pool.dev, &vs, &vp, NULL) != 0) {
    goto error;
  }
  if (n > 0) {
    const int here = is_current(pool.dev);
    if (here < 0) goto error;
    if (!here) {
      Py_DECREF(slots);
      return again_on(pool.dev, "append", args, nargs);
    }
    Launch l;
    int rc;
    if (read_launch(pool.dev, &l) != 0) goto error;
    LAUNCH(rc, st.append(P(kp), P(vp), n, ks, vs, P(sp), P(pool.ptr), pool.pages, pool.stride, (int)pool.kv_heads, kDim,
                         P(l.status), P(l.stream)));
    if (done(rc) != 0) goto error;
  }
  Py_DECREF(slots);
  Py_RETURN_NONE;
error:
  Py_XDECREF(slots);
  return NULL;
}

/* a norm weight: [128] fp16, or None */
static int read_weight(PyObject* t, const char* name, int64_t dev, uintptr_t* ptr) {
  *ptr = 0;
  if (t == Py_None) return 0;
  Tensor x;
  if (read_tensor(t, &x) != 0) return -1;
  if (x.dtype != st.f16 || x.nd != 1 || x.shape[0] != kDim || x.stride[0] != 1) {
    PyErr_Format(PyExc_ValueError, "%s must be a contiguous float16 [head_dim] tensor or None", name);
    return -1;
  }
  if (x.dev != dev) return off_device(name, t, dev);
  return address(t, ptr);
}

/* prologue(xq, xkv, q_weight, k_weight, eps, cos, sin, slots, pool, out or None) */
static PyObject* py_prologue(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  if (wanted(nargs, 10) != 0) return NULL;
  Pool pool;
  if (read_pool(args[8], &pool) != 0) return NULL;
  PyObject* slots = NULL;
  PyObject* out = args[9] == Py_None ? args[0] : args[9];
  Tensor q, kv, cos, sin;
  const double eps = PyFloat_AsDouble(args[4]);
  if (eps == -1.0 && PyErr_Occurred()) return NULL;
  if (read_tensor(args[0], &q) != 0) return NULL;
  if (q.nd != 3 || q.shape[1] == 0) return fail("xq must be float16 [n, q_heads, 128]"), NULL;
  const int64_t n = q.shape[0], q_heads = q.shape[1], row = 2 * pool.kv_heads * kDim;
  int64_t qs = 0, os = 0, rows = 0, n_slots = 0;
  uintptr_t qp = 0, op = 0, kvp = 0, cp = 0, sp = 0, qw = 0, kw = 0, slp = 0;
  if (check_rows(&q, "xq", q_heads, n, pool.dev, &qs, &qp) != 0) return NULL;
  if (out == args[0]) {
    op = qp;
    os = qs;
  } else {
    if (read_rows(out, "out", q_heads, n, pool.dev, &os, &op, &rows) != 0) return NULL;
    if (rows != n) return fail("out must match xq"), NULL;
  }
  if (read_tensor(args[1], &kv) != 0) return NULL;
  if (kv.dtype != st.f16 || kv.nd != 2 || kv.shape[0] != n || kv.shape[1] != row || kv.stride[1] != 1)
    return fail("xkv must be [n, 2*kv_heads*head_dim] float16, contiguous rows"), NULL;
  if (kv.dev != pool.dev) return off_device("xkv", args[1], pool.dev), NULL;
  if (read_tensor(args[5], &cos) != 0 || read_tensor(args[6], &sin) != 0) return NULL;
  if (cos.dtype != st.f16 || sin.dtype != st.f16) return fail("cos and sin must be float16"), NULL;
  if (cos.nd != 2 || sin.nd != 2 || cos.shape[0] != n || sin.shape[0] != n || sin.shape[1] != cos.shape[1] ||
      (cos.shape[1] != kDim && cos.shape[1] != kDim / 2) || cos.stride[1] != 1 || sin.stride[1] != 1 ||
      (n > 1 && cos.stride[0] != sin.stride[0]))
    return fail("cos and sin must be one row of head_dim (or head_dim/2) per token with equal strides"), NULL;
  if (cos.dev != pool.dev) return off_device("cos and sin", args[5], pool.dev), NULL;
  if (sin.dev != pool.dev) return off_device("cos and sin", args[6], pool.dev), NULL;
  if (read_weight(args[2], "q_norm_weight", pool.dev, &qw) != 0 || read_weight(args[3], "k_norm_weight", pool.dev, &kw) != 0)
    return NULL;
  if (address(args[1], &kvp) != 0 || address(args[5], &cp) != 0 || address(args[6], &sp) != 0) return NULL;
  if (read_slots(args[7], pool.dev, &slots, &n_slots, &slp) != 0) goto error;
  if (n_slots != n) {
    fail("Select_Index must name one slot per token");
    goto error;
  }
  if (n > 0) {
    const int here = is_current(pool.dev);
    if (here < 0) goto error;
    if (!here) {
      Py_DECREF(slots);
      return again_on(pool.dev, "prologue", args, nargs);
    }
    Launch l;
    int rc;
    if (read_launch(pool.dev, &l) != 0) goto error;
    LAUNCH(rc, st.prologue(P(qp), P(op), qs, os, P(kvp), n > 1 ? kv.stride[0] : row, P(qw), P(kw), (float)eps, P(cp), P(sp),
                           n > 1 ? cos.stride[0] : kDim, P(slp), P(pool.ptr), pool.pages, pool.stride, n, (int)q_heads,
                           (int)pool.kv_heads, kDim, P(l.status), P(l.stream)));
    if (done(rc) != 0) goto error;
  }
  Py_DECREF(slots);
  return Py_NewRef(out);
error:
  Py_XDECREF(slots);
  return NULL;
}

/* gather(pool, slots, out or None) */
static PyObject* py_gather(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  if (wanted(nargs, 3) != 0) return NULL;
  Pool pool;
  if (read_pool(args[0], &pool) != 0) return NULL;
  PyObject *slots = NULL, *out = NULL;
  int64_t n = 0, os = 0, rows = 0;
  uintptr_t sp = 0, op = 0;
  if (read_slots(args[1], pool.dev, &slots, &n, &sp) != 0) goto error;
  if (args[2] == Py_None) {
    if ((out = new_rows(n, 2 * pool.kv_heads, kDim, args[0])) == NULL || address(out, &op) != 0) goto error;
    os = 2 * pool.kv_heads * kDim;
  } else {
    out = Py_NewRef(args[2]);
    if (read_rows(out, "out", 2 * pool.kv_heads, n, pool.dev, &os, &op, &rows) != 0) goto error;
    if (rows != n) {
      PyErr_Format(PyExc_ValueError, "out must hold %lld rows", (long long)n);
      goto error;
    }
  }
  if (n > 0) {
    const int here = is_current(pool.dev);
    if (here < 0) goto error;
    if (!here) {
      PyObject* with_out[3] = {args[0], args[1], out};
      PyObject* r = again_on(pool.dev, "gather", with_out, 3);
      Py_DECREF(slots);
      Py_DECREF(out);
      return r;
    }
    Launch l;
    int rc;
    if (read_launch(pool.dev, &l) != 0) goto error;
    LAUNCH(rc, st.gather(P(pool.ptr), pool.pages, pool.stride, P(sp), n, P(op), os, (int)pool.kv_heads, kDim, P(l.status),
                         P(l.stream)));
    if (done(rc) != 0) goto error;
  }
  Py_DECREF(slots);
  return out;
error:
  Py_XDECREF(slots);
  Py_XDECREF(out);
  return NULL;
}

/* decode(q, pool, scale, table, lens, max_len, row ids or None, table_kind, page_size, out or None, metadata_fresh) */
static PyObject* py_decode(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  if (wanted(nargs, 11) != 0) return NULL;
  Pool pool;
  Tensor q;
  Table tbl;
  if (read_pool(args[1], &pool) != 0 || read_tensor(args[0], &q) != 0) return NULL;
  if (q.dtype != st.f16 || q.nd != 3 || q.shape[2] != kDim || q.stride[2] != 1)
    return fail("q must be float16 [batch, heads, 128], contiguous along head_dim"), NULL;
  if (q.dev != pool.dev) return off_device("q", args[0], pool.dev), NULL;
  const int64_t batch = q.shape[0], q_heads = q.shape[1];
  if (batch > INT32_MAX || q_heads > INT32_MAX) return fail("q is too large"), NULL;
  const double scale = PyFloat_AsDouble(args[2]);
  if (scale == -1.0 && PyErr_Occurred()) return NULL;
  const int64_t max_len = as_int(args[5]), page_size = as_int(args[8]);
  const int fresh = PyObject_IsTrue(args[10]);
  if (PyErr_Occurred()) return NULL;
  if (page_size < 0 || page_size > INT32_MAX) return fail("page_size is out of range"), NULL;
  int wide = 0;
  uintptr_t lens = 0, ids = 0, qp = 0, op = 0;
  if (read_table(args[3], args[7], pool.dev, &tbl) != 0 || read_ints(args[4], "b_seq_len", batch, pool.dev, &wide, &lens) != 0)
    return NULL;
  if (args[6] != Py_None) {
    if (read_ints(args[6], "b_req_idx", batch, pool.dev, NULL, &ids) != 0) return NULL;
  } else if (tbl.rows < batch) {
    return fail("the table has fewer rows than the batch"), NULL;
  }
  if (max_len < 0 || max_len > tbl.cols * (tbl.kind == B200KV_TABLE_BLOCK ? page_size : 1))
    return fail("max_actual_seq_len exceeds the table width"), NULL;
  PyObject *out = NULL, *ws = NULL;
  int64_t ob = q_heads * kDim, oh = kDim, ws_bytes = 0;
  uintptr_t wp = 0;
  if (args[9] == Py_None) {
    if ((out = rows_like(&q)) == NULL) return NULL;
  } else {
    Tensor o;
    if (read_tensor(args[9], &o) != 0) return NULL;
    if (o.dtype != st.f16 || o.nd != 3 || o.shape[0] != batch || o.shape[1] != q_heads || o.shape[2] != kDim || o.stride[2] != 1)
      return fail("out must match q"), NULL;
    if (o.dev != pool.dev) return off_device("out", args[9], pool.dev), NULL;
    ob = o.stride[0];
    oh = o.stride[1];
    out = Py_NewRef(args[9]);
  }
  if (batch > 0) {
    const int here = is_current(pool.dev);
    if (here < 0) goto error;
    if (!here) {
      PyObject* all[11];
      for (int i = 0; i < 11; ++i) all[i] = i == 9 ? out : args[i];
      PyObject* r = again_on(pool.dev, "decode", all, 11);
      Py_DECREF(out);
      return r;
    }
    Launch l;
    int rc;
    if (address(args[0], &qp) != 0 || address(out, &op) != 0 || read_launch(pool.dev, &l) != 0 ||
        read_scratch(pool.dev, l.stream, batch, 0, q_heads, pool.kv_heads, &ws, &wp, &ws_bytes) != 0)
      goto error;
    LAUNCH(rc, st.decode(P(qp), q.stride[0], q.stride[1], P(pool.ptr), pool.pages, pool.stride, P(tbl.ptr), tbl.stride, tbl.kind,
                         (int)tbl.rows, tbl.cols, P(ids), P(lens), wide, (int)batch, (int)q_heads, (int)pool.kv_heads, kDim,
                         (int)page_size, (float)scale, max_len, P(wp), (size_t)ws_bytes, P(op), ob, oh,
                         fresh ? B200KV_DECODE_SERIALIZED : 0, P(l.status), P(l.stream)));
    Py_XDECREF(ws);
    if (done(rc) != 0) goto error;
  }
  return out;
error:
  Py_XDECREF(out);
  return NULL;
}

/* prefill(q, pool, scale_log2, table, req ids, q_start, ctx_lens, q_lens, max_q_len, table_kind, page_size) */
static PyObject* py_prefill(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  if (wanted(nargs, 11) != 0) return NULL;
  Pool pool;
  Tensor q, ql;
  Table tbl;
  if (read_pool(args[1], &pool) != 0 || read_tensor(args[0], &q) != 0) return NULL;
  if (q.dtype != st.f16 || q.nd != 3 || q.shape[2] != kDim || q.stride[2] != 1)
    return fail("q must be float16 [tokens, heads, 128], contiguous along head_dim"), NULL;
  if (q.dev != pool.dev) return off_device("q", args[0], pool.dev), NULL;
  const int64_t total = q.shape[0], q_heads = q.shape[1];
  const double scale = PyFloat_AsDouble(args[2]);
  if (scale == -1.0 && PyErr_Occurred()) return NULL;
  const int64_t max_q = as_int(args[8]), page_size = as_int(args[10]);
  if (PyErr_Occurred()) return NULL;
  if (page_size < 0 || page_size > INT32_MAX || q_heads > INT32_MAX) return fail("page_size or heads are out of range"), NULL;
  if (read_table(args[3], args[9], pool.dev, &tbl) != 0 || read_tensor(args[7], &ql) != 0) return NULL;
  const int64_t batch = ql.nd == 1 ? ql.shape[0] : -1;
  if (batch > INT32_MAX) return fail("q_seq_lens is too long"), NULL;
  int wide = 0, ctx_wide = 0;
  uintptr_t qlens = 0, ctx = 0, ids = 0, start = 0, qp = 0, op = 0, wp = 0;
  if (check_ints(&ql, "q_seq_lens", batch, pool.dev, &wide, &qlens) != 0 ||
      read_ints(args[6], "context_lens", batch, pool.dev, &ctx_wide, &ctx) != 0)
    return NULL;
  if (wide != ctx_wide) return fail("context_lens and q_seq_lens must share dtype and shape"), NULL;
  if (read_ints(args[4], "req_ids", batch, pool.dev, NULL, &ids) != 0 ||
      read_ints(args[5], "q_start_loc", batch, pool.dev, NULL, &start) != 0)
    return NULL;
  const int work = total > 0 && q_heads > 0 && batch > 0;
  if (work) {
    const int here = is_current(pool.dev);
    if (here < 0) return NULL;
    if (!here) return again_on(pool.dev, "prefill", args, nargs);
  }
  PyObject *ws = NULL, *out = rows_like(&q);
  int64_t ws_bytes = 0;
  if (out == NULL || !work) return out;
  Launch l;
  int rc;
  if (address(args[0], &qp) != 0 || address(out, &op) != 0 || read_launch(pool.dev, &l) != 0) goto error;
  /* beyond 128 rows only their number of 128-row tiles counts for the scratch */
  const int64_t rows = max_q <= 128 ? max_q : (max_q + 127) / 128 * 128;
  if (rows > 0 && read_scratch(pool.dev, l.stream, batch, rows, q_heads, pool.kv_heads, &ws, &wp, &ws_bytes) != 0) goto error;
  LAUNCH(rc, st.prefill(P(qp), total > 1 ? q.stride[0] : q_heads * kDim, q_heads > 1 ? q.stride[1] : kDim, P(pool.ptr), pool.pages,
                        pool.stride, P(tbl.ptr), tbl.stride, tbl.kind, (int)tbl.rows, tbl.cols, P(ids), P(start), P(ctx), P(qlens),
                        wide, (int)batch, total, max_q, (int)q_heads, (int)pool.kv_heads, kDim, (int)page_size, (float)scale, P(op),
                        q_heads * kDim, kDim, P(wp), (size_t)ws_bytes, P(l.status), P(l.stream)));
  Py_XDECREF(ws);
  if (done(rc) != 0) goto error;
  return out;
error:
  Py_DECREF(out);
  return NULL;
}

/* setup(dict): the objects and entry points named in st */
static PyObject* py_setup(PyObject* self, PyObject* with) {
  if (!PyDict_Check(with)) return PyErr_SetString(PyExc_TypeError, "setup takes a dict"), NULL;
  struct { const char* name; PyObject** to; } objects[] = {
      {"float16", &st.f16}, {"int32", &st.i32}, {"int64", &st.i64}, {"uint8", &st.u8}, {"empty", &st.empty},
      {"empty_like", &st.empty_like}, {"status", &st.status},
      {"current_device", &st.current_device}, {"raw_stream", &st.raw_stream}, {"status_ptr", &st.status_ptr},
      {"workspace", &st.workspace}, {"on_device", &st.on_device}, {"refuse_cpu", &st.refuse_cpu}, {"check", &st.check}};
  struct { const char* name; void* to; } entries[] = {
      {"append", &st.append}, {"prologue", &st.prologue}, {"gather", &st.gather}, {"decode", &st.decode},
      {"prefill", &st.prefill}, {"capture_id", &st.capture_id}};
  for (size_t i = 0; i < sizeof(objects) / sizeof(objects[0]); ++i) {
    PyObject* o = PyDict_GetItemString(with, objects[i].name);
    if (o == NULL) return PyErr_Format(PyExc_KeyError, "%s", objects[i].name);
    Py_XSETREF(*objects[i].to, Py_NewRef(o));
  }
  if (!PyDict_Check(st.status)) return PyErr_SetString(PyExc_TypeError, "status must be a dict"), NULL;
  for (size_t i = 0; i < sizeof(entries) / sizeof(entries[0]); ++i) {
    PyObject* o = PyDict_GetItemString(with, entries[i].name);
    if (o == NULL) return PyErr_Format(PyExc_KeyError, "%s", entries[i].name);
    void* p = PyLong_AsVoidPtr(o);
    if (p == NULL) return PyErr_Occurred() ? NULL : PyErr_Format(PyExc_ValueError, "%s", entries[i].name);
    *(void**)entries[i].to = p;
  }
  Py_RETURN_NONE;
}

static PyMethodDef methods[] = {
    {"setup", py_setup, METH_O, NULL},
    {"forget", py_forget, METH_NOARGS, NULL},
    {"append", (PyCFunction)(void (*)(void))py_append, METH_FASTCALL, NULL},
    {"prologue", (PyCFunction)(void (*)(void))py_prologue, METH_FASTCALL, NULL},
    {"gather", (PyCFunction)(void (*)(void))py_gather, METH_FASTCALL, NULL},
    {"decode", (PyCFunction)(void (*)(void))py_decode, METH_FASTCALL, NULL},
    {"prefill", (PyCFunction)(void (*)(void))py_prefill, METH_FASTCALL, NULL},
    {NULL, NULL, 0, NULL}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kv4_native", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__kv4_native(void) {
  struct { const char* name; PyObject** to; } names[] = {
      {"shape", &s_shape}, {"stride", &s_stride}, {"dtype", &s_dtype}, {"get_device", &s_get_device},
      {"data_ptr", &s_data_ptr}, {"contiguous", &s_contiguous}, {"device", &s_device}};
  for (size_t i = 0; i < sizeof(names) / sizeof(names[0]); ++i)
    if ((*names[i].to = PyUnicode_InternFromString(names[i].name)) == NULL) return NULL;
  empty_names = Py_BuildValue("(ss)", "dtype", "device");
  return empty_names != NULL ? PyModule_Create(&module) : NULL;
}
