/* _g16fast: a CPython extension that calls the per-call entry points of libg16.so that sit on
 * latency-bound paths -- g16_skinny, g16_skinny_strips and their fp32 forms (mm_t at M <= 8 and the FastLinear decode
 * shortcut, the counterpart of the reference's PreparedLaunch, src/gtx16_fp16/kernels.py:324-338)
 * and g16_mm_t_gemm (mm_t's GEMM path, ops.py:86-108) -- with METH_FASTCALL argument parsing. Through ctypes the same calls spend
 * ~0.1 us per argument converting them; here the conversion is a few ns per argument.
 *
 * The module does not link libg16.so: bind() receives the addresses of the functions from the
 * library the ctypes binding already loaded, so both bindings call into the same instance. Pointer
 * arguments are Python ints or None (NULL); every call returns the entry point's int status. The
 * GIL is released around the call, as ctypes does.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <float.h>
#include <math.h>
#include <stddef.h>
#include <stdint.h>
#include <string.h>

#include "g16.h"

typedef int (*skinny_fn)(const void*, const void*, void*, const void*, int, int, int, int, void*, size_t, void*,
                         size_t, void*);
typedef int (*mm_t_gemm_fn)(const void*, int, const void*, void*, int, const void*, float, int, int, int, int, void*,
                            size_t, void*, size_t, void*, size_t, void*);

typedef int (*strips_fn)(const void*, const void*, void*, const void*, int, int, int, void*);
typedef int (*skinny_any_fn)(const void*, int, const void*, void*, int, const void*, int, int, int, int, void*, size_t,
                             void*, size_t, void*);
typedef int (*strips_any_fn)(const void*, int, const void*, void*, int, const void*, int, int, int, void*);
static skinny_any_fn g_skinny = NULL;
static strips_any_fn g_strips = NULL;
static skinny_fn g_skinny_f32in = NULL;
static strips_fn g_strips_f32in = NULL;
static mm_t_gemm_fn g_mm_t_gemm = NULL;

static int as_ptr(PyObject* o, void** out) {
  if (o == Py_None) {
    *out = NULL;
    return 0;
  }
  *out = PyLong_AsVoidPtr(o);
  return (*out == NULL && PyErr_Occurred()) ? -1 : 0;
}

static int as_int(PyObject* o, int* out) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) return -1;
  if (v < INT32_MIN || v > INT32_MAX) {
    PyErr_SetString(PyExc_OverflowError, "argument does not fit a C int");
    return -1;
  }
  *out = (int)v;
  return 0;
}

static int as_size(PyObject* o, size_t* out) {
  *out = PyLong_AsSize_t(o);
  return (*out == (size_t)-1 && PyErr_Occurred()) ? -1 : 0;
}

static int check_nargs(const char* name, Py_ssize_t nargs, Py_ssize_t want) {
  if (nargs == want) return 0;
  PyErr_Format(PyExc_TypeError, "%s() takes %zd arguments (%zd given)", name, want, nargs);
  return -1;
}

static PyObject* fast_bind(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  void *skinny, *gemm, *strips, *skinny_any, *strips_any;
  if (check_nargs("bind", nargs, 5) || as_ptr(args[0], &skinny) || as_ptr(args[1], &gemm) ||
      as_ptr(args[2], &strips) || as_ptr(args[3], &skinny_any) || as_ptr(args[4], &strips_any))
    return NULL;
  if (skinny == NULL || gemm == NULL || strips == NULL || skinny_any == NULL || strips_any == NULL) {
    PyErr_SetString(PyExc_ValueError, "bind() needs five non-NULL function addresses");
    return NULL;
  }
  g_skinny_f32in = (skinny_fn)skinny;
  g_mm_t_gemm = (mm_t_gemm_fn)gemm;
  g_strips_f32in = (strips_fn)strips;
  g_skinny = (skinny_any_fn)skinny_any;
  g_strips = (strips_any_fn)strips_any;
  Py_RETURN_NONE;
}

static int check_bound(const void* fn) {
  if (fn != NULL) return 0;
  PyErr_SetString(PyExc_RuntimeError, "_g16fast: bind() has not been called");
  return -1;
}

/* skinny_f32in(x, w_t, out, bias, M, N, K, ksplit, partials, partial_bytes, counters, counter_bytes,
 * stream) -> status of g16_skinny_f32in */
static PyObject* fast_skinny_f32in(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  void *x, *w, *out, *bias, *part, *cnt, *stream;
  int M, N, K, ksplit, st;
  size_t part_bytes, cnt_bytes;
  if (check_bound((const void*)g_skinny_f32in) || check_nargs("skinny_f32in", nargs, 13)) return NULL;
  if (as_ptr(args[0], &x) || as_ptr(args[1], &w) || as_ptr(args[2], &out) || as_ptr(args[3], &bias) ||
      as_int(args[4], &M) || as_int(args[5], &N) || as_int(args[6], &K) || as_int(args[7], &ksplit) ||
      as_ptr(args[8], &part) || as_size(args[9], &part_bytes) || as_ptr(args[10], &cnt) ||
      as_size(args[11], &cnt_bytes) || as_ptr(args[12], &stream))
    return NULL;
  Py_BEGIN_ALLOW_THREADS
  st = g_skinny_f32in(x, w, out, bias, M, N, K, ksplit, part, part_bytes, cnt, cnt_bytes, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(st);
}

/* skinny_strips_f32in(x, wd, out, bias, M, N, K, stream) -> status of g16_skinny_strips_f32in */
static PyObject* fast_strips_f32in(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  void *x, *wd, *out, *bias, *stream;
  int M, N, K, st;
  if (check_bound((const void*)g_strips_f32in) || check_nargs("skinny_strips_f32in", nargs, 8)) return NULL;
  if (as_ptr(args[0], &x) || as_ptr(args[1], &wd) || as_ptr(args[2], &out) || as_ptr(args[3], &bias) ||
      as_int(args[4], &M) || as_int(args[5], &N) || as_int(args[6], &K) || as_ptr(args[7], &stream))
    return NULL;
  Py_BEGIN_ALLOW_THREADS
  st = g_strips_f32in(x, wd, out, bias, M, N, K, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(st);
}

/* skinny(x, x_is_f32, w_t, out, out_is_f16, bias, M, N, K, ksplit, partials, partial_bytes, counters,
 * counter_bytes, stream) -> status of g16_skinny */
static PyObject* fast_skinny(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  void *x, *w, *out, *bias, *part, *cnt, *stream;
  int x_is_f32, out_is_f16, M, N, K, ksplit, st;
  size_t part_bytes, cnt_bytes;
  if (check_bound((const void*)g_skinny) || check_nargs("skinny", nargs, 15)) return NULL;
  if (as_ptr(args[0], &x) || as_int(args[1], &x_is_f32) || as_ptr(args[2], &w) || as_ptr(args[3], &out) ||
      as_int(args[4], &out_is_f16) || as_ptr(args[5], &bias) || as_int(args[6], &M) || as_int(args[7], &N) ||
      as_int(args[8], &K) || as_int(args[9], &ksplit) || as_ptr(args[10], &part) || as_size(args[11], &part_bytes) ||
      as_ptr(args[12], &cnt) || as_size(args[13], &cnt_bytes) || as_ptr(args[14], &stream))
    return NULL;
  Py_BEGIN_ALLOW_THREADS
  st = g_skinny(x, x_is_f32, w, out, out_is_f16, bias, M, N, K, ksplit, part, part_bytes, cnt, cnt_bytes, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(st);
}

/* skinny_strips(x, x_is_f32, wd, out, out_is_f16, bias, M, N, K, stream) -> status of g16_skinny_strips */
static PyObject* fast_strips(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  void *x, *wd, *out, *bias, *stream;
  int x_is_f32, out_is_f16, M, N, K, st;
  if (check_bound((const void*)g_strips) || check_nargs("skinny_strips", nargs, 10)) return NULL;
  if (as_ptr(args[0], &x) || as_int(args[1], &x_is_f32) || as_ptr(args[2], &wd) || as_ptr(args[3], &out) ||
      as_int(args[4], &out_is_f16) || as_ptr(args[5], &bias) || as_int(args[6], &M) || as_int(args[7], &N) ||
      as_int(args[8], &K) || as_ptr(args[9], &stream))
    return NULL;
  Py_BEGIN_ALLOW_THREADS
  st = g_strips(x, x_is_f32, wd, out, out_is_f16, bias, M, N, K, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(st);
}

/* mm_t_gemm(x, x_is_f32, w_t, out, out_is_f16, bias, thresh, M, N, K, num_cus, scratch, scratch_bytes,
 * workspace, workspace_bytes, counters, counter_bytes, stream) -> status of g16_mm_t_gemm */
static PyObject* fast_mm_t_gemm(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  void *x, *w, *out, *bias, *scratch, *ws, *cnt, *stream;
  int x_is_f32, out_is_f16, M, N, K, cus, st;
  size_t scratch_bytes, ws_bytes, cnt_bytes;
  double thresh;
  if (check_bound((const void*)g_mm_t_gemm) || check_nargs("mm_t_gemm", nargs, 18)) return NULL;
  if (as_ptr(args[0], &x) || as_int(args[1], &x_is_f32) || as_ptr(args[2], &w) || as_ptr(args[3], &out) ||
      as_int(args[4], &out_is_f16) || as_ptr(args[5], &bias))
    return NULL;
  thresh = PyFloat_AsDouble(args[6]);
  if (thresh == -1.0 && PyErr_Occurred()) return NULL;
  if (as_int(args[7], &M) || as_int(args[8], &N) || as_int(args[9], &K) || as_int(args[10], &cus) ||
      as_ptr(args[11], &scratch) || as_size(args[12], &scratch_bytes) || as_ptr(args[13], &ws) ||
      as_size(args[14], &ws_bytes) || as_ptr(args[15], &cnt) || as_size(args[16], &cnt_bytes) ||
      as_ptr(args[17], &stream))
    return NULL;
  Py_BEGIN_ALLOW_THREADS
  st = g_mm_t_gemm(x, x_is_f32, w, out, out_is_f16, bias, (float)thresh, M, N, K, cus, scratch, scratch_bytes, ws,
                   ws_bytes, cnt, cnt_bytes, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(st);
}

/* Entry points that take one struct of arguments whose last two fields are the workspace and its size:
 * `head` holds the fields before them. */
typedef size_t (*args_size_fn)(const void*);
typedef int (*args_call_fn)(const void*, void*);
enum { kMaxArgs = 512 };
typedef struct {
  void* workspace;
  int64_t workspace_bytes;
} args_tail;

static int join_args(PyObject* head, void* ws, size_t ws_bytes, unsigned char* out) {
  char* data;
  Py_ssize_t n;
  if (PyBytes_AsStringAndSize(head, &data, &n)) return -1;
  if (n % 8 != 0 || n > (Py_ssize_t)(kMaxArgs - sizeof(args_tail))) {
    PyErr_SetString(PyExc_ValueError, "argument struct of an unexpected size");
    return -1;
  }
  const args_tail tail = {ws, (int64_t)ws_bytes};
  memcpy(out, data, (size_t)n);
  memcpy(out + n, &tail, sizeof(tail));
  return 0;
}

/* args_size(fn_addr, head) -> size_t fn(const args*) */
static PyObject* fast_args_size(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  void* fn;
  _Alignas(16) unsigned char buf[kMaxArgs];
  if (check_nargs("args_size", nargs, 2) || as_ptr(args[0], &fn) || check_bound(fn) || join_args(args[1], NULL, 0, buf))
    return NULL;
  return PyLong_FromSize_t(((args_size_fn)fn)(buf));
}

/* args_call(fn_addr, head, workspace, workspace_bytes, stream) -> status of int fn(const args*, stream) */
static PyObject* fast_args_call(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  void *fn, *ws, *stream;
  size_t ws_bytes;
  int st;
  _Alignas(16) unsigned char buf[kMaxArgs];
  if (check_nargs("args_call", nargs, 5) || as_ptr(args[0], &fn) || check_bound(fn) || as_ptr(args[2], &ws) ||
      as_size(args[3], &ws_bytes) || as_ptr(args[4], &stream) || join_args(args[1], ws, ws_bytes, buf))
    return NULL;
  Py_BEGIN_ALLOW_THREADS
  st = ((args_call_fn)fn)(buf, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(st);
}

/* struct_call(fn_addr, args, stream) -> status of int fn(const args*, stream) */
static PyObject* fast_struct_call(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  void *fn, *stream;
  char* data;
  Py_ssize_t n;
  int st;
  _Alignas(16) unsigned char buf[kMaxArgs];
  if (check_nargs("struct_call", nargs, 3) || as_ptr(args[0], &fn) || check_bound(fn) || as_ptr(args[2], &stream) ||
      PyBytes_AsStringAndSize(args[1], &data, &n))
    return NULL;
  if (n % 8 != 0 || n > kMaxArgs) {
    PyErr_SetString(PyExc_ValueError, "argument struct of an unexpected size");
    return NULL;
  }
  memcpy(buf, data, (size_t)n);
  Py_BEGIN_ALLOW_THREADS
  st = ((args_call_fn)fn)(buf, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(st);
}

/* ---- the usual calls of attention, attention_decode, lora_mm_t and others, checked and packed here -------------
 * Each takes what its Python function takes and returns the output, or None for anything but a call that
 * could go straight to the kernels: operands of another type, shape, layout or device, a gradient wanted,
 * a scratch buffer that has to grow. The Python function then looks at the arguments one by one, copies
 * what has to be copied or says what is wrong with them. A tensor is read through its public attributes
 * (about 0.3 us of calls each, where the same checks in Python take 1). */
typedef struct {
  void* ptr;
  int64_t shape[4], stride[4]; /* in elements */
  int nd, device;
  PyObject* dtype; /* torch's own dtype objects live as long as torch */
} tensor_t;

static PyObject *s_dtype, *s_shape, *s_stride, *s_data_ptr, *s_get_device, *s_requires_grad, *s_new_empty;
static PyObject *g_f16 = NULL, *g_f32 = NULL, *g_i32 = NULL, *g_raw_stream = NULL, *g_grad_enabled = NULL, *g_ready = NULL,
                *g_scratch = NULL;
typedef size_t (*attention_size_fn)(const g16_attention_args*);
typedef int (*attention_fn)(const g16_attention_args*, void*);
static attention_size_fn g_attention_size[2];
static attention_fn g_attention[2];

#define MAX_DEVICES 64
static int g_device_cus[MAX_DEVICES]; /* 0: not asked yet, -1: not a device of these kernels */

static int int_tuple(PyObject* o, int64_t* out, int* n) {
  if (o == NULL || !PyTuple_Check(o) || PyTuple_GET_SIZE(o) > 4) {
    Py_XDECREF(o);
    return -1;
  }
  *n = (int)PyTuple_GET_SIZE(o);
  for (int i = 0; i < *n; ++i) out[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(o, i));
  Py_DECREF(o);
  return PyErr_Occurred() ? -1 : 0;
}

/* 0: t is filled in; -1: not a tensor that can be looked at (no error is left set) */
static int read_tensor(PyObject* o, tensor_t* t) {
  int n = 0;
  PyObject* x;
  if (int_tuple(PyObject_GetAttr(o, s_shape), t->shape, &t->nd) || int_tuple(PyObject_CallMethodNoArgs(o, s_stride), t->stride, &n) ||
      n != t->nd)
    goto no;
  x = PyObject_CallMethodNoArgs(o, s_data_ptr);
  if (x == NULL) goto no;
  t->ptr = PyLong_AsVoidPtr(x);
  Py_DECREF(x);
  x = PyObject_CallMethodNoArgs(o, s_get_device);
  if (x == NULL) goto no;
  t->device = (int)PyLong_AsLong(x);
  Py_DECREF(x);
  t->dtype = PyObject_GetAttr(o, s_dtype);
  if (t->dtype == NULL || PyErr_Occurred()) goto no;
  Py_DECREF(t->dtype);
  return 0;
no:
  PyErr_Clear();
  return -1;
}

/* Where a tensor that was made here lies; NULL where that cannot be told */
static void* pointer_of(PyObject* o) {
  PyObject* x = PyObject_CallMethodNoArgs(o, s_data_ptr);
  void* ptr = x == NULL ? NULL : PyLong_AsVoidPtr(x);
  Py_XDECREF(x);
  PyErr_Clear();
  return ptr;
}

/* Compute units of a device these kernels run on; -1 else */
static int device_cus(int device) {
  if (device < 0 || device >= MAX_DEVICES) return -1;
  if (g_device_cus[device] == 0) {
    PyObject* r = PyObject_CallFunction(g_ready, "i", device);
    long n = r == NULL ? -1 : PyLong_AsLong(r);
    Py_XDECREF(r);
    PyErr_Clear();
    g_device_cus[device] = n > 0 ? (int)n : -1;
  }
  return g_device_cus[device];
}

/* Whether a gradient is wanted of one of args[which[0]] .. (tensors or None) */
static int wants_grad(PyObject* const* args, const int* which, int n) {
  PyObject* r = PyObject_CallNoArgs(g_grad_enabled);
  int on = r != Py_False;
  Py_XDECREF(r);
  if (!on) return 0;
  for (int i = 0; i < n; ++i) {
    if (args[which[i]] == Py_None) continue;
    r = PyObject_GetAttr(args[which[i]], s_requires_grad);
    on = r != Py_False;
    Py_XDECREF(r);
    if (on) return 1;
  }
  return 0;
}

static int raw_stream(int device, void** out) {
  PyObject *i = PyLong_FromLong(device), *r = i == NULL ? NULL : PyObject_CallOneArg(g_raw_stream, i);
  Py_XDECREF(i);
  if (r == NULL) return -1;
  *out = PyLong_AsVoidPtr(r);
  Py_DECREF(r);
  return PyErr_Occurred() ? -1 : 0;
}

/* Pointer of the scratch buffer of (device, stream), at least `bytes` long */
static int scratch(int device, void* stream, size_t bytes, void** out) {
  PyObject* r = PyObject_CallFunction(g_scratch, "iKn", device, (unsigned long long)(uintptr_t)stream, (Py_ssize_t)bytes);
  if (r == NULL) return -1;
  *out = PyLong_AsVoidPtr(r);
  Py_DECREF(r);
  return PyErr_Occurred() ? -1 : 0;
}

static PyObject* empty_like(PyObject* o) {
  PyObject* shape = PyObject_GetAttr(o, s_shape);
  if (shape == NULL) return NULL;
  PyObject* argv[2] = {o, shape};
  PyObject* r = PyObject_VectorcallMethod(s_new_empty, argv, 2, NULL);
  Py_DECREF(shape);
  return r;
}

static int aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

/* Rows [.., token, head, d] that the kernels read in place (attn.py: _rows) */
static int rows_ok(const tensor_t* t, int size, int64_t d, int keys) {
  if (t->stride[t->nd - 1] != 1 || !aligned(t->ptr)) return 0;
  for (int i = 0; i < t->nd - 1; ++i)
    if (t->stride[i] * size % 16 != 0) return 0;
  const int64_t token = t->stride[t->nd - 3];
  return !keys || (token >= d && token * size < G16_ATTENTION_MAX_STRIDE);
}

/* A contiguous int32 or fp32 vector (NULL for None) */
static int vector(PyObject* o, PyObject* dtype, int64_t n, int device, const void** out) {
  tensor_t t;
  *out = NULL;
  if (o == Py_None) return 0;
  if (read_tensor(o, &t) || t.dtype != dtype || t.nd != 1 || t.shape[0] != n || t.device != device || (n > 1 && t.stride[0] != 1)) return -1;
  *out = t.ptr;
  return 0;
}

static int fits(int64_t v) { return v >= 0 && v <= INT32_MAX; }

static int heads_ok(const tensor_t* q, const tensor_t* k, const tensor_t* v, g16_attention_args* a) {
  const int64_t hq = q->shape[q->nd - 2], d = q->shape[q->nd - 1], hkv = k->shape[k->nd - 2];
  if ((q->dtype != g_f16 && q->dtype != g_f32) || k->dtype != q->dtype || v->dtype != q->dtype || k->device != q->device ||
      v->device != q->device || memcmp(k->shape, v->shape, sizeof(int64_t) * (size_t)k->nd) != 0 || k->shape[k->nd - 1] != d || d <= 0 ||
      d % 8 != 0 || d > G16_ATTENTION_MAX_D || !fits(hq) || !fits(hkv) || hkv == 0 || hq == 0 || hq % hkv != 0)
    return 0;
  a->hq = (int)hq;
  a->hkv = (int)hkv;
  a->d = (int)d;
  a->is_f32 = q->dtype == g_f32;
  a->num_cus = device_cus(q->device);
  const int size = a->is_f32 ? 4 : 2;
  return a->num_cus > 0 && rows_ok(q, size, d, 0) && rows_ok(k, size, d, 1) && rows_ok(v, size, d, 1);
}

/* scale, softcap, shared keys, slopes */
static int rest_ok(PyObject* scale, PyObject* cap, PyObject* sk, PyObject* sv, PyObject* slopes, int device, PyObject* dtype, g16_attention_args* a) {
  double c = PyFloat_AsDouble(cap), s = scale == Py_None ? 0.0 : PyFloat_AsDouble(scale);
  if (PyErr_Occurred()) return 0;
  if (scale == Py_None) {
    s = 1.0 / sqrt((double)a->d);
  }
  /* (what fp32 cannot hold is left to the Python function, which says so) */
  if (s != s || (fabs(s) > FLT_MAX && !isinf(s)) || !(c >= 0.0 && c <= FLT_MAX) || (c > 0.0 && (float)c == 0.0f)) return 0;
  a->scale = (float)s;
  a->softcap = (float)c;
  if (vector(slopes, g_f32, a->hq, device, (const void**)&a->slopes)) return 0;
  if ((sk == Py_None) != (sv == Py_None)) return 0;
  if (sk != Py_None) {
    tensor_t tk, tv;
    const int size = a->is_f32 ? 4 : 2;
    if (read_tensor(sk, &tk) || read_tensor(sv, &tv) || tk.nd != 3 || tv.nd != 3 || tk.dtype != dtype || tv.dtype != dtype ||
        tk.device != device || tv.device != device || memcmp(tk.shape, tv.shape, sizeof(int64_t) * 3) != 0 || tk.shape[1] != a->hkv ||
        tk.shape[2] != a->d || tk.shape[0] == 0 || !fits(tk.shape[0]) || !rows_ok(&tk, size, a->d, 1) || !rows_ok(&tv, size, a->d, 1))
      return 0;
    a->shared_k = tk.ptr;
    a->shared_v = tv.ptr;
    a->shared = (int)tk.shape[0];
    a->shared_k_token = tk.stride[0];
    a->shared_k_head = tk.stride[1];
    a->shared_v_token = tv.stride[0];
    a->shared_v_head = tv.stride[1];
  }
  return 1;
}

static PyObject* none_clear(void) {
  PyErr_Clear();
  Py_RETURN_NONE;
}

/* The output, or None with no error set where the library rejects the arguments (the Python function then
 * makes the same call and raises) */
static PyObject* run_attention(PyObject* q, int device, g16_attention_args* a, int decode) {
  void* stream;
  PyObject* out;
  int st;
  const size_t bytes = g_attention_size[decode](a);
  if (raw_stream(device, &stream) || (bytes > 0 && scratch(device, stream, bytes, &a->workspace))) return none_clear();
  if (bytes > 0 && a->workspace == NULL) Py_RETURN_NONE;
  a->workspace_bytes = (int64_t)bytes;
  out = empty_like(q);
  tensor_t t;
  if (out == NULL || read_tensor(out, &t)) {
    Py_XDECREF(out);
    return none_clear();
  }
  a->out = t.ptr;
  Py_BEGIN_ALLOW_THREADS
  st = g_attention[decode](a, stream);
  Py_END_ALLOW_THREADS
  if (st != 0) {
    Py_DECREF(out);
    Py_RETURN_NONE;
  }
  return out;
}

/* attention(q, k, v, q_offsets, k_offsets, causal, visible, shared_k, shared_v, scale, softcap, slopes) */
static const int kGradAttention[6] = {0, 1, 2, 7, 8, 11};
static PyObject* fast_attention(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  tensor_t q, k, v;
  g16_attention_args a;
  if (check_nargs("attention", nargs, 12)) return NULL;
  if (g_ready == NULL) Py_RETURN_NONE;
  memset(&a, 0, sizeof(a));
  const int packed = args[3] != Py_None;
  if (read_tensor(args[0], &q) || read_tensor(args[1], &k) || read_tensor(args[2], &v) || q.nd != (packed ? 3 : 4) || k.nd != q.nd ||
      v.nd != q.nd || !heads_ok(&q, &k, &v, &a) || wants_grad(args, kGradAttention, 6))
    return none_clear();
  if (packed) {
    tensor_t o;
    const PyObject* ko = args[4] == Py_None ? args[3] : args[4];
    if (read_tensor(args[3], &o) || o.nd != 1 || o.shape[0] < 2 || !fits(o.shape[0] - 1) ||
        vector(args[3], g_i32, o.shape[0], q.device, (const void**)&a.q_offsets) ||
        vector((PyObject*)ko, g_i32, o.shape[0], q.device, (const void**)&a.k_offsets))
      return none_clear();
    a.seqs = (int)(o.shape[0] - 1);
    a.q_token = q.stride[0], a.q_head = q.stride[1];
    a.k_token = k.stride[0], a.k_head = k.stride[1];
    a.v_token = v.stride[0], a.v_head = v.stride[1];
  } else {
    if (args[4] != Py_None || k.shape[0] != q.shape[0] || !fits(q.shape[0])) return none_clear();
    a.seqs = (int)q.shape[0];
    a.q_seq = q.stride[0], a.q_token = q.stride[1], a.q_head = q.stride[2];
    a.k_seq = k.stride[0], a.k_token = k.stride[1], a.k_head = k.stride[2];
    a.v_seq = v.stride[0], a.v_token = v.stride[1], a.v_head = v.stride[2];
  }
  const int64_t q_len = q.shape[q.nd - 3], k_len = k.shape[k.nd - 3];
  const int causal = PyObject_IsTrue(args[5]);
  if (!fits(q_len) || !fits(k_len) || q_len == 0 || a.seqs == 0 || causal < 0) return none_clear();
  a.q_len = (int)q_len;
  a.k_len = (int)k_len;
  a.causal = causal;
  if (vector(args[6], g_i32, a.seqs, q.device, (const void**)&a.visible) ||
      !rest_ok(args[9], args[10], args[7], args[8], args[11], q.device, q.dtype, &a))
    return none_clear();
  a.q = q.ptr, a.k = k.ptr, a.v = v.ptr;
  return run_attention(args[0], q.device, &a, 0);
}

/* attention_decode(q, k_cache, v_cache, lengths, pages, shared_k, shared_v, scale, softcap, slopes) */
static const int kGradDecode[6] = {0, 1, 2, 5, 6, 9};
static PyObject* fast_attention_decode(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  tensor_t q, k, v;
  g16_attention_args a;
  if (check_nargs("attention_decode", nargs, 10)) return NULL;
  if (g_ready == NULL) Py_RETURN_NONE;
  memset(&a, 0, sizeof(a));
  if (read_tensor(args[0], &q) || read_tensor(args[1], &k) || read_tensor(args[2], &v) || q.nd != 3 || k.nd != 4 || v.nd != 4 ||
      q.shape[0] == 0 || !fits(q.shape[0]) || !fits(k.shape[0]) || !fits(k.shape[1]) || k.shape[1] == 0 || !heads_ok(&q, &k, &v, &a) ||
      wants_grad(args, kGradDecode, 6) || vector(args[3], g_i32, q.shape[0], q.device, (const void**)&a.lengths) || a.lengths == NULL)
    return none_clear();
  a.seqs = (int)q.shape[0];
  a.q_len = 1;
  a.page = (int)k.shape[1];
  a.num_pages = (int)k.shape[0];
  a.k_len = a.page;
  if (args[4] != Py_None) {
    tensor_t t;
    if (read_tensor(args[4], &t) || t.dtype != g_i32 || t.nd != 2 || t.shape[0] != a.seqs || t.device != q.device || t.stride[1] != 1 ||
        t.stride[0] != t.shape[1] || t.shape[1] == 0 || !fits(t.shape[1] * a.page))
      return none_clear();
    a.pages = t.ptr;
    a.max_pages = (int)t.shape[1];
    a.k_len = a.max_pages * a.page;
  } else if (k.shape[0] != a.seqs) {
    Py_RETURN_NONE;
  }
  if (!rest_ok(args[7], args[8], args[5], args[6], args[9], q.device, q.dtype, &a)) return none_clear();
  a.q = q.ptr, a.k = k.ptr, a.v = v.ptr;
  a.q_seq = q.stride[0], a.q_head = q.stride[1];
  a.k_seq = k.stride[0], a.k_token = k.stride[1], a.k_head = k.stride[2];
  a.v_seq = v.stride[0], a.v_token = v.stride[1], a.v_head = v.stride[2];
  return run_attention(args[0], q.device, &a, 1);
}

typedef size_t (*lora_size_fn)(const g16_lora_args*);
typedef int (*lora_fn)(const g16_lora_args*, void*);
static lora_size_fn g_lora_size;
static lora_fn g_lora_shrink, g_lora_expand;
static PyObject* s_dtype_names = NULL;

static int packed_rows(const tensor_t* t, PyObject* dtype, int nd, int device) {
  int64_t step = 1;
  if (t->nd != nd || t->dtype != dtype || t->device != device || !aligned(t->ptr)) return 0;
  for (int i = nd - 1; i >= 0; --i) {
    if (t->shape[i] <= 0 || !fits(t->shape[i]) || (t->shape[i] > 1 && t->stride[i] != step)) return 0;
    step *= t->shape[i];
  }
  return 1;
}

static PyObject* new_matrix(PyObject* like, int64_t M, int64_t N, PyObject* dtype) {
  PyObject* shape = Py_BuildValue("(LL)", (long long)M, (long long)N);
  if (shape == NULL) return NULL;
  PyObject* argv[3] = {like, shape, dtype};
  PyObject* r = PyObject_VectorcallMethod(s_new_empty, argv, 2, s_dtype_names);
  Py_DECREF(shape);
  return r;
}

typedef int (*raw_fn)(const void*, const void*, int, void*, int, const void*, int, int, int, int, void*);
typedef int (*direct_fn)(const void*, const void*, int, void*, int, const void*, float, int, int, int, int, void*);
static raw_fn g_mm_t_raw;
static direct_fn g_mm_t_direct;
static PyObject* g_route = NULL;

/* The shared product as mm_t makes it, fp32 out */
typedef struct {
  int kind, ksplit; /* 0: skinny, 1: mm_t_gemm, 2: one launch that reads x itself */
  double thresh;
  void* ptr[3]; /* scratch, partials, counters */
  size_t bytes[3];
} product_t;

/* g_route(device, stream, M, N, K, x is fp32) -> (kind, ksplit, threshold, scratch, bytes, partials, bytes, counters,
 * bytes), or None where a buffer is not kept between calls */
static int product_route(int device, void* stream, const g16_lora_args* a, product_t* p) {
  PyObject* r = PyObject_CallFunction(g_route, "iKiiii", device, (unsigned long long)(uintptr_t)stream, a->M, a->N, a->K, a->x_is_f32);
  int bad = r == NULL || !PyTuple_Check(r) || PyTuple_GET_SIZE(r) != 9 || as_int(PyTuple_GET_ITEM(r, 0), &p->kind) ||
            as_int(PyTuple_GET_ITEM(r, 1), &p->ksplit);
  if (!bad) {
    p->thresh = PyFloat_AsDouble(PyTuple_GET_ITEM(r, 2));
    for (int i = 0; i < 3; ++i)
      bad = bad || as_ptr(PyTuple_GET_ITEM(r, 3 + 2 * i), &p->ptr[i]) || as_size(PyTuple_GET_ITEM(r, 4 + 2 * i), &p->bytes[i]);
  }
  Py_XDECREF(r);
  return bad || PyErr_Occurred() ? -1 : 0;
}

static int run_product(const product_t* p, const g16_lora_args* a, const void* w, const void* bias, void* stream) {
  void* y = (void*)a->y;
  if (p->kind == 0)
    return g_skinny(a->x, a->x_is_f32, w, y, 0, bias, a->M, a->N, a->K, p->ksplit, p->ptr[1], p->bytes[1], p->ptr[2], p->bytes[2], stream);
  if (p->kind == 1)
    return g_mm_t_gemm(a->x, a->x_is_f32, w, y, 0, bias, (float)p->thresh, a->M, a->N, a->K, a->num_cus, p->ptr[0], p->bytes[0], p->ptr[1],
                       p->bytes[1], p->ptr[2], p->bytes[2], stream);
  return a->x_is_f32 ? g_mm_t_direct(a->x, w, 0, y, 0, bias, (float)p->thresh, a->M, a->N, a->K, a->num_cus, stream)
                     : g_mm_t_raw(a->x, w, 0, y, 0, bias, a->M, a->N, a->K, a->num_cus, stream);
}

/* lora_mm_t(x2d, w_t, down, up, index, scale, bias, out_dtype) */
static const int kGradLora[6] = {0, 1, 2, 3, 5, 6};
static PyObject* fast_lora_mm_t(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  tensor_t x, w, down, up, t;
  g16_lora_args a;
  const void* bias;
  void* stream;
  product_t product;
  PyObject *y = NULL, *out = NULL;
  int st;
  if (check_nargs("lora_mm_t", nargs, 8)) return NULL;
  if (g_ready == NULL) Py_RETURN_NONE;
  memset(&a, 0, sizeof(a));
  if (read_tensor(args[0], &x) || x.nd != 2 || (x.dtype != g_f16 && x.dtype != g_f32) ||
      !packed_rows(&x, x.dtype, 2, x.device) || (a.num_cus = device_cus(x.device)) <= 0 || read_tensor(args[1], &w) ||
      !packed_rows(&w, g_f16, 2, x.device) || w.shape[0] != x.shape[1] || w.shape[0] % 8 != 0 || w.shape[1] % 8 != 0 ||
      w.shape[0] > G16_LORA_MAX_SIDE || w.shape[1] > G16_LORA_MAX_SIDE || read_tensor(args[2], &down) || !packed_rows(&down, g_f16, 3, x.device) || read_tensor(args[3], &up) ||
      !packed_rows(&up, g_f16, 3, x.device) || down.shape[2] != w.shape[0] || up.shape[1] != w.shape[1] || up.shape[0] != down.shape[0] ||
      up.shape[2] != down.shape[1] || down.shape[1] % 8 != 0 || down.shape[1] > G16_LORA_MAX_RANK ||
      vector(args[4], g_i32, x.shape[0], x.device, (const void**)&a.index) || a.index == NULL ||
      vector(args[5], g_f32, down.shape[0], x.device, (const void**)&a.scale) || vector(args[6], g_f32, w.shape[1], x.device, &bias) ||
      !aligned(bias) || (args[7] != g_f16 && args[7] != g_f32) || wants_grad(args, kGradLora, 6) || raw_stream(x.device, &stream))
    return none_clear();
  a.M = (int)x.shape[0], a.K = (int)w.shape[0], a.N = (int)w.shape[1];
  a.adapters = (int)down.shape[0], a.rank = (int)down.shape[1];
  a.x_is_f32 = x.dtype == g_f32, a.out_is_f16 = args[7] == g_f16;
  a.x = x.ptr, a.down = down.ptr, a.up = up.ptr;
  if (product_route(x.device, stream, &a, &product)) return none_clear();
  y = new_matrix(args[0], a.M, a.N, g_f32);
  out = y == NULL ? NULL : (a.out_is_f16 ? new_matrix(args[0], a.M, a.N, g_f16) : Py_NewRef(y));
  if (out == NULL || read_tensor(y, &t)) goto no;
  a.y = t.ptr;
  if (read_tensor(out, &t)) goto no;
  a.out = t.ptr;
  const size_t bytes = g_lora_size(&a);
  if (bytes > 0 && (scratch(x.device, stream, bytes, &a.workspace) || a.workspace == NULL)) goto no;
  a.workspace_bytes = (int64_t)bytes;
  Py_BEGIN_ALLOW_THREADS
  st = run_product(&product, &a, w.ptr, bias, stream);
  if (st == 0 && bytes > 0) st = g_lora_shrink(&a, stream);
  if (st == 0) st = g_lora_expand(&a, stream);
  Py_END_ALLOW_THREADS
  if (st != 0) goto no;
  Py_DECREF(y);
  return out;
no:
  Py_XDECREF(y);
  Py_XDECREF(out);
  return none_clear();
}

/* ---- rotary positions and caches in 8 bits --------------------------------------------------------------- */
static PyObject *g_i8 = NULL, *g_e4m3 = NULL, *g_capturing = NULL;
typedef int (*rotary_fn)(const g16_rotary_args*, void*);
typedef int (*cache_fn)(const g16_cache_args*, void*);
typedef size_t (*attention8_size_fn)(const g16_attention8_args*);
typedef int (*attention8_fn)(const g16_attention8_args*, void*);
static rotary_fn g_rotary;
static cache_fn g_cache_write, g_cache_read;
static attention8_size_fn g_attention8_size;
static attention8_fn g_attention8;

static int contiguous(const tensor_t* t) {
  int64_t step = 1;
  for (int i = t->nd - 1; i >= 0; --i) {
    if (t->shape[i] > 1 && t->stride[i] != step) return 0;
    step *= t->shape[i];
  }
  return 1;
}

/* rotary(x, positions, freqs, sections, interleaved) */
static const int kGradRotary[2] = {0, 2};
static PyObject* fast_rotary(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  tensor_t x, at, f;
  g16_rotary_args a;
  void* stream;
  PyObject* out;
  int st;
  if (check_nargs("rotary", nargs, 5)) return NULL;
  if (g_ready == NULL) Py_RETURN_NONE;
  memset(&a, 0, sizeof(a));
  if (read_tensor(args[0], &x) || (x.nd != 3 && x.nd != 4) || (x.dtype != g_f16 && x.dtype != g_f32) || device_cus(x.device) <= 0 ||
      !rows_ok(&x, x.dtype == g_f32 ? 4 : 2, 0, 0) || read_tensor(args[1], &at) || at.dtype != g_i32 || at.device != x.device || !contiguous(&at) ||
      read_tensor(args[2], &f) || f.dtype != g_f32 || f.nd != 1 || f.device != x.device || !contiguous(&f) || wants_grad(args, kGradRotary, 2))
    return none_clear();
  const int64_t d = x.shape[x.nd - 1], pairs = f.shape[0];
  if (d % 8 != 0 || d <= 0 || d > G16_ROTARY_MAX_D || 2 * pairs > d) return none_clear();
  const int lead = x.nd - 2;
  int skip = 0;
  if (args[3] == Py_None) {
    a.axes = 1;
    a.sections[0] = (int)pairs;
  } else {
    int64_t parts[4], sum = 0;
    Py_INCREF(args[3]);
    if (int_tuple(args[3], parts, &a.axes) || a.axes < 1 || a.axes > G16_ROTARY_MAX_AXES) return none_clear();
    for (int i = 0; i < a.axes; ++i) {
      if (parts[i] < 0 || parts[i] > pairs) return none_clear();
      a.sections[i] = (int)parts[i];
      sum += parts[i];
    }
    if (sum != pairs) return none_clear();
    skip = 1;
  }
  if (at.nd != lead + skip || (skip && at.shape[0] != a.axes)) return none_clear();
  for (int i = 0; i < lead; ++i)
    if (at.shape[skip + i] != x.shape[i]) return none_clear();
  for (int i = 0; i < x.nd; ++i)
    if (x.shape[i] <= 0 || !fits(x.shape[i])) return none_clear();
  const int interleaved = PyObject_IsTrue(args[4]);
  if (interleaved < 0 || raw_stream(x.device, &stream)) return none_clear();
  out = empty_like(args[0]);
  if (out == NULL || (a.out = pointer_of(out)) == NULL) {
    Py_XDECREF(out);
    return none_clear();
  }
  a.x = x.ptr, a.positions = at.ptr, a.freqs = f.ptr;
  a.x_seq = lead == 2 ? x.stride[0] : 0, a.x_token = x.stride[lead - 1], a.x_head = x.stride[lead];
  a.seqs = lead == 2 ? (int)x.shape[0] : 1, a.tokens = (int)x.shape[lead - 1], a.heads = (int)x.shape[lead];
  a.d = (int)d, a.pairs = (int)pairs, a.interleaved = interleaved, a.is_f32 = x.dtype == g_f32;
  Py_BEGIN_ALLOW_THREADS
  st = g_rotary(&a, stream);
  Py_END_ALLOW_THREADS
  if (st != 0) {
    Py_DECREF(out);
    Py_RETURN_NONE;
  }
  return out;
}

/* A cache that the kernels read in place: args k_cache, v_cache, k_scale, v_scale (check_cache in cache.py); its code, 0 else */
static int cache_ok(PyObject* const* args, tensor_t* kc, tensor_t* vc, tensor_t* ks, tensor_t* vs) {
  if (read_tensor(args[0], kc) || read_tensor(args[1], vc) || read_tensor(args[2], ks) || read_tensor(args[3], vs)) return 0;
  const int code = kc->dtype == g_i8 ? G16_CODE_INT8 : kc->dtype == g_e4m3 ? G16_CODE_E4M3 : 0;
  if (code == 0 || vc->dtype != kc->dtype || kc->nd != 4 || vc->nd != 4 || ks->nd != 3 || vs->nd != 3 || ks->dtype != g_f32 || vs->dtype != g_f32 ||
      vc->device != kc->device || ks->device != kc->device || vs->device != kc->device || device_cus(kc->device) <= 0)
    return 0;
  for (int i = 0; i < 4; ++i)
    if (kc->shape[i] <= 0 || !fits(kc->shape[i]) || vc->shape[i] != kc->shape[i] || (i < 3 && (ks->shape[i] != kc->shape[i] || vs->shape[i] != kc->shape[i])))
      return 0;
  if (kc->shape[3] % 8 != 0 || kc->shape[3] > G16_ATTENTION_MAX_D || kc->stride[3] != 1 || vc->stride[3] != 1 ||
      ((kc->stride[0] | kc->stride[1] | kc->stride[2] | vc->stride[0] | vc->stride[1] | vc->stride[2]) & 7) != 0 ||
      (((uintptr_t)kc->ptr | (uintptr_t)vc->ptr) & 7) != 0 || kc->shape[0] * kc->shape[1] > INT32_MAX)
    return 0;
  return code;
}

static void cache_args(g16_cache_args* a, const tensor_t* kc, const tensor_t* vc, const tensor_t* ks, const tensor_t* vs, const tensor_t* slots,
                       int code, int is_f32) {
  memset(a, 0, sizeof(*a));
  a->k_cache = kc->ptr, a->v_cache = vc->ptr, a->k_scale = ks->ptr, a->v_scale = vs->ptr, a->slots = slots->ptr;
  a->kc_page = kc->stride[0], a->kc_token = kc->stride[1], a->kc_head = kc->stride[2];
  a->vc_page = vc->stride[0], a->vc_token = vc->stride[1], a->vc_head = vc->stride[2];
  a->ks_page = ks->stride[0], a->ks_token = ks->stride[1], a->ks_head = ks->stride[2];
  a->vs_page = vs->stride[0], a->vs_token = vs->stride[1], a->vs_head = vs->stride[2];
  a->rows = (int)slots->shape[0], a->pages = (int)kc->shape[0], a->page = (int)kc->shape[1], a->hkv = (int)kc->shape[2], a->d = (int)kc->shape[3];
  a->code = code, a->is_f32 = is_f32;
}

/* A vector of slots on a device */
static int slots_ok(PyObject* o, int device, tensor_t* t) {
  return !read_tensor(o, t) && t->dtype == g_i32 && t->nd == 1 && t->device == device && contiguous(t) && t->shape[0] > 0 && fits(t->shape[0]);
}

/* cache_write(k, v, k_cache, v_cache, k_scale, v_scale, slots): true where it is done */
static const int kGradWrite[6] = {0, 1, 2, 3, 4, 5};
static PyObject* fast_cache_write(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  tensor_t k, v, kc, vc, ks, vs, slots;
  g16_cache_args a;
  void* stream;
  int st;
  if (check_nargs("cache_write", nargs, 7)) return NULL;
  if (g_ready == NULL) Py_RETURN_NONE;
  const int code = cache_ok(args + 2, &kc, &vc, &ks, &vs);
  if (code == 0 || read_tensor(args[0], &k) || read_tensor(args[1], &v) || k.nd != 3 || v.nd != 3 || (k.dtype != g_f16 && k.dtype != g_f32) ||
      v.dtype != k.dtype || k.device != kc.device || v.device != kc.device || !slots_ok(args[6], kc.device, &slots) || wants_grad(args, kGradWrite, 6))
    return none_clear();
  const int size = k.dtype == g_f32 ? 4 : 2;
  if (k.shape[0] != slots.shape[0] || k.shape[1] != kc.shape[2] || k.shape[2] != kc.shape[3] || memcmp(k.shape, v.shape, sizeof(int64_t) * 3) != 0 ||
      !rows_ok(&k, size, 0, 0) || !rows_ok(&v, size, 0, 0))
    return none_clear();
  const tensor_t* own[4] = {&kc, &vc, &ks, &vs};
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 3; ++j)
      if (own[i]->shape[j] > 1 && own[i]->stride[j] == 0) return none_clear();
  if (raw_stream(kc.device, &stream)) return none_clear();
  cache_args(&a, &kc, &vc, &ks, &vs, &slots, code, size == 4);
  a.k = k.ptr, a.v = v.ptr;
  a.k_token = k.stride[0], a.k_head = k.stride[1], a.v_token = v.stride[0], a.v_head = v.stride[1];
  Py_BEGIN_ALLOW_THREADS
  st = g_cache_write(&a, stream);
  Py_END_ALLOW_THREADS
  if (st != 0) Py_RETURN_NONE;
  Py_RETURN_TRUE;
}

/* cache_read(k_cache, v_cache, k_scale, v_scale, slots, out_dtype) -> (k, v) */
static const int kGradRead[4] = {0, 1, 2, 3};
static PyObject* fast_cache_read(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  tensor_t kc, vc, ks, vs, slots;
  g16_cache_args a;
  void* stream;
  PyObject *k = NULL, *v = NULL, *shape = NULL, *both = NULL;
  int st = -1;
  if (check_nargs("cache_read", nargs, 6)) return NULL;
  if (g_ready == NULL) Py_RETURN_NONE;
  const int code = cache_ok(args, &kc, &vc, &ks, &vs);
  if (code == 0 || !slots_ok(args[4], kc.device, &slots) || (args[5] != g_f16 && args[5] != g_f32) || wants_grad(args, kGradRead, 4) ||
      raw_stream(kc.device, &stream))
    return none_clear();
  cache_args(&a, &kc, &vc, &ks, &vs, &slots, code, args[5] == g_f32);
  shape = Py_BuildValue("(LLL)", (long long)slots.shape[0], (long long)kc.shape[2], (long long)kc.shape[3]);
  PyObject* argv[3] = {args[2], shape, args[5]};
  if (shape != NULL) k = PyObject_VectorcallMethod(s_new_empty, argv, 2, s_dtype_names);
  if (k != NULL) v = PyObject_VectorcallMethod(s_new_empty, argv, 2, s_dtype_names);
  if (v != NULL && (a.k = pointer_of(k)) != NULL && (a.v = pointer_of(v)) != NULL) {
    Py_BEGIN_ALLOW_THREADS
    st = g_cache_read(&a, stream);
    Py_END_ALLOW_THREADS
  }
  if (st == 0) both = PyTuple_Pack(2, k, v);
  Py_XDECREF(shape);
  Py_XDECREF(k);
  Py_XDECREF(v);
  return both != NULL ? both : none_clear();
}

/* attention_decode8(q, k_cache, v_cache, lengths, pages, shared_k, shared_v, scale, softcap, slopes, k_scale, v_scale) */
static const int kGradDecode8[8] = {0, 1, 2, 5, 6, 9, 10, 11};
static PyObject* fast_attention_decode8(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  tensor_t q, kc, vc, ks, vs, t;
  g16_attention8_args e;
  void* stream;
  PyObject* out;
  int st;
  if (check_nargs("attention_decode8", nargs, 12)) return NULL;
  if (g_ready == NULL) Py_RETURN_NONE;
  memset(&e, 0, sizeof(e));
  g16_attention_args* a = &e.a;
  PyObject* const cache[4] = {args[1], args[2], args[10], args[11]};
  e.code = cache_ok(cache, &kc, &vc, &ks, &vs);
  if (e.code == 0 || read_tensor(args[0], &q) || q.nd != 3 || (q.dtype != g_f16 && q.dtype != g_f32) || q.device != kc.device || q.shape[0] <= 0 ||
      !fits(q.shape[0]) || q.shape[1] <= 0 || !fits(q.shape[1]) || q.shape[1] % kc.shape[2] != 0 || q.shape[2] != kc.shape[3] ||
      !rows_ok(&q, q.dtype == g_f32 ? 4 : 2, 0, 0) || wants_grad(args, kGradDecode8, 8) ||
      vector(args[3], g_i32, q.shape[0], q.device, (const void**)&a->lengths) || a->lengths == NULL)
    return none_clear();
  a->is_f32 = q.dtype == g_f32, a->num_cus = device_cus(q.device);
  a->seqs = (int)q.shape[0], a->q_len = 1, a->hq = (int)q.shape[1], a->hkv = (int)kc.shape[2], a->d = (int)q.shape[2];
  a->page = (int)kc.shape[1], a->num_pages = (int)kc.shape[0], a->k_len = a->page;
  if (args[4] != Py_None) {
    if (read_tensor(args[4], &t) || t.dtype != g_i32 || t.nd != 2 || t.shape[0] != a->seqs || t.device != q.device || !contiguous(&t) || t.shape[1] == 0 ||
        !fits(t.shape[1] * a->page))
      return none_clear();
    a->pages = t.ptr;
    a->max_pages = (int)t.shape[1];
    a->k_len = a->max_pages * a->page;
  } else if (kc.shape[0] != a->seqs) {
    return none_clear();
  }
  if (!rest_ok(args[7], args[8], args[5], args[6], args[9], q.device, q.dtype, a)) return none_clear();
  a->q = q.ptr, a->k = kc.ptr, a->v = vc.ptr;
  a->q_seq = q.stride[0], a->q_head = q.stride[1];
  a->k_seq = kc.stride[0], a->k_token = kc.stride[1], a->k_head = kc.stride[2];
  a->v_seq = vc.stride[0], a->v_token = vc.stride[1], a->v_head = vc.stride[2];
  e.k_scale = ks.ptr, e.v_scale = vs.ptr;
  e.ks_seq = ks.stride[0], e.ks_token = ks.stride[1], e.ks_head = ks.stride[2];
  e.vs_seq = vs.stride[0], e.vs_token = vs.stride[1], e.vs_head = vs.stride[2];
  const size_t bytes = g_attention8_size(&e);
  if (bytes > 0) {  /* (a graph has a workspace of its own) */
    PyObject* capturing = PyObject_CallNoArgs(g_capturing);
    const int plain = capturing == Py_False;
    Py_XDECREF(capturing);
    if (!plain) return none_clear();
  }
  if (raw_stream(q.device, &stream) || (bytes > 0 && scratch(q.device, stream, bytes, &a->workspace))) return none_clear();
  if (bytes > 0 && a->workspace == NULL) Py_RETURN_NONE;
  a->workspace_bytes = (int64_t)bytes;
  out = empty_like(args[0]);
  if (out == NULL || (a->out = pointer_of(out)) == NULL) {
    Py_XDECREF(out);
    return none_clear();
  }
  Py_BEGIN_ALLOW_THREADS
  st = g_attention8(&e, stream);
  Py_END_ALLOW_THREADS
  if (st != 0) {
    Py_DECREF(out);
    Py_RETURN_NONE;
  }
  return out;
}

/* bind_torch(float16, float32, int32, raw_stream(device), is_grad_enabled(), ready(device) -> compute units or
 * -1, scratch(device, stream, bytes) -> pointer, route (see product_route), [addresses of
 * g16_attention_workspace_bytes, g16_attention, g16_attention_decode_workspace_bytes, g16_attention_decode,
 * g16_mm_t_raw, g16_mm_t_direct, g16_lora_workspace_bytes, g16_lora_shrink, g16_lora_expand, g16_rotary, g16_cache_write,
 * g16_cache_read, g16_attention_decode8_workspace_bytes, g16_attention_decode8], int8, float8_e4m3fn, capturing()) */
enum { kEntryPoints = 14 };
static PyObject* fast_bind_torch(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  void* fn[kEntryPoints];
  if (check_nargs("bind_torch", nargs, 12)) return NULL;
  for (int i = 0; i < kEntryPoints; ++i) {
    PyObject* o = PySequence_GetItem(args[8], i);
    const int bad = o == NULL || as_ptr(o, &fn[i]) || check_bound(fn[i]);
    Py_XDECREF(o);
    if (bad) return NULL;
  }
  for (int i = 0; i < 2; ++i) {
    g_attention_size[i] = (attention_size_fn)fn[2 * i];
    g_attention[i] = (attention_fn)fn[2 * i + 1];
  }
  g_mm_t_raw = (raw_fn)fn[4];
  g_mm_t_direct = (direct_fn)fn[5];
  g_lora_size = (lora_size_fn)fn[6];
  g_lora_shrink = (lora_fn)fn[7];
  g_lora_expand = (lora_fn)fn[8];
  g_rotary = (rotary_fn)fn[9];
  g_cache_write = (cache_fn)fn[10];
  g_cache_read = (cache_fn)fn[11];
  g_attention8_size = (attention8_size_fn)fn[12];
  g_attention8 = (attention8_fn)fn[13];
  PyObject** to[12] = {&g_f16, &g_f32, &g_i32, &g_raw_stream, &g_grad_enabled, &g_ready, &g_scratch, &g_route, NULL, &g_i8, &g_e4m3, &g_capturing};
  for (int i = 0; i < 12; ++i) {
    if (to[i] == NULL) continue;
    Py_INCREF(args[i]);
    Py_XSETREF(*to[i], args[i]);
  }
  memset(g_device_cus, 0, sizeof(g_device_cus));
  Py_RETURN_NONE;
}

static PyMethodDef fast_methods[] = {
    {"bind", (PyCFunction)(void (*)(void))fast_bind, METH_FASTCALL,
     "bind(skinny_f32in_addr, mm_t_gemm_addr, skinny_strips_f32in_addr, skinny_addr, skinny_strips_addr)"},
    {"skinny", (PyCFunction)(void (*)(void))fast_skinny, METH_FASTCALL,
     "g16_skinny with fast argument parsing; returns its status"},
    {"skinny_strips", (PyCFunction)(void (*)(void))fast_strips, METH_FASTCALL,
     "g16_skinny_strips with fast argument parsing; returns its status"},
    {"skinny_strips_f32in", (PyCFunction)(void (*)(void))fast_strips_f32in, METH_FASTCALL,
     "g16_skinny_strips_f32in with fast argument parsing; returns its status"},
    {"skinny_f32in", (PyCFunction)(void (*)(void))fast_skinny_f32in, METH_FASTCALL,
     "g16_skinny_f32in with fast argument parsing; returns its status"},
    {"mm_t_gemm", (PyCFunction)(void (*)(void))fast_mm_t_gemm, METH_FASTCALL,
     "g16_mm_t_gemm with fast argument parsing; returns its status"},
    {"bind_torch", (PyCFunction)(void (*)(void))fast_bind_torch, METH_FASTCALL, "torch's types and the callbacks of the calls below"},
    {"attention", (PyCFunction)(void (*)(void))fast_attention, METH_FASTCALL,
     "attention for arguments that need no copy; None for any others"},
    {"attention_decode", (PyCFunction)(void (*)(void))fast_attention_decode, METH_FASTCALL,
     "attention_decode for arguments that need no copy; None for any others"},
    {"lora_mm_t", (PyCFunction)(void (*)(void))fast_lora_mm_t, METH_FASTCALL,
     "lora_mm_t for arguments that need no copy; None for any others"},
    {"rotary", (PyCFunction)(void (*)(void))fast_rotary, METH_FASTCALL, "rotary for arguments that need no copy; None for any others"},
    {"cache_write", (PyCFunction)(void (*)(void))fast_cache_write, METH_FASTCALL,
     "cache_write for arguments that need no copy; None for any others"},
    {"cache_read", (PyCFunction)(void (*)(void))fast_cache_read, METH_FASTCALL,
     "cache_read for arguments that need no copy; None for any others"},
    {"attention_decode8", (PyCFunction)(void (*)(void))fast_attention_decode8, METH_FASTCALL,
     "attention_decode over a cache in 8 bits for arguments that need no copy; None for any others"},
    {"args_size", (PyCFunction)(void (*)(void))fast_args_size, METH_FASTCALL,
     "a *_workspace_bytes entry point, by address, on a struct of arguments; returns its size"},
    {"args_call", (PyCFunction)(void (*)(void))fast_args_call, METH_FASTCALL,
     "an entry point, by address, on a struct of arguments; returns its status"},
    {"struct_call", (PyCFunction)(void (*)(void))fast_struct_call, METH_FASTCALL,
     "an entry point without workspace, by address, on a struct of arguments; returns its status"},
    {NULL, NULL, 0, NULL},
};

static struct PyModuleDef fast_module = {PyModuleDef_HEAD_INIT, "_g16fast", NULL, -1, fast_methods,
                                         NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__g16fast(void) {
  s_dtype = PyUnicode_InternFromString("dtype");
  s_shape = PyUnicode_InternFromString("shape");
  s_stride = PyUnicode_InternFromString("stride");
  s_data_ptr = PyUnicode_InternFromString("data_ptr");
  s_get_device = PyUnicode_InternFromString("get_device");
  s_requires_grad = PyUnicode_InternFromString("requires_grad");
  s_new_empty = PyUnicode_InternFromString("new_empty");
  s_dtype_names = PyTuple_Pack(1, s_dtype);
  return PyModule_Create(&fast_module);
}
