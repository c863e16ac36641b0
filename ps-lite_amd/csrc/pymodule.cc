// The per-request half of the Python binding (ps-lite_amd/capi.py) as a CPython extension.
//
// A request from Python is a few checks on its arrays and one call of the C ABI. Through ctypes the
// checks cost more than the call: 1.7 us for the address of a numpy array, 3.4 us to wait for torch's
// current stream, 4.7 us of the 8.9 us of a device-resident push of 1,000 keys. Every function here
// takes the arrays themselves and returns None when one of them is not what the quick way takes (a list, another
// dtype, a non-contiguous array): capi.py then goes its general way, which converts or refuses it.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <hip/hip_runtime_api.h>
#define NPY_NO_DEPRECATED_API NPY_1_7_API_VERSION
#include <numpy/arrayobject.h>
#include <stdint.h>

#include <initializer_list>

#include "pskv/capi.h"

namespace {

// set once by setup(): torch's types, null when torch is not there
PyObject* g_tensor_type = nullptr;
PyObject *g_int64 = nullptr, *g_uint64 = nullptr, *g_float32 = nullptr, *g_int32 = nullptr;
PyObject* g_raw_stream = nullptr;  // callable: device index -> hipStream_t of torch's current stream, as an int
PyObject *g_float16 = nullptr, *g_bfloat16 = nullptr;
PyObject *s_dtype, *s_is_cuda, *s_is_contiguous, *s_numel, *s_data_ptr, *s_shape, *s_stride, *s_get_device, *s_nbytes;

enum Kind { kNone = -1, kHost = PSKV_MEM_HOST, kDevice = PSKV_MEM_DEVICE };

// One array argument. `type`: 'k' keys (64-bit), 'f' float32, 'i' int32.
class Arg {
 public:
  ~Arg() {
    if (viewed_) PyBuffer_Release(&view_);
  }
  // 1 taken, 0 not for the quick way, -1 a Python error is set
  int take(PyObject* o, char type) {
    if (o == Py_None) return 1;
    // (a numpy array is looked at itself: its buffer costs 50 ns to ask for and to give back, and a slice of a request has six.
    // The caller's arguments keep it.)
    if (PyArray_CheckExact(o)) return array(reinterpret_cast<PyArrayObject*>(o), type);
    if (g_tensor_type && PyObject_TypeCheck(o, reinterpret_cast<PyTypeObject*>(g_tensor_type))) return tensor(o, type);
    if (!PyObject_CheckBuffer(o)) return 0;
    if (PyObject_GetBuffer(o, &view_, PyBUF_C_CONTIGUOUS | PyBUF_FORMAT) != 0) {
      PyErr_Clear();
      return 0;
    }
    viewed_ = true;
    const char* f = view_.format;
    if (!f || f[0] == 0 || f[1] != 0) return 0;
    const bool fits = type == 'k'   ? (f[0] == 'L' || f[0] == 'Q') && view_.itemsize == 8
                      : type == 'f' ? f[0] == 'f' && view_.itemsize == 4
                                    : f[0] == 'i' && view_.itemsize == 4;
    if (!fits) return 0;
    n = (size_t)(view_.len / view_.itemsize);
    ptr = n ? view_.buf : nullptr;
    kind = kHost;
    return 1;
  }
  void* ptr = nullptr;
  size_t n = 0;
  int kind = kNone;
  PyObject* device_tensor = nullptr;  // borrowed

 private:
  int array(PyArrayObject* a, char type) {
    const int t = PyArray_TYPE(a);
    const bool fits = type == 'k'   ? t == NPY_ULONG || t == NPY_ULONGLONG
                      : type == 'f' ? t == NPY_FLOAT
                                    : t == NPY_INT;
    if (!fits || !PyArray_IS_C_CONTIGUOUS(a) || !PyArray_ISALIGNED(a) || !PyArray_ISNOTSWAPPED(a)) return 0;
    n = (size_t)PyArray_SIZE(a);
    ptr = n ? PyArray_DATA(a) : nullptr;
    kind = kHost;
    return 1;
  }
  int tensor(PyObject* o, char type) {
    PyObject* d = PyObject_GetAttr(o, s_dtype);
    if (!d) return -1;
    Py_DECREF(d);  // (dtypes live as long as torch does)
    const bool fits = type == 'k' ? d == g_int64 || d == g_uint64 : type == 'f' ? d == g_float32 : d == g_int32;
    if (!fits) return 0;
    PyObject* c = PyObject_CallMethodNoArgs(o, s_is_contiguous);
    if (!c) return -1;
    Py_DECREF(c);
    if (c != Py_True) return 0;
    PyObject* cuda = PyObject_GetAttr(o, s_is_cuda);
    if (!cuda) return -1;
    Py_DECREF(cuda);
    PyObject* count = PyObject_CallMethodNoArgs(o, s_numel);
    if (!count) return -1;
    n = PyLong_AsSize_t(count);
    Py_DECREF(count);
    if (n) {
      PyObject* p = PyObject_CallMethodNoArgs(o, s_data_ptr);
      if (!p) return -1;
      ptr = PyLong_AsVoidPtr(p);
      Py_DECREF(p);
    }
    if (PyErr_Occurred()) return -1;
    kind = cuda == Py_True ? kDevice : kHost;
    if (kind == kDevice) device_tensor = o;
    return 1;
  }
  Py_buffer view_;
  bool viewed_ = false;
};

// The C ABI wants device buffers complete before the call; torch fills and copies tensors on its current
// stream, which is waited for here. false: a Python error is set.
bool torch_is_done() {
  int device = 0;
  if (!g_raw_stream || hipGetDevice(&device) != hipSuccess) return true;
  PyObject* at = PyLong_FromLong(device);
  if (!at) return false;
  PyObject* raw = PyObject_CallOneArg(g_raw_stream, at);
  Py_DECREF(at);
  if (!raw) return false;
  void* stream = PyLong_AsVoidPtr(raw);
  Py_DECREF(raw);
  if (!stream && PyErr_Occurred()) return false;
  hipError_t e;
  Py_BEGIN_ALLOW_THREADS;
  e = hipStreamSynchronize(static_cast<hipStream_t>(stream));
  Py_END_ALLOW_THREADS;
  if (e != hipSuccess) {
    PyErr_Format(PyExc_RuntimeError, "waiting for torch's stream: %s", hipGetErrorString(e));
    return false;
  }
  return true;
}

// Takes `count` arrays of the given types; what they agree on goes to *kind. Device tensors are appended to `held`
// (a list, or None), which keeps them until the next wait. 1, 0 or -1 as Arg::take.
int take_all(Arg* args, PyObject* const* objects, const char* types, int count, PyObject* held, int* kind) {
  int k = kNone;
  for (int i = 0; i < count; ++i) {
    const int r = args[i].take(objects[i], types[i]);
    if (r != 1) return r;
    if (args[i].kind == kNone) continue;
    if (k != kNone && k != args[i].kind) return 0;
    k = args[i].kind;
  }
  *kind = k == kNone ? (int)kHost : k;
  if (*kind == kDevice) {
    if (!torch_is_done()) return -1;
    if (held != Py_None)
      for (int i = 0; i < count; ++i)
        if (args[i].device_tensor && PyList_Append(held, args[i].device_tensor) != 0) return -1;
  }
  return 1;
}

#define NOT_QUICK(r)                 \
  do {                               \
    const int r_ = (r);              \
    if (r_ < 0) return nullptr;      \
    if (r_ == 0) Py_RETURN_NONE;     \
  } while (0)

bool want(Py_ssize_t got, Py_ssize_t n) {
  if (got == n) return true;
  PyErr_Format(PyExc_TypeError, "%zd arguments expected, %zd given", n, got);
  return false;
}

// a status, or, for the calls that answer a size: the size when the status is 0, else (status, size)
PyObject* sized(int rc, size_t got) {
  if (rc == PSKV_OK) return PyLong_FromSize_t(got);
  return Py_BuildValue("(in)", rc, (Py_ssize_t)got);
}

// table_push(table, keys, vals, lens, held)
PyObject* table_push(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!want(n, 5)) return nullptr;
  pskv_table* t = static_cast<pskv_table*>(PyLong_AsVoidPtr(a[0]));
  if (PyErr_Occurred()) return nullptr;
  Arg x[3];
  int kind, rc;
  NOT_QUICK(take_all(x, a + 1, "kfi", 3, a[4], &kind));
  Py_BEGIN_ALLOW_THREADS;
  rc = pskv_push(t, static_cast<uint64_t*>(x[0].ptr), x[0].n, static_cast<float*>(x[1].ptr), x[1].n,
                 static_cast<int32_t*>(x[2].ptr), x[2].n, kind);
  Py_END_ALLOW_THREADS;
  return PyLong_FromLong(rc);
}

// table_pull(table, keys, out, out_lens, held)
PyObject* table_pull(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!want(n, 5)) return nullptr;
  pskv_table* t = static_cast<pskv_table*>(PyLong_AsVoidPtr(a[0]));
  if (PyErr_Occurred()) return nullptr;
  Arg x[3];
  int kind, rc;
  size_t got = 0;
  NOT_QUICK(take_all(x, a + 1, "kfi", 3, a[4], &kind));
  Py_BEGIN_ALLOW_THREADS;
  rc = pskv_pull(t, static_cast<uint64_t*>(x[0].ptr), x[0].n, static_cast<float*>(x[1].ptr), x[1].n,
                 static_cast<int32_t*>(x[2].ptr), &got, kind);
  Py_END_ALLOW_THREADS;
  return sized(rc, got);
}

// table_pushpull(table, keys, vals, lens, out, out_lens, held)
PyObject* table_pushpull(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!want(n, 7)) return nullptr;
  pskv_table* t = static_cast<pskv_table*>(PyLong_AsVoidPtr(a[0]));
  if (PyErr_Occurred()) return nullptr;
  Arg x[5];
  int kind, rc;
  size_t got = 0;
  NOT_QUICK(take_all(x, a + 1, "kfifi", 5, a[6], &kind));
  Py_BEGIN_ALLOW_THREADS;
  rc = pskv_pushpull(t, static_cast<uint64_t*>(x[0].ptr), x[0].n, static_cast<float*>(x[1].ptr), x[1].n,
                     static_cast<int32_t*>(x[2].ptr), x[2].n, static_cast<float*>(x[3].ptr), x[3].n,
                     static_cast<int32_t*>(x[4].ptr), &got, kind);
  Py_END_ALLOW_THREADS;
  return sized(rc, got);
}

// The tables of a group and the positions that its calls share: host arrays of S+1 entries (None: null).
struct GroupArgs {
  pskv_table* const* tables;
  size_t S;
  bool parse(PyObject* tables_at, PyObject* count) {
    tables = static_cast<pskv_table* const*>(PyLong_AsVoidPtr(tables_at));
    S = PyLong_AsSize_t(count);
    return !PyErr_Occurred();
  }
  // 1 / 0 / -1: a host array with at least S + 1 entries
  int positions(Arg* p, PyObject* o) {
    const int r = p->take(o, 'k');
    if (r != 1) return r;
    return p->kind == kNone || (p->kind == kHost && p->n >= S + 1) ? 1 : 0;
  }
};

// Every tensor of a group's call lives on the device.
int on_device(const Arg* x, int count) {
  for (int i = 0; i < count; ++i)
    if (x[i].kind == kHost) return 0;
  return 1;
}

// group_push(tables, S, keys, vals, lens, pos, val_pos, held)
PyObject* group_push(PyObject*, PyObject* const* a, Py_ssize_t n) {
  GroupArgs g;
  if (!want(n, 8) || !g.parse(a[0], a[1])) return nullptr;
  Arg x[3], pos, val_pos;
  int kind, rc;
  NOT_QUICK(g.positions(&pos, a[5]));
  NOT_QUICK(g.positions(&val_pos, a[6]));
  NOT_QUICK(take_all(x, a + 2, "kfi", 3, a[7], &kind));
  NOT_QUICK(on_device(x, 3));
  Py_BEGIN_ALLOW_THREADS;
  rc = pskv_push_multi(g.tables, g.S, static_cast<uint64_t*>(x[0].ptr), static_cast<uint64_t*>(pos.ptr),
                       static_cast<float*>(x[1].ptr), static_cast<uint64_t*>(val_pos.ptr),
                       static_cast<int32_t*>(x[2].ptr), PSKV_MEM_DEVICE);
  Py_END_ALLOW_THREADS;
  return PyLong_FromLong(rc);
}

// group_pull(tables, S, keys, out, out_lens, pos, out_pos, sizes, held)
PyObject* group_pull(PyObject*, PyObject* const* a, Py_ssize_t n) {
  GroupArgs g;
  if (!want(n, 9) || !g.parse(a[0], a[1])) return nullptr;
  Arg x[3], pos, out_pos, sizes;
  int kind, rc;
  NOT_QUICK(g.positions(&pos, a[5]));
  NOT_QUICK(g.positions(&out_pos, a[6]));
  NOT_QUICK(sizes.take(a[7], 'k'));
  NOT_QUICK(take_all(x, a + 2, "kfi", 3, a[8], &kind));
  NOT_QUICK(on_device(x, 3));
  Py_BEGIN_ALLOW_THREADS;
  rc = pskv_pull_multi(g.tables, g.S, static_cast<uint64_t*>(x[0].ptr), static_cast<uint64_t*>(pos.ptr),
                       static_cast<float*>(x[1].ptr), static_cast<uint64_t*>(out_pos.ptr),
                       static_cast<int32_t*>(x[2].ptr), static_cast<uint64_t*>(sizes.ptr), PSKV_MEM_DEVICE);
  Py_END_ALLOW_THREADS;
  return PyLong_FromLong(rc);
}

// group_pushpull(tables, S, keys, vals, lens, out, out_lens, pos, val_pos, out_pos, sizes, held)
PyObject* group_pushpull(PyObject*, PyObject* const* a, Py_ssize_t n) {
  GroupArgs g;
  if (!want(n, 12) || !g.parse(a[0], a[1])) return nullptr;
  Arg x[5], pos, val_pos, out_pos, sizes;
  int kind, rc;
  NOT_QUICK(g.positions(&pos, a[7]));
  NOT_QUICK(g.positions(&val_pos, a[8]));
  NOT_QUICK(g.positions(&out_pos, a[9]));
  NOT_QUICK(sizes.take(a[10], 'k'));
  NOT_QUICK(take_all(x, a + 2, "kfifi", 5, a[11], &kind));
  NOT_QUICK(on_device(x, 5));
  Py_BEGIN_ALLOW_THREADS;
  rc = pskv_pushpull_multi(g.tables, g.S, static_cast<uint64_t*>(x[0].ptr), static_cast<uint64_t*>(pos.ptr),
                           static_cast<float*>(x[1].ptr), static_cast<uint64_t*>(val_pos.ptr),
                           static_cast<int32_t*>(x[2].ptr), static_cast<float*>(x[3].ptr),
                           static_cast<uint64_t*>(out_pos.ptr), static_cast<int32_t*>(x[4].ptr),
                           static_cast<uint64_t*>(sizes.ptr), PSKV_MEM_DEVICE);
  Py_END_ALLOW_THREADS;
  return PyLong_FromLong(rc);
}

// slice(device, keys, lens, nvals, range_begin, range_end): (pos, val_pos, used), or a status
PyObject* slice(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!want(n, 6)) return nullptr;
  const long device = PyLong_AsLong(a[0]);
  const size_t nvals = PyLong_AsSize_t(a[3]);
  if (PyErr_Occurred()) {  // (a numpy integer, say)
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  Arg x[2], begin, end;
  int kind, rc;
  NOT_QUICK(begin.take(a[4], 'k'));
  NOT_QUICK(end.take(a[5], 'k'));
  const size_t S = begin.n;
  if (begin.kind != kHost || end.kind != kHost || end.n != S) Py_RETURN_NONE;
  NOT_QUICK(take_all(x, a + 1, "ki", 2, Py_None, &kind));
  npy_intp bounds = (npy_intp)S + 1, ranges = (npy_intp)S;
  PyObject* pos = PyArray_SimpleNew(1, &bounds, NPY_UINT64);
  PyObject* val_pos = PyArray_SimpleNew(1, &bounds, NPY_UINT64);
  PyObject* used = PyArray_SimpleNew(1, &ranges, NPY_UINT8);
  PyObject* result = nullptr;
  if (pos && val_pos && used) {
    uint64_t* p = static_cast<uint64_t*>(PyArray_DATA(reinterpret_cast<PyArrayObject*>(pos)));
    uint64_t* v = static_cast<uint64_t*>(PyArray_DATA(reinterpret_cast<PyArrayObject*>(val_pos)));
    uint8_t* u = static_cast<uint8_t*>(PyArray_DATA(reinterpret_cast<PyArrayObject*>(used)));
    Py_BEGIN_ALLOW_THREADS;
    rc = pskv_slice((int)device, static_cast<uint64_t*>(x[0].ptr), x[0].n, static_cast<int32_t*>(x[1].ptr), x[1].n,
                    nvals, static_cast<uint64_t*>(begin.ptr), static_cast<uint64_t*>(end.ptr), S, p, v, u, kind);
    Py_END_ALLOW_THREADS;
    result = rc ? PyLong_FromLong(rc) : PyTuple_Pack(3, pos, val_pos, used);
  }
  Py_XDECREF(pos);
  Py_XDECREF(val_pos);
  Py_XDECREF(used);
  return result;
}

// match(device, src_keys, src_vals, dst_keys, dst_vals, k, op)
PyObject* match(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!want(n, 7)) return nullptr;
  const long device = PyLong_AsLong(a[0]), op = PyLong_AsLong(a[6]);
  const size_t k = PyLong_AsSize_t(a[5]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  Arg x[4];
  int kind, rc;
  uint64_t got = 0;
  NOT_QUICK(take_all(x, a + 1, "kfkf", 4, Py_None, &kind));
  if (x[1].n != x[0].n * k || x[3].n != x[2].n * k) Py_RETURN_NONE;
  Py_BEGIN_ALLOW_THREADS;
  rc = pskv_match((int)device, static_cast<uint64_t*>(x[0].ptr), x[0].n, static_cast<float*>(x[1].ptr),
                  static_cast<uint64_t*>(x[2].ptr), x[2].n, static_cast<float*>(x[3].ptr), k, (int)op, &got, nullptr,
                  kind);
  Py_END_ALLOW_THREADS;
  return sized(rc, got);
}

// replay_run(recording)
PyObject* replay_run(PyObject*, PyObject* at) {
  pskv_replay* r = static_cast<pskv_replay*>(PyLong_AsVoidPtr(at));
  if (PyErr_Occurred()) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS;
  rc = pskv_replay_run(r);
  Py_END_ALLOW_THREADS;
  return PyLong_FromLong(rc);
}

// --- operators on rows --------------------------------------------------------------------------------------------------------
// These check their tensors here, once, and refuse what the calls do not take with TypeError or ValueError.

constexpr int kNoType = -1, kInt32 = 100, kInt64 = 101, kMemory = 102;  // beside PSKV_F32, PSKV_F16, PSKV_BF16

// A tensor on a GPU, as the calls see it.
struct Tensor {
  const char* name;
  void* ptr = nullptr;
  int type = kNoType, dims = 0, device = -1;
  int64_t n[4] = {1, 1, 1, 1}, by[4] = {0, 0, 0, 0};
  explicit Tensor(const char* what) : name(what) {}
  bool given() const { return type != kNoType; }
  int64_t count() const { return n[0] * n[1] * n[2] * n[3]; }
  // (torch leaves the strides of dimensions of one element to chance)
  size_t stride(int d, int64_t if_one) const { return (size_t)(n[d] > 1 ? by[d] : if_one); }

  bool fail(PyObject* error, const char* what) const {
    PyErr_Format(error, "%s: %s", name, what);
    return false;
  }
  bool take(PyObject* o, bool may_be_none = false) {
    if (may_be_none && o == Py_None) return true;
    if (!g_tensor_type || !PyObject_TypeCheck(o, reinterpret_cast<PyTypeObject*>(g_tensor_type)))
      return fail(PyExc_TypeError, "a torch tensor is expected");
    PyObject* at = PyObject_CallMethodNoArgs(o, s_get_device);
    if (!at) return false;
    device = (int)PyLong_AsLong(at);
    Py_DECREF(at);
    if (PyErr_Occurred()) return false;
    if (device < 0) return fail(PyExc_ValueError, "the tensor is not on the GPU");
    PyObject* d = PyObject_GetAttr(o, s_dtype);
    if (!d) return false;
    Py_DECREF(d);
    type = d == g_float32 ? PSKV_F32 : d == g_float16 ? PSKV_F16 : d == g_bfloat16 ? PSKV_BF16 : d == g_int32 ? kInt32
           : d == g_int64 || d == g_uint64 ? kInt64 : kNoType;
    if (type == kNoType) return fail(PyExc_TypeError, "not a type that a call takes");
    PyObject* shape = PyObject_GetAttr(o, s_shape);
    if (!shape) return false;
    PyObject* steps = PyObject_CallMethodNoArgs(o, s_stride);
    bool ok = steps && PyTuple_Check(shape) && PyTuple_Check(steps) && PyTuple_GET_SIZE(shape) == PyTuple_GET_SIZE(steps);
    if (ok) {
      dims = (int)PyTuple_GET_SIZE(shape);
      for (int i = 0; i < dims && i < 4; ++i) {
        n[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, i));
        by[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(steps, i));
      }
    }
    Py_DECREF(shape);
    Py_XDECREF(steps);
    if (PyErr_Occurred()) return false;
    if (!ok || dims > 4) return fail(PyExc_ValueError, "a tensor with up to four dimensions is expected");
    if (count() > 0) {
      PyObject* p = PyObject_CallMethodNoArgs(o, s_data_ptr);
      if (!p) return false;
      ptr = PyLong_AsVoidPtr(p);
      Py_DECREF(p);
      if (PyErr_Occurred()) return false;
    }
    return true;
  }
  // working memory, of any type; n[0]: bytes
  bool take_memory(PyObject* o) {
    if (o == Py_None) return true;
    if (!g_tensor_type || !PyObject_TypeCheck(o, reinterpret_cast<PyTypeObject*>(g_tensor_type)))
      return fail(PyExc_TypeError, "a torch tensor is expected");
    PyObject* at = PyObject_CallMethodNoArgs(o, s_get_device);
    PyObject* is = at ? PyObject_CallMethodNoArgs(o, s_is_contiguous) : nullptr;
    PyObject* size = is ? PyObject_GetAttr(o, s_nbytes) : nullptr;
    PyObject* p = size ? PyObject_CallMethodNoArgs(o, s_data_ptr) : nullptr;
    if (p) {
      device = (int)PyLong_AsLong(at);
      n[0] = PyLong_AsLongLong(size);
      ptr = PyLong_AsVoidPtr(p);
      type = kMemory;
    }
    const bool whole = is == Py_True;
    Py_XDECREF(at);
    Py_XDECREF(is);
    Py_XDECREF(size);
    Py_XDECREF(p);
    if (PyErr_Occurred()) return false;
    if (device < 0) return fail(PyExc_ValueError, "the tensor is not on the GPU");
    return whole || fail(PyExc_ValueError, "the tensor is not contiguous");
  }
  bool has_type(int t) const { return type == t || fail(PyExc_TypeError, t == PSKV_F32 ? "float32 is expected" : "int32 is expected"); }
  bool is_rows_type() const {
    return type == PSKV_F32 || type == PSKV_F16 || type == PSKV_BF16 || fail(PyExc_TypeError, "float32, float16 or bfloat16 is expected");
  }
  bool dense() const {
    int64_t want = 1;
    for (int d = dims; d-- > 0;) {
      if (n[d] > 1 && by[d] != want && count() > 0) return fail(PyExc_ValueError, "the tensor is not contiguous");
      want *= n[d];
    }
    return true;
  }
  // [n, k] with the elements of a row side by side
  bool is_matrix() const {
    if (dims != 2) return fail(PyExc_ValueError, "a matrix is expected");
    if (n[1] > 1 && by[1] != 1 && count() > 0) return fail(PyExc_ValueError, "the elements of a row do not lie side by side");
    return true;
  }
  bool like(const Tensor& o) const {
    if (type != o.type) return fail(PyExc_TypeError, "not of the type of the other rows");
    return true;
  }
  bool sized(int64_t rows, int64_t k) const {
    return (dims == 2 && n[0] == rows && n[1] == k) || fail(PyExc_ValueError, "its shape does not fit the other tensors'");
  }
};

// A whole number (a numpy one, too). false: a Python error is set.
bool whole_number(PyObject* o, unsigned long long* to) {
  PyObject* i = PyNumber_Index(o);
  if (!i) return false;
  *to = PyLong_AsUnsignedLongLong(i);
  Py_DECREF(i);
  return !PyErr_Occurred();
}
bool whole_number(PyObject* o, long long* to) {
  PyObject* i = PyNumber_Index(o);
  if (!i) return false;
  *to = PyLong_AsLongLong(i);
  Py_DECREF(i);
  return !PyErr_Occurred();
}

// All on one device.
bool together(std::initializer_list<const Tensor*> all, int* device) {
  *device = -1;
  for (const Tensor* t : all) {
    if (!t->given()) continue;
    if (*device >= 0 && t->device != *device) return t->fail(PyExc_ValueError, "the tensors of a call lie on one device");
    *device = t->device;
  }
  return true;
}

// The stream of a call: an address, or None for torch's current one on the tensors' device.
bool stream_of(PyObject* o, int device, void** stream) {
  if (o != Py_None) {
    *stream = PyLong_AsVoidPtr(o);
    return *stream || !PyErr_Occurred();
  }
  PyObject* at = PyLong_FromLong(device);
  PyObject* raw = at ? PyObject_CallOneArg(g_raw_stream, at) : nullptr;
  Py_XDECREF(at);
  if (!raw) return false;
  *stream = PyLong_AsVoidPtr(raw);
  Py_DECREF(raw);
  return *stream || !PyErr_Occurred();
}

#define NEED(x) \
  do {          \
    if (!(x)) return nullptr; \
  } while (0)

// A place of every choice of every token.
bool is_places(const Tensor& place) {
  return place.has_type(kInt32) && (place.dims == 2 || place.fail(PyExc_ValueError, "[tokens, choices] is expected")) && place.dense();
}

// [tokens, choices] of float32
bool is_weights(const Tensor& w, const Tensor& place) {
  return w.has_type(PSKV_F32) && w.sized(place.n[0], place.n[1]) && w.dense();
}

// Working memory of a call that was not given any, from allocate(bytes, a tensor of the call, stream); kept until the call has been
// enqueued.
class Room {
 public:
  ~Room() { Py_XDECREF(held_); }
  bool take(Tensor& work, size_t bytes, PyObject* allocate, PyObject* like, PyObject* stream) {
    if (work.given() || bytes == 0) return true;
    PyObject* size = PyLong_FromSize_t(bytes);
    if (!size) return false;
    PyObject* args[] = {size, like, stream};
    held_ = PyObject_Vectorcall(allocate, args, 3, nullptr);
    Py_DECREF(size);
    return held_ && work.take_memory(held_);
  }

 private:
  PyObject* held_ = nullptr;
};

// route_sort(experts, E, order, place, offsets, work, stream, allocate)
PyObject* route_sort(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NEED(want(n, 8));
  Tensor experts("experts"), order("order"), place("place"), offsets("offsets"), work("work");
  unsigned long long E;
  NEED(whole_number(a[1], &E));
  NEED(experts.take(a[0]) && order.take(a[2]) && place.take(a[3]) && offsets.take(a[4]) && work.take_memory(a[5]));
  if (experts.type != kInt32 && experts.type != kInt64) NEED(experts.fail(PyExc_TypeError, "int32 or int64 is expected"));
  NEED(experts.dense() && order.has_type(kInt32) && order.dense() && place.has_type(kInt32) && place.dense() &&
       offsets.has_type(kInt32) && offsets.dense());
  const int64_t count = experts.count();
  if (order.count() != count) NEED(order.fail(PyExc_ValueError, "as many entries as experts has are expected"));
  if (place.count() != count) NEED(place.fail(PyExc_ValueError, "as many entries as experts has are expected"));
  if ((uint64_t)offsets.count() != (uint64_t)E + 1) NEED(offsets.fail(PyExc_ValueError, "E + 1 entries are expected"));
  int device;
  void* stream;
  NEED(together({&experts, &order, &place, &offsets, &work}, &device) && stream_of(a[6], device, &stream));
  Room room;
  NEED(room.take(work, pskv_route_room((size_t)count, E), a[7], a[0], a[6]));
  int rc;
  Py_BEGIN_ALLOW_THREADS;
  rc = pskv_route_sort(device, stream, experts.ptr, experts.type == kInt64 ? 64 : 32, (size_t)count, E,
                       static_cast<int32_t*>(order.ptr), static_cast<int32_t*>(place.ptr), static_cast<int32_t*>(offsets.ptr),
                       work.ptr, work.given() ? (size_t)work.n[0] : 0);
  Py_END_ALLOW_THREADS;
  return PyLong_FromLong(rc);
}

// route_rows(x, place, rows, stream)
PyObject* route_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NEED(want(n, 4));
  Tensor x("x"), place("place"), rows("rows");
  NEED(x.take(a[0]) && place.take(a[1]) && rows.take(a[2]) && x.is_rows_type() && x.is_matrix() && is_places(place) &&
       rows.like(x) && rows.is_matrix() && rows.sized(rows.n[0], x.n[1]));
  if (place.n[0] != x.n[0]) NEED(place.fail(PyExc_ValueError, "its shape does not fit the other tensors'"));
  int device, rc;
  void* stream;
  NEED(together({&x, &place, &rows}, &device) && stream_of(a[3], device, &stream));
  Py_BEGIN_ALLOW_THREADS;
  rc = pskv_route_rows(device, stream, x.type, x.ptr, x.stride(0, x.n[1]), (size_t)x.n[0], (size_t)x.n[1],
                       static_cast<int32_t*>(place.ptr), (size_t)place.n[1], rows.ptr, rows.stride(0, rows.n[1]), (size_t)rows.n[0]);
  Py_END_ALLOW_THREADS;
  return PyLong_FromLong(rc);
}

// route_sum(rows, place, out, weights, stream)
PyObject* route_sum(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NEED(want(n, 5));
  Tensor rows("rows"), place("place"), out("out"), weights("weights");
  NEED(rows.take(a[0]) && place.take(a[1]) && out.take(a[2]) && weights.take(a[3], true) && rows.is_rows_type() &&
       rows.is_matrix() && is_places(place) && out.like(rows) && out.is_matrix() && out.sized(place.n[0], rows.n[1]));
  NEED(!weights.given() || is_weights(weights, place));
  int device, rc;
  void* stream;
  NEED(together({&rows, &place, &out, &weights}, &device) && stream_of(a[4], device, &stream));
  Py_BEGIN_ALLOW_THREADS;
  rc = pskv_route_sum(device, stream, rows.type, rows.ptr, rows.stride(0, rows.n[1]), (size_t)rows.n[0],
                      static_cast<int32_t*>(place.ptr), static_cast<float*>(weights.ptr), (size_t)place.n[1], out.ptr,
                      out.stride(0, out.n[1]), (size_t)out.n[0], (size_t)out.n[1]);
  Py_END_ALLOW_THREADS;
  return PyLong_FromLong(rc);
}

// route_sum_grad(grad, rows, place, weights, grad_rows, grad_weights, stream)
PyObject* route_sum_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NEED(want(n, 7));
  Tensor grad("grad"), rows("rows"), place("place"), weights("weights"), grad_rows("grad_rows"), grad_weights("grad_weights");
  NEED(grad.take(a[0]) && rows.take(a[1]) && place.take(a[2]) && weights.take(a[3]) && grad_rows.take(a[4]) &&
       grad_weights.take(a[5]));
  NEED(grad.is_rows_type() && grad.is_matrix() && is_places(place) && is_weights(weights, place) &&
       is_weights(grad_weights, place) && rows.like(grad) && rows.is_matrix() && grad_rows.like(grad) && grad_rows.is_matrix() &&
       rows.sized(rows.n[0], grad.n[1]) && grad_rows.sized(rows.n[0], grad.n[1]) && grad.sized(place.n[0], grad.n[1]));
  int device, rc;
  void* stream;
  NEED(together({&grad, &rows, &place, &weights, &grad_rows, &grad_weights}, &device) && stream_of(a[6], device, &stream));
  Py_BEGIN_ALLOW_THREADS;
  rc = pskv_route_sum_grad(device, stream, grad.type, grad.ptr, grad.stride(0, grad.n[1]), (size_t)grad.n[0], (size_t)grad.n[1],
                           rows.ptr, rows.stride(0, rows.n[1]), (size_t)rows.n[0], static_cast<int32_t*>(place.ptr),
                           static_cast<float*>(weights.ptr), (size_t)place.n[1], grad_rows.ptr,
                           grad_rows.stride(0, grad_rows.n[1]), static_cast<float*>(grad_weights.ptr));
  Py_END_ALLOW_THREADS;
  return PyLong_FromLong(rc);
}

// [batch, heads, queries, keys], or without the batch
struct Scores {
  size_t n[4];
  int64_t by[3];
  bool parse(const Tensor& t) {
    if (t.dims != 3 && t.dims != 4) return t.fail(PyExc_ValueError, "[heads, queries, keys] with or without a batch is expected");
    const int o = t.dims - 4;
    for (int d = 0; d < 4; ++d) n[d] = d + o < 0 ? 1 : (size_t)t.n[d + o];
    for (int d = 0; d < 3; ++d) by[d] = d + o < 0 || t.n[d + o] < 2 ? 0 : t.by[d + o];
    if (n[3] > 1 && t.by[3 + o] != 1 && t.count() > 0) return t.fail(PyExc_ValueError, "the keys of a query do not lie side by side");
    return true;
  }
};

bool is_positions(const Tensor& at, size_t batch) {
  if (!at.given()) return true;
  if (at.type != kInt64) return at.fail(PyExc_TypeError, "int64 is expected");
  if (at.dims != 1 || (size_t)at.n[0] != batch) return at.fail(PyExc_ValueError, "a position for each of the batch is expected");
  return at.dense();
}

// relbias(table, out, max_distance, two_sided, scores, q_first, k_first, q_at, stream)
PyObject* relbias(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NEED(want(n, 9));
  Tensor table("table"), out("out"), scores("scores"), at("q_at");
  unsigned long long far;
  long long q_first, k_first;
  const int two_sided = PyObject_IsTrue(a[3]);
  NEED(two_sided >= 0 && whole_number(a[2], &far) && whole_number(a[5], &q_first) && whole_number(a[6], &k_first));
  NEED(table.take(a[0]) && out.take(a[1]) && scores.take(a[4], true) && at.take(a[7], true) && table.has_type(PSKV_F32) &&
       table.dense() && out.is_rows_type());
  if (table.dims != 2) NEED(table.fail(PyExc_ValueError, "[buckets, heads] is expected"));
  Scores o, s{};
  NEED(o.parse(out) && is_positions(at, o.n[0]));
  if ((size_t)table.n[1] != o.n[1]) NEED(table.fail(PyExc_ValueError, "a column for each head is expected"));
  if (scores.given()) {
    NEED(scores.like(out) && s.parse(scores));
    bool same = scores.dims == out.dims;
    for (int d = 0; d < 4; ++d) same = same && s.n[d] == o.n[d];
    if (!same) NEED(scores.fail(PyExc_ValueError, "the shape of out is expected"));
  }
  int device, rc;
  void* stream;
  NEED(together({&table, &out, &scores, &at}, &device) && stream_of(a[8], device, &stream));
  Py_BEGIN_ALLOW_THREADS;
  rc = pskv_relbias(device, stream, out.type, static_cast<float*>(table.ptr), (size_t)table.n[0], o.n[1], far, two_sided, q_first,
                    k_first, static_cast<int64_t*>(at.ptr), scores.ptr, s.by, out.ptr, o.by, o.n[0], o.n[2], o.n[3]);
  Py_END_ALLOW_THREADS;
  return PyLong_FromLong(rc);
}

// relbias_grad(grad, grad_table, max_distance, two_sided, q_first, k_first, q_at, work, stream, allocate)
PyObject* relbias_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NEED(want(n, 10));
  Tensor grad("grad"), grad_table("grad_table"), at("q_at"), work("work");
  unsigned long long far;
  long long q_first, k_first;
  const int two_sided = PyObject_IsTrue(a[3]);
  NEED(two_sided >= 0 && whole_number(a[2], &far) && whole_number(a[4], &q_first) && whole_number(a[5], &k_first));
  NEED(grad.take(a[0]) && grad_table.take(a[1]) && at.take(a[6], true) && work.take_memory(a[7]) && grad.is_rows_type() &&
       grad_table.has_type(PSKV_F32) && grad_table.dense());
  Scores g;
  NEED(g.parse(grad) && is_positions(at, g.n[0]));
  if (grad_table.dims != 2 || (size_t)grad_table.n[1] != g.n[1])
    NEED(grad_table.fail(PyExc_ValueError, "[buckets, heads] is expected"));
  int device, rc;
  void* stream;
  NEED(together({&grad, &grad_table, &at, &work}, &device) && stream_of(a[8], device, &stream));
  const size_t buckets = (size_t)grad_table.n[0];
  Room room;
  NEED(room.take(work, pskv_relbias_grad_room(buckets, g.n[1], g.n[0], g.n[2], g.n[3], at.given() ? 1 : 0), a[9], a[0], a[8]));
  Py_BEGIN_ALLOW_THREADS;
  rc = pskv_relbias_grad(device, stream, grad.type, grad.ptr, g.by, buckets, g.n[1], far, two_sided, q_first, k_first,
                         static_cast<int64_t*>(at.ptr), g.n[0], g.n[2], g.n[3], static_cast<float*>(grad_table.ptr), work.ptr,
                         work.given() ? (size_t)work.n[0] : 0);
  Py_END_ALLOW_THREADS;
  return PyLong_FromLong(rc);
}

// dropout(x, out, p, seed, step, keys, first, stream)
PyObject* dropout(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NEED(want(n, 8));
  Tensor x("x"), out("out"), step("step"), keys("keys");
  const double p = PyFloat_AsDouble(a[2]);
  NEED(!PyErr_Occurred());
  unsigned long long seed, first;
  NEED(whole_number(a[3], &seed) && whole_number(a[6], &first));
  NEED(x.take(a[0]) && out.take(a[1]) && step.take(a[4], true) && keys.take(a[5], true) && x.is_rows_type() && x.is_matrix() &&
       out.like(x) && out.is_matrix() && out.sized(x.n[0], x.n[1]));
  if (step.given() && (step.type != kInt64 || step.count() != 1)) NEED(step.fail(PyExc_TypeError, "one word of 64 bits is expected"));
  if (keys.given()) {
    if (keys.type != kInt64) NEED(keys.fail(PyExc_TypeError, "keys of 64 bits are expected"));
    if (keys.count() != x.n[0]) NEED(keys.fail(PyExc_ValueError, "a key for each row is expected"));
    NEED(keys.dense());
  }
  int device, rc;
  void* stream;
  NEED(together({&x, &out, &step, &keys}, &device) && stream_of(a[7], device, &stream));
  Py_BEGIN_ALLOW_THREADS;
  rc = pskv_dropout(device, stream, x.type, x.ptr, x.stride(0, x.n[1]), out.ptr, out.stride(0, out.n[1]), (size_t)x.n[0],
                    (size_t)x.n[1], p, seed, static_cast<uint64_t*>(step.ptr), static_cast<uint64_t*>(keys.ptr), first);
  Py_END_ALLOW_THREADS;
  return PyLong_FromLong(rc);
}

// setup(tensor_type, int64, uint64, float32, int32, raw_stream, float16, bfloat16)
PyObject* setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!want(n, 8)) return nullptr;
  PyObject** to[8] = {&g_tensor_type, &g_int64, &g_uint64, &g_float32, &g_int32, &g_raw_stream, &g_float16, &g_bfloat16};
  for (int i = 0; i < 8; ++i) {
    Py_INCREF(a[i]);
    Py_XDECREF(*to[i]);
    *to[i] = a[i];
  }
  Py_RETURN_NONE;
}

#define FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(setup),      FAST(table_push), FAST(table_pull),     FAST(table_pushpull),
                         FAST(group_push), FAST(group_pull), FAST(group_pushpull), FAST(slice),
                         FAST(match),      FAST(route_sort), FAST(route_rows),     FAST(route_sum),
                         FAST(route_sum_grad), FAST(relbias), FAST(relbias_grad),  FAST(dropout),
                         {"replay_run", replay_run, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) {
  import_array();
  s_dtype = PyUnicode_InternFromString("dtype");
  s_is_cuda = PyUnicode_InternFromString("is_cuda");
  s_is_contiguous = PyUnicode_InternFromString("is_contiguous");
  s_numel = PyUnicode_InternFromString("numel");
  s_data_ptr = PyUnicode_InternFromString("data_ptr");
  s_shape = PyUnicode_InternFromString("shape");
  s_stride = PyUnicode_InternFromString("stride");
  s_get_device = PyUnicode_InternFromString("get_device");
  s_nbytes = PyUnicode_InternFromString("nbytes");
  if (!s_dtype || !s_is_cuda || !s_is_contiguous || !s_numel || !s_data_ptr || !s_shape || !s_stride || !s_get_device || !s_nbytes)
    return nullptr;
  return PyModule_Create(&module);
}
