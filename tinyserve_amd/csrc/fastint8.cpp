// The host path of hip_int8's calls without the interpreter: an eager call of a kernel of a few
// microseconds is bound by it. Takes the tensors, checks them, allocates the results and launches;
// for whatever it does not take (an argument that is refused, another current device, a tensor
// subclass) it returns None with nothing of the caller's written, and the Python function, whose
// rules these are, goes on. Without this module built every call goes that way.
//
// Host time of a call, from Python alone and from here (the launch takes about 2.8 us of it):
// int8_linear 7.8 and 4.2 us, add_rms_norm_rows_int8 9.2 and 4.6, dequantize_rows 7.3 and 3.9. Tensors
// come from the device's allocator without the dispatcher's way there (0.25 us each).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/tinyserve_amd.h"

namespace {

decltype(&ts_int8_quantize_rows) p_quantize;
decltype(&ts_int8_embedding) p_embedding;
decltype(&ts_int8_linear) p_linear;
decltype(&ts_int8_linear_workspace) p_workspace;
decltype(&ts_int8_pad_rows) p_pad;
PyTypeObject* rows_type;   // Int8Rows
PyObject* current_stream;  // device index -> the current stream's handle

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return TS_F32;
    case at::kHalf: return TS_F16;
    case at::kBFloat16: return TS_BF16;
    default: return -1;
  }
}

// The tensor of a Python argument; null for anything but a plain strided tensor on a device.
const at::Tensor* tensor(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.layout() == at::kStrided ? &t : nullptr;
}

bool row_contiguous(const at::Tensor& t) {
  return t.dim() == 2 && (t.stride(1) == 1 || t.size(1) <= 1) && t.size(0) <= TS_INT8_MAX_DIM && t.size(1) <= TS_INT8_MAX_DIM;
}

struct Rows {
  const at::Tensor *q = nullptr, *scale = nullptr;
  int64_t m = 0, k = 0;
};

bool rows_of(PyObject* o, Rows* r) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 2) return false;
  r->q = tensor(PyTuple_GET_ITEM(o, 0));
  r->scale = tensor(PyTuple_GET_ITEM(o, 1));
  if (!r->q || !r->scale || r->q->scalar_type() != at::kChar || !row_contiguous(*r->q)) return false;
  r->m = r->q->size(0);
  r->k = r->q->size(1);
  return r->scale->scalar_type() == at::kFloat && r->scale->dim() == 1 && r->scale->size(0) == r->m && r->scale->is_contiguous() &&
         r->scale->device() == r->q->device();
}

bool vector_like(const at::Tensor& w, const at::Tensor& x, int64_t n) {
  return w.scalar_type() == x.scalar_type() && w.dim() == 1 && w.size(0) == n && w.is_contiguous() && w.device() == x.device();
}

bool current(const at::Tensor& t) {
  const c10::impl::VirtualGuardImpl guard(t.device().type());
  return guard.getDevice() == t.device();
}

// The current stream's handle; false with a Python error set.
bool stream_of(const at::Tensor& t, void** out) {
  PyObject* dev = PyLong_FromLong(t.device().index());
  if (!dev) return false;
  PyObject* s = PyObject_CallOneArg(current_stream, dev);
  Py_DECREF(dev);
  if (!s) return false;
  *out = PyLong_AsVoidPtr(s);
  Py_DECREF(s);
  return !PyErr_Occurred();
}

// Whether every row may be read up to a whole 16 columns.
bool readable(const Rows& r) {
  const int64_t need = (r.k + 15) / 16 * 16, stride = r.q->stride(0);
  return stride >= need && r.q->storage_offset() + (r.m - 1) * stride + need <= static_cast<int64_t>(r.q->storage().nbytes());
}

// Whether tiles can read the rows (hip_int8._fits).
bool fits(const Rows& r) {
  const int64_t stride = r.q->stride(0);
  return reinterpret_cast<uintptr_t>(r.q->const_data_ptr()) % 16 == 0 && stride % 16 == 0 && stride <= (1 << 23) &&
         (r.k % 16 == 0 || readable(r));
}

bool scalar_type(PyObject* o, at::ScalarType* t, int* code) {
  if (!THPDtype_Check(o)) return false;
  *t = reinterpret_cast<THPDtype*>(o)->scalar_type;
  *code = dtype_code(*t);
  return *code >= 0;
}

// quantize(form, x, y, weight, eps) -> Int8Rows
PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 5 || !p_quantize) Py_RETURN_NONE;
  const long form = PyLong_AsLong(a[0]);
  if (form == -1 && PyErr_Occurred()) return nullptr;
  const at::Tensor *x = tensor(a[1]), *y = nullptr, *w = nullptr;
  if (!x || !row_contiguous(*x)) Py_RETURN_NONE;
  const int code = dtype_code(x->scalar_type());
  int64_t t = x->size(0), n = x->size(1);
  if (code < 0 || t == 0 || n == 0) Py_RETURN_NONE;
  double eps = 0.0;
  if (form == TS_INT8_NORM || form == TS_INT8_ADD_NORM) {
    w = tensor(a[3]);
    if (!w || !vector_like(*w, *x, n) || !PyFloat_CheckExact(a[4])) Py_RETURN_NONE;
    eps = PyFloat_AS_DOUBLE(a[4]);
    if (!(eps > 0)) Py_RETURN_NONE;
  }
  if (form == TS_INT8_ADD_NORM) {
    y = tensor(a[2]);
    if (!y || y->scalar_type() != x->scalar_type() || y->dim() != 2 || y->size(0) != t || y->size(1) != n ||
        (y->stride(1) != 1 && n > 1) || y->device() != x->device())
      Py_RETURN_NONE;
  }
  if (form == TS_INT8_SILU) {
    if (n % 2) Py_RETURN_NONE;
    n /= 2;
  }
  if (!current(*x)) Py_RETURN_NONE;
  void* stream;
  if (!stream_of(*x, &stream)) return nullptr;
  const int64_t stride = (n + 15) / 16 * 16;
  at::Tensor q = at::Tensor(at::detail::empty_cuda({t, stride}, at::kChar, x->device(), std::nullopt));
  at::Tensor scale = at::Tensor(at::detail::empty_cuda({t}, at::kFloat, x->device(), std::nullopt));
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = p_quantize(x->data_ptr(), y ? y->const_data_ptr() : nullptr, w ? w->const_data_ptr() : nullptr,
                  static_cast<int8_t*>(q.data_ptr()), static_cast<float*>(scale.data_ptr()), static_cast<int>(t),
                  static_cast<int>(n), x->stride(0), y ? y->stride(0) : 0, stride, static_cast<float>(eps),
                  static_cast<int>(form), code, stream);
  Py_END_ALLOW_THREADS
  if (rc) Py_RETURN_NONE;
  PyObject* pair = PyTuple_New(2);
  if (!pair) return nullptr;
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(stride == n ? q : q.narrow(1, 0, n)));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(scale));
  PyObject* args = PyTuple_GET_ITEM(pair, 0) && PyTuple_GET_ITEM(pair, 1) ? PyTuple_Pack(1, pair) : nullptr;
  Py_DECREF(pair);
  if (!args) return nullptr;
  PyObject* rows = PyTuple_Type.tp_new(rows_type, args, nullptr);
  Py_DECREF(args);
  return rows;
  END_HANDLE_TH_ERRORS
}

// linear(x, w, dtype, out) -> tensor
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  Rows x, w;
  at::ScalarType type;
  int code;
  if (n_args != 4 || !p_linear || !rows_of(a[0], &x) || !rows_of(a[1], &w) || !scalar_type(a[2], &type, &code)) Py_RETURN_NONE;
  const int64_t m = x.m, n = w.m, k = x.k;
  if (w.k != k || k > TS_INT8_MAX_K || m == 0 || n == 0 || x.q->device() != w.q->device() || !current(*x.q)) Py_RETURN_NONE;
  at::Tensor out;
  if (a[3] == Py_None) {
    out = at::Tensor(at::detail::empty_cuda({m, n}, type, x.q->device(), std::nullopt));
  } else {
    const at::Tensor* o = tensor(a[3]);
    if (!o || o->dim() != 2 || o->size(0) != m || o->size(1) != n || o->scalar_type() != type || (o->stride(1) != 1 && n > 1) ||
        (m > 1 && o->stride(0) < n) || o->device() != x.q->device())
      Py_RETURN_NONE;
    out = *o;
  }
  void* stream;
  if (!stream_of(*x.q, &stream)) return nullptr;
  const auto* xp = static_cast<const int8_t*>(x.q->const_data_ptr());
  const auto* wp = static_cast<const int8_t*>(w.q->const_data_ptr());
  int64_t xs = x.q->stride(0), ws = w.q->stride(0);
  const int64_t need = p_workspace(static_cast<int>(m), static_cast<int>(n), static_cast<int>(k));
  at::Tensor sums;
  if (need) sums = at::Tensor(at::detail::empty_cuda({need}, at::kByte, x.q->device(), std::nullopt));
  void* const sums_at = need ? sums.data_ptr() : nullptr;
  auto multiply = [&](int padded) {
    return p_linear(xp, xs, static_cast<const float*>(x.scale->const_data_ptr()), wp, ws,
                    static_cast<const float*>(w.scale->const_data_ptr()), out.data_ptr(), out.stride(0), static_cast<int>(m),
                    static_cast<int>(n), static_cast<int>(k), padded, code, sums_at, need, stream);
  };
  const int padded = k % 16 == 0 || (readable(x) && readable(w));
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = multiply(padded);
  Py_END_ALLOW_THREADS
  if (rc == TS_EUNSUPPORTED) {  // it runs in tiles, which need aligned rows
    const int64_t stride = (k + 15) / 16 * 16;
    at::Tensor xc, wc;
    if (!fits(x)) xc = at::detail::empty_cuda({m, stride}, at::kChar, x.q->device(), std::nullopt);
    if (!fits(w)) wc = at::detail::empty_cuda({n, stride}, at::kChar, x.q->device(), std::nullopt);
    auto* xo = xc.defined() ? static_cast<int8_t*>(xc.data_ptr()) : nullptr;
    auto* wo = wc.defined() ? static_cast<int8_t*>(wc.data_ptr()) : nullptr;
    Py_BEGIN_ALLOW_THREADS
    rc = p_pad(xp, xs, xo, xo ? static_cast<int>(m) : 0, wp, ws, wo, wo ? static_cast<int>(n) : 0, stride, static_cast<int>(k), stream);
    if (xo) xp = xo, xs = stride;
    if (wo) wp = wo, ws = stride;
    if (!rc) rc = multiply(1);
    Py_END_ALLOW_THREADS
  }
  if (rc) Py_RETURN_NONE;
  if (a[3] != Py_None) {
    Py_INCREF(a[3]);
    return a[3];
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// embedding(table, ids, dtype) -> tensor; ids None: every row
PyObject* embedding(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  Rows r;
  at::ScalarType type;
  int code;
  if (n_args != 3 || !p_embedding || !rows_of(a[0], &r) || !scalar_type(a[2], &type, &code)) Py_RETURN_NONE;
  int64_t t = r.m;
  const at::Tensor* ids = nullptr;
  if (a[1] != Py_None) {
    ids = tensor(a[1]);
    if (!ids || ids->dim() != 1 || ids->scalar_type() != at::kLong || !ids->is_contiguous() || ids->device() != r.q->device())
      Py_RETURN_NONE;
    t = ids->size(0);
  }
  if (t == 0 || t > TS_INT8_MAX_DIM || r.m == 0 || r.k == 0 || !current(*r.q)) Py_RETURN_NONE;
  void* stream;
  if (!stream_of(*r.q, &stream)) return nullptr;
  at::Tensor out = at::Tensor(at::detail::empty_cuda({t, r.k}, type, r.q->device(), std::nullopt));
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = p_embedding(static_cast<const int8_t*>(r.q->const_data_ptr()), r.q->stride(0), static_cast<const float*>(r.scale->const_data_ptr()),
                   r.m, ids ? static_cast<const int64_t*>(ids->const_data_ptr()) : nullptr, out.data_ptr(), r.k,
                   static_cast<int>(t), static_cast<int>(r.k), code, stream);
  Py_END_ALLOW_THREADS
  if (rc) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// bind(quantize, embedding, linear, its workspace, pad: the library's addresses; Int8Rows; the stream function)
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long q, e, l, s, p;
  PyObject *type, *stream;
  if (!PyArg_ParseTuple(args, "KKKKKOO", &q, &e, &l, &s, &p, &type, &stream)) return nullptr;
  if (!PyType_Check(type) || !PyType_IsSubtype(reinterpret_cast<PyTypeObject*>(type), &PyTuple_Type)) {
    PyErr_SetString(PyExc_TypeError, "bind takes a tuple type");
    return nullptr;
  }
  Py_INCREF(type);
  Py_INCREF(stream);
  Py_XDECREF(rows_type);
  Py_XDECREF(current_stream);
  rows_type = reinterpret_cast<PyTypeObject*>(type);
  current_stream = stream;
  p_quantize = reinterpret_cast<decltype(p_quantize)>(static_cast<uintptr_t>(q));
  p_embedding = reinterpret_cast<decltype(p_embedding)>(static_cast<uintptr_t>(e));
  p_linear = reinterpret_cast<decltype(p_linear)>(static_cast<uintptr_t>(l));
  p_workspace = reinterpret_cast<decltype(p_workspace)>(static_cast<uintptr_t>(s));
  p_pad = reinterpret_cast<decltype(p_pad)>(static_cast<uintptr_t>(p));
  Py_RETURN_NONE;
}

#define METHOD(NAME) {#NAME, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(NAME)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, nullptr}, METHOD(quantize), METHOD(linear), METHOD(embedding), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fastint8", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fastint8(void) { return PyModule_Create(&module); }
