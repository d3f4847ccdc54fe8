// The Python calls of the serving loop as one native step each: argument checks, the output
// allocation and the C-ABI call (include/kq.h), for torch tensors.
//
// A small linear is bound by the host: 9.0 us per call through Python checks (1.0), torch.empty
// (2.4, and 1 for its release), ctypes conversions (0.7) and the launch (2.7), where the kernel
// takes 4.  Here everything but the launch is about 1 us.
//
// Every function returns the result, an int (the kq_status of a call the library refused), or None
// when an argument is not of the plain form it handles (then the Python method goes on with its
// own checks and conversions, and raises what they raise).  A C++ exception inside one (an output that
// cannot be allocated, a tensor without memory) leaves as the Python exception torch makes of it.
#define PY_SSIZE_T_CLEAN
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <Python.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <exception>

namespace {

// Addresses of the library's entry points, handed over once (bind): this module does not link libkq,
// it calls the one the ctypes layer has loaded.
using LinearFn = int (*)(void*, uint64_t, uint64_t, int, uint64_t, uint64_t, uint32_t);
using FusedFn = int (*)(void*, uint32_t, const uint64_t*, uint64_t, int, uint64_t, float, const uint64_t*, uint64_t, const uint64_t*, uint32_t,
                        uint32_t);
using QuantizeFn = int (*)(void*, uint64_t, uint32_t, uint32_t, uint64_t, uint64_t);
using A8Fn = int (*)(void*, uint64_t, uint64_t, uint64_t, uint64_t, uint64_t, uint32_t);
using EmbeddingFn = int (*)(void*, uint64_t, uint64_t, uint32_t, uint64_t);
using RopeFn = int (*)(void*, uint64_t, int, uint32_t, uint32_t, uint32_t, uint64_t, uint64_t, uint64_t, uint32_t, uint32_t, uint32_t, uint64_t, uint64_t);
using AppendFn = int (*)(void*, uint64_t, uint64_t, uint64_t, uint64_t, uint64_t, int, uint32_t, uint64_t, uint32_t, uint64_t, uint64_t, uint32_t, uint64_t,
                         uint32_t, uint32_t, uint32_t);
using ReadFn = int (*)(void*, uint64_t, uint32_t, uint64_t, uint32_t, uint64_t, uint64_t, uint32_t, uint64_t, uint64_t);
using AttendFn = int (*)(void*, uint64_t, uint64_t, uint64_t, int, uint32_t, uint32_t, uint64_t, uint32_t, uint64_t, uint64_t, uint32_t, uint32_t, float,
                         uint32_t, uint64_t, uint32_t, uint32_t, uint32_t, uint64_t, uint64_t);
using AttendSharedFn = int (*)(void*, uint64_t, uint64_t, uint64_t, int, uint32_t, uint32_t, uint64_t, uint32_t, uint64_t, uint64_t, uint32_t, uint32_t, uint32_t,
                               uint64_t, uint64_t, uint64_t, float, uint32_t, uint64_t, uint32_t, uint32_t, uint32_t, uint64_t, uint64_t);
using AttendSelectedFn = int (*)(void*, uint64_t, uint64_t, uint64_t, int, uint32_t, uint32_t, uint64_t, uint32_t, uint64_t, uint64_t, uint32_t, uint64_t, uint32_t,
                                 float, uint64_t, uint32_t, uint32_t, uint32_t, uint64_t, uint64_t);
using SummarizeFn = int (*)(void*, uint64_t, uint64_t, uint64_t, uint32_t, uint64_t, uint32_t, uint64_t, uint64_t, uint32_t);
using SelectFn = int (*)(void*, uint64_t, uint64_t, uint64_t, uint64_t, uint64_t, int, uint32_t, uint32_t, uint64_t, uint32_t, uint64_t, uint64_t, uint32_t, uint32_t,
                         uint32_t, uint32_t, uint64_t, uint32_t, uint32_t, uint32_t, uint64_t);
using GrowFn = int (*)(void*, uint64_t, uint32_t, uint32_t, uint64_t, uint64_t, uint32_t, uint32_t, uint64_t, uint64_t);
using ForkFn = int (*)(void*, uint64_t, uint32_t, uint32_t, uint64_t, uint64_t, uint32_t, uint32_t, uint64_t, uint64_t, uint64_t, uint64_t);
using CompactFn = int (*)(void*, uint64_t, uint32_t, uint32_t, uint64_t, uint64_t, uint32_t, uint32_t, uint64_t, uint64_t);
using CopyFn = int (*)(void*, uint32_t, const uint64_t*, const uint64_t*, uint32_t, uint64_t, uint32_t, uint64_t);
AttendSharedFn g_attend_shared = nullptr;
AttendSelectedFn g_attend_selected = nullptr;
SummarizeFn g_summarize = nullptr;
SelectFn g_select = nullptr;
GrowFn g_grow = nullptr;
ForkFn g_fork = nullptr;
CompactFn g_compact = nullptr;
CopyFn g_copy = nullptr;
LinearFn g_linear = nullptr;
FusedFn g_fused = nullptr;
QuantizeFn g_quantize = nullptr;
A8Fn g_a8 = nullptr;
EmbeddingFn g_embedding = nullptr;
RopeFn g_rope = nullptr;
AppendFn g_append = nullptr;
ReadFn g_read = nullptr;
AttendFn g_attend = nullptr;

constexpr int kMaxMulti = 4;

// 0 / 1 / 2 = KQ_F32 / KQ_F16 / KQ_BF16, -1: not an activation type
int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kHalf: return 1;
    case at::kBFloat16: return 2;
    default: return -1;
  }
}
bool plain(const at::Tensor& t) { return t.is_cuda() && t.is_contiguous(); }
uint64_t ptr(const at::Tensor& t) { return reinterpret_cast<uint64_t>(t.data_ptr()); }
bool tensor_of(PyObject* o, const at::Tensor** out) {
  if (!THPVariable_Check(o)) return false;
  *out = &THPVariable_Unpack(o);
  return true;
}
at::Tensor empty_like_lead(const at::Tensor& x, int64_t last, at::ScalarType type) {
  c10::SmallVector<int64_t, 8> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = last;
  return at::detail::empty_cuda(shape, type, x.device(), c10::nullopt);
}
PyObject* status_of(int rc) { return PyLong_FromLong(rc); }
#define KQ_NONE Py_RETURN_NONE

// The library call while other Python threads run; the lock is back before anything, an exception too, goes on.
template <typename Call>
int without_gil(Call call) {
  struct Released {
    PyThreadState* state = PyEval_SaveThread();
    ~Released() { PyEval_RestoreThread(state); }
  } released;
  return call();
}

PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 17) {
    PyErr_SetString(PyExc_TypeError, "bind takes seventeen addresses");
    return nullptr;
  }
  g_linear = reinterpret_cast<LinearFn>(PyLong_AsVoidPtr(a[0]));
  g_fused = reinterpret_cast<FusedFn>(PyLong_AsVoidPtr(a[1]));
  g_quantize = reinterpret_cast<QuantizeFn>(PyLong_AsVoidPtr(a[2]));
  g_a8 = reinterpret_cast<A8Fn>(PyLong_AsVoidPtr(a[3]));
  g_embedding = reinterpret_cast<EmbeddingFn>(PyLong_AsVoidPtr(a[4]));
  g_rope = reinterpret_cast<RopeFn>(PyLong_AsVoidPtr(a[5]));
  g_append = reinterpret_cast<AppendFn>(PyLong_AsVoidPtr(a[6]));
  g_read = reinterpret_cast<ReadFn>(PyLong_AsVoidPtr(a[7]));
  g_attend = reinterpret_cast<AttendFn>(PyLong_AsVoidPtr(a[8]));
  g_attend_shared = reinterpret_cast<AttendSharedFn>(PyLong_AsVoidPtr(a[9]));
  g_attend_selected = reinterpret_cast<AttendSelectedFn>(PyLong_AsVoidPtr(a[10]));
  g_summarize = reinterpret_cast<SummarizeFn>(PyLong_AsVoidPtr(a[11]));
  g_select = reinterpret_cast<SelectFn>(PyLong_AsVoidPtr(a[12]));
  g_grow = reinterpret_cast<GrowFn>(PyLong_AsVoidPtr(a[13]));
  g_fork = reinterpret_cast<ForkFn>(PyLong_AsVoidPtr(a[14]));
  g_compact = reinterpret_cast<CompactFn>(PyLong_AsVoidPtr(a[15]));
  g_copy = reinterpret_cast<CopyFn>(PyLong_AsVoidPtr(a[16]));
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

// linear(ctx, handle, n, k, x, bias, out)
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  if (nargs != 7 || a[0] == Py_None) KQ_NONE;
  const int64_t n = PyLong_AsLongLong(a[2]), k = PyLong_AsLongLong(a[3]);
  const at::Tensor *x, *bias, *given = nullptr;
  if (!tensor_of(a[4], &x) || !tensor_of(a[5], &bias) || (a[6] != Py_None && !tensor_of(a[6], &given))) KQ_NONE;
  const int type = dtype_code(*x);
  if (type < 0 || !plain(*x) || x->dim() < 1 || x->size(-1) != k || k == 0 || bias->scalar_type() != at::kFloat || bias->dim() != 1 ||
      bias->size(0) != n)
    KQ_NONE;
  at::Tensor made;
  if (given == nullptr) made = empty_like_lead(*x, n, at::kFloat);
  const at::Tensor& out = given != nullptr ? *given : made;
  void* ctx = PyLong_AsVoidPtr(a[0]);
  const uint64_t handle = PyLong_AsUnsignedLongLong(a[1]);
  const uint64_t px = ptr(*x), pb = ptr(*bias), po = ptr(out);
  const uint32_t m = static_cast<uint32_t>(x->numel() / k);
  const int rc = without_gil([&] { return g_linear(ctx, handle, px, type, pb, po, m); });
  if (rc != 0) return status_of(rc);
  if (given != nullptr) return Py_NewRef(a[6]);
  return THPVariable_Wrap(std::move(made));
}

// linear_fused(ctx, handles, k, x, biases, outs, norm_weight, eps, residual, flags): `outs` a list of tensors
PyObject* linear_fused(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  if (nargs != 10 || a[0] == Py_None) KQ_NONE;
  PyObject *handles = a[1], *biases = a[4], *outs = a[5];
  if (!PyList_CheckExact(handles) || !PyList_CheckExact(biases) || !PyList_CheckExact(outs)) KQ_NONE;
  const Py_ssize_t count = PyList_GET_SIZE(handles);
  if (count < 1 || count > kMaxMulti || PyList_GET_SIZE(biases) != count || PyList_GET_SIZE(outs) < 1) KQ_NONE;
  const int64_t k = PyLong_AsLongLong(a[2]);
  const at::Tensor *x, *t, *norm = nullptr, *residual = nullptr;
  if (!tensor_of(a[3], &x) || (a[6] != Py_None && !tensor_of(a[6], &norm)) || (a[8] != Py_None && !tensor_of(a[8], &residual))) KQ_NONE;
  const int type = dtype_code(*x);
  if (type < 0 || !plain(*x) || x->dim() < 1 || x->size(-1) != k || k == 0) KQ_NONE;
  uint64_t w[kMaxMulti] = {}, b[kMaxMulti] = {}, o[kMaxMulti] = {};
  for (Py_ssize_t i = 0; i < count; ++i) {
    w[i] = PyLong_AsUnsignedLongLong(PyList_GET_ITEM(handles, i));
    if (!tensor_of(PyList_GET_ITEM(biases, i), &t)) KQ_NONE;
    b[i] = ptr(*t);
    if (i < PyList_GET_SIZE(outs)) {
      if (!tensor_of(PyList_GET_ITEM(outs, i), &t)) KQ_NONE;
      o[i] = ptr(*t);
    }
  }
  void* ctx = PyLong_AsVoidPtr(a[0]);
  const float eps = static_cast<float>(PyFloat_AsDouble(a[7]));
  const uint32_t flags = static_cast<uint32_t>(PyLong_AsUnsignedLong(a[9]));
  if (PyErr_Occurred()) return nullptr;
  const uint64_t px = ptr(*x), pn = norm != nullptr ? ptr(*norm) : 0, pr = residual != nullptr ? ptr(*residual) : 0;
  const uint32_t m = static_cast<uint32_t>(x->numel() / k);
  const int rc = without_gil([&] { return g_fused(ctx, static_cast<uint32_t>(count), w, px, type, pn, eps, b, pr, o, m, flags); });
  if (rc != 0) return status_of(rc);
  return Py_NewRef(outs);
}

// quantize_rows(ctx, x) -> (q, scale)
PyObject* quantize_rows(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  const at::Tensor* x;
  if (nargs != 2 || a[0] == Py_None || !tensor_of(a[1], &x) || x->scalar_type() != at::kFloat || !plain(*x) || x->dim() < 1) KQ_NONE;
  const int64_t dim = x->size(-1);
  if (dim == 0) KQ_NONE;
  at::Tensor q = at::detail::empty_cuda(x->sizes(), at::kChar, x->device(), c10::nullopt);
  at::Tensor scale = at::detail::empty_cuda(x->sizes().slice(0, x->dim() - 1), at::kFloat, x->device(), c10::nullopt);
  void* ctx = PyLong_AsVoidPtr(a[0]);
  const uint64_t px = ptr(*x), pq = ptr(q), ps = ptr(scale);
  const uint32_t rows = static_cast<uint32_t>(x->numel() / dim);
  const int rc = without_gil([&] { return g_quantize(ctx, px, rows, static_cast<uint32_t>(dim), pq, ps); });
  if (rc != 0) return status_of(rc);
  PyObject *pyq = THPVariable_Wrap(std::move(q)), *pys = THPVariable_Wrap(std::move(scale));
  PyObject* r = pyq != nullptr && pys != nullptr ? PyTuple_Pack(2, pyq, pys) : nullptr;
  Py_XDECREF(pyq);
  Py_XDECREF(pys);
  return r;
}

// linear_a8(ctx, handle, n, k, xq, xs, bias, out)
PyObject* linear_a8(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  if (nargs != 8 || a[0] == Py_None) KQ_NONE;
  const int64_t n = PyLong_AsLongLong(a[2]), k = PyLong_AsLongLong(a[3]);
  const at::Tensor *xq, *xs, *bias, *given = nullptr;
  if (!tensor_of(a[4], &xq) || !tensor_of(a[5], &xs) || !tensor_of(a[6], &bias) || (a[7] != Py_None && !tensor_of(a[7], &given))) KQ_NONE;
  if (xq->scalar_type() != at::kChar || !plain(*xq) || xq->dim() < 1 || xq->size(-1) != k || k == 0 || xs->scalar_type() != at::kFloat ||
      xs->numel() != xq->numel() / k || bias->scalar_type() != at::kFloat || bias->numel() != n)
    KQ_NONE;
  at::Tensor made;
  if (given == nullptr) made = empty_like_lead(*xq, n, at::kFloat);
  const at::Tensor& out = given != nullptr ? *given : made;
  void* ctx = PyLong_AsVoidPtr(a[0]);
  const uint64_t handle = PyLong_AsUnsignedLongLong(a[1]);
  const uint64_t pq = ptr(*xq), ps = ptr(*xs), pb = ptr(*bias), po = ptr(out);
  const uint32_t m = static_cast<uint32_t>(xq->numel() / k);
  const int rc = without_gil([&] { return g_a8(ctx, handle, pq, ps, pb, po, m); });
  if (rc != 0) return status_of(rc);
  if (given != nullptr) return Py_NewRef(a[7]);
  return THPVariable_Wrap(std::move(made));
}

// embedding(ctx, handle, k, index, out)
PyObject* embedding(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  if (nargs != 5 || a[0] == Py_None) KQ_NONE;
  const int64_t k = PyLong_AsLongLong(a[2]);
  const at::Tensor *index, *given = nullptr;
  if (!tensor_of(a[3], &index) || (a[4] != Py_None && !tensor_of(a[4], &given)) || index->scalar_type() != at::kInt || !plain(*index)) KQ_NONE;
  at::Tensor made;
  if (given == nullptr) {
    c10::SmallVector<int64_t, 8> shape(index->sizes().begin(), index->sizes().end());
    shape.push_back(k);
    made = at::detail::empty_cuda(shape, at::kFloat, index->device(), c10::nullopt);
  }
  const at::Tensor& out = given != nullptr ? *given : made;
  void* ctx = PyLong_AsVoidPtr(a[0]);
  const uint64_t handle = PyLong_AsUnsignedLongLong(a[1]);
  const uint64_t pi = ptr(*index), po = ptr(out);
  const uint32_t rows = static_cast<uint32_t>(index->numel());
  const int rc = without_gil([&] { return g_embedding(ctx, handle, pi, rows, po); });
  if (rc != 0) return status_of(rc);
  if (given != nullptr) return Py_NewRef(a[4]);
  return THPVariable_Wrap(std::move(made));
}

// ---- rotary positions, the packed cache and attention over it -----------------------------------------
// Rows [tokens, heads, dim] with dense heads and values; the elements between tokens.
bool rows_of(const at::Tensor& t, int64_t tokens, int64_t heads, int64_t dim, uint64_t* stride) {
  if (!t.is_cuda() || t.dim() != 3 || t.size(0) != tokens || t.size(1) != heads || t.size(2) != dim || t.stride(2) != 1 || (heads > 1 && t.stride(1) != dim) ||
      t.stride(0) < 0)
    return false;
  *stride = static_cast<uint64_t>(tokens > 1 ? t.stride(0) : heads * dim);
  return true;
}
// A tuple of whole numbers, as Rope.args and CacheBatch.args hold them; None stands for zeros.
template <int N>
bool numbers_of(PyObject* o, uint64_t (&v)[N]) {
  if (o == Py_None) {
    for (uint64_t& x : v) x = 0;
    return true;
  }
  if (!PyTuple_CheckExact(o) || PyTuple_GET_SIZE(o) != N) return false;
  for (int i = 0; i < N; ++i) v[i] = PyLong_AsUnsignedLongLong(PyTuple_GET_ITEM(o, i));
  return PyErr_Occurred() == nullptr;
}
uint32_t u32(uint64_t v) { return static_cast<uint32_t>(v); }

// rope(ctx, x, positions, rope args, out)
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  const at::Tensor *x, *positions, *given = nullptr;
  uint64_t table[4], x_stride, out_stride;
  if (nargs != 5 || a[0] == Py_None || !tensor_of(a[1], &x) || !tensor_of(a[2], &positions) || (a[4] != Py_None && !tensor_of(a[4], &given)) ||
      !numbers_of(a[3], table))
    KQ_NONE;
  const int type = dtype_code(*x);
  if (type < 0 || x->dim() != 3 || x->numel() == 0 || positions->scalar_type() != at::kInt || !plain(*positions) || positions->numel() != x->size(0)) KQ_NONE;
  const int64_t tokens = x->size(0), heads = x->size(1), dim = x->size(2);
  at::Tensor made;
  if (given == nullptr) made = at::detail::empty_cuda(x->sizes(), x->scalar_type(), x->device(), c10::nullopt);
  const at::Tensor& out = given != nullptr ? *given : made;
  if (out.scalar_type() != x->scalar_type() || !rows_of(*x, tokens, heads, dim, &x_stride) || !rows_of(out, tokens, heads, dim, &out_stride)) KQ_NONE;
  void* ctx = PyLong_AsVoidPtr(a[0]);
  const uint64_t px = ptr(*x), pp = ptr(*positions), po = ptr(out);
  const int rc = without_gil([&] {
    return g_rope(ctx, px, type, u32(tokens), u32(heads), u32(dim), x_stride, pp, table[0], u32(table[1]), u32(table[2]), u32(table[3]), po, out_stride);
  });
  if (rc != 0) return status_of(rc);
  if (given != nullptr) return Py_NewRef(a[4]);
  return THPVariable_Wrap(std::move(made));
}

// cache_append(ctx, handle, kv_heads, dim, k, v, batch args, rope args): 0, or the status
PyObject* cache_append(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  const at::Tensor *k, *v;
  uint64_t batch[6], table[4], k_stride, v_stride;
  if (nargs != 8 || a[0] == Py_None || !tensor_of(a[4], &k) || !tensor_of(a[5], &v) || !numbers_of(a[6], batch) || !numbers_of(a[7], table)) KQ_NONE;
  const int64_t heads = PyLong_AsLongLong(a[2]), dim = PyLong_AsLongLong(a[3]), tokens = static_cast<int64_t>(batch[5]);
  const int type = dtype_code(*k);
  if (type < 0 || v->scalar_type() != k->scalar_type() || !rows_of(*k, tokens, heads, dim, &k_stride) || !rows_of(*v, tokens, heads, dim, &v_stride)) KQ_NONE;
  void* ctx = PyLong_AsVoidPtr(a[0]);
  const uint64_t handle = PyLong_AsUnsignedLongLong(a[1]), pk = ptr(*k), pv = ptr(*v);
  if (PyErr_Occurred()) return nullptr;
  return status_of(without_gil([&] {
    return g_append(ctx, handle, pk, k_stride, pv, v_stride, type, u32(batch[0]), batch[1], u32(batch[2]), batch[3], batch[4], u32(batch[5]), table[0],
                    u32(table[1]), u32(table[2]), u32(table[3]));
  }));
}

// cache_read(ctx, handle, kv_heads, dim, device index, batch args) -> (k, v)
PyObject* cache_read(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  uint64_t batch[6];
  if (nargs != 6 || a[0] == Py_None || !numbers_of(a[5], batch)) KQ_NONE;
  const int64_t shape[3] = {static_cast<int64_t>(batch[5]), PyLong_AsLongLong(a[2]), PyLong_AsLongLong(a[3])};
  const at::Device device(at::kCUDA, static_cast<at::DeviceIndex>(PyLong_AsLong(a[4])));
  if (PyErr_Occurred()) return nullptr;
  at::Tensor k = at::detail::empty_cuda(shape, at::kFloat, device, c10::nullopt), v = at::detail::empty_cuda(shape, at::kFloat, device, c10::nullopt);
  void* ctx = PyLong_AsVoidPtr(a[0]);
  const uint64_t handle = PyLong_AsUnsignedLongLong(a[1]), pk = ptr(k), pv = ptr(v);
  const int rc =
      without_gil([&] { return g_read(ctx, handle, u32(batch[0]), batch[1], u32(batch[2]), batch[3], batch[4], u32(batch[5]), pk, pv); });
  if (rc != 0) return status_of(rc);
  PyObject *pyk = THPVariable_Wrap(std::move(k)), *pyv = THPVariable_Wrap(std::move(v));
  PyObject* r = pyk != nullptr && pyv != nullptr ? PyTuple_Pack(2, pyk, pyv) : nullptr;
  Py_XDECREF(pyk);
  Py_XDECREF(pyv);
  return r;
}

// The queries and the output of an attention call, made where none is given; false: not of the plain form.
struct Rows {
  const at::Tensor *q = nullptr, *given = nullptr;
  at::Tensor made;
  int type = -1;
  int64_t heads = 0;
  uint64_t pq = 0, po = 0, q_stride = 0, out_stride = 0;
  // device: the context's, or -1 for any
  bool of(PyObject* queries, PyObject* out, int64_t tokens, int64_t dim, int64_t device = -1) {
    if (!tensor_of(queries, &q) || (out != Py_None && !tensor_of(out, &given))) return false;
    type = dtype_code(*q);
    if (type < 0 || q->dim() != 3 || q->numel() == 0) return false;
    heads = q->size(1);
    if (!rows_of(*q, tokens, heads, dim, &q_stride) || (device >= 0 && q->get_device() != device)) return false;
    if (given != nullptr && device >= 0 && given->get_device() != device) return false;
    if (given == nullptr) made = at::detail::empty_cuda(q->sizes(), q->scalar_type(), q->device(), c10::nullopt);
    const at::Tensor& o = given != nullptr ? *given : made;
    if (o.scalar_type() != q->scalar_type() || !rows_of(o, tokens, heads, dim, &out_stride)) return false;
    pq = ptr(*q);
    po = ptr(o);
    return true;
  }
  PyObject* result(PyObject* out) { return given != nullptr ? Py_NewRef(out) : THPVariable_Wrap(std::move(made)); }
};

// cache_attention(ctx, handle, dim, q, batch args, most, scale, window, rope args, out)
PyObject* cache_attention(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  uint64_t batch[6], table[4];
  Rows r;
  if (nargs != 10 || a[0] == Py_None || !numbers_of(a[4], batch) || !numbers_of(a[8], table)) KQ_NONE;
  if (!r.of(a[3], a[9], static_cast<int64_t>(batch[5]), PyLong_AsLongLong(a[2]))) KQ_NONE;
  void* ctx = PyLong_AsVoidPtr(a[0]);
  const uint64_t handle = PyLong_AsUnsignedLongLong(a[1]);
  const uint32_t most = u32(PyLong_AsUnsignedLong(a[5])), window = u32(PyLong_AsUnsignedLong(a[7]));
  const float scale = static_cast<float>(PyFloat_AsDouble(a[6]));
  if (PyErr_Occurred()) return nullptr;
  const int rc = without_gil([&] {
    return g_attend(ctx, handle, r.pq, r.q_stride, r.type, u32(r.heads), u32(batch[0]), batch[1], u32(batch[2]), batch[3], batch[4], u32(batch[5]), most, scale, window,
                    table[0], u32(table[1]), u32(table[2]), u32(table[3]), r.po, r.out_stride);
  });
  return rc != 0 ? status_of(rc) : r.result(a[9]);
}

// cache_attention_shared(ctx, handle, dim, q, batch args, most, shared args, scale, window, rope args, out, device index)
PyObject* cache_attention_shared(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  uint64_t batch[6], table[4], groups[4];
  Rows r;
  if (nargs != 12 || a[0] == Py_None || !numbers_of(a[4], batch) || !numbers_of(a[6], groups) || !numbers_of(a[9], table)) KQ_NONE;
  if (!r.of(a[3], a[10], static_cast<int64_t>(batch[5]), PyLong_AsLongLong(a[2]), PyLong_AsLongLong(a[11]))) KQ_NONE;
  void* ctx = PyLong_AsVoidPtr(a[0]);
  const uint64_t handle = PyLong_AsUnsignedLongLong(a[1]);
  const uint32_t most = u32(PyLong_AsUnsignedLong(a[5])), window = u32(PyLong_AsUnsignedLong(a[8]));
  const float scale = static_cast<float>(PyFloat_AsDouble(a[7]));
  if (PyErr_Occurred()) return nullptr;
  const int rc = without_gil([&] {
    return g_attend_shared(ctx, handle, r.pq, r.q_stride, r.type, u32(r.heads), u32(batch[0]), batch[1], u32(batch[2]), batch[3], batch[4], u32(batch[5]), most,
                           u32(groups[0]), groups[1], groups[2], groups[3], scale, window, table[0], u32(table[1]), u32(table[2]), u32(table[3]), r.po, r.out_stride);
  });
  return rc != 0 ? status_of(rc) : r.result(a[10]);
}

// cache_attention_selected(ctx, handle, kv_heads, dim, q, batch args, selected, scale, rope args, out, device index)
PyObject* cache_attention_selected(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  uint64_t batch[6], table[4];
  const at::Tensor* selected;
  Rows r;
  if (nargs != 11 || a[0] == Py_None || !numbers_of(a[5], batch) || !numbers_of(a[8], table) || !tensor_of(a[6], &selected)) KQ_NONE;
  const int64_t device = PyLong_AsLongLong(a[10]);
  const int64_t tokens = static_cast<int64_t>(batch[5]);
  if (selected->scalar_type() != at::kInt || !plain(*selected) || selected->dim() != 3 || selected->size(0) != tokens ||
      selected->size(1) != PyLong_AsLongLong(a[2]) || selected->size(2) == 0 || selected->get_device() != device ||
      !r.of(a[4], a[9], tokens, PyLong_AsLongLong(a[3]), device))
    KQ_NONE;
  void* ctx = PyLong_AsVoidPtr(a[0]);
  const uint64_t handle = PyLong_AsUnsignedLongLong(a[1]), ps = ptr(*selected);
  const float scale = static_cast<float>(PyFloat_AsDouble(a[7]));
  const uint32_t budget = u32(static_cast<uint64_t>(selected->size(2)));
  if (PyErr_Occurred()) return nullptr;
  const int rc = without_gil([&] {
    return g_attend_selected(ctx, handle, r.pq, r.q_stride, r.type, u32(r.heads), u32(batch[0]), batch[1], u32(batch[2]), batch[3], batch[4], u32(batch[5]), ps, budget,
                             scale, table[0], u32(table[1]), u32(table[2]), u32(table[3]), r.po, r.out_stride);
  });
  return rc != 0 ? status_of(rc) : r.result(a[9]);
}

// cache_summarize(ctx, handle, summaries args, batch args): 0, or the status
PyObject* cache_summarize(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  uint64_t of[2], batch[6];
  if (nargs != 4 || a[0] == Py_None || !numbers_of(a[2], of) || !numbers_of(a[3], batch)) KQ_NONE;
  void* ctx = PyLong_AsVoidPtr(a[0]);
  const uint64_t handle = PyLong_AsUnsignedLongLong(a[1]);
  if (PyErr_Occurred()) return nullptr;
  return status_of(without_gil([&] { return g_summarize(ctx, handle, of[0], of[1], u32(batch[0]), batch[1], u32(batch[2]), batch[3], batch[4], u32(batch[5])); }));
}

// cache_select(ctx, handle, kv_heads, dim, summaries args, q, batch args, budget, first, last, rope args, out, device index)
PyObject* cache_select(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  uint64_t of[2], batch[6], table[4], q_stride;
  const at::Tensor *q, *given = nullptr;
  if (nargs != 13 || a[0] == Py_None || !numbers_of(a[4], of) || !tensor_of(a[5], &q) || !numbers_of(a[6], batch) || !numbers_of(a[10], table) ||
      (a[11] != Py_None && !tensor_of(a[11], &given)))
    KQ_NONE;
  const int64_t tokens = static_cast<int64_t>(batch[5]), kv_heads = PyLong_AsLongLong(a[2]), dim = PyLong_AsLongLong(a[3]);
  const int64_t budget = PyLong_AsLongLong(a[7]), first = PyLong_AsLongLong(a[8]), last = PyLong_AsLongLong(a[9]);
  const int64_t device = PyLong_AsLongLong(a[12]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    KQ_NONE;
  }
  const int type = q->get_device() == device ? dtype_code(*q) : -1;
  if (type < 0 || q->dim() != 3 || q->numel() == 0 || !rows_of(*q, tokens, q->size(1), dim, &q_stride) || budget <= 0 || budget > (1 << 20) || first < 0 ||
      first > budget || last < 0 || last > budget)
    KQ_NONE;
  const int64_t shape[3] = {tokens, kv_heads, budget};
  if (given != nullptr && (given->scalar_type() != at::kInt || !plain(*given) || given->get_device() != device || given->sizes() != at::IntArrayRef(shape))) KQ_NONE;
  at::Tensor made;
  if (given == nullptr) made = at::detail::empty_cuda(shape, at::kInt, q->device(), c10::nullopt);
  void* ctx = PyLong_AsVoidPtr(a[0]);
  const uint64_t handle = PyLong_AsUnsignedLongLong(a[1]), pq = ptr(*q), po = ptr(given != nullptr ? *given : made);
  const uint32_t heads = u32(static_cast<uint64_t>(q->size(1)));
  if (PyErr_Occurred()) return nullptr;
  const int rc = without_gil([&] {
    return g_select(ctx, handle, of[0], of[1], pq, q_stride, type, heads, u32(batch[0]), batch[1], u32(batch[2]), batch[3], batch[4], u32(batch[5]),
                    static_cast<uint32_t>(budget), static_cast<uint32_t>(first), static_cast<uint32_t>(last), table[0], u32(table[1]), u32(table[2]), u32(table[3]), po);
  });
  if (rc != 0) return status_of(rc);
  if (given != nullptr) return Py_NewRef(a[11]);
  return THPVariable_Wrap(std::move(made));
}

// ---- books of pages: (table, sequences, width, lengths, refs, pages, page_tokens, report) -----------------
// An i32 array with a number for each sequence, on the context's device.
bool each_sequence(PyObject* o, const uint64_t (&book)[8], int64_t device, uint64_t* address) {
  const at::Tensor* t;
  if (!tensor_of(o, &t) || t->scalar_type() != at::kInt || !plain(*t) || t->get_device() != device || static_cast<uint64_t>(t->numel()) != book[1]) return false;
  *address = ptr(*t);
  return true;
}
at::Tensor pairs_for(uint64_t count, int64_t device) {
  const int64_t shape[2] = {static_cast<int64_t>(count), 2};
  return at::detail::empty_cuda(shape, at::kInt, at::Device(at::kCUDA, static_cast<at::DeviceIndex>(device)), c10::nullopt);
}

// pages_grow(ctx, book args, news, device index): 0, or the status
PyObject* pages_grow(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  uint64_t k[8], news;
  if (nargs != 4 || a[0] == Py_None || !numbers_of(a[1], k) || !each_sequence(a[2], k, PyLong_AsLongLong(a[3]), &news)) KQ_NONE;
  void* ctx = PyLong_AsVoidPtr(a[0]);
  return status_of(without_gil([&] { return g_grow(ctx, k[0], u32(k[1]), u32(k[2]), k[3], k[4], u32(k[5]), u32(k[6]), k[7], news); }));
}

// pages_fork(ctx, book args, parents, keep, device index) -> pairs
PyObject* pages_fork(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  uint64_t k[8], parents, keep = 0;
  if (nargs != 5 || a[0] == Py_None || !numbers_of(a[1], k)) KQ_NONE;
  const int64_t device = PyLong_AsLongLong(a[4]);
  if (!each_sequence(a[2], k, device, &parents) || (a[3] != Py_None && !each_sequence(a[3], k, device, &keep))) KQ_NONE;
  at::Tensor pairs = pairs_for(k[1], device);
  void* ctx = PyLong_AsVoidPtr(a[0]);
  const uint64_t to = ptr(pairs);
  const int rc = without_gil([&] { return g_fork(ctx, k[0], u32(k[1]), u32(k[2]), k[3], k[4], u32(k[5]), u32(k[6]), k[7], parents, keep, to); });
  return rc != 0 ? status_of(rc) : THPVariable_Wrap(std::move(pairs));
}

// pages_compact(ctx, book args, device index) -> pairs
PyObject* pages_compact(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  uint64_t k[8];
  if (nargs != 3 || a[0] == Py_None || !numbers_of(a[1], k)) KQ_NONE;
  at::Tensor pairs = pairs_for(k[5], PyLong_AsLongLong(a[2]));
  void* ctx = PyLong_AsVoidPtr(a[0]);
  const uint64_t to = ptr(pairs);
  const int rc = without_gil([&] { return g_compact(ctx, k[0], u32(k[1]), u32(k[2]), k[3], k[4], u32(k[5]), u32(k[6]), k[7], to); });
  return rc != 0 ? status_of(rc) : THPVariable_Wrap(std::move(pairs));
}

// pages_copy(ctx, book args, pairs, pools, device index): tensors, or caches' page_args (pages, bytes of one, address, device); 0, or the status
PyObject* pages_copy(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  uint64_t k[8];
  const at::Tensor *pairs, *t;
  if (nargs != 5 || a[0] == Py_None || !numbers_of(a[1], k) || !tensor_of(a[2], &pairs) || !PyList_CheckExact(a[3])) KQ_NONE;
  const int64_t device = PyLong_AsLongLong(a[4]);
  if (pairs->get_device() != device || pairs->scalar_type() != at::kInt || !plain(*pairs) || pairs->dim() != 2 || pairs->size(1) != 2 || pairs->size(0) >= (1 << 30)) KQ_NONE;
  const Py_ssize_t count = PyList_GET_SIZE(a[3]);
  c10::SmallVector<uint64_t, 128> pools(count), bytes(count);
  for (Py_ssize_t i = 0; i < count; ++i) {
    PyObject* o = PyList_GET_ITEM(a[3], i);
    uint64_t of[4];
    if (tensor_of(o, &t)) {
      // (a pool without pages has no page's bytes: dividing by none would end the process)
      if (t->get_device() != device || !plain(*t) || t->dim() == 0 || t->size(0) == 0 || static_cast<uint64_t>(t->size(0)) < k[5]) KQ_NONE;
      bytes[i] = static_cast<uint64_t>(t->numel() / t->size(0)) * t->element_size();
      pools[i] = ptr(*t);
    } else {
      if (!PyTuple_CheckExact(o) || !numbers_of(o, of) || of[0] < k[5] || static_cast<int64_t>(of[3]) != device) KQ_NONE;
      bytes[i] = of[1];
      pools[i] = of[2];
    }
  }
  void* ctx = PyLong_AsVoidPtr(a[0]);
  const uint64_t pp = ptr(*pairs);
  const uint32_t most = static_cast<uint32_t>(pairs->size(0));
  return status_of(without_gil([&] { return g_copy(ctx, static_cast<uint32_t>(count), pools.data(), bytes.data(), u32(k[5]), pp, most, k[7]); }));
}

// CPython's frames have no handlers: what is thrown in a call must not leave it.
template <PyObject* (*kCall)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* a, Py_ssize_t nargs) {
  try {
    return kCall(self, a, nargs);
  } catch (...) {
    torch::translate_exception_to_python(std::current_exception());
    return nullptr;
  }
}

#define KQ_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<name>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {KQ_METHOD(bind),      KQ_METHOD(linear),    KQ_METHOD(linear_fused), KQ_METHOD(quantize_rows),
                         KQ_METHOD(linear_a8), KQ_METHOD(embedding), KQ_METHOD(rope),   KQ_METHOD(cache_append), KQ_METHOD(cache_read),
                         KQ_METHOD(cache_attention), KQ_METHOD(cache_attention_shared), KQ_METHOD(cache_attention_selected), KQ_METHOD(cache_summarize),
                         KQ_METHOD(cache_select), KQ_METHOD(pages_grow), KQ_METHOD(pages_fork), KQ_METHOD(pages_compact), KQ_METHOD(pages_copy), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kqtorch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__kqtorch() { return PyModule_Create(&module); }
