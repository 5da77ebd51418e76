// The usual call of the package in native code: tensors are checked, workspace and results allocated and the C ABI called
// without a round through the interpreter (16-19 us of host time per call there, 8.5 here; top-k 12.6 and 6.2).  Bound: two
// allocations by torch and two kernel launches.
//
// Only what needs no copy and no message is taken: plain tensors on the current device in a layout the kernels
// read.  Everything else returns None, and the Python functions of flash.py and cache.py, which do the same steps for any input, go on from there.
// Nothing is kept between calls.

#include <Python.h>

#include <ATen/Functions.h>
#include <ATen/core/Tensor.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "fcr.h"

namespace {

PyObject* g_check = nullptr;   // _lib.check: raises for a non-zero return code

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return FCR_DTYPE_F16;
    case at::kBFloat16: return FCR_DTYPE_BF16;
    case at::kFloat: return FCR_DTYPE_F32;
    default: return -1;
  }
}

// A plain dense tensor that is where its type says (no subclass, no wrapper of a transform).
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.has_storage()) return nullptr;
  const c10::DispatchKeySet odd({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                                 c10::DispatchKey::Functionalize, c10::DispatchKey::ZeroTensor, c10::DispatchKey::Negative});
  return t.key_set().has_any(odd) ? nullptr : &t;
}

// The layouts of flash.py::_device_layout that need no copy; strides of dimensions of size one as dense ones, which every
// check accepts.
bool layout(const at::Tensor& t, int64_t (&strides)[4]) {
  const int64_t al = 16 / t.element_size();
  const auto size = t.sizes(), stride = t.strides();
  if (size[3] % al != 0 || stride[3] != 1 || (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) != 0) return false;
  int64_t dense = size[3];
  for (int i = 2; i >= 0; --i) {
    strides[i] = size[i] == 1 ? dense : stride[i];
    if (strides[i] % al != 0 || strides[i] < 0) return false;
    dense = strides[i] * size[i];
  }
  strides[3] = 1;
  return strides[2] * t.element_size() < (1 << 25) && (size[2] <= 1 || strides[2] >= size[3]);
}

PyObject* failed(int rc) {
  PyObject* r = PyObject_CallFunction(g_check, "i", rc);
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "libfcr reported an error");
  return nullptr;
}

// reduce(query, key, reduction, is_causal, scale, out_dtype, pair): the result, (sums or means, maxima) with `pair`, or None.
PyObject* reduce(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS   // (C++ exceptions as the Python ones torch raises for them)
  if (n != 7) {
    PyErr_SetString(PyExc_TypeError, "reduce takes seven arguments");
    return nullptr;
  }
  const at::Tensor* const qp = plain(args[0]);
  const at::Tensor* const kp = plain(args[1]);
  if (!qp || !kp || !PyUnicode_Check(args[2])) Py_RETURN_NONE;
  const at::Tensor &q = *qp, &k = *kp;
  int red;
  if (PyUnicode_CompareWithASCIIString(args[2], "sum") == 0) red = FCR_REDUCE_SUM;
  else if (PyUnicode_CompareWithASCIIString(args[2], "mean") == 0) red = FCR_REDUCE_MEAN;
  else if (PyUnicode_CompareWithASCIIString(args[2], "max") == 0) red = FCR_REDUCE_MAX;
  else Py_RETURN_NONE;
  const int code = dtype_code(q.scalar_type());
  if (code < 0 || k.scalar_type() != q.scalar_type() || q.dim() != 4 || k.dim() != 4 || q.device() != k.device()) Py_RETURN_NONE;
  const auto qs = q.sizes(), ks = k.sizes();
  if (qs[0] != ks[0] || qs[1] != ks[1] || qs[3] != ks[3] || q.numel() == 0 || k.numel() == 0) Py_RETURN_NONE;
  if (qs[3] * q.element_size() > 1024 || qs[0] > INT32_MAX || qs[1] > INT32_MAX || qs[2] > INT32_MAX || ks[2] > INT32_MAX) Py_RETURN_NONE;
  at::ScalarType out_type = q.scalar_type();
  if (args[5] != Py_None) {
    if (!THPDtype_Check(args[5])) Py_RETURN_NONE;
    out_type = reinterpret_cast<THPDtype*>(args[5])->scalar_type;
    if (dtype_code(out_type) < 0) Py_RETURN_NONE;
  }
  double scale;
  if (args[4] == Py_None) scale = 1.0 / std::sqrt((double)qs[3]);
  else if (PyFloat_CheckExact(args[4])) scale = PyFloat_AS_DOUBLE(args[4]);
  else Py_RETURN_NONE;
  const int causal = PyObject_IsTrue(args[3]);
  const int pair = PyObject_IsTrue(args[6]);
  if (causal < 0 || pair < 0) return nullptr;
    int64_t qst[4], kst[4];
    if (!layout(q, qst) || !layout(k, kst) || c10::hip::current_device() != q.device().index()) Py_RETURN_NONE;
    const int b = (int)qs[0], h = (int)qs[1], m = (int)qs[2], nk = (int)ks[2], d = (int)qs[3];
    size_t bytes = fcr_workspace_bytes(code, b, h, m, nk, d);
    const size_t least = 4 * (size_t)b * (size_t)h * (size_t)m;
    if (bytes < least) bytes = least;
    const at::Tensor ws = at::empty({(int64_t)(bytes / 4)}, q.options().dtype(at::kFloat));
    const auto options = q.options().dtype(out_type);
    at::Tensor out = at::empty({qs[0], qs[1], ks[2]}, options), out2;
    if (pair) out2 = at::empty({qs[0], qs[1], ks[2]}, options);
    void* const stream = c10::hip::getCurrentHIPStream(q.device().index()).stream();
    const void *const qd = q.const_data_ptr(), *const kd = k.const_data_ptr();
    void *const wd = ws.mutable_data_ptr(), *const od = out.mutable_data_ptr(), *const od2 = pair ? out2.mutable_data_ptr() : nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fcr_colreduce_ws(qd, kd, od, od2, dtype_code(out_type), wd, bytes, code, b, h, m, nk, d, qst, kst, (float)scale, red, causal, stream);
    Py_END_ALLOW_THREADS
    if (rc) return failed(rc);
    if (!pair) return THPVariable_Wrap(std::move(out));
    PyObject* const a = THPVariable_Wrap(std::move(out));
    PyObject* const z = THPVariable_Wrap(std::move(out2));
    if (a && z) return Py_BuildValue("(NN)", a, z);
    Py_XDECREF(a);
    Py_XDECREF(z);
    return nullptr;
  END_HANDLE_TH_ERRORS
}

// keep(scores, k, with_threshold): the mask, (mask, threshold), or None.
PyObject* keep(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS   // (C++ exceptions as the Python ones torch raises for them)
  if (n != 3) {
    PyErr_SetString(PyExc_TypeError, "keep takes three arguments");
    return nullptr;
  }
  const at::Tensor* const sp = plain(args[0]);
  if (!sp || !PyLong_CheckExact(args[1])) Py_RETURN_NONE;
  const at::Tensor& s = *sp;
  const int code = dtype_code(s.scalar_type());
  int overflow = 0;
  const long long k = PyLong_AsLongLongAndOverflow(args[1], &overflow);
  if (code < 0 || overflow || k > INT32_MAX || k < INT32_MIN || s.dim() < 1 || s.numel() == 0 || !s.is_contiguous()) Py_RETURN_NONE;
  const int with_threshold = PyObject_IsTrue(args[2]);
  if (with_threshold < 0) return nullptr;
  const int64_t cols = s.size(-1), rows = s.numel() / cols;
  if (cols > INT32_MAX) Py_RETURN_NONE;
    if (c10::hip::current_device() != s.device().index()) Py_RETURN_NONE;
    at::Tensor mask = at::empty(s.sizes(), s.options().dtype(at::kBool)), threshold, ws;
    if (with_threshold) threshold = at::empty(s.sizes().slice(0, s.dim() - 1), s.options().dtype(at::kFloat));
    const size_t bytes = fcr_topk_bytes_typed(code, rows, (int)cols);
    if (bytes) ws = at::empty({(int64_t)bytes}, s.options().dtype(at::kByte));
    void* const stream = c10::hip::getCurrentHIPStream(s.device().index()).stream();
    const void* const sd = s.const_data_ptr();
    uint8_t* const md = static_cast<uint8_t*>(mask.mutable_data_ptr());
    float* const td = with_threshold ? static_cast<float*>(threshold.mutable_data_ptr()) : nullptr;
    void* const wd = bytes ? ws.mutable_data_ptr() : nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fcr_topk_mask_typed(sd, code, md, td, rows, (int)cols, (int)k, wd, bytes, stream);
    Py_END_ALLOW_THREADS
    if (rc) return failed(rc);
    if (!with_threshold) return THPVariable_Wrap(std::move(mask));
    PyObject* const a = THPVariable_Wrap(std::move(mask));
    PyObject* const z = THPVariable_Wrap(std::move(threshold));
    if (a && z) return Py_BuildValue("(NN)", a, z);
    Py_XDECREF(a);
    Py_XDECREF(z);
    return nullptr;
  END_HANDLE_TH_ERRORS
}

// The same for the calls on a cache (cache.py): one token of 64 sequences is written every 5 us here, every 18 through Python.
struct Cache {
  fcr_cache c;
  const at::Tensor* k;
};

// A KVCache of plain tensors on the current device; what is left to check is what the library checks.
bool cache_of(PyObject* o, Cache& out) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) return false;
  const at::Tensor *t[4];
  for (int i = 0; i < 4; ++i) {
    PyObject* const x = PyTuple_GET_ITEM(o, i);
    t[i] = x == Py_None ? nullptr : plain(x);
    if (x != Py_None && !t[i]) return false;
  }
  if (!t[0] || !t[1] || t[0]->dim() != 4 || t[0]->sizes() != t[1]->sizes() || t[0]->scalar_type() != t[1]->scalar_type()) return false;
  out.k = t[0];
  bool codes = true;
  switch (t[0]->scalar_type()) {
    case at::kHalf: out.c.dtype = FCR_DTYPE_F16, codes = false; break;
    case at::kBFloat16: out.c.dtype = FCR_DTYPE_BF16, codes = false; break;
    case at::kChar: out.c.dtype = FCR_DTYPE_INT8; break;
    case at::kFloat8_e4m3fn: out.c.dtype = FCR_DTYPE_E4M3; break;
    default: return false;
  }
  const auto size = t[0]->sizes();
  for (int i = 0; i < 4; ++i)
    if (size[i] < 1 || size[i] > INT32_MAX) return false;
  if (size[2] % 16 != 0 || size[3] % 16 != 0 || size[3] > 256 || t[0]->stride(3) != 1 || t[1]->stride(3) != 1) return false;
  out.c.pages = (int)size[0], out.c.H = (int)size[1], out.c.page_size = (int)size[2], out.c.D = (int)size[3];
  const auto device = t[0]->device();
  if (t[1]->device() != device || c10::hip::current_device() != device.index()) return false;
  out.c.k = t[0]->mutable_data_ptr(), out.c.v = t[1]->mutable_data_ptr();
  out.c.k_scale = out.c.v_scale = nullptr;
  for (int i = 0; i < 3; ++i) {
    out.c.k_strides[i] = t[0]->stride(i), out.c.v_strides[i] = t[1]->stride(i);
    out.c.k_scale_strides[i] = out.c.v_scale_strides[i] = 0;
  }
  for (int j = 2; j < 4; ++j) {
    if (codes != (t[j] != nullptr)) return false;
    if (!codes) continue;
    if (t[j]->scalar_type() != at::kFloat || t[j]->sizes() != size.slice(0, 3) || t[j]->device() != device) return false;
    (j == 2 ? out.c.k_scale : out.c.v_scale) = static_cast<float*>(t[j]->mutable_data_ptr());
    for (int i = 0; i < 3; ++i) (j == 2 ? out.c.k_scale_strides : out.c.v_scale_strides)[i] = t[j]->stride(i);
  }
  return true;
}

const at::Tensor* int_tensor(PyObject* o, const Cache& cache) {
  const at::Tensor* const t = plain(o);
  return t && t->scalar_type() == at::kInt && t->device() == cache.k->device() ? t : nullptr;
}

struct Table {
  const int32_t* at;
  int64_t stride;
  int pages, B;
};
bool table_of(PyObject* o, const Cache& cache, Table& out) {
  const at::Tensor* const t = int_tensor(o, cache);
  if (!t || t->dim() != 2 || t->size(0) < 1 || t->size(1) < 1 || t->size(0) > INT32_MAX || t->size(1) > INT32_MAX || (t->size(1) > 1 && t->stride(1) != 1))
    return false;
  out.at = static_cast<const int32_t*>(t->const_data_ptr()), out.stride = t->stride(0), out.pages = (int)t->size(1), out.B = (int)t->size(0);
  return true;
}

struct PerHead {   // int32 (B,) or (B, H)
  const int32_t* at;
  int64_t strides[2];
};
bool lengths_of(PyObject* o, const Cache& cache, int B, PerHead& out) {
  const at::Tensor* const t = int_tensor(o, cache);
  if (!t || t->dim() < 1 || t->dim() > 2 || t->size(0) != B || (t->dim() == 2 && t->size(1) != cache.c.H)) return false;
  out.at = static_cast<const int32_t*>(t->const_data_ptr());
  out.strides[0] = t->stride(0), out.strides[1] = t->dim() == 2 ? t->stride(1) : 0;
  return true;
}

// Rows that are read in place (cache.py::_rows).
bool rows_of(const at::Tensor& t, int64_t (&strides)[4]) {
  const int64_t al = 16 / t.element_size();
  if (t.stride(3) != 1 || (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) != 0) return false;
  for (int i = 0; i < 4; ++i) {
    strides[i] = t.stride(i);
    if (i < 3 && t.size(i) != 1 && strides[i] % al != 0) return false;
  }
  return true;
}

void* stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

PyObject* two(at::Tensor&& x, at::Tensor&& y) {
  PyObject* const a = THPVariable_Wrap(std::move(x));
  PyObject* const z = THPVariable_Wrap(std::move(y));
  if (a && z) return Py_BuildValue("(NN)", a, z);
  Py_XDECREF(a);
  Py_XDECREF(z);
  return nullptr;
}

// cache_write(cache, key, value, table, start, counts): True, or None.
PyObject* cache_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) {
    PyErr_SetString(PyExc_TypeError, "cache_write takes six arguments");
    return nullptr;
  }
  Cache cache;
  Table table;
  PerHead start, counts;
  const at::Tensor *const k = plain(args[1]), *const v = plain(args[2]);
  if (!k || !v || !cache_of(args[0], cache) || !table_of(args[3], cache, table) || !lengths_of(args[4], cache, table.B, start)) Py_RETURN_NONE;
  if (args[5] != Py_None && !lengths_of(args[5], cache, table.B, counts)) Py_RETURN_NONE;
  const int code = dtype_code(k->scalar_type());
  int64_t ks[4], vs[4];
  if (code < 0 || v->scalar_type() != k->scalar_type() || k->dim() != 4 || k->sizes() != v->sizes() || k->size(0) != table.B || k->size(1) != cache.c.H ||
      k->size(2) < 1 || k->size(2) > INT32_MAX || k->size(3) != cache.c.D || k->device() != cache.k->device() || v->device() != k->device() ||
      !rows_of(*k, ks) || !rows_of(*v, vs))
    Py_RETURN_NONE;
  const bool counted = args[5] != Py_None;
  const int T = (int)k->size(2);
  const void *const kd = k->const_data_ptr(), *const vd = v->const_data_ptr();
  void* const stream = stream_of(*cache.k);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = fcr_cache_write(&cache.c, table.at, table.stride, table.pages, start.at, start.strides, counted ? counts.at : nullptr,
                       counted ? counts.strides : nullptr, kd, vd, code, table.B, T, ks, vs, stream);
  Py_END_ALLOW_THREADS
  if (rc) return failed(rc);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// cache_read(cache, table, lengths, n, out_dtype): (key, value), or None.
PyObject* cache_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "cache_read takes five arguments");
    return nullptr;
  }
  Cache cache;
  Table table;
  PerHead lengths;
  if (!PyLong_CheckExact(args[3]) || !cache_of(args[0], cache) || !table_of(args[1], cache, table) || !lengths_of(args[2], cache, table.B, lengths))
    Py_RETURN_NONE;
  int overflow = 0;
  const long long rows = PyLong_AsLongLongAndOverflow(args[3], &overflow);
  if (overflow || rows < 1 || rows > INT32_MAX) Py_RETURN_NONE;
  at::ScalarType type = cache.c.k_scale ? at::kBFloat16 : cache.k->scalar_type();
  if (args[4] != Py_None) {
    if (!THPDtype_Check(args[4])) Py_RETURN_NONE;
    type = reinterpret_cast<THPDtype*>(args[4])->scalar_type;
  }
  const int code = dtype_code(type);
  if (code < 0) Py_RETURN_NONE;
  const auto options = cache.k->options().dtype(type);
  at::Tensor k = at::empty({table.B, cache.c.H, (int64_t)rows, cache.c.D}, options), v = at::empty(k.sizes(), options);
  void *const kd = k.mutable_data_ptr(), *const vd = v.mutable_data_ptr(), *const stream = stream_of(*cache.k);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = fcr_cache_read(&cache.c, table.at, table.stride, table.pages, lengths.at, lengths.strides, kd, vd, code, table.B, (int)rows, stream);
  Py_END_ALLOW_THREADS
  if (rc) return failed(rc);
  return two(std::move(k), std::move(v));
  END_HANDLE_TH_ERRORS
}

// cache_keep(cache, table, lengths, keep, into, into_table): the counts, or None.
PyObject* cache_keep(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) {
    PyErr_SetString(PyExc_TypeError, "cache_keep takes six arguments");
    return nullptr;
  }
  Cache cache, into;
  Table table, into_table;
  PerHead lengths;
  const at::Tensor* const mask = plain(args[3]);
  if (!mask || !cache_of(args[0], cache) || !cache_of(args[4], into) || !table_of(args[1], cache, table) || !table_of(args[5], into, into_table) ||
      !lengths_of(args[2], cache, table.B, lengths))
    Py_RETURN_NONE;
  if (into.c.dtype != cache.c.dtype || into.c.H != cache.c.H || into.c.D != cache.c.D || into.k->device() != cache.k->device() || into_table.B != table.B ||
      mask->scalar_type() != at::kBool || mask->dim() != 3 || mask->size(0) != table.B || mask->size(1) != cache.c.H || mask->size(2) < 1 ||
      mask->size(2) > INT32_MAX || mask->device() != cache.k->device() || !mask->is_contiguous() ||
      (into.c.k == cache.c.k && into_table.at == table.at))
    Py_RETURN_NONE;
  at::Tensor counts = at::empty({table.B, cache.c.H}, cache.k->options().dtype(at::kInt));
  const uint8_t* const md = static_cast<const uint8_t*>(mask->const_data_ptr());
  int32_t* const cd = static_cast<int32_t*>(counts.mutable_data_ptr());
  const int rows = (int)mask->size(2);
  void* const stream = stream_of(*cache.k);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = fcr_cache_keep(&cache.c, table.at, table.stride, table.pages, lengths.at, lengths.strides, md, rows, &into.c, into_table.at, into_table.stride,
                      into_table.pages, cd, table.B, stream);
  Py_END_ALLOW_THREADS
  if (rc) return failed(rc);
  return THPVariable_Wrap(std::move(counts));
  END_HANDLE_TH_ERRORS
}

// tree_attention(query, cache, table, context, tree_mask, scale, tree_lengths, with_lse): the result, (result, log-sum-exp), or None.
PyObject* tree_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) {
    PyErr_SetString(PyExc_TypeError, "tree_attention takes eight arguments");
    return nullptr;
  }
  Cache cache;
  Table table;
  PerHead context;
  const at::Tensor* const qp = plain(args[0]);
  if (!qp || !cache_of(args[1], cache) || !table_of(args[2], cache, table) || !lengths_of(args[3], cache, table.B, context)) Py_RETURN_NONE;
  const at::Tensor& q = *qp;
  const int code = dtype_code(q.scalar_type()), H = cache.c.H;
  int64_t qs[4];
  if ((code != FCR_DTYPE_F16 && code != FCR_DTYPE_BF16) || (!cache.c.k_scale && code != cache.c.dtype) || q.dim() != 4 || q.size(0) != table.B ||
      q.size(1) < 1 || q.size(1) % H != 0 || q.size(1) > INT32_MAX || q.size(2) < 1 || q.size(2) > INT32_MAX || q.size(3) != cache.c.D ||
      q.device() != cache.k->device() || !rows_of(q, qs))
    Py_RETURN_NONE;
  const int64_t T = q.size(2);
  const uint8_t* mask = nullptr;
  int64_t mask_stride = 0;
  if (args[4] != Py_None) {
    const at::Tensor* const m = plain(args[4]);
    if (!m || m->scalar_type() != at::kBool || m->device() != q.device() || !m->is_contiguous() || m->dim() < 2 || m->dim() > 3 ||
        m->size(-1) != T || m->size(-2) != T || (m->dim() == 3 && m->size(0) != table.B))
      Py_RETURN_NONE;
    mask = static_cast<const uint8_t*>(m->const_data_ptr());
    mask_stride = m->dim() == 3 ? T * T : 0;
  }
  double scale;
  if (args[5] == Py_None) scale = 1.0 / std::sqrt((double)cache.c.D);
  else if (PyFloat_CheckExact(args[5])) scale = PyFloat_AS_DOUBLE(args[5]);
  else Py_RETURN_NONE;
  const int32_t* tree_lengths = nullptr;
  if (args[6] != Py_None) {
    const at::Tensor* const t = int_tensor(args[6], cache);
    if (!t || t->dim() != 1 || t->size(0) != table.B || !t->is_contiguous()) Py_RETURN_NONE;
    tree_lengths = static_cast<const int32_t*>(t->const_data_ptr());
  }
  const int with_lse = PyObject_IsTrue(args[7]);
  if (with_lse < 0) return nullptr;
  const int G = (int)q.size(1) / H;
  const size_t bytes = fcr_tree_attention_bytes(table.B, H, G, (int)T, cache.c.D, (int64_t)table.pages * cache.c.page_size);
  if (!bytes) Py_RETURN_NONE;
  at::Tensor out = at::empty(q.sizes(), q.options()), lse;
  if (with_lse) lse = at::empty(q.sizes().slice(0, 3), q.options().dtype(at::kFloat));
  const at::Tensor ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
  const void* const qd = q.const_data_ptr();
  void *const od = out.mutable_data_ptr(), *const wd = ws.mutable_data_ptr(), *const stream = stream_of(q);
  float* const ld = with_lse ? static_cast<float*>(lse.mutable_data_ptr()) : nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = fcr_tree_attention(qd, &cache.c, table.at, table.stride, table.pages, context.at, context.strides, mask, mask_stride, tree_lengths, od, ld, wd, bytes,
                          code, table.B, G, (int)T, qs, (float)scale, stream);
  Py_END_ALLOW_THREADS
  if (rc) return failed(rc);
  if (!with_lse) return THPVariable_Wrap(std::move(out));
  return two(std::move(out), std::move(lse));
  END_HANDLE_TH_ERRORS
}

PyObject* on_error(PyObject*, PyObject* f) {
  Py_INCREF(f);
  Py_XSETREF(g_check, f);
  Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"reduce", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(reduce)), METH_FASTCALL, "reduce(query, key, reduction, is_causal, scale, out_dtype, pair)"},
    {"keep", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(keep)), METH_FASTCALL, "keep(scores, k, with_threshold)"},
    {"cache_write", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(cache_write)), METH_FASTCALL, "cache_write(cache, key, value, table, start, counts)"},
    {"cache_read", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(cache_read)), METH_FASTCALL, "cache_read(cache, table, lengths, n, out_dtype)"},
    {"cache_keep", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(cache_keep)), METH_FASTCALL, "cache_keep(cache, table, lengths, keep, into, into_table)"},
    {"tree_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(tree_attention)), METH_FASTCALL, "tree_attention(query, cache, table, context, tree_mask, scale, tree_lengths, with_lse)"},
    {"on_error", on_error, METH_O, "on_error(f): f(rc) raises for a return code of the library"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_host", "the usual call in native code", -1, g_methods};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&g_module); }
