// Argument path of the paged-cache ops from Python: reads the tensors, makes
// the outputs and calls the C ABI (include/ssa_b200.h).
//
// These ops run once per layer and token, so what a call costs on the host is
// what a small batch runs at; the same steps in Python through ctypes took about
// three times as long.  Only the plain case is handled here -- tensors of the
// right kinds, shapes and device, contiguous last dimensions, the current
// device -- and everything else is left to the Python code (ssa_b200/paged.py),
// which names what is wrong or makes the copies: these functions then return None
// and have done nothing.
#include <ATen/ATen.h>
#include <Python.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "../../include/ssa_b200.h"

namespace {

decltype(&ssa_paged_append) g_append;
decltype(&ssa_paged_attn_workspace_size) g_attn_size;
decltype(&ssa_paged_attn) g_attn;
decltype(&ssa_paged_evict) g_evict;

bool cuda_tensor(PyObject* o) { return THPVariable_Check(o) && THPVariable_Unpack(o).is_cuda(); }

bool dtype_of(const at::Tensor& t, ssa_dtype* d) {
  switch (t.scalar_type()) {
    case at::kFloat: *d = SSA_F32; return true;
    case at::kBFloat16: *d = SSA_BF16; return true;
    case at::kHalf: *d = SSA_F16; return true;
    default: return false;
  }
}

// int32 indices on device `dev`, contiguous rows.
bool index_of(PyObject* o, int dev, int dims, at::Tensor* t) {
  if (!cuda_tensor(o)) return false;
  *t = THPVariable_Unpack(o);
  return t->scalar_type() == at::kInt && t->dim() == dims && t->get_device() == dev && t->stride(dims - 1) == 1;
}

// The cache part common to the ops; false: not the plain case.
bool cache_of(PyObject* kp, PyObject* vp, PyObject* table, PyObject* lens, PyObject* weights, PyObject* word,
              SsaPagedCache* c, int* dev, at::Tensor* lens_t) {
  if (!cuda_tensor(kp) || !cuda_tensor(vp)) return false;
  const at::Tensor &k = THPVariable_Unpack(kp), &v = THPVariable_Unpack(vp);
  *dev = k.get_device();
  if (*dev != c10::cuda::current_device() || v.get_device() != *dev || k.dim() != 4 || k.sizes() != v.sizes() ||
      k.scalar_type() != v.scalar_type() || k.stride(3) != 1 || v.stride(3) != 1 || !dtype_of(k, &c->dtype))
    return false;
  at::Tensor t;
  if (!index_of(lens, *dev, 1, lens_t) || !index_of(table, *dev, 2, &t) || t.size(0) != lens_t->size(0)) return false;
  if (k.size(1) > 1024 || k.size(2) > 65535 || k.size(3) > 256 || t.size(0) > 65535 || t.size(1) > INT32_MAX) return false;
  c->batch = static_cast<int32_t>(t.size(0));
  c->max_pages = static_cast<int32_t>(t.size(1));
  c->num_pages = k.size(0);
  c->page_size = static_cast<int32_t>(k.size(1));
  c->h_kv = static_cast<int32_t>(k.size(2));
  c->d = static_cast<int32_t>(k.size(3));
  c->k_pages = k.data_ptr();
  c->k_stride_p = k.stride(0);
  c->k_stride_n = k.stride(1);
  c->k_stride_h = k.stride(2);
  c->v_pages = v.data_ptr();
  c->v_stride_p = v.stride(0);
  c->v_stride_n = v.stride(1);
  c->v_stride_h = v.stride(2);
  c->weights = nullptr;
  c->w_stride_p = c->w_stride_n = c->w_stride_h = 0;
  if (weights != Py_None) {
    if (!cuda_tensor(weights)) return false;
    const at::Tensor& w = THPVariable_Unpack(weights);
    if (w.get_device() != *dev || w.scalar_type() != at::kFloat || w.dim() != 3 || w.sizes() != k.sizes().slice(0, 3))
      return false;
    c->weights = static_cast<float*>(w.data_ptr());
    c->w_stride_p = w.stride(0);
    c->w_stride_n = w.stride(1);
    c->w_stride_h = w.stride(2);
  }
  c->page_table = static_cast<const int32_t*>(t.data_ptr());
  c->table_stride = t.stride(0);
  c->kv_lens = static_cast<const int32_t*>(lens_t->data_ptr());
  c->status = word == Py_None ? nullptr : static_cast<int32_t*>(PyLong_AsVoidPtr(word));
  return true;
}

// [rows, heads, d] of the cache's device and type, last dimension contiguous.
bool rows_of(PyObject* o, const SsaPagedCache& c, int dev, at::Tensor* t) {
  if (!cuda_tensor(o)) return false;
  *t = THPVariable_Unpack(o);
  ssa_dtype dt;
  return t->get_device() == dev && dtype_of(*t, &dt) && dt == c.dtype && t->dim() == 3 && t->size(2) == c.d &&
         t->stride(2) == 1;
}

void* stream_of(int dev) {
  return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream();
}

PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 4) {
    PyErr_SetString(PyExc_TypeError, "bind takes four addresses");
    return nullptr;
  }
  g_append = reinterpret_cast<decltype(g_append)>(PyLong_AsVoidPtr(a[0]));
  g_attn_size = reinterpret_cast<decltype(g_attn_size)>(PyLong_AsVoidPtr(a[1]));
  g_attn = reinterpret_cast<decltype(g_attn)>(PyLong_AsVoidPtr(a[2]));
  g_evict = reinterpret_cast<decltype(g_evict)>(PyLong_AsVoidPtr(a[3]));
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

// append(k_new, v_new, k_pages, v_pages, page_table, q_starts, kv_lens, weights, word) -> status or None
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  SsaPagedCache c;
  int dev;
  at::Tensor lens, k, v, starts;
  if (n != 9 || !cache_of(a[2], a[3], a[4], a[6], a[7], a[8], &c, &dev, &lens) || !rows_of(a[0], c, dev, &k) ||
      !rows_of(a[1], c, dev, &v) || k.sizes() != v.sizes() || k.size(1) != c.h_kv || !index_of(a[5], dev, 1, &starts) ||
      starts.size(0) != c.batch + 1)
    Py_RETURN_NONE;
  SsaPagedAppendArgs p;
  p.rows = k.size(0);
  p.q_starts = static_cast<const int32_t*>(starts.data_ptr());
  p.k_new = k.data_ptr();
  p.k_new_stride_n = k.stride(0);
  p.k_new_stride_h = k.stride(1);
  p.v_new = v.data_ptr();
  p.v_new_stride_n = v.stride(0);
  p.v_new_stride_h = v.stride(1);
  return PyLong_FromLong(g_append(&c, &p, stream_of(dev)));
  END_HANDLE_TH_ERRORS
}

// attend(q, k_pages, v_pages, page_table, q_starts, kv_lens, scale or None, is_causal, weights, return_lse, word,
//        workspace) -> (status, out, lse or None) or None (also where the workspace is too small)
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  SsaPagedCache c;
  int dev;
  at::Tensor lens, q, starts;
  if (n != 12 || !cache_of(a[1], a[2], a[3], a[5], a[8], a[10], &c, &dev, &lens) || !rows_of(a[0], c, dev, &q) ||
      c.h_kv < 1 || q.size(1) % c.h_kv != 0 || q.size(1) > INT32_MAX || !index_of(a[4], dev, 1, &starts) ||
      starts.size(0) != c.batch + 1 || !cuda_tensor(a[11]))
    Py_RETURN_NONE;
  const at::Tensor& ws = THPVariable_Unpack(a[11]);
  SsaPagedAttnArgs p;
  p.rows = q.size(0);
  p.q_starts = static_cast<const int32_t*>(starts.data_ptr());
  p.h_q = static_cast<int32_t>(q.size(1));
  p.causal = PyObject_IsTrue(a[7]);
  if (a[6] == Py_None) {
    p.scale = static_cast<float>(std::sqrt(static_cast<double>(c.d)));
  } else {
    p.scale = static_cast<float>(PyFloat_AsDouble(a[6]));
  }
  if (PyErr_Occurred()) return nullptr;
  p.q = q.data_ptr();
  p.q_stride_n = q.stride(0);
  p.q_stride_h = q.stride(1);
  p.out_stride_n = q.size(1) * q.size(2);
  p.out_stride_h = q.size(2);
  p.out = nullptr;
  p.lse = nullptr;
  const at::Tensor out = at::empty(q.sizes(), q.options());
  p.out = out.data_ptr();
  const size_t bytes = g_attn_size(&c, &p);
  if (bytes > static_cast<size_t>(ws.numel()) || ws.get_device() != dev) Py_RETURN_NONE;
  at::Tensor lse;
  if (PyObject_IsTrue(a[9])) {
    lse = at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat));
    p.lse = static_cast<float*>(lse.data_ptr());
  }
  const long status = g_attn(&c, &p, ws.data_ptr(), bytes, stream_of(dev));
  PyObject* r = PyTuple_New(3);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, PyLong_FromLong(status));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(out));
  if (lse.defined()) {
    PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(lse));
  } else {
    Py_INCREF(Py_None);
    PyTuple_SET_ITEM(r, 2, Py_None);
  }
  return r;
  END_HANDLE_TH_ERRORS
}

// evict(k_pages, v_pages, weights, page_table, kv_lens, new_table, budget, recent, word) -> (status, kept, lens) or None
PyObject* evict(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  SsaPagedCache c;
  int dev;
  at::Tensor lens, table;
  if (n != 9 || a[2] == Py_None || !cache_of(a[0], a[1], a[3], a[4], a[2], a[8], &c, &dev, &lens) ||
      !index_of(a[5], dev, 2, &table) || table.size(0) != c.batch || table.size(1) > INT32_MAX)
    Py_RETURN_NONE;
  const long long budget = PyLong_AsLongLong(a[6]), recent = PyLong_AsLongLong(a[7]);
  if (PyErr_Occurred()) return nullptr;
  if (budget < 1 || budget > INT32_MAX || recent < 0 || recent > budget) Py_RETURN_NONE;
  const at::Tensor kept = at::empty({c.batch, c.h_kv, budget}, lens.options());
  const at::Tensor new_lens = at::empty({c.batch}, lens.options());
  SsaPagedEvictArgs p;
  p.budget = static_cast<int32_t>(budget);
  p.recent = static_cast<int32_t>(recent);
  p.new_max_pages = static_cast<int32_t>(table.size(1));
  p.new_table = static_cast<const int32_t*>(table.data_ptr());
  p.new_table_stride = table.stride(0);
  p.kept = static_cast<int32_t*>(kept.data_ptr());
  p.new_lens = static_cast<int32_t*>(new_lens.data_ptr());
  const long status = g_evict(&c, &p, stream_of(dev));
  PyObject* r = PyTuple_New(3);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, PyLong_FromLong(status));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(kept));
  PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(new_lens));
  return r;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(bind)), METH_FASTCALL, nullptr},
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(append)), METH_FASTCALL, nullptr},
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(attend)), METH_FASTCALL, nullptr},
    {"evict", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(evict)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged_call(void) { return PyModule_Create(&module); }
