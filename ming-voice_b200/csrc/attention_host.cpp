// Host side of the attention calls (mingmoe/attention.py) in C++: reads the tensors, allocates the result, fills the C
// entry points' argument structs.
//
// A decode step's kernels take 3 to 10 us, and reading some 40 sizes, strides and addresses through Python attributes
// takes 5 to 7 us of every call. Here it takes under one. Only the plain case is handled: exact tensors on the cache's
// device with the right types, shapes and strides and a workspace that exists already. For anything else a function
// returns NotImplemented, and the Python code, which has the same checks, copies or refuses. The entry points are given
// by address (bind), so they are the ones of the library that mingmoe/_lib.py loaded.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <vector>

#include "../../include/mingmoe.h"

namespace {

int (*g_append)(const mv_kv_append_args*, void*, size_t, void*) = nullptr;
int (*g_paged)(const mv_attention_args*, void*, size_t, void*) = nullptr;
int (*g_prompt)(const mv_attention_args*, void*, size_t, void*) = nullptr;

struct Workspace {
  int device;
  void* stream;
  void* ptr;
  size_t bytes;
};
std::vector<Workspace>& workspaces() {  // under the GIL
  static std::vector<Workspace> w;
  return w;
}

struct Launch {
  void *stream, *ws;
  size_t bytes;
  // false also where another device is current: the entry points launch on the current one, and the Python code changes it
  bool find(int device) {
    if (c10::cuda::current_device() != device) return false;
    stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
    for (const Workspace& w : workspaces())
      if (w.device == device && w.stream == stream) {
        ws = w.ptr;
        bytes = w.bytes;
        return true;
      }
    return false;
  }
};

bool tensor(PyObject* o) { return THPVariable_CheckExact(o); }

bool on(const at::Tensor& t, int device) { return t.is_cuda() && t.device().index() == device; }

// a [T, heads, d] operand that the kernels take as it is
bool rows(PyObject* o, int d, at::ScalarType type, int device, const at::Tensor** out) {
  if (!tensor(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  *out = &t;
  if (t.dim() != 3 || t.scalar_type() != type || !on(t, device) || t.size(2) != d || t.stride(2) != 1) return false;
  const int64_t st = t.stride(0), sh = t.stride(1);
  return ((st | sh) & 7) == 0 && st >= d && sh >= d && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
}

bool ints(PyObject* o, int dim, int device, const at::Tensor** out) {
  if (!tensor(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  *out = &t;
  return t.dim() == dim && t.scalar_type() == at::kInt && on(t, device) &&
         (t.size(dim - 1) <= 1 || t.stride(dim - 1) == 1);
}

// the caller's result buffer, or a new one
bool result(PyObject* o, const at::Tensor& like, at::Tensor* out) {
  if (o == Py_None) {
    *out = at::empty_like(like);
    return out->stride(2) == 1;
  }
  if (!tensor(o)) return false;
  *out = THPVariable_Unpack(o);
  return out->sizes() == like.sizes() && out->scalar_type() == like.scalar_type() && out->device() == like.device() &&
         out->stride(2) == 1;
}

struct Batch {
  const at::Tensor *table, *cu, *lens;
  int B;
  bool read(PyObject* t, PyObject* c, PyObject* l, int device) {
    if (!ints(l, 1, device, &lens) || !ints(c, 1, device, &cu) || !ints(t, 2, device, &table)) return false;
    B = static_cast<int>(lens->size(0));
    return cu->size(0) == B + 1 && table->size(0) == B;
  }
};

const int* iptr(const at::Tensor* t) { return static_cast<const int*>(t->data_ptr()); }

at::ScalarType type_of(int code) { return code == MV_BF16 ? at::kBFloat16 : at::kHalf; }

PyObject* plain_not() { Py_RETURN_NOTIMPLEMENTED; }

bool number(PyObject* o, double* v) {
  *v = PyFloat_AsDouble(o);
  if (*v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

bool integer(PyObject* o, long* v) {
  if (!PyLong_Check(o)) return false;
  *v = PyLong_AsLong(o);
  if (*v == -1 && PyErr_Occurred()) PyErr_Clear();
  return *v >= 0 && *v <= 0x7fffffff;
}

bool flag(PyObject* o, bool* v) {
  const int t = PyObject_IsTrue(o);
  if (t < 0) PyErr_Clear();  // the Python code meets it again and raises
  *v = t == 1;
  return t >= 0;
}

PyObject* wrap(const at::Tensor& out, const at::Tensor& lse) {
  PyObject* o = THPVariable_Wrap(out);
  if (!lse.defined() || o == nullptr) return o;
  PyObject* l = THPVariable_Wrap(lse);
  return l == nullptr ? nullptr : Py_BuildValue("NN", o, l);
}

// scale, causal, return_lse, max_q of the attention calls
bool options(PyObject* max_q, PyObject* scale, PyObject* causal, PyObject* return_lse, int d, mv_attention_args* a,
             bool* with_lse) {
  bool c;
  if (!flag(causal, &c) || !flag(return_lse, with_lse)) return false;
  long m = a->T;
  if (max_q != Py_None && !integer(max_q, &m)) return false;
  double s = 1.0 / std::sqrt(static_cast<double>(d));
  if (scale != Py_None && !number(scale, &s)) return false;
  a->max_q = static_cast<int>(m);
  a->scale = static_cast<float>(s);
  a->causal = c;
  return true;
}

PyObject* guarded(PyObject* (*f)(PyObject* const*), PyObject* const* args) {
  try {
    return f(args);
  } catch (const std::exception&) {  // an allocation that failed: the Python code meets it again and raises torch's error
    return plain_not();
  }
}

// kv_append(cache address, device, k, v, page_table, cu_seqlens, kv_lens, q, q_out, cos_sin, positions, interleaved)
PyObject* append_impl(PyObject* const* o) {
  const auto* c = static_cast<const mv_paged_kv*>(PyLong_AsVoidPtr(o[0]));
  const int dev = static_cast<int>(PyLong_AsLong(o[1])), d = c->head_dim;
  const at::ScalarType type = type_of(c->dtype);
  const at::Tensor *k, *v, *q = nullptr;
  Batch b;
  Launch l;
  if (!rows(o[2], d, type, dev, &k) || !rows(o[3], d, type, dev, &v) || !b.read(o[4], o[5], o[6], dev))
    return plain_not();
  const int64_t T = k->size(0);
  if (k->size(1) != c->n_kv_heads || v->sizes() != k->sizes() || T > 0x7fffffff) return plain_not();
  mv_kv_append_args a{};
  a.cache = c;
  a.k = k->data_ptr(), a.v = v->data_ptr();
  a.k_st = k->stride(0), a.k_sh = k->stride(1), a.v_st = v->stride(0), a.v_sh = v->stride(1);
  a.page_table = iptr(b.table), a.cu_seqlens = iptr(b.cu), a.kv_lens = iptr(b.lens);
  a.pt_stride = b.table->stride(0), a.max_pages = static_cast<int>(b.table->size(1));
  a.T = static_cast<int>(T), a.B = b.B;
  if (o[9] != Py_None) {
    if (!tensor(o[9])) return plain_not();
    const at::Tensor& cs = THPVariable_Unpack(o[9]);
    if (cs.dim() != 2 || cs.scalar_type() != at::kFloat || !on(cs, dev) || cs.stride(1) != 1) return plain_not();
    a.cos_sin = static_cast<const float*>(cs.data_ptr());
    a.cs_stride = cs.stride(0), a.max_pos = static_cast<int>(cs.size(0)), a.rot_dim = static_cast<int>(cs.size(1));
  }
  if (o[10] != Py_None) {
    const at::Tensor* pos;
    if (!ints(o[10], 1, dev, &pos) || pos->size(0) != T) return plain_not();
    a.positions = iptr(pos);
  }
  bool interleaved;
  if (!flag(o[11], &interleaved)) return plain_not();
  a.interleaved = interleaved;
  at::Tensor qo;
  if (o[7] != Py_None) {
    if (!rows(o[7], d, type, dev, &q) || q->size(0) != T || !l.find(dev) || !result(o[8], *q, &qo)) return plain_not();
    a.q = q->data_ptr(), a.q_out = qo.data_ptr(), a.Hq = static_cast<int>(q->size(1));
    a.q_st = q->stride(0), a.q_sh = q->stride(1), a.qo_st = qo.stride(0), a.qo_sh = qo.stride(1);
  } else if (o[8] != Py_None || !l.find(dev)) {
    return plain_not();
  }
  const int rc = g_append(&a, l.ws, l.bytes, l.stream);
  if (rc != MV_OK) return PyLong_FromLong(rc);
  if (q == nullptr) Py_RETURN_NONE;
  return wrap(qo, at::Tensor());
}

// paged_attention(cache address, device, q, page_table, cu_seqlens, kv_lens, max_q, scale, causal, out, return_lse)
PyObject* paged_impl(PyObject* const* o) {
  const auto* c = static_cast<const mv_paged_kv*>(PyLong_AsVoidPtr(o[0]));
  const int dev = static_cast<int>(PyLong_AsLong(o[1])), d = c->head_dim;
  const at::Tensor* q;
  Batch b;
  Launch l;
  mv_attention_args a{};
  if (!rows(o[2], d, type_of(c->dtype), dev, &q) || !b.read(o[3], o[4], o[5], dev) || q->size(0) > 0x7fffffff)
    return plain_not();
  a.T = static_cast<int>(q->size(0)), a.Hq = static_cast<int>(q->size(1)), a.B = b.B;
  at::Tensor out, lse;
  bool with_lse;
  if (!options(o[6], o[7], o[8], o[10], d, &a, &with_lse) || !l.find(dev) || !result(o[9], *q, &out)) return plain_not();
  if (with_lse) lse = at::empty({a.T, a.Hq}, q->options().dtype(at::kFloat));
  a.cache = c;
  a.q = q->data_ptr(), a.out = out.data_ptr();
  a.lse = lse.defined() ? static_cast<float*>(lse.data_ptr()) : nullptr;
  a.cu_seqlens = iptr(b.cu), a.page_table = iptr(b.table), a.kv_lens = iptr(b.lens);
  a.q_st = q->stride(0), a.q_sh = q->stride(1), a.o_st = out.stride(0), a.o_sh = out.stride(1);
  a.pt_stride = b.table->stride(0), a.max_pages = static_cast<int>(b.table->size(1));
  const int rc = g_paged(&a, l.ws, l.bytes, l.stream);
  return rc != MV_OK ? PyLong_FromLong(rc) : wrap(out, lse);
}

// prompt_attention(q, k, v, cu_seqlens, cu_seqlens_k, max_q, scale, causal, out, return_lse)
PyObject* prompt_impl(PyObject* const* o) {
  if (!tensor(o[0])) return plain_not();
  const at::Tensor& q = THPVariable_Unpack(o[0]);
  if (q.dim() != 3 || !q.is_cuda() || (q.scalar_type() != at::kBFloat16 && q.scalar_type() != at::kHalf))
    return plain_not();
  const int dev = q.device().index(), d = static_cast<int>(q.size(2));
  const at::Tensor *pq, *k, *v, *cu, *cuk = nullptr;
  if (!rows(o[0], d, q.scalar_type(), dev, &pq) || !rows(o[1], d, q.scalar_type(), dev, &k) ||
      !rows(o[2], d, q.scalar_type(), dev, &v) || !ints(o[3], 1, dev, &cu))
    return plain_not();
  if (v->sizes() != k->sizes() || q.size(0) > 0x7fffffff || k->size(0) > 0x7fffffff || cu->size(0) < 1)
    return plain_not();
  if (o[4] != Py_None) {
    if (!ints(o[4], 1, dev, &cuk) || cuk->size(0) != cu->size(0)) return plain_not();
  } else if (k->size(0) != q.size(0)) {
    return plain_not();
  }
  Launch l;
  mv_attention_args a{};
  a.T = static_cast<int>(q.size(0)), a.Hq = static_cast<int>(q.size(1)), a.B = static_cast<int>(cu->size(0)) - 1;
  at::Tensor out, lse;
  bool with_lse;
  if (!options(o[5], o[6], o[7], o[9], d, &a, &with_lse) || !l.find(dev) || !result(o[8], q, &out)) return plain_not();
  if (with_lse) lse = at::empty({a.T, a.Hq}, q.options().dtype(at::kFloat));
  a.q = q.data_ptr(), a.k = k->data_ptr(), a.v = v->data_ptr(), a.out = out.data_ptr();
  a.lse = lse.defined() ? static_cast<float*>(lse.data_ptr()) : nullptr;
  a.cu_seqlens = iptr(cu), a.cu_seqlens_k = cuk == nullptr ? nullptr : iptr(cuk);
  a.q_st = q.stride(0), a.q_sh = q.stride(1), a.o_st = out.stride(0), a.o_sh = out.stride(1);
  a.k_st = k->stride(0), a.k_sh = k->stride(1), a.v_st = v->stride(0), a.v_sh = v->stride(1);
  a.Tk = static_cast<int>(k->size(0)), a.Hkv = static_cast<int>(k->size(1)), a.head_dim = d;
  a.dtype = q.scalar_type() == at::kBFloat16 ? MV_BF16 : MV_F16;
  const int rc = g_prompt(&a, l.ws, l.bytes, l.stream);
  return rc != MV_OK ? PyLong_FromLong(rc) : wrap(out, lse);
}

PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) { return n == 12 ? guarded(append_impl, a) : plain_not(); }
PyObject* paged(PyObject*, PyObject* const* a, Py_ssize_t n) { return n == 11 ? guarded(paged_impl, a) : plain_not(); }
PyObject* prompt(PyObject*, PyObject* const* a, Py_ssize_t n) { return n == 10 ? guarded(prompt_impl, a) : plain_not(); }

// bind(address of mv_kv_append, of mv_paged_attention, of mv_prompt_attention)
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long f[3];
  if (!PyArg_ParseTuple(args, "KKK", &f[0], &f[1], &f[2])) return nullptr;
  g_append = reinterpret_cast<decltype(g_append)>(f[0]);
  g_paged = reinterpret_cast<decltype(g_paged)>(f[1]);
  g_prompt = reinterpret_cast<decltype(g_prompt)>(f[2]);
  Py_RETURN_NONE;
}

// workspace(device, stream, address, bytes): the buffer of a stream's calls
PyObject* workspace(PyObject*, PyObject* args) {
  int device;
  unsigned long long stream, ptr, bytes;
  if (!PyArg_ParseTuple(args, "iKKK", &device, &stream, &ptr, &bytes)) return nullptr;
  workspaces().push_back(Workspace{device, reinterpret_cast<void*>(stream), reinterpret_cast<void*>(ptr),
                                   static_cast<size_t>(bytes)});
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"kv_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(append)), METH_FASTCALL, nullptr},
    {"paged_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(paged)), METH_FASTCALL, nullptr},
    {"prompt_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(prompt)), METH_FASTCALL, nullptr},
    {"bind", bind, METH_VARARGS, nullptr},
    {"workspace", workspace, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_attention_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__attention_host() { return PyModule_Create(&module); }
