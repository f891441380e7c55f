// Host side of mingmoe.fp8, mingmoe.sampling and mingmoe.paging in C++: reads the tensors, allocates the results, fills the C
// entry points' argument structs.
//
// The kernels of a small call take 3 to 10 us, and reading its sizes, strides and addresses through Python attributes as long
// again. Only the plain case is handled: exact tensors on the current device with the right types, shapes and strides. For
// anything else a function returns NotImplemented, and the Python code, which has the same checks, copies or refuses. The
// entry points are given by address (bind), so they are the ones of the library that mingmoe/_lib.py loaded.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <vector>

#include "../../include/mingmoe.h"

namespace {

int (*g_linear)(const mv_fp8_linear_args*, void*, size_t, void*) = nullptr;
size_t (*g_linear_scratch)(int, int, int) = nullptr;
int (*g_sample)(const mv_sample_args*, void*) = nullptr;
int (*g_plan)(const mv_plan_args*, void*) = nullptr;

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

PyObject* plain_not() { Py_RETURN_NOTIMPLEMENTED; }

const at::Tensor* tensor(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

bool on(const at::Tensor& t, int device) { return t.is_cuda() && t.device().index() == device; }

void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream(); }

int code(at::ScalarType t) {
  return t == at::kBFloat16 ? MV_BF16 : t == at::kHalf ? MV_F16 : t == at::kFloat ? MV_F32 : -1;
}

bool unit(const at::Tensor& t) { return t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1); }

// a tensor whose leading axes are one of rows: rows and their stride
bool rows_of(const at::Tensor& t, int64_t* rows, int64_t* stride) {
  const int64_t d = t.dim();
  if (d < 1 || (t.size(d - 1) > 1 && t.stride(d - 1) != 1)) return false;
  if (d == 2) {
    *rows = t.size(0), *stride = t.stride(0);
    return true;
  }
  if (!t.is_contiguous()) return false;
  *rows = t.size(d - 1) > 0 ? t.numel() / t.size(d - 1) : 0;
  *stride = t.size(d - 1);
  return t.size(d - 1) > 0;
}

PyObject* guarded(PyObject* (*f)(PyObject* const*), PyObject* const* args) {
  // results are new tensors, or views of those, without a history: no dispatch through the layers that keep one
  at::AutoDispatchBelowADInplaceOrView guard;
  try {
    return f(args);
  } catch (const std::exception&) {  // an allocation that failed: the Python code meets it again and raises torch's error
    return plain_not();
  }
}

// fp8_linear(x, wq, ws, residual, out, out_dtype)
PyObject* linear_impl(PyObject* const* o) {
  const at::Tensor *x = tensor(o[0]), *wq = tensor(o[1]), *ws = tensor(o[2]);
  if (x == nullptr || wq == nullptr || ws == nullptr || !x->is_cuda()) return plain_not();
  const int dev = x->device().index();
  const int xt = code(x->scalar_type());
  if (c10::cuda::current_device() != dev || !on(*wq, dev) || !on(*ws, dev) || (xt != MV_BF16 && xt != MV_F16) ||
      wq->scalar_type() != at::kFloat8_e4m3fn || ws->scalar_type() != at::kFloat || !unit(*wq) || !unit(*ws))
    return plain_not();
  at::ScalarType ot = x->scalar_type();
  if (o[5] != Py_None) {
    if (!THPDtype_Check(o[5])) return plain_not();
    ot = reinterpret_cast<THPDtype*>(o[5])->scalar_type;
  }
  const int64_t n = wq->size(0), k = wq->size(1), blocks = (k + 127) / 128;
  int64_t rows, x_st;
  if (code(ot) < 0 || k < 1 || !rows_of(*x, &rows, &x_st) || x->size(x->dim() - 1) != k || ws->size(0) != (n + 127) / 128 ||
      ws->size(1) != blocks || rows > 0x7fffffff || n > 0x7fffffff || k > 0x7fffffff)
    return plain_not();
  auto shape = x->sizes().vec();
  shape.back() = n;
  mv_fp8_linear_args a{};
  if (o[3] != Py_None) {
    const at::Tensor* r = tensor(o[3]);
    int64_t r_rows, r_st;
    if (r == nullptr || !on(*r, dev) || r->scalar_type() != ot || r->sizes() != at::IntArrayRef(shape) ||
        !rows_of(*r, &r_rows, &r_st))
      return plain_not();
    a.residual = r->data_ptr(), a.r_st = r_st;
  }
  at::Tensor out;
  int64_t o_rows, o_st;
  if (o[4] == Py_None) {
    out = at::empty(shape, x->options().dtype(ot));
  } else {
    const at::Tensor* t = tensor(o[4]);
    if (t == nullptr || !on(*t, dev) || t->scalar_type() != ot || t->sizes() != at::IntArrayRef(shape)) return plain_not();
    out = *t;
  }
  if (!rows_of(out, &o_rows, &o_st)) return plain_not();
  void* stream = stream_of(dev);
  const Workspace* found = nullptr;
  for (const Workspace& w : workspaces())
    if (w.device == dev && w.stream == stream) found = &w;
  if (found == nullptr) return plain_not();
  a.T = static_cast<int>(rows), a.N = static_cast<int>(n), a.K = static_cast<int>(k);
  const size_t bytes = g_linear_scratch(a.T, a.N, a.K);
  at::Tensor scratch;
  if (bytes > 0) {
    scratch = at::empty({static_cast<int64_t>(bytes)}, x->options().dtype(at::kByte));
    a.scratch = scratch.data_ptr();
  }
  a.x = x->data_ptr(), a.wq = wq->data_ptr(), a.ws = static_cast<const float*>(ws->data_ptr()), a.out = out.data_ptr();
  a.x_st = x_st, a.w_st = wq->stride(0), a.ws_st = ws->stride(0), a.o_st = o_st, a.scratch_bytes = bytes;
  a.x_dtype = xt, a.out_dtype = code(ot);
  const int rc = g_linear(&a, found->ptr, found->bytes, stream);
  return rc != MV_OK ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
}

// a setting of sample: a tensor of b values of `type`, or a number
bool setting(PyObject* o, at::ScalarType type, int64_t b, int dev, const void** p, double* value) {
  if (const at::Tensor* t = tensor(o)) {
    *p = t->data_ptr();
    return on(*t, dev) && t->scalar_type() == type && t->dim() == 1 && t->size(0) == b && (b <= 1 || t->stride(0) == 1);
  }
  if (type == at::kInt) {
    if (!PyLong_Check(o)) return false;
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) PyErr_Clear();
    *value = static_cast<double>(v);
    return v >= 0 && v <= 0x7fffffff;
  }
  *value = PyFloat_AsDouble(o);
  if (*value == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

// sample(logits, u, temperature, top_k, top_p, min_p, out, return_logprob)
PyObject* sample_impl(PyObject* const* o) {
  const at::Tensor *l = tensor(o[0]), *u = tensor(o[1]);
  if (l == nullptr || u == nullptr || !l->is_cuda() || l->dim() != 2 || code(l->scalar_type()) < 0) return plain_not();
  const int dev = l->device().index();
  const int64_t b = l->size(0), v = l->size(1);
  const void *pu, *pt = nullptr, *pk = nullptr, *pp = nullptr, *pm = nullptr;
  double unused, t = 0, k = 0, p = 0, m = 0;
  if (c10::cuda::current_device() != dev || (v > 1 && l->stride(1) != 1) || b > 0x7fffffff || v > 0x7fffffff ||
      !setting(o[1], at::kFloat, b, dev, &pu, &unused) || !setting(o[2], at::kFloat, b, dev, &pt, &t) ||
      !setting(o[3], at::kInt, b, dev, &pk, &k) || !setting(o[4], at::kFloat, b, dev, &pp, &p) ||
      !setting(o[5], at::kFloat, b, dev, &pm, &m))
    return plain_not();
  const int with = PyObject_IsTrue(o[7]);
  if (with < 0) {
    PyErr_Clear();  // the Python code meets it again and raises
    return plain_not();
  }
  at::Tensor out, logprob;
  if (o[6] == Py_None) {
    out = at::empty({b}, l->options().dtype(at::kLong));
  } else {
    const at::Tensor* given = tensor(o[6]);
    if (given == nullptr || !on(*given, dev) || given->scalar_type() != at::kLong || given->dim() != 1 || given->size(0) != b ||
        !given->is_contiguous())
      return plain_not();
    out = *given;
  }
  if (with) logprob = at::empty({b}, l->options().dtype(at::kFloat));
  mv_sample_args a{};
  a.logits = l->data_ptr(), a.u = static_cast<const float*>(pu), a.temperature = static_cast<const float*>(pt);
  a.top_p = static_cast<const float*>(pp), a.min_p = static_cast<const float*>(pm), a.top_k = static_cast<const int*>(pk);
  a.tokens = static_cast<long long*>(out.data_ptr());
  a.logprob = with ? static_cast<float*>(logprob.data_ptr()) : nullptr;
  a.st = l->stride(0);
  a.temperature_value = static_cast<float>(t), a.top_p_value = static_cast<float>(p), a.min_p_value = static_cast<float>(m);
  a.top_k_value = static_cast<int>(k), a.B = static_cast<int>(b), a.V = static_cast<int>(v), a.dtype = code(l->scalar_type());
  const int rc = g_sample(&a, stream_of(dev));
  if (rc != MV_OK) return PyLong_FromLong(rc);
  PyObject* first = THPVariable_Wrap(out);
  if (!with || first == nullptr) return first;
  PyObject* second = THPVariable_Wrap(logprob);
  return second == nullptr ? nullptr : Py_BuildValue("NN", first, second);
}

// contiguous int32
bool ints(PyObject* o, int64_t size, int dev, const at::Tensor** out) {
  const at::Tensor* t = tensor(o);
  *out = t;
  return t != nullptr && on(*t, dev) && t->scalar_type() == at::kInt && t->dim() == 1 && (size < 0 || t->size(0) == size) &&
         (t->size(0) <= 1 || t->stride(0) == 1);
}

// plan_step(new, lens, pages, free, n_free, page_size, num_tokens, seqs, max_len, lens_out, n_free_out, prompts):
// (cu_seqlens, kv_lens, page_table, slots, positions, ok)
PyObject* plan_impl(PyObject* const* o) {
  const at::Tensor *fresh, *lens, *pages = tensor(o[2]), *free_pages, *n_free, *seqs = nullptr, *lens_out, *n_free_out;
  if (pages == nullptr || !pages->is_cuda() || pages->scalar_type() != at::kInt || !unit(*pages)) return plain_not();
  const int dev = pages->device().index();
  const int64_t s = pages->size(0), p = pages->size(1);
  if (c10::cuda::current_device() != dev || !ints(o[0], -1, dev, &fresh) || !ints(o[1], s, dev, &lens) ||
      !ints(o[3], -1, dev, &free_pages) || !ints(o[4], 1, dev, &n_free))
    return plain_not();
  const int64_t b = fresh->size(0);
  if (o[7] == Py_None ? b != s : !ints(o[7], b, dev, &seqs)) return plain_not();
  lens_out = lens, n_free_out = n_free;
  if ((o[9] != Py_None && !ints(o[9], s, dev, &lens_out)) || (o[10] != Py_None && !ints(o[10], 1, dev, &n_free_out)))
    return plain_not();
  if (!PyLong_Check(o[5]) || !PyLong_Check(o[6]) || (o[8] != Py_None && !PyLong_Check(o[8]))) return plain_not();
  const long long page = PyLong_AsLongLong(o[5]), tokens = PyLong_AsLongLong(o[6]);
  long long max_len = p * page;
  if (o[8] != Py_None) max_len = PyLong_AsLongLong(o[8]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return plain_not();
  }
  const int prompts = PyObject_IsTrue(o[11]);
  if (prompts < 0) {
    PyErr_Clear();  // the Python code meets it again and raises
    return plain_not();
  }
  if (page < 0 || page > 0x7fffffff || tokens < 0 || tokens > 0x7fffffff - 3 * b - 4 || max_len < 0) return plain_not();
  const auto options = pages->options();
  // cu_seqlens, kv_lens, ok, scratch, positions side by side
  at::Tensor all = at::empty({3 * b + 4 + tokens}, options);
  at::Tensor slots = at::empty({tokens}, options.dtype(at::kLong));
  at::Tensor table = seqs == nullptr ? *pages : at::empty({b, p}, options);
  const auto part = [&](int64_t from, int64_t n) { return all.as_strided({n}, {1}, from); };
  at::Tensor cu = part(0, b + 1), kv = part(b + 1, b), ok = part(2 * b + 1, 1), positions = part(3 * b + 4, tokens);
  int* base = static_cast<int*>(all.data_ptr());
  mv_plan_args a{};
  a.new_tokens = static_cast<const int*>(fresh->data_ptr()), a.lens = static_cast<const int*>(lens->data_ptr());
  a.n_free = static_cast<const int*>(n_free->data_ptr()), a.free_pages = static_cast<int*>(free_pages->data_ptr());
  a.pages = static_cast<int*>(pages->data_ptr()), a.lens_out = static_cast<int*>(lens_out->data_ptr());
  a.n_free_out = static_cast<int*>(n_free_out->data_ptr());
  if (seqs != nullptr) {
    a.seqs = static_cast<const int*>(seqs->data_ptr()), a.table = static_cast<int*>(table.data_ptr());
    a.table_st = p;
  }
  a.cu_seqlens = base, a.kv_lens = base + b + 1, a.ok = base + 2 * b + 1, a.scratch = base + 2 * b + 2;
  a.positions = base + 3 * b + 4, a.slots = static_cast<long long*>(slots.data_ptr());
  a.pages_st = pages->stride(0), a.B = static_cast<int>(b), a.max_seqs = static_cast<int>(s);
  a.max_pages = static_cast<int>(p), a.page_size = static_cast<int>(page);
  a.max_len = static_cast<int>(max_len < 0x7fffffff ? max_len : 0x7fffffff);
  a.num_pages = static_cast<int>(free_pages->size(0)), a.T = static_cast<int>(tokens), a.prompts = prompts;
  const int rc = g_plan(&a, stream_of(dev));
  if (rc != MV_OK) return PyLong_FromLong(rc);
  if (seqs == nullptr) Py_INCREF(o[2]);
  return Py_BuildValue("NNNNNN", THPVariable_Wrap(cu), THPVariable_Wrap(kv), seqs == nullptr ? o[2] : THPVariable_Wrap(table),
                       THPVariable_Wrap(slots), THPVariable_Wrap(positions), THPVariable_Wrap(ok));
}

PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) { return n == 6 ? guarded(linear_impl, a) : plain_not(); }
PyObject* sample(PyObject*, PyObject* const* a, Py_ssize_t n) { return n == 8 ? guarded(sample_impl, a) : plain_not(); }
PyObject* plan(PyObject*, PyObject* const* a, Py_ssize_t n) { return n == 12 ? guarded(plan_impl, a) : plain_not(); }

// bind(addresses of mv_fp8_linear, mv_fp8_linear_scratch_bytes, mv_sample, mv_plan_step)
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long f[4];
  if (!PyArg_ParseTuple(args, "KKKK", &f[0], &f[1], &f[2], &f[3])) return nullptr;
  g_linear = reinterpret_cast<decltype(g_linear)>(f[0]);
  g_linear_scratch = reinterpret_cast<decltype(g_linear_scratch)>(f[1]);
  g_sample = reinterpret_cast<decltype(g_sample)>(f[2]);
  g_plan = reinterpret_cast<decltype(g_plan)>(f[3]);
  Py_RETURN_NONE;
}

// workspace(device, stream, address, bytes): the header of a stream's products
PyObject* workspace(PyObject*, PyObject* args) {
  int device;
  unsigned long long stream, ptr, bytes;
  if (!PyArg_ParseTuple(args, "iKKK", &device, &stream, &ptr, &bytes)) return nullptr;
  workspaces().push_back(Workspace{device, reinterpret_cast<void*>(stream), reinterpret_cast<void*>(ptr),
                                   static_cast<size_t>(bytes)});
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"fp8_linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(linear)), METH_FASTCALL, nullptr},
    {"sample", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(sample)), METH_FASTCALL, nullptr},
    {"plan_step", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(plan)), METH_FASTCALL, nullptr},
    {"bind", bind, METH_VARARGS, nullptr},
    {"workspace", workspace, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving_host() { return PyModule_Create(&module); }
