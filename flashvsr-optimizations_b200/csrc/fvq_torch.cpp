// fvq_torch.cpp -- short path from torch's eager mode to the C ABI for the block operators.
//
// A decode step calls these operators on a few rows at a time, where the Python side of a call
// (argument checks, output allocation, ctypes) takes longer than the kernel.  Each function here
// takes the common call -- plain CUDA tensors on the current device, contiguous, aligned, of the
// right types and shapes, with no gradient to record and no mode, trace or transform active --
// checks all of that, allocates the outputs and calls libfvq.so, whose entry points ops.py hands
// over with bind().  Anything else returns None, and the Python implementation (which copies,
// converts or raises) takes the call.  Nothing is computed here.
#include <Python.h>

#include <cstdint>
#include <optional>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include "../../include/fvq.h"

namespace {

struct Entries {
  decltype(&fvq_rms_norm) rms_norm = nullptr;
  decltype(&fvq_linear_act) linear_act = nullptr;
  decltype(&fvq_fp8_scaled_mm_act) fp8_scaled_mm_act = nullptr;
  decltype(&fvq_fp8_cache_write) cache_write = nullptr;
  decltype(&fvq_fp8_cache_read) cache_read = nullptr;
} entries;

// Whether something has to see the call that only the dispatcher shows it to: a dispatch mode,
// torch.jit.trace (which would record the outputs as constants) or a functorch transform, all of
// them keys that the thread includes beside the ones it starts with; a function mode; a forward-mode
// level, whose tangents the Python path refuses.
bool interposed() {
  return !(c10::impl::tls_local_dispatch_key_set().included_ - c10::default_included_set).empty() ||
         at::impl::torch_function_mode_enabled() ||
         torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr;
}

// The keys of a strided CUDA tensor in memory; any other (a conjugate or negated view, zeros without
// storage, a wrapper) makes it one for the dispatcher.
bool plain_keys(const at::Tensor& t) {
  constexpr c10::DispatchKeySet kPlain({c10::DispatchKey::CUDA, c10::DispatchKey::AutogradCUDA,
                                        c10::DispatchKey::ADInplaceOrView, c10::DispatchKey::AutocastCUDA});
  const c10::DispatchKeySet keys = t.key_set();
  return (keys.raw_repr() & ~kPlain.raw_repr()) == 0 && keys.has(c10::DispatchKey::CUDA);
}

bool aligned(const at::Tensor& t, uintptr_t to) {
  return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & (to - 1)) == 0;
}

// The tensor behind obj when it is a plain one of type `type` on device `dev`; otherwise null.
const at::Tensor* plain(PyObject* obj, at::ScalarType type, c10::DeviceIndex dev) {
  if (!THPVariable_CheckExact(obj)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(obj);
  if (!t.defined() || !plain_keys(t) || !t.has_storage() || t.scalar_type() != type || t.get_device() != dev)
    return nullptr;
  if (t.requires_grad() && c10::GradMode::is_enabled()) return nullptr;
  return &t;
}

// Contiguous and aligned besides; None gives null with *ok kept.
const at::Tensor* dense(PyObject* obj, at::ScalarType type, c10::DeviceIndex dev, uintptr_t to, bool* ok,
                        bool optional = false) {
  if (optional && obj == Py_None) return nullptr;
  const at::Tensor* t = plain(obj, type, dev);
  if (t == nullptr || !t->is_contiguous() || !aligned(*t, to)) {
    *ok = false;
    return nullptr;
  }
  return t;
}

const void* ptr(const at::Tensor* t) { return t == nullptr ? nullptr : t->const_data_ptr(); }

template <class T>
const T* in(const at::Tensor* t) {
  return static_cast<const T*>(ptr(t));
}

void* stream_of(c10::DeviceIndex dev) { return c10::cuda::getCurrentCUDAStream(dev).stream(); }

// Releases the interpreter's lock; taken again before an exception (a tensor whose memory may not be
// written throws at data_ptr) becomes a Python error.
struct Unlocked {
  PyThreadState* const state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// The device the fast path works on, or -1 when nothing is to be done here.
c10::DeviceIndex usable_device(const void* entry, PyObject* first) {
  if (entry == nullptr || !THPVariable_CheckExact(first) || interposed()) return -1;
  const at::Tensor& t = THPVariable_Unpack(first);
  if (!t.defined() || !t.is_cuda() || t.get_device() != c10::cuda::current_device()) return -1;
  return t.get_device();
}

// What at::empty ends in for a CUDA tensor, without the dispatch on the way there.
at::Tensor output(const at::Tensor& like, at::IntArrayRef sizes, at::ScalarType type) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}

// rms_norm(x, weight, residual, eps, fp8) -> (y | q, scale | None, new residual | None)
PyObject* py_rms_norm(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 5) Py_RETURN_NONE;
  const auto dev = usable_device(reinterpret_cast<const void*>(entries.rms_norm), args[0]);
  if (dev < 0) Py_RETURN_NONE;
  bool ok = true;
  const at::Tensor* x = plain(args[0], at::kBFloat16, dev);
  const at::Tensor* w = dense(args[1], at::kBFloat16, dev, 2, &ok, true);
  if (x == nullptr || !ok || x->dim() < 1 || x->numel() == 0) Py_RETURN_NONE;
  const auto sizes = x->sizes();
  const int64_t d = sizes.back(), rows = x->numel() / d;
  int64_t inner = 1, outer = d, step = 0;
  if (!x->is_contiguous()) {
    if (x->stride(-1) != 1 || x->dim() < 2 || x->dim() > 3) Py_RETURN_NONE;
    outer = x->stride(0);
    if (x->dim() == 3) inner = x->size(1), step = x->stride(1);
  }
  if (w != nullptr && w->numel() != d) Py_RETURN_NONE;
  const at::Tensor* r = nullptr;
  bool f32 = false;
  if (args[2] != Py_None) {
    if (!THPVariable_CheckExact(args[2])) Py_RETURN_NONE;
    f32 = THPVariable_Unpack(args[2]).scalar_type() == at::kFloat;
    r = dense(args[2], f32 ? at::kFloat : at::kBFloat16, dev, f32 ? 4 : 2, &ok);
    if (!ok || r->sizes() != sizes) Py_RETURN_NONE;
  }
  const double eps = PyFloat_AsDouble(args[3]);
  if (eps == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  const bool fp8 = args[4] == Py_True;
  at::Tensor y = output(*x, sizes, fp8 ? at::kFloat8_e4m3fn : at::kBFloat16), scale, fresh;
  if (fp8) {
    c10::SmallVector<int64_t, 5> s(sizes.begin(), sizes.end());
    s.back() = 1;
    scale = output(*x, s, at::kFloat);
  }
  if (r != nullptr) fresh = output(*x, sizes, r->scalar_type());
  int rc;
  {
    const Unlocked unlocked;
    rc = entries.rms_norm(in<uint16_t>(x), rows, inner, outer, step, d, in<uint16_t>(w),
                          static_cast<float>(eps), ptr(r), f32 ? 1 : 0,
                          r != nullptr ? fresh.data_ptr() : nullptr,
                          fp8 ? nullptr : static_cast<uint16_t*>(y.data_ptr()),
                          fp8 ? static_cast<uint8_t*>(y.data_ptr()) : nullptr,
                          fp8 ? static_cast<float*>(scale.data_ptr()) : nullptr, stream_of(dev));
  }
  if (rc != FVQ_OK) Py_RETURN_NONE;  // the Python path repeats the call and raises
  PyObject* out = PyTuple_New(3);
  if (out == nullptr) return nullptr;
  const auto put = [&](int i, at::Tensor& t) {
    if (!t.defined()) Py_INCREF(Py_None);
    PyTuple_SET_ITEM(out, i, t.defined() ? THPVariable_Wrap(std::move(t)) : Py_None);
  };
  put(0, y);
  put(1, scale);
  put(2, fresh);
  return out;
  END_HANDLE_TH_ERRORS
}

// Shapes shared by the two products; false when the Python path has to look at the call.
struct Product {
  int64_t m, k, n, wn, stride;
  c10::SmallVector<int64_t, 5> out;
};

bool product_shape(const at::Tensor& x, const at::Tensor& w, const at::Tensor* bias,
                   const at::Tensor* residual, bool gated, int64_t per16, Product* p) {
  if (x.dim() < 1 || w.dim() != 2 || x.numel() == 0 || w.numel() == 0) return false;
  p->k = x.size(-1);
  p->wn = w.size(0);
  if (w.size(1) != p->k || (gated && p->wn % 2 != 0)) return false;
  p->n = gated ? p->wn / 2 : p->wn;
  p->m = x.numel() / p->k;
  p->stride = p->k;
  if (!x.is_contiguous()) {
    if (x.dim() != 2 || x.stride(1) != 1) return false;
    p->stride = p->m > 1 ? x.stride(0) : p->k;
    if (p->stride < p->k || p->stride % per16 != 0) return false;
  }
  if (!aligned(x, 16)) return false;
  p->out.assign(x.sizes().begin(), x.sizes().end());
  p->out.back() = p->n;
  if (bias != nullptr && bias->numel() != p->wn) return false;
  return residual == nullptr || residual->sizes() == at::IntArrayRef(p->out);
}

// linear_act(x, weight, bias, act, gated, residual) -> y
PyObject* py_linear_act(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 6 || !PyLong_Check(args[3]) || !PyBool_Check(args[4])) Py_RETURN_NONE;
  const auto dev = usable_device(reinterpret_cast<const void*>(entries.linear_act), args[0]);
  if (dev < 0) Py_RETURN_NONE;
  bool ok = true;
  const at::Tensor* x = plain(args[0], at::kBFloat16, dev);
  const at::Tensor* w = dense(args[1], at::kBFloat16, dev, 16, &ok);
  const at::Tensor* bias = dense(args[2], at::kBFloat16, dev, 16, &ok, true);
  const at::Tensor* residual = dense(args[5], at::kBFloat16, dev, 16, &ok, true);
  const bool gated = args[4] == Py_True;
  Product p;
  if (x == nullptr || !ok || !product_shape(*x, *w, bias, residual, gated, 8, &p)) Py_RETURN_NONE;
  const int act = static_cast<int>(PyLong_AsLong(args[3]));
  at::Tensor y = output(*x, p.out, at::kBFloat16);
  int rc;
  {
    const Unlocked unlocked;
    rc = entries.linear_act(in<uint16_t>(x), p.m, p.k, p.stride, in<uint16_t>(w), p.n, in<uint16_t>(bias),
                            act, gated ? 1 : 0, in<uint16_t>(residual), static_cast<uint16_t*>(y.data_ptr()),
                            stream_of(dev));
  }
  if (rc != FVQ_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// fp8_scaled_mm_act(a, scale_a, w, scale_w, bias, act, gated, residual) -> y
PyObject* py_fp8_scaled_mm_act(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 8 || !PyLong_Check(args[5]) || !PyBool_Check(args[6])) Py_RETURN_NONE;
  const auto dev = usable_device(reinterpret_cast<const void*>(entries.fp8_scaled_mm_act), args[0]);
  if (dev < 0) Py_RETURN_NONE;
  bool ok = true;
  const at::Tensor* a = plain(args[0], at::kFloat8_e4m3fn, dev);
  const at::Tensor* sa = dense(args[1], at::kFloat, dev, 4, &ok);
  const at::Tensor* w = dense(args[2], at::kFloat8_e4m3fn, dev, 16, &ok);
  const at::Tensor* sw = dense(args[3], at::kFloat, dev, 16, &ok);
  const at::Tensor* bias = dense(args[4], at::kBFloat16, dev, 16, &ok, true);
  const at::Tensor* residual = dense(args[7], at::kBFloat16, dev, 16, &ok, true);
  const bool gated = args[6] == Py_True;
  Product p;
  if (a == nullptr || !ok || !product_shape(*a, *w, bias, residual, gated, 16, &p) ||
      sa->numel() != p.m || sw->numel() != p.wn)
    Py_RETURN_NONE;
  const int act = static_cast<int>(PyLong_AsLong(args[5]));
  at::Tensor y = output(*a, p.out, at::kBFloat16);
  int rc;
  {
    const Unlocked unlocked;
    rc = entries.fp8_scaled_mm_act(in<uint8_t>(a), in<float>(sa), p.m, p.k, p.stride, in<uint8_t>(w),
                                   in<float>(sw), p.n, in<uint16_t>(bias), act, gated ? 1 : 0,
                                   in<uint16_t>(residual), static_cast<uint16_t*>(y.data_ptr()),
                                   stream_of(dev));
  }
  if (rc != FVQ_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// The store's four tensors; false when one is not as fvq_fp8_cache_* takes them.
bool store_of(PyObject* const* args, c10::DeviceIndex dev, const at::Tensor* (&t)[4]) {
  bool ok = true;
  t[0] = dense(args[0], at::kFloat8_e4m3fn, dev, 8, &ok);
  t[1] = dense(args[1], at::kFloat, dev, 4, &ok);
  t[2] = dense(args[2], at::kFloat8_e4m3fn, dev, 8, &ok);
  t[3] = dense(args[3], at::kFloat, dev, 4, &ok);
  return ok && t[0]->dim() == 4 && t[2]->sizes() == t[0]->sizes() &&
         t[1]->sizes() == t[0]->sizes().slice(0, 3) && t[3]->sizes() == t[0]->sizes().slice(0, 3);
}

bool token_rows(const at::Tensor& x, const at::Tensor& codes) {
  return x.dim() == 3 && x.size(1) == codes.size(2) && x.size(2) == codes.size(3) && x.stride(2) == 1 &&
         x.stride(0) % 8 == 0 && x.stride(1) % 8 == 0 && aligned(x, 16);
}

// fp8_cache_write(k, v, slots, k_codes, k_scale, v_codes, v_scale) -> True
PyObject* py_cache_write(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 7) Py_RETURN_NONE;
  const auto dev = usable_device(reinterpret_cast<const void*>(entries.cache_write), args[0]);
  if (dev < 0) Py_RETURN_NONE;
  bool ok = true;
  const at::Tensor* k = plain(args[0], at::kBFloat16, dev);
  const at::Tensor* v = plain(args[1], at::kBFloat16, dev);
  const at::Tensor* slots = dense(args[2], at::kLong, dev, 8, &ok);
  const at::Tensor* t[4];
  if (k == nullptr || v == nullptr || !ok || !store_of(args + 3, dev, t) || !token_rows(*k, *t[0]) ||
      !token_rows(*v, *t[0]) || k->sizes() != v->sizes() || k->numel() == 0 || slots->dim() != 1 ||
      slots->size(0) != k->size(0))
    Py_RETURN_NONE;
  int rc;
  {
    const Unlocked unlocked;
    rc = entries.cache_write(in<uint16_t>(k), in<uint16_t>(v), k->size(0), k->size(1), k->size(2),
                             k->stride(0), k->stride(1), v->stride(0), v->stride(1), in<int64_t>(slots),
                             static_cast<uint8_t*>(t[0]->data_ptr()), static_cast<float*>(t[1]->data_ptr()),
                             static_cast<uint8_t*>(t[2]->data_ptr()), static_cast<float*>(t[3]->data_ptr()),
                             t[0]->size(0) * t[0]->size(1), stream_of(dev));
  }
  if (rc != FVQ_OK) Py_RETURN_NONE;
  for (const auto* s : t)  // written in place
    if (!s->is_inference()) s->unsafeGetTensorImpl()->bump_version();
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// fp8_cache_read(k_codes, k_scale, v_codes, v_scale, page_table, lengths, max_len) -> (k, v)
PyObject* py_cache_read(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 7 || !PyLong_Check(args[6])) Py_RETURN_NONE;
  const auto dev = usable_device(reinterpret_cast<const void*>(entries.cache_read), args[0]);
  if (dev < 0) Py_RETURN_NONE;
  bool ok = true;
  const at::Tensor* t[4];
  const at::Tensor* table = dense(args[4], at::kInt, dev, 4, &ok);
  const at::Tensor* lengths = dense(args[5], at::kInt, dev, 4, &ok);
  const int64_t max_len = PyLong_AsLongLong(args[6]);
  if (max_len == -1 && PyErr_Occurred()) PyErr_Clear();
  if (!ok || !store_of(args, dev, t) || table->dim() != 2 || table->numel() == 0 || lengths->dim() != 1 ||
      lengths->size(0) != table->size(0) || max_len <= 0 || t[0]->size(2) * t[0]->size(3) == 0)
    Py_RETURN_NONE;
  const int64_t sizes[4] = {table->size(0), max_len, t[0]->size(2), t[0]->size(3)};
  at::Tensor k = output(*t[0], sizes, at::kBFloat16), v = output(*t[0], sizes, at::kBFloat16);
  int rc;
  {
    const Unlocked unlocked;
    rc = entries.cache_read(in<uint8_t>(t[0]), in<float>(t[1]), in<uint8_t>(t[2]), in<float>(t[3]),
                            t[0]->size(0), t[0]->size(1), sizes[2], sizes[3], in<int32_t>(table), sizes[0],
                            table->size(1), in<int32_t>(lengths), max_len,
                            static_cast<uint16_t*>(k.data_ptr()), static_cast<uint16_t*>(v.data_ptr()),
                            stream_of(dev));
  }
  if (rc != FVQ_OK) Py_RETURN_NONE;
  PyObject* out = PyTuple_New(2);
  if (out == nullptr) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(k)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(v)));
  return out;
  END_HANDLE_TH_ERRORS
}

// bind(rms_norm, linear_act, fp8_scaled_mm_act, cache_write, cache_read): addresses in libfvq.so
PyObject* py_bind(PyObject*, PyObject* const* args, Py_ssize_t count) {
  void* at[5];
  if (count != 5) {
    PyErr_SetString(PyExc_TypeError, "bind takes five addresses");
    return nullptr;
  }
  for (int i = 0; i < 5; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (at[i] == nullptr && PyErr_Occurred()) return nullptr;
  }
  entries.rms_norm = reinterpret_cast<decltype(entries.rms_norm)>(at[0]);
  entries.linear_act = reinterpret_cast<decltype(entries.linear_act)>(at[1]);
  entries.fp8_scaled_mm_act = reinterpret_cast<decltype(entries.fp8_scaled_mm_act)>(at[2]);
  entries.cache_write = reinterpret_cast<decltype(entries.cache_write)>(at[3]);
  entries.cache_read = reinterpret_cast<decltype(entries.cache_read)>(at[4]);
  Py_RETURN_NONE;
}

template <class F>
PyCFunction fast(F f) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f));
}

PyMethodDef methods[] = {
    {"bind", fast(py_bind), METH_FASTCALL, "hand over the entry points of libfvq.so"},
    {"rms_norm", fast(py_rms_norm), METH_FASTCALL, "None when the Python path has to take the call"},
    {"linear_act", fast(py_linear_act), METH_FASTCALL, "None when the Python path has to take the call"},
    {"fp8_scaled_mm_act", fast(py_fp8_scaled_mm_act), METH_FASTCALL,
     "None when the Python path has to take the call"},
    {"fp8_cache_write", fast(py_cache_write), METH_FASTCALL,
     "None when the Python path has to take the call"},
    {"fp8_cache_read", fast(py_cache_read), METH_FASTCALL,
     "None when the Python path has to take the call"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fvq_torch", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

#define FVQ_TEXT_(x) #x
#define FVQ_TEXT(x) FVQ_TEXT_(x)

PyMODINIT_FUNC PyInit__fvq_torch() {
  PyObject* m = PyModule_Create(&module);
  // compared by the loader: what is used of torch changes between its versions
  if (m != nullptr && PyModule_AddStringConstant(m, "built_for",
                                                 TORCH_VERSION " " FVQ_TEXT(PY_MAJOR_VERSION) "." FVQ_TEXT(
                                                     PY_MINOR_VERSION)) != 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
