// Python module libfdl_direct: the paged-cache and scoring operators for calls
// of a few microseconds, where the dispatcher's boxing of a dozen arguments is
// a third of the call: the same functions that torch_ops.cpp registers, taken
// from Python without it.  Only plain CUDA tensors go this way, and only while
// nothing watches the dispatcher; for everything else (subclasses, wrapped or
// fake tensors, dispatch and function modes, torch.jit.trace, the profiler) the
// entry returns NotImplemented and the caller uses torch.ops.fdl.  A library
// of its own, so that libfdl_torch.so needs no interpreter.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/record_function.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>

#include "torch_ops.h"

namespace {

using at::Tensor;

constexpr c10::DispatchKeySet kPlainKeys =
    c10::DispatchKeySet({c10::DispatchKey::CUDA, c10::DispatchKey::ADInplaceOrView, c10::DispatchKey::AutogradCUDA,
                         c10::DispatchKey::AutocastCUDA});

bool plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return false;
  const Tensor& t = THPVariable_Unpack(o);
  const auto keys = t.key_set();
  // (the difference of two sets keeps its backend bits)
  return keys.has(c10::DispatchKey::CUDA) && ((keys - kPlainKeys).raw_repr() & ~c10::full_backend_mask) == 0 &&
         !t._fw_grad(0).defined();
}
bool plain_or_none(PyObject* o) { return o == Py_None || plain(o); }
const Tensor& tensor(PyObject* o) { return THPVariable_Unpack(o); }
std::optional<Tensor> maybe(PyObject* o) {
  if (o == Py_None) return std::nullopt;
  return THPVariable_Unpack(o);
}
int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
// A dispatch mode, a trace or a transform adds keys to the thread's own; a
// function mode and the profiler show elsewhere.
bool watched() {
  const auto keys = c10::impl::tls_local_dispatch_key_set().included_;
  return !(keys - c10::default_included_set).empty() || c10::impl::TorchDispatchModeTLS::any_modes_set() ||
         at::impl::torch_function_mode_enabled() || at::hasCallbacks();
}
bool direct(PyObject* const* a, Py_ssize_t n, Py_ssize_t want, std::initializer_list<int> tensors,
            std::initializer_list<int> optional = {}) {
  if (n != want || watched()) return false;
  for (int i : tensors)
    if (!plain(a[i])) return false;
  for (int i : optional)
    if (!plain_or_none(a[i])) return false;
  return true;
}
struct NoGil {
  PyThreadState* s = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(s); }
};

PyObject* py_page_slots(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!direct(a, n, 11, {0, 1, 2, 3, 4, 6, 7, 8}, {9, 10})) Py_RETURN_NOTIMPLEMENTED;
  const Tensor lens = tensor(a[0]), n_new = tensor(a[1]), table = tensor(a[2]), pages = tensor(a[3]),
               count = tensor(a[4]), slots = tensor(a[6]), pos = tensor(a[7]), cu = tensor(a[8]);
  const int64_t page = integer(a[5]);
  const auto nl = maybe(a[9]), nc = maybe(a[10]);
  {
    NoGil g;
    fdl_torch::page_slots(lens, n_new, table, pages, count, page, slots, pos, cu, nl, nc);
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* py_norm_rope_store(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!direct(a, n, 12, {0, 1, 2, 8, 9, 10, 11}, {3, 4})) Py_RETURN_NOTIMPLEMENTED;
  const Tensor y = tensor(a[0]), pos = tensor(a[1]), freq = tensor(a[2]), q = tensor(a[8]), k = tensor(a[9]),
               v = tensor(a[10]), slots = tensor(a[11]);
  const auto qw = maybe(a[3]), kw = maybe(a[4]);
  const double eps = number(a[5]), scale = number(a[7]);
  const int inter = PyObject_IsTrue(a[6]);
  if (inter < 0) throw python_error();
  {
    NoGil g;
    fdl_torch::norm_rope_store(y, pos, freq, qw, kw, eps, inter != 0, scale, q, k, v, slots);
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* py_paged_decode_attn(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!direct(a, n, 7, {0, 1, 2, 3, 4, 6})) Py_RETURN_NOTIMPLEMENTED;
  const Tensor q = tensor(a[0]), k = tensor(a[1]), v = tensor(a[2]), table = tensor(a[3]), lens = tensor(a[4]),
               out = tensor(a[6]);
  const double scale = number(a[5]);
  {
    NoGil g;
    fdl_torch::paged_decode_attn(q, k, v, table, lens, scale, out);
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* py_token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!direct(a, n, 3, {0, 1})) Py_RETURN_NOTIMPLEMENTED;
  const Tensor logits = tensor(a[0]), targets = tensor(a[1]);
  const int64_t top = integer(a[2]);
  fdl_torch::Scores r;
  {
    NoGil g;
    r = fdl_torch::token_logprobs(logits, targets, top, true);
  }
  return Py_BuildValue("(NNNN)", THPVariable_Wrap(std::get<0>(r)), THPVariable_Wrap(std::get<1>(r)),
                       THPVariable_Wrap(std::get<2>(r)), THPVariable_Wrap(std::get<3>(r)));
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(F)), METH_FASTCALL, nullptr};
}
PyMethodDef kMethods[] = {method<py_page_slots>("page_slots"), method<py_norm_rope_store>("norm_rope_store"),
                          method<py_paged_decode_attn>("paged_decode_attn"),
                          method<py_token_logprobs>("token_logprobs"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "libfdl_direct", nullptr, -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit_libfdl_direct(void) { return PyModule_Create(&kModule); }
