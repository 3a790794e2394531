// What the dispatcher entries of kv_attention._native share: the library's functions, argument checks, layouts, and the reading of Python's
// arguments.
#pragma once
#include <Python.h>
#include <dlfcn.h>

#include <mutex>
#include <string>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/library.h>

#include "../../include/kv_attention.h"

namespace kv_native {

using at::Tensor;
using c10::SymInt;
using OptTensor = std::optional<Tensor>;

// ---- the shared library -------------------------------------------------------------------------------------
struct Api {
  decltype(&kv_cross_forward) cross_forward;
  decltype(&kv_cross_forward_workspace) cross_forward_workspace;
  decltype(&kv_cross_backward) cross_backward;
  decltype(&kv_cross_backward_workspace) cross_backward_workspace;
  decltype(&kv_paged_forward) paged_forward;
  decltype(&kv_paged_forward_workspace) paged_forward_workspace;
  decltype(&kv_paged_append) paged_append;
  decltype(&kv_paged_append_rope) paged_append_rope;
  decltype(&kv_paged_tree_forward) paged_tree_forward;
  decltype(&kv_paged_tree_forward_workspace) paged_tree_forward_workspace;
  decltype(&kv_paged_keep) paged_keep;
  decltype(&kv_qk_norm_rope) qk_norm_rope;
  decltype(&kv_qk_norm_rope_backward) qk_norm_rope_backward;
  decltype(&kv_qk_norm_rope_backward_workspace) qk_norm_rope_backward_workspace;
  decltype(&kv_error_string) error_string;
};

const Api& api();   // kv_torch.cpp; opened on the first call
inline void check(int64_t rc, const char* what) {
  TORCH_CHECK(rc >= 0, what, " failed with code ", rc, ": ", api().error_string((int)rc));
}
inline void check_launch(int rc, const char* what) {
  TORCH_CHECK(rc == 0, what, " failed with code ", rc, ": ", api().error_string(rc));
}

// ---- argument checks and layout -------------------------------------------------------------------------------
inline int dtype_id(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kHalf: return 1;
    case at::kBFloat16: return 2;
    default: return -1;
  }
}
inline bool known_head_dim(int64_t d) { return d == 16 || d == 32 || d == 64 || d == 128 || d == 256; }
inline bool alike(const Tensor& a, const Tensor& b) { return a.device() == b.device() && a.scalar_type() == b.scalar_type(); }
inline bool is_lengths(const OptTensor& l, const Tensor& q) {
  return !l || (l->scalar_type() == at::kInt && l->dim() == 1 && l->size(0) == q.size(0) && l->device() == q.device());
}
inline bool is_scale(double sm_scale) { return std::fabs(sm_scale) <= 0x1p127; }   // times log2(e) in float32's range
inline bool small(int64_t n) { return n <= 0x7fffffff; }
inline bool small_sizes(const Tensor& t) { return small(t.size(0)) && small(t.size(1)) && small(t.size(2)); }

inline bool is_cross(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lens, const OptTensor& q_lens, double sm_scale) {
  if (q.dim() != 4 || k.dim() != 4 || dtype_id(q) < 0 || !known_head_dim(q.size(3)) || !alike(q, k) || !alike(q, v)) return false;
  if (v.sizes() != k.sizes() || k.size(0) != q.size(0) || k.size(3) != q.size(3) || k.size(1) < 1 || q.size(1) < 1 || q.size(1) % k.size(1) != 0)
    return false;
  return small_sizes(q) && small_sizes(k) && is_lengths(lens, q) && is_lengths(q_lens, q) && is_scale(sm_scale);
}
// A cache in pages and the table of its sequences.
inline bool is_pages(const Tensor& k_pages, const Tensor& v_pages, const Tensor& table) {
  if (k_pages.dim() != 4 || dtype_id(k_pages) < 0 || !known_head_dim(k_pages.size(3)) || !alike(k_pages, v_pages)) return false;
  if (v_pages.sizes() != k_pages.sizes() || k_pages.size(2) < 1 || k_pages.size(1) < 1) return false;
  if (table.dim() != 2 || table.scalar_type() != at::kInt || table.device() != k_pages.device()) return false;
  for (const Tensor* t : {&k_pages, &v_pages}) {   // read and written in place: no copy stands in for them
    const int64_t vec = 16 / t->element_size();
    if (t->numel() == 0) continue;
    if (t->stride(3) != 1 || reinterpret_cast<uintptr_t>(t->const_data_ptr()) % 16 != 0) return false;
    for (int i = 0; i < 3; ++i)
      if (t->size(i) > 1 && (t->stride(i) % vec != 0 || t->stride(i) <= 0)) return false;
  }
  return small_sizes(k_pages) && small(table.size(0)) && small(table.size(1)) && table.size(1) * k_pages.size(2) <= (int64_t(1) << 30);
}
inline bool is_cache(const Tensor& x, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& lens,
                     const OptTensor& new_lens) {
  if (x.dim() != 4 || !alike(x, k_pages) || !is_pages(k_pages, v_pages, table) || k_pages.size(3) != x.size(3) || x.size(1) < 1) return false;
  return small_sizes(x) && table.size(0) == x.size(0) && is_lengths(lens, x) && is_lengths(new_lens, x);
}

inline PyObject* wrap(const OptTensor& t) {
  if (t) return THPVariable_Wrap(*t);
  Py_RETURN_NONE;
}
inline PyObject* wrap(std::optional<double> x) {
  if (x) return PyFloat_FromDouble(*x);
  Py_RETURN_NONE;
}
// Have Python's checks name what is wrong; takes the references.
[[noreturn]] inline void explain(const char* function, std::initializer_list<PyObject*> args) {
  PyObject* tuple = PyTuple_New((Py_ssize_t)args.size());
  Py_ssize_t i = 0;
  for (PyObject* a : args) PyTuple_SET_ITEM(tuple, i++, a);
  PyObject* m = PyImport_ImportModule("kv_attention.ops");
  PyObject* f = m ? PyObject_GetAttrString(m, function) : nullptr;
  PyObject* r = f ? PyObject_CallObject(f, tuple) : nullptr;
  Py_XDECREF(r);
  Py_XDECREF(f);
  Py_XDECREF(m);
  Py_DECREF(tuple);
  if (PyErr_Occurred()) throw python_error();
  TORCH_CHECK(false, "unsupported arguments");
}
struct Gil {
  PyGILState_STATE s = PyGILState_Ensure();
  ~Gil() { PyGILState_Release(s); }
};

// The tensor itself when the kernels can read it in place (unit stride along the head dimension, the others and the base
// address multiples of 16 bytes, rows that advance), otherwise a contiguous copy.  offsets32: rows of one head are addressed with 32-bit byte offsets.
inline Tensor kernel_layout(const Tensor& t, bool offsets32 = true) {
  const int64_t es = t.element_size(), vec = 16 / es, T = t.size(2);
  const auto s = t.strides();
  bool ok = (s[3] == 1 || t.size(3) == 1) && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
  for (int i = 0; i < 3; ++i) ok = ok && (t.size(i) <= 1 || s[i] % vec == 0);
  ok = ok && (T <= 1 || (s[2] > 0 && (!offsets32 || s[2] <= 0xffffffffLL / es / (T + 1024))));
  if (ok) return t;
  return t.is_contiguous() ? t.clone(at::MemoryFormat::Contiguous) : t.contiguous();
}
struct Strides {   // a dimension of one element may have any stride: 0 here
  int64_t s[4];
  explicit Strides(const Tensor& t) {
    for (int i = 0; i < 3; ++i) s[i] = t.size(i) > 1 ? t.stride(i) : 0;
    s[3] = 1;
  }
  operator const int64_t*() const { return s; }
};
inline Tensor unit_rows(const Tensor& table) { return table.size(1) <= 1 || table.stride(1) == 1 ? table : table.contiguous(); }
inline const void* ptr(const Tensor& t) { return t.const_data_ptr(); }
inline void* out_ptr(const Tensor& t) { return t.mutable_data_ptr(); }
struct Lengths {
  const int32_t* p = nullptr;
  int64_t stride = 0;
  explicit Lengths(const OptTensor& l) {
    if (l) p = l->const_data_ptr<int32_t>(), stride = l->stride(0);
  }
};
inline int clamp_int(int64_t x) { return (int)std::min<int64_t>(x, 0x7fffffff); }
inline void* current_stream(const Tensor& q) { return c10::hip::getCurrentHIPStream(q.device().index()).stream(); }
// From the caching allocator: a workspace belongs to the call and its stream (or to the graph that captures it).
inline Tensor workspace(const Tensor& q, int64_t bytes) { return at::empty({bytes}, q.options().dtype(at::kByte)); }
inline Tensor empty_rows(const Tensor& q) { return at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat)); }
inline Tensor empty_same(const Tensor& q) { return at::empty(q.sizes(), q.options()); }

template <typename F> const c10::TypedOperatorHandle<F> find_op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").template typed<F>();
}
inline bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->requires_grad()) return true;
  return false;
}
inline bool has_tangent(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t->_fw_grad(0).defined()) return true;
  return false;
}

// ---- arguments from Python, positional and complete ---------------------------------------------------------
inline bool tensor_arg(PyObject* x, Tensor& t) {
  if (!THPVariable_Check(x)) return false;
  t = THPVariable_Unpack(x);
  return true;
}
inline bool optional_arg(PyObject* x, OptTensor& t) {
  if (x == Py_None) return true;
  if (!THPVariable_Check(x)) return false;
  t = THPVariable_Unpack(x);
  return true;
}
inline bool int_arg(PyObject* x, int64_t& value) {
  int overflow = 0;
  if (!PyLong_CheckExact(x)) return false;
  value = PyLong_AsLongLongAndOverflow(x, &overflow);
  return overflow == 0;
}
inline bool scale_arg(PyObject* x, const Tensor& q, double& value) {
  if (q.dim() < 1 || (x != Py_None && !PyFloat_CheckExact(x))) return false;
  value = x == Py_None ? 1.0 / std::sqrt((double)q.size(-1)) : PyFloat_AS_DOUBLE(x);
  return true;
}
// None or a float
inline bool eps_arg(PyObject* x, std::optional<double>& value) {
  if (x == Py_None) return true;
  if (!PyFloat_CheckExact(x)) return false;
  value = PyFloat_AS_DOUBLE(x);
  return true;
}

}  // namespace kv_native

// kv_rope_torch.cpp
PyObject* py_qk_norm_rope(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_paged_append_rope(PyObject*, PyObject* const* args, Py_ssize_t n);
