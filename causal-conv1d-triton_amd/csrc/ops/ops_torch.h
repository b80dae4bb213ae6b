/* What the CPython extension `_ccv1d_ops` shares between its sources: reading and checking arguments, brought
 * to the forms that the library takes, and calling it. */
#pragma once

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <exception>
#include <initializer_list>
#include <optional>
#include <utility>

#include "ccv1d_layer.h"
#include "ccv1d_ops.h"

namespace ccv1d_torch {

inline PyObject* g_error_type = nullptr;

// Thrown with a Python error set.
struct Raised {};

[[noreturn]] inline void raise(PyObject* type, const char* msg) {
  PyErr_SetString(type, msg);
  throw Raised{};
}

inline void check(bool ok, const char* msg) {
  if (!ok) raise(PyExc_AssertionError, msg);
}

// A tangent of forward-mode differentiation would be lost without a word.
inline const at::Tensor& tensor(PyObject* o, const char* msg) {
  if (!THPVariable_Check(o)) raise(PyExc_TypeError, msg);
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
    raise(PyExc_NotImplementedError, "the operators have no forward-mode derivatives");
  return t;
}

// An optional tensor; undefined for None.
inline at::Tensor optional(PyObject* o, const char* msg) {
  return o == Py_None ? at::Tensor() : tensor(o, msg);
}

inline int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised{};
  return v;
}

inline double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised{};
  return v;
}

inline bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Raised{};
  return v != 0;
}

inline int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return CCV1D_F32;
    case at::kHalf: return CCV1D_F16;
    case at::kBFloat16: return CCV1D_BF16;
    default: raise(PyExc_TypeError, "unsupported dtype (fp32, fp16 or bf16 expected)");
  }
}

inline bool shaped(const at::Tensor& t, std::initializer_list<int64_t> s) {
  return t.sizes() == at::IntArrayRef(s);
}

inline at::Tensor unit_last(const at::Tensor& t) {
  return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

// Contiguous and of a type; as it is where it is both (a call into torch costs 0.2 us also then).
inline at::Tensor as_type(const at::Tensor& t, at::ScalarType type) {
  if (!t.defined() || (t.scalar_type() == type && t.is_contiguous())) return t;
  return t.to(type).contiguous();
}

inline at::Tensor as_f32(const at::Tensor& t) { return as_type(t, at::kFloat); }
inline at::Tensor as_i32(const at::Tensor& t) { return as_type(t, at::kInt); }

// Whether int32 cannot hold all whole numbers of a tensor's type.
inline bool past_i32(const at::Tensor& t) {
  return t.scalar_type() == at::kLong || t.scalar_type() == at::kUInt32 || t.scalar_type() == at::kUInt64;
}

// Whole numbers as int32; those outside its range stay outside any index or length.
inline at::Tensor as_index(const at::Tensor& t) {
  if (t.defined() && past_i32(t))
    return t.to(at::kLong).clamp(INT32_MIN, INT32_MAX).to(at::kInt).contiguous();
  return as_i32(t);
}

// Sequence ids as they are in 32 or 64 bits: a shorter one could join two sequences or turn one to padding.
inline at::Tensor as_ids(const at::Tensor& t) {
  return as_type(t, t.defined() && past_i32(t) ? at::kLong : at::kInt);
}

// Tells autograd that a tensor was written to.
inline void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// A contiguous tensor in the storage of `base`, from byte `at` on (a multiple of its element's size):
// several small outputs share one allocation.
inline at::Tensor inside(const at::Tensor& base, int64_t at, at::ScalarType type, int64_t n) {
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(
      c10::Storage(base.storage()), base.key_set(), c10::scalarTypeToTypeMeta(type));
  t.unsafeGetTensorImpl()->set_storage_offset(at / (int64_t)c10::elementSize(type));
  t.unsafeGetTensorImpl()->set_sizes_contiguous(at::IntArrayRef(&n, 1));
  return t;
}

// The address of a tensor, null where there is none. One without memory of its own (a subclass that wraps
// other tensors, a fake tensor) is refused: to the library its null would mean that the tensor is absent.
template <typename P = void>
P* ptr(const at::Tensor& t) {
  if (!t.defined()) return nullptr;
  void* p = t.data_ptr();
  if (!p && t.numel() > 0)
    raise(PyExc_TypeError, "a tensor without memory of its own (a wrapper subclass, say) is not supported");
  return static_cast<P*>(p);
}

inline void* stream_of(int64_t dev) {
  return c10::hip::getCurrentHIPStream(static_cast<c10::DeviceIndex>(dev)).stream();
}

inline at::Tensor scratch(size_t bytes, const at::Tensor& like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : at::Tensor();
}

template <typename A>
inline void call(int (*fn)(const A*), const A& a) {
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = fn(&a);
  Py_END_ALLOW_THREADS
  if (rc) {
    PyErr_Format(g_error_type ? g_error_type : PyExc_RuntimeError, "libccv1d error %d: %s", rc,
                 ccv1d_last_error());
    throw Raised{};
  }
}

// A tuple of tensors, None for undefined ones.
inline PyObject* tuple_of(std::initializer_list<at::Tensor> ts) {
  PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
  if (!r) throw Raised{};
  Py_ssize_t i = 0;
  for (const at::Tensor& t : ts) {
    PyObject* o = t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None);
    if (!o) {
      Py_DECREF(r);
      throw Raised{};
    }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

// Writes in place are not recorded by autograd.
inline void no_grad_through(std::initializer_list<const at::Tensor*> ts, const char* msg) {
  if (!c10::GradMode::is_enabled()) return;
  for (const at::Tensor* t : ts) check(!t->defined() || !t->requires_grad(), msg);
}

// The interpreter's lock, which the autograd engine's threads do not hold: errors are Python's.
struct Interpreter {
  PyGILState_STATE state = PyGILState_Ensure();
  ~Interpreter() { PyGILState_Release(state); }
};

// Gradients whose own gradient is refused when it is asked for.
inline void refuse_second(torch::autograd::variable_list& grads, const char* what) {
  torch::autograd::variable_list some;
  for (const at::Tensor& g : grads)
    if (g.defined()) some.push_back(g.detach().set_requires_grad(true));
  torch::autograd::DelayedError error(what, (int64_t)some.size());
  some = error.apply(std::move(some));
  size_t i = 0;
  for (at::Tensor& g : grads)
    if (g.defined()) g = some[i++];
}

// The operators of ccv1d_layer_torch.cpp.
PyObject* delta_fwd(PyObject* const* o);
PyObject* delta_bwd(PyObject* const* o);
PyObject* delta_train(PyObject* const* o);
PyObject* delta_update(PyObject* const* o);
PyObject* norm_fwd(PyObject* const* o);
PyObject* norm_bwd(PyObject* const* o);
PyObject* norm_train(PyObject* const* o);

}  // namespace ccv1d_torch
