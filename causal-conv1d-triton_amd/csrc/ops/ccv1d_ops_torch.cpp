/* CPython extension `_ccv1d_ops`: the operators of include/ccv1d_ops.h over torch tensors, each in
 * one native call: argument checks, allocation of outputs and workspaces with torch's caching
 * allocator, and the library call on torch's current stream. The Python side (recurrence.py,
 * paged.py) holds the documentation and the autograd wiring. Built with g++ like ccv1d_torch.cpp,
 * for the same reason: a decode step's operators are bound by the host, and reading attributes and
 * allocating cost microseconds in Python and tens of nanoseconds here.
 */
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

#include "ccv1d_ops.h"

namespace {

PyObject* g_error_type = nullptr;

// Thrown with a Python error set.
struct Raised {};

[[noreturn]] void raise(PyObject* type, const char* msg) {
  PyErr_SetString(type, msg);
  throw Raised{};
}

void check(bool ok, const char* msg) {
  if (!ok) raise(PyExc_AssertionError, msg);
}

// A tangent of forward-mode differentiation would be lost without a word.
const at::Tensor& tensor(PyObject* o, const char* msg) {
  if (!THPVariable_Check(o)) raise(PyExc_TypeError, msg);
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
    raise(PyExc_NotImplementedError, "the operators have no forward-mode derivatives");
  return t;
}

// An optional tensor; undefined for None.
at::Tensor optional(PyObject* o, const char* msg) {
  return o == Py_None ? at::Tensor() : tensor(o, msg);
}

int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised{};
  return v;
}

double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised{};
  return v;
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Raised{};
  return v != 0;
}

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return CCV1D_F32;
    case at::kHalf: return CCV1D_F16;
    case at::kBFloat16: return CCV1D_BF16;
    default: raise(PyExc_TypeError, "unsupported dtype (fp32, fp16 or bf16 expected)");
  }
}

bool shaped(const at::Tensor& t, std::initializer_list<int64_t> s) {
  return t.sizes() == at::IntArrayRef(s);
}

at::Tensor unit_last(const at::Tensor& t) {
  return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

// Contiguous and of a type; as it is where it is both (a call into torch costs 0.2 us also then).
at::Tensor as_type(const at::Tensor& t, at::ScalarType type) {
  if (!t.defined() || (t.scalar_type() == type && t.is_contiguous())) return t;
  return t.to(type).contiguous();
}

at::Tensor as_f32(const at::Tensor& t) { return as_type(t, at::kFloat); }
at::Tensor as_i32(const at::Tensor& t) { return as_type(t, at::kInt); }

// Whether int32 cannot hold all whole numbers of a tensor's type.
bool past_i32(const at::Tensor& t) {
  return t.scalar_type() == at::kLong || t.scalar_type() == at::kUInt32 || t.scalar_type() == at::kUInt64;
}

// Whole numbers as int32; those outside its range stay outside any index or length.
at::Tensor as_index(const at::Tensor& t) {
  if (t.defined() && past_i32(t))
    return t.to(at::kLong).clamp(INT32_MIN, INT32_MAX).to(at::kInt).contiguous();
  return as_i32(t);
}

// Sequence ids as they are in 32 or 64 bits: a shorter one could join two sequences or turn one to padding.
at::Tensor as_ids(const at::Tensor& t) {
  return as_type(t, t.defined() && past_i32(t) ? at::kLong : at::kInt);
}

// Tells autograd that a tensor was written to.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// A contiguous tensor in the storage of `base`, from byte `at` on (a multiple of its element's size):
// several small outputs share one allocation.
at::Tensor inside(const at::Tensor& base, int64_t at, at::ScalarType type, int64_t n) {
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

void* stream_of(int64_t dev) {
  return c10::hip::getCurrentHIPStream(static_cast<c10::DeviceIndex>(dev)).stream();
}

at::Tensor scratch(size_t bytes, const at::Tensor& like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : at::Tensor();
}

template <typename A>
void call(int (*fn)(const A*), const A& a) {
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
PyObject* tuple_of(std::initializer_list<at::Tensor> ts) {
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
void no_grad_through(std::initializer_list<const at::Tensor*> ts, const char* msg) {
  if (!c10::GradMode::is_enabled()) return;
  for (const at::Tensor* t : ts) check(!t->defined() || !t->requires_grad(), msg);
}

// ------------------------------------------------------------------------------- recurrence

struct Rec {
  at::Tensor x, gate, decay, igate, seq, init;
  at::ScalarType decay_type{}, init_type{};  // as given
  ccv1d_rec_args a{};
};

// x, gate, decay, input_gate, seq_idx, initial_states, decay_scale
void rec_inputs(PyObject* const* o, Rec& r) {
  r.x = tensor(o[0], "x must be a tensor");
  r.gate = tensor(o[1], "gate must be a tensor");
  r.decay = optional(o[2], "decay must be a tensor or None");
  r.igate = optional(o[3], "input_gate must be a tensor or None");
  r.seq = optional(o[4], "seq_idx must be a tensor or None");
  r.init = optional(o[5], "initial_states must be a tensor or None");
  r.a.decay_scale = (float)number(o[6]);
}

// Checks the inputs and brings them to the form that the library takes.
void rec_check(Rec& r) {
  ccv1d_rec_args& a = r.a;
  check(r.x.dim() == 3, "x must be (batch, seqlen, dim)");
  a.batch = r.x.size(0), a.seqlen = r.x.size(1), a.dim = r.x.size(2);
  check(r.gate.sizes() == r.x.sizes(), "gate must have the shape of x");
  check(!r.igate.defined() || r.igate.sizes() == r.x.sizes(), "input_gate must have the shape of x");
  check(!r.decay.defined() || shaped(r.decay, {a.dim}), "decay must be (dim,)");
  check(!r.seq.defined() || shaped(r.seq, {a.batch, a.seqlen}), "seq_idx must be (batch, seqlen)");
  check(!r.init.defined() || shaped(r.init, {a.batch, a.dim}), "initial_states must be (batch, dim)");
  check(!r.seq.defined() || at::isIntegralType(r.seq.scalar_type(), false),
        "seq_idx must hold integers");
  check(!r.decay.defined() || r.decay.is_floating_point(), "decay must be floating point");
  check(!r.init.defined() || r.init.is_floating_point(), "initial_states must be floating point");
  check(a.decay_scale >= 0.0f, "decay_scale must not be negative");
  check(r.x.is_cuda(), "x must be on a GPU");
  const int64_t dev = r.x.get_device();
  check(r.gate.get_device() == dev, "gate must be on the device of x");
  check(!r.igate.defined() || r.igate.get_device() == dev, "input_gate must be on the device of x");
  check(!r.decay.defined() || r.decay.get_device() == dev, "decay must be on the device of x");
  check(!r.seq.defined() || r.seq.get_device() == dev, "seq_idx must be on the device of x");
  check(!r.init.defined() || r.init.get_device() == dev, "initial_states must be on the device of x");
  a.dtype = dtype_code(r.x);
  check(r.gate.scalar_type() == r.x.scalar_type() &&
            (!r.igate.defined() || r.igate.scalar_type() == r.x.scalar_type()),
        "gate and input_gate must have the dtype of x");
  r.x = unit_last(r.x);
  r.gate = unit_last(r.gate);
  if (r.igate.defined()) r.igate = unit_last(r.igate);
  if (r.decay.defined()) r.decay_type = r.decay.scalar_type();
  if (r.init.defined()) r.init_type = r.init.scalar_type();
  r.decay = as_f32(r.decay);
  r.init = as_f32(r.init);
  r.seq = as_ids(r.seq);
  a.x = ptr(r.x), a.x_stride_b = r.x.stride(0), a.x_stride_t = r.x.stride(1);
  a.gate = ptr(r.gate), a.gate_stride_b = r.gate.stride(0), a.gate_stride_t = r.gate.stride(1);
  if (r.igate.defined()) {
    a.input_gate = ptr(r.igate);
    a.input_gate_stride_b = r.igate.stride(0), a.input_gate_stride_t = r.igate.stride(1);
  }
  a.decay = ptr<float>(r.decay);
  a.seq_idx = ptr(r.seq);
  a.seq_idx_64 = r.seq.defined() && r.seq.scalar_type() == at::kLong;
  a.initial_states = ptr<float>(r.init);
  a.device = (int)dev;
  a.stream = stream_of(dev);
}

struct RecOut {
  at::Tensor out, fin, saved;
};

RecOut rec_forward(Rec& r, bool final_states, bool save) {
  rec_check(r);
  ccv1d_rec_args& a = r.a;
  const auto f32 = r.x.options().dtype(at::kFloat);
  at::Tensor out = at::empty({a.batch, a.seqlen, a.dim}, r.x.options()), fin, saved;
  if (final_states) fin = at::empty({a.batch, a.dim}, f32);
  if (save)
    saved = at::empty(
        {a.batch, (a.seqlen + CCV1D_REC_SAVED_ROWS - 1) / CCV1D_REC_SAVED_ROWS, a.dim}, f32);
  a.workspace_bytes = ccv1d_rec_workspace_bytes(a.batch, a.seqlen, a.dim, 0);
  at::Tensor ws = scratch(a.workspace_bytes, r.x);
  a.out = ptr(out), a.final_states = ptr<float>(fin), a.saved = ptr<float>(saved);
  a.workspace = ptr(ws);
  call(ccv1d_rec_fwd, a);
  return {out, fin, saved};
}

/* rec_fwd(x, gate, decay, input_gate, seq_idx, initial_states, decay_scale, return_final, save)
 *   -> (out, final_states or None, saved or None) */
PyObject* rec_fwd(PyObject* const* o) {
  Rec r;
  rec_inputs(o, r);
  const RecOut res = rec_forward(r, truth(o[7]), truth(o[8]));
  return tuple_of({res.out, res.fin, res.saved});
}

struct RecGrads {
  at::Tensor x, gate, decay, igate, init;  // of the inputs' own types
};

RecGrads rec_backward(Rec& r, const at::Tensor& saved, at::Tensor dout, at::Tensor dfin,
                      bool need_dinitial) {
  rec_check(r);
  ccv1d_rec_args& a = r.a;
  const int64_t dev = a.device;
  check(dout.sizes() == r.x.sizes(), "the gradient of out must have the shape of x");
  check(dout.get_device() == dev, "the gradient of out must be on the device of x");
  check(dout.scalar_type() == r.x.scalar_type(), "the gradient of out must have the dtype of x");
  check(!dfin.defined() || shaped(dfin, {a.batch, a.dim}),
        "the gradient of final_states must be (batch, dim)");
  check(!dfin.defined() || dfin.get_device() == dev,
        "the gradient of final_states must be on the device of x");
  check(saved.scalar_type() == at::kFloat && saved.is_contiguous() && saved.get_device() == dev &&
            shaped(saved, {a.batch,
                           (a.seqlen + CCV1D_REC_SAVED_ROWS - 1) / CCV1D_REC_SAVED_ROWS, a.dim}),
        "saved must be what the forward kept");
  dout = unit_last(dout);
  dfin = as_f32(dfin);
  const auto f32 = r.x.options().dtype(at::kFloat);
  const at::IntArrayRef shape = r.x.sizes();
  at::Tensor dx = at::empty(shape, r.x.options()), dgate = at::empty(shape, r.x.options());
  at::Tensor dig = r.igate.defined() ? at::empty(shape, r.x.options()) : at::Tensor();
  at::Tensor ddecay = r.decay.defined() ? at::empty({a.dim}, f32) : at::Tensor();
  at::Tensor dinit = need_dinitial ? at::empty({a.batch, a.dim}, f32) : at::Tensor();
  a.workspace_bytes = ccv1d_rec_workspace_bytes(a.batch, a.seqlen, a.dim, 1);
  at::Tensor ws = scratch(a.workspace_bytes, r.x);
  a.saved = ptr<float>(saved);
  a.dout = ptr(dout), a.dout_stride_b = dout.stride(0), a.dout_stride_t = dout.stride(1);
  a.dfinal_states = ptr<float>(dfin);
  a.dx = ptr(dx), a.dgate = ptr(dgate), a.dinput_gate = ptr(dig);
  a.ddecay = ptr<float>(ddecay), a.dinitial_states = ptr<float>(dinit);
  a.workspace = ptr(ws);
  call(ccv1d_rec_bwd, a);
  if (ddecay.defined()) ddecay = ddecay.to(r.decay_type);
  if (dinit.defined() && r.init.defined()) dinit = dinit.to(r.init_type);
  return {dx, dgate, ddecay, dig, dinit};
}

/* rec_bwd(x, gate, decay, input_gate, seq_idx, initial_states, decay_scale, saved, dout,
 *         dfinal_states, need_dinitial)
 *   -> (dx, dgate, ddecay or None, dinput_gate or None, dinitial_states or None), the last three of
 *      the inputs' own types */
PyObject* rec_bwd(PyObject* const* o) {
  Rec r;
  rec_inputs(o, r);
  const RecGrads g = rec_backward(r, tensor(o[7], "saved must be a tensor"),
                                  tensor(o[8], "dout must be a tensor"),
                                  optional(o[9], "dfinal_states must be a tensor or None"),
                                  truth(o[10]));
  return tuple_of({g.x, g.gate, g.decay, g.igate, g.init});
}

// The interpreter's lock, which the autograd engine's threads do not hold: errors are Python's.
struct Interpreter {
  PyGILState_STATE state = PyGILState_Ensure();
  ~Interpreter() { PyGILState_Release(state); }
};

/* The autograd node of gated_recurrence_fn. Kept for the backward: the inputs, and the state in front of
 * every 64th row in fp32, from which the backward makes the states between again. In C++ because a
 * training call of little work is bound by the host, and a Python node is a part of that (forward and backward
 * on one machine, runs in turn, which differ by when the engine's thread wakes: B=11 T=38 D=3693 bf16 without
 * decay Python 78 to 81 us, C++ 38 to 65; B=3 T=159 D=320 with decay 105 to 109 and 56 to 93). */
struct RecNode : torch::autograd::Function<RecNode> {
  using Maybe = std::optional<at::Tensor>;
  using Context = torch::autograd::AutogradContext;
  using List = torch::autograd::variable_list;

  static List forward(Context* ctx, const at::Tensor& x, const at::Tensor& gate, const Maybe& decay,
                      const Maybe& igate, const Maybe& seq, const Maybe& init, double decay_scale,
                      bool final_states) {
    Rec r;
    r.x = x, r.gate = gate, r.decay = decay.value_or(at::Tensor());
    r.igate = igate.value_or(at::Tensor()), r.seq = seq.value_or(at::Tensor());
    r.init = init.value_or(at::Tensor());
    r.a.decay_scale = (float)decay_scale;
    List keep = {r.x, r.gate, r.decay, r.igate, r.seq, r.init};
    const RecOut res = rec_forward(r, final_states, true);
    keep.push_back(res.saved);
    ctx->save_for_backward(std::move(keep));
    ctx->saved_data["decay_scale"] = decay_scale;
    ctx->set_materialize_grads(false);
    return final_states ? List{res.out, res.fin} : List{res.out};
  }

  static List backward(Context* ctx, const List& up) {
    const bool graph = c10::GradMode::is_enabled();
    List grads(8);
    {
      const c10::AutoGradMode off(false);
      const List kept = ctx->get_saved_variables();
      Rec r;
      r.x = kept[0], r.gate = kept[1], r.decay = kept[2], r.igate = kept[3], r.seq = kept[4];
      r.init = kept[5];
      r.a.decay_scale = (float)ctx->saved_data["decay_scale"].toDouble();
      const at::Tensor dout = up[0].defined() ? up[0] : at::zeros(r.x.sizes(), r.x.options());
      const bool need = r.init.defined() && r.init.requires_grad();
      const Interpreter held;
      try {
        RecGrads g = rec_backward(r, kept[6], dout, up.size() > 1 ? up[1] : at::Tensor(), need);
        grads[0] = g.x, grads[1] = g.gate, grads[2] = g.decay, grads[3] = g.igate, grads[5] = g.init;
      } catch (const Raised&) {
        python_error e;
        e.persist();
        throw e;
      }
    }
    if (graph) refuse_second(grads);
    return grads;
  }

  // Gradients whose own gradient is refused when it is asked for.
  static void refuse_second(List& grads) {
    List some;
    for (const at::Tensor& g : grads)
      if (g.defined()) some.push_back(g.detach().set_requires_grad(true));
    torch::autograd::DelayedError error("gated_recurrence_fn has no second derivatives",
                                        (int64_t)some.size());
    some = error.apply(std::move(some));
    size_t i = 0;
    for (at::Tensor& g : grads)
      if (g.defined()) g = some[i++];
  }
};

/* rec_train(x, gate, decay, input_gate, seq_idx, initial_states, decay_scale, return_final)
 *   -> (out, final_states or None), recorded by autograd */
PyObject* rec_train(PyObject* const* o) {
  Rec r;
  rec_inputs(o, r);
  auto maybe = [](const at::Tensor& t) { return t.defined() ? RecNode::Maybe(t) : std::nullopt; };
  const RecNode::List res =
      RecNode::apply(r.x, r.gate, maybe(r.decay), maybe(r.igate), maybe(r.seq), maybe(r.init),
                     number(o[6]), truth(o[7]));
  return tuple_of({res[0], res.size() > 1 ? res[1] : at::Tensor()});
}

/* rec_update(x, gate, state, decay, input_gate, state_indices, decay_scale) -> out */
PyObject* rec_update(PyObject* const* o) {
  at::Tensor x = tensor(o[0], "x must be a tensor"), gate = tensor(o[1], "gate must be a tensor");
  const at::Tensor& state = tensor(o[2], "state must be a tensor");
  at::Tensor decay = optional(o[3], "decay must be a tensor or None");
  at::Tensor igate = optional(o[4], "input_gate must be a tensor or None");
  at::Tensor idx = optional(o[5], "state_indices must be a tensor or None");
  ccv1d_rec_update_args a{};
  a.decay_scale = (float)number(o[6]);
  check(a.decay_scale >= 0.0f, "decay_scale must not be negative");
  check(x.dim() == 2, "x must be (rows, dim)");
  a.rows = x.size(0), a.dim = x.size(1);
  check(gate.sizes() == x.sizes(), "gate must have the shape of x");
  check(!igate.defined() || igate.sizes() == x.sizes(), "input_gate must have the shape of x");
  check(!decay.defined() || shaped(decay, {a.dim}), "decay must be (dim,)");
  check(state.dim() == 2 && state.size(1) == a.dim, "state must be (slots, dim)");
  a.slots = state.size(0);
  check(!idx.defined() || shaped(idx, {a.rows}), "state_indices must be (rows,)");
  check(idx.defined() || a.slots >= a.rows, "state must have a slot for each row");
  check(state.scalar_type() == at::kFloat, "state must be fp32");
  check(a.slots == 0 || a.dim <= 1 || state.stride(1) == 1, "state must have a unit channel stride");
  check(a.slots <= 1 || state.stride(0) >= a.dim, "slots of state must not overlap");
  check(!idx.defined() || at::isIntegralType(idx.scalar_type(), false),
        "state_indices must hold integers");
  check(!decay.defined() || decay.is_floating_point(), "decay must be floating point");
  check(x.is_cuda(), "x must be on a GPU");
  const int64_t dev = x.get_device();
  check(gate.get_device() == dev, "gate must be on the device of x");
  check(state.get_device() == dev, "state must be on the device of x");
  check(!igate.defined() || igate.get_device() == dev, "input_gate must be on the device of x");
  check(!decay.defined() || decay.get_device() == dev, "decay must be on the device of x");
  check(!idx.defined() || idx.get_device() == dev, "state_indices must be on the device of x");
  a.dtype = dtype_code(x);
  check(gate.scalar_type() == x.scalar_type() &&
            (!igate.defined() || igate.scalar_type() == x.scalar_type()),
        "gate and input_gate must have the dtype of x");
  no_grad_through({&x, &gate, &decay, &igate, &state},
                  "gated_recurrence_update has no backward: call it under torch.no_grad()");
  x = unit_last(x), gate = unit_last(gate), decay = as_f32(decay), idx = as_index(idx);
  if (igate.defined()) {
    igate = unit_last(igate);
    a.input_gate = ptr(igate), a.input_gate_stride = igate.stride(0);
  }
  at::Tensor out = at::empty({a.rows, a.dim}, x.options());
  a.x = ptr(x), a.x_stride = x.stride(0), a.gate = ptr(gate), a.gate_stride = gate.stride(0);
  a.decay = ptr<float>(decay);
  a.state = ptr<float>(state), a.state_stride = state.stride(0);
  a.state_indices = ptr<int32_t>(idx);
  a.out = ptr(out);
  a.device = (int)dev, a.stream = stream_of(dev);
  call(ccv1d_rec_update, a);
  written(state);
  return tuple_of({out});
}

// ------------------------------------------------------------------------------- paging

// (n,) int32 on a GPU, contiguous.
void check_i32(const at::Tensor& t, int64_t n, int64_t dev, const char* shape, const char* rest) {
  check(t.dim() == 1 && (n < 0 || t.size(0) == n), shape);
  check(t.scalar_type() == at::kInt && t.is_contiguous() && t.get_device() == dev, rest);
}

/* paged_plan(cached_lens, new_lens, block_tables, free_pages, num_free, page_size, max_tokens)
 *   -> (seq_lens, query_start, positions, request_ids, slot_mapping, num_free) */
PyObject* paged_plan(PyObject* const* o) {
  const at::Tensor& cached = tensor(o[0], "cached_lens must be a tensor");
  const at::Tensor& fresh = tensor(o[1], "new_lens must be a tensor");
  const at::Tensor& tables = tensor(o[2], "block_tables must be a tensor");
  const at::Tensor& free = tensor(o[3], "free_pages must be a tensor");
  const at::Tensor& num = tensor(o[4], "num_free must be a tensor");
  ccv1d_paged_plan_args a{};
  a.page_size = integer(o[5]);
  a.max_tokens = integer(o[6]);
  check(a.page_size >= 1, "page_size must be at least 1");
  check(a.max_tokens >= 0, "max_tokens must not be negative");
  check(cached.dim() == 1, "cached_lens must be (requests,)");
  check(cached.is_cuda(), "cached_lens must be on a GPU");
  const int64_t R = cached.size(0), dev = cached.get_device();
  check_i32(cached, R, dev, "cached_lens must be (requests,)", "cached_lens must be contiguous int32");
  check_i32(fresh, R, dev, "new_lens must be (requests,)",
            "new_lens must be contiguous int32 on the device of cached_lens");
  check_i32(free, -1, dev, "free_pages must be (pages,)",
            "free_pages must be contiguous int32 on the device of cached_lens");
  check_i32(num, 1, dev, "num_free must be (1,)",
            "num_free must be int32 on the device of cached_lens");
  check(tables.dim() == 2 && tables.size(0) == R, "block_tables must be (requests, max_pages)");
  check(tables.scalar_type() == at::kInt && tables.get_device() == dev,
        "block_tables must be int32 on the device of cached_lens");
  check(tables.size(1) <= 1 || tables.stride(1) == 1, "rows of block_tables must be contiguous");
  check(R <= 1 || tables.stride(0) >= tables.size(1), "rows of block_tables must not overlap");
  const int64_t N = a.max_tokens;
  // slot_mapping first: its elements are 8 bytes
  const at::Tensor all = at::empty({16 * N + 4 * (R + R + 1 + 1)}, cached.options().dtype(at::kByte));
  int64_t at = 0;
  auto next = [&](at::ScalarType type, int64_t n) {
    at::Tensor t = inside(all, at, type, n);
    at += n * (int64_t)c10::elementSize(type);
    return t;
  };
  at::Tensor slots = next(at::kLong, N), pos = next(at::kInt, N), ids = next(at::kInt, N);
  at::Tensor lens = next(at::kInt, R), start = next(at::kInt, R + 1), left = next(at::kInt, 1);
  a.cached_lens = ptr<int32_t>(cached), a.new_lens = ptr<int32_t>(fresh);
  a.block_tables = ptr<int32_t>(tables), a.block_table_stride = tables.stride(0);
  a.free_pages = ptr<int32_t>(free), a.num_free = ptr<int32_t>(num);
  a.requests = R, a.max_pages = tables.size(1), a.num_free_pages = free.size(0);
  a.seq_lens = ptr<int32_t>(lens), a.query_start = ptr<int32_t>(start);
  a.positions = ptr<int32_t>(pos), a.request_ids = ptr<int32_t>(ids);
  a.slot_mapping = ptr<int64_t>(slots), a.num_free_out = ptr<int32_t>(left);
  a.device = (int)dev, a.stream = stream_of(dev);
  call(ccv1d_paged_plan, a);
  written(tables);
  return tuple_of({lens, start, pos, ids, slots, left});
}

void check_cache(const at::Tensor& t, const at::Tensor& like, const char* shape) {
  check(t.dim() == 4 && t.sizes() == like.sizes(), shape);
  check(t.size(3) <= 1 || t.stride(3) == 1, "the caches must have a unit last stride");
}

// Whether no two elements of a cache share memory: each stride, from the smallest on, passes all that those
// before it reach. (Strides that interleave without meeting are taken to meet.)
bool distinct(const at::Tensor& t) {
  if (t.is_contiguous()) return true;
  std::array<std::pair<int64_t, int64_t>, 4> dims;  // strides and sizes; of one element: (0, 1)
  for (int d = 0; d < 4; ++d)
    dims[d] = t.size(d) > 1 ? std::pair(t.stride(d), t.size(d)) : std::pair(int64_t(0), int64_t(1));
  std::sort(dims.begin(), dims.end());
  int64_t reach = 0;
  for (const auto& [stride, size] : dims) {
    if (size > 1 && stride <= reach) return false;
    reach += (size - 1) * stride;
  }
  return true;
}

/* paged_cache_write(k, v, k_cache, v_cache, slot_mapping) */
PyObject* paged_cache_write(PyObject* const* o) {
  at::Tensor k = tensor(o[0], "k must be a tensor"), v = tensor(o[1], "v must be a tensor");
  const at::Tensor& kc = tensor(o[2], "k_cache must be a tensor");
  const at::Tensor& vc = tensor(o[3], "v_cache must be a tensor");
  const at::Tensor& slots = tensor(o[4], "slot_mapping must be a tensor");
  ccv1d_paged_write_args a{};
  check(kc.dim() == 4, "k_cache must be (num_pages, page_size, kv_heads, head_dim)");
  a.num_pages = kc.size(0), a.page_size = kc.size(1), a.kv_heads = kc.size(2), a.head_dim = kc.size(3);
  check(a.page_size >= 1, "page_size must be at least 1");
  check_cache(kc, kc, "");
  check_cache(vc, kc, "v_cache must have the shape of k_cache");
  check(kc.numel() == 0 || (distinct(kc) && distinct(vc)), "rows of the caches must not overlap");
  check(k.dim() == 3 && k.size(1) == a.kv_heads && k.size(2) == a.head_dim,
        "k must be (tokens, kv_heads, head_dim)");
  check(v.sizes() == k.sizes(), "v must have the shape of k");
  a.tokens = k.size(0);
  check(shaped(slots, {a.tokens}), "slot_mapping must be (tokens,)");
  check(at::isIntegralType(slots.scalar_type(), false), "slot_mapping must hold integers");
  check(k.is_cuda(), "k must be on a GPU");
  const int64_t dev = k.get_device();
  check(v.get_device() == dev && kc.get_device() == dev && vc.get_device() == dev &&
            slots.get_device() == dev,
        "v, the caches and slot_mapping must be on the device of k");
  a.dtype = dtype_code(k);
  check(v.scalar_type() == k.scalar_type() && kc.scalar_type() == k.scalar_type() &&
            vc.scalar_type() == k.scalar_type(),
        "v and the caches must have the dtype of k");
  no_grad_through({&k, &v, &kc, &vc},
                  "paged_cache_write has no backward: call it under torch.no_grad()");
  k = unit_last(k), v = unit_last(v);
  const at::Tensor s = as_type(slots, at::kLong);
  a.k = ptr(k), a.k_stride_t = k.stride(0), a.k_stride_h = k.stride(1);
  a.v = ptr(v), a.v_stride_t = v.stride(0), a.v_stride_h = v.stride(1);
  a.k_cache = ptr(kc), a.v_cache = ptr(vc);
  a.k_cache_stride_p = kc.stride(0), a.k_cache_stride_t = kc.stride(1), a.k_cache_stride_h = kc.stride(2);
  a.v_cache_stride_p = vc.stride(0), a.v_cache_stride_t = vc.stride(1), a.v_cache_stride_h = vc.stride(2);
  a.slot_mapping = ptr<int64_t>(s);
  a.device = (int)dev, a.stream = stream_of(dev);
  call(ccv1d_paged_write, a);
  written(kc);
  written(vc);
  Py_RETURN_NONE;
}

/* paged_attention(q, k_cache, v_cache, block_tables, seq_lens, request_ids, softmax_scale or None,
 *                 window, max_seq_len, return_lse) -> (out, lse or None) */
PyObject* paged_attention(PyObject* const* o) {
  at::Tensor q = tensor(o[0], "q must be a tensor");
  const at::Tensor& kc = tensor(o[1], "k_cache must be a tensor");
  const at::Tensor& vc = tensor(o[2], "v_cache must be a tensor");
  const at::Tensor& tables = tensor(o[3], "block_tables must be a tensor");
  at::Tensor lens = tensor(o[4], "seq_lens must be a tensor");
  at::Tensor ids = optional(o[5], "request_ids must be a tensor or None");
  ccv1d_paged_attn_args a{};
  a.window = integer(o[7]), a.max_seq_len = integer(o[8]);
  check(q.dim() == 3, "q must be (rows, q_heads, head_dim)");
  check(kc.dim() == 4, "k_cache must be (num_pages, page_size, kv_heads, head_dim)");
  a.rows = q.size(0), a.q_heads = q.size(1), a.head_dim = q.size(2);
  a.num_pages = kc.size(0), a.page_size = kc.size(1), a.kv_heads = kc.size(2);
  check(a.page_size >= 1, "page_size must be at least 1");
  check(kc.size(3) == a.head_dim, "the caches must have the head_dim of q");
  check_cache(kc, kc, "");
  check_cache(vc, kc, "v_cache must have the shape of k_cache");
  check(a.kv_heads > 0 && a.q_heads % a.kv_heads == 0, "q_heads must be a multiple of kv_heads");
  check(a.head_dim >= 8 && a.head_dim % 8 == 0 && a.head_dim <= CCV1D_PAGED_MAX_HEAD_DIM,
        "head_dim must be a multiple of 8, at most 256");
  check(shaped(lens, {a.rows}), "seq_lens must be (rows,)");
  check(!ids.defined() || shaped(ids, {a.rows}), "request_ids must be (rows,)");
  check(tables.dim() == 2, "block_tables must be (requests, max_pages)");
  a.requests = tables.size(0), a.max_pages = tables.size(1);
  check(ids.defined() || a.requests >= a.rows, "block_tables must have a row for each row of q");
  check(a.window >= 0, "window must be at least 1");
  check(a.max_seq_len >= 0, "max_seq_len must not be negative");
  check(tables.scalar_type() == at::kInt, "block_tables must be int32");
  check(a.max_pages <= 1 || tables.stride(1) == 1, "rows of block_tables must be contiguous");
  check(at::isIntegralType(lens.scalar_type(), false) &&
            (!ids.defined() || at::isIntegralType(ids.scalar_type(), false)),
        "seq_lens and request_ids must hold integers");
  check(q.is_cuda(), "q must be on a GPU");
  const int64_t dev = q.get_device();
  check(kc.get_device() == dev && vc.get_device() == dev && tables.get_device() == dev &&
            lens.get_device() == dev && (!ids.defined() || ids.get_device() == dev),
        "the caches, block_tables, seq_lens and request_ids must be on the device of q");
  a.dtype = dtype_code(q);
  check(kc.scalar_type() == q.scalar_type() && vc.scalar_type() == q.scalar_type(),
        "the caches must have the dtype of q");
  no_grad_through({&q, &kc, &vc}, "paged_attention has no backward: call it under torch.no_grad()");
  a.scale = o[6] == Py_None ? 1.0f / std::sqrt((float)a.head_dim) : (float)number(o[6]);
  q = unit_last(q), lens = as_index(lens), ids = as_index(ids);
  at::Tensor out = at::empty({a.rows, a.q_heads, a.head_dim}, q.options());
  at::Tensor lse = truth(o[9]) ? at::empty({a.rows, a.q_heads}, q.options().dtype(at::kFloat))
                               : at::Tensor();
  a.q = ptr(q), a.q_stride_r = q.stride(0), a.q_stride_h = q.stride(1);
  a.k_cache = ptr(kc), a.v_cache = ptr(vc);
  a.k_cache_stride_p = kc.stride(0), a.k_cache_stride_t = kc.stride(1), a.k_cache_stride_h = kc.stride(2);
  a.v_cache_stride_p = vc.stride(0), a.v_cache_stride_t = vc.stride(1), a.v_cache_stride_h = vc.stride(2);
  a.block_tables = ptr<int32_t>(tables), a.block_table_stride = tables.stride(0);
  a.seq_lens = ptr<int32_t>(lens), a.request_ids = ptr<int32_t>(ids);
  a.out = ptr(out), a.lse = ptr<float>(lse);
  a.device = (int)dev, a.stream = stream_of(dev);
  a.workspace_bytes = ccv1d_paged_attn_workspace_bytes(&a);
  at::Tensor ws = scratch(a.workspace_bytes, q);
  a.workspace = ptr(ws);
  call(ccv1d_paged_attn, a);
  return tuple_of({out, lse});
}

template <PyObject* (*IMPL)(PyObject* const*), Py_ssize_t N>
PyObject* native_call(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "takes %zd arguments (%zd given)", N, n);
    return nullptr;
  }
  try {
    return IMPL(a);
  } catch (const Raised&) {
    return nullptr;
  } catch (const std::exception&) {  // torch's, with their types: out of memory among them
    torch::translate_exception_to_python(std::current_exception());
    return nullptr;
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown error");
    return nullptr;
  }
}

PyObject* set_error_type(PyObject*, PyObject* t) {
  if (!PyType_Check(t) || !PyType_IsSubtype(reinterpret_cast<PyTypeObject*>(t),
                                            reinterpret_cast<PyTypeObject*>(PyExc_Exception))) {
    PyErr_SetString(PyExc_TypeError, "an exception type is expected");
    return nullptr;
  }
  Py_INCREF(t);
  Py_XDECREF(g_error_type);
  g_error_type = t;
  Py_RETURN_NONE;
}

template <PyObject* (*IMPL)(PyObject* const*), Py_ssize_t N>
PyMethodDef method(const char* name, const char* doc) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(native_call<IMPL, N>)),
          METH_FASTCALL, doc};
}

PyMethodDef methods[] = {
    method<rec_fwd, 9>("rec_fwd", "forward of the gated recurrence"),
    method<rec_bwd, 11>("rec_bwd", "backward of the gated recurrence"),
    method<rec_train, 8>("rec_train", "the gated recurrence, recorded by autograd"),
    method<rec_update, 7>("rec_update", "one token of each request, states in place"),
    method<paged_plan, 7>("paged_plan", "plan of a batch over paged caches"),
    method<paged_cache_write, 5>("paged_cache_write", "keys and values to their slots"),
    method<paged_attention, 10>("paged_attention", "attention of one token over paged caches"),
    {"set_error_type", set_error_type, METH_O, "exception type for library errors"},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {
    PyModuleDef_HEAD_INIT, "_ccv1d_ops",
    "the operators of ccv1d_ops.h over torch tensors, each in one native call", -1, methods,
    nullptr, nullptr, nullptr, nullptr,
};

}  // namespace

PyMODINIT_FUNC PyInit__ccv1d_ops(void) { return PyModule_Create(&module); }
