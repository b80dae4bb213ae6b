/* The operators of include/ccv1d_layer.h over torch tensors, a part of the extension `_ccv1d_ops`: the gated delta
 * rule and the norms around a block. The Python side is delta.py and norm.py. */
#include "ops_torch.h"

namespace ccv1d_torch {

namespace {

using Maybe = std::optional<at::Tensor>;
using Context = torch::autograd::AutogradContext;
using List = torch::autograd::variable_list;

Maybe maybe(const at::Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }

// A backward pass in the engine's thread: Python's errors become torch's.
template <typename F>
void in_engine(F&& body) {
  const Interpreter held;
  try {
    body();
  } catch (const Raised&) {
    python_error e;
    e.persist();
    throw e;
  }
}

// ------------------------------------------------------------------------------- delta rule

struct Delta {
  at::Tensor q, k, v, g, beta, seq, init;
  at::ScalarType init_type{};  // as given
  std::optional<double> scale;
  ccv1d_delta_args a{};
};

// q, k, v, log_decay, beta, seq_idx, initial_states, scale or None
void delta_inputs(PyObject* const* o, Delta& d) {
  d.q = tensor(o[0], "q must be a tensor");
  d.k = tensor(o[1], "k must be a tensor");
  d.v = tensor(o[2], "v must be a tensor");
  d.g = tensor(o[3], "log_decay must be a tensor");
  d.beta = tensor(o[4], "beta must be a tensor");
  d.seq = optional(o[5], "seq_idx must be a tensor or None");
  d.init = optional(o[6], "initial_states must be a tensor or None");
  if (o[7] != Py_None) d.scale = number(o[7]);
}

float scale_of(const std::optional<double>& scale, int64_t key_dim) {
  return scale ? (float)*scale : 1.0f / std::sqrt((float)key_dim);
}

// Checks the inputs and brings them to the form that the library takes.
void delta_check(Delta& d) {
  ccv1d_delta_args& a = d.a;
  check(d.k.dim() == 4, "k must be (batch, seqlen, key_heads, key_dim)");
  check(d.v.dim() == 4, "v must be (batch, seqlen, heads, value_dim)");
  check(d.q.sizes() == d.k.sizes(), "q must have the shape of k");
  a.batch = d.k.size(0), a.seqlen = d.k.size(1), a.key_heads = d.k.size(2), a.key_dim = d.k.size(3);
  a.heads = d.v.size(2), a.value_dim = d.v.size(3);
  check(d.v.size(0) == a.batch && d.v.size(1) == a.seqlen, "v must have the batch and seqlen of k");
  check(a.key_heads > 0 && a.heads > 0 && a.heads % a.key_heads == 0,
        "the heads of v must be a multiple of the heads of k");
  check(a.key_dim >= 1 && a.key_dim <= CCV1D_DELTA_MAX_KEY_DIM, "key_dim must be 1 to 256");
  check(a.value_dim >= 1, "value_dim must be at least 1");
  check(shaped(d.g, {a.batch, a.seqlen, a.heads}), "log_decay must be (batch, seqlen, heads)");
  check(shaped(d.beta, {a.batch, a.seqlen, a.heads}), "beta must be (batch, seqlen, heads)");
  check(!d.seq.defined() || shaped(d.seq, {a.batch, a.seqlen}), "seq_idx must be (batch, seqlen)");
  check(!d.seq.defined() || at::isIntegralType(d.seq.scalar_type(), false), "seq_idx must hold integers");
  check(!d.init.defined() || shaped(d.init, {a.batch, a.heads, a.key_dim, a.value_dim}),
        "initial_states must be (batch, heads, key_dim, value_dim)");
  check(!d.init.defined() || d.init.is_floating_point(), "initial_states must be floating point");
  check(d.k.is_cuda(), "k must be on a GPU");
  const int64_t dev = d.k.get_device();
  check(d.q.get_device() == dev && d.v.get_device() == dev && d.g.get_device() == dev &&
            d.beta.get_device() == dev && (!d.seq.defined() || d.seq.get_device() == dev) &&
            (!d.init.defined() || d.init.get_device() == dev),
        "q, v, log_decay, beta, seq_idx and initial_states must be on the device of k");
  a.dtype = dtype_code(d.k);
  check(d.q.scalar_type() == d.k.scalar_type() && d.v.scalar_type() == d.k.scalar_type(),
        "q and v must have the dtype of k");
  a.log_decay_dtype = dtype_code(d.g), a.beta_dtype = dtype_code(d.beta);
  d.q = unit_last(d.q), d.k = unit_last(d.k), d.v = unit_last(d.v);
  if (d.init.defined()) d.init_type = d.init.scalar_type();
  d.init = as_f32(d.init);
  d.seq = as_ids(d.seq);
  a.scale = scale_of(d.scale, a.key_dim);
  a.q = ptr(d.q), a.q_stride_b = d.q.stride(0), a.q_stride_t = d.q.stride(1), a.q_stride_h = d.q.stride(2);
  a.k = ptr(d.k), a.k_stride_b = d.k.stride(0), a.k_stride_t = d.k.stride(1), a.k_stride_h = d.k.stride(2);
  a.v = ptr(d.v), a.v_stride_b = d.v.stride(0), a.v_stride_t = d.v.stride(1), a.v_stride_h = d.v.stride(2);
  a.log_decay = ptr(d.g), a.log_decay_stride_b = d.g.stride(0), a.log_decay_stride_t = d.g.stride(1);
  a.log_decay_stride_h = d.g.stride(2);
  a.beta = ptr(d.beta), a.beta_stride_b = d.beta.stride(0), a.beta_stride_t = d.beta.stride(1);
  a.beta_stride_h = d.beta.stride(2);
  a.seq_idx = ptr(d.seq);
  a.seq_idx_64 = d.seq.defined() && d.seq.scalar_type() == at::kLong;
  a.initial_states = ptr<float>(d.init);
  a.device = (int)dev;
  a.stream = stream_of(dev);
}

struct DeltaOut {
  at::Tensor out, fin, saved;
};

DeltaOut delta_forward(Delta& d, bool final_states, bool save) {
  delta_check(d);
  ccv1d_delta_args& a = d.a;
  const auto f32 = d.k.options().dtype(at::kFloat);
  at::Tensor out = at::empty({a.batch, a.seqlen, a.heads, a.value_dim}, d.k.options()), fin, saved;
  if (final_states) fin = at::empty({a.batch, a.heads, a.key_dim, a.value_dim}, f32);
  if (save) saved = at::empty({(int64_t)ccv1d_delta_saved_floats(&a)}, f32);
  a.workspace_bytes = ccv1d_delta_workspace_bytes(&a, 0);
  const at::Tensor ws = scratch(a.workspace_bytes, d.k);
  a.out = ptr(out), a.final_states = ptr<float>(fin), a.saved = ptr<float>(saved);
  a.workspace = ptr(ws);
  call(ccv1d_delta_fwd, a);
  return {out, fin, saved};
}

struct DeltaGrads {
  at::Tensor q, k, v, g, beta, init;  // of the inputs' own types
};

DeltaGrads delta_backward(Delta& d, const at::Tensor& saved, at::Tensor dout, at::Tensor dfin, bool need_dinitial) {
  delta_check(d);
  ccv1d_delta_args& a = d.a;
  const int64_t dev = a.device;
  check(dout.sizes() == d.v.sizes(), "the gradient of out must have the shape of v");
  check(dout.get_device() == dev, "the gradient of out must be on the device of k");
  check(dout.scalar_type() == d.k.scalar_type(), "the gradient of out must have the dtype of k");
  check(!dfin.defined() || shaped(dfin, {a.batch, a.heads, a.key_dim, a.value_dim}),
        "the gradient of final_states must be (batch, heads, key_dim, value_dim)");
  check(!dfin.defined() || dfin.get_device() == dev, "the gradient of final_states must be on the device of k");
  check(saved.scalar_type() == at::kFloat && saved.is_contiguous() && saved.get_device() == dev &&
            shaped(saved, {(int64_t)ccv1d_delta_saved_floats(&a)}),
        "saved must be what the forward kept");
  dout = unit_last(dout);
  dfin = as_f32(dfin);
  DeltaGrads r;
  r.q = at::empty(d.q.sizes(), d.q.options()), r.k = at::empty(d.k.sizes(), d.k.options());
  r.v = at::empty(d.v.sizes(), d.v.options());
  r.g = at::empty(d.g.sizes(), d.g.options()), r.beta = at::empty(d.beta.sizes(), d.beta.options());
  if (need_dinitial)
    r.init = at::empty({a.batch, a.heads, a.key_dim, a.value_dim}, d.k.options().dtype(at::kFloat));
  a.workspace_bytes = ccv1d_delta_workspace_bytes(&a, 1);
  const at::Tensor ws = scratch(a.workspace_bytes, d.k);
  a.saved = ptr<float>(saved);
  a.dout = ptr(dout), a.dout_stride_b = dout.stride(0), a.dout_stride_t = dout.stride(1);
  a.dout_stride_h = dout.stride(2);
  a.dfinal_states = ptr<float>(dfin);
  a.dq = ptr(r.q), a.dk = ptr(r.k), a.dv = ptr(r.v), a.dlog_decay = ptr(r.g), a.dbeta = ptr(r.beta);
  a.dinitial_states = ptr<float>(r.init);
  a.workspace = ptr(ws);
  call(ccv1d_delta_bwd, a);
  if (r.init.defined() && d.init.defined()) r.init = r.init.to(d.init_type);
  return r;
}

/* The autograd node of gated_delta_fn. Kept for the backward: the inputs, and in fp32 the state in front of every
 * chunk of 64 rows and the rows' corrections (`saved`). */
struct DeltaNode : torch::autograd::Function<DeltaNode> {
  static List forward(Context* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& g,
                      const at::Tensor& beta, const Maybe& seq, const Maybe& init, std::optional<double> scale,
                      bool final_states) {
    Delta d;
    d.q = q, d.k = k, d.v = v, d.g = g, d.beta = beta;
    d.seq = seq.value_or(at::Tensor()), d.init = init.value_or(at::Tensor());
    d.scale = scale;
    List keep = {d.q, d.k, d.v, d.g, d.beta, d.seq, d.init};
    const DeltaOut res = delta_forward(d, final_states, true);
    keep.push_back(res.saved);
    ctx->save_for_backward(std::move(keep));
    ctx->saved_data["scale"] = (double)d.a.scale;
    ctx->set_materialize_grads(false);
    return final_states ? List{res.out, res.fin} : List{res.out};
  }

  static List backward(Context* ctx, const List& up) {
    const bool graph = c10::GradMode::is_enabled();
    List grads(9);
    {
      const c10::AutoGradMode off(false);
      const List kept = ctx->get_saved_variables();
      Delta d;
      d.q = kept[0], d.k = kept[1], d.v = kept[2], d.g = kept[3], d.beta = kept[4], d.seq = kept[5];
      d.init = kept[6];
      d.scale = ctx->saved_data["scale"].toDouble();
      const at::Tensor dout = up[0].defined() ? up[0] : at::zeros(d.v.sizes(), d.v.options());
      const bool need = d.init.defined() && d.init.requires_grad();
      in_engine([&] {
        const DeltaGrads r = delta_backward(d, kept[7], dout, up.size() > 1 ? up[1] : at::Tensor(), need);
        grads[0] = r.q, grads[1] = r.k, grads[2] = r.v, grads[3] = r.g, grads[4] = r.beta, grads[6] = r.init;
      });
    }
    if (graph) refuse_second(grads, "gated_delta_fn has no second derivatives");
    return grads;
  }
};

// ------------------------------------------------------------------------------- norms

struct Norm {
  at::Tensor x, residual, post, gate, scale, pre;
  double factor = 1.0, eps = 0.0;
  int activation = 0;
  ccv1d_norm_args a{};
};

// x, residual, post_weight, gate, scale (a tensor, a number or None), pre_weight, eps, activation
void norm_inputs(PyObject* const* o, Norm& n) {
  n.x = tensor(o[0], "x must be a tensor");
  n.residual = optional(o[1], "residual must be a tensor or None");
  n.post = optional(o[2], "post_weight must be a tensor or None");
  n.gate = optional(o[3], "gate must be a tensor or None");
  if (THPVariable_Check(o[4])) n.scale = tensor(o[4], "");
  else if (o[4] != Py_None) n.factor = number(o[4]);
  n.pre = optional(o[5], "pre_weight must be a tensor or None");
  n.eps = number(o[6]);
  n.activation = (int)integer(o[7]);
}

struct Rows {
  int64_t outer, inner, stride_o, stride_i;
};

// The leading dimensions of a tensor as two, with a stride for each; whether that is possible.
bool two_strides(const at::Tensor& t, int64_t outer, int64_t inner, int64_t lead_inner, Rows& r) {
  // merges dimensions [from, to) into one stride
  auto merged = [&](int64_t from, int64_t to, int64_t& stride) {
    stride = 0;
    int64_t size = 1;
    for (int64_t d = to - 1; d >= from; --d) {
      if (t.size(d) == 1) continue;
      if (size == 1) stride = t.stride(d);
      else if (t.stride(d) != stride * size) return false;
      size *= t.size(d);
    }
    return true;
  };
  r.outer = outer, r.inner = inner;
  return merged(0, lead_inner, r.stride_o) && merged(lead_inner, t.dim() - 1, r.stride_i);
}

// A tensor of rows as the library takes it: unit last stride, two strides for its rows.
Rows as_rows(at::Tensor& t, int64_t outer, int64_t inner, int64_t lead_inner) {
  Rows r;
  t = unit_last(t);
  if (!two_strides(t, outer, inner, lead_inner, r)) {
    t = t.contiguous();
    two_strides(t, outer, inner, lead_inner, r);
  }
  return r;
}

void norm_check(Norm& n) {
  ccv1d_norm_args& a = n.a;
  check(n.x.dim() >= 1, "x must be (..., dim)");
  a.dim = n.x.size(-1);
  check(a.dim >= 1 && a.dim <= CCV1D_NORM_MAX_DIM, "dim must be 1 to 8192");
  check(n.post.defined() || n.pre.defined(), "post_weight or pre_weight must be given");
  check(!n.residual.defined() || n.residual.sizes() == n.x.sizes(), "residual must have the shape of x");
  check(!n.gate.defined() || n.gate.sizes() == n.x.sizes(), "gate must have the shape of x");
  check(!n.post.defined() || shaped(n.post, {a.dim}), "post_weight must be (dim,)");
  check(!n.scale.defined() || shaped(n.scale, {a.dim}), "scale must be a number or (dim,)");
  check(!n.pre.defined() || shaped(n.pre, {a.dim}), "pre_weight must be (dim,)");
  check(n.eps >= 0.0, "eps must not be negative");
  check(n.x.is_cuda(), "x must be on a GPU");
  const int64_t dev = n.x.get_device();
  for (const at::Tensor* t : {&n.residual, &n.post, &n.gate, &n.scale, &n.pre})
    check(!t->defined() || t->get_device() == dev,
          "residual, gate, scale and the weights must be on the device of x");
  a.dtype = a.residual_dtype = dtype_code(n.x);
  check(!n.gate.defined() || n.gate.scalar_type() == n.x.scalar_type(), "gate must have the dtype of x");
  if (n.residual.defined()) {
    a.residual_dtype = dtype_code(n.residual);
    check(a.residual_dtype == a.dtype || a.residual_dtype == CCV1D_F32,
          "residual must have the dtype of x or be fp32");
  }
  if (n.post.defined()) a.post_dtype = dtype_code(n.post), n.post = n.post.contiguous();
  if (n.scale.defined()) a.scale_dtype = dtype_code(n.scale), n.scale = n.scale.contiguous();
  if (n.pre.defined()) a.pre_dtype = dtype_code(n.pre), n.pre = n.pre.contiguous();
  // Rows by two indices: the last leading dimension that a tensor's strides keep apart from the ones before
  // it is the inner one; one cut serves all.
  const int64_t lead = n.x.dim() - 1;
  int64_t cut = lead > 1 ? lead - 1 : lead;
  a.inner = 1;
  for (int64_t d = cut; d < lead; ++d) a.inner *= n.x.size(d);
  a.outer = 1;
  for (int64_t d = 0; d < cut; ++d) a.outer *= n.x.size(d);
  Rows r = as_rows(n.x, a.outer, a.inner, cut);
  a.x = ptr(n.x), a.x_stride_o = r.stride_o, a.x_stride_i = r.stride_i;
  if (n.gate.defined()) {
    r = as_rows(n.gate, a.outer, a.inner, cut);
    a.gate = ptr(n.gate), a.gate_stride_o = r.stride_o, a.gate_stride_i = r.stride_i;
  }
  if (n.residual.defined()) {
    r = as_rows(n.residual, a.outer, a.inner, cut);
    a.residual = ptr(n.residual), a.residual_stride_o = r.stride_o, a.residual_stride_i = r.stride_i;
  }
  a.post_weight = ptr(n.post), a.scale_weight = ptr(n.scale), a.pre_weight = ptr(n.pre);
  a.scale = (float)n.factor, a.eps = (float)n.eps;
  a.activation = n.activation;
  a.device = (int)dev;
  a.stream = stream_of(dev);
}

at::ScalarType residual_type(const Norm& n) {
  return n.residual.defined() ? n.residual.scalar_type() : n.x.scalar_type();
}

struct NormOut {
  at::Tensor y, r;
};

NormOut norm_forward(Norm& n) {
  norm_check(n);
  ccv1d_norm_args& a = n.a;
  const at::IntArrayRef shape = n.x.sizes();
  NormOut o;
  o.r = at::empty(shape, n.x.options().dtype(residual_type(n)));
  if (n.pre.defined()) o.y = at::empty(shape, n.x.options());
  a.r = ptr(o.r), a.y = ptr(o.y);
  call(ccv1d_norm_fwd, a);
  return o;
}

struct NormGrads {
  at::Tensor x, residual, post, gate, scale, pre;
};

NormGrads norm_backward(Norm& n, at::Tensor dr, at::Tensor dy, bool need_dresidual) {
  norm_check(n);
  ccv1d_norm_args& a = n.a;
  const int64_t dev = a.device, lead = n.x.dim() - 1, cut = lead > 1 ? lead - 1 : lead;
  const at::IntArrayRef shape = n.x.sizes();
  check(!dr.defined() || dr.sizes() == shape, "the gradient of r must have the shape of x");
  check(!dy.defined() || dy.sizes() == shape, "the gradient of y must have the shape of x");
  check(!dr.defined() || dr.scalar_type() == residual_type(n), "the gradient of r must have r's dtype");
  check(!dy.defined() || (n.pre.defined() && dy.scalar_type() == n.x.scalar_type()),
        "the gradient of y must have the dtype of x");
  check((!dr.defined() || dr.get_device() == dev) && (!dy.defined() || dy.get_device() == dev),
        "the gradients must be on the device of x");
  if (dr.defined()) {
    const Rows r = as_rows(dr, a.outer, a.inner, cut);
    a.dr = ptr(dr), a.dr_stride_o = r.stride_o, a.dr_stride_i = r.stride_i;
  }
  if (dy.defined()) {
    const Rows r = as_rows(dy, a.outer, a.inner, cut);
    a.dy = ptr(dy), a.dy_stride_o = r.stride_o, a.dy_stride_i = r.stride_i;
  }
  NormGrads g;
  auto like = [](const at::Tensor& t) { return t.defined() ? at::empty(t.sizes(), t.options()) : at::Tensor(); };
  g.x = like(n.x), g.gate = like(n.gate), g.post = like(n.post), g.scale = like(n.scale), g.pre = like(n.pre);
  if (need_dresidual) g.residual = like(n.residual);
  a.dx = ptr(g.x), a.dgate = ptr(g.gate), a.dresidual = ptr(g.residual);
  a.dpost_weight = ptr(g.post), a.dscale_weight = ptr(g.scale), a.dpre_weight = ptr(g.pre);
  a.workspace_bytes = ccv1d_norm_workspace_bytes(&a);
  const at::Tensor ws = scratch(a.workspace_bytes, n.x);
  a.workspace = ptr(ws);
  call(ccv1d_norm_bwd, a);
  return g;
}

/* The autograd node of block_norm_fn. Kept for the backward: the inputs alone, from which r and the rows'
 * norms are made again. */
struct NormNode : torch::autograd::Function<NormNode> {
  static List forward(Context* ctx, const at::Tensor& x, const Maybe& residual, const Maybe& post, const Maybe& gate,
                      const Maybe& scale, const Maybe& pre, double factor, double eps, int64_t activation) {
    Norm n;
    n.x = x, n.residual = residual.value_or(at::Tensor()), n.post = post.value_or(at::Tensor());
    n.gate = gate.value_or(at::Tensor()), n.scale = scale.value_or(at::Tensor()), n.pre = pre.value_or(at::Tensor());
    n.factor = factor, n.eps = eps, n.activation = (int)activation;
    List keep = {n.x, n.residual, n.post, n.gate, n.scale, n.pre};
    const NormOut res = norm_forward(n);
    ctx->save_for_backward(std::move(keep));
    ctx->saved_data["factor"] = factor;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["activation"] = activation;
    ctx->set_materialize_grads(false);
    return res.y.defined() ? List{res.r, res.y} : List{res.r};
  }

  static List backward(Context* ctx, const List& up) {
    const bool graph = c10::GradMode::is_enabled();
    List grads(9);
    {
      const c10::AutoGradMode off(false);
      const List kept = ctx->get_saved_variables();
      Norm n;
      n.x = kept[0], n.residual = kept[1], n.post = kept[2], n.gate = kept[3], n.scale = kept[4], n.pre = kept[5];
      n.factor = ctx->saved_data["factor"].toDouble();
      n.eps = ctx->saved_data["eps"].toDouble();
      n.activation = (int)ctx->saved_data["activation"].toInt();
      const bool need = n.residual.defined() && n.residual.requires_grad();
      in_engine([&] {
        const NormGrads g = norm_backward(n, up[0], up.size() > 1 ? up[1] : at::Tensor(), need);
        grads[0] = g.x, grads[1] = g.residual, grads[2] = g.post, grads[3] = g.gate, grads[4] = g.scale;
        grads[5] = g.pre;
      });
    }
    if (graph) refuse_second(grads, "block_norm_fn has no second derivatives");
    return grads;
  }
};

}  // namespace

/* delta_fwd(q, k, v, log_decay, beta, seq_idx, initial_states, scale or None, return_final, save)
 *   -> (out, final_states or None, saved or None) */
PyObject* delta_fwd(PyObject* const* o) {
  Delta d;
  delta_inputs(o, d);
  const DeltaOut res = delta_forward(d, truth(o[8]), truth(o[9]));
  return tuple_of({res.out, res.fin, res.saved});
}

/* delta_bwd(q, k, v, log_decay, beta, seq_idx, initial_states, scale or None, saved, dout, dfinal_states,
 *           need_dinitial) -> (dq, dk, dv, dlog_decay, dbeta, dinitial_states or None) */
PyObject* delta_bwd(PyObject* const* o) {
  Delta d;
  delta_inputs(o, d);
  const DeltaGrads r = delta_backward(d, tensor(o[8], "saved must be a tensor"),
                                      tensor(o[9], "dout must be a tensor"),
                                      optional(o[10], "dfinal_states must be a tensor or None"), truth(o[11]));
  return tuple_of({r.q, r.k, r.v, r.g, r.beta, r.init});
}

/* delta_train(q, k, v, log_decay, beta, seq_idx, initial_states, scale or None, return_final)
 *   -> (out, final_states or None), recorded by autograd */
PyObject* delta_train(PyObject* const* o) {
  Delta d;
  delta_inputs(o, d);
  const List res = DeltaNode::apply(d.q, d.k, d.v, d.g, d.beta, maybe(d.seq), maybe(d.init), d.scale, truth(o[8]));
  return tuple_of({res[0], res.size() > 1 ? res[1] : at::Tensor()});
}

/* delta_update(q, k, v, log_decay, beta, state, state_indices, scale or None) -> out */
PyObject* delta_update(PyObject* const* o) {
  at::Tensor q = tensor(o[0], "q must be a tensor"), k = tensor(o[1], "k must be a tensor");
  at::Tensor v = tensor(o[2], "v must be a tensor");
  const at::Tensor& g = tensor(o[3], "log_decay must be a tensor");
  const at::Tensor& beta = tensor(o[4], "beta must be a tensor");
  const at::Tensor& state = tensor(o[5], "state must be a tensor");
  at::Tensor idx = optional(o[6], "state_indices must be a tensor or None");
  std::optional<double> scale;
  if (o[7] != Py_None) scale = number(o[7]);
  ccv1d_delta_update_args a{};
  check(k.dim() == 3, "k must be (rows, key_heads, key_dim)");
  check(v.dim() == 3, "v must be (rows, heads, value_dim)");
  check(q.sizes() == k.sizes(), "q must have the shape of k");
  a.rows = k.size(0), a.key_heads = k.size(1), a.key_dim = k.size(2), a.heads = v.size(1), a.value_dim = v.size(2);
  check(v.size(0) == a.rows, "v must have the rows of k");
  check(a.key_heads > 0 && a.heads > 0 && a.heads % a.key_heads == 0,
        "the heads of v must be a multiple of the heads of k");
  check(a.key_dim >= 1 && a.key_dim <= CCV1D_DELTA_MAX_KEY_DIM, "key_dim must be 1 to 256");
  check(a.value_dim >= 1, "value_dim must be at least 1");
  check(shaped(g, {a.rows, a.heads}), "log_decay must be (rows, heads)");
  check(shaped(beta, {a.rows, a.heads}), "beta must be (rows, heads)");
  check(state.dim() == 4 && state.size(1) == a.heads && state.size(2) == a.key_dim && state.size(3) == a.value_dim,
        "state must be (slots, heads, key_dim, value_dim)");
  a.slots = state.size(0);
  check(!idx.defined() || shaped(idx, {a.rows}), "state_indices must be (rows,)");
  check(idx.defined() || a.slots >= a.rows, "state must have a slot for each row");
  check(state.scalar_type() == at::kFloat, "state must be fp32");
  check(a.slots == 0 || state[0].is_contiguous(), "each slot of state must be contiguous");
  check(a.slots <= 1 || state.stride(0) >= a.heads * a.key_dim * a.value_dim, "slots of state must not overlap");
  check(!idx.defined() || at::isIntegralType(idx.scalar_type(), false), "state_indices must hold integers");
  check(k.is_cuda(), "k must be on a GPU");
  const int64_t dev = k.get_device();
  check(q.get_device() == dev && v.get_device() == dev && g.get_device() == dev && beta.get_device() == dev &&
            state.get_device() == dev && (!idx.defined() || idx.get_device() == dev),
        "q, v, log_decay, beta, state and state_indices must be on the device of k");
  a.dtype = dtype_code(k);
  check(q.scalar_type() == k.scalar_type() && v.scalar_type() == k.scalar_type(), "q and v must have the dtype of k");
  a.log_decay_dtype = dtype_code(g), a.beta_dtype = dtype_code(beta);
  no_grad_through({&q, &k, &v, &g, &beta, &state},
                  "gated_delta_update has no backward: call it under torch.no_grad()");
  q = unit_last(q), k = unit_last(k), v = unit_last(v), idx = as_index(idx);
  at::Tensor out = at::empty({a.rows, a.heads, a.value_dim}, k.options());
  a.q = ptr(q), a.q_stride_r = q.stride(0), a.q_stride_h = q.stride(1);
  a.k = ptr(k), a.k_stride_r = k.stride(0), a.k_stride_h = k.stride(1);
  a.v = ptr(v), a.v_stride_r = v.stride(0), a.v_stride_h = v.stride(1);
  a.log_decay = ptr(g), a.log_decay_stride_r = g.stride(0), a.log_decay_stride_h = g.stride(1);
  a.beta = ptr(beta), a.beta_stride_r = beta.stride(0), a.beta_stride_h = beta.stride(1);
  a.scale = scale_of(scale, a.key_dim);
  a.state = ptr<float>(state), a.state_stride = state.stride(0);
  a.state_indices = ptr<int32_t>(idx);
  a.out = ptr(out);
  a.device = (int)dev, a.stream = stream_of(dev);
  call(ccv1d_delta_update, a);
  written(state);
  return tuple_of({out});
}

/* norm_fwd(x, residual, post_weight, gate, scale, pre_weight, eps, activation) -> (r, y or None) */
PyObject* norm_fwd(PyObject* const* o) {
  Norm n;
  norm_inputs(o, n);
  const NormOut res = norm_forward(n);
  return tuple_of({res.r, res.y});
}

/* norm_bwd(x, residual, post_weight, gate, scale, pre_weight, eps, activation, dr or None, dy or None,
 *          need_dresidual) -> (dx, dresidual, dpost_weight, dgate, dscale, dpre_weight), None for absent ones */
PyObject* norm_bwd(PyObject* const* o) {
  Norm n;
  norm_inputs(o, n);
  const NormGrads g = norm_backward(n, optional(o[8], "dr must be a tensor or None"),
                                    optional(o[9], "dy must be a tensor or None"), truth(o[10]));
  return tuple_of({g.x, g.residual, g.post, g.gate, g.scale, g.pre});
}

/* norm_train(x, residual, post_weight, gate, scale, pre_weight, eps, activation) -> (r, y or None), recorded
 * by autograd */
PyObject* norm_train(PyObject* const* o) {
  Norm n;
  norm_inputs(o, n);
  const List res = NormNode::apply(n.x, maybe(n.residual), maybe(n.post), maybe(n.gate), maybe(n.scale), maybe(n.pre),
                                   n.factor, n.eps, (int64_t)n.activation);
  return tuple_of({res[0], res.size() > 1 ? res[1] : at::Tensor()});
}

}  // namespace ccv1d_torch
