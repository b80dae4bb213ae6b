"""Gated delta rule over channels-last heads, the linear attention that the causal convolution's queries, keys and
values go into, with forward and backward. Per head, in fp32 whatever the inputs' type, with a state S of
(key_dim, value_dim):

    S'   = exp(log_decay[t]) * S[t - 1]
    u[t] = beta[t] * (v[t] - S'^T k[t])
    S[t] = S' + k[t] u[t]^T
    o[t] = scale * S[t]^T q[t]

`gated_delta_fn` runs whole sequences, training included; `gated_delta_update` one token of each request of a
serving batch, the states in a pool. Packing (`seq_idx`) and states follow causal_conv1d_fn and
gated_recurrence_fn. Queries and keys are taken as they are: a model of this kind gives them unit length
(block_norm_fn with a constant weight does that), and keys much longer than that make the recurrence grow.
The kernels are hand-written HIP kernels of libccv1d.so (include/ccv1d_layer.h). The reference package has no such
operator.
"""

import torch
from torch import Tensor

from ._ops import native


# The two passes as torch.library operators, for torch.compile, and the forward without what the backward needs. Absent
# outputs are empty tensors.


@torch.library.custom_op("causal_conv1d_amd::gated_delta", mutates_args=(), device_types="cuda")
def _fwd_op(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, beta: Tensor, seq_idx: Tensor | None,
            initial_states: Tensor | None, scale: float) -> tuple[Tensor, Tensor, Tensor]:
    return native().delta_fwd(q, k, v, log_decay, beta, seq_idx, initial_states, scale, True, True)


@_fwd_op.register_fake
def _fwd_fake(q, k, v, log_decay, beta, seq_idx, initial_states, scale):
    B, T, H, Dv = v.shape
    Dk, N = k.shape[3], (T + 63) // 64
    dk, dvp = (64 if Dk <= 64 else 128 if Dk <= 128 else 256), (Dv + 31) // 32 * 32
    return (v.new_empty(B, T, H, Dv), v.new_empty(B, H, Dk, Dv, dtype=torch.float32),
            v.new_empty(B * H * N * (dk + 64) * dvp, dtype=torch.float32))


@torch.library.custom_op("causal_conv1d_amd::gated_delta_bwd", mutates_args=(), device_types="cuda")
def _bwd_op(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, beta: Tensor, seq_idx: Tensor | None,
            initial_states: Tensor | None, scale: float, saved: Tensor, dout: Tensor,
            dfinal_states: Tensor | None,
            need_dinitial: bool) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    res = native().delta_bwd(q, k, v, log_decay, beta, seq_idx, initial_states, scale, saved, dout,
                             dfinal_states, need_dinitial)
    return tuple(q.new_empty(0) if t is None else t for t in res)


@_bwd_op.register_fake
def _bwd_fake(q, k, v, log_decay, beta, seq_idx, initial_states, scale, saved, dout, dfinal_states,
              need_dinitial):
    return (q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape),
            log_decay.new_empty(log_decay.shape), beta.new_empty(beta.shape),
            initial_states.new_empty(initial_states.shape) if need_dinitial else q.new_empty(0))


def _op_setup(ctx, inputs, output):
    *tensors, ctx.scale = inputs
    ctx.save_for_backward(*tensors, output[2])


def _op_backward(ctx, dout, dfinal, _):
    q, k, v, log_decay, beta, seq_idx, init, saved = ctx.saved_tensors
    need = init is not None and ctx.needs_input_grad[6]
    if dout is None:
        dout = torch.zeros_like(v)
    dq, dk, dv, dg, dbeta, dinit = _bwd_op(q, k, v, log_decay, beta, seq_idx, init, ctx.scale, saved, dout,
                                           dfinal, need)
    return dq, dk, dv, dg, dbeta, None, dinit if need else None, None


_fwd_op.register_autograd(_op_backward, setup_context=_op_setup)


@torch.library.custom_op("causal_conv1d_amd::gated_delta_infer", mutates_args=(), device_types="cuda")
def _infer_op(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, beta: Tensor, seq_idx: Tensor | None,
              initial_states: Tensor | None, scale: float, final_states: bool) -> tuple[Tensor, Tensor]:
    out, fin, _ = native().delta_fwd(q, k, v, log_decay, beta, seq_idx, initial_states, scale, final_states, False)
    return out, v.new_empty(0) if fin is None else fin


@_infer_op.register_fake
def _infer_fake(q, k, v, log_decay, beta, seq_idx, initial_states, scale, final_states):
    B, T, H, Dv = v.shape
    return (v.new_empty(B, T, H, Dv),
            v.new_empty(B, H, k.shape[3], Dv, dtype=torch.float32) if final_states else v.new_empty(0))


def gated_delta_fn(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    log_decay: Tensor,
    beta: Tensor,
    seq_idx: Tensor | None = None,
    initial_states: Tensor | None = None,
    return_final_states: bool = False,
    scale: float | None = None,
) -> Tensor | tuple[Tensor, Tensor]:
    """The gated delta rule along time, with autograd (the module's docstring has the recurrence).

    Arguments:
      q, k: (batch, seqlen, key_heads, key_dim), v: (batch, seqlen, heads, value_dim) on a GPU, bf16, fp16 or
         fp32, one type for all, unit last stride (other strides are free, so slices of one projection go in as
         they are; a tensor without a unit stride is copied first). heads is a multiple of key_heads: head h has
         the queries and keys of key head h // (heads // key_heads). key_dim is 1 to 256.
      log_decay, beta: (batch, seqlen, heads), each fp32, fp16 or bf16, any strides. A log-decay below -104, whose
         exponential is zero in fp32, empties the state.
      seq_idx: optional (batch, seqlen) integer ids marking packed sequences: the state starts at zero in each
         row whose id differs from the row before; rows with a negative id are padding, whose outputs and
         gradients are zero whatever the inputs hold there. initial_states belong to the sequence of seq_idx[:, 0].
         An infinity or NaN in a row that is no padding, or a log-decay above 88.7, whose exponential is infinite in
         fp32, on a state, spoils that sequence from there on (and its gradients), no other; only finite keys so long,
         or log-decays of several rows so far above zero, that the products of 64 rows overflow fp32 can.
      initial_states: optional (batch, heads, key_dim, value_dim), any float type, the state in front of row 0.
      return_final_states: also return the state behind the last row (zero where that is padding, so prompts of
         unequal length take a call each), of the shape of initial_states in fp32, which is the initial_states of a
         following chunk; gradients flow through it.
      scale: of the outputs, key_dim ** -0.5 without.

    Returns `out` (batch, seqlen, heads, value_dim), rounded once to v's dtype, or `(out, final_states)`.
    Gradients: q, k, v, log_decay, beta and initial_states. Results are deterministic. Training keeps, beside the
    inputs, ceil(seqlen / 64) * (K + 64) * V fp32 numbers of each batch and head until the backward, K being key_dim
    raised to 64, 128 or 256 and V value_dim to a multiple of 32; the backward takes as many again while it runs.
    """
    train = torch.is_grad_enabled() and any(
        getattr(t, "requires_grad", False) for t in (q, k, v, log_decay, beta, initial_states))
    if torch.compiler.is_compiling():
        if scale is None:
            scale = k.shape[-1] ** -0.5
        if train:
            out, final, _ = _fwd_op(q, k, v, log_decay, beta, seq_idx, initial_states, scale)
        else:
            out, final = _infer_op(q, k, v, log_decay, beta, seq_idx, initial_states, scale, return_final_states)
    elif train:
        out, final = native().delta_train(q, k, v, log_decay, beta, seq_idx, initial_states, scale,
                                          return_final_states)
    else:
        out, final, _ = native().delta_fwd(q, k, v, log_decay, beta, seq_idx, initial_states, scale,
                                           return_final_states, False)
    return (out, final) if return_final_states else out


def gated_delta_update(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    log_decay: Tensor,
    beta: Tensor,
    state: Tensor,
    state_indices: Tensor | None = None,
    scale: float | None = None,
) -> Tensor:
    """One token of each request: the state of row r's slot takes a step of the gated delta rule, in place, and is
    read along q. No backward.

    Arguments:
      q, k: (rows, key_heads, key_dim), v: (rows, heads, value_dim), log_decay, beta: (rows, heads), as in
         gated_delta_fn.
      state: (slots, heads, key_dim, value_dim) fp32, a pool of states, each slot contiguous, updated in place.
      state_indices: optional (rows,) integers, the slot of each row (row r uses slot r without). Rows whose
         index lies outside the pool, -1 above all, are left out: their output is zero. Two rows of one slot
         race: what they leave there and return is not defined.

    Returns out (rows, heads, value_dim).
    """
    return native().delta_update(q, k, v, log_decay, beta, state, state_indices, scale)[0]
