"""Gated linear recurrence over channels-last inputs, the operator that follows the causal convolution
in a recurrent block, with forward and backward. Per channel d, in fp32 whatever the inputs' type:

    r = sigmoid(gate), i = sigmoid(input_gate)            (i = 1 without an input gate)
    a = exp(-decay_scale * softplus(decay[d]) * r),  beta = sqrt(1 - a^2)     with a decay
    a = r,                                           beta = 1 - r             without
    h[t] = a[t] * h[t - 1] + beta[t] * i[t] * x[t]

A sequence's first row has the beta of any other (some models of this family take 1 there).
`gated_recurrence_fn` runs whole sequences, training included; `gated_recurrence_update` one token of
each request of a serving batch, the states in a pool. Layout, packing (`seq_idx`) and states follow
causal_conv1d_fn, so that one block hands the same tensors to both. The kernels are hand-written HIP
kernels of libccv1d.so (include/ccv1d_ops.h). The reference package has no such operator.
"""

import torch
from torch import Tensor

from ._ops import native


# The two passes as torch.library operators, for torch.compile. Absent outputs are empty tensors.


@torch.library.custom_op("causal_conv1d_amd::gated_recurrence", mutates_args=(), device_types="cuda")
def _fwd_op(x: Tensor, gate: Tensor, decay: Tensor | None, input_gate: Tensor | None,
            seq_idx: Tensor | None, initial_states: Tensor | None,
            decay_scale: float) -> tuple[Tensor, Tensor, Tensor]:
    return native().rec_fwd(x, gate, decay, input_gate, seq_idx, initial_states, decay_scale, True,
                            True)


@_fwd_op.register_fake
def _fwd_fake(x, gate, decay, input_gate, seq_idx, initial_states, decay_scale):
    B, T, D = x.shape
    return (x.new_empty(B, T, D), x.new_empty(B, D, dtype=torch.float32),
            x.new_empty(B, (T + 63) // 64, D, dtype=torch.float32))


@torch.library.custom_op("causal_conv1d_amd::gated_recurrence_bwd", mutates_args=(),
                         device_types="cuda")
def _bwd_op(x: Tensor, gate: Tensor, decay: Tensor | None, input_gate: Tensor | None,
            seq_idx: Tensor | None, initial_states: Tensor | None, decay_scale: float,
            saved: Tensor, dout: Tensor, dfinal_states: Tensor | None,
            need_dinitial: bool) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    res = native().rec_bwd(x, gate, decay, input_gate, seq_idx, initial_states, decay_scale, saved,
                           dout, dfinal_states, need_dinitial)
    return tuple(x.new_empty(0) if t is None else t for t in res)


@_bwd_op.register_fake
def _bwd_fake(x, gate, decay, input_gate, seq_idx, initial_states, decay_scale, saved, dout,
              dfinal_states, need_dinitial):
    none = x.new_empty(0)
    return (x.new_empty(x.shape), x.new_empty(x.shape),
            none if decay is None else decay.new_empty(decay.shape),
            none if input_gate is None else x.new_empty(x.shape),
            initial_states.new_empty(initial_states.shape) if need_dinitial else none)


def _op_setup(ctx, inputs, output):
    *tensors, ctx.decay_scale = inputs
    ctx.save_for_backward(*tensors, output[2])


def _op_backward(ctx, dout, dfinal, _):
    x, gate, decay, input_gate, seq_idx, init, saved = ctx.saved_tensors
    need = init is not None and ctx.needs_input_grad[5]
    if dout is None:
        dout = torch.zeros_like(x)
    dx, dgate, ddecay, dig, dinit = _bwd_op(x, gate, decay, input_gate, seq_idx, init,
                                            ctx.decay_scale, saved, dout, dfinal, need)
    return (dx, dgate, None if decay is None else ddecay, None if input_gate is None else dig, None,
            dinit if need else None, None)


_fwd_op.register_autograd(_op_backward, setup_context=_op_setup)


def gated_recurrence_fn(
    x: Tensor,
    gate: Tensor,
    decay: Tensor | None = None,
    input_gate: Tensor | None = None,
    seq_idx: Tensor | None = None,
    initial_states: Tensor | None = None,
    return_final_states: bool = False,
    decay_scale: float = 8.0,
) -> Tensor | tuple[Tensor, Tensor]:
    """h[t] = a[t] * h[t - 1] + beta[t] * i[t] * x[t] along time, with autograd (the module's
    docstring has a, beta and i).

    Arguments:
      x, gate, input_gate: (batch, seqlen, dim) on a GPU, bf16, fp16 or fp32, one type for all, unit
         stride along dim (other strides are free, so slices of one projection go in as they are; a
         tensor without a unit stride is copied first). gate and input_gate are pre-activations.
      decay: optional (dim,), any float type; its gradient comes back in that type.
      seq_idx: optional (batch, seqlen) integer ids below 2^63 (causal_conv1d_fn tells its ids apart by
         their low 32 bits) marking packed sequences: the state starts at zero
         in each row whose id differs from the row before; rows with a negative id are padding, whose
         outputs and gradients are zero whatever x and the gates hold there. initial_states belong to
         the sequence of seq_idx[:, 0].
      initial_states: optional (batch, dim), any float type, the state in front of x[:, 0].
      return_final_states: also return the state of the last row, (batch, dim) in fp32, which is the
         initial_states of a following chunk; gradients flow through it.
      decay_scale: the factor in the decay's exponent.

    Returns `out` (batch, seqlen, dim), h rounded once to x's dtype, or `(out, final_states)`.
    Gradients: x, gate, decay, input_gate and initial_states. Results are deterministic.
    """
    if torch.compiler.is_compiling():
        out, final, _ = _fwd_op(x, gate, decay, input_gate, seq_idx, initial_states, decay_scale)
    elif torch.is_grad_enabled() and any(
            getattr(t, "requires_grad", False)
            for t in (x, gate, decay, input_gate, initial_states)):
        out, final = native().rec_train(x, gate, decay, input_gate, seq_idx, initial_states,
                                        decay_scale, return_final_states)
    else:
        out, final, _ = native().rec_fwd(x, gate, decay, input_gate, seq_idx, initial_states,
                                         decay_scale, return_final_states, False)
    return (out, final) if return_final_states else out


def gated_recurrence_update(
    x: Tensor,
    gate: Tensor,
    state: Tensor,
    decay: Tensor | None = None,
    input_gate: Tensor | None = None,
    state_indices: Tensor | None = None,
    decay_scale: float = 8.0,
) -> Tensor:
    """One token of each request: the state of row r's slot becomes a * state + beta * i * x[r], in
    place, and is returned rounded to x's dtype. No backward.

    Arguments:
      x, gate, input_gate: (rows, dim), as in gated_recurrence_fn.
      state: (slots, dim) fp32 with a unit channel stride, a pool of states, updated in place.
      state_indices: optional (rows,) integers, the slot of each row (row r uses slot r without). Rows
         whose index lies outside the pool, -1 above all, are left out: their output is zero. Two rows
         of one slot race: what they leave there and return is not defined.

    Returns out (rows, dim).
    """
    return native().rec_update(x, gate, state, decay, input_gate, state_indices, decay_scale)[0]
