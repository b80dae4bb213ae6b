"""Norms before and after a block, fused with the block's gate, the scale of its output and the residual stream, with
forward and backward: what stands around the convolution, the gated recurrence, the gated delta rule and
attention in a model. The kernels are hand-written HIP kernels of libccv1d.so (include/ccv1d_layer.h). The reference
package has no such operator.
"""

import torch
from torch import Tensor

from ._ops import native

_ACTIVATIONS = {None: 0, "silu": 1, "sigmoid": 2}


# The two passes as torch.library operators, for torch.compile. Absent outputs are empty tensors.


@torch.library.custom_op("causal_conv1d_amd::block_norm", mutates_args=(), device_types="cuda")
def _fwd_op(x: Tensor, residual: Tensor | None, post_weight: Tensor | None, gate: Tensor | None,
            scale: Tensor | None, factor: float, pre_weight: Tensor | None, eps: float,
            activation: int) -> tuple[Tensor, Tensor]:
    r, y = native().norm_fwd(x, residual, post_weight, gate, factor if scale is None else scale, pre_weight,
                             eps, activation)
    return r, x.new_empty(0) if y is None else y


@_fwd_op.register_fake
def _fwd_fake(x, residual, post_weight, gate, scale, factor, pre_weight, eps, activation):
    return ((x if residual is None else residual).new_empty(x.shape),
            x.new_empty(0 if pre_weight is None else x.shape))


@torch.library.custom_op("causal_conv1d_amd::block_norm_bwd", mutates_args=(), device_types="cuda")
def _bwd_op(x: Tensor, residual: Tensor | None, post_weight: Tensor | None, gate: Tensor | None,
            scale: Tensor | None, factor: float, pre_weight: Tensor | None, eps: float, activation: int,
            dr: Tensor | None, dy: Tensor | None,
            need_dresidual: bool) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    res = native().norm_bwd(x, residual, post_weight, gate, factor if scale is None else scale, pre_weight, eps,
                            activation, dr, dy, need_dresidual)
    return tuple(x.new_empty(0) if t is None else t for t in res)


@_bwd_op.register_fake
def _bwd_fake(x, residual, post_weight, gate, scale, factor, pre_weight, eps, activation, dr, dy,
              need_dresidual):
    return tuple(x.new_empty(0) if t is None else t.new_empty(t.shape) for t in (
        x, residual if need_dresidual else None, post_weight, gate, scale, pre_weight))


def _op_setup(ctx, inputs, output):
    *tensors, ctx.factor, pre_weight, ctx.eps, ctx.activation = inputs
    ctx.save_for_backward(*tensors, pre_weight)


def _op_backward(ctx, dr, dy):
    x, residual, post, gate, scale, pre = ctx.saved_tensors
    need = residual is not None and ctx.needs_input_grad[1]
    grads = _bwd_op(x, residual, post, gate, scale, ctx.factor, pre, ctx.eps, ctx.activation, dr,
                    None if pre is None else dy, need)
    dx, dres, dpost, dgate, dscale, dpre = (
        None if t is None else g
        for g, t in zip(grads, (x, residual if need else None, post, gate, scale, pre)))
    return dx, dres, dpost, dgate, dscale, None, dpre, None, None


_fwd_op.register_autograd(_op_backward, setup_context=_op_setup)


def block_norm_fn(
    x: Tensor,
    residual: Tensor | None = None,
    post_weight: Tensor | None = None,
    gate: Tensor | None = None,
    scale: Tensor | float | None = None,
    pre_weight: Tensor | None = None,
    eps: float = 1e-6,
    activation: str | None = "silu",
) -> Tensor | tuple[Tensor, Tensor]:
    """What stands between a block's output x and the next block's input, with autograd; each part is left out where
    its argument is None:

        m = x * post_weight / sqrt(mean(x^2) + eps)      the norm after the block
        m = m * act(gate)                                its gate
        r = residual + scale * m                         back to the residual stream
        y = r * pre_weight / sqrt(mean(r^2) + eps)       the norm before the next block

    over the last dimension, in fp32 whatever the types, every result rounded once (y from the unrounded r). So a row whose
    squares add up to more than fp32 holds, with elements beyond 1e17 or so, comes out of a norm as zero.

    Arguments:
      x: (..., dim) on a GPU, bf16, fp16 or fp32, dim at most 8192. Unit last stride and rows that two
         strides describe (slices of a projection, heads beside each other, rows that are expanded); others are
         copied first. So gate, residual and the incoming gradients.
      residual: optional, of x's shape, of x's dtype or fp32.
      post_weight, pre_weight: optional (dim,), fp32, fp16 or bf16; one of the two at least.
      gate: optional, of x's shape and dtype, before its activation.
      scale: optional number, or tensor (dim,) of fp32, fp16 or bf16.
      activation: of the gate, "silu", "sigmoid" or None.

    Returns r, of residual's dtype (x's without one), or with pre_weight `(y, r)`, y of x's dtype. Gradients: x,
    residual, gate and the weights (scale where it is a tensor). Results are deterministic.
    """
    if activation not in _ACTIVATIONS:
        raise NotImplementedError("activation must be None, 'silu' or 'sigmoid'")
    act = _ACTIVATIONS[activation]
    if torch.compiler.is_compiling():
        tensor = isinstance(scale, Tensor)
        r, y = _fwd_op(x, residual, post_weight, gate, scale if tensor else None,
                       1.0 if tensor or scale is None else float(scale), pre_weight, eps, act)
    elif torch.is_grad_enabled() and any(
            getattr(t, "requires_grad", False)
            for t in (x, residual, post_weight, gate, scale, pre_weight)):
        r, y = native().norm_train(x, residual, post_weight, gate, scale, pre_weight, eps, act)
    else:
        r, y = native().norm_fwd(x, residual, post_weight, gate, scale, pre_weight, eps, act)
    return r if pre_weight is None else (y, r)
