"""Norms around a block over no rows beside a residual stream of another type, whose pointer is then null."""

import ctypes as C

import pytest
import torch

from test_layer_abi import BF16, F32, Norm, lib  # noqa: F401  (fixture)


@pytest.mark.parametrize("outer,inner", [(0, 4), (4, 0), (0, 0)])
def test_no_rows_in_c(lib, outer, inner):  # noqa: F811
    a = Norm(dtype=BF16, residual_dtype=F32, post_weight=4096, pre_weight=4096, dim=8, outer=outer, inner=inner, scale=1.0)
    assert lib.ccv1d_norm_fwd(C.byref(a)) == 0, lib.ccv1d_last_error()
    assert lib.ccv1d_norm_workspace_bytes(C.byref(a)) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 30), (2, 0, 30), (0, 3, 30)])
def test_no_rows(shape):
    from causal_conv1d_triton.norm import block_norm_fn
    x, gate = (torch.zeros(shape, device="cuda", dtype=torch.bfloat16, requires_grad=True) for _ in range(2))
    residual = torch.zeros(shape, device="cuda", requires_grad=True)
    post, scale, pre = (torch.ones(30, device="cuda", requires_grad=True) for _ in range(3))
    y, r = block_norm_fn(x, residual, post, gate, scale, pre)
    assert y.shape == r.shape == shape and (y.dtype, r.dtype) == (torch.bfloat16, torch.float32)
    leaves = (x, residual, post, gate, scale, pre)
    for t, g in zip(leaves, torch.autograd.grad([y, r], leaves, [torch.ones_like(y), torch.ones_like(r)])):
        assert g.shape == t.shape and g.dtype == t.dtype and not g.any()
    with torch.no_grad():
        assert block_norm_fn(x, residual, post).shape == shape
