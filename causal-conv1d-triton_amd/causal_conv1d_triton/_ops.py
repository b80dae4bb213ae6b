"""Binding of the operators around the convolution (include/ccv1d_ops.h): the CPython extension
`_ccv1d_ops` (csrc/ops/ccv1d_ops_torch.cpp), which checks arguments, allocates and calls libccv1d.so.
There is no other compute path: without the extension every call raises."""

from ._ffi import CCV1DError

try:
    from . import _ccv1d_ops as _native
except ImportError:
    _native = None
else:
    _native.set_error_type(CCV1DError)


def native():
    if _native is None:
        raise RuntimeError("the extension _ccv1d_ops is not built; run "
                           "`make -C causal-conv1d-triton_amd` (or __graft_entry__.build()) first")
    return _native
