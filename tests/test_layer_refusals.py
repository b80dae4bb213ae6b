"""What the operators of a linear-attention layer refuse on a GPU: tensors of other devices and types, calls that
autograd would have to record, wrapper subclasses. Each is refused before anything is launched."""

import pytest
import torch

from causal_conv1d_triton.delta import gated_delta_fn, gated_delta_update
from causal_conv1d_triton.norm import block_norm_fn
from test_ops_refusals import Wrapper

pytestmark = pytest.mark.gpu
F = torch.float32


def z(*s, dtype=torch.bfloat16):
    return torch.zeros(*s, device="cuda", dtype=dtype)


def delta(**kw):
    d = dict(q=z(1, 5, 2, 8), k=z(1, 5, 2, 8), v=z(1, 5, 4, 6), log_decay=z(1, 5, 4, dtype=F), beta=z(1, 5, 4))
    return gated_delta_fn(**{**d, **kw})


@pytest.mark.parametrize("name,shape", [("q", (1, 5, 2, 8)), ("v", (1, 5, 4, 6)), ("log_decay", (1, 5, 4)),
                                        ("beta", (1, 5, 4)), ("seq_idx", (1, 5)), ("initial_states", (1, 4, 8, 6))])
def test_delta_devices(name, shape):
    x = torch.zeros(shape, dtype=torch.int32 if name == "seq_idx" else torch.bfloat16)
    with pytest.raises(AssertionError) as e:
        delta(**{name: x})
    assert "must be on the device of k" in str(e.value)


def test_delta_types():
    with pytest.raises(AssertionError) as e:
        delta(v=z(1, 5, 4, 6, dtype=F))
    assert "must have the dtype of k" in str(e.value)
    for kw in (dict(log_decay=z(1, 5, 4, dtype=torch.float64)), dict(beta=z(1, 5, 4, dtype=torch.int32)),
               dict(q=z(1, 5, 2, 8, dtype=torch.float64), k=z(1, 5, 2, 8, dtype=torch.float64),
                    v=z(1, 5, 4, 6, dtype=torch.float64))):
        with pytest.raises(TypeError) as e:
            delta(**kw)
        assert "unsupported dtype" in str(e.value)


def update(**kw):
    d = dict(q=z(3, 2, 8), k=z(3, 2, 8), v=z(3, 4, 6), log_decay=z(3, 4, dtype=F), beta=z(3, 4),
             state=z(3, 4, 8, 6, dtype=F))
    return gated_delta_update(**{**d, **kw})


@pytest.mark.parametrize("kw,msg", [
    (lambda: dict(state=torch.zeros(3, 4, 8, 6)), "on the device of k"),
    (lambda: dict(state_indices=torch.zeros(3, dtype=torch.int32)), "on the device of k"),
    (lambda: dict(q=z(3, 2, 8, dtype=F)), "the dtype of k"),
    (lambda: dict(q=z(3, 2, 8).requires_grad_()), "no backward"),
    (lambda: dict(beta=z(3, 4).requires_grad_()), "no backward"),
    (lambda: dict(state=z(3, 4, 8, 6, dtype=F).requires_grad_()), "no backward"),
])
def test_update(kw, msg):
    with pytest.raises(AssertionError) as e:
        update(**kw())
    assert msg in str(e.value)


@pytest.mark.parametrize("kw,err,msg", [
    (lambda: dict(residual=torch.zeros(3, 8)), AssertionError, "on the device of x"),
    (lambda: dict(post_weight=torch.zeros(8)), AssertionError, "on the device of x"),
    (lambda: dict(scale=torch.zeros(8)), AssertionError, "on the device of x"),
    (lambda: dict(gate=z(3, 8, dtype=F)), AssertionError, "gate must have the dtype of x"),
    (lambda: dict(residual=z(3, 8, dtype=torch.float16)), AssertionError, "the dtype of x or be fp32"),
    (lambda: dict(post_weight=z(8, dtype=torch.float64)), TypeError, "unsupported dtype"),
    (lambda: dict(residual=z(3, 8, dtype=torch.int32)), TypeError, "unsupported dtype"),
])
def test_norm(kw, err, msg):
    with pytest.raises(err) as e:
        block_norm_fn(**{**dict(x=z(3, 8), post_weight=z(8)), **kw()})
    assert msg in str(e.value)


@pytest.mark.parametrize("call", [
    lambda: delta(beta=Wrapper(z(1, 5, 4))),
    lambda: delta(seq_idx=Wrapper(z(1, 5, dtype=torch.int32))),
    lambda: delta(initial_states=Wrapper(z(1, 4, 8, 6, dtype=F))),
    lambda: delta(q=z(1, 5, 2, 8).requires_grad_(), initial_states=Wrapper(z(1, 4, 8, 6, dtype=F))),
    lambda: update(state_indices=Wrapper(z(3, dtype=torch.int32))),
    lambda: block_norm_fn(z(3, 8), Wrapper(z(3, 8)), z(8)),
    lambda: block_norm_fn(z(3, 8), None, z(8), pre_weight=Wrapper(z(8))),
    lambda: block_norm_fn(z(3, 8).requires_grad_(), None, z(8), scale=Wrapper(z(8))),
])
def test_wrappers(call):
    with pytest.raises(TypeError) as e:
        call()
    assert "memory of its own" in str(e.value)


def test_backward_gradients_of_another_shape():
    """The library reads as many elements of the incoming gradients as the outputs have."""
    from causal_conv1d_triton._ops import native
    k, v, g = z(1, 70, 2, 8), z(1, 70, 2, 8), z(1, 70, 2, dtype=F)
    args = (k, k, v, g, g, None, None, None)
    out, _, saved = native().delta_fwd(*args, False, True)
    for dout, sv, dfin, msg in ((out[:, :69], saved, None, "gradient of out must have the shape"),
                                (out.float(), saved, None, "must have the dtype of k"),
                                (out.cpu(), saved, None, "gradient of out must be on"),
                                (out, saved, z(1, 2, 8, 7, dtype=F), "gradient of final_states must be (batch"),
                                (out, saved[1:], None, "saved must be what the forward kept")):
        with pytest.raises(AssertionError) as e:
            native().delta_bwd(*args, sv, dout, dfin, False)
        assert msg in str(e.value)
    x, w = z(4, 8), z(8)
    args = (x, x, w, None, None, w, 1e-6, 1)
    for dr, dy, msg in ((x[:3], None, "gradient of r must have the shape"), (x.float(), None, "r's dtype"),
                        (None, x.float(), "dtype of x"), (None, x[:, :7], "gradient of y must have the shape"),
                        (x.cpu(), None, "on the device")):
        with pytest.raises(AssertionError) as e:
            native().norm_bwd(*args, dr, dy, True)
        assert msg in str(e.value)


def test_out_of_memory_keeps_its_type():
    x = z(1, 64).expand(1 << 26, 64)
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    try:
        torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (1 << 30)) / total)
        with pytest.raises(torch.OutOfMemoryError):
            block_norm_fn(x, None, z(64))
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert block_norm_fn(x[:100], None, z(64)).shape == (100, 64)
