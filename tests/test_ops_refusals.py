"""What the operators around the convolution refuse on a GPU: tensors of other devices and types, and
calls that autograd would have to record. Each is refused before anything is launched."""

import pytest
import torch

from causal_conv1d_triton.paged import paged_attention, paged_cache_write, paged_plan
from causal_conv1d_triton.recurrence import gated_recurrence_fn, gated_recurrence_update

pytestmark = pytest.mark.gpu


def z(*s, dtype=torch.bfloat16):
    return torch.zeros(*s, device="cuda", dtype=dtype)


def i32(*s):
    return z(*s, dtype=torch.int32)


F = torch.float32


@pytest.mark.parametrize("make,err,msg", [
    (lambda: (z(1, 2, 3), torch.zeros(1, 2, 3)), AssertionError, "gate must be on the device of x"),
    (lambda: (z(1, 2, 3), z(1, 2, 3), torch.zeros(3)), AssertionError, "decay must be on the device"),
    (lambda: (z(1, 2, 3), z(1, 2, 3), None, torch.zeros(1, 2, 3)), AssertionError, "input_gate must be on"),
    (lambda: (z(1, 2, 3), z(1, 2, 3), None, None, torch.zeros(1, 2, dtype=torch.int32)), AssertionError,
     "seq_idx must be on the device"),
    (lambda: (z(1, 2, 3), z(1, 2, 3), None, None, None, torch.zeros(1, 3)), AssertionError,
     "initial_states must be on the device"),
    (lambda: (z(1, 2, 3), z(1, 2, 3, dtype=F)), AssertionError, "must have the dtype of x"),
    (lambda: (z(1, 2, 3), z(1, 2, 3), None, z(1, 2, 3, dtype=F)), AssertionError, "must have the dtype"),
    (lambda: (z(1, 2, 3, dtype=torch.float64),) * 2, TypeError, "unsupported dtype"),
    (lambda: (i32(1, 2, 3),) * 2, TypeError, "unsupported dtype"),
])
def test_recurrence(make, err, msg):
    with pytest.raises(err) as e:
        gated_recurrence_fn(*make())
    assert msg in str(e.value)


@pytest.mark.parametrize("make,err,msg", [
    (lambda: (z(2, 3), z(2, 3), torch.zeros(2, 3)), AssertionError, "state must be on the device of x"),
    (lambda: (z(2, 3), z(2, 3), z(2, 3, dtype=F), None, None, torch.zeros(2, dtype=torch.int32)),
     AssertionError, "state_indices must be on the device"),
    (lambda: (z(2, 3), z(2, 3, dtype=F), z(2, 3, dtype=F)), AssertionError, "must have the dtype of x"),
    (lambda: (z(2, 3).requires_grad_(), z(2, 3), z(2, 3, dtype=F)), AssertionError, "no backward"),
    (lambda: (z(2, 3), z(2, 3), z(2, 3, dtype=F).requires_grad_()), AssertionError, "no backward"),
])
def test_update(make, err, msg):
    with pytest.raises(err) as e:
        gated_recurrence_update(*make())
    assert msg in str(e.value)


@pytest.mark.parametrize("make,msg", [
    (lambda: (i32(2), torch.zeros(2, dtype=torch.int32), i32(2, 4), i32(9), i32(1), 16, 4), "new_lens must be"),
    (lambda: (i32(2), i32(3), i32(2, 4), i32(9), i32(1), 16, 4), "new_lens must be (requests,)"),
    (lambda: (i32(2).long(), i32(2), i32(2, 4), i32(9), i32(1), 16, 4), "cached_lens must be contiguous"),
    (lambda: (i32(2), i32(4)[::2], i32(2, 4), i32(9), i32(1), 16, 4), "new_lens must be contiguous"),
    (lambda: (i32(2), i32(2), i32(3, 4), i32(9), i32(1), 16, 4), "block_tables must be (requests"),
    (lambda: (i32(2), i32(2), i32(2, 8)[:, ::2], i32(9), i32(1), 16, 4), "rows of block_tables must be"),
    (lambda: (i32(2), i32(2), i32(1, 4).expand(2, 4), i32(9), i32(1), 16, 4), "must not overlap"),
    (lambda: (i32(2), i32(2), i32(2, 4).long(), i32(9), i32(1), 16, 4), "block_tables must be int32"),
    (lambda: (i32(2), i32(2), i32(2, 4), i32(3, 3), i32(1), 16, 4), "free_pages must be"),
    (lambda: (i32(2), i32(2), i32(2, 4), i32(9), i32(2), 16, 4), "num_free must be (1,)"),
])
def test_plan(make, msg):
    with pytest.raises(AssertionError) as e:
        paged_plan(*make())
    assert msg in str(e.value)


@pytest.mark.parametrize("make,msg", [
    (lambda: (z(5, 2, 8), z(5, 2, 8), z(3, 4, 2, 8), torch.zeros(3, 4, 2, 8), i32(5)), "on the device of k"),
    (lambda: (z(5, 2, 8), z(5, 2, 8), z(3, 4, 2, 8), z(3, 4, 2, 8), torch.zeros(5, dtype=torch.int32)),
     "on the device of k"),
    (lambda: (z(5, 2, 8), z(5, 2, 8, dtype=F), z(3, 4, 2, 8), z(3, 4, 2, 8), i32(5)), "the dtype of k"),
    (lambda: (z(5, 2, 8), z(5, 2, 8), z(3, 4, 2, 8), z(3, 4, 2, 8, dtype=F), i32(5)), "the dtype of k"),
    (lambda: (z(5, 2, 8).requires_grad_(), z(5, 2, 8), z(3, 4, 2, 8), z(3, 4, 2, 8), i32(5)), "no backward"),
])
def test_write(make, msg):
    with pytest.raises(AssertionError) as e:
        paged_cache_write(*make())
    assert msg in str(e.value)


@pytest.mark.parametrize("make,msg", [
    (lambda: (z(2, 4, 8), torch.zeros(3, 4, 2, 8), z(3, 4, 2, 8), i32(2, 3), i32(2)), "on the device of q"),
    (lambda: (z(2, 4, 8), z(3, 4, 2, 8), z(3, 4, 2, 8), torch.zeros(2, 3, dtype=torch.int32), i32(2)),
     "on the device of q"),
    (lambda: (z(2, 4, 8), z(3, 4, 2, 8), z(3, 4, 2, 8), i32(2, 3), torch.zeros(2, dtype=torch.int32)),
     "on the device of q"),
    (lambda: (z(2, 4, 8), z(3, 4, 2, 8, dtype=F), z(3, 4, 2, 8, dtype=F), i32(2, 3), i32(2)),
     "the dtype of q"),
    (lambda: (z(2, 4, 8).requires_grad_(), z(3, 4, 2, 8), z(3, 4, 2, 8), i32(2, 3), i32(2)), "no backward"),
])
def test_attention(make, msg):
    with pytest.raises(AssertionError) as e:
        paged_attention(*make())
    assert msg in str(e.value)


@pytest.mark.parametrize("train", [False, True])
def test_out_of_memory_keeps_its_type(train):
    """Serving loops catch torch.OutOfMemoryError. The process's share of the card is made small: the output,
    of a row that the input's strides repeat, does not fit it."""
    x = z(1, 1, 64).requires_grad_(train).expand(1, 1 << 26, 64)
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    try:
        torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (1 << 30)) / total)
        with pytest.raises(torch.OutOfMemoryError):
            gated_recurrence_fn(x, x)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert gated_recurrence_fn(x[:, :100], x[:, :100]).shape == (1, 100, 64)


class Wrapper(torch.Tensor):
    """A subclass that holds another tensor and has no memory of its own."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, strides=inner.stride(), dtype=inner.dtype,
                                                   device=inner.device)

    def __init__(self, inner):
        self.inner = inner

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        plain = torch.utils._pytree.tree_map(lambda t: t.inner if isinstance(t, cls) else t, (args, kwargs or {}))
        return torch.utils._pytree.tree_map(lambda t: cls(t) if isinstance(t, torch.Tensor) else t,
                                            func(*plain[0], **plain[1]))


@pytest.mark.parametrize("call", [
    lambda: gated_recurrence_fn(z(1, 2, 3), z(1, 2, 3), Wrapper(z(3, dtype=F))),
    lambda: gated_recurrence_fn(z(1, 2, 3), z(1, 2, 3), None, Wrapper(z(1, 2, 3))),
    lambda: gated_recurrence_fn(z(1, 2, 3), z(1, 2, 3), None, None, Wrapper(i32(1, 2))),
    lambda: gated_recurrence_fn(z(1, 2, 3), z(1, 2, 3), None, None, None, Wrapper(z(1, 3, dtype=F))),
    lambda: gated_recurrence_fn(z(1, 2, 3).requires_grad_(), z(1, 2, 3), None, None, Wrapper(i32(1, 2))),
    lambda: gated_recurrence_update(z(2, 3), z(2, 3), z(2, 3, dtype=F), None, None, Wrapper(i32(2))),
    lambda: gated_recurrence_update(z(2, 3), z(2, 3), z(2, 3, dtype=F), Wrapper(z(3, dtype=F))),
    lambda: paged_attention(z(2, 4, 8), z(3, 4, 2, 8), z(3, 4, 2, 8), i32(2, 3), i32(2),
                            request_ids=Wrapper(i32(2))),
    lambda: paged_attention(Wrapper(z(2, 4, 8)), z(3, 4, 2, 8), z(3, 4, 2, 8), i32(2, 3), i32(2)),
    lambda: paged_plan(Wrapper(i32(2)), i32(2), i32(2, 4), i32(9), i32(1), 16, 4),
    lambda: paged_cache_write(z(5, 2, 8), z(5, 2, 8), Wrapper(z(3, 4, 2, 8)), z(3, 4, 2, 8), i32(5)),
])
def test_wrappers(call):
    """Taken for their null address, an optional one would count as absent."""
    with pytest.raises(TypeError) as e:
        call()
    assert "memory of its own" in str(e.value)


def test_backward_gradients_of_another_shape():
    """The library reads as many elements of the incoming gradients as x has."""
    from causal_conv1d_triton._ops import native
    x, saved = z(2, 70, 8), z(2, 2, 8, dtype=F)
    args = (x, x, None, None, None, None, 8.0)
    for dout, sv, dfin, msg in ((z(2, 69, 8), saved, None, "gradient of out must have the shape"),
                                (z(2, 70, 8, dtype=F), saved, None, "must have the dtype of x"),
                                (torch.zeros(2, 70, 8), saved, None, "gradient of out must be on"),
                                (x, saved, z(2, 7, dtype=F), "gradient of final_states must be (batch"),
                                (x, saved[:, :1], None, "saved must be what the forward kept")):
        with pytest.raises(AssertionError) as e:
            native().rec_bwd(*args, sv, dout, dfin, False)
        assert msg in str(e.value)
