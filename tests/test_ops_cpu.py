"""The operators around the convolution without a GPU: import surface, the refusals of the public
functions that need no GPU tensor, the operators' fake implementations, and the 64-bit definitions
that the GPU tests compare with, against themselves written another way and against differences."""

import inspect
import math

import pytest
import torch

import ops_oracle as oracle
from causal_conv1d_triton import paged, recurrence
from causal_conv1d_triton._ops import native
from causal_conv1d_triton.paged import paged_attention, paged_cache_write, paged_plan
from causal_conv1d_triton.recurrence import gated_recurrence_fn, gated_recurrence_update


def test_import_surface():
    assert native() is not None
    assert list(inspect.signature(gated_recurrence_fn).parameters) == [
        "x", "gate", "decay", "input_gate", "seq_idx", "initial_states", "return_final_states",
        "decay_scale"]
    assert list(inspect.signature(gated_recurrence_update).parameters) == [
        "x", "gate", "state", "decay", "input_gate", "state_indices", "decay_scale"]
    assert paged.PagedPlan._fields == ("seq_lens", "query_start", "positions", "request_ids",
                                       "slot_mapping", "num_free")
    assert list(inspect.signature(paged_attention).parameters) == [
        "q", "k_cache", "v_cache", "block_tables", "seq_lens", "softmax_scale", "window",
        "request_ids", "max_seq_len", "return_lse"]


Z = torch.zeros
I = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731


@pytest.mark.parametrize("args,msg", [
    ((Z(2, 3), Z(2, 3)), "x must be (batch, seqlen, dim)"),
    ((Z(1, 2, 3), Z(1, 2, 4)), "gate must have the shape of x"),
    ((Z(1, 2, 3), Z(1, 2, 3), Z(4)), "decay must be (dim,)"),
    ((Z(1, 2, 3), Z(1, 2, 3), I(3)), "decay must be floating point"),
    ((Z(1, 2, 3), Z(1, 2, 3), None, Z(1, 2)), "input_gate must have the shape of x"),
    ((Z(1, 2, 3), Z(1, 2, 3), None, None, I(2, 1)), "seq_idx must be (batch, seqlen)"),
    ((Z(1, 2, 3), Z(1, 2, 3), None, None, Z(1, 2)), "seq_idx must hold integers"),
    ((Z(1, 2, 3), Z(1, 2, 3), None, None, None, Z(1, 1, 3)), "initial_states must be (batch, dim)"),
    ((Z(1, 2, 3), Z(1, 2, 3), None, None, None, I(1, 3)), "initial_states must be floating point"),
    ((Z(1, 2, 3), Z(1, 2, 3), None, None, None, None, False, -1.0), "decay_scale"),
    ((Z(1, 2, 3), Z(1, 2, 3)), "x must be on a GPU"),
])
def test_recurrence_refuses(args, msg):
    with pytest.raises(AssertionError) as e:
        gated_recurrence_fn(*args)
    assert msg in str(e.value)


@pytest.mark.parametrize("args,msg", [
    ((Z(3), Z(3), Z(2, 3)), "x must be (rows, dim)"),
    ((Z(2, 3), Z(3, 2), Z(2, 3)), "gate must have the shape of x"),
    ((Z(2, 3), Z(2, 3), Z(2, 4)), "state must be (slots, dim)"),
    ((Z(2, 3), Z(2, 3), Z(1, 3)), "a slot for each row"),
    ((Z(2, 3), Z(2, 3), Z(2, 3).half()), "state must be fp32"),
    ((Z(2, 3), Z(2, 3), Z(3, 2).t()), "unit channel stride"),
    ((Z(2, 3), Z(2, 3), Z(1, 3).expand(2, 3)), "must not overlap"),
    ((Z(2, 3), Z(2, 3), Z(2, 3), Z(2)), "decay must be (dim,)"),
    ((Z(2, 3), Z(2, 3), Z(2, 3), None, None, I(3)), "state_indices must be (rows,)"),
    ((Z(2, 3), Z(2, 3), Z(2, 3), None, None, Z(2)), "state_indices must hold integers"),
    ((Z(2, 3), Z(2, 3), Z(2, 3)), "x must be on a GPU"),
])
def test_update_refuses(args, msg):
    with pytest.raises(AssertionError) as e:
        gated_recurrence_update(*args)
    assert msg in str(e.value)


def test_not_tensors():
    with pytest.raises(TypeError):
        gated_recurrence_fn([1], Z(1, 2, 3))
    with pytest.raises(TypeError):
        gated_recurrence_update(Z(2, 3), Z(2, 3), 5)
    with pytest.raises(TypeError):
        paged_attention(Z(1, 1, 8), Z(1, 1, 1, 8), Z(1, 1, 1, 8), I(1, 1), [3])
    with pytest.raises(TypeError):
        paged_plan(I(1), I(1), I(1, 1), I(1), I(1), "16", 4)


@pytest.mark.parametrize("args,msg", [
    ((I(2), I(2), I(2, 4), I(9), I(1), 0, 4), "page_size must be at least 1"),
    ((I(2), I(2), I(2, 4), I(9), I(1), 16, -1), "max_tokens must not be negative"),
    ((I(2, 1), I(2), I(2, 4), I(9), I(1), 16, 4), "cached_lens must be (requests,)"),
    ((I(2), I(2), I(2, 4), I(9), I(1), 16, 4), "cached_lens must be on a GPU"),
])
def test_plan_refuses(args, msg):
    with pytest.raises(AssertionError) as e:
        paged_plan(*args)
    assert msg in str(e.value)


C4 = Z(3, 4, 2, 8)


@pytest.mark.parametrize("args,msg", [
    ((Z(5, 2, 8), Z(5, 2, 8), Z(3, 4, 2), C4, I(5)), "k_cache must be (num_pages"),
    ((Z(5, 2, 8), Z(5, 2, 8), C4, Z(3, 4, 2, 9), I(5)), "v_cache must have the shape of k_cache"),
    ((Z(5, 2, 8), Z(5, 2, 8), Z(3, 4, 2, 16)[..., ::2], C4, I(5)), "unit last stride"),
    ((Z(5, 3, 8), Z(5, 2, 8), C4, C4, I(5)), "k must be (tokens, kv_heads, head_dim)"),
    ((Z(5, 2, 8), Z(4, 2, 8), C4, C4, I(5)), "v must have the shape of k"),
    ((Z(5, 2, 8), Z(5, 2, 8), C4, C4, I(4)), "slot_mapping must be (tokens,)"),
    ((Z(5, 2, 8), Z(5, 2, 8), C4, C4, Z(5)), "slot_mapping must hold integers"),
    ((Z(5, 2, 8), Z(5, 2, 8), C4, C4, I(5)), "k must be on a GPU"),
])
def test_write_refuses(args, msg):
    with pytest.raises(AssertionError) as e:
        paged_cache_write(*args)
    assert msg in str(e.value)


@pytest.mark.parametrize("cache", [
    Z(1, 4, 2, 8).expand(3, 4, 2, 8), Z(3, 1, 2, 8).expand(3, 4, 2, 8), Z(3, 4, 1, 8).expand(3, 4, 2, 8),
    Z(200).as_strided((3, 4, 2, 8), (60, 16, 8, 1)), Z(200).as_strided((3, 4, 2, 8), (64, 16, 7, 1)),
    Z(200).as_strided((3, 4, 2, 8), (16, 16, 8, 1))])
def test_write_refuses_caches_that_overlap(cache):
    """Rows written by two workgroups at once would hold whichever came last."""
    for caches in ((cache, C4), (C4, cache)):
        with pytest.raises(AssertionError) as e:
            paged_cache_write(Z(5, 2, 8), Z(5, 2, 8), *caches, I(5))
        assert "must not overlap" in str(e.value)


@pytest.mark.parametrize("cache", [
    C4, Z(3, 2, 4, 8).transpose(1, 2), Z(3, 4, 4, 8)[:, :, 1:3], Z(3, 4, 2, 11)[..., 2:10], Z(4, 3, 2, 8).transpose(0, 1),
    Z(3, 2, 2, 4, 11)[:, 1].transpose(1, 2)[..., :8], Z(9, 4, 2, 8)[::3]])
def test_write_takes_caches_with_strides(cache):
    with pytest.raises(AssertionError) as e:
        paged_cache_write(Z(5, 2, 8), Z(5, 2, 8), cache, C4, I(5))
    assert "k must be on a GPU" in str(e.value)


@pytest.mark.parametrize("args,kw,msg", [
    ((Z(2, 8), C4, C4, I(2, 3), I(2)), {}, "q must be (rows, q_heads, head_dim)"),
    ((Z(2, 4, 9), C4, C4, I(2, 3), I(2)), {}, "the caches must have the head_dim of q"),
    ((Z(2, 3, 8), C4, C4, I(2, 3), I(2)), {}, "q_heads must be a multiple of kv_heads"),
    ((Z(2, 4, 12), Z(3, 4, 2, 12), Z(3, 4, 2, 12), I(2, 3), I(2)), {}, "multiple of 8, at most 256"),
    ((Z(2, 4, 264), Z(3, 4, 2, 264), Z(3, 4, 2, 264), I(2, 3), I(2)), {}, "multiple of 8"),
    ((Z(2, 4, 8), C4, C4, I(2, 3), I(3)), {}, "seq_lens must be (rows,)"),
    ((Z(2, 4, 8), C4, C4, I(2), I(2)), {}, "block_tables must be (requests, max_pages)"),
    ((Z(2, 4, 8), C4, C4, I(1, 3), I(2)), {}, "block_tables must have a row for each row of q"),
    ((Z(2, 4, 8), C4, C4, I(2, 3), I(2)), dict(request_ids=I(3)), "request_ids must be (rows,)"),
    ((Z(2, 4, 8), C4, C4, I(2, 3).long(), I(2)), {}, "block_tables must be int32"),
    ((Z(2, 4, 8), C4, C4, I(2, 6)[:, ::2], I(2)), {}, "rows of block_tables must be contiguous"),
    ((Z(2, 4, 8), C4, C4, I(2, 3), Z(2)), {}, "must hold integers"),
    ((Z(2, 4, 8), C4, C4, I(2, 3), I(2)), dict(window=0), "window must be at least 1"),
    ((Z(2, 4, 8), C4, C4, I(2, 3), I(2)), dict(max_seq_len=-1), "max_seq_len must not be negative"),
    ((Z(2, 4, 8), C4, C4, I(2, 3), I(2)), {}, "q must be on a GPU"),
])
def test_attention_refuses(args, kw, msg):
    with pytest.raises(AssertionError) as e:
        paged_attention(*args, **kw)
    assert msg in str(e.value)


@pytest.mark.parametrize("decay,igate,init", [(True, True, True), (True, False, False),
                                              (False, True, True), (False, False, False)])
def test_fake_shapes(decay, igate, init):
    """The registered operators' fake implementations give the real outputs' shapes and types."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        f = lambda *s, t=torch.bfloat16: torch.empty(*s, device="cuda", dtype=t)  # noqa: E731
        x, gate = f(2, 130, 8), f(2, 130, 8)
        d, i = f(8, t=torch.float32) if decay else None, f(2, 130, 8) if igate else None
        s = f(2, 8, t=torch.float16) if init else None
        out, fin, saved = recurrence._fwd_op(x, gate, d, i, None, s, 8.0)
        assert out.shape == x.shape and out.dtype == x.dtype
        assert fin.shape == (2, 8) and fin.dtype == torch.float32
        assert saved.shape == (2, 3, 8) and saved.dtype == torch.float32
        g = recurrence._bwd_op(x, gate, d, i, None, s, 8.0, saved, out, fin, init)
        assert g[0].shape == g[1].shape == x.shape
        assert g[2].shape == ((8,) if decay else (0,))
        assert g[3].shape == (x.shape if igate else (0,))
        assert g[4].shape == ((2, 8) if init else (0,))
        assert not init or g[4].dtype == torch.float16


@pytest.mark.parametrize("call", [
    lambda d: gated_recurrence_fn(d(1, 2, 3), Z(1, 2, 3)),
    lambda d: gated_recurrence_fn(Z(1, 2, 3), Z(1, 2, 3), d(3)),
    lambda d: gated_recurrence_fn(Z(1, 2, 3).requires_grad_(), d(1, 2, 3)),
    lambda d: gated_recurrence_update(Z(2, 3), Z(2, 3), d(2, 3)),
    lambda d: paged_cache_write(Z(5, 2, 8), d(5, 2, 8), C4, C4, I(5)),
    lambda d: paged_attention(d(2, 4, 8), C4, C4, I(2, 3), I(2)),
])
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(call, grad):
    """Autograd is off for one-token calls, which leaves tangents on."""
    import torch.autograd.forward_ad as ad
    with ad.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(NotImplementedError) as e:
            call(lambda *s: ad.make_dual(Z(*s), torch.ones(*s)))
        assert "forward-mode" in str(e.value)
        with ad._set_fwd_grad_enabled(False), pytest.raises(AssertionError) as e:  # as if there were none
            call(lambda *s: ad.make_dual(Z(*s), torch.ones(*s)))
        assert "must be on a GPU" in str(e.value)


def test_tensors_without_memory_are_refused():
    """An address of null means an absent tensor to the library."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(2, 13, 8, device="cuda")
        with pytest.raises(TypeError) as e:
            gated_recurrence_fn(x, x)
        assert "memory of its own" in str(e.value)
        with pytest.raises(TypeError) as e:
            gated_recurrence_update(x[0], x[0], x[0])
        assert "memory of its own" in str(e.value)


# ------------------------------------------------------------------------------ the oracle


def _case(decay, igate, packed, T=12):
    g = torch.Generator().manual_seed(3)
    n = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    seq = None
    if packed:
        seq = torch.tensor([[0, 0, 0, 1, 1, -1, -1, 2, 2, 2, 3, -1], [4] * 12])[:, :T]
    return dict(x=n(2, T, 3), gate=n(2, T, 3), decay=n(3) - 3 if decay else None,
                igate=n(2, T, 3) if igate else None, seq=seq, init=n(2, 3)), n(2, T, 3), n(2, 3)


def _plain(x, gate, decay, igate, seq, init):
    """Element by element, in Python's floats."""
    B, T, D = x.shape
    out, fin = torch.zeros(B, T, D, dtype=torch.float64), torch.zeros(B, D, dtype=torch.float64)
    for b in range(B):
        for d in range(D):
            h = float(init[b, d])
            for t in range(T):
                r = 1 / (1 + math.exp(-float(gate[b, t, d])))
                i = 1.0 if igate is None else 1 / (1 + math.exp(-float(igate[b, t, d])))
                if decay is None:
                    a, beta = r, 1 - r
                else:
                    a = math.exp(-8.0 * math.log1p(math.exp(float(decay[d]))) * r)
                    beta = math.sqrt(1 - a * a)
                if seq is not None and seq[b, t] < 0:
                    h = 0.0
                else:
                    if seq is not None and t > 0 and seq[b, t] != seq[b, t - 1]:
                        h = 0.0
                    h = a * h + beta * i * float(x[b, t, d])
                out[b, t, d] = h
            fin[b, d] = h
    return out, fin


@pytest.mark.parametrize("decay", [True, False])
@pytest.mark.parametrize("igate", [True, False])
@pytest.mark.parametrize("packed", [True, False])
def test_oracle_recurrence(decay, igate, packed):
    """The oracle's states are the definition's, and its gradients those of differences."""
    t, dy, dfin = _case(decay, igate, packed)
    res = oracle.recurrence(**t, dy=dy, dfinal=dfin)
    out, fin = _plain(**t)
    assert torch.allclose(res["out"][0], out, rtol=1e-12, atol=1e-13)
    assert torch.allclose(res["final"][0], fin, rtol=1e-12, atol=1e-13)

    def loss(u):
        o, f = _plain(**u)
        live = 1.0 if t["seq"] is None else (t["seq"] >= 0)[..., None].double()
        end = 1.0 if t["seq"] is None else (t["seq"][:, -1] >= 0)[:, None].double()
        return float((o * dy * live).sum() + (f * dfin * end).sum())

    for k in ("x", "gate", "decay", "igate", "init"):
        if t[k] is None:
            continue
        g, eps = torch.zeros_like(t[k]), 1e-5
        for j in range(t[k].numel()):
            up, down = t[k].clone(), t[k].clone()
            up.view(-1)[j] += eps
            down.view(-1)[j] -= eps
            g.view(-1)[j] = (loss({**t, k: up}) - loss({**t, k: down})) / (2 * eps)
        # second-order differences: eps^2 of the third derivative, and rounding over eps
        assert torch.allclose(res[k][0], g, rtol=1e-6, atol=1e-7), k


def test_oracle_attention():
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(6, 4, 2, 8, generator=g) for _ in range(2))
    tables = torch.tensor([[5, 2, 0, 3], [1, 4, -1, 9]], dtype=torch.int32)
    q = torch.randn(2, 4, 8, generator=g)
    (out, _), (lse, _) = oracle.attention(q, k, v, tables, torch.tensor([14, 16]), window=9)
    for r, keep in ((0, range(5, 14)), (1, range(7, 8))):
        kk = torch.stack([k[tables[r, p // 4], p % 4] for p in keep]).double()
        vv = torch.stack([v[tables[r, p // 4], p % 4] for p in keep]).double()
        for h in range(4):
            s = kk[:, h // 2] @ q[r, h].double() / math.sqrt(8)
            assert torch.allclose(out[r, h], torch.softmax(s, 0) @ vv[:, h // 2])
            assert torch.allclose(lse[r, h], torch.logsumexp(s, 0))


def test_oracle_plan():
    """Two requests that share a short free list, by hand."""
    res = oracle.plan(torch.tensor([3, 4, 0]), torch.tensor([2, 1, 1]),
                      torch.tensor([[7, -1], [8, -1], [-1, -1]]), torch.tensor([1, 2]), 2, 4, 6)
    assert res["tables"].tolist() == [[7, 2], [8, 1], [-1, -1]]  # the third finds no page
    assert res["seq_lens"].tolist() == [5, 5, 0]
    assert res["query_start"].tolist() == [0, 2, 3, 4]
    assert res["positions"].tolist() == [3, 4, 4, -1, -1, -1]
    assert res["request_ids"].tolist() == [0, 0, 1, -1, -1, -1]
    assert res["slot_mapping"].tolist() == [31, 8, 4, -1, -1, -1]
    assert res["num_free"].tolist() == [0]
