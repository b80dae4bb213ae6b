"""The operators of a linear-attention layer without a GPU: signatures, the refusals that need no GPU tensor, the
registered operators' fake implementations, and the 64-bit definitions that the GPU tests compare with, against the
same written another way and against differences."""

import inspect
import math

import pytest
import torch

import layer_oracle as oracle
from causal_conv1d_triton import delta, norm
from causal_conv1d_triton.delta import gated_delta_fn, gated_delta_update
from causal_conv1d_triton.norm import block_norm_fn

Z = torch.zeros
I = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731


def test_signatures():
    assert list(inspect.signature(gated_delta_fn).parameters) == [
        "q", "k", "v", "log_decay", "beta", "seq_idx", "initial_states", "return_final_states", "scale"]
    assert list(inspect.signature(gated_delta_update).parameters) == [
        "q", "k", "v", "log_decay", "beta", "state", "state_indices", "scale"]
    assert list(inspect.signature(block_norm_fn).parameters) == [
        "x", "residual", "post_weight", "gate", "scale", "pre_weight", "eps", "activation"]


K, V, G = Z(1, 5, 2, 8), Z(1, 5, 4, 6), Z(1, 5, 4)


@pytest.mark.parametrize("args,msg", [
    ((Z(5, 2, 8), Z(5, 2, 8), V, G, G), "k must be (batch, seqlen"),
    ((K, K, Z(5, 4, 6), G, G), "v must be (batch, seqlen"),
    ((Z(1, 5, 2, 7), K, V, G, G), "q must have the shape of k"),
    ((K, K, Z(1, 6, 4, 6), G, G), "the batch and seqlen of k"),
    ((K, K, Z(1, 5, 3, 6), Z(1, 5, 3), Z(1, 5, 3)), "multiple of the heads of k"),
    ((K, K, Z(1, 5, 0, 6), Z(1, 5, 0), Z(1, 5, 0)), "multiple of the heads of k"),
    ((Z(1, 5, 2, 257), Z(1, 5, 2, 257), V, G, G), "key_dim must be 1 to 256"),
    ((Z(1, 5, 2, 0), Z(1, 5, 2, 0), V, G, G), "key_dim must be 1 to 256"),
    ((K, K, Z(1, 5, 4, 0), G, G), "value_dim must be at least 1"),
    ((K, K, V, Z(1, 5, 2), G), "log_decay must be (batch"),
    ((K, K, V, G, Z(1, 4, 4)), "beta must be (batch"),
    ((K, K, V, G, G, I(1, 4)), "seq_idx must be (batch, seqlen)"),
    ((K, K, V, G, G, Z(1, 5)), "seq_idx must hold integers"),
    ((K, K, V, G, G, None, Z(1, 4, 6, 8)), "initial_states must be (batch"),
    ((K, K, V, G, G, None, I(1, 4, 8, 6)), "initial_states must be floating point"),
    ((K, K, V, G, G), "k must be on a GPU"),
])
def test_delta_refuses(args, msg):
    with pytest.raises(AssertionError) as e:
        gated_delta_fn(*args)
    assert msg in str(e.value)


k2, v2, g2, s2 = Z(3, 2, 8), Z(3, 4, 6), Z(3, 4), Z(3, 4, 8, 6)


@pytest.mark.parametrize("args,msg", [
    ((Z(3, 8), Z(3, 8), v2, g2, g2, s2), "k must be (rows"),
    ((k2, k2, Z(3, 6), g2, g2, s2), "v must be (rows"),
    ((Z(3, 2, 7), k2, v2, g2, g2, s2), "q must have the shape of k"),
    ((k2, k2, Z(4, 4, 6), g2, g2, s2), "v must have the rows of k"),
    ((k2, k2, Z(3, 5, 6), Z(3, 5), Z(3, 5), Z(3, 5, 8, 6)), "multiple of the heads of k"),
    ((k2, k2, v2, Z(3, 2), g2, s2), "log_decay must be (rows, heads)"),
    ((k2, k2, v2, g2, Z(3), s2), "beta must be (rows, heads)"),
    ((k2, k2, v2, g2, g2, Z(3, 4, 6, 8)), "state must be (slots"),
    ((k2, k2, v2, g2, g2, Z(2, 4, 8, 6)), "a slot for each row"),
    ((k2, k2, v2, g2, g2, s2.half()), "state must be fp32"),
    ((k2, k2, v2, g2, g2, Z(3, 4, 6, 8).transpose(2, 3)), "each slot of state must be contiguous"),
    ((k2, k2, v2, g2, g2, Z(1, 4, 8, 6).expand(3, -1, -1, -1)), "must not overlap"),
    ((k2, k2, v2, g2, g2, s2, I(2)), "state_indices must be (rows,)"),
    ((k2, k2, v2, g2, g2, s2, Z(3)), "state_indices must hold integers"),
    ((k2, k2, v2, g2, g2, s2), "k must be on a GPU"),
])
def test_update_refuses(args, msg):
    with pytest.raises(AssertionError) as e:
        gated_delta_update(*args)
    assert msg in str(e.value)


X, W = Z(3, 8), Z(8)


@pytest.mark.parametrize("args,msg", [
    ((X,), "post_weight or pre_weight must be given"),
    ((Z(()), None, Z(1)), "x must be (..., dim)"),
    ((Z(3, 0), None, Z(0)), "dim must be 1 to 8192"),
    ((Z(1, 8193), None, Z(8193)), "dim must be 1 to 8192"),
    ((X, Z(2, 8), W), "residual must have the shape of x"),
    ((X, None, Z(7)), "post_weight must be (dim,)"),
    ((X, None, W, Z(3, 4)), "gate must have the shape of x"),
    ((X, None, W, None, Z(3)), "scale must be a number or (dim,)"),
    ((X, None, None, None, None, Z(3, 8)), "pre_weight must be (dim,)"),
    ((X, None, W, None, None, None, -1.0), "eps must not be negative"),
    ((X, None, W, None, None, None, math.nan), "eps must not be negative"),
    ((X, None, W), "x must be on a GPU"),
])
def test_norm_refuses(args, msg):
    with pytest.raises(AssertionError) as e:
        block_norm_fn(*args)
    assert msg in str(e.value)


def test_other_refusals():
    with pytest.raises(NotImplementedError):
        block_norm_fn(X, None, W, activation="gelu")
    with pytest.raises(TypeError):
        block_norm_fn(X, None, W, scale="2")
    with pytest.raises(TypeError):
        gated_delta_fn([1.0], K, V, G, G)
    with pytest.raises(TypeError):
        gated_delta_fn(K, K, V, G, G, scale="1")


@pytest.mark.parametrize("call", [
    lambda d: gated_delta_fn(d(1, 5, 2, 8), K, V, G, G),
    lambda d: gated_delta_fn(K, K, V, G, d(1, 5, 4)),
    lambda d: gated_delta_update(k2, k2, v2, g2, g2, d(3, 4, 8, 6)),
    lambda d: block_norm_fn(d(3, 8), None, W),
    lambda d: block_norm_fn(X, None, W, scale=d(8)),
])
def test_forward_mode_is_refused(call):
    import torch.autograd.forward_ad as ad
    with ad.dual_level(), pytest.raises(NotImplementedError) as e:
        call(lambda *s: ad.make_dual(Z(*s), torch.ones(*s)))
    assert "forward-mode" in str(e.value)


def test_fake_shapes():
    """The registered operators' fake implementations give the real outputs' shapes and types, and as many saved
    numbers as the library asks for (tests/test_layer_abi.py has the same formula)."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        f = lambda *s, t=torch.bfloat16: torch.empty(*s, device="cuda", dtype=t)  # noqa: E731
        q, v, g, b = f(2, 130, 3, 72), f(2, 130, 6, 40), f(2, 130, 6, t=torch.float32), f(2, 130, 6)
        s = f(2, 6, 72, 40, t=torch.float16)
        out, fin, saved = delta._fwd_op(q, q, v, g, b, None, s, 1.0)
        assert out.shape == v.shape and out.dtype == v.dtype
        assert fin.shape == s.shape and fin.dtype == torch.float32
        assert saved.shape == (2 * 6 * 3 * (128 + 64) * 64,)
        grads = delta._bwd_op(q, q, v, g, b, None, s, 1.0, saved, out, fin, True)
        assert [(x.shape, x.dtype) for x in grads] == [(x.shape, x.dtype) for x in (q, q, v, g, b, s)]
        x, r, w = f(4, 9, 30), f(4, 9, 30, t=torch.float32), f(30, t=torch.float32)
        got = norm._fwd_op(x, r, None, x, w, 1.0, w, 1e-6, 1)
        assert [(t.shape, t.dtype) for t in got] == [(r.shape, r.dtype), (x.shape, x.dtype)]
        got = norm._fwd_op(x, None, w, None, None, 1.0, None, 1e-6, 1)
        assert got[0].shape == x.shape and got[1].shape == (0,)
        grads = norm._bwd_op(x, r, None, x, w, 1.0, w, 1e-6, 1, r, x, True)
        assert [t.shape for t in grads] == [x.shape, r.shape, (0,), x.shape, w.shape, w.shape]


def test_tensors_without_memory_are_refused():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        f = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
        for call in (lambda: gated_delta_fn(f(1, 5, 2, 8), f(1, 5, 2, 8), f(1, 5, 2, 8), f(1, 5, 2), f(1, 5, 2)),
                     lambda: block_norm_fn(f(3, 8), None, f(8))):
            with pytest.raises(TypeError) as e:
                call()
            assert "memory of its own" in str(e.value)


# ------------------------------------------------------------------------------ the oracle


def _case(T=11):
    gen = torch.Generator().manual_seed(3)
    n = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    seq = torch.tensor([[0, 0, 0, 1, 1, -1, -1, 2, 2, 3, -1], [4] * 11])
    return [n(2, T, 1, 3), n(2, T, 1, 3), n(2, T, 2, 4), -n(2, T, 2).abs(), torch.sigmoid(n(2, T, 2)), seq,
            n(2, 2, 3, 4)]


def test_oracle_delta_is_the_recurrence():
    """Element by element, in Python's floats."""
    q, k, v, g, beta, seq, init = _case()
    out, final = oracle.delta(q, k, v, g, beta, seq, init)
    for b in range(2):
        for h in range(2):
            S = init[b, h].tolist()
            for t in range(11):
                if seq[b, t] < 0 or (t and seq[b, t] != seq[b, t - 1]):
                    S = [[0.0] * 4 for _ in range(3)]
                else:
                    S = [[math.exp(g[b, t, h]) * x for x in row] for row in S]
                if seq[b, t] < 0:
                    assert not out[b, t, h].any()
                    continue
                kt, qt = k[b, t, 0].tolist(), q[b, t, 0].tolist()
                for c in range(4):
                    u = float(beta[b, t, h]) * (float(v[b, t, h, c]) - sum(kt[i] * S[i][c] for i in range(3)))
                    for i in range(3):
                        S[i][c] += kt[i] * u
                want = [sum(qt[i] * S[i][c] for i in range(3)) * 3 ** -0.5 for c in range(4)]
                torch.testing.assert_close(out[b, t, h], torch.tensor(want, dtype=torch.float64))
            torch.testing.assert_close(final[b, h], torch.tensor(S, dtype=torch.float64))


def test_oracle_delta_against_differences():
    q, k, v, g, beta, seq, init = _case()
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v, g, beta, init)]
    torch.autograd.gradcheck(lambda *x: oracle.delta(*x[:5], seq, x[5]), leaves, atol=1e-6)


def test_oracle_norm_against_differences():
    gen = torch.Generator().manual_seed(3)
    n = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64).requires_grad_(True)  # noqa: E731
    for activation in ("silu", "sigmoid", None):
        torch.autograd.gradcheck(
            lambda x, r, p, z, s, w: oracle.norm(x, r, p, z, s, w, activation=activation),
            [n(3, 5), n(3, 5), n(5), n(3, 5), n(5), n(5)])


def test_a_mistake_is_outside_the_bounds():
    """What the comparison has to catch: a decay left out, a rate on the wrong row, a state lost at a chunk's end."""
    gen = torch.Generator().manual_seed(5)
    n = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    k = torch.nn.functional.normalize(n(1, 130, 1, 64), dim=-1)
    t = {"q": k.roll(1, 1), "k": k, "v": n(1, 130, 1, 16), "g": -0.05 * n(1, 130, 1).abs(),
         "beta": torch.sigmoid(n(1, 130, 1))}
    want = oracle.delta_all(t)["out"]
    wrong = [dict(t, g=t["g"] * 0), dict(t, beta=t["beta"].roll(1, 1)),
             dict(t, g=torch.where(torch.arange(130)[None, :, None] == 64, torch.tensor(-50.0), t["g"]))]
    oracle.delta_close(want.float(), want, "out", t)
    for w in wrong:
        with pytest.raises(AssertionError):
            oracle.delta_close(oracle.delta_all(w)["out"].float(), want, "out", t)
