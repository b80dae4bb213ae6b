"""How many bits the operators of a linear-attention layer keep: bounds close to what fp32 arithmetic gives, where those
of test_layer_delta.py and test_layer_norm.py hold for every element at its worst."""

import pytest
import torch

import layer_oracle as oracle
from causal_conv1d_triton.norm import block_norm_fn
from test_layer_delta import BF, F, HF, make, run
from test_layer_norm import make as make_norm, run as run_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Dk", [64, 128, 200])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_outputs_of_16_bits_are_the_nearest(dtype, Dk):
    """Of an fp32 number whose error has a mean of e, rounded to a type whose steps are s apart, 2 e / s come out as the
    number beside the nearest one (so near lies the middle between two). With e = 2^-21 of the outputs' root mean
    square, eight units of fp32, and outputs of a quarter of that and more, whose steps are more than 2^-8 (bf16) or
    2^-11 (fp16) of themselves: 2^-10 or 2^-7 of them."""
    t = make(Dk, B=2, T=300, Hk=2, H=4, Dk=Dk, Dv=64, dtype=dtype, init=True, grad=False)
    share = oracle.share_beside(run(t)["out"], oracle.delta_all(t)["out"])
    assert share <= {BF: 2.0 ** -10, HF: 2.0 ** -7}[dtype], share


def trained(seed, **kw):
    t = make(seed, init=True, **kw)
    t["beta"] = t["beta"].float()
    final = torch.randn(t["init"].shape, generator=torch.Generator().manual_seed(seed))
    return run(t, final), oracle.delta_all(t, final)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("Dk,Dv,T", [(64, 40, 64), (64, 64, 300), (100, 33, 129), (128, 64, 300), (130, 40, 70), (256, 64, 300)])
@pytest.mark.parametrize("dtype", [F, BF, HF])
def test_delta_in_fp32(dtype, Dk, Dv, T, packed):
    """Everything that is kept in fp32, in the root mean square; results of 16 bits are the nearest numbers."""
    got, want = trained(Dk + T, B=2, T=T, Hk=2, H=4, Dk=Dk, Dv=Dv, dtype=dtype, packed=packed)
    for n, x in got.items():
        if x.dtype == F:
            oracle.rms_close(x, want[n], n)
        else:
            # as the outputs above, with the means of e = 2^-20: sums over heads and small tensors
            assert oracle.share_beside(x, want[n]) <= {BF: 2.0 ** -9, HF: 2.0 ** -6}[dtype], n


@pytest.mark.parametrize("dtype", [F, BF, HF])
def test_update_in_fp32(dtype):
    from causal_conv1d_triton.delta import gated_delta_update
    t = make(41, B=1, T=50, Hk=2, H=4, Dk=128, Dv=128, dtype=dtype, grad=False)
    gen = torch.Generator().manual_seed(1)
    state = torch.randn(50, 4, 128, 128, generator=gen)
    names = ("q", "k", "v", "g", "beta")
    one = {n: t[n][0][:, None] for n in names}
    want = oracle.delta_all(dict(one, init=state))
    pool = state.cuda()
    with torch.no_grad():
        out = gated_delta_update(*(t[n][0].cuda() for n in names), pool)
    oracle.rms_close(pool, want["final"], "final")
    if dtype == F:
        oracle.rms_close(out[:, None], want["out"], "out")
    else:
        assert oracle.share_beside(out[:, None], want["out"]) <= {BF: 2.0 ** -10, HF: 2.0 ** -7}[dtype]


@pytest.mark.parametrize("rows,D", [(33, 64), (33, 300), (1025, 2048), (7, 8192), (40000, 128)])
@pytest.mark.parametrize("dtype", [F, BF, HF])
def test_norms_in_fp32(dtype, rows, D):
    """The weights' gradients, sums over all rows in 32 lines of 1024 at most, and in fp32 everything, in the root mean
    square: a row left out of 40000 would be 5000 units and more, a sum kept in 16 bits 74."""
    t = make_norm(rows + D, (rows, D), dtype, F, True, True, "tensor", True)
    got, want = run_norm(t), oracle.norm_all(t)
    for n, x in got.items():
        if x.dtype == F:
            oracle.rms_close(x, want[n], n)
        else:
            assert oracle.share_beside(x, want[n]) <= {BF: 2.0 ** -9, HF: 2.0 ** -6}[dtype], n


@pytest.mark.parametrize("activation", ["silu", "sigmoid"])
def test_gates_far_from_zero_are_no_less_exact(activation):
    """Rows of 64 behind a norm with unit weights, gates from -86 to 86, in units of 2^-24 of each element: the sum of
    squares 8 terms a lane and 4 steps of a tree, half of their 12 roundings in the root; 1 / 64 and eps 1/2, root 2,
    quotient 2; three products 3; the exponential 2, its argument's correction and factor 2, the sum with one 1, the
    reciprocal 2; 24 together. (With the argument rounded to fp32 it is 2^-18 ln 2 alone, 44 units, at -80.)"""
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(500, 64, generator=gen)
    gate = 172 * torch.rand(500, 64, generator=gen) - 86
    with torch.no_grad():
        got = block_norm_fn(x.cuda(), None, torch.ones(64, device="cuda"), gate.cuda(), activation=activation).cpu().double()
    want, _ = oracle.norm(x.double(), post=torch.ones(64, dtype=torch.float64), gate=gate.double(), activation=activation)
    units = ((got - want).abs() / want.abs()).max() * 2.0 ** 24
    assert float(units) <= 24, float(units)
