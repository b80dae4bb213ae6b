"""How many bits the operators of a linear-attention layer keep: bounds close to what fp32 arithmetic gives, where those
of test_layer_delta.py and test_layer_norm.py hold for every element at its worst."""

import pytest
import torch

import layer_oracle as oracle
from causal_conv1d_triton.norm import block_norm_fn
from test_layer_delta import BF, F, HF, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Dk", [64, 128, 200])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_outputs_of_16_bits_are_the_nearest(dtype, Dk):
    """Of an fp32 number whose error has a mean of e, rounded to a type whose steps are s apart, 2 e / s come out as the
    number beside the nearest one (so near lies the middle between two). With e = 2^-21 of the outputs' root mean
    square, eight units of fp32, and outputs of a quarter of that and more, whose steps are more than 2^-8 (bf16) or
    2^-11 (fp16) of themselves: 2^-10 or 2^-7 of them."""
    t = make(Dk, B=2, T=300, Hk=2, H=4, Dk=Dk, Dv=64, dtype=dtype, init=True, grad=False)
    got, want = run(t)["out"].cpu(), oracle.delta_all(t)["out"]
    large = want.abs() >= 0.25 * want.square().mean().sqrt()
    share = float((got != want.to(dtype))[large].double().mean())
    assert share <= {BF: 2.0 ** -10, HF: 2.0 ** -7}[dtype], share


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
