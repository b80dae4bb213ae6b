"""How many bits the operators of a linear-attention layer keep: bounds close to what fp32 arithmetic gives, where those
of test_layer_delta.py and test_layer_norm.py hold for every element at its worst."""

import pytest
import torch

import layer_oracle as oracle
from test_layer_delta import BF, HF, make, run

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
