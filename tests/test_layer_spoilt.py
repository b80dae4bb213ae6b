"""Infinities and NaN in the gated delta rule's sequences whose decays are zero in fp32 by the product of many, none
of them alone: the sequence stays spoilt, as the recurrence has it, and no other does."""

import math

import pytest
import torch

from test_layer_delta import BF, F, HF, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("decay", [-3.0, -20.0, -95.0, -103.0])
@pytest.mark.parametrize("dtype,Dk", [(BF, 64), (HF, 128), (F, 100), (BF, 256)])
def test_a_strong_decay_leaves_what_is_no_number(dtype, Dk, decay):
    """Two sequences, cut within the third 64 rows; the first one's row 5 holds a NaN value."""
    t = make(31, B=1, T=260, Hk=1, H=1, Dk=Dk, Dv=40, dtype=dtype, init=True, grad=False)
    t["g"][:] = decay
    t["seq"] = (torch.arange(260) >= 150).int()[None]
    clean = run(t)
    t["v"] = t["v"].clone()
    t["v"][:, 5] = math.nan
    got = run(t)
    assert torch.equal(got["out"][:, :5], clean["out"][:, :5]) and torch.equal(got["out"][:, 150:], clean["out"][:, 150:])
    assert not torch.isfinite(got["out"][:, 5:150]).any()
    assert torch.isfinite(clean["out"]).all() and torch.equal(got["final"], clean["final"])
    t["seq"] = None
    assert not torch.isfinite(run(t)["final"]).any()


@pytest.mark.parametrize("first", [-95.0, -60.0])
def test_a_strong_decay_in_one_row(first):
    """Of the first row of 64 alone."""
    t = make(32, B=1, T=200, Hk=1, H=1, dtype=BF, init=True, grad=False)
    t["g"][:, 64] = t["g"][:, 128] = first
    t["init"] = t["init"] * math.inf
    got = run(t)
    assert not torch.isfinite(got["out"]).any() and not torch.isfinite(got["final"]).any()


@pytest.mark.parametrize("dtype,Dk", [(BF, 64), (HF, 128), (F, 100), (BF, 256)])
def test_gradients_in_front_of_a_strong_decay(dtype, Dk):
    """A gradient that is no number reaches every row of its sequence in front of it, and no other sequence."""
    t = make(33, B=1, T=260, Hk=1, H=1, Dk=Dk, Dv=40, dtype=dtype, init=True)
    t["g"][:] = -3.0
    t["seq"] = (torch.arange(260) >= 20).int()[None]
    clean = run(t)
    t["do"] = t["do"].clone()
    t["do"][:, 200] = math.nan
    got = run(t)
    for n in ("k", "v", "beta"):
        assert not torch.isfinite(got[n][:, 20:201]).any(), n
    for n in ("q", "k", "v", "g", "beta"):
        assert torch.equal(got[n][:, :20], clean[n][:, :20]), n
        assert torch.equal(got[n][:, 201:], clean[n][:, 201:]), n
    assert torch.equal(got["init"], clean["init"]) and torch.equal(got["out"], clean["out"])
    t["seq"] = None
    assert not torch.isfinite(run(t)["init"]).any()


@pytest.mark.parametrize("row", [50, 70])
@pytest.mark.parametrize("dtype,Dk", [(BF, 64), (HF, 128), (F, 100), (BF, 256)])
def test_an_infinite_decay_spoils_its_own_sequence(dtype, Dk, row):
    """A finite log-decay whose exponential is infinite in fp32; in the first row of a sequence it multiplies nothing."""
    t = make(34, B=1, T=270, Hk=1, H=2, Dk=Dk, Dv=40, dtype=dtype, init=True)
    starts = torch.tensor([0, 17, 40, 75, 90, 150, 192, 263])
    t["seq"] = (torch.arange(270)[:, None] >= starts).sum(1).int()[None]
    clean = run(t)
    t["g"] = t["g"].clone()
    t["g"][:, row] = 200.0
    t["g"][:, 90] = 200.0
    got = run(t)
    own = (torch.arange(270) >= 40) & (torch.arange(270) < 75)
    for n in ("out", "q", "k", "v", "g", "beta"):
        assert torch.equal(got[n][:, ~own], clean[n][:, ~own]), n
    for n in ("final", "init"):
        assert torch.equal(got[n], clean[n]), n
    assert torch.equal(got["out"][:, 40:row], clean["out"][:, 40:row])
    assert not torch.isfinite(got["out"][:, row:75]).any()
