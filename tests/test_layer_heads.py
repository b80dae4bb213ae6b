"""The delta rule with many heads of a key, in the workgroups that make the systems of all heads of a chunk (512 chunks of
keys and more), four at a time, and in those that make one head's each."""

import math

import pytest
import torch

import layer_oracle as oracle
from test_layer_delta import BF, F, HF, check, make, run

pytestmark = pytest.mark.gpu

SIZES = dict(B=8, T=520, Hk=8, Dk=16, Dv=16)  # 8 * 8 * 9 chunks


@pytest.mark.parametrize("group", [3, 4, 5, 6, 9])
@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_heads_of_a_key_in_one_workgroup(dtype, group):
    t = make(group, H=8 * group, dtype=dtype, packed=True, **SIZES)
    got = run(t)
    pick = {n: None if x is None else x[5:6] for n, x in t.items()}
    want = oracle.delta_all(pick)
    for n, x in got.items():
        oracle.delta_close(x[5:6], want[n], n, pick)
        if x.dtype == F and want[n].any():
            oracle.rms_close(x[5:6], want[n], n)


@pytest.mark.parametrize("Dk", [64, 256])
def test_wide_heads_of_a_key_in_one_workgroup(Dk):
    t = make(50 + Dk, B=9, T=500, Hk=8, H=40, Dk=Dk, Dv=16, dtype=BF)
    got = run(t)
    pick = {n: None if x is None else x[8:] for n, x in t.items()}
    want = oracle.delta_all(pick)
    for n, x in got.items():
        oracle.delta_close(x[8:], want[n], n, pick)
        if x.dtype == F:
            oracle.rms_close(x[8:], want[n], n)


@pytest.mark.parametrize("name,bad", [("k", math.inf), ("q", math.nan), ("v", math.nan), ("beta", math.inf), ("g", math.nan)])
@pytest.mark.parametrize("dtype", [BF, F])
def test_spoilt_rows_of_some_heads(dtype, name, bad):
    """Of a key, all heads that share it; of the others, the head whose it is."""
    t = make(7, H=48, dtype=dtype, **SIZES)
    t["seq"] = ((torch.arange(520) >= 30).int() + (torch.arange(520) >= 50).int())[None].expand(8, -1).contiguous()
    clean = run(t)
    t[name] = t[name].clone()
    t[name][3, 40, 5] = bad  # a key head, or a head of key head 0
    got = run(t)
    own = torch.zeros(8, 520, dtype=torch.bool)
    own[3, 30:50] = True
    heads = range(30, 36) if name in ("q", "k") else [5]
    for n in ("out", "v", "g", "beta"):
        rest = torch.ones(48, dtype=torch.bool)
        rest[list(heads)] = False
        assert torch.equal(got[n][:, :, rest], clean[n][:, :, rest]), n
    for n in ("out", "q", "k", "v", "g", "beta"):
        assert torch.equal(got[n][~own], clean[n][~own]), n
    for h in heads:
        assert not torch.isfinite(got["out"][3, 40, h]).any()
    assert torch.equal(got["final"], clean["final"])


@pytest.mark.parametrize("Hk,H", [(1, 3), (2, 8), (1, 6)])
def test_shared_keys_in_fp16(Hk, H):
    check(make(7 * H + Hk, T=90, Hk=Hk, H=H, dtype=HF))
