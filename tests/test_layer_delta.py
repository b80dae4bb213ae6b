"""The gated delta rule on the GPU against its definition in 64 bits (tests/layer_oracle.py, which derives the
bounds), forward and backward: types, lengths from one row, odd head sizes, shared keys, strides, packed
sequences and padding, decays at the ends of their range, states, streams and graphs; and its single-token form."""

import math

import pytest
import torch

import layer_oracle as oracle
from causal_conv1d_triton.delta import gated_delta_fn, gated_delta_update

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F = torch.bfloat16, torch.float16, torch.float32
LEAVES = ("q", "k", "v", "g", "beta", "init")


def ids(gen, B, T):
    seq = torch.zeros(B, T, dtype=torch.int32)
    for b in range(B):
        cuts = torch.randint(0, T + 1, (5,), generator=gen).sort().values.tolist()
        for j, c in enumerate(cuts):
            seq[b, c:] = j + 1
        seq[b, T - T // 10:] = -1
        if T > 20:
            seq[b, cuts[2]:cuts[2] + 3] = -1
    return seq


def make(seed, B=2, T=100, Hk=2, H=2, Dk=64, Dv=32, dtype=BF, packed=False, init=False, grad=True):
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    unit = lambda x: x / x.norm(dim=-1, keepdim=True).clamp(min=1e-6) * 0.99  # noqa: E731
    t = {"q": unit(n(B, T, Hk, Dk)).to(dtype), "k": unit(0.3 + n(B, T, Hk, Dk)).to(dtype), "v": n(B, T, H, Dv).to(dtype),
         "g": -torch.nn.functional.softplus(n(B, T, H) - 2), "beta": torch.sigmoid(n(B, T, H)).to(dtype),
         "seq": ids(gen, B, T) if packed else None, "init": n(B, H, Dk, Dv) if init else None,
         "do": n(B, T, H, Dv).to(dtype) if grad else None}
    return t


def run(t, dfinal=None, scale=None):
    d = {n: None if x is None else x.to(DEV) for n, x in t.items()}
    names = [n for n in LEAVES if d[n] is not None]
    if d["do"] is None:
        with torch.no_grad():
            out, fin = gated_delta_fn(*(d[n] for n in LEAVES[:5]), d["seq"], d["init"], return_final_states=True,
                                      scale=scale)
        return {"out": out, "final": fin}
    for n in names:
        d[n] = d[n].detach().requires_grad_(True)
    out, fin = gated_delta_fn(*(d[n] for n in LEAVES[:5]), d["seq"], d["init"], return_final_states=True, scale=scale)
    outs, ups = [out], [d["do"]]
    if dfinal is not None:
        outs.append(fin)
        ups.append(dfinal.to(DEV))
    grads = torch.autograd.grad(outs, [d[n] for n in names], ups)
    return {"out": out, "final": fin, **dict(zip(names, grads))}


def check(t, dfinal=None, scale=None):
    got = run(t, dfinal, scale)
    want = oracle.delta_all(t, dfinal, scale)
    for n, x in got.items():
        oracle.delta_close(x, want[n], n, t)
    return got


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300])
@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_lengths(T, dtype):
    check(make(T, T=T, dtype=dtype, init=T % 2 == 1))


@pytest.mark.parametrize("Dk", [1, 3, 16, 63, 64, 65, 96, 128, 130, 200, 256])
@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_key_sizes(Dk, dtype):
    check(make(Dk, T=70, Dk=Dk, Dv=40, dtype=dtype, init=True))


@pytest.mark.parametrize("Dv", [1, 2, 15, 16, 17, 31, 33, 64, 100, 129])
@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_value_sizes(Dv, dtype):
    check(make(Dv, T=70, Dk=48, Dv=Dv, dtype=dtype, init=True))


@pytest.mark.parametrize("Hk,H", [(1, 1), (1, 3), (2, 4), (3, 3), (2, 8)])
@pytest.mark.parametrize("dtype", [BF, F])
def test_shared_keys(Hk, H, dtype):
    check(make(7 * H + Hk, T=90, Hk=Hk, H=H, dtype=dtype))


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("Dk", [64, 128, 256])
@pytest.mark.parametrize("init", [False, True])
def test_packed(dtype, Dk, init):
    check(make(11, B=3, T=203, Hk=1, H=2, Dk=Dk, dtype=dtype, packed=True, init=init))


@pytest.mark.parametrize("Dk,Dv,dtype", [(64, 64, BF), (128, 96, BF), (128, 128, BF), (64, 72, HF)])
def test_two_tiles_a_workgroup(Dk, Dv, dtype):
    """More tiles of values than CUs."""
    heads = 4 * (256 // (4 * ((Dv + 31) // 32 * 2)) + 1)
    t = make(Dk + Dv, B=heads // 4, T=130, Hk=4, H=4, Dk=Dk, Dv=Dv, dtype=dtype, init=True)
    check(t)


def test_many_chunks_with_shared_keys():
    """More than 512 chunks of keys: a workgroup makes the systems of all heads of a key."""
    t = make(5, B=8, T=520, Hk=8, H=16, Dk=16, Dv=16)
    got = run(t)
    pick = {n: None if x is None else x[:1] for n, x in t.items()}
    want = oracle.delta_all(pick)
    for n, x in got.items():
        oracle.delta_close(x[:1], want[n], n, pick)


@pytest.mark.parametrize("dtype", [BF, F])
def test_decays(dtype):
    """None, strong, past fp32's range, infinite; and rates of zero, one and two."""
    t = make(3, T=140, dtype=dtype, init=True)
    for at, x in ((5, 0.0), (20, -30.0), (40, -103.0), (41, -105.0), (60, -1000.0), (64, -math.inf), (65, 0.0),
                  (100, -3e38), (127, -math.inf), (128, -math.inf)):
        t["g"][:, at] = x
    t["beta"][:, 7:90:3] = 0
    t["beta"][:, 8:90:3] = 1
    t["beta"][:, 9:90:3] = 2
    check(t)


def test_growth_within_a_chunk():
    """A log-decay above zero is a factor like any other."""
    t = make(4, T=60, dtype=F)
    t["g"] = t["g"] * 0 + 0.02
    check(t)


@pytest.mark.parametrize("gtype", [BF, HF, F])
@pytest.mark.parametrize("btype", [BF, HF, F])
def test_types_of_gates(gtype, btype):
    t = make(6, T=75, packed=True)
    t["g"], t["beta"] = t["g"].to(gtype), t["beta"].to(btype)
    got = check(t)
    assert got["g"].dtype == gtype and got["beta"].dtype == btype


def test_type_of_states():
    t = make(8, T=66, init=True)
    t["init"] = t["init"].to(BF)
    got = run(t)
    assert got["init"].dtype == BF and got["final"].dtype == F
    want = oracle.delta_all(t)
    oracle.delta_close(got["init"], want["init"], "init", t)
    oracle.delta_close(got["out"], want["out"], "out", t)


@pytest.mark.parametrize("scale", [1.0, 0.0, -2.5])
def test_scale(scale):
    check(make(9, T=80, dtype=F), scale=scale)


@pytest.mark.parametrize("dtype", [BF, F])
def test_strides(dtype):
    """Slices of one projection, transposed batches, gates of any strides: the bits of contiguous copies."""
    B, T, H, Dk, Dv = 2, 133, 3, 40, 24
    t = make(10, B=B, T=T, Hk=H, H=H, Dk=Dk, Dv=Dv, dtype=dtype, init=True)
    wide = torch.cat([t[n].flatten(2) for n in ("q", "k", "v")], -1).transpose(0, 1).contiguous().transpose(0, 1).to(DEV)
    parts = dict(zip(("q", "k", "v"), wide.split([H * Dk, H * Dk, H * Dv], -1)))
    lean = {n: x.to(DEV) for n, x in t.items() if x is not None}
    odd = dict(lean, **{n: parts[n].unflatten(-1, (H, -1)) for n in parts})
    odd["g"] = lean["g"].permute(2, 0, 1).contiguous().permute(1, 2, 0)
    odd["beta"] = torch.stack([lean["beta"]] * 2, -1)[..., 0]
    odd["do"] = torch.stack([lean["do"]] * 3, -1)[..., 1]  # no unit stride: copied
    res = []
    for d in (lean, odd):
        leaves = [d[n].detach().requires_grad_(True) for n in LEAVES]
        out = gated_delta_fn(*leaves[:5], None, leaves[5])
        res.append([out.detach(), *torch.autograd.grad(out, leaves, d["do"])])
    for a, b in zip(*res):
        assert torch.equal(a, b)


def test_expanded_inputs():
    """One query and one rate for all: their gradients are summed by autograd over the expanded dimensions."""
    t = make(12, B=2, T=50, dtype=F)
    q1 = t["q"][:1, :1].to(DEV).requires_grad_(True)
    b1 = t["beta"][:, :, :1].to(DEV).requires_grad_(True)
    rest = [t[n].to(DEV) for n in ("k", "v", "g")]
    out = gated_delta_fn(q1.expand(2, 50, -1, -1), *rest, b1.expand(-1, -1, 2))
    got = torch.autograd.grad(out, [q1, b1], t["do"].to(DEV))
    t["q"], t["beta"] = t["q"][:1, :1].expand(2, 50, -1, -1), t["beta"][:, :, :1].expand(-1, -1, 2)
    want = oracle.delta_all(t)
    oracle.close(got[0], want["q"].sum((0, 1), keepdim=True), 1e-3 * 100 ** 0.5, "q")
    oracle.delta_close(got[1], want["beta"].sum(2, keepdim=True), "beta", t)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [BF, F])
def test_padding_may_hold_anything(bad, dtype):
    t = make(13, B=2, T=200, Hk=1, H=2, dtype=dtype, packed=True, init=True)
    pad = t["seq"] < 0
    clean = run(t)
    for n in ("q", "k", "v", "g", "beta", "do"):
        t[n] = t[n].clone()
        t[n][pad] = bad
    got = run(t)
    for n in clean:
        assert torch.equal(got[n], clean[n]), n
    for n in ("out", "q", "k", "v", "g", "beta"):
        assert not got[n][pad.to(DEV)].any(), n


@pytest.mark.parametrize("dtype", [BF, F])
def test_other_sequences_in_other_chunks(dtype):
    """A value that is no number spoils its sequence, and at most the rows of its own 64."""
    t = make(14, B=1, T=256, Hk=1, H=1, dtype=dtype)
    t["seq"] = (torch.arange(256) // 128).int()[None]
    clean = run(t)
    t["v"] = t["v"].clone()
    t["v"][:, 5] = math.nan
    t["k"] = t["k"].clone()
    t["k"][:, 70] = math.inf
    got = run(t)
    assert not torch.isfinite(got["out"][:, 70:128]).any()
    for n in ("out", "q", "k", "v", "g", "beta"):
        assert torch.equal(got[n][:, 128:], clean[n][:, 128:]), n
    assert torch.equal(got["final"], clean["final"])


SPOILT = [("q", math.nan), ("k", math.inf), ("v", -math.inf), ("v", math.nan), ("g", math.inf), ("g", math.nan),
          ("beta", math.inf), ("beta", math.nan), ("do", math.inf)]


@pytest.mark.parametrize("row", [50, 70])
@pytest.mark.parametrize("name,bad", SPOILT)
@pytest.mark.parametrize("dtype,Dk", [(BF, 64), (BF, 130), (HF, 40), (F, 100)])
def test_other_sequences_in_the_same_chunk(dtype, Dk, name, bad, row):
    """A row that holds an infinity or NaN spoils its sequence from there on (gradients: up to there, too), and
    no bit of any other, wherever in the 64 rows these begin and end."""
    t = make(16, B=1, T=270, Hk=1, H=2, Dk=Dk, Dv=40, dtype=dtype, init=True)
    starts = torch.tensor([0, 17, 40, 75, 90, 150, 192, 263])
    t["seq"] = (torch.arange(270)[:, None] >= starts).sum(1).int()[None]
    clean = run(t)
    t[name] = t[name].clone()
    t[name][:, row] = bad
    got = run(t)
    own = (torch.arange(270) >= 40) & (torch.arange(270) < 75)
    for n in ("out", "q", "k", "v", "g", "beta"):
        assert torch.equal(got[n][:, ~own], clean[n][:, ~own]), n
    for n in ("final", "init"):
        assert torch.equal(got[n], clean[n]), n
    assert torch.equal(got["out"][:, 40:row], clean["out"][:, 40:row])
    if name == "do":
        assert torch.equal(got["out"], clean["out"])
        for n in ("q", "k", "v", "g", "beta"):
            assert torch.equal(got[n][:, row + 1:75], clean[n][:, row + 1:75]), n
            if n != "q":
                assert not torch.isfinite(got[n][:, 40:row]).all(), n
    else:
        assert not torch.isfinite(got["out"][:, row]).any()
        if name == "q":
            assert torch.equal(got["out"][:, row + 1:], clean["out"][:, row + 1:])
        else:
            assert not torch.isfinite(got["out"][:, row:75]).any()


def test_a_spoilt_initial_state_and_a_start_within_the_chunk():
    t = make(17, B=1, T=130, Hk=1, H=1, init=True, grad=False)
    t["seq"] = (torch.arange(130) >= 21).int()[None]
    t["init"] = t["init"] * math.inf
    got = run(t)
    t["init"] = None
    want = run(t)
    assert torch.equal(got["out"][:, 21:], want["out"][:, 21:]) and torch.equal(got["final"], want["final"])
    assert not torch.isfinite(got["out"][:, :21]).any()


def test_a_spoiled_initial_state_ends_with_its_sequence():
    t = make(15, B=1, T=130, Hk=1, H=1, init=True, grad=False)
    t["seq"] = (torch.arange(130) >= 64).int()[None]
    t["init"] = t["init"] * math.inf
    got = run(t)
    t["init"] = None
    want = run(t)
    assert torch.equal(got["out"][:, 64:], want["out"][:, 64:]) and torch.equal(got["final"], want["final"])


def test_all_padding():
    t = make(16, T=90, init=True)
    t["seq"] = torch.full((2, 90), -3, dtype=torch.int32)
    got = run(t, dfinal=torch.ones(2, 2, 64, 32))
    for n, x in got.items():
        assert not x.any(), n


@pytest.mark.parametrize("T", [9, 150])
def test_ids_of_64_bits(T):
    """Ids that agree in their low 32 bits are other sequences."""
    t = make(17, B=1, T=T, packed=True)
    wide = dict(t, seq=torch.where(t["seq"] < 0, t["seq"].long(), t["seq"].long() << 33))
    a, b = run(t), run(wide)
    for n in a:
        assert torch.equal(a[n], b[n]), n


def test_empty():
    for B, T in ((0, 5), (2, 0), (0, 0)):
        t = make(18, B=B, T=T, init=True)
        got = run(t, dfinal=torch.ones(B, 2, 64, 32))
        assert got["out"].shape == (B, T, 2, 32) and got["q"].shape == (B, T, 2, 64)
        assert torch.equal(got["final"].cpu(), t["init"])
        assert torch.equal(got["init"].cpu(), torch.ones(B, 2, 64, 32))


def test_final_states_alone():
    t = make(19, T=150, init=True, packed=False)
    t["do"] = torch.zeros_like(t["do"])
    gen = torch.Generator().manual_seed(1)
    check(t, dfinal=torch.randn(2, 2, 64, 32, generator=gen))
    d = {n: t[n].to(DEV).requires_grad_(True) for n in LEAVES}
    _, fin = gated_delta_fn(*(d[n] for n in LEAVES[:5]), None, d["init"], return_final_states=True)
    (gi,) = torch.autograd.grad(fin.sum(), [d["init"]])
    want = oracle.delta_all(t, torch.ones(2, 2, 64, 32))
    oracle.delta_close(gi, want["init"], "init", t)


@pytest.mark.parametrize("dtype", [BF, F])
def test_chunks_continue(dtype):
    """A prompt in pieces, the states carried: the whole prompt's outputs, cut at other places."""
    t = make(20, T=201, dtype=dtype, grad=False)
    whole = run(t)
    state, outs = None, []
    for lo, hi in ((0, 1), (1, 70), (70, 134), (134, 201)):
        part = {n: x if x is None or n in ("init", "seq") else x[:, lo:hi] for n, x in t.items()}
        got = run(dict(part, init=state))
        outs.append(got["out"])
        state = got["final"]
    want = oracle.delta_all(t)
    oracle.delta_close(torch.cat(outs, 1), want["out"], "out", t)
    oracle.delta_close(state, whole["final"].double().cpu(), "final", t)


@pytest.mark.parametrize("dtype", [BF, F])
def test_against_differences(dtype):
    """A step along a direction changes the loss as the gradients say: differences of the operator's own fp32
    outputs would drown, so those of the definition in 64 bits."""
    t = make(21, B=1, T=40, Hk=1, H=2, Dk=16, Dv=16, dtype=dtype, init=True)
    got = run(t)
    gen = torch.Generator().manual_seed(2)
    for n in LEAVES:
        step = torch.randn(t[n].shape, generator=gen, dtype=torch.float64)
        loss = []
        for sign in (1, -1):
            moved = {m: None if x is None else x.double() for m, x in t.items()}
            moved[n] = moved[n] + sign * 1e-5 * step
            out, _ = oracle.delta(*(moved[m] for m in LEAVES[:5]), None, moved["init"])
            loss.append((out * moved["do"]).sum())
        slope, said = float(loss[0] - loss[1]) / 2e-5, float((got[n].double().cpu() * step).sum())
        # each element is off by half a step of its type at most, added without cancelling at worst
        room = float((got[n].double().cpu().abs() * step.abs()).sum()) * oracle.UNIT[got[n].dtype] * 2 + 1e-4 * abs(slope)
        assert abs(slope - said) <= room + 1e-3, (n, slope, said)


def test_deterministic_across_streams_and_graphs():
    t = {n: x if x is None else x.to(DEV) for n, x in make(22, T=300, H=4, Dv=100, packed=True, init=True).items()}

    @torch.enable_grad()
    def once():
        leaves = [t[n].detach().requires_grad_(True) for n in LEAVES]
        out, fin = gated_delta_fn(*leaves[:5], t["seq"], leaves[5], return_final_states=True)
        return [out.detach(), fin.detach(), *torch.autograd.grad(out, leaves, t["do"])]

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = once()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, again):
        assert torch.equal(a, b)
    with torch.no_grad():
        args = [t[n] for n in LEAVES[:5]]
        gated_delta_fn(*args, t["seq"], t["init"], return_final_states=True)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, fin = gated_delta_fn(*args, t["seq"], t["init"], return_final_states=True)
        for i in range(4):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, first[0]) and torch.equal(fin, first[1]), i
            once()
            torch.cuda.synchronize()
        t["v"].mul_(2)
        graph.replay()
        want = gated_delta_fn(*args, t["seq"], t["init"])
        assert torch.equal(out, want)


def test_compiled():
    t = {n: x if x is None else x.to(DEV) for n, x in make(23, T=130, packed=True, init=True).items()}

    def f(q, k, v, g, beta, init):
        out, fin = gated_delta_fn(q, k, v, g, beta, t["seq"], init, return_final_states=True)
        return out * 2, fin

    res = []
    for fn in (f, torch.compile(f, backend="aot_eager", fullgraph=True)):
        leaves = [t[n].detach().requires_grad_(True) for n in LEAVES]
        out, fin = fn(*leaves)
        res.append([out, fin, *torch.autograd.grad([out, fin], leaves, [t["do"], torch.ones_like(fin)])])
    for a, b in zip(*res):
        assert torch.equal(a, b)


def test_second_derivatives_are_refused():
    t = make(24, T=20)
    leaves = [t[n].to(DEV).requires_grad_(True) for n in LEAVES[:5]]
    out = gated_delta_fn(*leaves)
    (g,) = torch.autograd.grad(out.float().square().sum(), leaves[:1], create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        g.float().sum().backward()


def test_gradients_of_some_inputs_and_twice():
    t = {n: x if x is None else x.to(DEV) for n, x in make(25, T=100).items()}
    full = run(make(25, T=100))
    v = t["v"].requires_grad_(True)
    out = gated_delta_fn(t["q"], t["k"], v, t["g"], t["beta"])
    a = torch.autograd.grad(out, v, t["do"], retain_graph=True)[0]
    b = torch.autograd.grad(out, v, t["do"])[0]
    assert torch.equal(a, b) and torch.equal(a, full["v"])


def test_offsets_past_32_bits():
    """A batch whose values lie past 2^31 elements of their start."""
    B, T, H, Dv = 3, 70, 2, 32
    t = make(26, B=B, T=T, H=H, Dv=Dv, grad=False)
    stride = (1 << 30) + (1 << 27)
    room = torch.empty(2 * stride + T * H * Dv, dtype=BF, device=DEV)
    v = room.as_strided((B, T, H, Dv), (stride, H * Dv, Dv, 1))
    v.copy_(t["v"])
    with torch.no_grad():
        out = gated_delta_fn(*(t[n].to(DEV) for n in ("q", "k")), v, t["g"].to(DEV), t["beta"].to(DEV))
    assert torch.equal(out, run(t)["out"])


# ------------------------------------------------------------------------------- one token


def update_inputs(seed, R, Hk, H, Dk, Dv, dtype, pool):
    t = make(seed, B=1, T=R, Hk=Hk, H=H, Dk=Dk, Dv=Dv, dtype=dtype, grad=False)
    gen = torch.Generator().manual_seed(seed + 1)
    d = {n: t[n][0] for n in LEAVES[:5]}
    d["state"] = torch.randn(pool, H, Dk, Dv, generator=gen)
    d["idx"] = torch.randperm(pool, generator=gen)[:R].int()
    return d


@pytest.mark.parametrize("R,Hk,H,Dk,Dv", [(1, 1, 1, 1, 1), (3, 1, 2, 64, 64), (5, 2, 4, 128, 128), (2, 1, 1, 256, 100),
                                          (4, 3, 3, 65, 67), (40, 2, 2, 100, 130)])
@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_update(R, Hk, H, Dk, Dv, dtype):
    d = update_inputs(R + Dk, R, Hk, H, Dk, Dv, dtype, R + 3)
    state = d["state"].to(DEV)
    with torch.no_grad():
        out = gated_delta_update(*(d[n].to(DEV) for n in LEAVES[:5]), state, d["idx"].to(DEV))
    at = d["idx"].long()
    t = {n: d[n][:, None] for n in LEAVES[:5]}
    want = oracle.delta_all(dict(t, init=d["state"][at]))
    oracle.delta_close(out[:, None], want["out"], "out", dict(t, init=d["state"][at]))
    oracle.delta_close(state[at.to(DEV)], want["final"], "final", dict(t, init=d["state"][at]))
    left = torch.ones(R + 3, dtype=torch.bool)
    left[at] = False
    assert torch.equal(state.cpu()[left], d["state"][left])


def test_update_without_indices_and_outside_the_pool():
    d = update_inputs(3, 6, 2, 2, 64, 48, BF, 6)
    args = [d[n].to(DEV) for n in LEAVES[:5]]
    with torch.no_grad():
        a, b = d["state"].to(DEV), d["state"].to(DEV)
        assert torch.equal(gated_delta_update(*args, a), gated_delta_update(*args, b, torch.arange(6, device=DEV)))
        assert torch.equal(a, b)
        c = d["state"].to(DEV)
        idx = torch.tensor([-1, 2, 6, 4, 1 << 40, -(1 << 40)], device=DEV)
        out = gated_delta_update(*(x if i else x for i, x in enumerate(args)), c, idx)
        assert not out[[0, 2, 4, 5]].any() and out[[1, 3]].all(-1).any()
        assert torch.equal(c[[0, 1, 3, 5]].cpu(), d["state"][[0, 1, 3, 5]])
        e = d["state"].to(DEV)
        assert gated_delta_update(*(x[:0] for x in args), e).shape == (0, 2, 48)
        assert torch.equal(e.cpu(), d["state"])


def test_update_of_a_strided_pool_and_slices():
    d = update_inputs(4, 4, 2, 4, 72, 40, BF, 7)
    args = [d[n].to(DEV) for n in LEAVES[:5]]
    room = torch.zeros(7, 2, 4, 72, 40, device=DEV)
    pool = room[:, 1]
    pool.copy_(d["state"])
    plain = d["state"].to(DEV)
    wide = torch.cat([x.flatten(1) for x in args[:3]], 1)
    parts = [x.unflatten(1, (h, -1)) for x, h in zip(wide.split([144, 144, 160], 1), (2, 2, 4))]
    with torch.no_grad():
        a = gated_delta_update(*args, plain, d["idx"].to(DEV))
        b = gated_delta_update(*parts, args[3].t().contiguous().t(), args[4], pool, d["idx"].long().to(DEV))
    assert torch.equal(a, b) and torch.equal(plain, pool) and not room[:, 0].any()


@pytest.mark.parametrize("g", [-math.inf, -1000.0])
def test_update_empties_the_state(g):
    """A decay of zero leaves nothing of the state, whatever it held."""
    d = update_inputs(5, 2, 1, 1, 64, 64, F, 2)
    d["g"][:] = g
    bad = torch.full_like(d["state"], math.nan).to(DEV)
    with torch.no_grad():
        out = gated_delta_update(*(d[n].to(DEV) for n in LEAVES[:5]), bad)
    t = {n: d[n][:, None] for n in LEAVES[:5]}
    want = oracle.delta_all(dict(t, g=torch.zeros_like(t["g"])))
    oracle.delta_close(out[:, None], want["out"], "out", t)
    oracle.delta_close(bad, want["final"], "final", t)


@pytest.mark.parametrize("dtype", [BF, F])
def test_tokens_one_by_one(dtype):
    """A prompt, then tokens: the states and outputs of the whole sequence."""
    t = make(27, B=3, T=80, Hk=1, H=2, dtype=dtype, grad=False)
    want = oracle.delta_all(t)
    state = torch.zeros(5, 2, 64, 32, device=DEV)
    slots = torch.tensor([4, 0, 2], device=DEV, dtype=torch.int32)
    head = run({n: x if x is None else x[:, :70] for n, x in t.items()})
    state[slots.long()] = head["final"]
    outs = [head["out"]]
    with torch.no_grad():
        for s in range(70, 80):
            outs.append(gated_delta_update(*(t[n][:, s].to(DEV) for n in LEAVES[:5]), state, slots)[:, None])
    oracle.delta_close(torch.cat(outs, 1), want["out"], "out", t)
    oracle.delta_close(state[slots.long()], want["final"], "final", t)


def test_update_in_a_graph():
    d = update_inputs(6, 8, 2, 4, 128, 128, BF, 12)
    args = [d[n].to(DEV) for n in LEAVES[:5]]
    idx = d["idx"].to(DEV)
    state, eager = d["state"].to(DEV), d["state"].to(DEV)
    with torch.no_grad():
        warm = state.clone()
        gated_delta_update(*args, warm, idx)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = gated_delta_update(*args, state, idx)
        for _ in range(4):
            graph.replay()
            want = gated_delta_update(*args, eager, idx)
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(state, eager)


def test_in_place_writes_count():
    d = update_inputs(7, 2, 1, 1, 64, 64, BF, 2)
    state = d["state"].to(DEV)
    before = state._version
    with torch.no_grad():
        gated_delta_update(*(d[n].to(DEV) for n in LEAVES[:5]), state)
    assert state._version > before
