"""The gated linear recurrence on the GPU against its definition in 64 bits (tests/ops_oracle.py, which
also derives the bounds), forward and backward: types, sizes from one row and one channel on, odd
channel counts, strides, packed sequences and padding, states, streams and graphs."""

import pytest
import torch

import ops_oracle as oracle
from causal_conv1d_triton import causal_conv1d_fn
from causal_conv1d_triton.recurrence import gated_recurrence_fn, gated_recurrence_update

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


def make(seed, B, T, D, dtype, decay=True, igate=True, packed=False, init=False, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t = {"x": n(B, T, D).to(dtype), "gate": (spread * n(B, T, D) + (0 if decay else 1)).to(dtype),
         "decay": None, "igate": (spread * n(B, T, D)).to(dtype) if igate else None, "seq": None,
         "init": n(B, D) if init else None, "dy": n(B, T, D).to(dtype)}
    if decay:
        keep = 0.9 + 0.0999 * torch.rand(D, generator=g)
        t["decay"] = torch.log(torch.expm1(-torch.log(keep) / 8))
    if packed:
        seq = torch.zeros(B, T, dtype=torch.int32)
        for b in range(B):
            cuts = torch.randint(0, T + 1, (5,), generator=g).sort().values.tolist()
            for j, c in enumerate(cuts):
                seq[b, c:] = j + 1
            seq[b, T - T // 10:] = -1
            if T > 20:
                seq[b, cuts[2]:cuts[2] + 3] = -1
        t["seq"] = seq
    return t


def run(t, final=False, dfinal=None, train=True):
    d = {k: None if v is None else v.to(DEV) for k, v in t.items()}
    leaves = [k for k in ("x", "gate", "decay", "igate", "init") if d[k] is not None]
    if train:
        for k in leaves:
            d[k].requires_grad_(True)
    res = gated_recurrence_fn(d["x"], d["gate"], d["decay"], d["igate"], d["seq"], d["init"],
                              return_final_states=final)
    out, fin = res if final else (res, None)
    got = {"out": out, "final": fin}
    if train:
        outs, gs = [out], [d["dy"]]
        if dfinal is not None:
            outs.append(fin)
            gs.append(dfinal.to(DEV))
        got.update(zip(leaves, torch.autograd.grad(outs, [d[k] for k in leaves], gs)))
    return got


def check(t, final=False, dfinal=None, train=True):
    got = run(t, final, dfinal, train)
    want = oracle.recurrence(t["x"], t["gate"], t["decay"], t["igate"], t["seq"], t["init"],
                             dy=t["dy"] if train else None, dfinal=dfinal)
    for k, v in got.items():
        if v is not None:
            oracle.assert_close(v, want[k], k)


LENGTHS = [1, 2, 3, 31, 63, 64, 65, 127, 128, 129, 255, 257, 700, 1030, 2500]


@pytest.mark.parametrize("T", LENGTHS)
@pytest.mark.parametrize("dtype", [BF, F])
def test_lengths(T, dtype):
    check(make(T, 2, T, 70, dtype, init=T % 2 == 1))


@pytest.mark.parametrize("D", [1, 2, 3, 5, 63, 64, 65, 127, 128, 130, 257, 1000])
@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_channels(D, dtype):
    check(make(D, 2, 150, D, dtype, init=True))


@pytest.mark.parametrize("decay", [True, False])
@pytest.mark.parametrize("igate", [True, False])
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_variants(decay, igate, packed, dtype):
    t = make(7, 3, 333, 66, dtype, decay, igate, packed, init=True)
    dfin = torch.randn(3, 66, generator=torch.Generator().manual_seed(1))
    check(t, final=True, dfinal=dfin)


def test_long():
    check(make(3, 1, 20001, 3, F, init=True), final=True)
    check(make(4, 1, 9000, 130, BF, packed=True))


def test_many_rows():
    check(make(5, 300, 9, 130, BF, init=True), final=True)


@pytest.mark.parametrize("decay", [True, False])
def test_wide_gates(decay):
    """Gates far into saturation: a near 0 and near 1, where beta and 1 - r cancel in a plain form."""
    check(make(6, 2, 200, 66, F, decay=decay, spread=6.0, init=True))


@pytest.mark.parametrize("decay", [True, False])
@pytest.mark.parametrize("igate", [True, False])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_wide_gates_of_16_bits(decay, igate, dtype):
    check(make(16, 2, 200, 66, dtype, decay, igate, spread=6.0, init=True))


# A gate far below zero counts as 2^-126 in some of the forms, and the root of that, 2^-63, is the largest
# trace of it in beta and the gradients; the other factors here (states, x, dout, the decay's exponent)
# stay below 2^5 each, three of them in a product.
CLOSED = 2.0 ** -48


@pytest.mark.parametrize("decay", [True, False])
@pytest.mark.parametrize("igate", [True, False])
@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_gates_at_the_ends_of_their_type(decay, igate, dtype):
    """Gates that are infinite or their type's largest and lowest value, as masks are: sigmoid is 1 or 0
    there, forward and backward, and in the form for one token."""
    ends = torch.tensor([float("inf"), float("-inf"), torch.finfo(dtype).max, torch.finfo(dtype).min])
    t = make(19, 2, 150, 70, dtype, decay, igate, init=True)
    g = torch.Generator().manual_seed(4)
    for k in ("gate", "igate"):
        if t[k] is not None:
            at = torch.rand(t[k].shape, generator=g) < 0.2
            t[k][at] = ends[torch.randint(0, 4, (int(at.sum()),), generator=g)].to(dtype)
    dfin = torch.randn(2, 70, generator=g)
    want = oracle.recurrence(t["x"], t["gate"], t["decay"], t["igate"], None, t["init"], dy=t["dy"], dfinal=dfin)
    for k, v in run(t, final=True, dfinal=dfin).items():
        if v is not None:
            oracle.assert_close(v, (want[k][0], want[k][1] + CLOSED), k)
    state = t["init"].to(DEV)
    d = {k: None if v is None else v.to(DEV) for k, v in t.items()}
    for j in range(20):
        out = gated_recurrence_update(d["x"][:, j], d["gate"][:, j], state, d["decay"],
                                      None if d["igate"] is None else d["igate"][:, j])
        oracle.assert_close(out, (want["out"][0][:, j], want["out"][1][:, j] + CLOSED))


@pytest.mark.parametrize("decay", [True, False])
@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_gates_that_are_no_numbers(dtype, decay):
    """They reach the rows that the formulas lead to, forward and backward, and the rest keeps its bits."""
    t = make(23, 2, 150, 70, dtype, decay, init=True)
    t["seq"] = (torch.arange(150) // 40).int().expand(2, 150).contiguous()
    clean = run(t)
    t["gate"][0, 20, 5] = t["igate"][1, 30, 6] = float("nan")
    got = run(t)
    where = {k: torch.zeros(2, 150, 70, dtype=torch.bool) for k in ("out", "x", "gate", "igate")}
    where["out"][0, 20:40, 5] = where["out"][1, 30:40, 6] = True  # the state from the row on
    where["x"][0, :21, 5] = True  # the incoming gradient up to the row, and beta in it
    where["x"][1, 30, 6] = where["igate"][1, 30, 6] = True  # i alone
    where["gate"][0, :40, 5] = where["gate"][1, 30:40, 6] = True  # the state before, or the gradient
    where["igate"][0, :21, 5] = True
    for k, bad in where.items():
        v, ref = got[k].cpu(), clean[k].cpu()
        assert v[bad].isnan().all(), k
        assert torch.equal(v[~bad], ref[~bad]), k
    assert got["init"][0, 5].isnan() and got["init"].isnan().sum() == 1


@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_decay_that_never_forgets(dtype):
    """A decay of -infinity or the lowest number: softplus is 0, a is 1, beta 0 and so is its gradient."""
    t = make(20, 2, 150, 70, dtype, init=True)
    ends = [0, 1, 33, 69]
    t["decay"][ends] = torch.tensor([float("-inf"), torch.finfo(F).min, float("-inf"), -200.0])
    got = run(t, final=True)
    want = oracle.recurrence(t["x"], t["gate"], t["decay"], t["igate"], None, t["init"], dy=t["dy"])
    live = torch.ones(70, dtype=torch.bool)
    live[ends] = False
    assert not got["decay"].cpu()[~live].any()
    for k, v in got.items():
        value, bound = want[k]
        if k == "decay":  # the oracle divides by the softplus
            oracle.assert_close(v.cpu()[live], (value[live], bound[live]), k)
        else:
            oracle.assert_close(v, (value, bound + CLOSED), k)
    state = t["init"].to(DEV)
    out = gated_recurrence_update(t["x"][:, 0].to(DEV), t["gate"][:, 0].to(DEV), state, t["decay"].to(DEV),
                                  t["igate"][:, 0].to(DEV))
    oracle.assert_close(out, (want["out"][0][:, 0], want["out"][1][:, 0] + CLOSED))


@pytest.mark.parametrize("B,T", [(128, 129), (128, 200), (130, 256), (127, 256), (128, 257)])
@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("packed", [True, False])
def test_around_one_chunk(B, T, dtype, packed):
    """Lengths and batches on both sides of the rule that takes 256 rows in one chunk."""
    t = make(17, B, T, 6, dtype, packed=packed, init=True)
    check(t, final=True, dfinal=torch.randn(B, 6, generator=torch.Generator().manual_seed(2)))


@pytest.mark.parametrize("D", [66, 129])
def test_strides(D):
    """Slices of one projection, an upstream gradient and gates with strides of their own."""
    t = make(8, 3, 140, D, BF, init=True)
    got = run(t)
    wide = torch.randn(3, 140, 4 * D + 3, device=DEV).to(BF)
    wide[..., 1:1 + D], wide[..., D + 1:2 * D + 1] = t["x"].to(DEV), t["gate"].to(DEV)
    wide[..., 2 * D + 2:3 * D + 2] = t["igate"].to(DEV)
    wide.requires_grad_(True)
    dec, init = t["decay"].to(DEV), t["init"].to(DEV)
    out = gated_recurrence_fn(wide[..., 1:1 + D], wide[..., D + 1:2 * D + 1], dec,
                              wide[..., 2 * D + 2:3 * D + 2], None, init)
    dy = torch.empty(140, 3, 2 * D, device=DEV, dtype=BF).transpose(0, 1)[..., ::2]
    dy.copy_(t["dy"])
    (dw,) = torch.autograd.grad(out, [wide], dy)
    assert torch.equal(out, got["out"])
    assert torch.equal(dw[..., 1:1 + D], got["x"])
    assert torch.equal(dw[..., D + 1:2 * D + 1], got["gate"])
    assert torch.equal(dw[..., 2 * D + 2:3 * D + 2], got["igate"])
    # time-major storage and a broadcast upstream gradient (the gradient of a sum)
    xt = t["x"].to(DEV).transpose(0, 1).contiguous().transpose(0, 1)
    out2 = gated_recurrence_fn(xt, t["gate"].to(DEV), dec, t["igate"].to(DEV), None, init)
    assert torch.equal(out2, got["out"])
    x = t["x"].to(DEV).requires_grad_(True)
    gated_recurrence_fn(x, t["gate"].to(DEV), dec, t["igate"].to(DEV), None, init).sum().backward()
    t["dy"] = torch.ones_like(t["dy"])
    assert torch.equal(x.grad, run(t)["x"])


def test_types_of_side_tensors():
    t = make(9, 2, 40, 64, BF, init=True)
    dec = t["decay"].to(DEV).to(BF).requires_grad_(True)
    init = t["init"].to(DEV).to(HF).requires_grad_(True)
    x = t["x"].to(DEV)
    out = gated_recurrence_fn(x, t["gate"].to(DEV), dec, t["igate"].to(DEV),
                              torch.zeros(2, 40, dtype=torch.int64, device=DEV), init)
    gd, gi = torch.autograd.grad(out, [dec, init], t["dy"].to(DEV))
    assert gd.dtype == BF and gi.dtype == HF
    want = oracle.recurrence(t["x"], t["gate"], t["decay"].to(BF), t["igate"], None,
                             t["init"].to(HF), dy=t["dy"])
    oracle.assert_close(gd, want["decay"])
    oracle.assert_close(gi, want["init"])


def test_empty():
    for B, T, D in ((0, 5, 8), (2, 5, 0), (2, 0, 8)):
        t = make(1, B, T, D, BF, init=True)
        dfin = torch.randn(B, D, generator=torch.Generator().manual_seed(2))
        got = run(t, final=True, dfinal=dfin)
        assert got["out"].shape == (B, T, D) and got["final"].shape == (B, D)
        assert got["x"].shape == (B, T, D)
        if T == 0:
            assert torch.equal(got["final"].cpu(), t["init"])
            assert torch.equal(got["init"].cpu(), dfin)
        assert not got["decay"].any()


def test_final_state_gradient_alone():
    t = make(2, 2, 100, 64, F, init=True)
    d = {k: None if v is None else v.to(DEV) for k, v in t.items()}
    d["x"].requires_grad_(True)
    dfin = torch.randn(2, 64, generator=torch.Generator().manual_seed(3))
    _, fin = gated_recurrence_fn(d["x"], d["gate"], d["decay"], d["igate"], None, d["init"], True)
    (dx,) = torch.autograd.grad(fin, [d["x"]], dfin.to(DEV))
    want = oracle.recurrence(t["x"], t["gate"], t["decay"], t["igate"], None, t["init"],
                             dy=torch.zeros_like(t["dy"]), dfinal=dfin)
    oracle.assert_close(dx, want["x"])


@pytest.mark.parametrize("decay", [True, False])
def test_values_in_padding_and_other_sequences_stay_there(decay):
    """NaN and infinities in padding change nothing; those of one sequence reach its own later rows
    (and, backwards, its earlier ones) and no other sequence or channel."""
    t = make(10, 2, 400, 70, BF, decay=decay, init=True)
    seq = torch.zeros(2, 400, dtype=torch.int32)
    seq[:, 130:] = 1
    seq[:, 150:180] = -1
    seq[:, 180:] = 2
    t["seq"] = seq
    clean = run(t)
    for bad in (float("nan"), float("inf"), torch.finfo(BF).min):
        u = {k: None if v is None else v.clone() for k, v in t.items()}
        for k in ("x", "gate", "igate", "dy"):
            u[k][:, 150:180] = bad
        got = run(u)
        for k, v in clean.items():
            assert v is None or torch.equal(got[k], v), (bad, k)
        assert not got["out"][:, 150:180].any() and not got["gate"][:, 150:180].any()
    u = {k: None if v is None else v.clone() for k, v in t.items()}
    u["x"][0, 20, 5] = float("nan")
    u["x"][1, 200, 6] = float("inf")
    u["dy"][0, 300, 7] = float("nan")
    got = run(u)
    out, ref = got["out"].float().cpu(), clean["out"].float().cpu()
    assert out[0, 20:130, 5].isnan().all() and out[1, 200:, 6].isinf().all()
    hit = torch.zeros(2, 400, 70, dtype=torch.bool)
    hit[0, 20:130, 5] = hit[1, 200:, 6] = True
    assert torch.equal(out[~hit], ref[~hit])
    dx, ref = got["x"].float().cpu(), clean["x"].float().cpu()
    assert dx[0, 180:301, 7].isnan().all()
    hit[:] = False
    hit[0, 180:301, 7] = True
    assert torch.equal(dx[~hit], ref[~hit])


@pytest.mark.parametrize("T", [9, 150, 1200])
@pytest.mark.parametrize("decay", [True, False])
def test_ids_of_64_bits(T, decay):
    """Ids that 32 bits cannot hold or tell apart: the bits of the same sequences under small ids."""
    t = make(21, 2, T, 70, BF, decay=decay, init=True)
    big = [2 ** 31, 2 ** 32 + 2 ** 31, 5, 5 + 2 ** 32, 5 + 2 ** 33, -1, 2 ** 32 - 1, -2 ** 32, 2 ** 62, 0, -2 ** 63]
    small = torch.full((2, T), 0, dtype=torch.int32)
    wide = torch.full((2, T), big[0], dtype=torch.int64)
    for b in range(2):
        cuts = [0, *(torch.randint(1, T, (len(big) - 1,), generator=torch.Generator().manual_seed(b)).sort()
                     .values.tolist())]
        for j, (c, n) in enumerate(zip(cuts, big)):
            wide[b, c:] = n
            small[b, c:] = j if n >= 0 else -1
    dfin = torch.randn(2, 70, generator=torch.Generator().manual_seed(3))
    t["seq"] = small
    want = run(t, final=True, dfinal=dfin)
    t["seq"] = wide
    got = run(t, final=True, dfinal=dfin)
    for k, v in want.items():
        assert v is None or torch.equal(got[k], v), k
    t["seq"] = wide.repeat(1, 2)[:, ::2].contiguous()  # the forward alone, from ids with strides
    wide2 = torch.stack([t["seq"], t["seq"] + 1], 2).to(DEV)[..., 0]
    t["seq"] = None
    d = {k: None if v is None else v.to(DEV) for k, v in t.items()}
    args = (d["x"], d["gate"], d["decay"], d["igate"])
    assert torch.equal(gated_recurrence_fn(*args, wide2, d["init"]),
                       gated_recurrence_fn(*args, wide2.contiguous(), d["init"]))


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.uint32])
def test_ids_of_other_types(dtype):
    t = make(22, 2, 150, 70, BF)
    ids = torch.tensor([100, 3, 0, 127, 4])[torch.arange(150) // 32].expand(2, 150)
    t["seq"] = ids.int()
    want = run(t, train=False)["out"]
    if dtype == torch.uint32:
        ids = ids + 2 ** 31
    t["seq"] = ids.to(dtype)
    assert torch.equal(run(t, train=False)["out"], want)


def test_all_padding():
    t = make(11, 2, 100, 64, BF, init=True)
    t["seq"] = torch.full((2, 100), -1, dtype=torch.int32)
    got = run(t, final=True, dfinal=torch.ones(2, 64))
    for k, v in got.items():
        assert v is None or not v.any(), k


def test_chunks_continue():
    """A sequence cut at any row, its state handed over, is the whole one's up to the rounding of the
    carried sums; one row at a time too."""
    t = make(12, 2, 300, 66, F)
    d = {k: None if v is None else v.to(DEV) for k, v in t.items()}
    want = oracle.recurrence(t["x"], t["gate"], t["decay"], t["igate"])
    for cuts in ([0, 1, 130, 300], list(range(0, 301, 7)) + [300]):
        state, outs = None, []
        for a, b in zip(cuts[:-1], cuts[1:]):
            o, state = gated_recurrence_fn(d["x"][:, a:b], d["gate"][:, a:b], d["decay"],
                                           d["igate"][:, a:b], None, state, True)
            outs.append(o)
        oracle.assert_close(torch.cat(outs, 1), want["out"])
        oracle.assert_close(state, want["final"])


def test_deterministic_across_streams_and_graphs():
    t = make(13, 2, 1500, 192, BF, packed=True, init=True)
    ref = run(t)
    side = torch.cuda.Stream()
    for _ in range(3):
        got = run(t)
        with torch.cuda.stream(side):
            other = run(t)
        side.synchronize()
        for k, v in ref.items():
            assert v is None or (torch.equal(got[k], v) and torch.equal(other[k], v)), k
    d = {k: None if v is None else v.to(DEV) for k, v in t.items()}
    leaves = [d[k].requires_grad_(True) for k in ("x", "gate", "decay", "igate", "init")]

    def step():
        out = gated_recurrence_fn(d["x"], d["gate"], d["decay"], d["igate"], d["seq"], d["init"])
        return (out, *torch.autograd.grad(out, leaves, d["dy"]))

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = step()
    names = ("out", "x", "gate", "decay", "igate", "init")
    for i in range(4):
        with torch.no_grad():
            d["x"].copy_(t["x"].roll(i, 0))
        for o in outs:
            o.detach().fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        u = dict(t, x=t["x"].roll(i, 0))
        for k, o in zip(names, outs):
            assert torch.equal(o, run(u)[k]), (i, k)


def test_after_the_convolution_compiled():
    """The block that the two operators make, compiled without a graph break: the eager bits."""
    t = make(14, 2, 200, 64, BF)
    w = (torch.randn(64, 4, generator=torch.Generator().manual_seed(1)) / 2).to(DEV)
    d = {k: None if v is None else v.to(DEV) for k, v in t.items()}

    def block(x, gate, decay, igate):
        return gated_recurrence_fn(causal_conv1d_fn(x, w), gate, decay, igate,
                                   return_final_states=True)

    def grads(fn):
        leaves = [d[k].detach().requires_grad_(True) for k in ("x", "gate", "decay", "igate")]
        out, fin = fn(*leaves)
        return (out, fin, *torch.autograd.grad(out, leaves, d["dy"]))

    for a, b in zip(grads(block), grads(torch.compile(block, fullgraph=True))):
        assert torch.equal(a, b)


def test_registered_operators():
    """Schema, fake implementations, autograd registration and AOT dispatch of the two operators."""
    from causal_conv1d_triton import recurrence
    t = make(15, 2, 130, 66, BF, packed=True, init=True)
    d = {k: None if v is None else v.to(DEV) for k, v in t.items()}
    for k in ("x", "gate", "decay", "igate", "init"):
        d[k].requires_grad_(True)
    torch.library.opcheck(recurrence._fwd_op, (d["x"], d["gate"], d["decay"], d["igate"], d["seq"],
                                               d["init"], 8.0))
    torch.library.opcheck(recurrence._fwd_op, (d["x"], d["gate"], None, None, None, None, 8.0))


def test_second_derivatives_are_refused():
    x = torch.randn(1, 5, 8, device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad(gated_recurrence_fn(x, x).square().sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_second_derivatives_are_refused_where_the_incoming_gradient_is_a_constant():
    """The gradient still depends on x, so a sum with x must not leave that part out silently."""
    x = torch.randn(1, 5, 8, device=DEV, requires_grad=True)
    h0 = torch.randn(1, 8, device=DEV, requires_grad=True)
    out, fin = gated_recurrence_fn(x, x, initial_states=h0, return_final_states=True)
    g, gh = torch.autograd.grad(out.sum() + fin.sum(), [x, h0], create_graph=True)
    with pytest.raises(RuntimeError):
        ((g * x).sum() + gh.sum()).backward()


def test_gradients_of_some_inputs_and_twice():
    """A graph that is kept gives the same bits again; gradients of a part of the inputs are those of all."""
    t = make(16, 2, 130, 66, BF, init=True)
    d = {k: None if v is None else v.to(DEV) for k, v in t.items()}
    names = ("x", "gate", "decay", "igate", "init")
    for k in names:
        d[k].requires_grad_(True)
    out = gated_recurrence_fn(d["x"], d["gate"], d["decay"], d["igate"], None, d["init"])
    every = torch.autograd.grad(out, [d[k] for k in names], d["dy"], retain_graph=True)
    for k, g in zip(names, every):
        (again,) = torch.autograd.grad(out, [d[k]], d["dy"], retain_graph=True)
        assert again.dtype == d[k].dtype and torch.equal(again, g)
    with torch.no_grad():
        d["x"].mul_(2)
    with pytest.raises(RuntimeError):  # an input that was changed since
        torch.autograd.grad(out, [d["gate"]], d["dy"])


@pytest.mark.parametrize("R,D", [(1, 1), (1, 130), (5, 66), (16, 2048), (300, 97)])
@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("decay", [True, False])
def test_update(R, D, dtype, decay):
    t = make(R + D, R, 1, D, dtype, decay=decay, igate=R != 5)
    g = torch.Generator().manual_seed(1)
    pool = torch.randn(R + 3, D, generator=g)
    idx = torch.randperm(R + 3, generator=g)[:R].to(torch.int32)
    state = pool.to(DEV)
    ig = None if t["igate"] is None else t["igate"][:, 0].to(DEV)
    dec = None if t["decay"] is None else t["decay"].to(DEV)
    out = gated_recurrence_update(t["x"][:, 0].to(DEV), t["gate"][:, 0].to(DEV), state, dec, ig,
                                  idx.to(DEV))
    want = oracle.recurrence(t["x"], t["gate"], t["decay"], t["igate"], None, pool[idx.long()])
    oracle.assert_close(out, (want["out"][0][:, 0], want["out"][1][:, 0]))
    oracle.assert_close(state[idx.long().to(DEV)], want["final"])
    rest = torch.ones(R + 3, dtype=torch.bool)
    rest[idx.long()] = False
    assert torch.equal(state.cpu()[rest], pool[rest])


def test_update_skips_rows_outside_the_pool():
    t = make(1, 6, 1, 70, BF)
    pool = torch.randn(4, 2 * 70, generator=torch.Generator().manual_seed(1))
    state = pool.to(DEV)[:, 3:73]  # rows with a stride and an odd start
    idx = torch.tensor([2, -1, 4, 0, 2 ** 32 + 1, -2 ** 32 + 1], dtype=torch.int64)
    out = gated_recurrence_update(t["x"][:, 0].to(DEV), t["gate"][:, 0].to(DEV), state,
                                  t["decay"].to(DEV), t["igate"][:, 0].to(DEV), idx.to(DEV))
    assert not out[[1, 2, 4, 5]].any()
    sel = [0, 3]
    want = oracle.recurrence(t["x"][sel], t["gate"][sel], t["decay"], t["igate"][sel], None,
                             pool[[2, 0], 3:73])
    oracle.assert_close(out[sel], (want["out"][0][:, 0], want["out"][1][:, 0]))
    oracle.assert_close(state[[2, 0]], want["final"])
    assert torch.equal(state[[1, 3]].cpu(), pool[[1, 3], 3:73])
    # every index that int32 can hold
    edge = torch.tensor([-1, 4, 2 ** 31 - 1, -2 ** 31, 5, -2], dtype=torch.int32, device=DEV)
    out = gated_recurrence_update(t["x"][:, 0].to(DEV), t["gate"][:, 0].to(DEV), state,
                                  state_indices=edge)
    assert not out.any() and torch.equal(state[[1, 3]].cpu(), pool[[1, 3], 3:73])
    # a write in place is one to autograd too
    version = state._version
    gated_recurrence_update(t["x"][:, 0].to(DEV), t["gate"][:, 0].to(DEV), state, state_indices=edge)
    assert state._version > version
    # without indices row r uses slot r
    state = pool.to(DEV)[:, :70].contiguous()
    gated_recurrence_update(t["x"][:4, 0].to(DEV), t["gate"][:4, 0].to(DEV), state)
    want = oracle.recurrence(t["x"][:4], t["gate"][:4], None, None, None, pool[:, :70])
    oracle.assert_close(state, want["final"])


@pytest.mark.parametrize("dtype", [torch.uint32, torch.uint64])
def test_update_with_unsigned_indices(dtype):
    """Those that int32 cannot hold lie outside the pool, whatever their low bits."""
    t = make(1, 4, 1, 70, BF)
    pool = torch.randn(4, 70, generator=torch.Generator().manual_seed(1))
    state = pool.to(DEV)
    far = 2 ** 32 - 1 if dtype == torch.uint32 else 2 ** 32 + 1
    idx = torch.tensor([2, far, 0, 2 ** 31], dtype=torch.int64).to(dtype).to(DEV)
    out = gated_recurrence_update(t["x"][:, 0].to(DEV), t["gate"][:, 0].to(DEV), state, state_indices=idx)
    want = oracle.recurrence(t["x"][[0, 2]], t["gate"][[0, 2]], None, None, None, pool[[2, 0]])
    oracle.assert_close(out[[0, 2]], (want["out"][0][:, 0], want["out"][1][:, 0]))
    assert not out[[1, 3]].any() and torch.equal(state[[1, 3]].cpu(), pool[[1, 3]])


def test_offsets_past_32_bits():
    """Batch rows, time rows and slots further apart than 32 bits of elements."""
    n = 2 ** 32 + 5 * 70
    store = torch.zeros(n, dtype=BF, device=DEV)
    t = make(18, 2, 5, 70, BF)
    d = {k: None if v is None else v.to(DEV) for k, v in t.items()}
    want = gated_recurrence_fn(d["x"], d["gate"], d["decay"], d["igate"])
    x = store.as_strided((2, 5, 70), (2 ** 32, 70, 1))
    x.copy_(d["x"])
    assert torch.equal(gated_recurrence_fn(x, d["gate"], d["decay"], d["igate"]), want)
    x = store.as_strided((1, 3, 70), (70, 2 ** 31, 1))
    x.copy_(d["x"][:1, :3])
    cut = [d[k][:1, :3] for k in ("gate", "igate")]
    assert torch.equal(gated_recurrence_fn(x, cut[0], d["decay"], cut[1]), want[:1, :3])
    pool = store[:2 ** 32].view(F).as_strided((2, 70), (2 ** 31 - 70, 1))
    pool.copy_(torch.ones(2, 70))
    small = pool.clone()
    args = (d["x"][:, 0], d["gate"][:, 0])
    idx = torch.tensor([1, 0], device=DEV)
    out = gated_recurrence_update(*args, pool, d["decay"], state_indices=idx)
    assert torch.equal(out, gated_recurrence_update(*args, small, d["decay"], state_indices=idx))
    assert torch.equal(pool, small)
