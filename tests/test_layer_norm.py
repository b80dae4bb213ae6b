"""The norms around a block on the GPU against their definition in 64 bits (tests/layer_oracle.py, which derives the
bounds), forward and backward: every combination of parts, row lengths around each launch's limits, types, strides
and broadcast inputs, extreme values, streams and graphs."""

import itertools
import math

import pytest
import torch

import layer_oracle as oracle
from causal_conv1d_triton.norm import block_norm_fn

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F = torch.bfloat16, torch.float16, torch.float32
NAMES = ("x", "residual", "post", "gate", "scale", "pre")


def make(seed, shape, dtype=BF, residual=None, post=False, gate=False, scale=None, pre=False, wtype=F, dy=True, dr=True):
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    D = shape[-1]
    t = {"x": n(*shape).to(dtype), "residual": n(*shape).to(residual) if residual else None,
         "post": (1 + 0.1 * n(D)).to(wtype) if post else None, "gate": n(*shape).to(dtype) if gate else None,
         "scale": (0.5 + 0.1 * n(D)).to(wtype) if scale == "tensor" else scale,
         "pre": (1 + 0.1 * n(D)).to(wtype) if pre else None}
    t["dr"] = n(*shape).to(residual or dtype) if dr else None
    t["dy"] = n(*shape).to(dtype) if dy and pre else None
    return t


def run(t, eps=1e-6, activation="silu"):
    d = {n: t[n].detach().to(DEV) if isinstance(t[n], torch.Tensor) else t[n] for n in (*NAMES, "dr", "dy")}
    grad = d["dr"] is not None or d["dy"] is not None
    names = [n for n in NAMES if isinstance(d[n], torch.Tensor)]
    if grad:
        for n in names:
            d[n].requires_grad_(True)
    res = block_norm_fn(*(d[n] for n in NAMES), eps=eps, activation=activation)
    y, r = res if d["pre"] is not None else (None, res)
    got = {"r": r.detach(), "y": None if y is None else y.detach()}
    if grad:
        outs, ups = zip(*((o, u) for o, u in ((r, d["dr"]), (y, d["dy"])) if u is not None))
        grads = torch.autograd.grad(outs, [d[n] for n in names], ups, allow_unused=True)
        got.update({"d" + n: g for n, g in zip(names, grads)})
    return got


def check(t, eps=1e-6, activation="silu"):
    got = run(t, eps, activation)
    want = oracle.norm_all(t, eps, activation)
    for n, x in got.items():
        if x is not None:
            oracle.norm_close(x, want[n], n, t)
    return got


@pytest.mark.parametrize("D", [1, 2, 7, 8, 9, 64, 127, 128, 129, 500, 512, 513, 2047, 2048, 2049, 4096, 4097, 8191, 8192])
@pytest.mark.parametrize("dtype,residual", [(BF, BF), (BF, F), (HF, HF), (HF, F), (F, F)])
def test_row_lengths(D, dtype, residual):
    check(make(D, (5, D), dtype, residual, True, True, "tensor", True))


PARTS = [p for p in itertools.product((None, "own", "fp32"), (False, True), (False, True), (None, 0.3, "tensor"),
                                      (False, True)) if p[1] or p[4]]


@pytest.mark.parametrize("residual,post,gate,scale,pre", PARTS)
def test_parts(residual, post, gate, scale, pre):
    check(make(1, (9, 200), BF, {None: None, "own": BF, "fp32": F}[residual], post, gate, scale, pre))


@pytest.mark.parametrize("dy,dr", [(True, False), (False, True)])
@pytest.mark.parametrize("post", [False, True])
def test_one_gradient_alone(dy, dr, post):
    check(make(2, (7, 130), BF, F, post, True, "tensor", True, dy=dy, dr=dr))


@pytest.mark.parametrize("activation", ["silu", "sigmoid", None])
@pytest.mark.parametrize("dtype", [BF, HF, F])
def test_activations(activation, dtype):
    t = make(3, (6, 96), dtype, None, True, True)
    t["gate"] = (t["gate"].float() * 4).to(dtype)
    check(t, activation=activation)


@pytest.mark.parametrize("wtype", [BF, HF, F])
def test_types_of_weights(wtype):
    got = check(make(4, (40, 300), BF, BF, True, True, "tensor", True, wtype=wtype))
    assert all(got["d" + n].dtype == wtype for n in ("post", "scale", "pre"))


@pytest.mark.parametrize("rows,D", [(1, 64), (15, 64), (16, 128), (17, 128), (3, 512), (5, 500), (1023, 300), (1025, 300),
                                    (5000, 40), (40000, 128), (2100, 2048)])
def test_numbers_of_rows(rows, D):
    """Below, at and above the workgroups that the backward has at most, and rows of a workgroup."""
    check(make(rows, (rows, D), BF, F, True, True, "tensor", True))


def test_shapes():
    for shape in ((30,), (3, 30), (2, 3, 30), (2, 1, 3, 30), (2, 2, 2, 3, 30), (0, 30), (2, 0, 30)):
        check(make(5, shape, BF, BF, True, True, "tensor", True))


@pytest.mark.parametrize("dtype", [BF, F])
def test_strides(dtype):
    """Heads as slices of a projection, transposed batches, gradients that autograd expands: the bits of contiguous
    copies."""
    t = {n: x.to(DEV) if isinstance(x, torch.Tensor) else x
         for n, x in make(6, (3, 17, 4, 40), dtype, dtype, True, True, "tensor", True).items()}
    wide = torch.cat([t["x"].flatten(2), t["gate"].flatten(2)], -1)
    odd = dict(t, x=wide[..., :160].unflatten(-1, (4, 40)), gate=wide[..., 160:].unflatten(-1, (4, 40)),
               residual=t["residual"].transpose(0, 1).contiguous().transpose(0, 1))
    res = []
    for d in (t, odd):
        leaves = [d[n].detach().requires_grad_(True) for n in NAMES]
        y, r = block_norm_fn(*leaves)
        res.append([y.detach(), r.detach(), *torch.autograd.grad([y, r], leaves, [t["dy"], t["dr"]])])
        res.append([y.detach(), r.detach(), *torch.autograd.grad(block_norm_fn(*leaves)[0].sum(), leaves)])
    for a, b in zip(res[0] + res[1], res[2] + res[3]):
        assert torch.equal(a, b)


def test_expanded_inputs():
    """A gate and a residual of one row for all: autograd adds their gradients over the rows."""
    t = make(7, (50, 64), F, F, True, True, None, True)
    g1, r1 = (t[n][:1].to(DEV).requires_grad_(True) for n in ("gate", "residual"))
    x, post, pre = (t[n].to(DEV) for n in ("x", "post", "pre"))
    y, r = block_norm_fn(x, r1.expand(50, -1), post, g1.expand(50, -1), None, pre)
    got = torch.autograd.grad([y, r], [g1, r1], [t["dy"].to(DEV), t["dr"].to(DEV)])
    t["gate"], t["residual"] = t["gate"][:1].expand(50, -1), t["residual"][:1].expand(50, -1)
    want = oracle.norm_all(t)
    for g, n in zip(got, ("dgate", "dresidual")):
        oracle.close(g, want[n].sum(0, keepdim=True), 50 * 64 * oracle.U * float(want[n].abs().max()), n)


def test_zero_rows_and_large_values():
    t = make(8, (6, 300), F, F, True, True, "tensor", True)
    t["x"][1] = 0
    t["x"][2] *= 1e15
    t["x"][3] *= 1e-15
    t["residual"][1] = 0
    check(t)


def test_gates_far_from_zero():
    """silu of large magnitudes is the gate itself, or zero; no number comes from an overflow."""
    t = make(9, (4, 64), BF, None, True, True)
    t["gate"][0], t["gate"][1], t["gate"][2], t["gate"][3] = 100.0, -100.0, 3e38, -1e38
    got = run(t)
    assert all(torch.isfinite(got[n][:2]).all() for n in ("r", "dx", "dgate"))
    assert not got["r"][1].any() and not got["r"][3].any()
    want = oracle.norm_all({n: x if x is None or not isinstance(x, torch.Tensor) or x.dim() < 2 else x[:2]
                            for n, x in t.items()})
    for n in ("r", "dx", "dgate"):
        oracle.norm_close(got[n][:2], want[n], n, t)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_rows_do_not_meet(bad):
    """A row that holds no number spoils itself alone (and the weights' sums)."""
    t = make(10, (33, 100), BF, F, True, True, "tensor", True)
    clean = run(t)
    t["x"][5, 7] = bad
    got = run(t)
    rest = [i for i in range(33) if i != 5]
    for n in ("r", "y", "dx", "dgate", "dresidual"):
        assert torch.equal(got[n][rest], clean[n][rest]), n


@pytest.mark.parametrize("shape", [(1, 8), (5, 64), (17, 128), (3, 512), (3, 1024)])
def test_no_eps_and_rows_that_fill_no_workgroup(shape):
    """Weights' sums take nothing of the rows behind the last, whose inverse norm would be infinite."""
    check(make(12, shape, F, F, True, True, "tensor", True), eps=0.0)


def test_eps():
    for eps in (0.0, 1e-3, 1.0):
        check(make(11, (5, 77), F, F, True, True, None, True), eps=eps)


@pytest.mark.parametrize("dtype", [BF, F])
def test_against_differences(dtype):
    t = make(12, (3, 40), dtype, F, True, True, "tensor", True)
    got = run(t)
    gen = torch.Generator().manual_seed(2)
    for n in NAMES:
        step = torch.randn(t[n].shape, generator=gen, dtype=torch.float64)
        loss = []
        for sign in (1, -1):
            moved = {m: t[m].double() for m in NAMES}
            moved[n] = moved[n] + sign * 1e-5 * step
            r, y = oracle.norm(**moved)
            loss.append((r * t["dr"]).sum() + (y * t["dy"]).sum())
        slope, said = float(loss[0] - loss[1]) / 2e-5, float((got["d" + n].double().cpu() * step).sum())
        room = float((got["d" + n].double().cpu().abs() * step.abs()).sum()) * oracle.UNIT[got["d" + n].dtype] * 2
        assert abs(slope - said) <= room + 1e-4 * abs(slope) + 1e-3, (n, slope, said)


def test_deterministic_across_streams_and_graphs():
    t = {n: x.to(DEV) if isinstance(x, torch.Tensor) else x
         for n, x in make(13, (700, 300), BF, F, True, True, "tensor", True).items()}

    @torch.enable_grad()
    def once():
        leaves = [t[n].detach().requires_grad_(True) for n in NAMES]
        y, r = block_norm_fn(*leaves)
        return [y.detach(), r.detach(), *torch.autograd.grad([y, r], leaves, [t["dy"], t["dr"]])]

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = once()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, again):
        assert torch.equal(a, b)
    with torch.no_grad():
        args = [t[n] for n in NAMES]
        block_norm_fn(*args)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, r = block_norm_fn(*args)
        for _ in range(4):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, first[0]) and torch.equal(r, first[1])
            once()
            torch.cuda.synchronize()


def test_compiled():
    t = {n: x.to(DEV) if isinstance(x, torch.Tensor) else x
         for n, x in make(14, (20, 130), BF, F, True, True, "tensor", True).items()}
    for parts in (NAMES, ("x", "post", "gate"), ("x", "residual", "pre")):
        def f(*leaves, parts=parts):
            d = dict.fromkeys(NAMES)
            d.update(zip(parts, leaves))
            res = block_norm_fn(*(d[n] for n in NAMES))
            return res if isinstance(res, tuple) else (res,)

        out = []
        for fn in (f, torch.compile(f, backend="aot_eager", fullgraph=True)):
            leaves = [t[n].detach().requires_grad_(True) for n in parts]
            res = fn(*leaves)
            out.append([*res, *torch.autograd.grad(res, leaves, [torch.ones_like(x) for x in res])])
        for a, b in zip(*out):
            assert torch.equal(a, b)


def test_second_derivatives_are_refused():
    t = make(15, (4, 30), BF, None, True)
    x, post = t["x"].to(DEV).requires_grad_(True), t["post"].to(DEV)
    (g,) = torch.autograd.grad(block_norm_fn(x, None, post).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        g.float().sum().backward()


def test_unit_keys():
    """A constant weight of dim ** -0.5 gives rows unit length, as the delta rule takes its keys."""
    x = torch.randn(50, 3, 64, device=DEV)
    w = torch.full((64,), 64 ** -0.5, device=DEV)
    torch.testing.assert_close(block_norm_fn(x, post_weight=w, eps=0.0), torch.nn.functional.normalize(x, dim=-1))
