"""The gradients of every weight of the example's block, through the convolution, the delta rule and the norms, against the
same block in plain operations in 64 bits."""

import pytest
import torch
import torch.nn.functional as nnf

import layer_oracle as oracle
from test_layer_example import example  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


def plain(b, w, x, residual, seq):
    """The block of examples/delta_serving.py; w holds its weights, everything is 64 bits on the CPU."""
    z = x @ w["w_in"].T
    mixed, gate, decay, beta = z.split([b.mixed, b.H * b.Dv, b.H, b.H], -1)
    width = w["w_conv"].shape[1]
    rows = torch.zeros_like(mixed)
    for back in range(width):  # rows of the same document alone
        moved = nnf.pad(mixed, (0, 0, back, 0))[:, :mixed.shape[1]]
        same = (nnf.pad(seq, (back, 0), value=-1)[:, :mixed.shape[1]] == seq)[..., None]
        rows = rows + torch.where(same, moved, torch.zeros_like(moved)) * w["w_conv"][:, width - 1 - back]
    mixed = rows * torch.sigmoid(rows)
    q, k, v = mixed.split([b.Hk * b.Dk, b.Hk * b.Dk, b.H * b.Dv], -1)

    def heads(t, n):
        return t.unflatten(-1, (n, -1))

    def unit(t):
        return t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6) * b.Dk ** -0.5

    o, _ = oracle.delta(unit(heads(q, b.Hk)), unit(heads(k, b.Hk)), heads(v, b.H),
                        -w["rate"] * nnf.softplus(decay + w["shift"]), torch.sigmoid(beta), seq)
    o, _ = oracle.norm(o, post=w["w_head"], gate=heads(gate, b.H))
    r, y = oracle.norm(o.flatten(-2) @ w["w_out"].T, residual, pre=w["w_next"])
    return y, r


def test_every_weight_of_a_block(example):  # noqa: F811
    """About ten tensors between the operators are rounded to bf16, 2^-9 of each element and 0.6 of that in the mean, in
    the forward and again in the backward: 20 such roundings are 0.5 % of a gradient's norm when they are independent. The
    sums that they go through (decays over the rows, two normalisations) can make three or four times as much of it: 2 %.
    A factor left out or a term lost is tens of per cent."""
    model = example.Model(seed=4, layers=1)
    b = model.blocks[0]
    gen = torch.Generator("cuda").manual_seed(6)
    x = torch.randn(2, 80, 256, generator=gen, device="cuda").to(torch.bfloat16)
    residual = torch.randn(2, 80, 256, generator=gen, device="cuda")
    ups = [torch.randn(2, 80, 256, generator=gen, device="cuda").to(torch.bfloat16),
           torch.randn(2, 80, 256, generator=gen, device="cuda")]
    seq = (torch.arange(80, device="cuda") // 33).int().expand(2, 80).contiguous()
    leaves = [getattr(b, n).detach().requires_grad_(True) for n in b.NAMES]
    for n, t in zip(b.NAMES, leaves):
        setattr(b, n, t)
    out = b.forward(x, residual, seq)
    got = torch.autograd.grad(out, leaves, ups)
    w = {n: t.detach().cpu().double().requires_grad_(True) for n, t in zip(b.NAMES, leaves)}
    y, r = plain(b, w, x.cpu().double(), residual.cpu().double(), seq.cpu())
    want = torch.autograd.grad([y, r], list(w.values()), [u.cpu().double() for u in ups])
    for n, a, e in zip(b.NAMES, got, want):
        assert float(e.norm()) > 0 and a.shape == e.shape
        off = float((a.double().cpu() - e).norm() / e.norm())
        assert off < 0.02, (n, off)
    for a, e in zip(out, (y, r)):
        assert float((a.detach().double().cpu() - e.detach()).norm() / e.detach().norm()) < 0.02
