"""Training passes of the delta rule and the norms around a block, as a layer runs them, captured in a graph: every replay
has the eager bits, beside eager work and with other inputs in the same places."""

import pytest
import torch

from causal_conv1d_triton.delta import gated_delta_fn
from causal_conv1d_triton.norm import block_norm_fn

pytestmark = pytest.mark.gpu
BF, F = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype,Dk,packed", [(BF, 64, True), (BF, 128, False), (F, 72, True), (BF, 256, False)])
def test_training_in_a_graph(dtype, Dk, packed):
    gen = torch.Generator("cuda").manual_seed(0)
    n = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    B, T, Hk, H, Dv = 2, 300, 2, 4, 40
    q, k = n(B, T, Hk, Dk).to(dtype), n(B, T, Hk, Dk).to(dtype)
    v, gate, stream = n(B, T, H, Dv).to(dtype), n(B, T, H, Dv).to(dtype), n(B, T, H * Dv)
    g, beta, init = -n(B, T, H).abs(), torch.sigmoid(n(B, T, H)).to(dtype), n(B, H, Dk, Dv)
    unit, w1, w2 = torch.full((Dk,), Dk ** -0.5, device="cuda"), 1 + 0.1 * n(Dv), 1 + 0.1 * n(H * Dv)
    seq = (torch.arange(T, device="cuda") // 110).int().expand(B, T).contiguous() if packed else None
    dy, dr, dfinal = n(B, T, H * Dv).to(dtype), n(B, T, H * Dv), n(B, H, Dk, Dv)
    leaves = [t.requires_grad_(True) for t in (q, k, v, gate, stream, g, beta, init, w1, w2)]

    def step():
        kn, qn = (block_norm_fn(t, post_weight=unit) for t in (k, q))
        o, final = gated_delta_fn(qn, kn, v, g, beta, seq, init, return_final_states=True)
        o = block_norm_fn(o, post_weight=w1, gate=gate)
        y, r = block_norm_fn(o.flatten(-2), stream, pre_weight=w2)
        grads = torch.autograd.grad([y, r, final], leaves, [dy, dr, dfinal])
        return [t.detach() for t in (y, r, final, *grads)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = step()
    for i in range(4):
        with torch.no_grad():
            v.copy_(v.roll(1, 0))
        for o in outs:
            o.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step()):
            assert torch.equal(a, b), i
