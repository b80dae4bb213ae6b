"""The delta rule under torch.compile without gradients: the operator that keeps nothing for a backward is the one that is
traced, its results are the eager call's, and its memory too."""

import pytest
import torch

from causal_conv1d_triton import delta
from causal_conv1d_triton.delta import gated_delta_fn

BF, F = torch.bfloat16, torch.float32


def traced(call):
    """Names of the operators of this package in the graph of a call; nothing is run."""
    seen = []

    def backend(gm, inputs):
        seen.extend(str(n.target) for n in gm.graph.nodes if "causal_conv1d_amd" in str(n.target))

        def nothing(*args):
            raise StopIteration
        return nothing

    torch._dynamo.reset()
    with pytest.raises(StopIteration):
        torch.compile(call, backend=backend, fullgraph=True)()
    return seen


@pytest.mark.parametrize("final", [False, True])
@pytest.mark.parametrize("grad_mode,leaf,op", [(True, True, "gated_delta"), (True, False, "gated_delta_infer"),
                                               (False, True, "gated_delta_infer"), (False, False, "gated_delta_infer")])
def test_which_operator_is_traced(grad_mode, leaf, op, final):
    q, v, g = torch.zeros(1, 5, 2, 8, dtype=BF), torch.zeros(1, 5, 4, 6, dtype=BF), torch.zeros(1, 5, 4)
    v.requires_grad_(leaf)
    with torch.set_grad_enabled(grad_mode):
        seen = traced(lambda: gated_delta_fn(q, q, v, g, g, return_final_states=final))
    assert [s.split(".")[1] for s in seen] == [op], seen


def test_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        f = lambda *s, t=BF: torch.empty(*s, device="cuda", dtype=t)  # noqa: E731
        q, v, g = f(2, 130, 3, 72), f(2, 130, 6, 40), f(2, 130, 6, t=F)
        for final, shape in ((True, (2, 6, 72, 40)), (False, (0,))):
            out, fin = delta._infer_op(q, q, v, g, g, None, None, 1.0, final)
            assert out.shape == v.shape and out.dtype == BF and fin.shape == shape
            assert not final or fin.dtype == F


@pytest.mark.gpu
@pytest.mark.parametrize("final", [False, True])
def test_inference_is_the_eager_call(final):
    """Bits and peak memory. Training's call would keep 2 * 4 * 16 * (64 + 64) * 64 numbers beside them, 4 MiB."""
    gen = torch.Generator("cuda").manual_seed(0)
    n = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    q, v, g = torch.nn.functional.normalize(n(2, 1000, 4, 64), dim=-1).to(BF), n(2, 1000, 4, 64).to(BF), -n(2, 1000, 4).abs()
    beta, init = torch.sigmoid(n(2, 1000, 4)), n(2, 4, 64, 64)

    def f(q, v, g, beta, init):
        return gated_delta_fn(q, q, v, g, beta, None, init, return_final_states=final)

    torch._dynamo.reset()
    results, peaks = [], []
    with torch.no_grad():
        for fn in (f, torch.compile(f, backend="aot_eager", fullgraph=True)):
            for _ in range(2):  # the second time nothing is traced
                torch.cuda.synchronize()
                torch.cuda.reset_peak_memory_stats()
                before = torch.cuda.memory_allocated()
                res = fn(q, v, g, beta, init)
                torch.cuda.synchronize()
                peak = torch.cuda.max_memory_allocated() - before
            results.append(res if final else (res,))
            peaks.append(peak)
    for a, b in zip(*results):
        assert torch.equal(a, b)
    assert abs(peaks[1] - peaks[0]) < 1 << 20, peaks
