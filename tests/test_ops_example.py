"""The example that runs the operators together: a training step over packed documents, and serving."""

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                        "hybrid_serving.py")
    spec = importlib.util.spec_from_file_location("hybrid_serving", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_example_runs(example):
    """Token by token or all at once, the model says the same: both round every layer's activations to
    bf16 (2^-8) in four layers, in another order of sums, so 5 % of the logits' norm is far outside what
    rounding does and far inside what a lost state or key would."""
    loss, grads, off = example.main()
    assert torch.isfinite(loss) and all(torch.isfinite(g).all() and g.any() for g in grads)
    assert off < 0.05


def test_the_comparison_tells(example):
    """What the last test's bound has to catch is outside it: a step from lost states, or lost keys."""
    layers, embed, gen = example.build(seed=2)
    said, logits = example.serve(layers, embed, gen)
    for lost in (0, 2):  # a recurrent layer, the attention layer
        server = example.Server(layers, embed, len(said), 64, 16, 16)
        server.prompts([s[:-1] for s in said])
        for t in server.state[lost]:
            t.zero_()
        off = server.step(torch.stack([s[-1] for s in said])).float() - logits.float()
        assert float(off.norm() / logits.float().norm()) > 0.05, lost


def test_packed_documents_are_the_separate_ones(example):
    """The plan's request ids as seq_idx: a packed pass gives each request its own rows."""
    layers, embed, gen = example.build(seed=1)
    server = example.Server(layers, embed, 3, 64, 16, 16)
    prompts = [torch.randint(0, 512, (n,), generator=gen, device="cuda") for n in (33, 1, 90)]
    _, plan = server.prompts(prompts)
    x = embed[torch.cat(prompts)]
    u, gate, igate = layers[0].project(x)
    conv = example.causal_conv1d_fn(u[None], layers[0].w_conv, layers[0].b_conv,
                                    plan.request_ids[None], activation="silu")
    h = example.gated_recurrence_fn(conv, gate[None], layers[0].decay, igate[None],
                                    plan.request_ids[None])
    at = 0
    for p in prompts:
        n = len(p)
        s = slice(at, at + n)
        c1 = example.causal_conv1d_fn(u[None, s], layers[0].w_conv, layers[0].b_conv,
                                      activation="silu")
        h1 = example.gated_recurrence_fn(c1, gate[None, s], layers[0].decay, igate[None, s])
        assert torch.equal(conv[:, s], c1)
        # the same rows, cut into waves at other places
        assert torch.allclose(h[:, s].float(), h1.float(), rtol=2 ** -7, atol=1e-5)
        at += n
