"""The operators of a linear-attention layer together, as the example runs them: training on packed documents, and
serving."""

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "delta_serving.py")
    spec = importlib.util.spec_from_file_location("delta_serving", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_example_runs(example):
    """Token by token or all at once, the model says the same: both round every layer's activations to bf16 (2^-8)
    in three layers, in another order of sums; 5 % of the logits' norm is far outside what rounding does."""
    loss, grads, off = example.main()
    assert torch.isfinite(loss) and all(torch.isfinite(g).all() and g.any() for g in grads)
    assert off < 0.05


def test_the_comparison_tells(example):
    """What the last test's bound has to catch is outside it: a step from a lost state, of either kind."""
    model = example.Model(seed=2)
    said, logits = model.serve()
    slots = torch.arange(len(said), device="cuda", dtype=torch.int32)
    for lost in (0, 1):
        states = model.states(len(said))
        model.prompts([s[:-1] for s in said], states)
        states[0][lost].zero_()
        off = model.step(torch.stack([s[-1] for s in said]), states, slots).float() - logits.float()
        assert float(off.norm() / logits.float().norm()) > 0.05, lost


def test_packed_documents_are_the_separate_ones(example):
    """A packed pass gives each document its own rows: through the convolution, the rule and the norms."""
    model = example.Model(seed=1)
    docs = [torch.randint(0, 512, (n,), generator=model.gen, device="cuda") for n in (33, 1, 90)]
    seq = torch.cat([torch.full((len(d),), i, device="cuda") for i, d in enumerate(docs)]).int()[None]
    with torch.no_grad():
        x, stream = model.start(torch.cat(docs)[None])
        both = model.blocks[0].forward(x, stream, seq)
        at = 0
        for d in docs:
            s = slice(at, at + len(d))
            alone = model.blocks[0].forward(x[:, s], stream[:, s])
            for a, b in zip(both, alone):  # rounded to bf16 in between, cut into chunks at other places
                assert float((a[:, s].float() - b.float()).norm() / b.float().norm()) < 2 ** -7
            at += len(d)


def test_gradients_of_a_block(example):
    """The block's backward against differences of its own loss along the gradient: both sides pass bf16 values
    between the operators (2^-8 each), so a tenth is far outside what rounding does over 2 * 64 rows."""
    model = example.Model(seed=3, layers=1)
    b = model.blocks[0]
    tokens = torch.randint(0, 512, (2, 65), generator=model.gen, device="cuda")

    def loss(rate):
        b.rate = rate
        x, stream = model.start(tokens[:, :-1])
        x, stream = b.forward(x, stream)
        return torch.nn.functional.cross_entropy(model.logits(x).float().flatten(0, 1), tokens[:, 1:].flatten())

    rate = b.rate.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(loss(rate), rate)
    with torch.no_grad():
        step = 0.5 * g / g.norm()
        slope = float(loss(rate + step) - loss(rate - step)) / 2
    said = float((g * step).sum())
    assert abs(slope - said) < 0.25 * abs(said) + 2e-4, (slope, said)
