"""What the bounds of test_layer_accuracy.py have to catch, without a GPU: the delta rule with one of its parts kept in
fewer bits, and sums of the norms' weights without one row, are outside them; fp32 is inside."""

import pytest
import torch

import layer_oracle as oracle

LEAVES = ("q", "k", "v", "g", "beta", "init")


def rounded(x, bits):
    """To so many significant bits; gradients pass."""
    m, e = torch.frexp(x.detach())
    return x + (torch.ldexp(torch.round(m * 2.0 ** bits), e - bits) - x.detach())


def delta(d, part, bits):
    """The recurrence with a part in fewer bits: an operand, the states between chunks of 64 rows (of the gradients,
    too), or the corrections."""
    r = lambda x, name: rounded(x, bits) if part == name else x  # noqa: E731

    def back(x, name):
        if part == "d" + name:
            x.register_hook(lambda g: rounded(g, bits))
        return x

    q, k, S = r(d["q"], "q"), r(d["k"], "k"), d["init"]
    outs = []
    for t in range(q.shape[1]):
        if t % 64 == 0:
            S = back(r(S, "state"), "state")
        S = torch.exp(d["g"][:, t])[..., None, None] * S
        u = d["beta"][:, t][..., None] * (d["v"][:, t] - torch.einsum("bhk,bhkv->bhv", k[:, t], S))
        u = back(r(u, "u"), "u")
        S = S + k[:, t][..., None] * u[..., None, :]
        outs.append(q.shape[-1] ** -0.5 * torch.einsum("bhk,bhkv->bhv", q[:, t], S))
    return torch.stack(outs, 1), S


def results(T, part=None, bits=0):
    gen = torch.Generator().manual_seed(T)
    n = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
    d = {"q": unit(n(1, T, 2, 64)), "k": unit(0.3 + n(1, T, 2, 64)), "v": n(1, T, 2, 32),
         "g": -torch.nn.functional.softplus(n(1, T, 2) - 2), "beta": torch.sigmoid(n(1, T, 2)), "init": n(1, 2, 64, 32)}
    do, dfinal = n(1, T, 2, 32).double(), n(1, 2, 64, 32).double()
    d = {m: x.double().requires_grad_(True) for m, x in d.items()}
    out, final = delta(d, part, bits)
    grads = torch.autograd.grad([out, final], [d[m] for m in LEAVES], [do, dfinal])
    return {"out": out.detach(), "final": final.detach(), **dict(zip(LEAVES, grads))}


@pytest.mark.parametrize("T", [17, 65, 300])
@pytest.mark.parametrize("bits", [16, 18])
@pytest.mark.parametrize("part,seen", [("q", ("out", "init")), ("k", ("final", "v")), ("u", ("final", "q", "k")),
                                       ("state", ("out", "q")), ("du", ("v", "beta")), ("dstate", ("init",))])
def test_fewer_bits_are_outside(part, seen, bits, T):
    want, got = results(T), results(T, part, bits)
    for n, x in want.items():
        oracle.rms_close(x.float(), x, n)  # one rounding to fp32
    for n in seen:
        with pytest.raises(AssertionError):
            oracle.rms_close(got[n].float(), want[n], n)


def test_a_row_left_out_is_outside():
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(40000, 16, generator=gen, dtype=torch.float64)
    h = x / x.square().mean(-1, keepdim=True).sqrt()
    terms = h * torch.randn(40000, 16, generator=gen, dtype=torch.float64)
    want = terms.sum(0)
    oracle.rms_close(terms.float().sum(0), want, "dpost")
    with pytest.raises(AssertionError):
        oracle.rms_close(terms[1:].sum(0).float(), want, "dpost")
