"""Plain 64-bit implementations of the operators of a linear-attention layer, on the CPU, whose gradients are torch's
own of these few lines. Test infrastructure only.

Bounds of the delta rule. Keys have at most unit length, decays are at most one and 0 <= beta <= 2, so a step neither
stretches the state nor an error in it: I - beta k k^T has norm one at most. What a chunk of 64 rows adds in fp32
comes from sums of at most 256 products (the keys' elements) and 64 (the rows), a triangular system of 64 rows whose
substitution is exact for a matrix 64 units away, and from the products of pieces left out, 2^-22 of the largest: below
256 units of 2^-24 of the largest that the column of values holds (state, value or output), and the chunks' errors
add up. A gradient is such a sum of products of two such quantities, forward and backward, each off by as much, and
passes the triangular system twice: 1024 units a chunk of the tensor's largest element. A result of 16 bits is rounded
once more, half a step.

Bounds of the norms. A row's sum of squares has at most 8192 positive terms, in 256 lanes of 32 that are joined in a
tree: 64 roundings at most, half of that in the inverse root; the factors of an element are a handful of roundings and
the hardware's exponential (1 ulp, and |z| 2^-24 from its argument). 64 units of the element's own size for results
without a difference; a difference (the backward's centring, the residual sum) of the size of its two terms."""

import torch

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}
U = 2.0 ** -24


def delta(q, k, v, g, beta, seq=None, init=None, scale=None):
    """(out, final) in 64 bits, token after token, differentiable."""
    B, T, Hk, Dk = k.shape
    H, Dv = v.shape[2:]
    scale = Dk ** -0.5 if scale is None else scale
    q, k = (x.repeat_interleave(H // Hk, 2) for x in (q, k))
    S = torch.zeros(B, H, Dk, Dv, dtype=torch.float64) if init is None else init
    outs = []
    for t in range(T):
        live = torch.ones(B, dtype=torch.bool)
        keep = torch.ones(B, dtype=torch.bool)
        if seq is not None:
            live = seq[:, t] >= 0
            if t:
                keep = seq[:, t] == seq[:, t - 1]
        cut = (~(live & keep))[:, None, None, None]

        def alive(x):
            m = live.view(-1, *[1] * (x.dim() - 1))
            return torch.where(m, x, torch.zeros_like(x))

        kt, qt, vt = alive(k[:, t]), alive(q[:, t]), alive(v[:, t])
        S = torch.where(cut, torch.zeros_like(S), alive(torch.exp(g[:, t]))[..., None, None] * S)
        u = alive(beta[:, t])[..., None] * (vt - torch.einsum("bhk,bhkv->bhv", kt, S))
        S = S + kt[..., None] * u[..., None, :]
        outs.append(scale * torch.einsum("bhk,bhkv->bhv", qt, S))
    out = torch.stack(outs, 1) if outs else torch.zeros(B, 0, H, Dv, dtype=torch.float64)
    return out, S


def delta_all(t, dfinal=None, scale=None):
    """dict of out, final and the gradients of t's tensors (keys q k v g beta init, seq and do), in 64 bits."""
    d = {n: None if t.get(n) is None else t[n].detach().cpu().double().requires_grad_(True)
         for n in ("q", "k", "v", "g", "beta", "init")}
    seq = None if t.get("seq") is None else t["seq"].cpu().long()
    out, final = delta(*(d[n] for n in ("q", "k", "v", "g", "beta")), seq, d["init"], scale)
    res = {"out": out.detach(), "final": final.detach()}
    if t.get("do") is not None:
        total = (out * t["do"].cpu().double()).sum()
        if dfinal is not None:
            total = total + (final * dfinal.cpu().double()).sum()
        names = [n for n in d if d[n] is not None]
        grads = torch.autograd.grad(total, [d[n] for n in names], allow_unused=True)
        res.update({n: torch.zeros_like(d[n]) if x is None else x for n, x in zip(names, grads)})
    return res


def delta_close(got, want, name, t):
    """got against want within the bound at the head of this file."""
    got = got.detach().cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    chunks = (t["k"].shape[1] + 63) // 64 + 1
    size = want.abs().max() if want.numel() else torch.tensor(0.0)
    if name in ("out", "final"):
        units = 256
        size = max([float(size)] + [float(t[n].double().abs().max()) for n in ("v", "init") if t.get(n) is not None])
    else:
        units = 1024
    close(got, want, units * chunks * U * size, name)


def close(got, want, bound, name):
    got = got.detach().cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    err = (got.double() - want).abs()
    room = bound + UNIT[got.dtype] * (want.abs() + bound) + TINY[got.dtype]
    bad = ~(err <= room)
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} off, worst "
                           f"{float((err / room).nan_to_num(float('inf')).max()):.3g} of its bound")


def act(z, activation):
    s = torch.sigmoid(z)
    return {"silu": z * s, "sigmoid": s, None: z}[activation]


def norm(x, residual=None, post=None, gate=None, scale=None, pre=None, eps=1e-6, activation="silu"):
    """(r, y or None) in 64 bits, differentiable."""
    m = x
    if post is not None:
        m = m * post / torch.sqrt((m * m).mean(-1, keepdim=True) + eps)
    if gate is not None:
        m = m * act(gate, activation)
    r = m if scale is None else scale * m
    if residual is not None:
        r = residual + r
    y = None if pre is None else r * pre / torch.sqrt((r * r).mean(-1, keepdim=True) + eps)
    return r, y


def norm_all(t, eps=1e-6, activation="silu"):
    """dict of r, y and the gradients of t's tensors under the incoming dr and dy."""
    d = {n: t[n].detach().cpu().double().requires_grad_(True) if isinstance(t.get(n), torch.Tensor) else t.get(n)
         for n in ("x", "residual", "post", "gate", "scale", "pre")}
    r, y = norm(**d, eps=eps, activation=activation)
    res = {"r": r.detach(), "y": None if y is None else y.detach()}
    total = 0.0
    if t.get("dr") is not None:
        total = total + (r * t["dr"].cpu().double()).sum()
    if t.get("dy") is not None:
        total = total + (y * t["dy"].cpu().double()).sum()
    if isinstance(total, torch.Tensor):
        names = [n for n in d if isinstance(d[n], torch.Tensor)]
        grads = torch.autograd.grad(total, [d[n] for n in names], allow_unused=True)
        res.update({"d" + n: torch.zeros_like(d[n]) if g is None else g for n, g in zip(names, grads)})
    return res


def norm_close(got, want, name, t):
    """The weights' gradients are sums over the rows of terms of both signs, and a row's results differences of
    terms of the size of the row's largest: 64 units of that, times the square root of the number of rows."""
    rows = max(1, want.numel() // max(1, want.shape[-1])) if want.dim() > 1 else 1
    n_rows = t["x"].numel() // max(1, t["x"].shape[-1])
    if name in ("dpost", "dscale", "dpre"):
        bound = 64 * U * max(1.0, n_rows ** 0.5) * (float(want.abs().max()) + 8 * n_rows ** 0.5) if n_rows else 0.0
    else:
        size = want.abs().reshape(rows, -1).amax(-1).view(*want.shape[:-1], 1) if want.numel() else want
        parts = max([1.0] + [float(t[n].double().abs().max()) for n in ("dr", "dy", "residual")
                             if t.get(n) is not None and t[n].numel()])
        bound = 64 * U * (size + parts)
    close(got, want, bound, name)


# Root mean squares, in units of 2^-24 of the tensor's own. A step of a sum in fp32 rounds by 0.3 units of its result in
# the mean; a product over the keys' elements or the rows is up to 48 steps (8 instructions for each of six pairs of
# pieces), whose partial sums are smaller than the last: 2 units. Three such products follow one another in a chunk, a chunk's
# error shrinks with its state, and the backward goes through as many again: 5 units. The gradient of the log-decays is
# a difference of sums over the rows behind, whose parts are up to three times as large.
RMS_UNITS = {"g": 24}


def rms_units(got, want):
    off = (got.detach().double().cpu() - want).square().mean().sqrt()
    return float(off / want.square().mean().sqrt()) / U


def rms_close(got, want, name):
    assert got.dtype == torch.float32 and got.shape == want.shape
    if want.any():
        units = rms_units(got, want)
        assert units <= RMS_UNITS.get(name, 8), (name, units)
    else:
        assert not got.any(), name


def share_beside(got, want):
    """Of results of 16 bits of a quarter of their root mean square and more, the share that is not the nearest number."""
    large = want.abs() >= 0.25 * want.square().mean().sqrt()
    return float((got.cpu() != want.to(got.dtype))[large].double().mean())
