"""Plain 64-bit implementations of the operators around the convolution, on the CPU, with a bound of
the rounding error that an fp32 evaluation of the same formulas makes. Test infrastructure only.

Bounds. One fp32 evaluation of a row's factors a, beta, i and of its multiply-add is off by at most
EPS of its value (a: the exponent k r is off by a few units of 2^-24 of itself, |k r| is of order one
wherever a is not negligible, and the exponential adds one). An error made in row s reaches row t
multiplied by the factors between, so with A[t] = a[t] A[t-1] + |u[t]| (the recurrence over absolute
values) the state is off by at most EPS times E[t] = a[t] E[t-1] + A[t]. The gradients are products
of such quantities and their bounds follow by the product rule. A result stored in 16 bits is rounded
once more."""

import math

import torch

EPS = 1e-6
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}


def _walk(f, u):
    """h[t] = f[t] h[t-1] + u[t] along dim 1 from zero; a factor of zero cuts."""
    h = torch.empty_like(u)
    s = torch.zeros_like(u[:, 0])
    for t in range(u.shape[1]):
        s = torch.where(f[:, t] == 0, u[:, t], f[:, t] * s + u[:, t])
        h[:, t] = s
    return h


def recurrence(x, gate, decay=None, igate=None, seq=None, init=None, scale=8.0, dy=None, dfinal=None):
    """dict of out, final and, with dy, the gradients; each a pair (value, error bound)."""
    x, gate = x.double(), gate.double()
    B, T, D = x.shape
    r, not_r = torch.sigmoid(gate), torch.sigmoid(-gate)  # 1 - r itself cancels, in 64 bits too
    if decay is None:
        la, a, beta = None, r, not_r
    else:
        decay = decay.double()
        sp = torch.nn.functional.softplus(decay, threshold=50)
        la = -scale * sp * r
        a, beta = torch.exp(la), torch.sqrt(-torch.expm1(2 * la))
    i = torch.ones_like(x) if igate is None else torch.sigmoid(igate.double())
    not_i = None if igate is None else torch.sigmoid(-igate.double())
    f, live = a.clone(), torch.ones(B, T, 1, dtype=torch.bool)
    if seq is not None:
        seq = seq.long()
        live = (seq >= 0)[..., None]
        f[:, 1:] = f[:, 1:] * (seq[:, 1:] == seq[:, :-1])[..., None]
        f = torch.where(live, f, 0)
    zero = torch.zeros_like(x)
    v = torch.where(live, i * x, zero)
    beta = torch.where(live, beta, zero)
    u = beta * v
    h0 = torch.zeros(B, D, dtype=torch.float64) if init is None else init.double()

    def states(u, first):
        u = u.clone()
        if T:
            u[:, 0] += torch.where(f[:, 0] == 0, 0, f[:, 0] * first)
        return _walk(f, u)

    h = states(u, h0)
    A = states(u.abs(), h0.abs())
    E = states(A, h0.abs())
    last = lambda h, first: h[:, -1] if T else first  # noqa: E731
    res = {"out": (h, EPS * E), "final": (last(h, h0), EPS * last(E, h0.abs()))}
    if dy is None:
        return res

    def back(dy, dfin):  # dh[t] = dy[t] + f[t+1] dh[t+1], dh of the last row with dfinal
        dy = torch.where(live, dy, zero)
        if T and dfin is not None:
            dy = dy.clone()
            dy[:, -1] += torch.where(live[:, -1], dfin, torch.zeros_like(dfin))
        g = torch.cat([torch.zeros_like(f[:, :1]), f.flip(1)[:, :-1]], 1)
        return _walk(g, dy.flip(1)).flip(1)

    dfin = None if dfinal is None else dfinal.double()
    dh = back(dy.double(), dfin)
    dA = back(dy.double().abs(), None if dfin is None else dfin.abs())
    dE = back(dA, None if dfin is None else dfin.abs())
    keep = f != 0

    def before(h, first):
        return torch.where(keep, torch.cat([first[:, None], h[:, :-1]], 1), zero)

    hp, Ap, Ep = before(h, h0), before(A, h0.abs()), before(E, h0.abs())
    res["x"] = (dh * beta * i, 4 * EPS * dE * beta * i)
    if igate is not None:
        xx = torch.where(live, x, zero)
        w = beta * xx * i * not_i
        res["igate"] = (dh * w, 4 * EPS * dE * w.abs())
    if decay is None:
        w = torch.where(live, r * not_r, zero)
        res["gate"] = (dh * (hp - v) * w, 4 * EPS * w * (dE * (Ap + v.abs()) + dA * Ep))
    else:
        over = torch.where(beta > 0, a * a / beta, zero)
        q = dh * la * (a * hp - v * over)
        eq = 4 * EPS * la.abs() * (dE * (a * Ap + v.abs() * over) + dA * a * Ep)
        res["gate"] = (q * not_r, eq * not_r)
        ratio = torch.sigmoid(decay) / sp
        res["decay"] = (q.sum((0, 1)) * ratio, (eq + EPS * q.abs()).sum((0, 1)) * ratio)
    if T:
        res["init"] = (torch.where(keep[:, 0], f[:, 0] * dh[:, 0], 0), EPS * f[:, 0] * (dE + dA)[:, 0])
    else:
        res["init"] = (torch.zeros(B, D, dtype=torch.float64) if dfin is None else dfin,
                       torch.zeros(B, D, dtype=torch.float64))
    return res


def assert_close(got, want, what=""):
    """got against (value, bound): the bound, and one rounding to got's type."""
    value, bound = want
    got = got.detach().cpu()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    u, tiny = UNIT[got.dtype], TINY[got.dtype]
    err = (got.double() - value).abs()
    room = bound + u * (value.abs() + bound) + tiny
    bad = ~(err <= room)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
                           f"{float((err / room).nan_to_num(math.inf).max()):.3g} of its bound")


def plan(cached, new, tables, free, num_free, page_size, max_tokens):
    """One request after the other, in Python integers."""
    M = tables.shape[1]
    tables = [list(map(int, row)) for row in tables.tolist()]
    free = free.tolist()
    nf = min(max(int(num_free), 0), len(free))
    seq_lens, start = [], [0]
    pos, ids, slots = [], [], []
    upto = used = 0
    for r, (c, n) in enumerate(zip(cached.tolist(), new.tolist())):
        c, n = max(c, 0), max(n, 0)
        have, want = -(-c // page_size), -(-(c + n) // page_size)
        need = want - have if want <= M else 0
        ok = want <= M and (need == 0 or upto + need <= nf)
        if ok:
            for j in range(need):
                tables[r][have + j] = free[nf - 1 - upto - j]
            if need:
                used = upto + need
        upto += need
        seq_lens.append(c + n if ok else c)
        start.append(start[-1] + n)
        for t in range(min(n, max(0, max_tokens - len(pos)))):
            p = c + t
            page = tables[r][p // page_size] if ok else -1
            pos.append(p if ok else -1)
            ids.append(r if ok else -1)
            slots.append(page * page_size + p % page_size if page >= 0 else -1)

    def places(v):
        return torch.tensor((v + [-1] * max_tokens)[:max_tokens], dtype=torch.int64)

    return {"tables": torch.tensor(tables, dtype=torch.int64).reshape(len(tables), M),
            "seq_lens": torch.tensor(seq_lens, dtype=torch.int64),
            "query_start": torch.tensor(start), "positions": places(pos),
            "request_ids": places(ids), "slot_mapping": places(slots),
            "num_free": torch.tensor([nf - used])}


def attention(q, k_cache, v_cache, tables, lens, scale=None, window=None, ids=None):
    """((out, bound), (lse, bound)) of one row after the other. Bounds: a score is off by the rounding
    of its sum of products, which moves every weight by as much, and a weight's own representation by
    at most 2^-15 of it (two 8-bit pieces) or 2^-24 of the largest."""
    R, Hq, Dh = q.shape
    P, ps, H, _ = k_cache.shape
    G = Hq // H
    scale = Dh ** -0.5 if scale is None else scale
    out = torch.zeros(R, Hq, Dh, dtype=torch.float64)
    bound = torch.zeros_like(out)
    lse = torch.full((R, Hq), -math.inf, dtype=torch.float64)
    lbound = torch.zeros_like(lse)
    for r in range(R):
        req = r if ids is None else int(ids[r])
        if req < 0 or req >= tables.shape[0]:
            continue
        n = min(int(lens[r]), tables.shape[1] * ps)
        lo = max(0, n - window) if window else 0
        at = [(int(tables[req, p // ps]), p % ps) for p in range(lo, n)]
        at = [(g, o) for g, o in at if 0 <= g < P]
        if not at:
            continue
        pg, off = (torch.tensor(v) for v in zip(*at))
        k, v = k_cache[pg, off].double(), v_cache[pg, off].double()
        for h in range(Hq):
            s = (k[:, h // G] @ q[r, h].double()) * scale
            top = s.max()
            w = torch.exp(s - top) if torch.isfinite(top) else torch.zeros_like(s)
            e = (Dh + 8) * 2.0 ** -24 * (k[:, h // G].abs() @ q[r, h].double().abs()).max() * scale
            e = e + 2.0 ** -22 * (1 + s.abs().max())
            if float(w.sum()) == 0:
                continue
            lse[r, h] = top + torch.log(w.sum())
            lbound[r, h] = e + 2.0 ** -22 + len(at) ** 0.5 * 2.0 ** -24
            w = w / w.sum()
            vv = v[:, h // G]
            out[r, h] = w @ vv
            bound[r, h] = (2.0 ** -15 + 2 * e) * (w @ vv.abs()) + 2.0 ** -24 * w.max() * vv.abs().sum(0)
    return (out, bound), (lse, lbound)
