"""Measured workloads of the layer that the short convolution feeds in a linear-attention model: the gated
delta rule over its queries, keys and values (training, prompts, single tokens over a pool of states), and
the norms around a block, fused with the block's gate, the scale of its output and the residual stream.

A case is a dict of plain values:
  name     its name (listed cases only)
  op       "train"  gated_delta_fn, then the gradients of every differentiable input
           "infer"  gated_delta_fn with autograd off, states in and out
           "step"   gated_delta_update of one token per request, states in a pool
           "norm"   block_norm_fn, then (train) the gradients of every differentiable input
  dtype    of the activations; states and log-decays are fp32
Delta rule: B, T (batch, seqlen; "step": R requests of a pool of `pool` states), Hk heads of queries and
  keys of Dk, H heads of values of Dv (H / Hk of them share a key), packed (seq_idx of packed sequences, the
  last 5 % of a row padding), init (initial states and their gradient)
Norms: rows of D ("heads": so many rows lie beside each other, as a layer's heads do), post (norm of the
  block's output), gate, residual (its type, "" without), scale (per channel), pre (norm of the sum)
"""

import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ESIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6
CHUNK = 64


def _named(name, c):
    return dict(c, name=name) if name else c


def _delta(name, op, B, T, Hk, H, Dk, Dv, dtype="bf16", packed=False, init=False):
    return _named(name, dict(op=op, B=B, T=T, Hk=Hk, H=H, Dk=Dk, Dv=Dv, dtype=dtype, packed=packed,
                             init=init))


def _step(name, R, pool, Hk, H, Dk, Dv, dtype="bf16"):
    return _named(name, dict(op="step", R=R, pool=pool, Hk=Hk, H=H, Dk=Dk, Dv=Dv, dtype=dtype))


def _norm(name, rows, D, heads=1, dtype="bf16", post=False, gate=False, residual="", scale=False,
          pre=False, train=False):
    return _named(name, dict(op="norm", rows=rows, D=D, heads=heads, dtype=dtype, post=post, gate=gate,
                             residual=residual, scale=scale, pre=pre, train=train))


def listed():
    return [
        # One generated token of a small serving batch.
        _step("delta_step", 4, 16, 8, 8, 128, 128),
        # One generated token of a busy server: every state is read and written.
        _step("delta_step_busy", 128, 160, 16, 32, 128, 128),
        # Chunked prefill: 256 tokens of each request per call, states carried between calls.
        _delta("delta_chunk", "infer", 4, 256, 8, 16, 128, 128, init=True),
        # A whole long prompt of one request.
        _delta("delta_prompt", "infer", 1, 16384, 16, 16, 128, 128),
        # Training; two value heads share a key head.
        _delta("delta_train", "train", 4, 4096, 8, 16, 128, 128),
        # Training on packed documents, small heads.
        _delta("delta_train_packed", "train", 2, 8192, 16, 16, 64, 128, packed=True),
        # Full precision, lengths and heads that no tile divides, states trained.
        _delta("delta_train_odd_fp32", "train", 3, 777, 4, 4, 72, 100, dtype="fp32", init=True),
        # The norm of a decode step: the block's output joins the residual stream.
        _norm("norm_step", 16, 2048, residual="bf16", pre=True),
        # The norm of the delta rule's heads with the output gate, in training.
        _norm("norm_heads_train", 65536, 128, heads=16, post=True, gate=True, train=True),
        # Norms after and before a block with its scale and an fp32 residual stream, in training.
        _norm("norm_block_train", 16384, 2048, post=True, residual="fp32", scale=True, pre=True,
              train=True),
        # The same with a gate in a prompt, 16-bit residual stream.
        _norm("norm_block_prompt", 32768, 4096, post=True, gate=True, residual="bf16", scale=True,
              pre=True),
        # Row lengths that no access width divides.
        _norm("norm_odd_fp16", 5003, 1501, dtype="fp16", gate=True, residual="fp16", pre=True,
              train=True),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["train", "train", "infer", "infer", "step", "norm", "norm", "norm"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "norm":
        heads = rng.choice([1, 1, log(2, 32)])
        D = (rng.choice([64, 128, 256, rng.randint(16, 256)]) if heads > 1 else
             rng.choice([64 * log(4, 128), log(16, 8192)]))
        most = (64 << 20) // (2 if dtype == "fp32" else 1)
        rows = heads * max(1, min(log(1, 65536), most // (D * heads)))
        residual = rng.choice(["", dtype, dtype, "fp32"])
        post = rng.random() < 0.6
        return _norm(None, rows, D, heads, dtype, post, rng.random() < 0.5, residual,
                     bool(residual) and rng.random() < 0.4, bool(residual) or not post,
                     rng.random() < 0.6)
    Dk = rng.choice([64, 128, 128, 256, 96, rng.randint(16, 256)])
    Dv = rng.choice([64, 128, 128, 256, 96, rng.randint(16, 256)])
    Hk = rng.choice([1, 2, 4, 8, 16, rng.randint(1, 16)])
    H = Hk * rng.choice([1, 1, 1, 2, 4])
    if op == "step":
        R = max(1, min(log(1, 256), (1 << 28) // (H * Dk * Dv * 4)))
        return _step(None, R, R + log(1, 32), Hk, H, Dk, Dv, dtype)
    # Products of at most the listed cases' size.
    most = (4 * 4096 * 16 * 128 * 128) // ((4 if dtype == "fp32" else 1) * H * Dk * Dv)
    T = max(1, min(log(2, 16384), most))
    B = max(1, min(log(1, 16), most // T))
    return _delta(None, op, B, T, Hk, H, Dk, Dv, dtype, packed=T >= 64 and rng.random() < 0.3,
                  init=op == "infer" or rng.random() < 0.3)


def _ids(rng, B, T):
    ids = np.empty((B, T), np.int32)
    for b in range(B):
        t = n = 0
        while t < T:
            length = int(rng.integers(min(32, T), 2049))
            ids[b, t:t + length] = n
            t += length
            n += 1
        ids[b, T - T // 20:] = -1
    return ids


def prepare(case, seed):
    """Queries and keys are unit vectors, made from silu(N(0, 1)) as the convolution gives it, values
    silu(N(0, 1)), beta sigmoid(N(0, 1)); the decay is -rate * softplus(N(0, 1) + shift) with rates of 1 to
    16 and shifts that make the step 0.001 to 0.1, as such layers start training. Norms: N(0, 1), weights
    near one, scales near 0.1."""
    s, op = {"case": case}, case["op"]
    g = torch.Generator(DEV).manual_seed(seed)
    rng = np.random.default_rng(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device=DEV)

    if op == "norm":
        D, heads = case["D"], case["heads"]
        shape = (case["rows"] // heads, heads, D) if heads > 1 else (case["rows"], D)
        s["x"] = normal(*shape, dtype=dt)
        # the gate is a slice of a projection that makes other things too
        s["gate"] = None
        if case["gate"]:
            wide = normal(shape[0], 2 * heads * D, dtype=dt)
            s["gate"] = wide[:, heads * D:].unflatten(-1, (heads, D)) if heads > 1 else wide[:, D:]
        s["residual"] = normal(*shape, dtype=DTYPES[case["residual"]]) if case["residual"] else None
        s["post"] = 1 + 0.1 * normal(D) if case["post"] else None
        s["scale"] = 0.1 + 0.02 * normal(D) if case["scale"] else None
        s["pre"] = 1 + 0.1 * normal(D) if case["pre"] else None
        s["wrt"] = [k for k in ("x", "gate", "residual", "post", "scale", "pre") if s[k] is not None]
        if case["train"]:
            s["dr"] = normal(*shape, dtype=(s["x"] if s["residual"] is None else s["residual"]).dtype)
            s["dy"] = normal(*shape, dtype=dt) if case["pre"] else None
            for k in s["wrt"]:
                s[k] = s[k].detach().requires_grad_(True)
        return s

    H, Hk, Dk, Dv = case["H"], case["Hk"], case["Dk"], case["Dv"]
    lead = (case["R"],) if op == "step" else (case["B"], case["T"])
    silu = torch.nn.functional.silu
    for n in ("q", "k"):
        x = silu(normal(*lead, Hk, Dk))
        s[n] = (x / x.norm(dim=-1, keepdim=True)).to(dt)
    s["v"] = silu(normal(*lead, H, Dv)).to(dt)
    s["beta"] = torch.sigmoid(normal(*lead, H)).to(dt)
    rate = 1 + 15 * uniform(H)
    step = torch.exp(math.log(0.001) + (math.log(0.1) - math.log(0.001)) * uniform(H))
    shift = step + torch.log(-torch.expm1(-step))
    s["g"] = -rate * torch.nn.functional.softplus(normal(*lead, H) + shift)
    if op == "step":
        s["state"] = 0.3 * normal(case["pool"], H, Dk, Dv)
        s["slots"] = torch.from_numpy(rng.permutation(case["pool"])[:case["R"]].astype(np.int32)).to(DEV)
        return s
    s["seq"] = torch.from_numpy(_ids(rng, case["B"], case["T"])).to(DEV) if case["packed"] else None
    s["init"] = 0.3 * normal(case["B"], H, Dk, Dv) if case["init"] else None
    s["wrt"] = [k for k in ("q", "k", "v", "g", "beta", "init") if s[k] is not None]
    if op == "train":
        s["do"] = normal(*lead, H, Dv, dtype=dt)
        for k in s["wrt"]:
            s[k].requires_grad_(True)
    return s


# The framework's operators.


def _own(s):
    at = os.path.join(os.getcwd(), "causal-conv1d-triton_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    case, op = s["case"], s["case"]["op"]
    if op == "norm":
        from causal_conv1d_triton.norm import block_norm_fn
        args = (s["x"], s["residual"], s["post"], s["gate"], s["scale"], s["pre"])
        if not case["train"]:
            with torch.no_grad():
                res = block_norm_fn(*args, eps=EPS)
            return dict(zip(("y", "r"), res)) if case["pre"] else {"r": res}
        res = block_norm_fn(*args, eps=EPS)
        up = (s["dy"], s["dr"]) if case["pre"] else s["dr"]
        grads = torch.autograd.grad(res, [s[k] for k in s["wrt"]], up)
        out = dict(zip(("y", "r"), res)) if case["pre"] else {"r": res}
        return {**{k: v.detach() for k, v in out.items()},
                **{"d" + k: v for k, v in zip(s["wrt"], grads)}}
    from causal_conv1d_triton.delta import gated_delta_fn, gated_delta_update
    if op == "step":
        with torch.no_grad():
            out = gated_delta_update(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"],
                                     state_indices=s["slots"])
        return {"out": out, "state": s["state"]}
    if op == "infer":
        with torch.no_grad():
            out, final = gated_delta_fn(s["q"], s["k"], s["v"], s["g"], s["beta"], s["seq"], s["init"],
                                        return_final_states=True)
        return {"out": out, "final": final}
    out = gated_delta_fn(s["q"], s["k"], s["v"], s["g"], s["beta"], s["seq"], s["init"])
    grads = torch.autograd.grad(out, [s[k] for k in s["wrt"]], s["do"])
    return {"out": out.detach(), **{"d" + k: v for k, v in zip(s["wrt"], grads)}}


# The plain forms.


def _rms(x, weight):
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return y * weight.float()


def _norm_forward(x, residual, post, gate, scale, pre):
    m = x.float()
    if post is not None:
        m = _rms(m, post)
    if gate is not None:
        z = gate.float()
        m = m * z * torch.sigmoid(z)
    r = m if scale is None else scale.float() * m
    if residual is not None:
        r = residual.float() + r
    return r, None if pre is None else _rms(r, pre)


def _plain_norm(s):
    train = s["case"]["train"]
    names = ("x", "residual", "post", "gate", "scale", "pre")
    with torch.set_grad_enabled(train):
        t = {n: s[n] if s[n] is None else s[n].detach().float().requires_grad_(train) for n in names}
        r, y = _norm_forward(*(t[n] for n in names))
    res = {"r": r.detach().to(s["x"].dtype if s["residual"] is None else s["residual"].dtype)}
    if y is not None:
        res["y"] = y.detach().to(s["x"].dtype)
    if train:
        outs, ups = ([r], [s["dr"].float()]) if y is None else ([r, y], [s["dr"].float(), s["dy"].float()])
        grads = torch.autograd.grad(outs, [t[n] for n in s["wrt"]], ups)
        res.update({"d" + n: v.to(s[n].dtype) for n, v in zip(s["wrt"], grads)})
    return res


def _chunked(q, k, v, g, beta, seq, init):
    """The delta rule in chunks of rows: within one, the rows' corrections u solve a unit triangular
    system; between chunks the state is carried. fp32, but the decays' sums and the triangular inverse,
    which is a product of powers, in 64 bits. q, k: (B, T, Hk, Dk), v: (B, T, H, Dv), g, beta: (B, T, H)."""
    B, T, Hk, Dk = k.shape
    H, Dv, C = v.shape[2], v.shape[3], CHUNK
    N = -(-T // C)
    live = torch.ones(B, T, dtype=torch.bool, device=DEV) if seq is None else seq >= 0
    run = torch.zeros(B, T, dtype=torch.int64, device=DEV)
    if seq is not None:  # the number of the run of equal ids that a row lies in
        run = torch.cat([torch.zeros_like(run[:, :1]), (seq[:, 1:] != seq[:, :-1]).long()], 1).cumsum(1)

    def cut(x, fill=0.0):  # (B, T, H, ...) -> (B, H, N, C, ...)
        x = torch.cat([x, torch.full((B, N * C - T, *x.shape[2:]), fill, dtype=x.dtype, device=DEV)], 1)
        return x.unflatten(1, (N, C)).movedim(3, 1)

    def masked(x):
        return x.masked_fill(~live.view(B, T, *[1] * (x.dim() - 2)), 0)

    q, k = (cut(masked(x).repeat_interleave(H // Hk, 2)) for x in (q * Dk ** -0.5, k))
    v, g, beta = cut(masked(v)), cut(masked(g)), cut(masked(beta))
    run = cut(run[:, :, None], -1).squeeze(1).view(B, 1, N, C)
    last = torch.cat([torch.zeros_like(run[:, :, :1, :1]), run[:, :, :-1, -1:]], 2)
    if T % C:
        run = torch.where(run < 0, run.amax(dim=(2, 3), keepdim=True), run)
    first = run == last  # rows that the carried state reaches
    first = first.float()
    end = (run == run[..., -1:]).float()
    through = first[..., -1]  # whether it reaches the chunk's end
    sums = g.double().cumsum(-1)
    i = torch.arange(C, device=DEV)
    same = (run[..., :, None] == run[..., None, :]) & (i[:, None] >= i)
    decay = torch.exp((sums[..., :, None] - sums[..., None, :]).masked_fill(~same, -math.inf)).float()
    into = torch.exp(sums).float() * first
    rest = torch.exp(sums[..., -1:] - sums).float() * end
    whole = torch.exp(sums[..., -1]).float() * through
    kk = torch.matmul(k, k.transpose(-1, -2).contiguous())
    qk = torch.matmul(q, k.transpose(-1, -2).contiguous()) * decay
    n = (-beta[..., None] * kk * decay).double().masked_fill(i[:, None] <= i, 0)
    inv = torch.eye(C, device=DEV, dtype=torch.float64) + n
    for _ in range(C.bit_length() - 2):
        n = torch.matmul(n, n)
        inv = inv + torch.matmul(n, inv)
    inv = inv.float()
    state = torch.zeros(B, H, Dk, Dv, device=DEV) if init is None else init.float()
    bv, kin = beta[..., None] * v, (beta * into)[..., None] * k
    u0, w = torch.matmul(inv, bv), torch.matmul(inv, kin)
    qin, kout = into[..., None] * q, (rest[..., None] * k).transpose(-1, -2).contiguous()
    outs = []
    for c in range(N):
        u = u0[:, :, c] - torch.matmul(w[:, :, c], state)
        outs.append(torch.matmul(qin[:, :, c], state) + torch.matmul(qk[:, :, c], u))
        state = whole[:, :, c, None, None] * state + torch.matmul(kout[:, :, c], u)
    out = torch.stack(outs, 2).flatten(2, 3)[:, :, :T].movedim(1, 2)
    if seq is not None:
        out = out.masked_fill(~live[..., None, None], 0)
        state = state * live[:, -1, None, None, None]
    return out, state


def _plain_delta(s):
    train = s["case"]["op"] == "train"
    names = ("q", "k", "v", "g", "beta", "init")
    with torch.set_grad_enabled(train):
        t = {n: s[n] if s[n] is None else s[n].detach().float().requires_grad_(train) for n in names}
        out, final = _chunked(t["q"], t["k"], t["v"], t["g"], t["beta"], s["seq"], t["init"])
    res = {"out": out.detach().to(s["v"].dtype)}
    if not train:
        return {**res, "final": final.detach()}
    grads = torch.autograd.grad(out, [t[n] for n in s["wrt"]], s["do"].float())
    return {**res, **{"d" + n: v.to(s[n].dtype) for n, v in zip(s["wrt"], grads)}}


def _plain_step(s):
    c, at = s["case"], s["slots"].long()
    q, k = (s[n].float().repeat_interleave(c["H"] // c["Hk"], 1) for n in ("q", "k"))
    state = torch.exp(s["g"].float())[..., None, None] * s["state"][at]
    u = s["beta"].float()[..., None] * (s["v"].float() - (k[..., None] * state).sum(-2))
    state = state + k[..., None] * u[..., None, :]
    s["state"].index_copy_(0, at, state)
    out = (q[..., None] * state).sum(-2) * c["Dk"] ** -0.5
    return {"out": out.to(s["v"].dtype), "state": s["state"]}


_PLAIN = {"train": _plain_delta, "infer": _plain_delta, "step": _plain_step, "norm": _plain_norm}


def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        return _PLAIN[s["case"]["op"]](s)


def work(case):
    """Every input read once, every output written once. Operations of the delta rule: for each token and
    head the state is multiplied by the key, updated by the outer product and multiplied by the query, with
    two products for each of these in the backward; of the norms about ten an element and direction."""
    op, e = case["op"], ESIZE[case["dtype"]]
    if op == "norm":
        n, D = case["rows"] * case["D"], case["D"]
        er = ESIZE[case["residual"]] if case["residual"] else 0
        eo = er or e
        weights = 4 * D * (case["post"] + case["scale"] + case["pre"])
        byts = n * (e * (1 + case["gate"] + case["pre"]) + er + eo) + weights
        if not case["train"]:
            return {"bytes": byts, "flops": 10 * n}
        byts += n * (e * (1 + case["gate"] + case["pre"]) + er + eo) + weights
        return {"bytes": byts, "flops": 30 * n}
    H, Hk, Dk, Dv = case["H"], case["Hk"], case["Dk"], case["Dv"]
    rows = case["R"] if op == "step" else case["B"] * case["T"]
    tokens = rows * (e * (2 * Hk * Dk + H * Dv) + H * (4 + e))  # q, k, v, log-decay, beta
    out = rows * H * Dv * e
    state = 4 * H * Dk * Dv * (case["R"] if op == "step" else case["B"])
    product = 2 * rows * H * Dk * Dv
    if op == "step":
        return {"bytes": tokens + out + 2 * state + 4 * rows, "flops": 3 * product}
    byts = tokens + out + state * case["init"] + 4 * rows * case["packed"]
    if op == "infer":
        return {"bytes": byts + state, "flops": 3 * product}
    return {"bytes": 2 * byts + tokens - 4 * rows * case["packed"], "flops": 9 * product}


# The same from the definitions in 64 bits.


def _exact_norm(s):
    train = s["case"]["train"]
    x = s["x"].detach().double()
    d = {n: None if s[n] is None else s[n].detach().double()
         for n in ("residual", "post", "gate", "scale", "pre")}
    inv1 = 1 / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS)
    h1 = x * inv1
    n1 = x if d["post"] is None else h1 * d["post"]
    sig = None if d["gate"] is None else 1 / (1 + torch.exp(-d["gate"]))
    act = 1.0 if sig is None else d["gate"] * sig
    m = n1 * act
    scale = 1.0 if d["scale"] is None else d["scale"]
    r = scale * m + (0.0 if d["residual"] is None else d["residual"])
    res = {"r": r}
    inv2 = 1 / torch.sqrt(r.pow(2).mean(-1, keepdim=True) + EPS)
    if d["pre"] is not None:
        res["y"] = r * inv2 * d["pre"]
    if not train:
        return res
    lead = tuple(range(x.dim() - 1))
    dr = s["dr"].double()
    if d["pre"] is not None:
        dy = s["dy"].double()
        h2, t = r * inv2, dy * d["pre"]
        dr = dr + inv2 * (t - h2 * (h2 * t).mean(-1, keepdim=True))
        res["dpre"] = (dy * h2).sum(lead)
    if d["residual"] is not None:
        res["dresidual"] = dr
    if d["scale"] is not None:
        res["dscale"] = (dr * m).sum(lead)
    dm = dr * scale
    if sig is not None:
        res["dgate"] = dm * n1 * sig * (1 + d["gate"] * (1 - sig))
    dn = dm * act
    if d["post"] is None:
        res["dx"] = dn
    else:
        res["dpost"] = (dn * h1).sum(lead)
        t = dn * d["post"]
        res["dx"] = inv1 * (t - h1 * (h1 * t).mean(-1, keepdim=True))
    return res


def _exact_delta(s):
    """Token after token: decay the state, correct it along the key, read it along the query. Backwards the
    same in reverse, with the states of a span of rows made again from the one in front of it."""
    c = s["case"]
    train = c["op"] == "train"
    G, scale = c["H"] // c["Hk"], c["Dk"] ** -0.5
    q, k = (s[n].detach().double().repeat_interleave(G, 2).transpose(0, 1).contiguous()
            for n in ("q", "k"))
    v, beta, alpha = (x.transpose(0, 1).contiguous() for x in (
        s["v"].detach().double(), s["beta"].detach().double(), torch.exp(s["g"].detach().double())))
    T, B, H, Dk = k.shape
    keep = torch.ones(T, B, 1, dtype=torch.float64, device=DEV)
    live = torch.ones_like(keep)
    if s["seq"] is not None:
        seq = s["seq"].T
        live[..., 0] = (seq >= 0).double()
        keep[1:, :, 0] = (seq[1:] == seq[:-1]).double()
    beta, keep = beta * live, keep * live
    a = alpha * keep
    state = torch.zeros(B, H, Dk, c["Dv"], dtype=torch.float64, device=DEV)
    if s["init"] is not None:
        state = s["init"].detach().double()

    def one(state, t):
        old = a[t, ..., None, None] * state
        err = v[t] - (old * k[t, ..., None]).sum(-2)
        return old, err, torch.addcmul(old, k[t, ..., None], (beta[t, ..., None] * err)[..., None, :])

    span = 128
    out, starts = torch.empty_like(v), []
    for t in range(T):
        if t % span == 0:
            starts.append(state)
        state = one(state, t)[2]
        out[t] = (state * q[t, ..., None]).sum(-2) * scale
    out = out * live[..., None]
    if not train:
        return {"out": out.transpose(0, 1), "final": state}
    do = s["do"].double().transpose(0, 1) * live[..., None] * scale
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    dg, dbeta = torch.empty_like(alpha), torch.empty_like(beta)
    ds = torch.zeros_like(state)
    for first in reversed(range(0, T, span)):
        state, kept = starts[first // span], []
        for t in range(first, min(T, first + span)):
            old, err, after = one(state, t)
            kept.append((state, old, err, after))
            state = after
        for t in reversed(range(first, min(T, first + span))):
            before, old, err, after = kept.pop()
            ds = torch.addcmul(ds, q[t, ..., None], do[t, ..., None, :])
            dq[t] = (after * do[t, ..., None, :]).sum(-1)
            du = (ds * k[t, ..., None]).sum(-2)
            db = beta[t, ..., None] * du
            dv[t] = db
            dbeta[t] = (du * err).sum(-1)
            dk[t] = (ds * (beta[t, ..., None] * err)[..., None, :]).sum(-1) - (
                old * db[..., None, :]).sum(-1)
            ds = torch.addcmul(ds, k[t, ..., None], db[..., None, :], value=-1)
            dg[t] = a[t] * (ds * before).sum((-1, -2))
            ds = a[t, ..., None, None] * ds
    one_live = live[..., None]

    def back(x):
        return x.transpose(0, 1)

    def shared(x):  # the heads of one key
        return back(x * one_live).unflatten(2, (c["Hk"], G)).sum(3)

    res = {"out": back(out), "dq": shared(dq), "dk": shared(dk), "dv": back(dv * one_live),
           "dg": back(dg * live), "dbeta": back(dbeta * live)}
    if s["init"] is not None:
        res["dinit"] = ds
    return res


def _exact_step(s):
    c, at = s["case"], s["slots"].long()
    q, k = (s[n].double().repeat_interleave(c["H"] // c["Hk"], 1) for n in ("q", "k"))
    state = s["state"].double()
    old = torch.exp(s["g"].double())[..., None, None] * state[at]
    u = s["beta"].double()[..., None] * (s["v"].double() - torch.matmul(
        k[..., None, :], old).squeeze(-2))
    new = old + k[..., None] * u[..., None, :]
    state[at] = new
    out = torch.matmul(q[..., None, :], new).squeeze(-2) * c["Dk"] ** -0.5
    return {"out": out, "state": state}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("train", "infer"):
        # a row is some tens of launches and some passes over the states, of 5 TB/s at the best
        row = 120e-6 + case["B"] * case["H"] * case["Dk"] * case["Dv"] * 8 * 30 / 2e12
        if case["T"] * row * (3 if case["op"] == "train" else 1) > 20:
            return None
    with torch.no_grad():
        return {"train": _exact_delta, "infer": _exact_delta, "step": _exact_step,
                "norm": _exact_norm}[case["op"]](s)
