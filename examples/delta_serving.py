"""A small language model of gated-delta-rule blocks, trained for a step and served.

A block: a projection to queries, keys, values, an output gate, decays and rates; the causal convolution over the
first three; queries and keys brought to unit length; the gated delta rule; the norm of its heads with the output
gate; a projection back, which joins an fp32 residual stream in the same pass as the next block's norm. Training runs
packed documents (seq_idx); serving runs each prompt, then one token of every request per step with the convolution's
and the rule's states in pools of slots. Weights are random; nothing is read from disk.

    python examples/delta_serving.py
"""

import math
import os
import sys

import torch
import torch.nn.functional as nnf

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "causal-conv1d-triton_amd"))

from causal_conv1d_triton import causal_conv1d_fn  # noqa: E402
from causal_conv1d_triton.delta import gated_delta_fn, gated_delta_update  # noqa: E402
from causal_conv1d_triton.norm import block_norm_fn  # noqa: E402

DEV, DT = "cuda", torch.bfloat16


class DeltaBlock:
    def __init__(self, dim, key_heads, heads, key_dim, value_dim, width, gen):
        self.Hk, self.H, self.Dk, self.Dv = key_heads, heads, key_dim, value_dim
        self.mixed = 2 * key_heads * key_dim + heads * value_dim  # what the convolution sees
        n = lambda *s, scale=1.0: scale * torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
        rows = self.mixed + heads * value_dim + 2 * heads
        self.w_in, self.w_out = n(rows, dim, scale=dim ** -0.5).to(DT), n(dim, heads * value_dim, scale=0.05).to(DT)
        self.w_conv = n(self.mixed, width, scale=width ** -0.5)
        self.rate, self.shift = 1 + 3 * torch.rand(heads, generator=gen, device=DEV), n(heads) - 3
        self.w_head, self.w_next = torch.ones(value_dim, device=DEV), torch.ones(dim, device=DEV)
        self.unit = torch.full((key_dim,), key_dim ** -0.5, device=DEV)  # a norm of one

    NAMES = ("w_in", "w_out", "w_conv", "rate", "shift", "w_head", "w_next")

    def project(self, x):
        mixed, gate, decay, beta = nnf.linear(x, self.w_in).split(
            [self.mixed, self.H * self.Dv, self.H, self.H], -1)
        return mixed, gate.unflatten(-1, (self.H, self.Dv)), -self.rate * nnf.softplus(
            decay.float() + self.shift), torch.sigmoid(beta)

    def heads(self, mixed):
        """Queries, keys and values after the convolution; the first two of unit length."""
        q, k, v = mixed.split([self.Hk * self.Dk, self.Hk * self.Dk, self.H * self.Dv], -1)
        q, k = (block_norm_fn(t.unflatten(-1, (self.Hk, self.Dk)), post_weight=self.unit) for t in (q, k))
        return q, k, v.unflatten(-1, (self.H, self.Dv))

    def back(self, o, gate, residual):
        """The gated norm of the heads, the projection back and the next block's norm: (its input, the stream)."""
        o = block_norm_fn(o, post_weight=self.w_head, gate=gate)
        return block_norm_fn(nnf.linear(o.flatten(-2), self.w_out), residual, pre_weight=self.w_next)

    def forward(self, x, residual, seq_idx=None):
        mixed, gate, decay, beta = self.project(x)
        mixed = causal_conv1d_fn(mixed, self.w_conv, None, seq_idx, activation="silu")
        return self.back(gated_delta_fn(*self.heads(mixed), decay, beta, seq_idx), gate, residual)

    def states(self, slots):
        return [torch.zeros(slots, self.w_conv.shape[1] - 1, self.mixed, device=DEV, dtype=DT),
                torch.zeros(slots, self.H, self.Dk, self.Dv, device=DEV)]

    def prompt(self, x, residual, state, slot):
        mixed, gate, decay, beta = self.project(x)
        mixed, state[0][slot:slot + 1] = causal_conv1d_fn(mixed, self.w_conv, None, return_final_states=True,
                                                          activation="silu")
        o, state[1][slot:slot + 1] = gated_delta_fn(*self.heads(mixed), decay, beta, return_final_states=True)
        return self.back(o, gate, residual)

    def step(self, x, residual, state, slots):
        mixed, gate, decay, beta = self.project(x)
        at = slots.long()
        mixed, last = causal_conv1d_fn(mixed[:, None], self.w_conv, None, initial_states=state[0][at],
                                       return_final_states=True, activation="silu")
        state[0].index_copy_(0, at, last)
        o = gated_delta_update(*self.heads(mixed[:, 0]), decay, beta, state[1], slots)
        return self.back(o, gate, residual)


class Model:
    def __init__(self, seed=0, layers=3, dim=256, vocab=512, key_heads=2, heads=4, key_dim=64, value_dim=64, width=4):
        self.gen = torch.Generator(DEV).manual_seed(seed)
        self.blocks = [DeltaBlock(dim, key_heads, heads, key_dim, value_dim, width, self.gen) for _ in range(layers)]
        self.embed = torch.randn(vocab, dim, generator=self.gen, device=DEV).to(DT)
        self.w_first = torch.ones(dim, device=DEV)

    def start(self, tokens):
        stream = self.embed[tokens].float()
        return block_norm_fn(stream, post_weight=self.w_first).to(DT), stream

    def logits(self, x):
        return nnf.linear(x, self.embed) / math.sqrt(self.embed.shape[1])

    def train_step(self, T=512):
        """Packed documents; the loss and every weight's gradient."""
        kept = [{n: getattr(b, n) for n in b.NAMES} for b in self.blocks]
        params = [t.detach().requires_grad_(True) for k in kept for t in k.values()]
        for b, i in zip(self.blocks, range(0, len(params), len(DeltaBlock.NAMES))):
            for n, p in zip(b.NAMES, params[i:]):
                setattr(b, n, p)
        tokens = torch.randint(0, self.embed.shape[0], (2, T + 1), generator=self.gen, device=DEV)
        seq_idx = (torch.arange(T, device=DEV) // 200).int().expand(2, T).contiguous()
        seq_idx[:, -20:] = -1
        x, stream = self.start(tokens[:, :-1])
        for b in self.blocks:
            x, stream = b.forward(x, stream, seq_idx)
        live = seq_idx >= 0
        loss = nnf.cross_entropy(self.logits(x).float()[live], tokens[:, 1:][live])
        grads = torch.autograd.grad(loss, params)
        for b, k in zip(self.blocks, kept):
            for n, t in k.items():
                setattr(b, n, t)
        return loss.detach(), grads

    @torch.no_grad()
    def prompts(self, prompts, states):
        """The prompts one after the other, request r in slot r; the logits of each one's last token."""
        out = []
        for slot, tokens in enumerate(prompts):
            x, stream = self.start(tokens[None])
            for b, s in zip(self.blocks, states):
                x, stream = b.prompt(x, stream, s, slot)
            out.append(x[0, -1])
        return self.logits(torch.stack(out))

    @torch.no_grad()
    def step(self, tokens, states, slots):
        x, stream = self.start(tokens)
        for b, s in zip(self.blocks, states):
            x, stream = b.step(x, stream, s, slots)
        return self.logits(x)

    def states(self, slots):
        return [b.states(slots) for b in self.blocks]

    def serve(self, lengths=(37, 5, 70, 1), steps=12):
        """Greedy generation; (tokens of each request, the last logits)."""
        prompts = [torch.randint(0, self.embed.shape[0], (n,), generator=self.gen, device=DEV) for n in lengths]
        states, slots = self.states(len(lengths)), torch.arange(len(lengths), device=DEV, dtype=torch.int32)
        logits = self.prompts(prompts, states)
        said = [list(p) for p in prompts]
        for _ in range(steps):
            tokens = logits.argmax(-1)
            for r, t in enumerate(tokens):
                said[r].append(t)
            logits = self.step(tokens, states, slots)
        return [torch.stack(s) for s in said], logits


def main():
    model = Model()
    loss, grads = model.train_step()
    print(f"training step: loss {loss:.3f}, {len(grads)} gradients, largest "
          f"{max(float(g.abs().max()) for g in grads):.3g}")
    said, logits = model.serve()
    again = model.prompts(said, model.states(len(said)))
    off = float((again.float() - logits.float()).norm() / logits.float().norm())
    print(f"served {len(said)} requests of {[len(s) for s in said]} tokens; the same tokens as prompts "
          f"give logits {off:.2e} apart")
    return loss, grads, off


if __name__ == "__main__":
    main()
