"""A small language model of recurrent and attention blocks, trained for a step and served.

A recurrent block is a projection, the causal convolution, the gated linear recurrence over it and a
projection back; an attention block keeps its keys and values in a paged cache. Training runs packed
documents through the recurrent blocks (seq_idx); serving admits requests of any length with
`paged_plan`, runs their prompts, and then one token of every request per step, the recurrent states in
pools of slots. Weights are random; nothing is read from disk.

    python examples/hybrid_serving.py
"""

import math
import os
import sys

import torch
import torch.nn.functional as nnf

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "causal-conv1d-triton_amd"))

from causal_conv1d_triton import causal_conv1d_fn  # noqa: E402
from causal_conv1d_triton.paged import paged_attention, paged_cache_write, paged_plan  # noqa: E402
from causal_conv1d_triton.recurrence import (  # noqa: E402
    gated_recurrence_fn, gated_recurrence_update)

DEV, DT = "cuda", torch.bfloat16


class RecurrentBlock:
    def __init__(self, dim, width, gen):
        self.dim, self.width = dim, width
        n = lambda *s, scale: scale * torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
        self.w_in = n(3 * dim, dim, scale=dim ** -0.5).to(DT)
        self.w_out = n(dim, dim, scale=dim ** -0.5).to(DT)
        self.w_conv, self.b_conv = n(dim, width, scale=width ** -0.5), n(dim, scale=0.1)
        keep = 0.9 + 0.099 * torch.rand(dim, generator=gen, device=DEV)
        self.decay = torch.log(torch.expm1(-torch.log(keep) / 8))

    def parameters(self):
        return [self.w_in, self.w_out, self.w_conv, self.b_conv, self.decay]

    def project(self, x):
        """The convolution's input and the two gates: slices of one projection, used as they are."""
        return nnf.linear(x, self.w_in).split(self.dim, -1)

    def forward(self, x, seq_idx=None):
        u, gate, igate = self.project(x)
        u = causal_conv1d_fn(u, self.w_conv, self.b_conv, seq_idx, activation="silu")
        h = gated_recurrence_fn(u, gate, self.decay, igate, seq_idx)
        return x + nnf.linear(h, self.w_out)

    def states(self, slots):
        return [torch.zeros(slots, self.width - 1, self.dim, device=DEV, dtype=DT),
                torch.zeros(slots, self.dim, device=DEV)]

    def prompt(self, x, state, slot):
        """One request's prompt (1, T, dim); its final states go to its slot."""
        u, gate, igate = self.project(x)
        u, state[0][slot:slot + 1] = causal_conv1d_fn(u, self.w_conv, self.b_conv,
                                                      return_final_states=True, activation="silu")
        h, state[1][slot:slot + 1] = gated_recurrence_fn(u, gate, self.decay, igate,
                                                         return_final_states=True)
        return x + nnf.linear(h, self.w_out)

    def step(self, x, state, slots):
        """One token of each request (R, dim); slots says where its states are."""
        u, gate, igate = self.project(x)
        at = slots.long()
        u, last = causal_conv1d_fn(u[:, None], self.w_conv, self.b_conv,
                                   initial_states=state[0][at], return_final_states=True,
                                   activation="silu")
        state[0].index_copy_(0, at, last)
        h = gated_recurrence_update(u[:, 0], gate, state[1], self.decay, igate, slots)
        return x + nnf.linear(h, self.w_out)


class AttentionBlock:
    def __init__(self, dim, heads, kv_heads, window, gen):
        self.heads, self.kv_heads, self.window = heads, kv_heads, window
        self.head_dim = dim // heads
        rows = (heads + 2 * kv_heads) * self.head_dim
        self.w_qkv = (torch.randn(rows, dim, generator=gen, device=DEV) / math.sqrt(dim)).to(DT)
        self.w_out = (torch.randn(dim, dim, generator=gen, device=DEV) / math.sqrt(dim)).to(DT)

    def cache(self, pages, page_size):
        shape = (pages, page_size, self.kv_heads, self.head_dim)
        return [torch.zeros(shape, device=DEV, dtype=DT) for _ in range(2)]

    def tokens(self, x, cache, tables, plan, places):
        """Any tokens of any requests (N, dim) at the given places of a plan: their keys and values are
        written first, then each attends up to itself."""
        H, K = self.heads, self.kv_heads
        qkv = nnf.linear(x, self.w_qkv).view(-1, H + 2 * K, self.head_dim)
        paged_cache_write(qkv[:, H:H + K], qkv[:, H + K:], *cache, plan.slot_mapping[places])
        out = paged_attention(qkv[:, :H], *cache, tables, plan.positions[places] + 1,
                              window=self.window, request_ids=plan.request_ids[places])
        return x + nnf.linear(out.flatten(1), self.w_out)


class Server:
    """Requests of a fixed number of slots over shared pages."""

    def __init__(self, layers, embed, slots, pages, page_size, max_pages):
        self.layers, self.embed, self.page_size = layers, embed, page_size
        self.state = [b.states(slots) if isinstance(b, RecurrentBlock) else b.cache(pages, page_size)
                      for b in layers]
        self.tables = torch.full((slots, max_pages), -1, device=DEV, dtype=torch.int32)
        self.lens = torch.zeros(slots, device=DEV, dtype=torch.int32)
        self.free = torch.arange(pages, device=DEV, dtype=torch.int32)
        self.num_free = torch.tensor([pages], device=DEV, dtype=torch.int32)

    def plan(self, new_lens, max_tokens):
        plan = paged_plan(self.lens, new_lens, self.tables, self.free, self.num_free, self.page_size,
                          max_tokens)
        self.lens, self.num_free = plan.seq_lens, plan.num_free
        return plan

    @torch.no_grad()
    def prompts(self, prompts):
        """All prompts at once; the logits of each one's last token. Returns the plan too."""
        sizes = [len(p) for p in prompts]
        plan = self.plan(torch.tensor(sizes, device=DEV, dtype=torch.int32), sum(sizes))
        x = self.embed[torch.cat(prompts)]
        for block, state in zip(self.layers, self.state):
            if isinstance(block, RecurrentBlock):
                x = torch.cat([block.prompt(part[None], state, slot)[0]
                               for slot, part in enumerate(x.split(sizes))])
            else:
                x = block.tokens(x, state, self.tables, plan, slice(None))
        return nnf.linear(x[plan.query_start[1:] - 1], self.embed), plan

    @torch.no_grad()
    def step(self, tokens):
        """The next token of every request; its logits."""
        R = tokens.numel()
        plan = self.plan(torch.ones(R, device=DEV, dtype=torch.int32), R)
        x = self.embed[tokens]
        for block, state in zip(self.layers, self.state):
            if isinstance(block, RecurrentBlock):
                x = block.step(x, state, plan.request_ids)
            else:
                x = block.tokens(x, state, self.tables, plan, slice(None))
        return nnf.linear(x, self.embed)


def build(seed=0, dim=256, vocab=512, heads=8, kv_heads=2, window=64, width=4):
    gen = torch.Generator(DEV).manual_seed(seed)
    layers = [RecurrentBlock(dim, width, gen), RecurrentBlock(dim, width, gen),
              AttentionBlock(dim, heads, kv_heads, window, gen), RecurrentBlock(dim, width, gen)]
    embed = torch.randn(vocab, dim, generator=gen, device=DEV).to(DT)
    return layers, embed, gen


def train_step(layers, embed, gen, T=512):
    """Packed documents through the recurrent blocks; the loss and every parameter's gradient."""
    blocks = [b for b in layers if isinstance(b, RecurrentBlock)]
    params = [p.detach().requires_grad_(True) for b in blocks for p in b.parameters()]
    for i, b in enumerate(blocks):
        b.w_in, b.w_out, b.w_conv, b.b_conv, b.decay = params[5 * i:5 * i + 5]
    tokens = torch.randint(0, embed.shape[0], (2, T + 1), generator=gen, device=DEV)
    seq_idx = (torch.arange(T, device=DEV) // 200).int().expand(2, T).contiguous()
    seq_idx[:, -20:] = -1
    x = embed[tokens[:, :-1]]
    for b in blocks:
        x = b.forward(x, seq_idx)
    loss = nnf.cross_entropy(nnf.linear(x, embed).float()[seq_idx >= 0] / math.sqrt(embed.shape[1]),
                             tokens[:, 1:][seq_idx >= 0])
    grads = torch.autograd.grad(loss, params)
    for b in blocks:
        b.w_in, b.w_out, b.w_conv, b.b_conv, b.decay = (p.detach() for p in b.parameters())
    return loss.detach(), grads


def serve(layers, embed, gen, lengths=(37, 5, 70, 1), steps=12):
    """Greedy generation; (tokens of each request, the last logits)."""
    server = Server(layers, embed, len(lengths), pages=64, page_size=16, max_pages=16)
    prompts = [torch.randint(0, embed.shape[0], (n,), generator=gen, device=DEV) for n in lengths]
    logits, _ = server.prompts(prompts)
    said = [list(p) for p in prompts]
    for _ in range(steps):
        tokens = logits.argmax(-1)
        for r, t in enumerate(tokens):
            said[r].append(t)
        logits = server.step(tokens)
    return [torch.stack(s) for s in said], logits


def main():
    layers, embed, gen = build()
    loss, grads = train_step(layers, embed, gen)
    print(f"training step: loss {loss:.3f}, {len(grads)} gradients, largest "
          f"{max(float(g.abs().max()) for g in grads):.3g}")
    said, logits = serve(layers, embed, gen)
    again, _ = Server(layers, embed, len(said), 64, 16, 16).prompts(said)
    off = float((again.float() - logits.float()).norm() / logits.float().norm())
    print(f"served {len(said)} requests of {[len(s) for s in said]} tokens; the same tokens as prompts "
          f"give logits {off:.2e} apart")
    return loss, grads, off


if __name__ == "__main__":
    main()
