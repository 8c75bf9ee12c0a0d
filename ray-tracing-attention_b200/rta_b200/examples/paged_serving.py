"""Serve samples of one prompt from a paged K/V cache: prefill in chunks, fork, decode, free, compact.

    python -m rta_b200.examples.paged_serving [--prompt 700] [--samples 6] [--tokens 24]

A small random attention model (rotary positions, grouped K/V heads, a sliding window with the first tokens kept) reads
a prompt in chunks, the sequence is forked into `samples` continuations that share its full pages, every decode step --
reserve, per layer append and decode, readout -- is one CUDA graph, half of the samples end early and their pages are
given back, and the others go on in a compacted pool.  The hidden states of the survivors are compared with the same
model computed without a cache.
"""
from __future__ import annotations

import argparse

import torch

from ..paged import PagedCache


class Model:
    """Attention layers only: h += Wo attention(Wq h, Wk h, Wv h)."""

    def __init__(self, layers=3, hidden=512, heads=8, kv_heads=2, head_dim=128, vocab=1000, window=256, sinks=4, seed=0,
                 device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)

        def rand(*shape):
            return (torch.randn(*shape, generator=g, device=device) * shape[0] ** -0.5).bfloat16()

        self.layers, self.heads, self.kv_heads, self.head_dim = layers, heads, kv_heads, head_dim
        self.window, self.sinks = window, sinks
        self.qkv = [rand(hidden, (heads + 2 * kv_heads) * head_dim) for _ in range(layers)]
        self.out = [rand(heads * head_dim, hidden) for _ in range(layers)]
        self.embed, self.read = rand(vocab, hidden) * vocab ** 0.5, rand(hidden, vocab)
        self.freq = 10000.0 ** (-torch.arange(0, head_dim, 2, device=device) / head_dim)

    def project(self, layer, h, positions):
        """q, k (rotated) and v of rows h at their positions, views of one projection."""
        x = (h @ self.qkv[layer]).view(h.shape[0], self.heads + 2 * self.kv_heads, self.head_dim)
        turned = x[:, :self.heads + self.kv_heads]
        angle = positions[:, None, None] * self.freq
        cos, sin = angle.cos(), angle.sin()
        a, b = turned[..., 0::2].float(), turned[..., 1::2].float()
        turned[..., 0::2], turned[..., 1::2] = (a * cos - b * sin).bfloat16(), (a * sin + b * cos).bfloat16()
        return x[:, :self.heads], x[:, self.heads:self.heads + self.kv_heads], x[:, self.heads + self.kv_heads:]

    def mix(self, layer, h, attention):
        return h + attention.reshape(h.shape[0], -1) @ self.out[layer]

    def logits(self, h):
        return h.float() @ self.read.float()

    def plain(self, tokens):
        """Hidden states of a whole sequence without a cache, attention in fp32."""
        h = self.embed[tokens]
        t = torch.arange(len(tokens), device=h.device)
        see = (t[None] <= t[:, None]) & ((t[None] > t[:, None] - self.window) | (t[None] < self.sinks))
        for layer in range(self.layers):
            q, k, v = (x.float().transpose(0, 1) for x in self.project(layer, h, t))
            group = self.heads // self.kv_heads
            s = q @ k.repeat_interleave(group, 0).transpose(1, 2) * self.head_dim ** -0.5
            a = s.masked_fill(~see, float("-inf")).softmax(-1) @ v.repeat_interleave(group, 0)
            h = self.mix(layer, h, a.transpose(0, 1).bfloat16())
        return h


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def serve(prompt=700, samples=6, tokens=24, chunk=256, page_size=16, seed=0):
    """Runs the program; returns the tokens of the surviving samples and the worst relative error of their states."""
    model = Model(seed=seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    ids = torch.randint(0, model.embed.shape[0], (prompt,), generator=g, device="cuda")
    longest = prompt + 2 * tokens + page_size
    pages = -(-longest // page_size) + samples * (2 + 2 * tokens // page_size + 1)
    cache = PagedCache.create(model.layers, pages, page_size, model.kv_heads, model.head_dim, samples + 1, longest,
                              torch.bfloat16)
    attention = dict(window=model.window, sinks=model.sinks)

    # the prompt, in chunks, into slot 0
    for first in range(0, prompt, chunk):
        part = ids[first:first + chunk]
        n = len(part)
        cache.reserve(ints(n))
        starts, h = ints(0, n), model.embed[part]
        positions = torch.arange(first, first + n, device="cuda")
        for layer in range(model.layers):
            q, k, v = model.project(layer, h, positions)
            cache.append(k, v, starts, layer=layer)
            h = model.mix(layer, h, cache.prefill(q, starts, layer=layer, **attention))
    last = h[-1]

    # samples 1 .. n share the prompt's pages; sample i begins with the i-th best token
    slots = ints(*range(1, samples + 1))
    cache.fork(ints(*[0] * samples), slots)
    cache.free(ints(0))
    start = model.logits(last[None])[0].topk(samples).indices

    def steps(slots, token, first, count):
        """`count` decode steps of some samples as replays of one graph: their tokens [count][n], the last states."""
        n = len(slots)
        counts, starts = ints(*[1] * n), ints(*range(n + 1))
        token, position = token.clone(), torch.full((n,), first, device="cuda")
        said, state = [], torch.empty(n, model.embed.shape[1], device="cuda", dtype=torch.bfloat16)

        def step():
            cache.reserve(counts, slots)
            h = model.embed[token]
            for layer in range(model.layers):
                q, k, v = model.project(layer, h, position)
                cache.append(k, v, starts, layer=layer, slots=slots)
                h = model.mix(layer, h, cache.decode(q, layer=layer, slots=slots, **attention))
            state.copy_(h)
            token.copy_(model.logits(h).argmax(-1))
            position.add_(1)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            said.append(token.clone())
            step()  # the first step sets the kernels up; the others replay it
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                step()
            for _ in range(count - 1):
                said.append(token.clone())
                graph.replay()
        torch.cuda.current_stream().wait_stream(side)
        cache.check()
        return torch.stack(said), token, state

    said, token, _ = steps(slots, start, prompt, tokens)
    keep = samples - samples // 2
    cache.free(slots[keep:].contiguous())  # half of them have ended
    live = ints(0)
    cache.compact(live=live)
    more, _, state = steps(slots[:keep].contiguous(), token[:keep], prompt + tokens, tokens)
    worst = 0.0
    for i in range(keep):
        whole = torch.cat([ids, said[:, i], more[:, i]])
        want = model.plain(whole)[-1].double()
        worst = max(worst, ((state[i].double() - want).norm() / want.norm()).item())
    used = int((cache.map.refs > 0).sum())
    return torch.cat([said[:, :keep], more]).T, worst, int(live), used, pages


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--prompt", type=int, default=700)
    ap.add_argument("--samples", type=int, default=6)
    ap.add_argument("--tokens", type=int, default=24)
    a = ap.parse_args()
    said, worst, live, used, pages = serve(a.prompt, a.samples, a.tokens)
    print(f"{said.shape[0]} of {a.samples} samples went on to {said.shape[1]} tokens each, the first: {said[0].tolist()}")
    print(f"pages in use after compaction {live}, at the end {used} of {pages}; states within {worst:.2e} of the model "
          "without a cache")


if __name__ == "__main__":
    main()
