"""Several generations decoded from one paged key-value cache.

A small decoder with random weights (RMSNorm, grouped-query attention with
rotary positions and a sliding window, SwiGLU, a head tied with the
embeddings, as crates/llm-core/src/model.rs has them) serves a batch of
prompts. A step is

  PagePool.plan        pages, slots and positions for the new tokens
  KVCache.append       each layer's rotated keys, and its values, into them
  KVCache.attend       each layer's attention over a request's pages
  Sampler.sample_tied_head_device   logits and the next token

with everything on the device. Prompts go in one token a step, as the
reference's prefill does (model.rs:311-322); requests end at their own
lengths and give their pages back.

With --dtype i8 the caches are of 8 bits with a scale for each block of tokens
(BlockKVCache), which follow from what is written.

  python examples/paged_decode.py [--dtype bf16|f16|f32|e4m3|i8] [--steps N]
"""
from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from scriptonait_amd.kv import KVCache, PagePool, Rope  # noqa: E402
from scriptonait_amd.kv_blocks import BlockKVCache  # noqa: E402
from scriptonait_amd.sampler import Sampler, SamplingConfig  # noqa: E402


class Decoder:
    """Weights of a small decoder, and its caches."""

    def __init__(self, sampler, vocab=1000, hidden=256, layers=2, heads=8, kv_heads=2, window=48, theta=10000.0, batch=4,
                 context=96, page_size=16, pages=24, dtype="bf16", seed=0):
        dev = torch.device("cuda:0")
        g = torch.Generator().manual_seed(seed)
        self.dtype = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "e4m3": torch.bfloat16,
                      "i8": torch.bfloat16}[dtype]
        cached = torch.float8_e4m3fn if dtype == "e4m3" else self.dtype
        self.sampler, self.hidden, self.heads, self.kv_heads, self.window = sampler, hidden, heads, kv_heads, window
        self.dim = hidden // heads
        rnd = lambda *s: (torch.randn(*s, generator=g) / math.sqrt(s[0])).to(dev, self.dtype)  # noqa: E731
        self.embed = (torch.randn(vocab, hidden, generator=g) / math.sqrt(hidden)).to(dev)
        self.layers = [dict(qkv=rnd(hidden, (heads + 2 * kv_heads) * self.dim), o=rnd(hidden, hidden), up=rnd(hidden, 4 * hidden),
                            gate=rnd(hidden, 4 * hidden), down=rnd(4 * hidden, hidden)) for _ in range(layers)]
        self.rope = Rope(self.dim, theta, "halves")
        self.pool = PagePool(sampler, pages, page_size)
        scales = [torch.full((kv_heads,), 0.02, device=dev) for _ in range(2)] if dtype == "e4m3" else []
        shape = (pages, page_size, kv_heads, self.dim)
        if dtype == "i8":
            blocks = (pages, page_size // math.gcd(page_size, 16), kv_heads)
            self.caches = [BlockKVCache(sampler, *[torch.zeros(shape, dtype=torch.int8, device=dev) for _ in range(2)],
                                        *[torch.zeros(blocks, device=dev) for _ in range(2)]) for _ in range(layers)]
        else:
            self.caches = [KVCache(sampler, *[torch.zeros(shape, device=dev).to(cached) for _ in range(2)], *scales)
                           for _ in range(layers)]
        self.workspace = self.caches[0].workspace(heads)
        i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
        self.lens, self.granted, self.start = i32(batch), i32(batch), i32(batch + 1)
        self.table = i32(batch, context // page_size)
        self.slots, self.positions = torch.zeros(batch, dtype=torch.int64, device=dev), i32(batch)
        self.q = torch.zeros(batch, heads, self.dim, dtype=self.dtype, device=dev)
        self.attended = torch.zeros_like(self.q)

    def plan(self, wants, release):
        """Pages for the requests that add a token (wants: [B] int32 of 0 and
        1); those in release give theirs back. Each request's slot (-1: none)
        and position; the plan packs the tokens that are asked for, this
        example keeps a place for every request."""
        self.pool.plan(self.lens, self.table, self.lens, self.granted, self.start, self.slots, self.positions,
                       new_tokens=wants, release=release)
        place = self.start[:-1].long().clamp(max=len(wants) - 1)
        return torch.where(self.granted > 0, self.slots[place], -1), self.positions[place]

    def forward(self, tokens, slots, positions):
        """The normalized last hidden state after one token for each request."""
        x = self.embed[tokens].to(self.dtype)
        for w, cache in zip(self.layers, self.caches):
            rows = (norm(x) @ w["qkv"]).view(len(tokens), -1, self.dim)
            H, K = self.heads, self.kv_heads
            cache.append(rows[:, H:H + K], rows[:, H + K:], slots, q=rows[:, :H], out_q=self.q, positions=positions,
                         rope=self.rope)
            cache.attend(self.q, self.table, self.lens, self.attended, self.workspace, window=self.window)
            x = x + self.attended.view(len(tokens), -1) @ w["o"]
            y = norm(x)
            x = x + (torch.nn.functional.silu(y @ w["gate"]) * (y @ w["up"])) @ w["down"]
        return norm(x).float()


def norm(x):
    y = x.float()
    return (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-5)).to(x.dtype)


def generate(sampler, prompts, steps, config=None, seeds=None, on_step=None, make=Decoder, **model):
    """Decodes every prompt until it and its new tokens are `steps` long, or
    its own limit (a (prompt, limit) pair) is reached; the token lists. The
    cache has room for all of them, unless `model` says how much it has."""
    prompts = [p if isinstance(p, tuple) else (p, steps) for p in prompts]
    B, dev = len(prompts), torch.device("cuda:0")
    page = model.setdefault("page_size", 16)
    model.setdefault("context", -(-steps // page) * page)
    model.setdefault("pages", B * (model["context"] // page))
    m = make(sampler, batch=B, **model)
    config = SamplingConfig(temperature=0.8, top_k=20, repetition_penalty=1.0) if config is None else config
    rng = torch.tensor(np.arange(B) if seeds is None else seeds, dtype=torch.int64, device=dev)
    ids = torch.zeros(B, dtype=torch.int32, device=dev)
    told = torch.zeros(B, steps, dtype=torch.int32, device=dev)
    for b, (p, _) in enumerate(prompts):
        told[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
    given = torch.tensor([len(p) for p, _ in prompts], device=dev)
    limit = torch.tensor([min(n, steps) for _, n in prompts], device=dev)
    refused = torch.zeros((), dtype=torch.bool, device=dev)
    for t in range(steps):
        wants = (limit > t).int()
        slots, positions = m.plan(wants, (limit == t).int())
        refused |= (m.granted < wants).any()
        hidden = m.forward(told[:, t].long(), slots, positions)
        if on_step is not None:
            on_step(t, hidden)
        sampler.sample_tied_head_device(hidden, m.embed, config.to_params(), rng, ids)
        if t + 1 < steps:
            told[:, t + 1] = torch.where((t + 1 >= given) & (t + 1 < limit), ids, told[:, t + 1])
    torch.cuda.synchronize()
    if sampler.status().flags:
        raise RuntimeError("a kernel flagged its input")
    if refused:  # such a token is in no cache: what followed did not see it
        raise RuntimeError("the cache had no room for a token")
    return [told[b, :int(limit[b])].tolist() for b in range(B)], m


def main():
    a = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    a.add_argument("--dtype", choices=["bf16", "f16", "f32", "e4m3", "i8"], default="bf16")
    a.add_argument("--steps", type=int, default=64)
    args = a.parse_args()
    prompts = [([1, 2, 3], args.steps), ([10, 11, 12, 13, 14], args.steps // 2), ([7], args.steps), ([5, 6], args.steps * 3 // 4)]
    with Sampler(0) as s:
        out, m = generate(s, prompts, args.steps, dtype=args.dtype)
    for tokens in out:
        print(tokens)
    print(f"free pages: {int(m.pool.free_state[1])} of {m.pool.pages}")


if __name__ == "__main__":
    main()
