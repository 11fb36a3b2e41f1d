"""A quantized decoder served over a paged key-value cache.

One step takes a token of every request through all layers: block tables and slots from the
requests' lengths (``paged_tables``), then per layer the 4-bit projections (``affine_qmv``), the
cache (``paged_append``, ``paged_attention``), the 4-bit MLP (``affine_mlp``) and the norms around
them (``residual_norm``: each block's own norm, the scaled residual and the next block's norm in one
pass). Lengths, tables and the free list stay on the device, so a step is captured once into a HIP
graph and replayed. Weights are random; prompts go through the same one-token step.

    python examples/paged_decode.py --requests 32 --steps 64
"""

from __future__ import annotations

import argparse
import os
import sys
import time
from dataclasses import dataclass

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import metile_amd as mt  # noqa: E402


@dataclass(frozen=True)
class Config:
    layers: int = 4
    hidden: int = 1536
    inter: int = 8960
    heads: int = 12
    kv_heads: int = 2
    head_dim: int = 128
    vocab: int = 32000
    residual_scale: float = 1.0
    theta: float = 1e6


class Decoder:
    """Random 4-bit weights (MLX affine format, groups of 64) and 16-bit norms."""

    def __init__(self, config: Config, *, dtype=torch.bfloat16, device="cuda", seed=0):
        self.config, self.dtype, self.device = config, dtype, torch.device(device)
        g = torch.Generator(device).manual_seed(seed)
        c = config

        def randn(*shape, scale=1.0, mean=0.0):
            return (torch.randn(*shape, generator=g, device=device) * scale + mean).to(dtype)

        def quantized(n, k):
            return mt.affine_quantize(randn(n, k, scale=k ** -0.5), group_size=64, bits=4)

        heads, kv = c.heads * c.head_dim, c.kv_heads * c.head_dim
        self.embedding = randn(c.vocab, c.hidden)
        self.layers = [dict(qkv=quantized(heads + 2 * kv, c.hidden), out=quantized(c.hidden, heads),
                            gate=quantized(c.inter, c.hidden), up=quantized(c.inter, c.hidden),
                            down=quantized(c.hidden, c.inter),
                            norms=[randn(c.hidden, scale=0.1, mean=1.0) for _ in range(4)])
                       for _ in range(c.layers)]
        self.final_norm = randn(c.hidden, scale=0.1, mean=1.0)
        self.head = quantized(c.vocab, c.hidden)
        self.inverse_frequency = c.theta ** (
            -torch.arange(0, c.head_dim, 2, device=device, dtype=torch.float32) / c.head_dim)

    def rotate(self, x, positions):
        """Rotary embedding of [requests, heads, head_dim] at each request's position."""
        angle = positions.float()[:, None, None] * self.inverse_frequency
        a, b = x.float().chunk(2, dim=-1)
        cos, sin = angle.cos(), angle.sin()
        return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1).to(x.dtype)


class Batch:
    """The requests being served: a cache per layer, one block table, and lengths on the device."""

    def __init__(self, decoder: Decoder, requests, *, pages, page_size=16, cache_dtype=None,
                 longest=None):
        c, device = decoder.config, decoder.device
        self.decoder = decoder
        self.caches = [mt.PagedCache.allocate(pages, page_size, c.kv_heads, c.head_dim,
                                              dtype=cache_dtype or decoder.dtype, device=device)
                       for _ in range(c.layers)]
        width = -(-(longest or pages * page_size) // page_size)
        self.page_size = page_size
        self.tables = torch.full((requests, width), -1, dtype=torch.int32, device=device)
        self.free = torch.arange(pages, dtype=torch.int32, device=device)
        self.taken = torch.zeros(1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(requests, dtype=torch.int32, device=device)
        self.tokens = torch.zeros(requests, dtype=torch.int64, device=device)
        self.active = torch.ones(requests, dtype=torch.int32, device=device)

    def step(self):
        """Logits of every request's next token; ``self.tokens`` of the active ones enter the cache."""
        d, c = self.decoder, self.decoder.config
        requests = self.tokens.shape[0]
        # a token of every active request, in order: the packed batch has a row for each request,
        # and rows of idle ones (and padding behind the last) have no slot
        plan = mt.paged_tables(self.lengths, self.active, self.tables, self.free,
                               page_size=self.page_size, tokens=requests, free_start=self.taken)
        # (rows are packed: row t is request plan.requests[t])
        owner = plan.requests.clamp(min=0).long()
        residual = d.embedding[self.tokens[owner]]
        tables, lengths = self.tables[owner], torch.where(plan.requests >= 0, plan.positions + 1, 0)
        residual, h = mt.residual_norm(residual, weight=d.layers[0]["norms"][0])
        for i, (layer, cache) in enumerate(zip(d.layers, self.caches)):
            heads, kv = c.heads * c.head_dim, c.kv_heads * c.head_dim
            q, k, v = mt.affine_qmv(h, *layer["qkv"]).split([heads, kv, kv], dim=1)
            q = d.rotate(q.unflatten(1, (c.heads, c.head_dim)), plan.positions)
            k = d.rotate(k.unflatten(1, (c.kv_heads, c.head_dim)), plan.positions)
            mt.paged_append(k, v.unflatten(1, (c.kv_heads, c.head_dim)), cache, plan.slots)
            mixed = mt.paged_attention(q, cache, tables, lengths.int())
            block = mt.affine_qmv(mixed.flatten(1), *layer["out"])
            norms = layer["norms"]
            residual, h = mt.residual_norm(residual, block, post_weight=norms[1], weight=norms[2],
                                           residual_scale=c.residual_scale)
            block = mt.affine_mlp(h, layer["gate"], layer["up"], layer["down"])
            last = i + 1 == len(d.layers)
            residual, h = mt.residual_norm(
                residual, block, post_weight=norms[3],
                weight=d.final_norm if last else d.layers[i + 1]["norms"][0],
                residual_scale=c.residual_scale)
        packed = mt.affine_qmv(h, *d.head)
        logits = torch.zeros(requests + 1, c.vocab, dtype=packed.dtype, device=packed.device)
        logits[torch.where(plan.requests >= 0, plan.requests.long(), requests)] = packed
        self.lengths.copy_(plan.lengths)
        self.taken.add_(plan.taken)
        return logits[:requests]

    def choose(self, logits):
        """Greedy next tokens of the active requests in place; idle ones keep theirs."""
        self.tokens.copy_(torch.where(self.active > 0, logits.argmax(-1), self.tokens))


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--requests", type=int, default=32)
    p.add_argument("--steps", type=int, default=64)
    p.add_argument("--layers", type=int, default=Config.layers)
    p.add_argument("--cache", choices=("bf16", "fp8"), default="bf16")
    a = p.parse_args()
    decoder = Decoder(Config(layers=a.layers))
    pages = a.requests * -(-(a.steps + 2) // 16)
    batch = Batch(decoder, a.requests, pages=pages, longest=a.steps + 2,
                  cache_dtype=torch.float8_e4m3fn if a.cache == "fp8" else None)
    batch.tokens.copy_(torch.arange(a.requests) + 1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        batch.choose(batch.step())  # once outside capture: the stream's workspace
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            batch.choose(batch.step())
        stream.synchronize()
        began = time.perf_counter()
        for _ in range(a.steps):
            graph.replay()
        stream.synchronize()
        seconds = time.perf_counter() - began
    print(f"{a.requests} requests, {a.layers} layers, {a.steps} steps: "
          f"{1e3 * seconds / a.steps:.3f} ms a step, {a.requests * a.steps / seconds:.0f} tokens/s, "
          f"lengths {batch.lengths.unique().tolist()}, pages taken {int(batch.taken)} of {pages}")


if __name__ == "__main__":
    main()
