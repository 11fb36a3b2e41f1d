"""A quantized decoder served over a paged key-value cache.

One step takes a token of every request through all layers: block tables and slots from the
requests' lengths (``paged_tables``), then per layer the 4-bit projections (``affine_qmv``), the
cache (``paged_append``, ``paged_attention``), the 4-bit MLP (``affine_mlp``) and the norms around
them (``residual_norm``: each block's own norm, the scaled residual and the next block's norm in one
pass). Lengths, tables and the free list stay on the device, so a step is captured once into a HIP
graph and replayed. Weights are random.

Prompts go through the layers at once (``paged_chunk_attention``), or token by token through the same
step. A prompt can be answered several times: its requests share its full pages (``paged_fork``,
``paged_copy``) and begin with different tokens (``token_logprobs``), whose log probabilities are summed
up. Requests that end give back their pages (``paged_free``), and those in use can be put together
(``paged_compact``).

    python examples/paged_decode.py --requests 32 --steps 64
    python examples/paged_decode.py --requests 32 --steps 64 --prompt 1000 --answers 4
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
        self.missing = torch.zeros(1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(requests, dtype=torch.int32, device=device)
        self.tokens = torch.zeros(requests, dtype=torch.int64, device=device)
        self.active = torch.ones(requests, dtype=torch.int32, device=device)
        self.scores = torch.zeros(requests, dtype=torch.float32, device=device)

    def take(self, pages):
        """Counts pages that were taken: the list's end where it held fewer, and how many were missing."""
        most = self.free.shape[0]
        self.missing.add_((self.taken + pages - most).clamp(min=0))
        self.taken.add_(pages).clamp_(max=most)

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
        tables, lengths = self.tables[owner], torch.where(plan.requests >= 0, plan.positions + 1, 0)
        h = self.layers(self.tokens[owner], plan, lambda q, cache: mt.paged_attention(
            q, cache, tables, lengths.int()))
        packed = mt.affine_qmv(h, *d.head)
        logits = torch.zeros(requests + 1, c.vocab, dtype=packed.dtype, device=packed.device)
        logits[torch.where(plan.requests >= 0, plan.requests.long(), requests)] = packed
        self.lengths.copy_(plan.lengths)
        self.take(plan.taken)
        return logits[:requests]

    def layers(self, tokens, plan, attend):
        """The last norm of a packed batch of tokens, which enter the cache."""
        d, c = self.decoder, self.decoder.config
        residual = d.embedding[tokens]
        residual, h = mt.residual_norm(residual, weight=d.layers[0]["norms"][0])
        for i, (layer, cache) in enumerate(zip(d.layers, self.caches)):
            heads, kv = c.heads * c.head_dim, c.kv_heads * c.head_dim
            q, k, v = mt.affine_qmv(h, *layer["qkv"]).split([heads, kv, kv], dim=1)
            q = d.rotate(q.unflatten(1, (c.heads, c.head_dim)), plan.positions)
            k = d.rotate(k.unflatten(1, (c.kv_heads, c.head_dim)), plan.positions)
            mt.paged_append(k, v.unflatten(1, (c.kv_heads, c.head_dim)), cache, plan.slots)
            mixed = attend(q, cache)
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
        return h

    def prefill(self, tokens, counts, *, score=False):
        """Logits behind the last of each request's next ``counts`` tokens (int32 ``[requests]``; the
        packed ``tokens`` are int64), which enter the cache. With ``score`` also the log probability of
        each of ``tokens`` but a request's first (-inf there)."""
        d = self.decoder
        plan = mt.paged_tables(self.lengths, counts, self.tables, self.free,
                               page_size=self.page_size, tokens=tokens.shape[0],
                               free_start=self.taken)
        h = self.layers(tokens, plan, lambda q, cache: mt.paged_chunk_attention(
            q, cache, self.tables, plan.lengths, plan.starts))
        self.lengths.copy_(plan.lengths)
        self.take(plan.taken)
        last = plan.starts[1:].long() - 1
        logits = mt.affine_qmv(h[last.clamp(min=0)], *d.head)
        if not score:
            return logits
        # (row t has the distribution of token t + 1, if that is the same request's)
        first = torch.ones_like(tokens, dtype=torch.bool)
        first[1:] = plan.requests[1:] != plan.requests[:-1]
        after = torch.where(first, -1, tokens).roll(-1)
        scores = mt.token_logprobs(mt.affine_qmv(h, *d.head), after).logprobs.roll(1)
        return logits, torch.where(first, float("-inf"), scores)

    def fork(self, sources, targets):
        """Requests ``targets`` (int32) go on from the tokens of ``sources``."""
        plan = mt.paged_fork(self.tables, self.lengths, sources, targets, self.free,
                             page_size=self.page_size, free_start=self.taken)
        mt.paged_copy(self.caches, plan.sources, plan.targets)
        self.take(plan.taken)
        self.tokens[targets.long()] = self.tokens[sources.long()]
        self.scores[targets.long()] = self.scores[sources.long()]

    def release(self, kept):
        """Requests give back the pages behind their first ``kept`` tokens (int32 ``[requests]``)."""
        pages = self.caches[0].pages
        freed = mt.paged_free(self.tables, self.lengths, kept, self.free, page_size=self.page_size,
                              pages=pages, free_start=self.taken)
        self.taken.sub_(freed)
        self.lengths.copy_(kept)

    def compact(self):
        """The pages in use become the lowest ones."""
        plan = mt.paged_compact(self.tables, self.lengths, self.free, page_size=self.page_size,
                                pages=self.caches[0].pages, free_start=self.taken)
        mt.paged_copy(self.caches, plan.sources, plan.targets)
        self.tables.copy_(plan.block_tables)
        self.free.copy_(plan.free_pages)

    def choose(self, logits):
        """Greedy next tokens of the active requests in place; idle ones keep theirs."""
        self.tokens.copy_(torch.where(self.active > 0, logits.argmax(-1), self.tokens))

    def choose_scored(self, logits):
        """The same, and the log probabilities of the chosen tokens onto ``self.scores``."""
        best = mt.token_logprobs(logits, top=1)
        on = self.active > 0
        self.tokens.copy_(torch.where(on, best.top_tokens[:, 0], self.tokens))
        self.scores.add_(torch.where(on, best.top_logprobs[:, 0], 0.0))

    def answer(self, answers, logits):
        """Requests ``answers * r`` have prompts, whose last logits these are: those behind each go on
        from its tokens, with the likeliest next token, the second, and so on."""
        requests = self.tokens.shape[0]
        rows = torch.arange(requests, dtype=torch.int32, device=self.tokens.device)
        at = rows % answers
        self.fork((rows - at)[at > 0], rows[at > 0])
        best = mt.token_logprobs(logits[::answers], top=answers)
        self.tokens.copy_(best.top_tokens.flatten()[:requests])
        self.scores.copy_(best.top_logprobs.flatten()[:requests])


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--requests", type=int, default=32)
    p.add_argument("--steps", type=int, default=64)
    p.add_argument("--layers", type=int, default=Config.layers)
    p.add_argument("--cache", choices=("bf16", "fp8"), default="bf16")
    p.add_argument("--prompt", type=int, default=0, help="tokens of each request's prompt")
    p.add_argument("--answers", type=int, default=1, help="requests that answer one prompt")
    a = p.parse_args()
    if a.answers < 1 or a.answers > 32 or a.requests % a.answers or (a.answers > 1 and not a.prompt):
        p.error("answers must be 1 to 32 of a prompt and divide the requests")
    decoder = Decoder(Config(layers=a.layers))
    longest = a.prompt + a.steps + 2
    pages = a.requests * -(-longest // 16)
    batch = Batch(decoder, a.requests, pages=pages, longest=longest,
                  cache_dtype=torch.float8_e4m3fn if a.cache == "fp8" else None)
    batch.tokens.copy_(torch.arange(a.requests) + 1)
    choose = batch.choose
    if a.prompt:
        choose = batch.choose_scored
        counts = torch.zeros_like(batch.lengths)
        counts[::a.answers] = a.prompt
        tokens = torch.randint(decoder.config.vocab, (a.requests // a.answers * a.prompt,), device="cuda")
        batch.prefill(tokens, counts)  # once before the clock runs
        batch.release(torch.zeros_like(counts))
        torch.cuda.synchronize()
        began = time.perf_counter()
        batch.answer(a.answers, batch.prefill(tokens, counts))
        torch.cuda.synchronize()
        seconds = time.perf_counter() - began
        print(f"{tokens.shape[0]} tokens of prompts: {1e3 * seconds:.3f} ms, "
              f"{tokens.shape[0] / seconds:.0f} tokens/s")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        choose(batch.step())  # once outside capture: the stream's workspace
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            choose(batch.step())
        stream.synchronize()
        began = time.perf_counter()
        for _ in range(a.steps):
            graph.replay()
        stream.synchronize()
        seconds = time.perf_counter() - began
    print(f"{a.requests} requests, {a.layers} layers, {a.steps} steps: "
          f"{1e3 * seconds / a.steps:.3f} ms a step, {a.requests * a.steps / seconds:.0f} tokens/s, "
          f"lengths {batch.lengths.unique().tolist()}, pages taken {int(batch.taken)} of {pages}"
          + (f", {int(batch.missing)} missing" if int(batch.missing) else ""))
    if a.answers > 1:
        best = batch.scores.view(-1, a.answers).argmax(1, keepdim=True)
        kept = torch.arange(a.answers, device="cuda") == best
        batch.release(torch.where(kept.flatten(), batch.lengths, 0).int())
        batch.compact()
        print(f"the likeliest answers hold {int(batch.taken)} pages")


if __name__ == "__main__":
    main()
