"""The paged decode example, step by step against a decoder in 64 bits that keeps its history in plain
tensors, with requests that start and stop, in both cache types and from a replayed graph."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import metile_amd as mt
from examples.paged_decode import Batch, Config, Decoder

pytestmark = pytest.mark.gpu

CONFIG = Config(layers=2, hidden=256, inter=512, heads=6, kv_heads=2, head_dim=64, vocab=320,
                residual_scale=0.75)


class Plain:
    """The same decoder in 64 bits on dequantized weights; keys and values as lists."""

    def __init__(self, decoder):
        self.d, self.c = decoder, decoder.config
        self.past = {}

    def weight(self, triple):
        w, s, b = triple
        return mt.affine_dequantize(w, s, b, group_size=64, bits=4).double()

    def norm(self, x, w):
        return x / torch.sqrt((x * x).mean() + 1e-6) * w.double()

    def rotate(self, x, position):
        angle = position * self.d.inverse_frequency.double()
        a, b = x.chunk(2, dim=-1)
        return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1)

    def step(self, request, token, position):
        c, d = self.c, self.d
        x = d.embedding[token].double()
        for i, layer in enumerate(d.layers):
            n = layer["norms"]
            h = self.norm(x, n[0])
            q, k, v = (self.weight(layer["qkv"]) @ h).split(
                [c.heads * c.head_dim, c.kv_heads * c.head_dim, c.kv_heads * c.head_dim])
            past = self.past.setdefault((request, i), [])
            past.append((self.rotate(k.view(c.kv_heads, -1), position), v.view(c.kv_heads, -1)))
            q = self.rotate(q.view(c.heads, -1), position)
            keys, values = (torch.stack([p[j] for p in past]).repeat_interleave(
                c.heads // c.kv_heads, 1) for j in (0, 1))
            p = torch.softmax((keys * q).sum(-1) * c.head_dim ** -0.5, 0)
            block = self.weight(layer["out"]) @ (p[..., None] * values).sum(0).flatten()
            x = c.residual_scale * x + self.norm(block, n[1])
            h = self.norm(x, n[2])
            gate = self.weight(layer["gate"]) @ h
            block = self.weight(layer["down"]) @ (
                torch.nn.functional.silu(gate) * (self.weight(layer["up"]) @ h))
            x = c.residual_scale * x + self.norm(block, n[3])
        return self.weight(d.head) @ self.norm(x, d.final_norm)


@pytest.mark.parametrize("cache,bound", [(None, 0.03), (torch.float8_e4m3fn, 0.12)])
def test_steps_against_a_plain_decoder(cache, bound):
    # 16-bit activations round some ten times a layer (2^-9 of the value in the mean): 0.01 to
    # 0.02 of the logits over two layers. 8-bit keys and values add 2^-5 of theirs in each layer.
    decoder = Decoder(CONFIG, seed=3)
    batch = Batch(decoder, 3, pages=12, page_size=4, longest=24, cache_dtype=cache)
    plain = Plain(decoder)
    rng = np.random.RandomState(0)
    lengths = [0, 0, 0]
    for step in range(9):
        active = [1, int(step >= 2), int(step % 3 != 1)]
        tokens = rng.randint(0, CONFIG.vocab, 3)
        batch.tokens.copy_(torch.from_numpy(tokens))
        batch.active.copy_(torch.tensor(active))
        logits = batch.step()
        for r in range(3):
            if not active[r]:
                continue
            want = plain.step(r, int(tokens[r]), lengths[r])
            lengths[r] += 1
            off = (logits[r].double() - want).norm() / want.norm()
            assert float(off) < bound, (step, r, float(off))
        assert batch.lengths.tolist() == lengths
    assert int(batch.taken) == sum(-(-n // 4) for n in lengths)
    used = [p for p in batch.tables.flatten().tolist() if p >= 0]
    assert sorted(used) == list(range(int(batch.taken)))


def test_graph_replays_match_eager_steps():
    decoder = Decoder(CONFIG, seed=5)
    eager, graphed = (Batch(decoder, 2, pages=12, page_size=4, longest=24) for _ in range(2))
    for b in (eager, graphed):
        b.tokens.copy_(torch.tensor([5, 17]))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for b in (eager, graphed):
            b.choose(b.step())
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            logits = graphed.step()
            graphed.choose(logits)
        for _ in range(12):
            graph.replay()
            want = eager.step()
            eager.choose(want)
            stream.synchronize()
            assert torch.equal(logits, want)
            assert graphed.tokens.tolist() == eager.tokens.tolist()
    assert graphed.lengths.tolist() == eager.lengths.tolist() == [13, 13]
