"""The serving operators together: prompts, forks, decode steps, releases and compactions of one cache,
against 64 bits, and the paged decode example with all of them."""

from __future__ import annotations

import sys

import pytest
import torch

import metile_amd as mt
from examples import paged_decode
from examples.paged_decode import Batch, Decoder
from tests import serving_reference as ref
from tests.test_gpu_paged import FP8, i32
from tests.test_gpu_paged_decode import CONFIG, Plain

pytestmark = pytest.mark.gpu


class Loop:
    """One layer's cache served by the operators; `held` has the keys and values of each request's
    tokens, as they went in, and `step` compares what each new token attends to."""

    def __init__(self, requests, cache_dtype, dtype=torch.bfloat16, page=8, seed=0):
        self.g = torch.Generator("cuda").manual_seed(seed)
        self.heads, self.kv, self.dim, self.page, self.dtype = 6, 2, 64, page, dtype
        self.pages = 96
        self.caches = [mt.PagedCache.allocate(self.pages, page, self.kv, self.dim, dtype=cache_dtype)
                       for _ in range(2)]
        self.tables = torch.full((requests, 24), -1, dtype=torch.int32, device="cuda")
        self.lengths, self.start = i32([0] * requests), i32([0])
        self.free = torch.randperm(self.pages, generator=self.g, device="cuda").int()
        self.held = [[] for _ in range(requests)]  # (key, value) rows of the caches

    def step(self, new):
        """Tokens of each request: their attention, checked."""
        tokens, counts = sum(new) + 3, i32(new)
        plan = mt.paged_tables(self.lengths, counts, self.tables, self.free, page_size=self.page,
                               tokens=tokens, free_start=self.start)
        self.lengths.copy_(plan.lengths)
        self.start.add_(plan.taken)
        q = torch.randn(tokens, self.heads, self.dim, generator=self.g, device="cuda").to(self.dtype)
        for layer, cache in enumerate(self.caches):
            k, v = (torch.randn(tokens, self.kv, self.dim, generator=self.g, device="cuda").to(self.dtype)
                    for _ in range(2))
            mt.paged_append(k, v, cache, plan.slots)
            if max(new) > 1:
                got, lse = mt.paged_chunk_attention(q, cache, self.tables, plan.lengths, plan.starts,
                                                    return_lse=True)
            else:
                owner = plan.requests.clamp(min=0).long()
                lengths = torch.where(plan.requests >= 0, plan.positions + 1, 0).int()
                got, lse = mt.paged_attention(q, cache, self.tables[owner], lengths, return_lse=True)
            if layer == 0:
                row = 0
                for r, n in enumerate(new):
                    self.held[r] += [(k[row + i], v[row + i]) for i in range(n)]
                    row += n
                self.compare(q, cache, plan, got, lse)

    def compare(self, q, cache, plan, got, lse):
        # each request's tokens as they went in, a request a page of a plain cache
        longest = max(map(len, self.held))
        plain = [torch.zeros(len(self.held), longest, self.kv, self.dim, dtype=cache.key.dtype,
                             device="cuda")
                 for _ in range(2)]
        for r, rows in enumerate(self.held):
            for side, out in enumerate(plain):
                if rows:
                    out[r, :len(rows)] = torch.stack([t[side] for t in rows]).to(out.dtype)
        want, want_lse, tol, lse_tol = ref.chunk_attention(
            q, *plain, torch.arange(len(self.held))[:, None], [len(h) for h in self.held],
            plan.starts.tolist(), self.dim ** -0.5)
        assert bool(((got.double().cpu() - want).abs() <= tol).all())
        live = torch.isfinite(want_lse)
        assert bool(((lse.double().cpu() - want_lse).abs()[live] <= lse_tol[live]).all())
        assert torch.equal(torch.isinf(lse.cpu()), ~live)
        assert self.lengths.tolist() == [len(h) for h in self.held]

    def fork(self, sources, targets, tokens=None):
        plan = mt.paged_fork(self.tables, self.lengths, i32(sources), i32(targets), self.free,
                             page_size=self.page, free_start=self.start,
                             tokens=None if tokens is None else i32(tokens))
        mt.paged_copy(self.caches, plan.sources, plan.targets)
        self.start.add_(plan.taken)
        for i, (s, t) in enumerate(zip(sources, targets)):
            self.held[t] = self.held[s][:tokens[i] if tokens else None]

    def release(self, kept):
        freed = mt.paged_free(self.tables, self.lengths, i32(kept), self.free, page_size=self.page,
                              pages=self.pages, free_start=self.start)
        self.start.sub_(freed)
        self.lengths.copy_(i32(kept))
        self.held = [h[:n] for h, n in zip(self.held, kept)]
        used = ref.in_use(self.tables.tolist(), kept, self.page, self.pages)
        assert int(self.start) == len(used)
        assert used.isdisjoint(self.free.tolist()[int(self.start):])

    def compact(self):
        plan = mt.paged_compact(self.tables, self.lengths, self.free, page_size=self.page,
                                pages=self.pages, free_start=self.start)
        mt.paged_copy(self.caches, plan.sources, plan.targets)
        self.tables.copy_(plan.block_tables)
        self.free.copy_(plan.free_pages)
        used = ref.in_use(self.tables.tolist(), self.lengths.tolist(), self.page, self.pages)
        assert used == set(range(int(self.start)))


@pytest.mark.parametrize("cache", [torch.bfloat16, FP8])
def test_operators_together(cache):
    loop = Loop(6, cache)
    loop.step([37, 0, 16, 0, 0, 5])                 # prompts
    loop.fork([0, 0, 2], [1, 3, 4])                 # answered several times
    loop.step([1, 1, 1, 1, 1, 1])
    loop.step([4, 9, 1, 0, 2, 30])                  # drafts, and the rest of a prompt
    loop.release([38, 41, 0, 38, 18, 36])           # drafts taken back, one request ends
    loop.step([1, 1, 0, 1, 1, 1])
    loop.compact()
    loop.step([1, 1, 40, 1, 0, 1])                  # another takes its place
    loop.release([0, len(loop.held[1]), 40, 0, 0, 0])
    loop.fork([1, 1, 2], [0, 3, 5], [20, 33, 16])   # from the middle of what there is
    loop.compact()
    loop.step([3, 1, 1, 7, 2, 1])
    loop.step([1, 1, 1, 1, 1, 0])
    loop.release([0] * 6)
    assert int(loop.start) == 0 and sorted(loop.free.tolist()) == list(range(loop.pages))


@pytest.mark.parametrize("cache,bound", [(None, 0.03), (FP8, 0.12)])
def test_example_against_a_plain_decoder(cache, bound):
    # 16-bit activations round some ten times a layer (2^-9 of the value in the mean): 0.01 to
    # 0.02 of the logits over two layers. 8-bit keys and values add 2^-5 of theirs in each layer.
    decoder = Decoder(CONFIG, seed=3)
    batch = Batch(decoder, 4, pages=40, page_size=4, longest=40, cache_dtype=cache)
    plain = Plain(decoder)
    lengths = [0] * 4

    def prefill(counts):
        tokens = torch.randint(CONFIG.vocab, (sum(counts),), device="cuda")
        logits, scores = batch.prefill(tokens, i32(counts), score=True)
        at = 0
        for r, n in enumerate(counts):
            want = None
            for i in range(n):
                token = int(tokens[at + i])
                if i:
                    # (a log probability is off by at most twice the largest error of a logit, and the
                    # errors that `bound` allows spread evenly: eight times their root mean square)
                    lp = torch.log_softmax(want, 0)[token]
                    assert abs(float(scores[at + i]) - float(lp)) <= 16 * bound * float(want.std() + 1)
                else:
                    assert float(scores[at]) == float("-inf")
                want = plain.step(r, token, lengths[r])
                lengths[r] += 1
            at += n
            if n:
                off = (logits[r].double() - want).norm() / want.norm()
                assert float(off) < bound, (r, float(off))
        assert batch.lengths.tolist() == lengths
        return logits

    def fork(source, target):
        batch.fork(i32([source]), i32([target]))
        lengths[target] = lengths[source]
        for i in range(CONFIG.layers):
            plain.past[target, i] = list(plain.past[source, i])

    def step(active):
        batch.active.copy_(torch.tensor(active))
        tokens = batch.tokens.tolist()
        before = batch.scores.clone()
        logits = batch.step()
        batch.choose_scored(logits)
        for r in range(4):
            if active[r]:
                want = plain.step(r, tokens[r], lengths[r])
                lengths[r] += 1
                off = (logits[r].double() - want).norm() / want.norm()
                assert float(off) < bound, (r, float(off))
                best = torch.log_softmax(logits[r].double(), 0).max()
                assert abs(float(batch.scores[r] - before[r]) - float(best)) < 1e-4
                assert int(batch.tokens[r]) == int(logits[r].argmax())
            else:
                assert int(batch.tokens[r]) == tokens[r] and batch.scores[r] == before[r]
        assert batch.lengths.tolist() == lengths

    prefill([9, 0, 3, 0])
    fork(0, 1)
    prefill([0, 2, 6, 0])
    step([1, 1, 1, 0])
    fork(2, 3)
    step([1, 1, 0, 1])
    batch.release(i32([0, lengths[1], 0, lengths[3]]))
    lengths[0] = lengths[2] = 0
    for i in range(CONFIG.layers):
        plain.past[0, i], plain.past[2, i] = [], []
    batch.compact()
    prefill([0, 0, 5, 2])
    step([0, 1, 1, 1])


def test_answers_begin_with_the_likeliest_tokens():
    decoder = Decoder(CONFIG, seed=1)
    batch = Batch(decoder, 6, pages=40, page_size=4, longest=30)
    tokens = torch.randint(CONFIG.vocab, (14,), device="cuda")
    logits = batch.prefill(tokens, i32([6, 0, 0, 8, 0, 0]))
    batch.answer(3, logits)
    assert batch.lengths.tolist() == [6] * 3 + [8] * 3
    for r in (0, 3):
        want = torch.log_softmax(logits[r].double(), 0)
        first = sorted(range(CONFIG.vocab), key=lambda t: (-float(want[t]), t))[:3]
        assert batch.tokens[r:r + 3].tolist() == first
        assert torch.allclose(batch.scores[r:r + 3].double(), want[first], atol=1e-5)
    # one full page that three share and one of each; two full ones that three share
    assert int(batch.taken) == 1 + 3 + 2


@pytest.mark.parametrize("cache", ["bf16", "fp8"])
def test_example_runs(cache, capsys, monkeypatch):
    monkeypatch.setattr(sys, "argv", ["paged_decode.py", "--requests", "6", "--steps", "5", "--layers", "1",
                                      "--prompt", "50", "--answers", "3", "--cache", cache])
    paged_decode.main()
    said = capsys.readouterr().out
    assert "100 tokens of prompts" in said and "lengths [56]" in said
    assert "the likeliest answers hold 8 pages" in said
