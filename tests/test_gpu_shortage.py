"""Free lists that run out: what is there is handed out once, and comes back whole."""

from __future__ import annotations

import pytest
import torch

from examples.paged_decode import Batch, Decoder
from tests.test_gpu_paged import i32
from tests.test_gpu_paged_decode import CONFIG

pytestmark = pytest.mark.gpu


def test_example_comes_back_from_an_exhausted_list():
    """Prompts, forks and steps beyond the pool, then everything is released: each page is free, once."""
    decoder = Decoder(CONFIG, seed=2)
    batch = Batch(decoder, 6, pages=7, page_size=4, longest=40)
    tokens = torch.randint(CONFIG.vocab, (20,), device="cuda")

    def release():
        batch.release(torch.zeros_like(batch.lengths))
        assert int(batch.taken) == 0 and sorted(batch.free.tolist()) == list(range(7))

    batch.prefill(tokens[:10], i32([6, 0, 4, 0, 0, 0]))    # 3 of 7 pages
    assert batch.missing.tolist() == [0]
    batch.fork(i32([0, 0, 0, 2]), i32([1, 3, 4, 5]))       # 3 begun pages more
    batch.choose(batch.step())                             # requests 2 and 5 need a page each: one is there
    assert batch.missing.tolist() == [1]
    batch.release(i32([7, 7, 5, 0, 7, 0]))                 # one page comes back
    batch.fork(i32([0, 0]), i32([3, 5]))                   # and two are wanted
    assert batch.missing.tolist() == [2] and int(batch.taken) == 7
    release()
    batch.prefill(tokens, i32([20, 0, 0, 0, 0, 0]))
    batch.fork(i32([0]), i32([1]))
    batch.prefill(tokens, i32([20, 0, 0, 0, 0, 0]))        # 3 of 5 pages are missing
    assert batch.missing.tolist() == [5]
    batch.compact()
    assert sorted(p for p in batch.tables[0].tolist() if p >= 0) == list(range(7))
    release()
    logits = batch.prefill(tokens[:8], i32([8, 0, 0, 0, 0, 0]))
    assert bool(torch.isfinite(logits[0]).all()) and int(batch.taken) == 2
