"""Idle requests of the paged decode example keep the token that waits for them."""

from __future__ import annotations

import pytest
import torch

from examples.paged_decode import Batch, Config, Decoder


def test_choose_keeps_the_tokens_of_idle_requests():
    batch = Batch.__new__(Batch)
    batch.tokens = torch.tensor([3, 4, 5])
    batch.active = torch.tensor([1, 0, 1], dtype=torch.int32)
    logits = torch.zeros(3, 9)
    logits[0, 7] = logits[2, 8] = 1.0
    batch.choose(logits)
    assert batch.tokens.tolist() == [7, 4, 8]


CONFIG = Config(layers=2, hidden=256, inter=512, heads=6, kv_heads=2, head_dim=64, vocab=320)


def generate(decoder, pauses, steps, *, graph=False):
    """Each request's chosen tokens; request r is idle in the steps of ``pauses[r]``."""
    batch = Batch(decoder, len(pauses), pages=24, page_size=4, longest=24)
    batch.tokens.copy_(torch.arange(len(pauses)) + 11)
    chosen = [[] for _ in pauses]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        replay = None
        for step in range(steps):
            active = [int(step not in p) for p in pauses]
            batch.active.copy_(torch.tensor(active))
            if replay is None:
                batch.choose(batch.step())
            else:
                replay.replay()
            stream.synchronize()
            if graph and replay is None:  # (the step above gave the stream its workspace)
                replay = torch.cuda.CUDAGraph()
                with torch.cuda.graph(replay, stream=stream):
                    batch.choose(batch.step())
            for r, on in enumerate(active):
                if on:
                    chosen[r].append(int(batch.tokens[r]))
    return chosen


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
def test_a_paused_request_goes_on_where_it_stopped(graph):
    decoder = Decoder(CONFIG, seed=5)
    steps = 12
    want = generate(decoder, [(), (), ()], steps)
    pauses = [(3, 4), (), (2, 6, 7, 9)]
    got = generate(decoder, pauses, steps, graph=graph)
    for r, p in enumerate(pauses):
        assert got[r] == want[r][:steps - len(p)]
