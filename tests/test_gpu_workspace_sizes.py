"""Sizes of workspaces that a cache remembers: those of decode steps stay while chunks come in every size."""

from __future__ import annotations

import pytest
import torch

import metile_amd as mt
from metile_amd import _lib
from tests.test_gpu_paged import i32

pytestmark = pytest.mark.gpu


def test_chunks_of_many_sizes_do_not_make_decode_steps_ask_again(monkeypatch):
    cache = mt.PagedCache.allocate(4, 16, 2, 64)
    cache.key.zero_(), cache.value.zero_()
    q = torch.randn(600, 4, 64, device="cuda").bfloat16()
    table = i32([[0, 1, 2, 3]])
    asked, lib = [], _lib.lib()

    class Counted:
        def __getattr__(self, name):
            if name == "mt_paged_attention_workspace_bytes":
                asked.append(name)
            return getattr(lib, name)

    monkeypatch.setattr(_lib, "lib", lambda counted=Counted(): counted)
    for tokens in range(1, 601):
        mt.paged_chunk_attention(q[:tokens], cache, table, i32([64]), i32([0, min(tokens, 64)]))
        mt.paged_attention(q[:1], cache, table, i32([64]))
    assert len(asked) == 1
    assert len(cache._chunk_workspaces) <= 256
