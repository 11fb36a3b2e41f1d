"""Attention of chunks through the C entry, its outputs and workspace between guard bands: starts in any order
write nothing but the rows of the batch, and rows in front of the first request and behind the last are
zeros."""

from __future__ import annotations

import math
import random

import pytest
import torch

import metile_amd as mt
from metile_amd import _lib
from tests.test_gpu_chunk_attention import case, compare, expect
from tests.test_gpu_paged import FP8, i32

pytestmark = pytest.mark.gpu
BAND = 1 << 16


def guarded(nbytes):
    """Bytes between two bands, and a check of these."""
    held = torch.full((nbytes + 2 * BAND,), 0xA5, dtype=torch.uint8, device="cuda")

    def untouched():
        return bool((held[:BAND] == 0xA5).all()) and bool((held[-BAND:] == 0xA5).all())

    return held[BAND:held.numel() - BAND], untouched


def call(c):
    """(out, lse) of the C entry; nothing else has changed."""
    cache = mt.PagedCache(c["key"], c["value"], key_scale=c["scales"][0], value_scale=c["scales"][1])
    query, tables, starts, lengths = (c[n].contiguous() for n in ("query", "tables", "starts", "lengths"))
    tokens, heads, dim = query.shape
    requests, width = tables.shape
    lib = _lib.lib()
    shape = (tokens, requests, heads, width, c["window"])
    need = lib.mt_paged_chunk_attention_workspace_bytes(cache._ref, *shape)
    assert need > 0
    (ws, ws_ok), (out, out_ok), (lse, lse_ok) = (
        guarded(-(-n // 256) * 256) for n in (need, query.numel() * 2, tokens * heads * 4))
    inputs = [c["key"].view(torch.uint8), c["value"].view(torch.uint8), query, tables, starts, lengths]
    before = [t.clone() for t in inputs]
    args = _lib.PAGED_CHUNK_ATTENTION_ARGS.pack(
        query.data_ptr(), heads * dim, dim, tables.data_ptr(), width, lengths.data_ptr(), starts.data_ptr(),
        out.data_ptr(), lse.data_ptr(), *shape[:4], c["window"], dim ** -0.5,
        {torch.bfloat16: _lib.MT_BF16, torch.float16: _lib.MT_F16}[query.dtype])
    stream = torch.cuda.current_stream().cuda_stream
    _lib.check(lib.mt_paged_chunk_attention(cache._ref, args, ws.data_ptr(), need, stream))
    assert ws_ok() and out_ok() and lse_ok()
    assert bool((ws[need:] == 0xA5).all())
    assert all(torch.equal(a, b) for a, b in zip(inputs, before))
    for t, n in ((out, query.numel() * 2), (lse, tokens * heads * 4)):
        assert bool((t[n:] == 0xA5).all())
    return (out[:query.numel() * 2].view(query.dtype).view(query.shape),
            lse[:tokens * heads * 4].view(torch.float32).view(tokens, heads))


@pytest.mark.parametrize("past", [30, 3000])
@pytest.mark.parametrize("starts", [[0, 40, 20, 60], [0, -5, 2 ** 31 - 1, 60], [0, 64, 0, 64], [60, 40, 20, 0],
                                    [-2 ** 31, 2 ** 31 - 1, -1, 2 ** 31 - 1]])
def test_starts_out_of_order_write_no_other_memory(starts, past):
    for dim, dtype in ((64, torch.bfloat16), (80, FP8), (256, torch.bfloat16)):
        c = case([20, 20, 20], [past] * 3, heads=2, kv=1, dim=dim, cache=dtype, padding=4)
        call({**c, "starts": i32(starts)})


def test_starts_of_many_requests_out_of_order_write_no_other_memory():
    rng = random.Random(3)
    c = case([rng.randint(0, 5) for _ in range(90)], [rng.choice((9, 2500)) for _ in range(90)], heads=6,
             kv=2, dim=64, padding=3)
    for _ in range(5):
        order = c["starts"].tolist()
        rng.shuffle(order)
        call({**c, "starts": i32(order)})


@pytest.mark.parametrize("requests", [3, 70])
@pytest.mark.parametrize("front", [1, 40])
def test_rows_in_front_of_the_first_request_are_zeros(requests, front):
    new, past = [(7 * r) % 23 for r in range(requests)], [(3 * r) % 90 for r in range(requests)]
    c = case(new, past, heads=4, kv=2, dim=64, padding=6)
    want = expect(c)
    rows = torch.randn(front, 4, 64, device="cuda").bfloat16()
    out, lse = call({**c, "query": torch.cat([rows, c["query"]]), "starts": c["starts"] + front})
    assert bool((out[:front] == 0).all()) and bool((lse[:front] == -math.inf).all())
    compare((out[front:], lse[front:]), want)


def test_a_batch_of_rows_without_requests():
    c = case([20, 20, 20], [30, 30, 30], heads=2, kv=1, dim=64, padding=4)
    for at in (0, 1, 63, 64, 900):
        out, lse = call({**c, "starts": i32([at] * 4)})
        assert bool((out == 0).all()) and bool((lse == -math.inf).all())
