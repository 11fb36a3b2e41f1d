"""The serving operators without a GPU: argument checks of the C ABI, and the restatements that the GPU
tests compare with."""

from __future__ import annotations

import ctypes
import math
import random
import re
import struct
from pathlib import Path

import pytest
import torch

import metile_amd as mt
from metile_amd import _lib
from tests import serving_reference as ref
from tests.test_decode_operators import BAD_CACHES, BUF, cache, message


def test_argument_blocks_are_laid_out_as_the_header_says():
    header = (Path(__file__).resolve().parents[1] / "include" / "metile_amd.h").read_text()
    for name, packer in (("mt_paged_chunk_attention_args", _lib.PAGED_CHUNK_ATTENTION_ARGS),
                         ("mt_paged_copy_args", _lib.PAGED_COPY_ARGS),
                         ("mt_paged_fork_args", _lib.PAGED_FORK_ARGS),
                         ("mt_paged_free_args", _lib.PAGED_FREE_ARGS),
                         ("mt_paged_compact_args", _lib.PAGED_COMPACT_ARGS),
                         ("mt_token_logprobs_args", _lib.TOKEN_LOGPROBS_ARGS)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, header, re.S).group(1)
        letters = ""
        for line in body.strip().split(";")[:-1]:
            kind, names = re.match(r"\s*(?:const )?(\w+)(.*)", line, re.S).groups()
            for field in names.split(","):
                count = int(re.search(r"\[(\d)\]", field).group(1)) if "[" in field else 1
                letters += ("P" if "*" in field else
                            {"int64_t": "q", "int": "i", "float": "f"}[kind]) * count
        assert packer.format == "@" + letters + "0P", name


def attend(desc, ws=None, nbytes=0, **changes):
    a = dict(query=256, qs=128, qh=128, tables=256, ts=4, lengths=256, starts=256, out=256, lse=0,
             tokens=8, requests=1, heads=1, width=4, window=0, scale=1.0, dtype=0)
    a.update(changes)
    return _lib.lib().mt_paged_chunk_attention(
        desc, _lib.PAGED_CHUNK_ATTENTION_ARGS.pack(*a.values()), ws, nbytes, None)


@pytest.mark.parametrize("changes,text", BAD_CACHES)
def test_caches_are_checked(changes, text):
    assert text in message(attend(cache(**changes)))
    assert _lib.lib().mt_paged_chunk_attention_workspace_bytes(cache(**changes), 8, 1, 1, 4, 0) == 0
    good, bad = cache()._obj, cache(**changes)._obj
    addresses = struct.pack("@2P", ctypes.addressof(good), ctypes.addressof(bad))
    args = _lib.PAGED_COPY_ARGS.pack(256, 256, 1)
    assert text in message(_lib.lib().mt_paged_copy(addresses, 2, args, None))


@pytest.mark.parametrize("changes,text", [
    (dict(tokens=0), "tokens"), (dict(requests=0), "requests"), (dict(heads=0), "heads"),
    (dict(width=0), "width"), (dict(width=1 << 27), "2^31"), (dict(width=(1 << 27) - 3), "2^31"),
    (dict(window=-1), "window"), (dict(dtype=2), "dtype"), (dict(dtype=1), "query's dtype"),
    (dict(scale=float("nan")), "finite"), (dict(scale=3e38), "finite"), (dict(query=0), "null"),
    (dict(starts=0), "null"), (dict(out=264), "16 bytes"), (dict(qh=100), "16 bytes"),
    (dict(qs=-128), "16 bytes"), (dict(tokens=1 << 25, heads=64), "2^31"),
    (dict(requests=1 << 24), "2^24")])
def test_chunk_attention_arguments_are_checked(changes, text):
    assert text in message(attend(cache(), **changes))


def test_chunk_attention_needs_its_workspace():
    lib = _lib.lib()
    need = lib.mt_paged_chunk_attention_workspace_bytes(cache(), 8, 3, 8, 40, 0)
    assert need > 0
    assert attend(cache(), requests=3, heads=8, width=40) == _lib.MT_ERR_WORKSPACE
    assert attend(cache(), requests=3, heads=8, width=40, ws=BUF,
                  nbytes=need - 1) == _lib.MT_ERR_WORKSPACE
    assert "aligned" in message(attend(cache(), requests=3, heads=8, width=40,
                                       ws=ctypes.c_void_p(264), nbytes=need))
    # parts are bounded whatever the shapes
    most = [lib.mt_paged_chunk_attention_workspace_bytes(cache(), n, 3, 8, 1 << 20, 0)
            for n in (1 << 16, 1 << 20)]
    assert most[0] == most[1] < 1 << 28


def test_pages_arguments_are_checked():
    lib = _lib.lib()
    fork = dict(tables=256, stride=4, lengths=256, sources=256, targets=256, tokens=0, free=256, start=0,
                cs=256, ct=256, taken=256, requests=2, width=4, count=3, page=16, forks=1)
    release = dict(tables=256, stride=4, lengths=256, kept=256, free=256, start=256, freed=256, requests=2,
                   width=4, count=3, page=16, pages=9)
    compact = dict(tables=256, stride=4, lengths=256, free=256, start=256, nt=256, nf=256, sources=256,
                   targets=256, moves=256, requests=2, width=4, count=3, page=16, pages=9, most=4)
    calls = (
        (fork, lambda a: lib.mt_paged_fork(_lib.PAGED_FORK_ARGS.pack(*a.values()), None)),
        (release, lambda a: lib.mt_paged_free(_lib.PAGED_FREE_ARGS.pack(*a.values()), None, 0, None)),
        (compact, lambda a: lib.mt_paged_compact(_lib.PAGED_COMPACT_ARGS.pack(*a.values()), None, 0, None)))
    for good, call in calls:
        for changes, text in ((dict(requests=-1), "requests"), (dict(requests=1 << 24), "requests"),
                              (dict(page=0), "page_size"), (dict(width=0), "width"),
                              (dict(width=1 << 27), "2^31"), (dict(stride=3), "overlap"),
                              (dict(count=-1), "negative"), (dict(tables=0), "null"),
                              (dict(lengths=0), "null"), (dict(free=0), "null")):
            assert text in message(call({**good, **changes})), changes
    for changes, text in ((dict(forks=-1), "forks"), (dict(forks=1 << 23), "forks"),
                          (dict(taken=0), "null"), (dict(sources=0), "null"), (dict(ct=0), "null")):
        assert text in message(calls[0][1]({**fork, **changes}))
    for good, call in calls[1:]:
        assert call(good) == _lib.MT_ERR_WORKSPACE
        for changes, text in ((dict(pages=0), "pages"), (dict(start=0), "null")):
            assert text in message(call({**good, **changes}))
    assert "kept" not in compact and "null" in message(calls[1][1]({**release, "kept": 0}))
    for changes, text in ((dict(most=3), "most_moves"), (dict(nt=0), "null"), (dict(nf=0), "null"),
                          (dict(moves=0), "null"), (dict(targets=0), "null")):
        assert text in message(calls[2][1]({**compact, **changes}))
    assert lib.mt_paged_free_workspace_bytes(0) == lib.mt_paged_compact_workspace_bytes(-1) == 0
    # marks of the largest pool do not pass the counts' bits
    assert 2 << 31 <= lib.mt_paged_free_workspace_bytes((1 << 31) - 1) < 3 << 31


def test_copy_arguments_are_checked():
    lib = _lib.lib()
    one = struct.pack("@P", ctypes.addressof(cache()._obj))
    desc = cache()  # kept while its address is used
    one = struct.pack("@P", ctypes.addressof(desc._obj))
    for args, count, text in (((256, 256, -1), 1, "negative"), ((256, 256, 1), -1, "negative"),
                              ((0, 256, 1), 1, "null"), ((256, 0, 1), 1, "null")):
        assert text in message(lib.mt_paged_copy(one, count, _lib.PAGED_COPY_ARGS.pack(*args), None))
    assert lib.mt_paged_copy(one, 1, _lib.PAGED_COPY_ARGS.pack(0, 0, 0), None) == _lib.MT_OK
    assert lib.mt_paged_copy(None, 0, _lib.PAGED_COPY_ARGS.pack(256, 256, 1), None) == _lib.MT_OK
    assert "null" in message(lib.mt_paged_copy(None, 1, _lib.PAGED_COPY_ARGS.pack(256, 256, 1), None))


def test_logprobs_arguments_are_checked():
    lib = _lib.lib()
    good = dict(logits=256, stride=100, tokens=256, logprobs=256, entropies=256, ranks=256, tl=256, tt=256,
                rows=4, vocab=100, top=5, dtype=0, temperature=1.0)

    def call(**changes):
        return lib.mt_token_logprobs(_lib.TOKEN_LOGPROBS_ARGS.pack(*{**good, **changes}.values()), None,
                                     0, None)

    for changes, text in ((dict(dtype=3), "dtype"), (dict(rows=-1), "rows"), (dict(vocab=0), "vocab"),
                          (dict(vocab=(1 << 24) + 1), "vocab"), (dict(top=33), "top"),
                          (dict(top=-1), "top"), (dict(top=6, vocab=5), "top"),
                          (dict(temperature=0.0), "temperature"), (dict(temperature=-1.0), "temperature"),
                          (dict(temperature=math.nan), "temperature"),
                          (dict(temperature=math.inf), "temperature"),
                          (dict(temperature=1e-39), "temperature"), (dict(stride=-1), "row_stride"),
                          (dict(logits=0), "null"), (dict(entropies=0), "null"), (dict(ranks=0), "null"),
                          (dict(tl=0), "null")):
        assert text in message(call(**changes)), changes
    assert call(rows=0) == _lib.MT_OK
    assert call(rows=2, vocab=1 << 20) == _lib.MT_ERR_WORKSPACE
    assert lib.mt_token_logprobs_workspace_bytes(0, 100, 5) == 0
    assert lib.mt_token_logprobs_workspace_bytes(1, 1 << 24, 32) < 1 << 20


def test_guards_before_the_device():
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="ROCm device"):
        mt.token_logprobs(torch.zeros(3, 5))
    with pytest.raises(ValueError, match="ROCm device"):
        mt.paged_fork(i[:, None], i, i, i, i, page_size=4)
    with pytest.raises(ValueError, match="ROCm device"):
        mt.paged_free(i[:, None], i, i, i, page_size=4, pages=3, free_start=i[:1])
    with pytest.raises(ValueError, match="ROCm device"):
        mt.paged_compact(i[:, None], i, i, page_size=4, pages=3, free_start=i[:1])


# ---- the restatements ----------------------------------------------------------------------------------


def test_reference_chunks_against_torch():
    g = torch.Generator().manual_seed(0)
    key, value = torch.randn(2, 5, 4, 2, 8, generator=g, dtype=torch.float64)
    query = torch.randn(6, 4, 8, generator=g).half()
    tables = torch.tensor([[3, 1, 4], [0, 2, -1]])
    out, lse, _, _ = ref.chunk_attention(query, key, value, tables, [10, 7], [0, 4, 6], 0.3, window=5)
    for r, (rows, n) in enumerate(((slice(0, 4), 10), (slice(4, 6), 7))):
        k, v = (t[tables[r][:-(-n // 4)]].reshape(-1, 2, 8)[:n].repeat_interleave(2, 1) for t in (key, value))
        new = rows.stop - rows.start
        place = n - new + torch.arange(new)[:, None]
        seen = (torch.arange(n) <= place) & (torch.arange(n) > place - 5)
        q = query[rows].double().transpose(0, 1)
        want = torch.nn.functional.scaled_dot_product_attention(q, k.transpose(0, 1), v.transpose(0, 1),
                                                                attn_mask=seen, scale=0.3)
        assert torch.allclose(out[rows], want.transpose(0, 1), atol=1e-12)
        logits = (q @ k.permute(1, 2, 0)) * 0.3
        assert torch.allclose(lse[rows], logits.masked_fill(~seen, -math.inf).logsumexp(-1).T, atol=1e-12)


def test_reference_pages_by_hand():
    tables = [[5, 3, 9], [5, 7, -1], [-1, -1, -1]]
    assert ref.fork(tables, [10, 6, 0], [0], [2], [0, 2], 4, 1) == (
        [[5, 3, 9], [5, 7, -1], [5, 3, 2]], [10, 6, 10], [9], [2], [1])
    assert ref.fork(tables, [10, 6, 0], [1], [2], [0, 2], 4, tokens=[4]) == (
        [[5, 3, 9], [5, 7, -1], [5, -1, -1]], [10, 6, 4], [-1], [-1], [0])
    assert ref.free(tables, [10, 6, 0], [5, 0, 0], [-1, -1, -1, 2], 4, 10, 3) == ([-1, 7, 9, 2], [2])
    assert ref.free(tables, [10, 6, 0], [0, 6, 0], [-1, -1], 4, 10, 1) == ([9, -1], [2])
    # in use 3 5 7 9, free 1 2 6: the lowest four are 1 2 3 5
    assert ref.compact(tables, [10, 6, 0], [-1, 6, 1, 2], 4, 10, 1) == (
        [[5, 3, 1], [5, 2, -1], [-1, -1, -1]], [-1, 6, 7, 9], [9, 7] + [-1] * 3, [1, 2] + [-1] * 3, [2])


def test_reference_logprobs_against_torch():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 40, generator=g, dtype=torch.float64)
    x[2, 3:] = -math.inf
    t = torch.tensor([1, 2, 0, 39, 7])
    lp, h, rank, top, best = ref.logprobs(x, t, 3, 0.7)
    d = torch.distributions.Categorical(logits=x / 0.7)
    assert torch.allclose(lp, d.log_prob(t))
    assert torch.allclose(h[[0, 1, 3, 4]], d.entropy()[[0, 1, 3, 4]])
    assert torch.allclose(h[2], torch.distributions.Categorical(logits=x[2, :3] / 0.7).entropy())
    for r in range(5):
        order = sorted(range(40), key=lambda i: (-float(x[r, i]), i))
        assert best[r].tolist() == order[:3] and int(rank[r]) == order.index(int(t[r]))
        assert torch.allclose(top[r], d.logits[r, order[:3]])


def test_reference_pages_keep_every_page_once():
    rng = random.Random(0)
    for _ in range(50):
        lengths = [rng.randint(0, 30) for _ in range(6)]
        numbers = rng.sample(range(64), 64)
        tables = [[numbers.pop() if c * 4 < n else -1 for c in range(8)] for n in lengths]
        new, free, _, _, moves = ref.compact(tables, lengths, numbers, 4, 64, 0)
        used = ref.in_use(new, lengths, 4, 64)
        assert used == set(range(len(used))) and sorted(used | set(free)) == list(range(64))
