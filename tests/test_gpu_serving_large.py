"""The serving operators where counts of tokens, pages, columns and forks come near 2^31, or near the most that
is accepted."""

from __future__ import annotations

import pytest
import torch

import metile_amd as mt
from tests.test_gpu_paged import i32

pytestmark = pytest.mark.gpu
MOST = (1 << 31) - 1


def long_row(rows=1):
    """Rows of 2^31 - 1 pages of a token each: the first 30000 again and again, and two others near the end."""
    tables = torch.empty(rows, MOST, dtype=torch.int32, device="cuda")
    torch.arange(MOST, dtype=torch.int32, device="cuda", out=tables[0])
    tables[0].remainder_(30000)
    tables[0, -70000], tables[0, -1] = 39998, 39999
    return tables


def test_free_of_the_longest_rows():
    tables = long_row()
    free = torch.full((40000,), -1, dtype=torch.int32, device="cuda")
    free[30002:] = torch.arange(30000, 39998, device="cuda")
    before = free.clone()
    for kept, gone in ((MOST - 70001, [39998, 39999]), (MOST - 1, [39999]), (MOST, [])):
        list_ = before.clone()
        freed = mt.paged_free(tables, i32([MOST]), i32([kept]), list_, page_size=1, pages=40000,
                              free_start=i32([30002]))
        assert freed.tolist() == [len(gone)]
        assert list_[30002 - len(gone):30002].tolist() == gone
        assert torch.equal(list_[30002:], before[30002:]) and bool((list_[:30002 - len(gone)] == -1).all())


def test_compaction_of_the_longest_rows():
    tables = long_row()
    free = torch.full((40000,), -1, dtype=torch.int32, device="cuda")
    free[30002:] = torch.arange(30000, 39998, device="cuda")
    plan = mt.paged_compact(tables, i32([MOST]), free, page_size=1, pages=40000, free_start=i32([30002]))
    assert plan.moves.tolist() == [2]
    assert plan.sources[:3].tolist() == [39999, 39998, -1] and plan.targets[:3].tolist() == [30000, 30001, -1]
    assert plan.free_pages[30002:].tolist() == list(range(30002, 40000))
    tables[0, -70000], tables[0, -1] = 30001, 30000
    assert torch.equal(plan.block_tables, tables)


def test_fork_of_the_longest_rows():
    tables = long_row(2)
    tables[1].fill_(-1)
    lengths = i32([MOST, 0])
    fork = mt.paged_fork(tables, lengths, i32([0]), i32([1]), i32([]), page_size=1)
    assert [t.tolist() for t in fork] == [[-1], [-1], [0]] and lengths.tolist() == [MOST, MOST]
    assert torch.equal(tables[0], tables[1])


def test_nearly_2_31_rows_of_padding():
    """A call of one request and the most rows that are accepted for it: all but its own are zeros."""
    tokens, dim = 128 * ((1 << 24) - (1 << 16)) - 129, 16
    cache = mt.PagedCache.allocate(1, 16, 1, dim)
    cache.key.normal_(), cache.value.normal_()
    query = torch.randn(1, 1, dim, device="cuda").bfloat16().expand(tokens, 1, dim)
    tables, lengths = i32([[0]]), i32([16])
    few = mt.paged_chunk_attention(query[:5], cache, tables, lengths, i32([0, 5]))
    out, lse = mt.paged_chunk_attention(query, cache, tables, lengths, i32([0, 5]), return_lse=True)
    assert torch.equal(out[:5], few)
    assert bool((lse[5:] == -float("inf")).all())
    rest = out[5:].flatten().view(torch.int16)
    assert not any(bool(part.any()) for part in rest.split(1 << 30))


@pytest.mark.parametrize("forks", [1023, 2559, 2560, 4095, 4096, 4097, 50001, (1 << 23) - 1])
def test_many_forks(forks):
    """Sources with and without a begun page, some forks left out, the list too short for the last."""
    g = torch.Generator("cuda").manual_seed(forks)
    live, page = 1000, 4
    requests = live + forks
    lengths = torch.zeros(requests, dtype=torch.int32, device="cuda")
    lengths[:live] = torch.randint(0, 9, (live,), generator=g, device="cuda")
    tables = torch.full((requests, 3), -1, dtype=torch.int32, device="cuda")
    tables[:live] = torch.randint(0, 5000, (live, 3), generator=g, device="cuda", dtype=torch.int32)
    sources = torch.randint(-20, live, (forks,), generator=g, device="cuda", dtype=torch.int32)
    targets = live + torch.randperm(forks, generator=g, device="cuda").int()
    targets[5::97] = requests
    kept = torch.randint(0, 12, (forks,), generator=g, device="cuda", dtype=torch.int32)
    ok = (sources >= 0) & (targets < requests)
    source = sources.clamp(min=0).long()
    n = torch.where(ok, torch.minimum(lengths[source], kept), 0)
    begun = n % page > 0
    before = begun.long().cumsum(0) - begun.long()
    free = torch.randperm(int(begun.sum()), generator=g, device="cuda").int()  # from entry 2 on: two short
    at = before + 2
    there = begun & (at < free.numel())
    fresh = torch.where(there, free[at.clamp(max=free.numel() - 1)], -1)
    full = (n // page).long()
    old = tables[source].gather(1, full.clamp(max=2)[:, None])[:, 0]
    want_tables, want_lengths = tables.clone(), lengths.clone()
    column = torch.arange(3, device="cuda")
    rows = torch.where(column < full[:, None], tables[source], -1)
    rows = torch.where((column == full[:, None]) & begun[:, None], fresh[:, None], rows)
    want_tables[targets[ok].long()] = rows[ok]
    want_lengths[targets[ok].long()] = n[ok]
    fork = mt.paged_fork(tables, lengths, sources, targets, free, page_size=page, free_start=i32([2]),
                         tokens=kept)
    assert torch.equal(fork.sources, torch.where(there, old, -1))
    assert torch.equal(fork.targets, fresh.int())
    assert int(fork.taken) == int(begun.sum())
    assert torch.equal(tables, want_tables) and torch.equal(lengths, want_lengths)


def test_parts_of_more_blocks_than_fp32_counts():
    """Requests of up to 110 million keys, all of them one page's, whose blocks sum up past 2^24, in parts of
    which a lost or misplaced one would show: the page's result. A part's sums have some 2^16 equal terms
    (blocks), each rounded by at most 2^-24 of the sum."""
    page, dim, heads = 64, 16, 130
    cache = mt.PagedCache.allocate(1, page, 1, dim)
    g = torch.Generator("cuda").manual_seed(3)
    cache.key.normal_(generator=g), cache.value.normal_(generator=g)
    widths, new = [1699999, 300001, 77777, 1234567], [9, 1, 1, 5]
    starts = i32([0, 9, 10, 11, 16])
    tables = torch.zeros(4, max(widths), dtype=torch.int32, device="cuda")
    q = torch.randn(1, heads, dim, generator=g, device="cuda").bfloat16().repeat(16, 1, 1)
    # (each request's new tokens are its page's last: a token sees `widths` whole pages and some)
    out, lse = mt.paged_chunk_attention(q, cache, tables, i32([w * page for w in widths]), starts,
                                        return_lse=True)
    want, want_lse = mt.paged_chunk_attention(q[:1], cache, tables[:1], i32([page]), i32([0, 1]),
                                              return_lse=True)
    blocks = torch.tensor([float(w) for w, n in zip(widths, new) for _ in range(n)]).log().cuda()
    assert float((lse - want_lse - blocks[:, None]).abs().max()) <= 2.0 ** -8 + 2.0 ** -16
    assert float((out.float() - want.float()).abs().max()) <= (2.0 ** -7 + 2.0 ** -7) * float(
        cache.value.abs().max())


def test_pools_of_nearly_2_31_pages():
    """Pages of one token, the highest numbers in use, freed and compacted."""
    pages = MOST
    rows = [[pages - 1, 7, pages - 3], [pages - 3, 1 << 30, -1]]
    tables, lengths, start = i32(rows), i32([3, 2]), i32([4])
    listed = [-1, -1, -1, -1, pages - 2, 5, 1 << 20, 3]
    free = i32(listed)
    freed = mt.paged_free(tables, lengths, i32([1, 1]), free, page_size=1, pages=pages, free_start=start)
    assert freed.tolist() == [2]  # (the second keeps what the first gives up)
    assert free.tolist() == [-1, -1, 7, 1 << 30] + listed[4:]
    plan = mt.paged_compact(tables, lengths, i32(listed), page_size=1, pages=pages, free_start=start)
    # in use 7, 2^30, and two of the highest; free 3, 5, 2^20 and the highest but one
    assert plan.moves.tolist() == [3]
    assert plan.sources.tolist() == [pages - 1, pages - 3, 1 << 30, -1, -1, -1]
    assert plan.targets.tolist() == [3, 5, 1 << 20, -1, -1, -1]
    assert plan.block_tables.tolist() == [[3, 7, 5], [5, 1 << 20, -1]]
    assert plan.free_pages.tolist() == [-1, -1, -1, -1, 1 << 30, pages - 3, pages - 2, pages - 1]


def test_many_forks_in_a_replayed_graph():
    live, forks, page = 50, 3000, 4
    tables = torch.zeros(live + forks, 3, dtype=torch.int32, device="cuda")
    lengths = torch.zeros(live + forks, dtype=torch.int32, device="cuda")
    sources = torch.zeros(forks, dtype=torch.int32, device="cuda")
    targets = live + torch.arange(forks, dtype=torch.int32, device="cuda")
    free, start = torch.arange(forks, device="cuda").int(), i32([0])

    def call():
        return mt.paged_fork(tables, lengths, sources, targets, free, page_size=page, free_start=start)

    def fill(seed):
        g = torch.Generator("cuda").manual_seed(seed)
        tables.copy_(torch.randint(0, 900, tables.shape, generator=g, device="cuda"))
        lengths.copy_(torch.randint(0, 12, lengths.shape, generator=g, device="cuda"))
        sources.copy_(torch.randint(-3, live, sources.shape, generator=g, device="cuda"))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = call()
    torch.cuda.synchronize()
    for seed in range(4):
        fill(seed)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        after = [t.clone() for t in (*got, tables, lengths)]
        fill(seed)
        eager = call()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(after, (*eager, tables, lengths)))
        source, known = sources.clamp(min=0).long(), sources >= 0
        begun = known & (lengths[source] % page > 0)
        assert int(eager.taken) == int(begun.sum())
        before = (begun.long().cumsum(0) - begun.long()).int()
        assert torch.equal(eager.targets, torch.where(begun, before, -1))
