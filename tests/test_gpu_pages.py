"""Copies, forks, freeing and compaction of a paged cache's pages on the GPU, exactly."""

from __future__ import annotations

import random

import pytest
import torch

import metile_amd as mt
from tests import serving_reference as ref
from tests.test_gpu_paged import FP8, as_bits, i32, pool

pytestmark = pytest.mark.gpu


def state(requests, longest, page, *, seed=0, shared=3, spare=0.4, extra_columns=1, stray=False):
    """Tables over a pool in random order, some requests sharing the first pages of others, and its free
    list; with `stray`, entries and listed pages that are none of the pool's."""
    rng = random.Random(seed)
    lengths = [rng.choice((0, 1, page, longest, rng.randint(0, longest))) for _ in range(requests)]
    width = max(1, -(-longest // page)) + extra_columns
    counts = [-(-n // page) for n in lengths]
    pages = max(2, int(sum(counts) * (1 + spare)) + 2)
    numbers = list(range(pages))
    rng.shuffle(numbers)
    tables = [[numbers.pop() if c < n else rng.choice((-1, 3)) for c in range(width)] for n in counts]
    for r in range(1, requests):
        if shared and r % shared == 0:
            half = min(counts[r], counts[r - 1]) // 2
            numbers += tables[r][:half]
            tables[r][:half] = tables[r - 1][:half]
    rng.shuffle(numbers)
    used = {p for row, n in zip(tables, counts) for p in row[:n]}
    numbers = [p for p in numbers if p not in used]
    if stray and requests:
        for _ in range(1 + requests // 4):
            r = rng.randrange(requests)
            tables[r][rng.randrange(width)] = rng.choice((-1, -9, pages, 2 ** 31 - 1))
        numbers += [pages, -4] + numbers[:2]
    start = rng.randint(0, 5) if stray else pages - len(numbers)
    free = [-1] * start + numbers
    return dict(tables=tables, lengths=lengths, free=free, start=start, pages=pages, page=page)


# ---- copies --------------------------------------------------------------------------------------------


@pytest.mark.parametrize("layout", ["outer", "inner", "mixed"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, FP8])
@pytest.mark.parametrize("page,heads,dim", [(16, 2, 64), (1, 1, 16), (5, 3, 80), (64, 8, 128), (7, 1, 256)])
def test_copy(layout, dtype, page, heads, dim):
    rng = random.Random(page)
    pages = 37
    caches = [mt.PagedCache(pool(pages, page, heads, dim, dtype, layout, seed=2 * i),
                            pool(pages, page, heads, dim, dtype, layout, seed=2 * i + 1))
              for i in range(3)]
    numbers = rng.sample(range(pages), pages)
    sources, targets = [numbers[i % 9] for i in range(14)], numbers[9:23]
    for i, bad in ((2, -1), (5, pages), (7, -2 ** 31)):
        sources[i] = bad
    for i, bad in ((3, -1), (9, pages), (11, 2 ** 31 - 1)):
        targets[i] = bad
    want = []
    for c in caches:
        for t in (c.key, c.value):
            bits = as_bits(t)
            for s, d in zip(sources, targets):
                if 0 <= s < pages and 0 <= d < pages:
                    bits[d] = as_bits(t)[s]
            want.append(bits)
    mt.paged_copy(caches, i32(sources), i32(targets))
    got = [as_bits(t) for c in caches for t in (c.key, c.value)]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_copy_of_different_caches_and_many_layers():
    shapes = [(40, 16, 2, 64, torch.bfloat16, "outer")] * 70 + [
        (50, 8, 1, 128, torch.float16, "inner"), (40, 16, 2, 64, FP8, "outer"),
        (40, 16, 2, 64, torch.bfloat16, "outer")]
    caches = [mt.PagedCache(pool(*s, seed=i), pool(*s, seed=i + 1000)) for i, s in enumerate(shapes)]
    before = [as_bits(c.key) for c in caches], [as_bits(c.value) for c in caches]
    mt.paged_copy(tuple(caches), i32([1, 45, 3]), i32([7, 2, 48]))
    for i, (c, k, v) in enumerate(zip(caches, *before)):
        for t, bits in ((c.key, k), (c.value, v)):
            bits[7] = bits[1]
            if c.pages == 50:
                bits[2], bits[48] = bits[45].clone(), bits[3].clone()
            assert torch.equal(as_bits(t), bits), i


def test_copy_with_different_strides_of_keys_and_values():
    key, value = pool(9, 5, 3, 32, torch.bfloat16, "outer"), pool(9, 5, 3, 32, torch.bfloat16, "mixed")
    cache = mt.PagedCache(key, value)
    want = [as_bits(key), as_bits(value)]
    for bits in want:
        bits[8] = bits[0]
    rest = as_bits(value._base)
    mt.paged_copy(cache, i32([0]), i32([8]))
    assert torch.equal(as_bits(key), want[0]) and torch.equal(as_bits(value), want[1])
    rest[8, 1] = rest[0, 1]  # and nothing between the value's pages
    assert torch.equal(as_bits(value._base), rest)


def test_copy_of_nothing():
    cache = mt.PagedCache.allocate(3, 4, 1, 16)
    mt.paged_copy(cache, i32([]), i32([]))
    mt.paged_copy([], i32([1]), i32([2]))


def test_copy_of_more_pairs_than_a_launch_counts():
    """The largest page is so large that a launch takes a few pairs of it."""
    key = torch.zeros(8, 1 << 20, 1, 256, dtype=FP8, device="cuda")
    value = torch.zeros(8, 1 << 20, 1, 256, dtype=FP8, device="cuda")
    bits = key.view(torch.uint8)
    for p in range(8):
        bits[p] = p + 1
    cache = mt.PagedCache(key, value)
    sources, targets = [0, 1] * 300, [-1] * 600
    for at, target in ((0, 2), (599, 3), (300, 4), (301, 5)):
        targets[at] = target
    mt.paged_copy(cache, i32(sources), i32(targets))
    for p, held in enumerate((1, 2, 1, 2, 1, 2, 7, 8)):
        assert bool((bits[p] == held).all()), p


@pytest.mark.parametrize("size", [(1 << 32) + (1 << 20), 11 << 30])
def test_copy_beyond_32_bits(size):
    apart = size // 9 // 2 // 16 * 16
    cache = mt.PagedCache(*(torch.empty(9 * apart, dtype=torch.bfloat16, device="cuda").as_strided(
        (9, 16, 2, 64), (apart, 128, 64, 1)) for _ in range(2)))
    for t in (cache.key, cache.value):
        t.copy_(torch.randn(9, 16, 2, 64, device="cuda"))
    want = [as_bits(t) for t in (cache.key, cache.value)]
    for bits in want:
        bits[8], bits[7] = bits[0].clone(), bits[5].clone()
    mt.paged_copy(cache, i32([0, 5]), i32([8, 7]))
    assert all(torch.equal(as_bits(t), bits) for t, bits in zip((cache.key, cache.value), want))


# ---- forks ---------------------------------------------------------------------------------------------


def check_fork(s, sources, targets, tokens=None, start=None):
    want = ref.fork(s["tables"], s["lengths"], sources, targets, s["free"], s["page"],
                    s["start"] if start is None else start, tokens)
    tables, lengths = i32(s["tables"]), i32(s["lengths"])
    got = mt.paged_fork(tables, lengths, i32(sources), i32(targets), i32(s["free"]),
                        page_size=s["page"], free_start=i32([s["start"] if start is None else start]),
                        tokens=None if tokens is None else i32(tokens))
    assert tables.tolist() == want[0] and lengths.tolist() == want[1]
    for a, b, name in zip(got, want[2:], mt.PagedFork._fields):
        assert a.tolist() == b, name


@pytest.mark.parametrize("page", [1, 5, 16, 64])
@pytest.mark.parametrize("forks", [1, 3, 40, 300, 700])
def test_fork(page, forks):
    rng = random.Random(forks * 100 + page)
    s = state(2 * forks, 150, page, seed=forks, spare=2.0 + page)
    rows = list(range(2 * forks))
    rng.shuffle(rows)
    sources = [rows[rng.randrange(forks)] for _ in range(forks)]
    check_fork(s, sources, rows[forks:])
    check_fork(s, sources, rows[forks:], [rng.choice((0, 1, page, 30, 10 ** 6, -3)) for _ in range(forks)])


def test_fork_edges():
    s = state(8, 90, 16, seed=4, spare=2.0)
    s["lengths"][:4] = [33, 32, 0, 10 ** 9]
    check_fork(s, [0, 1, 2, 3], [4, 5, 6, 7])
    check_fork(s, [0, -1, 8, 2 ** 31 - 1, 0], [4, 5, 6, 7, -1])   # rows that there are not
    check_fork(s, [0, 0, 0], [4, 5, 6], start=len(s["free"]) - 1)  # the list runs out
    check_fork(s, [0, 0], [4, 5], start=-1)
    check_fork(s, [0, 0], [4, 5], start=2 ** 31 - 1)
    s["lengths"][0] = -5
    check_fork(s, [0], [4])
    check_fork(s, [], [])


def test_fork_without_start_and_strided_tables():
    s = state(4, 60, 8, seed=1, spare=2.0)
    free = s["free"][s["start"]:]
    want = ref.fork(s["tables"], s["lengths"], [0], [2], free, 8)
    wide = torch.full((4, 30), 77, dtype=torch.int32, device="cuda")
    view = wide[:, 3:3 + len(s["tables"][0])]
    view.copy_(i32(s["tables"]))
    lengths = i32(s["lengths"])
    got = mt.paged_fork(view, lengths, i32([0, 9])[:1], i32([2]), i32(free), page_size=8)
    assert view.tolist() == want[0] and lengths.tolist() == want[1]
    assert [t.tolist() for t in got] == list(want[2:])
    assert bool((wide[:, :3] == 77).all()) and bool((wide[:, 3 + view.shape[1]:] == 77).all())


# ---- freeing -------------------------------------------------------------------------------------------


def check_free(s, kept, start=None):
    start = s["start"] if start is None else start
    want = ref.free(s["tables"], s["lengths"], kept, s["free"], s["page"], s["pages"], start)
    tables, lengths, free = i32(s["tables"]), i32(s["lengths"]), i32(s["free"])
    before = tables.clone(), lengths.clone()
    freed = mt.paged_free(tables, lengths, i32(kept), free, page_size=s["page"], pages=s["pages"],
                          free_start=i32([start]))
    assert freed.tolist() == want[1] and free.tolist() == want[0]
    assert torch.equal(tables, before[0]) and torch.equal(lengths, before[1])


@pytest.mark.parametrize("page", [1, 5, 16])
@pytest.mark.parametrize("requests", [1, 2, 30, 500])
@pytest.mark.parametrize("stray", [False, True])
def test_free(page, requests, stray):
    rng = random.Random(requests + page)
    s = state(requests, 220, page, seed=requests, stray=stray)
    check_free(s, [rng.choice((0, n, n - 1, n // 2, n + 5, -3)) for n in s["lengths"]])
    check_free(s, [0] * requests)
    check_free(s, s["lengths"])


@pytest.mark.parametrize("start", [0, 1, 7, -3, 2 ** 31 - 1, -2 ** 31])
def test_free_into_a_list_that_has_no_room(start):
    s = state(12, 100, 8, seed=2)
    check_free(s, [0] * 12, start=start)


def test_free_of_a_large_pool_and_long_rows():
    """Several workgroups a scan, and rows of several pieces."""
    s = state(6, 9000, 1, seed=3, spare=0.1)
    assert s["pages"] > 3 * 4096 and len(s["tables"][0]) > 4096
    check_free(s, [n // 3 if i % 2 else 0 for i, n in enumerate(s["lengths"])])


@pytest.mark.parametrize("requests,longest,page,spare", [
    (256, 500, 4, 0.2), (256, 512, 4, 0.2), (257, 500, 4, 0.2), (40, 900, 1, 0.2), (7, 2300, 1, 0.4),
    (64, 700, 1, 0.1), (3, 20, 16, 3000.0), (1, 16300, 1, 0.0), (1, 16500, 1, 0.0)])
def test_sizes_about_those_of_one_workgroup(requests, longest, page, spare):
    s = state(requests, longest, page, seed=requests, spare=spare, stray=True)
    rng = random.Random(requests)
    check_free(s, [rng.choice((0, n, n // 2)) for n in s["lengths"]])
    check_compact(s)


@pytest.mark.parametrize("pages", [16383, 16384, 16385])
def test_pools_about_those_of_one_workgroup(pages):
    """Every page in use or free, moves from one end to the other."""
    numbers = list(range(pages))
    for used in (1, pages // 2, pages - 1, pages):
        rows = [numbers[::-1][:used][i::4] for i in range(4)]
        s = dict(tables=[row + [-1] * (used // 4 + 1 - len(row)) for row in rows],
                 lengths=[len(row) for row in rows], free=[-1] * used + numbers[:pages - used], start=used,
                 pages=pages, page=1)
        check_compact(s)
        check_free(s, [n // 2 for n in s["lengths"]])


def test_free_without_requests():
    free = i32([-1, 4])
    freed = mt.paged_free(torch.empty(0, 3, dtype=torch.int32, device="cuda"), i32([]), i32([]), free,
                          page_size=4, pages=9, free_start=i32([1]))
    assert freed.tolist() == [0] and free.tolist() == [-1, 4]


# ---- compaction ----------------------------------------------------------------------------------------


def check_compact(s, start=None):
    start = s["start"] if start is None else start
    want = ref.compact(s["tables"], s["lengths"], s["free"], s["page"], s["pages"], start)
    tables, lengths, free = i32(s["tables"]), i32(s["lengths"]), i32(s["free"])
    before = tables.clone(), free.clone()
    plan = mt.paged_compact(tables, lengths, free, page_size=s["page"], pages=s["pages"],
                            free_start=i32([start]))
    for got, expect, name in zip(plan, want, mt.PagedCompaction._fields):
        assert got.tolist() == expect, name
    assert torch.equal(tables, before[0]) and torch.equal(free, before[1])


@pytest.mark.parametrize("page", [1, 5, 16])
@pytest.mark.parametrize("requests", [1, 2, 30, 500])
@pytest.mark.parametrize("stray", [False, True])
@pytest.mark.parametrize("spare", [0.0, 0.3, 3.0])
def test_compact(page, requests, stray, spare):
    check_compact(state(requests, 220, page, seed=requests, stray=stray, spare=spare))


def test_compact_edges():
    s = state(12, 100, 8, seed=2)
    for start in (0, len(s["free"]), len(s["free"]) - 1, -7, 2 ** 31 - 1):
        check_compact(s, start=start)
    check_compact({**s, "lengths": [0] * 12})          # nothing in use
    check_compact({**s, "lengths": [10 ** 9] * 12})    # entries behind the last page are none
    check_compact({**s, "free": [], "start": 0})
    check_compact({**s, "free": s["free"] + s["free"][-3:]})  # listed twice


def test_compact_of_a_large_pool():
    check_compact(state(6, 9000, 1, seed=3, spare=1.0))


def test_compacted_requests_read_the_same():
    """Attention over the pages gives the same bits before and after."""
    s = state(9, 150, 16, seed=8, spare=1.0)
    cache = mt.PagedCache(pool(s["pages"], 16, 2, 64, torch.bfloat16, "outer", seed=1),
                          pool(s["pages"], 16, 2, 64, torch.bfloat16, "outer", seed=2))
    q = torch.randn(9, 4, 64, device="cuda").bfloat16()
    tables, lengths, free = i32(s["tables"]), i32(s["lengths"]), i32(s["free"])
    before = mt.paged_attention(q, cache, tables, lengths)
    plan = mt.paged_compact(tables, lengths, free, page_size=16, pages=s["pages"],
                            free_start=i32([s["start"]]))
    mt.paged_copy(cache, plan.sources, plan.targets)
    assert int(plan.moves) > 0
    assert torch.equal(before, mt.paged_attention(q, cache, plan.block_tables, lengths))
    used = len(ref.in_use(s["tables"], s["lengths"], 16, s["pages"]))
    live = ref.in_use(plan.block_tables.tolist(), s["lengths"], 16, s["pages"])
    assert live == set(range(used))


# ---- graphs and streams ----------------------------------------------------------------------------


def test_graph_replays():
    """A captured release, fork and compaction, replayed with other contents."""
    states = [state(40, 200, 8, seed=n, spare=1.5) for n in (1, 2, 3)]
    pages = max(s["pages"] for s in states)
    length = max(len(s["free"]) for s in states)
    width = max(len(s["tables"][0]) for s in states)
    tables = torch.zeros(40, width, dtype=torch.int32, device="cuda")
    lengths, kept = i32([0] * 40), i32([0] * 40)
    free, start = i32([0] * length), i32([0])
    sources, targets = i32([0]), i32([1])

    def call():
        freed = mt.paged_free(tables, lengths, kept, free, page_size=8, pages=pages, free_start=start)
        fork = mt.paged_fork(tables, lengths, sources, targets, free, page_size=8, free_start=start)
        plan = mt.paged_compact(tables, lengths, free, page_size=8, pages=pages, free_start=start)
        return [freed, *fork, *plan]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = call()
    torch.cuda.synchronize()
    for turn in range(6):
        s = states[turn % 3]
        padded = [row + [-1] * (width - len(row)) for row in s["tables"]]
        listed = [-1] * (length - len(s["free"])) + s["free"]
        begin = s["start"] + length - len(s["free"])

        def fill():
            tables.copy_(i32(padded))
            lengths.copy_(i32(s["lengths"]))
            kept.copy_(i32([n // 2 for n in s["lengths"]]))
            free.copy_(i32(listed))
            start.copy_(i32([begin]))

        fill()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        state_after = [t.tolist() for t in (*got, tables, lengths, free)]
        fill()
        eager = call()
        assert state_after == [t.tolist() for t in (*eager, tables, lengths, free)]


def test_refusals():
    tables, lengths, free, start = i32([[0, 1], [2, 3]]), i32([5, 6]), i32([4, 5]), i32([0])
    one, cache = i32([1]), mt.PagedCache.allocate(6, 4, 1, 16)

    def fork(t=tables, n=lengths, s=i32([0]), d=one, f=free, **kw):
        return mt.paged_fork(t, n, s, d, f, **{"page_size": 4, **kw})

    def release(t=tables, n=lengths, k=lengths, f=free, **kw):
        return mt.paged_free(t, n, k, f, **{"page_size": 4, "pages": 6, "free_start": start, **kw})

    def compact(t=tables, n=lengths, f=free, **kw):
        return mt.paged_compact(t, n, f, **{"page_size": 4, "pages": 6, "free_start": start, **kw})

    for call in (fork, release, compact):
        call()
        for kwargs, text in ((dict(t=tables.long()), "int32"), (dict(t=tables[0]), "int32"),
                             (dict(n=one), "same requests"), (dict(n=lengths.float()), "int32"),
                             (dict(page_size=0), "page_size"), (dict(page_size=1 << 30), "2^31"),
                             (dict(t=tables.t()), "contiguous rows"), (dict(t=tables[:, :0]), "column"),
                             (dict(free_start=i32([1, 2])), "one element"),
                             (dict(free_start=start.long()), "int32"), (dict(f=free.cpu()), "ROCm device")):
            with pytest.raises(ValueError, match=text.replace("^", r"\^")):
                call(**kwargs)
    for kwargs, text in ((dict(s=i32([0, 1])), "same forks"), (dict(tokens=lengths), "same forks"),
                         (dict(n=i32([1, 2, 3, 4])[::2]), "contiguous")):
        with pytest.raises(ValueError, match=text):
            fork(**kwargs)
    for call in (release, compact):
        with pytest.raises(ValueError, match="pages"):
            call(pages=0)
    with pytest.raises(ValueError, match="contiguous"):
        release(f=i32([1, 2, 3, 4])[::2])
    for args, text in (((cache, one.long(), one), "int32"), ((cache, one, i32([1, 2])), "pairs"),
                       ((cache, one.cpu(), one), "ROCm device")):
        with pytest.raises(ValueError, match=text):
            mt.paged_copy(*args)
