"""Paged key-value cache on the GPU: tables and slot maps exactly, append bit for bit, attention
against 64 bits, at the sizes, layouts, masks and contents where they can go wrong."""

from __future__ import annotations

import random

import pytest
import torch

import metile_amd as mt
from metile_amd.quantized import workspace
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---- block tables and slot maps ---------------------------------------------------------------------


def check_tables(cached, new, page, width, *, tokens=None, free=None, start=None, seed=0):
    rng = random.Random(seed)
    requests = len(cached)
    had = [-(-min(max(0, n), width * page) // page) for n in cached]
    most = sum(-(-min(max(0, a) + max(0, b), width * page) // page) - h
               for a, b, h in zip(cached, new, had))
    numbers = list(range(sum(had) + most + 7))
    rng.shuffle(numbers)
    table = [[numbers.pop() if c < h else -5 for c in range(width)] for h in had]
    free = numbers if free is None else numbers[:free]
    tokens = sum(max(0, n) for n in new) if tokens is None else tokens
    want = ref.tables(cached, new, table, free, page, tokens, start or 0)
    on_gpu = i32(table) if table else torch.empty(0, width, dtype=torch.int32, device="cuda")
    step = mt.paged_tables(i32(cached), i32(new), on_gpu, i32(free), page_size=page, tokens=tokens,
                           free_start=None if start is None else i32([start]))
    assert on_gpu.tolist() == want[0]
    for got, expect, name in zip(step, want[1:], mt.PagedStep._fields):
        assert got.tolist() == expect, name
    assert step.slots.dtype == torch.int64 and step.taken.dtype == torch.int32


@pytest.mark.parametrize("page", [1, 5, 16, 64, 256])
@pytest.mark.parametrize("requests", [1, 3, 64, 257])
def test_tables_ragged(requests, page):
    rng = random.Random(requests * 1000 + page)
    cached = [rng.choice((0, 0, 1, page - 1, page, page + 1, rng.randint(0, 300)))
              for _ in range(requests)]
    new = [rng.choice((0, 1, 1, page, page + 1, rng.randint(0, 90))) for _ in range(requests)]
    check_tables(cached, new, page, max(1, -(-400 // page)))


def test_tables_decode_step_and_idle_requests():
    check_tables([15, 16, 0, 31, 32, 7], [1, 1, 0, 1, 1, 0], 16, 4)
    check_tables([0], [1], 16, 1)
    check_tables([0], [0], 16, 1)
    check_tables([16, 16], [0, 0], 16, 2, tokens=0)


@pytest.mark.parametrize("requests", [4096, 4097, 9000])
def test_tables_of_more_requests_than_one_scan_holds(requests):
    rng = random.Random(requests)
    check_tables([rng.randint(0, 40) for _ in range(requests)],
                 [rng.choice((0, 1, 1, 1, rng.randint(0, 9))) for _ in range(requests)], 16, 4)


def test_tables_long_prompts_fill_many_workgroups():
    check_tables([0, 100, 3], [70001, 1, 33333], 16, 4400)


def test_tables_padding_shortage_and_narrow_tables():
    check_tables([3, 30, 0], [5, 9, 2], 8, 8, tokens=64)              # padded batch
    check_tables([3, 30, 0], [25, 29, 20], 8, 8, free=4)              # free list runs out
    check_tables([3, 30, 0], [25, 29, 20], 8, 4)                      # table too narrow
    check_tables([3, 99, 40], [25, 29, 0], 8, 4)                      # cached beyond the table
    check_tables([3, 30, 0], [25, 29, 20], 8, 8, start=3)             # list begun further on
    check_tables([3, 30, 0], [5, 9, 2], 8, 8, start=1 << 30)          # and past its end
    check_tables([3, 30, 0], [5, 9, 2], 8, 8, start=-2)
    check_tables([-4, 30, 0], [5, -9, 2], 8, 8)                       # negative counts are none


def test_tables_no_requests():
    step = mt.paged_tables(i32([]), i32([]), torch.empty(0, 4, dtype=torch.int32, device="cuda"),
                           i32([1]), page_size=16, tokens=5)
    assert step.slots.tolist() == [-1] * 5 and step.requests.tolist() == [-1] * 5
    assert step.starts.tolist() == [0] and step.taken.tolist() == [0]


def test_tables_drop_tokens_beyond_the_batch():
    # the caller's bound is too small: nothing is written past it
    check_tables([0, 8], [20, 20], 8, 8, tokens=25)


def test_tables_huge_counts_stop_at_the_largest_int():
    top = 2 ** 31 - 1
    table = torch.full((3, 4), -1, dtype=torch.int32, device="cuda")
    step = mt.paged_tables(i32([top, top, 0]), i32([top, 1, 2]), table, i32(list(range(20))),
                           page_size=16, tokens=8)
    assert step.lengths.tolist() == [top, top, 2]
    assert step.starts.tolist() == [0, top, top, top]
    assert step.slots.tolist() == [-1] * 8


def test_tables_strided_rows_keep_their_neighbours():
    wide = torch.full((3, 10), 77, dtype=torch.int32, device="cuda")
    view = wide[:, 2:6]
    view.fill_(-1)
    mt.paged_tables(i32([0, 0, 0]), i32([4, 9, 16]), view, i32(list(range(9))), page_size=4,
                    tokens=29)
    assert view.tolist() == [[0, -1, -1, -1], [1, 2, 3, -1], [4, 5, 6, 7]]
    assert bool((wide[:, :2] == 77).all()) and bool((wide[:, 6:] == 77).all())


# ---- append -------------------------------------------------------------------------------------------


def pool(pages, page, heads, dim, dtype, layout, fill=None, seed=0):
    """A cache tensor [pages, page, heads, dim]: heads outside or inside the slots, or interleaved
    with another tensor (odd page strides)."""
    g = torch.Generator("cuda").manual_seed(seed)
    shape = {"outer": (pages, heads, page, dim), "inner": (pages, page, heads, dim),
             "mixed": (pages, 3, page, heads, dim)}[layout]
    t = torch.randn(shape, generator=g, device="cuda")
    if fill is not None:
        t = torch.full_like(t, fill)
    t = t.to(dtype)
    return {"outer": lambda: t.transpose(1, 2), "inner": lambda: t, "mixed": lambda: t[:, 1]}[
        layout]()


def as_bits(t):
    return t.contiguous().view(torch.uint8 if t.dtype == FP8 else torch.int16).cpu()


@pytest.mark.parametrize("layout", ["outer", "inner", "mixed"])
@pytest.mark.parametrize("dtype,cache", [(torch.bfloat16, torch.bfloat16),
                                         (torch.float16, torch.float16), (torch.bfloat16, FP8),
                                         (torch.float16, FP8)])
@pytest.mark.parametrize("tokens,heads,dim,page", [(1, 2, 128, 16), (7, 1, 16, 1), (33, 3, 80, 20),
                                                   (300, 8, 64, 64), (65, 5, 256, 8)])
def test_append(tokens, heads, dim, page, dtype, cache, layout):
    g = torch.Generator("cuda").manual_seed(tokens)
    pages = 2 * tokens // page + 3
    keys, values = (pool(pages, page, heads, dim, cache, layout, seed=s) for s in (1, 2))
    scales = (0.7, 1.9) if cache == FP8 else (1.0, 1.0)
    fused = torch.randn(tokens, (3 * heads + 1) * dim, generator=g, device="cuda") * 100
    fused = fused.to(dtype)
    key = fused[:, dim:(heads + 1) * dim].unflatten(1, (heads, dim))
    value = fused[:, -heads * dim:].unflatten(1, (heads, dim))
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    slots[1::5] = -1
    slots[3::5] += pages * page  # past the cache
    want = []
    for rows, t, scale in ((key, keys, scales[0]), (value, values, scales[1])):
        held = rows
        if cache == FP8:
            held = torch.from_numpy(ref.fp8_values(
                (rows.float() / scale).double().cpu().numpy())).float().to(FP8).cuda()
        t = t.clone()
        view = t.view(torch.uint8) if cache == FP8 else t
        held = held.view(torch.uint8) if cache == FP8 else held
        for i, s in enumerate(slots.tolist()):
            if 0 <= s < pages * page:
                view[s // page, s % page] = held[i]
        want.append(as_bits(t))
    mt.paged_append(key, value, mt.PagedCache(keys, values, key_scale=scales[0],
                                              value_scale=scales[1]), slots)
    for got, expect in zip((keys, values), want):
        assert torch.equal(as_bits(got), expect)


def test_append_special_values_to_8_bits():
    special = [0.0, -0.0, float("inf"), -float("inf"), 448.0, 464.0, 480.0, 1e4, -1e4, 2.0 ** -9,
               2.0 ** -10, 1.5 * 2.0 ** -10, 2.0 ** -11, 17.0, 19.0, -18.0]
    key = torch.tensor(special, dtype=torch.bfloat16, device="cuda").reshape(1, 1, 16)
    cache = mt.PagedCache.allocate(1, 4, 1, 16, dtype=FP8)
    mt.paged_append(key, key, cache, torch.tensor([2], device="cuda"))
    got = cache.key[:, :, 0].float()[0, 2].double().cpu()
    clipped = [max(-448.0, min(448.0, x)) for x in special]
    assert got.tolist() == ref.fp8_values(clipped).tolist()
    nan = torch.full_like(key, float("nan"))
    mt.paged_append(nan, nan, cache, torch.tensor([0], device="cuda"))
    assert bool(torch.isnan(cache.value[:, :, 0].float()[0, 0]).all())


def test_append_unaligned_rows_and_no_tokens():
    base = torch.randn(6, 2 * 16 + 3, device="cuda").to(torch.float16)
    key = base[:, 3:].unflatten(1, (2, 16))  # rows 70 bytes apart
    cache = mt.PagedCache.allocate(2, 4, 2, 16, dtype=torch.float16)
    cache.key.zero_(), cache.value.zero_()
    slots = torch.arange(6, device="cuda") + 1
    mt.paged_append(key, key, cache, slots)
    got = cache.value.reshape(8, 2, 16)
    assert torch.equal(got[1:7], key) and not bool(got[0].any()) and not bool(got[7].any())
    mt.paged_append(key[:0], key[:0], cache, slots[:0])


# ---- attention ----------------------------------------------------------------------------------------


def attention_case(lengths, heads, kv_heads, dim, page, *, dtype=torch.bfloat16, cache=None,
                   layout="outer", window=0, scale=None, width=None, seed=0, spread=1.0):
    """Query, cache with NaN in every slot that no request's tokens use, tables whose unused entries
    are no pages at all, and lengths."""
    cache = cache or dtype
    g = torch.Generator("cuda").manual_seed(seed)
    counts = [-(-max(0, n) // page) for n in lengths]
    width = width or max(1, max(counts))
    pages = sum(counts) + 2
    keys, values = (pool(pages, page, kv_heads, dim, cache, layout, fill=float("nan"))
                    for _ in range(2))
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    table = torch.full((len(lengths), width), 2 ** 31 - 1, dtype=torch.int32)
    scales = (0.5, 2.0) if cache == FP8 else (1.0, 1.0)
    handle = mt.PagedCache(keys, values, key_scale=scales[0], value_scale=scales[1])
    slots = []
    for r, (n, c) in enumerate(zip(lengths, counts)):
        mine = [order.pop() for _ in range(c)]
        table[r, :min(c, width)] = torch.tensor(mine[:width], dtype=torch.int32)
        slots += [mine[t // page] * page + t % page for t in range(max(0, n))]
    if slots:
        rows = [(torch.randn(len(slots), kv_heads, dim, generator=g, device="cuda") * spread)
                .to(dtype) for _ in range(2)]
        mt.paged_append(*rows, handle, torch.tensor(slots, device="cuda"))
    query = torch.randn(len(lengths), heads, dim, generator=g, device="cuda").to(dtype)
    return query, handle, table.cuda(), i32(lengths)


def check_attention(query, cache, tables, lengths, *, window=0, scale=None):
    out, lse = mt.paged_attention(query, cache, tables, lengths, scale=scale, window=window or None,
                                  return_lse=True)
    want, want_lse, tol, lse_tol = ref.attention(
        query, cache.key, cache.value, tables.cpu(), lengths.tolist(),
        query.shape[2] ** -0.5 if scale is None else scale, window, cache.key_scale,
        cache.value_scale)
    assert out.dtype == query.dtype and out.shape == query.shape
    off = (out.double().cpu() - want).abs() - tol
    assert float(off.max()) <= 0, float(off.max())
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse.cpu()), empty)
    off = ((lse.double().cpu() - want_lse).abs() - lse_tol)[~empty]
    assert off.numel() == 0 or float(off.max()) <= 0, float(off.max())
    return out


RAGGED = [0, 1, 2, 7, 8, 9, 31, 32, 33, 127, 128, 129, 255, 300, 0, 513]


@pytest.mark.parametrize("dtype,cache", [(torch.bfloat16, torch.bfloat16),
                                         (torch.float16, torch.float16), (torch.bfloat16, FP8),
                                         (torch.float16, FP8)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(12, 2, 128), (14, 2, 64), (4, 4, 80), (24, 3, 96),
                                                (16, 1, 256), (5, 5, 16), (10, 2, 192),
                                                (7, 1, 112)])
def test_attention_types_and_heads(heads, kv_heads, dim, dtype, cache):
    check_attention(*attention_case(RAGGED, heads, kv_heads, dim, 16, dtype=dtype, cache=cache))


@pytest.mark.parametrize("cache", [torch.bfloat16, FP8])
@pytest.mark.parametrize("page", [1, 3, 8, 20, 24, 64, 256])
@pytest.mark.parametrize("layout", ["outer", "inner", "mixed"])
def test_attention_pages_and_layouts(layout, page, cache):
    check_attention(*attention_case(RAGGED, 8, 2, 64, page, cache=cache, layout=layout))


@pytest.mark.parametrize("heads,kv_heads", [(17, 1), (32, 1), (48, 1), (40, 2), (130, 2)])
def test_attention_many_heads_of_one(heads, kv_heads):
    check_attention(*attention_case([5, 0, 200, 1000], heads, kv_heads, 64, 16))


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 128, 511, 5000])
@pytest.mark.parametrize("page", [16, 5])
def test_attention_window(window, page):
    q, cache, tables, lengths = attention_case(RAGGED + [1400], 8, 2, 64, page)
    # pages wholly before the window may be gone
    for r, n in enumerate(lengths.tolist()):
        tables[r, :max(0, n - window) // page] = -1
    check_attention(q, cache, tables, lengths, window=window)


@pytest.mark.parametrize("requests", [1, 2, 65, 700])
def test_attention_rows_shared_by_many_workgroups(requests):
    lengths = [9000] if requests == 1 else [5000, 3] if requests == 2 else [
        (7 * i * i) % 97 + (3000 if i == 11 else 0) for i in range(requests)]
    check_attention(*attention_case(lengths, 4, 2, 64, 16))


@pytest.mark.parametrize("length,heads,kv_heads,dim", [
    (70000, 2, 1, 64),    # some 550 workgroups a row: two levels of joins of 32
    (20000, 16, 1, 256),  # some 160 of large parts: three levels of joins of 8
    (9000, 20, 1, 128)])  # two tiles of query heads, each joined by itself
def test_attention_joins_of_several_levels(length, heads, kv_heads, dim):
    case = attention_case([length, 0, 40], heads, kv_heads, dim, 16)
    first = check_attention(*case)
    again = mt.paged_attention(*case)
    assert torch.equal(first.view(torch.int16), again.view(torch.int16))
    assert not bool(workspace(torch.device("cuda", 0), 1)[:65536].any())


@pytest.mark.parametrize("seed", range(24))
def test_attention_random_shapes(seed):
    rng = random.Random(seed)
    dtype = rng.choice((torch.bfloat16, torch.float16))
    kv_heads = rng.choice((1, 2, 3, 8))
    most = rng.choice((3, 40, 300, 2500))
    lengths = [rng.choice((0, 1, rng.randint(0, most), rng.randint(0, most)))
               for _ in range(rng.randint(1, 40))]
    window = rng.choice((0, 0, rng.randint(1, most + 5)))
    case = attention_case(lengths, kv_heads * rng.choice((1, 2, 5, 8, 16, 18)), kv_heads,
                          16 * rng.randint(1, 16), rng.choice((1, 2, 7, 8, 16, 24, 30, 128)),
                          dtype=dtype, cache=rng.choice((dtype, dtype, FP8)),
                          layout=rng.choice(("outer", "inner", "mixed")), seed=seed)
    check_attention(*case, window=window, scale=rng.choice((None, 0.05, 1.0)))


def test_attention_more_requests_than_one_scan():
    lengths = [(13 * i) % 5 for i in range(4500)]
    check_attention(*attention_case(lengths, 2, 1, 32, 4))


def test_attention_lengths_are_limited_to_the_table():
    q, cache, tables, _ = attention_case([64, 40, 64], 4, 2, 64, 16)
    check_attention(q, cache, tables, i32([2 ** 31 - 1, -7, 65]))


def test_attention_leaves_out_what_is_no_page():
    q, cache, tables, lengths = attention_case([100, 40, 300, 16], 4, 2, 64, 16)
    tables[0, 2] = -1
    tables[0, 6] = 10 ** 6
    tables[2, ::2] = -(2 ** 31)
    tables[3] = -1  # nothing is left
    out = check_attention(q, cache, tables, lengths)
    assert not bool(out[3].any())


def test_attention_extreme_scores():
    # scores up to about +-30000: one token takes all, others underflow; no overflow anywhere
    q, cache, tables, lengths = attention_case([1, 77, 900], 4, 2, 128, 16, spread=30.0)
    check_attention(q, cache, tables, lengths, scale=8.0)
    check_attention(q, cache, tables, lengths, scale=-8.0)
    check_attention(q, cache, tables, lengths, scale=0.0)


def test_attention_small_probabilities_add_up_in_f16():
    # one token far ahead of many: each of the others is below f16's range, together they count
    n, dim = 40000, 64
    cache = mt.PagedCache.allocate(n // 16, 16, 1, dim, dtype=torch.float16)
    cache.key.zero_(), cache.value.fill_(1000.0)
    cache.key[0, 0, 0, 0] = 16.5
    cache.value[0, 0].zero_()
    q = torch.zeros(1, 1, dim, dtype=torch.float16, device="cuda")
    q[..., 0] = 1.0
    check_attention(q, cache, torch.arange(n // 16, dtype=torch.int32, device="cuda")[None],
                    i32([n]), scale=1.0)


def test_attention_infinities_and_nan_of_the_cache():
    q, cache, tables, lengths = attention_case([40, 40, 40, 40], 4, 2, 64, 16)
    table = tables.tolist()
    cache.value[table[0][1], 3, 0, 5] = float("inf")
    cache.key[table[1][0], 2, 1, 7] = float("nan")
    cache.key[table[2][0], :, :, 0] = 0.0
    out = mt.paged_attention(q, cache, tables, lengths)
    assert bool(torch.isinf(out[0, :2, 5]).all()) and bool(torch.isfinite(out[0, 2:]).all())
    assert bool(torch.isfinite(out[0, :2, :5]).all()) and bool(torch.isfinite(out[0, :2, 6:]).all())
    assert bool(torch.isnan(out[1, 2:]).all()) and bool(torch.isfinite(out[1, :2]).all())
    assert bool(torch.isfinite(out[2:]).all())
    cache.value[table[3][2], 1, 1, 9] = float("nan")
    cache.value[table[3][0], 4, 1, 10] = -float("inf")
    out = mt.paged_attention(q, cache, tables, lengths)[3]
    assert bool(torch.isnan(out[2:, 9]).all()) and bool((out[2:, 10] == -float("inf")).all())
    assert bool(torch.isfinite(out[:2]).all()) and bool(torch.isfinite(out[2:, 11:]).all())


def test_attention_offsets_past_32_bits():
    # 2.6e9 elements a side: pages whose offsets pass 2^32 bytes and 2^31 elements
    pages, page, kv_heads, dim = 20000, 64, 8, 256
    cache = mt.PagedCache.allocate(pages, page, kv_heads, dim)
    used = [0, pages - 1, pages // 2, pages - 2, 11000]
    g = torch.Generator("cuda").manual_seed(3)
    n = 64 * 5 - 9
    slots = torch.tensor([used[t // page] * page + t % page for t in range(n)], device="cuda")
    key, value = (torch.randn(n, kv_heads, dim, generator=g, device="cuda").bfloat16()
                  for _ in range(2))
    mt.paged_append(key, value, cache, slots)
    got = cache.key[pages - 1, :4]
    assert torch.equal(got, key[64:68])
    q = torch.randn(1, 16, dim, generator=g, device="cuda").bfloat16()
    check_attention(q, cache, i32([used]), i32([n]))


def test_attention_strided_and_unaligned_queries():
    _, cache, tables, lengths = attention_case([33, 100], 4, 2, 64, 16)
    fused = torch.randn(2, 10 * 64 + 1, device="cuda").bfloat16()
    check_attention(fused[:, 64:5 * 64].unflatten(1, (4, 64)), cache, tables, lengths)
    check_attention(fused[:, 1:4 * 64 + 1].unflatten(1, (4, 64)), cache, tables, lengths)
    wide = torch.zeros(2, 40, dtype=torch.int32, device="cuda")
    wide[:, 3:3 + tables.shape[1]] = tables
    check_attention(fused[:, :256].unflatten(1, (4, 64)), cache, wide[:, 3:3 + tables.shape[1]],
                    lengths)
    wide = wide.t().contiguous().t()[:, 3:3 + tables.shape[1]]
    check_attention(fused[:, :256].unflatten(1, (4, 64)), cache, wide, lengths)


def test_attention_no_requests_and_no_columns():
    q, cache, tables, lengths = attention_case([33, 100], 4, 2, 64, 16)
    assert mt.paged_attention(q[:0], cache, tables[:0], lengths[:0]).shape == (0, 4, 64)
    out, lse = mt.paged_attention(q, cache, tables[:, :0], lengths, return_lse=True)
    assert not bool(out.any()) and bool((lse == -float("inf")).all())


def test_attention_is_deterministic_and_leaves_its_counters_at_zero():
    case = attention_case([9000, 0, 77, 2500], 8, 2, 128, 16)
    first = mt.paged_attention(*case)
    for _ in range(5):
        assert torch.equal(mt.paged_attention(*case).view(torch.int16), first.view(torch.int16))
    assert not bool(workspace(torch.device("cuda", 0), 1)[:65536].any())


def test_attention_on_its_own_stream_and_in_a_graph():
    q, cache, tables, lengths = attention_case([700, 0, 77], 8, 2, 128, 16)
    one, none = torch.ones_like(lengths), i32([])
    want = mt.paged_attention(q, cache, tables, lengths)
    step = mt.paged_tables(lengths - 1, one, tables.clone(), none, page_size=16, tokens=3)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        assert torch.equal(mt.paged_attention(q, cache, tables, lengths), want)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        scratch = tables.clone()
        with torch.cuda.graph(graph, stream=stream):
            again = mt.paged_tables(lengths - 1, one, scratch, none, page_size=16, tokens=3)
            out = mt.paged_attention(q, cache, scratch, lengths)
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(again.slots[:1], step.slots[:1])
        # other work of the program between the replays, and other lengths in place
        mt.paged_attention(q, cache, tables, lengths)
        lengths.copy_(i32([700 - i, 0, 77]))
        want = mt.paged_attention(q, cache, tables, lengths)
        step = mt.paged_tables(lengths - 1, one, tables.clone(), none, page_size=16, tokens=3)


def test_a_step_end_to_end_over_two_steps():
    """Prompts, then one token each, through tables, append and attention, against a cache kept as
    plain lists."""
    page, kv_heads, heads, dim = 8, 2, 6, 32
    g = torch.Generator("cuda").manual_seed(9)
    cache = mt.PagedCache.allocate(40, page, kv_heads, dim)
    free = torch.randperm(40, generator=g, device="cuda").int()
    table = torch.full((3, 9), -1, dtype=torch.int32, device="cuda")
    cached, start = i32([0, 0, 0]), i32([0])
    seen = [[], [], []]
    for new in ([30, 8, 1], [1, 1, 0], [1, 1, 1], [1, 0, 1]):
        step = mt.paged_tables(cached, i32(new), table, free, page_size=page, tokens=sum(new) + 2,
                               free_start=start)
        start = start + step.taken
        key, value = (torch.randn(sum(new) + 2, kv_heads, dim, generator=g,
                                  device="cuda").bfloat16() for _ in range(2))
        mt.paged_append(key, value, cache, step.slots)
        for t, r in enumerate(step.requests.tolist()):
            if r >= 0:
                seen[r].append((key[t], value[t]))
        cached = step.lengths
        query = torch.randn(3, heads, dim, generator=g, device="cuda").bfloat16()
        out = mt.paged_attention(query, cache, table, cached)
        for r in range(3):
            k, v = (torch.stack([s[i] for s in seen[r]])[:, None] for i in (0, 1))
            whole = torch.zeros(1, len(seen[r]), dtype=torch.int32)
            whole[0] = torch.arange(len(seen[r]))
            want, _, tol, _ = ref.attention(query[r:r + 1], k, v, whole, [len(seen[r])],
                                            dim ** -0.5)
            assert bool(((out[r].double().cpu() - want[0]).abs() <= tol[0]).all())
    assert start.item() == len({int(p) for p in table.flatten().tolist() if p >= 0})


# ---- refusals -----------------------------------------------------------------------------------------


def test_refusals():
    q, cache, tables, lengths = attention_case([33, 100], 4, 2, 64, 16)
    bad = [
        (lambda: mt.paged_attention(q.float(), cache, tables, lengths), "bfloat16 or float16"),
        (lambda: mt.paged_attention(q.half(), cache, tables, lengths), "queries' dtype"),
        (lambda: mt.paged_attention(q[..., :32], cache, tables, lengths), "head_dim"),
        (lambda: mt.paged_attention(q[:, :3], cache, tables, lengths), "multiple of the cache"),
        (lambda: mt.paged_attention(q, cache, tables.long(), lengths), "int32"),
        (lambda: mt.paged_attention(q, cache, tables, lengths.long()), "int32"),
        (lambda: mt.paged_attention(q, cache, tables[:1], lengths), "same requests"),
        (lambda: mt.paged_attention(q, cache, tables, lengths, window=0), "window"),
        (lambda: mt.paged_attention(q, cache, tables, lengths, scale=float("nan")), "finite"),
        (lambda: mt.paged_attention(q.cpu(), cache, tables, lengths), "one ROCm device"),
        (lambda: mt.paged_append(q, q, cache, lengths.long()), "cache's heads"),
        (lambda: mt.paged_append(q[:, :2], q[:, :2], cache, lengths), "int64"),
        (lambda: mt.paged_append(q[:, :2].half(), q[:, :2].half(), cache, lengths.long()),
         "dtype"),
        (lambda: mt.PagedCache(cache.key, cache.value[:1]), "one shape"),
        (lambda: mt.PagedCache(cache.key.float(), cache.value.float()), "float8_e4m3fn"),
        (lambda: mt.PagedCache(cache.key, cache.value, key_scale=2.0), "scales"),
        (lambda: mt.PagedCache.allocate(1, 16, 1, 72), "multiple of 16"),
        (lambda: mt.PagedCache.allocate(1, 16, 1, 272), "multiple of 16"),
        (lambda: mt.PagedCache.allocate(1, 16, 1, 64, dtype=FP8, key_scale=0.0), "positive"),
        (lambda: mt.PagedCache(cache.key[..., 4:52], cache.value[..., 4:52]), "16 bytes"),
        (lambda: mt.paged_tables(lengths, lengths, tables.long(), lengths, page_size=16,
                                 tokens=4), "int32"),
        (lambda: mt.paged_tables(lengths[:1], lengths, tables, lengths, page_size=16, tokens=4),
         "same requests"),
        (lambda: mt.paged_tables(lengths, lengths, tables, lengths, page_size=0, tokens=4),
         "page_size"),
        (lambda: mt.paged_tables(lengths, lengths, tables, lengths, page_size=16, tokens=-1),
         "tokens"),
        (lambda: mt.paged_tables(lengths, lengths, tables, lengths, page_size=16, tokens=4,
                                 free_start=lengths), "free_start"),
    ]
    for call, message in bad:
        with pytest.raises(ValueError, match=message):
            call()
