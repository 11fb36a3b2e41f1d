"""Attention of chunks of new tokens over a paged cache on the GPU, against 64 bits, at the sizes, layouts,
masks and contents where it can go wrong."""

from __future__ import annotations

import math
import random

import pytest
import torch

import metile_amd as mt
from tests import serving_reference as ref
from tests.test_gpu_paged import FP8, i32, pool

pytestmark = pytest.mark.gpu


def case(new, past, *, heads=8, kv=2, dim=128, page=16, dtype=torch.bfloat16, cache=None, window=0,
         layout="outer", padding=0, seed=0, extra_columns=0, magnitude=1.0):
    """A packed batch of requests with `new` tokens each behind `past` ones."""
    g = torch.Generator("cuda").manual_seed(seed)
    rng = random.Random(seed)
    lengths = [a + b for a, b in zip(new, past)]
    width = max(1, -(-max(lengths, default=1) // page)) + extra_columns
    counts = [-(-n // page) for n in lengths]
    pages = max(1, sum(counts) + 3)
    numbers = list(range(pages))
    rng.shuffle(numbers)
    tables = [[numbers.pop() if c < n else -7 for c in range(width)] for n in counts]
    cache = cache or dtype
    scales = (0.5, 1.5) if cache == FP8 else (1.0, 1.0)
    key = pool(pages, page, kv, dim, cache, layout, seed=seed + 1)
    value = pool(pages, page, kv, dim, cache, layout, seed=seed + 2)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    query = (torch.randn(starts[-1] + padding, heads, dim, generator=g, device="cuda") * magnitude
             ).to(dtype)
    return dict(query=query, key=key, value=value, tables=i32(tables).reshape(len(new), width),
                lengths=i32(lengths), starts=i32(starts), window=window, scales=scales)


def run(c, **kwargs):
    cache = mt.PagedCache(c["key"], c["value"], key_scale=c["scales"][0], value_scale=c["scales"][1])
    return mt.paged_chunk_attention(c["query"], cache, c["tables"], c["lengths"], c["starts"],
                                    window=c["window"] or None, return_lse=True, **kwargs)


def expect(c, scale=None):
    scale = c["query"].shape[2] ** -0.5 if scale is None else scale
    return ref.chunk_attention(c["query"], c["key"], c["value"], c["tables"], c["lengths"].tolist(),
                               c["starts"].tolist(), scale, c["window"], *c["scales"])


def compare(got, want):
    out, lse = (t.double().cpu() for t in got)
    w_out, w_lse, out_tol, lse_tol = want
    for x, w, tol in ((out, w_out, out_tol), (lse, w_lse, lse_tol)):
        fine = torch.isfinite(w)
        assert torch.equal(torch.isnan(x), torch.isnan(w))
        assert torch.equal(x[~fine & ~torch.isnan(w)], w[~fine & ~torch.isnan(w)])
        off = (x - w).abs()[fine] - tol[fine]
        assert not off.numel() or float(off.max()) <= 0, float(off.max())


def check(*args, scale=None, **kwargs):
    c = case(*args, **kwargs)
    compare(run(c) if scale is None else run(c, scale=scale), expect(c, scale))
    return c


@pytest.mark.parametrize("new,past", [([1], [0]), ([1], [1]), ([2], [0]), ([31], [33]), ([33], [31]),
                                      ([64], [0]), ([65], [63]), ([129], [0]), ([5], [700]),
                                      ([300], [5]), ([17, 1, 40], [0, 129, 64])])
def test_small_shapes(new, past):
    check(new, past)


@pytest.mark.parametrize("heads,kv", [(1, 1), (2, 2), (7, 1), (12, 2), (14, 2), (28, 4), (20, 5), (48, 1),
                                      (33, 1), (129, 1), (130, 2)])
def test_head_layouts(heads, kv):
    check([9, 50], [100, 3], heads=heads, kv=kv, dim=64)


@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128, 144, 192, 208, 256])
@pytest.mark.parametrize("dtype,cache", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                         (torch.bfloat16, FP8), (torch.float16, FP8)])
def test_head_sizes_and_types(dim, dtype, cache):
    check([70, 3, 40], [90, 200, 0], heads=6, kv=2, dim=dim, dtype=dtype, cache=cache, seed=dim)


@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 64, 100, 256])
@pytest.mark.parametrize("layout", ["outer", "inner", "mixed"])
def test_pages_and_layouts(page, layout):
    check([33, 90, 1], [77, 0, 150], heads=4, kv=2, dim=64, page=page, layout=layout, extra_columns=2)


@pytest.mark.parametrize("window", [1, 2, 31, 64, 65, 130, 1000])
@pytest.mark.parametrize("group", [1, 4])
def test_windows(window, group):
    check([150, 1, 64], [20, 300, 64], heads=2 * group, kv=2, dim=64, window=window)


def test_ragged_batch_with_idle_requests_and_padding():
    rng = random.Random(5)
    new = [rng.choice((0, 0, 1, 2, rng.randint(1, 90))) for _ in range(70)]
    past = [rng.choice((0, 1, rng.randint(0, 400))) for _ in range(70)]
    c = check(new, past, heads=4, kv=2, dim=64, padding=13)
    out, lse = run(c)
    behind = c["starts"].tolist()[-1]
    assert bool((out[behind:] == 0).all()) and bool((lse[behind:] == -math.inf).all())


@pytest.mark.parametrize("requests", [64, 65, 1025, 4099])
def test_many_requests(requests):
    """More requests than a wave or the planning workgroup holds one each."""
    rng = random.Random(requests)
    new = [rng.choice((0, 1, 1, 2, 5)) for _ in range(requests)]
    past = [rng.randint(0, 12) for _ in range(requests)]
    check(new, past, heads=2, kv=1, dim=32, page=8, padding=2)


@pytest.mark.parametrize("dtype,cache", [(torch.bfloat16, torch.bfloat16), (torch.float16, FP8)])
def test_long_context_is_split(dtype, cache):
    """Few rows over many keys: the keys are split, the parts joined."""
    check([9], [9000], heads=8, kv=2, dim=128, dtype=dtype, cache=cache, page=64)
    check([1, 40, 3], [5000, 2500, 0], heads=4, kv=4, dim=80, dtype=dtype, cache=cache)
    check([30], [4000], heads=3, kv=1, dim=256, dtype=dtype, cache=cache, window=3000)


@pytest.mark.parametrize("past", [120, 185, 190, 250, 2000, 9000, 33000, 70000])
@pytest.mark.parametrize("heads,kv,dim", [(12, 2, 128), (3, 1, 64), (40, 1, 80), (2, 1, 256)])
def test_few_rows_in_few_and_many_parts(heads, kv, dim, past):
    check([6], [past], heads=heads, kv=kv, dim=dim, page=64, dtype=torch.float16)


@pytest.mark.parametrize("new,past", [(300, 8000), (1100, 3000)])
@pytest.mark.parametrize("heads,kv,dim,dtype", [(14, 2, 64, torch.float16), (24, 3, 96, torch.bfloat16),
                                                (20, 5, 192, torch.bfloat16), (16, 1, 256, FP8),
                                                (9, 1, 128, torch.float16)])
def test_one_request_in_parts_that_fill_rounds(heads, kv, dim, dtype, new, past):
    check([new], [past], heads=heads, kv=kv, dim=dim, page=64, cache=dtype,
          dtype=torch.bfloat16 if dtype == FP8 else dtype)


def test_many_parts_beside_requests_with_none():
    """Some tiles of a call are split and some are not, in both ways of counting them."""
    for requests in (60, 70):
        new = [(r % 4) * 3 for r in range(requests)]
        past = [9000 if r % 9 == 5 else r for r in range(requests)]
        check(new, past, heads=4, kv=1, dim=64, padding=5, seed=requests)


def test_large_scores_and_f16_probabilities():
    """Scores of hundreds, in rising and falling order along the keys."""
    for dtype in (torch.bfloat16, torch.float16):
        for order in (1, -1):
            c = case([40], [400], heads=2, kv=1, dim=64, dtype=dtype)
            ramp = torch.linspace(-3, 3, 440, device="cuda")[::1] * order
            ramp = (ramp if order == 1 else ramp)
            table = c["tables"][0].long()
            at = torch.arange(440, device="cuda")
            c["key"][table[at // 16], at % 16, 0] = ramp[:, None].to(dtype).expand(-1, 64)
            c["query"].fill_(2.0)
            compare(run(c), expect(c))


def test_scales():
    for scale in (0.0, -0.25, 1.0, 0.01):
        check([40, 3], [30, 200], heads=4, kv=2, dim=64, scale=scale)


def test_strided_queries_tables_and_vectors():
    c = case([30, 60], [50, 10], heads=6, kv=2, dim=64)
    want = expect(c)
    fused = torch.zeros(90, 10 * 64, dtype=torch.bfloat16, device="cuda")
    fused[:, 64:7 * 64] = c["query"].flatten(1)
    views = dict(query=fused[:, 64:7 * 64].unflatten(1, (6, 64)),
                 tables=torch.stack([c["tables"]] * 3, -1)[..., 1],
                 lengths=torch.stack([c["lengths"]] * 2, -1)[:, 0],
                 starts=torch.stack([c["starts"]] * 2, -1)[:, 1])
    compare(run({**c, **views}), want)
    odd = torch.zeros(90 * 6 * 64 + 3, dtype=torch.bfloat16, device="cuda")[3:].view(90, 6, 64)
    odd.copy_(c["query"])
    compare(run({**c, "query": odd}), want)
    turned = c["query"].transpose(0, 1).contiguous().transpose(0, 1)
    compare(run({**c, "query": turned}), want)
    wide = torch.full((2, c["tables"].shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    wide[:, 2:-3] = c["tables"]
    compare(run({**c, "tables": wide[:, 2:-3]}), want)


def test_tokens_on_no_page_are_left_out():
    for bad in (-1, 10 ** 6, -2 ** 31):
        c = case([70, 5], [60, 100], heads=4, kv=2, dim=64)
        c["tables"][0, 2] = bad
        c["tables"][0, 8] = bad   # the page of the last tokens
        c["tables"][1].fill_(bad)  # nothing at all
        compare(run(c), expect(c))


def test_lengths_beyond_the_table_below_the_chunk_and_negative():
    c = case([20, 20, 20, 20], [30, 30, 30, 30], heads=2, kv=1, dim=64)
    most = c["tables"].shape[1] * 16
    c["lengths"].copy_(i32([most + 9, 12, -5, 2 ** 31 - 1]))
    compare(run(c), expect(c))


def test_starts_out_of_order_stay_in_bounds():
    c = case([20, 20, 20], [30, 30, 30], heads=2, kv=1, dim=64, padding=4)
    for starts in ([0, 40, 20, 60], [0, -5, 2 ** 31 - 1, 60], [64, 64, 64, 64], [0, 64, 0, 64]):
        out, lse = run({**c, "starts": i32(starts)})
        assert out.shape == c["query"].shape and lse.shape == (64, 2)
    torch.cuda.synchronize()


@pytest.mark.parametrize("content", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("past", [0, 100, 3000])
def test_what_no_token_sees_does_not_matter(content, dtype, past):
    """Slots behind the last token, pages of no request, and later tokens of the chunk."""
    c = case([50, 20], [past, 7], heads=4, kv=2, dim=64, dtype=dtype)
    want = expect(c)
    length = int(c["lengths"][0])
    for side in (c["key"], c["value"]):
        used = torch.zeros(side.shape[:2], dtype=torch.bool, device="cuda")
        for r in range(2):
            at = torch.arange(int(c["lengths"][r]), device="cuda")
            used[c["tables"][r].long()[at // 16], at % 16] = True
        side[~used] = content
    compare(run(c), want)
    # the last three tokens' values: theirs alone; the keys: the rows that see them have no numbers
    for back in (1, 2, 3):
        page = int(c["tables"][0, (length - back) // 16])
        c["value"][page, (length - back) % 16, 0, 5] = content
    got, want = run(c), expect(c)
    compare(got, want)
    assert bool(torch.isfinite(got[0][:47]).all())
    assert not bool(torch.isfinite(got[0][47:50, :2, 5]).any())


def test_infinite_value_of_a_small_probability():
    """exp(-200) is below every type's range, but not nothing: infinity, not NaN."""
    for dtype in (torch.bfloat16, torch.float16):
        for past in (0, 4000):
            c = case([40], [past], heads=1, kv=1, dim=64, dtype=dtype)
            c["query"].fill_(1.0)
            c["key"].fill_(0.0)
            length = past + 40
            table = c["tables"][0].long().tolist()

            def place(j):
                return table[j // 16], j % 16
            c["key"][place(1)] = -25.0  # a score of -200, then zeros
            c["value"][place(1)] = math.inf
            got, want = run(c), expect(c)
            compare(got, want)
            assert bool((got[0][-1] == math.inf).all())
            c["value"][place(length - 2)][0, 3] = -math.inf  # +inf and -inf: no number
            got = run(c)
            assert bool(torch.isnan(got[0][-1, 0, 3])) and bool((got[0][-1, 0, 4:] == math.inf).all())


def test_empty_batches():
    cache = mt.PagedCache.allocate(2, 16, 2, 64)
    q = torch.randn(5, 4, 64, device="cuda").bfloat16()
    empty = torch.empty(0, 3, dtype=torch.int32, device="cuda")
    out, lse = mt.paged_chunk_attention(q, cache, empty, i32([]), i32([0]), return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    out = mt.paged_chunk_attention(q[:0], cache, i32([[0]]), i32([3]), i32([0, 0]))
    assert out.shape == (0, 4, 64)
    out = mt.paged_chunk_attention(q, cache, i32([[0], [1]]), i32([0, 0]), i32([0, 0, 0]))
    assert bool((out == 0).all())


def test_one_new_token_agrees_with_decode_attention():
    c = case([1] * 9, [0, 1, 15, 16, 63, 64, 500, 2000, 90], heads=8, kv=2, dim=128)
    cache = mt.PagedCache(c["key"], c["value"])
    want, want_lse = mt.paged_attention(c["query"], cache, c["tables"], c["lengths"], return_lse=True)
    out, lse = run(c)
    # two results of the same sums, rounded once each, and probabilities rounded to 2^-8 in one
    spread = 2.0 ** -7 * want.float().abs() + 2.0 ** -8 * c["value"].float().abs().max()
    assert bool(((out.float() - want.float()).abs() <= spread).all())
    assert torch.allclose(lse, want_lse, rtol=2e-6, atol=2e-6)


def test_results_do_not_change_from_run_to_run():
    c = case([100, 3, 300], [2000, 4000, 0], heads=8, kv=2, dim=128)
    first = run(c)
    for _ in range(5):
        again = run(c)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_graph_replays_with_other_lengths_and_another_stream():
    c = case([40, 30], [100, 2500], heads=4, kv=2, dim=64, padding=10, extra_columns=4)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run(c)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = run(c)
    for lengths, starts in (([140, 2530], [0, 40, 70]), ([60, 2000], [0, 50, 75]), ([5, 1], [0, 5, 6]),
                            ([0, 2530], [0, 0, 80])):
        c["lengths"].copy_(i32(lengths))
        c["starts"].copy_(i32(starts))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager = run(c)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))
        compare(got, expect(c))


def test_calls_on_two_streams_at_once():
    cases = [case([60, 9], [3000, 1000], heads=8, kv=2, dim=128, seed=s) for s in (1, 2)]
    want = [run(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(10):
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(run(c))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))


def far_pool(pages, page, heads, dim, dtype, apart, seed):
    """A cache whose pages lie `apart` values from each other."""
    t = torch.empty(pages * apart, dtype=dtype, device="cuda").as_strided(
        (pages, page, heads, dim), (apart, heads * dim, dim, 1))
    t.copy_(pool(pages, page, heads, dim, dtype, "inner", seed=seed))
    return t


@pytest.mark.parametrize("dim,dtype", [(64, torch.bfloat16), (80, FP8), (96, torch.bfloat16),
                                       (128, torch.bfloat16), (128, FP8), (192, FP8),
                                       (256, torch.bfloat16)])
@pytest.mark.parametrize("size", [(1 << 32) - (1 << 20), (1 << 32) + (1 << 20), 11 << 30])
def test_offsets_about_and_beyond_32_bits(dim, dtype, size):
    """Keys and values that end just below 4 GiB, just above, and far above."""
    pages, page, heads = 9, 16, 2
    apart = size // (pages * dtype.itemsize) // 16 * 16
    c = case([70, 1], [40, 10], heads=4, kv=heads, dim=dim, page=page, cache=dtype)
    c["scales"] = (1.0, 1.0)
    c["tables"] = i32([[8, 0, 7, 1, 6, 2, 5], [4, 8, 3, 0, 1, 2, 5]])
    c["key"], c["value"] = (far_pool(pages, page, heads, dim, dtype, apart, s) for s in (1, 2))
    compare(run(c), expect(c))


def test_largest_window_of_a_chunk_longer_than_its_request():
    c = case([300], [0], heads=2, kv=1, dim=64, window=(1 << 31) - 1)
    c["lengths"].copy_(i32([200]))
    compare(run(c), expect(c))


def test_longest_table():
    """2^31 - 128 keys, all of them one page's: the page's result. A part's sums have 2^16 equal terms (blocks),
    each rounded by at most 2^-24 of the sum, so they are off by 2^-8 of it at most."""
    page, dim = 64, 16
    key, value = (pool(1, page, 1, dim, torch.bfloat16, "inner", seed=s) for s in (1, 2))
    cache = mt.PagedCache(key, value)
    width = (1 << 25) - 2
    tables = torch.zeros(1, width, dtype=torch.int32, device="cuda")
    q = torch.randn(1, 1, dim, device="cuda").bfloat16()
    one, starts = i32([page]), i32([0, 1])
    out, lse = mt.paged_chunk_attention(q, cache, tables, i32([width * page]), starts, return_lse=True)
    want, want_lse = mt.paged_chunk_attention(q, cache, tables, one, starts, return_lse=True)
    assert float((lse - want_lse - math.log(width)).abs().max()) <= 2.0 ** -8 + 2.0 ** -20
    # (numerator and denominator, a rounding of either result)
    assert float((out.float() - want.float()).abs().max()) <= (2.0 ** -7 + 2.0 ** -7) * float(value.abs().max())
    over = mt.paged_chunk_attention(q, cache, tables, i32([(1 << 31) - 1]), starts)
    assert torch.equal(over, out)


@pytest.mark.parametrize("odd", [math.nan, math.inf])
def test_queries_that_are_no_numbers_keep_to_themselves(odd):
    c = case([40, 3], [200, 3000], heads=4, kv=2, dim=64)
    clean = run(c)
    want = expect(c)
    c["query"][5, 2, 7] = odd
    c["query"][41, 0, 0] = odd
    out, lse = run(c)
    for row, head in ((5, 2), (41, 0)):
        assert bool(torch.isnan(out[row, head]).all()) and not bool(torch.isfinite(lse[row, head]))
        out[row, head], lse[row, head] = clean[0][row, head], clean[1][row, head]
    compare((out, lse), want)


def test_8_bit_nan_that_no_token_sees():
    c = case([30], [70], heads=4, kv=2, dim=64, cache=FP8, extra_columns=1)
    want = expect(c)
    used = set(c["tables"][0, :7].tolist())
    for t in (c["key"], c["value"]):
        bits = t.view(torch.uint8)
        for p in range(t.shape[0]):
            if p not in used:
                bits[p] = 0x7f
        bits[int(c["tables"][0, 6]), 4:] = 0x7f  # behind the 100 tokens
    compare(run(c), want)


def test_refusals():
    cache = mt.PagedCache.allocate(4, 16, 2, 64)
    q = torch.zeros(5, 4, 64, dtype=torch.bfloat16, device="cuda")
    t, n, s = i32([[0, 1]]), i32([5]), i32([0, 5])

    def call(query=q, c=cache, tables=t, lengths=n, starts=s, **kwargs):
        return mt.paged_chunk_attention(query, c, tables, lengths, starts, **kwargs)

    call()
    for kwargs, text in ((dict(query=q.float()), "bfloat16 or float16"), (dict(query=q.half()), "queries' dtype"),
                         (dict(query=q[..., :32]), "head_dim"), (dict(query=q[:, :3]), "multiple"),
                         (dict(query=q[0]), "head_dim"), (dict(tables=t.long()), "int32"),
                         (dict(tables=t[0]), "int32"), (dict(lengths=i32([5, 5])), "same requests"),
                         (dict(starts=i32([0])), "same requests"), (dict(starts=s.long()), "int32"),
                         (dict(window=0), "window"), (dict(scale=float("nan")), "finite"),
                         (dict(lengths=n.cpu()), "ROCm device")):
        with pytest.raises(ValueError, match=text):
            call(**kwargs)
