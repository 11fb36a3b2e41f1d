"""Log probabilities, ranks, entropies and alternatives on the GPU against 64 bits: order exactly, values by
the rounding of fp32 sums."""

from __future__ import annotations

import math

import pytest
import torch

import metile_amd as mt
from tests import serving_reference as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def check(logits, tokens, top, temperature=1.0):
    got = mt.token_logprobs(logits, tokens, top=top, temperature=temperature)
    rows, vocab = logits.shape
    want = ref.logprobs(logits, tokens, top, temperature)
    # A thread's sum runs over vocab / 256 terms (or a part's share), then over some hundred threads and
    # parts in a tree: relative errors of a few units of 2^-24 in each factor (the difference, the
    # reciprocal of the temperature, the exponential of an argument of size x: |x| units), and less than
    # `vocab / 256` of them added up in the sum at worst. What is measured is far less.
    x = logits.double().cpu()
    fine = torch.where(torch.isfinite(x), x, 0.0)
    spread = ((fine.amax(-1) - fine.amin(-1)) / temperature).clamp(min=1.0)
    unit = 2.0 ** -24 * (8 + min(vocab, 8192 * 32) / 256)
    tol = unit * 4 + 2.0 ** -21 * torch.log(torch.tensor(float(vocab) + 1))
    if tokens is not None:
        lp = got.logprobs.double().cpu()
        gone = torch.isinf(want[0])
        assert torch.equal(lp[gone], want[0][gone])
        assert bool(((lp - want[0]).abs() <= tol + 2.0 ** -22 * want[0].abs())[~gone].all())
        assert got.ranks.tolist() == want[2].tolist() and got.ranks.dtype == torch.int32
    else:
        assert got.logprobs is None and got.ranks is None
    h = got.entropies.double().cpu()
    assert bool(((h - want[1]).abs() <= tol + unit * spread * 4).all()), float((h - want[1]).abs().max())
    assert got.top_tokens.tolist() == want[4].tolist() and got.top_tokens.dtype == torch.int64
    best = got.top_logprobs.double().cpu()
    gone = torch.isinf(want[3])
    assert torch.equal(best[gone], want[3][gone])
    assert bool(((best - want[3]).abs() <= tol + 2.0 ** -22 * want[3].abs())[~gone].all())
    return got


def randn(rows, vocab, dtype, seed=0, scale=3.0):
    g = torch.Generator("cuda").manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g, device="cuda") * scale).to(dtype)
    return x, torch.randint(vocab, (rows,), generator=g, device="cuda")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 63, 255, 257, 2047, 2049, 8191, 8192, 8193, 16385, 50001,
                                   152064])
def test_vocabularies(vocab, dtype):
    x, t = randn(5, vocab, dtype, seed=vocab)
    check(x, t, min(vocab, 20))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 2, 63, 200, 1500])
def test_rows(rows, dtype):
    x, t = randn(rows, 20011, dtype, seed=rows)
    check(x, t, 5)


@pytest.mark.parametrize("top", [0, 1, 2, 31, 32])
@pytest.mark.parametrize("rows,vocab", [(3, 32), (3, 40000), (1100, 9000)])
def test_numbers_of_alternatives(top, rows, vocab):
    x, t = randn(rows, vocab, torch.bfloat16, seed=top)
    check(x, t, top)
    check(x, None, top)


@pytest.mark.parametrize("temperature", [0.01, 0.7, 3.0, 1000.0])
def test_temperatures(temperature):
    x, t = randn(7, 30000, torch.float32, scale=1.0)
    check(x, t, 8, temperature)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [2, 1300])
def test_ties_go_to_the_lowest_index(dtype, rows):
    for vocab in (300, 17000):
        x = torch.full((rows, vocab), 1.5, dtype=dtype, device="cuda")  # one value
        t = torch.arange(rows, device="cuda") * 7 % vocab
        check(x, t, 32)
        x = (torch.arange(vocab, device="cuda") % 5).to(dtype).expand(rows, vocab).contiguous()
        check(x, t, 32)
        x = torch.zeros(rows, vocab, dtype=dtype, device="cuda")  # zeros of both signs are equal
        x[:, ::3] = -0.0
        check(x, t, 20)
        x = -torch.ones(rows, vocab, dtype=dtype, device="cuda")  # few that differ, at the end
        x[:, -3:] = 2.0
        x[:, vocab // 2] = 3.0
        check(x, t, 32)


@pytest.mark.parametrize("dtype", TYPES)
def test_sorted_rows(dtype):
    """All alternatives in one group of values, first or last."""
    for vocab in (1000, 40000):
        up = torch.linspace(-10, 10, vocab, device="cuda").to(dtype)
        x = torch.stack([up, up.flip(0)])
        check(x, torch.tensor([3, vocab - 2], device="cuda"), 32)


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_tokens(dtype):
    lowest = torch.finfo(dtype).min
    for mask in (-math.inf, lowest):
        x, t = randn(6, 30000, dtype)
        x[0, 100:] = mask
        x[1, :-1] = mask            # one token left
        x[2, ::2] = mask
        x[3, :] = mask
        x[3, 77], x[3, 20000] = 1.0, 2.0
        x[4, 5] = mask
        t[0], t[1], t[4] = 50, 29999, 5
        check(x, t, 20)
    x = torch.full((2, 9000), lowest, dtype=dtype, device="cuda")  # nothing but the lowest
    check(x, torch.tensor([4, 8999], device="cuda"), 3)


@pytest.mark.parametrize("rows,vocab", [(1, 1), (2, 300), (3, 40000), (1200, 9000)])
def test_rows_that_allow_nothing(rows, vocab):
    x = torch.full((rows, vocab), -math.inf, dtype=torch.bfloat16, device="cuda")
    k = min(vocab, 4)
    got = mt.token_logprobs(x, torch.zeros(rows, dtype=torch.int64, device="cuda"), top=k)
    assert bool((got.logprobs == -math.inf).all()) and bool((got.entropies == 0).all())
    assert bool((got.top_logprobs == -math.inf).all())
    assert got.top_tokens.tolist() == [list(range(k))] * rows and bool((got.ranks == 0).all())


@pytest.mark.parametrize("rows,vocab", [(2, 300), (2, 40000), (1200, 9000)])
@pytest.mark.parametrize("odd", [math.nan, math.inf])
def test_rows_without_numbers(rows, vocab, odd):
    x, t = randn(rows, vocab, torch.float32)
    clean = ref.logprobs(x, t, 5)
    x[1, 17] = odd
    got = mt.token_logprobs(x, t, top=5)
    assert bool(torch.isnan(got.logprobs[1])) and bool(torch.isnan(got.entropies[1]))
    assert bool(torch.isnan(got.top_logprobs[1]).all())
    if odd != odd:  # no alternative; the others in their order
        x[1, 17] = -math.inf
        assert got.top_tokens[1].tolist() == ref.logprobs(x[1:2], t[1:2], 5)[4][0].tolist()
    else:
        assert int(got.top_tokens[1, 0]) == 17
    assert torch.allclose(got.logprobs[:1].double().cpu(), clean[0][:1], rtol=1e-5)
    x[:] = math.nan
    x[0, 9] = 1.0
    got = mt.token_logprobs(x, t, top=3)
    assert got.top_tokens[:2].tolist() == [[9, -1, -1], [-1, -1, -1]]


def test_tokens_outside_the_vocabulary():
    x, t = randn(6, 12000, torch.float16)
    want = check(x, t, 2)
    outside = t.clone()
    outside[1], outside[3], outside[4] = -1, 12000, 2 ** 62
    got = mt.token_logprobs(x, outside, top=2)
    gone = torch.tensor([False, True, False, True, True, False], device="cuda")
    assert bool((got.logprobs[gone] == -math.inf).all()) and bool((got.ranks[gone] == -1).all())
    assert torch.equal(got.logprobs[~gone], want.logprobs[~gone])
    assert torch.equal(got.ranks[~gone], want.ranks[~gone])


@pytest.mark.parametrize("dtype", TYPES)
def test_likely_tokens_keep_their_small_log_probabilities(dtype):
    """-log1p of what is left, to an error of 2^-23 of the whole."""
    x = torch.full((3, 20000), -20.0, dtype=dtype, device="cuda")
    x[:, 11] = torch.tensor([0.0, 8.0, 20.0], device="cuda").to(dtype)
    got = check(x, torch.full((3,), 11, device="cuda"), 1)
    want = ref.logprobs(x, torch.full((3,), 11), 1)[0]
    assert bool(((got.logprobs.double().cpu() - want).abs() <= 2.0 ** -22).all())


def test_strides_shapes_and_alignment():
    base, t = randn(12, 20003, torch.bfloat16)
    want = mt.token_logprobs(base, t, top=7)
    wide = torch.zeros(12, 20003 + 61, dtype=torch.bfloat16, device="cuda")
    for offset in (0, 1, 5, 8):
        wide.zero_()
        view = wide[:, offset:offset + 20003]
        view.copy_(base)
        for a, b in zip(want, mt.token_logprobs(view, t, top=7)):
            assert torch.equal(a, b)
    for a, b in zip(want, mt.token_logprobs(base.t().contiguous().t(), t, top=7)):
        assert torch.equal(a, b)
    shaped = mt.token_logprobs(base.view(3, 4, -1), t.view(3, 4), top=7)
    assert shaped.logprobs.shape == (3, 4) and shaped.top_tokens.shape == (3, 4, 7)
    for a, b in zip(want, shaped):
        assert torch.equal(a.flatten(), b.flatten())
    one = mt.token_logprobs(base[0], t[0], top=7)
    assert one.entropies.shape == () and one.top_logprobs.shape == (7,)
    same = mt.token_logprobs(base[:1].expand(12, -1), t, top=2)
    assert torch.equal(same.entropies, same.entropies[:1].expand(12))
    f32 = torch.zeros(3, 20003 * 4 + 1, device="cuda")[:, 1:20004]
    f32.copy_(base[:3])
    check(f32, t[:3], 5)


def test_vocabulary_in_several_parts_and_the_largest():
    x, t = randn(2, 600011, torch.bfloat16)
    check(x, t, 20)
    x = torch.randn(1, 1 << 24, device="cuda").bfloat16()
    x[0, -1] = 30.0
    got = mt.token_logprobs(x, torch.tensor([(1 << 24) - 1], device="cuda"), top=2)
    assert int(got.ranks) == 0 and int(got.top_tokens[0, 0]) == (1 << 24) - 1


def test_ties_in_long_rows():
    """Many equal maxima over several batches of a workgroup and several parts, of every kind of row."""
    for rows, vocab in ((3, 70001), (3, 300007), (256, 70001), (257, 40000)):
        x = torch.full((rows, vocab), -2.0, dtype=torch.bfloat16, device="cuda")
        x[:, ::3] = 1.0
        x[0, vocab - 5:] = 4.0
        x[1, 60:90] = 5.0
        check(x, torch.full((rows,), vocab - 1, device="cuda"), 32)


def test_more_rows_than_one_launch_takes():
    rows = (1 << 22) + 5
    x = torch.zeros(rows, 9, dtype=torch.float16, device="cuda")
    t = torch.arange(rows, device="cuda") % 9
    x[torch.arange(rows, device="cuda"), t] = (t + 1).to(torch.float16)
    got = mt.token_logprobs(x, t, top=2)
    few = mt.token_logprobs(x[:9], t[:9], top=2)
    want = ref.logprobs(x[:9], t[:9], 2)
    assert bool(((few.logprobs.double().cpu() - want[0]).abs() <= 2.0 ** -20).all())
    for a, b in zip(got, few):
        assert torch.equal(a, b[t])


def test_empty():
    got = mt.token_logprobs(torch.empty(0, 50, device="cuda"),
                            torch.empty(0, dtype=torch.int64, device="cuda"), top=3)
    assert got.logprobs.shape == (0,) and got.top_tokens.shape == (0, 3)


@pytest.mark.parametrize("rows", [3, 600])
def test_the_same_bits_each_time_in_graphs_and_on_other_streams(rows):
    x, t = randn(rows, 50001, torch.bfloat16)
    want = mt.token_logprobs(x, t, top=9)
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(want, mt.token_logprobs(x, t, top=9)))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        mt.token_logprobs(x, t, top=9)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = mt.token_logprobs(x, t, top=9)
    for seed in (0, 5, 6):
        fresh, tokens = randn(rows, 50001, torch.bfloat16, seed=seed)
        x.copy_(fresh)
        t.copy_(tokens)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager = mt.token_logprobs(x, t, top=9)
        assert all(torch.equal(a, b) for a, b in zip(got, eager))


def test_refusals():
    x, t = randn(3, 100, torch.bfloat16)
    for args, kwargs, text in (((x.double(), t), {}, "bfloat16, float16 or float32"),
                               ((x, t.int()), {}, "int64"), ((x, t[:2]), {}, "int64"),
                               ((x, t), dict(top=33), "top"), ((x, t), dict(top=-1), "top"),
                               ((x[:, :4], t), dict(top=5), "top"), ((x[:, :0], t), {}, "vocab"),
                               ((x, t), dict(temperature=0.0), "temperature"),
                               ((x, t), dict(temperature=-1.0), "temperature"),
                               ((x, t), dict(temperature=float("nan")), "temperature"),
                               ((x, t.cpu()), {}, "ROCm device"), ((x.cpu(), t.cpu()), {}, "ROCm device")):
        with pytest.raises(ValueError, match=text):
            mt.token_logprobs(*args, **kwargs)
