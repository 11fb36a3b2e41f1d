"""Paged attention beside infinities: what is finite keeps the precision it has without them."""

from __future__ import annotations

import pytest
import torch

import metile_amd as mt
from tests import paged_reference as ref
from tests.test_gpu_paged import attention_case

pytestmark = pytest.mark.gpu


def held(cache):
    """The cache's tensors and scales for the 64-bit form, which only reads them."""
    return cache.key.clone(), cache.value.clone()


def outside(out, want, tol):
    return float(((out.double().cpu() - want).abs() - tol).max())


# One wave's rows (up to 128 tokens) and rows that waves and workgroups share.
LENGTHS = [[2], [33, 5, 100, 128], [129, 700], [6000, 40]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (16, 1, 128), (3, 1, 80), (8, 2, 256)])
@pytest.mark.parametrize("lengths", LENGTHS)
def test_columns_beside_an_infinite_value(lengths, heads, kv_heads, dim, dtype):
    q, cache, tables, n = attention_case(lengths, heads, kv_heads, dim, 16, dtype=dtype)
    key, value = held(cache)
    table = tables.tolist()
    for r, length in enumerate(lengths):
        for t, d in ((length // 2, 3), (length - 1, dim - 1)):
            cache.value[table[r][t // 16], t % 16, 0, d] = float("inf")
            value[table[r][t // 16], t % 16, 0, d] = 0.0
    out, lse = mt.paged_attention(q, cache, tables, n, return_lse=True)
    want, want_lse, tol, lse_tol = ref.attention(q, key, value, tables.cpu(), lengths, dim ** -0.5)
    group = heads // kv_heads
    for d in (3, dim - 1):
        assert bool((out[:, :group, d] == float("inf")).all())
        out[:, :group, d] = 0.0
        want[:, :group, d] = 0.0
    assert outside(out, want, tol) <= 0
    assert outside(lse, want_lse, lse_tol) <= 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths", LENGTHS)
def test_heads_that_an_infinite_key_leaves_out(lengths, dtype):
    # the score is -inf for heads whose query is negative there: the token has no part in them
    q, cache, tables, n = attention_case(lengths, 6, 1, 64, 1, dtype=dtype)
    q[:, :, 9] = q[:, :, 9].abs() + 0.25
    q[:, 1::2, 9] *= -1
    without = tables.cpu()
    for r, length in enumerate(lengths):
        t = length // 3
        cache.key[int(tables[r, t]), 0, 0, 9] = float("inf")
        without[r, t] = -1
    key, value = held(cache)
    out, lse = mt.paged_attention(q, cache, tables, n, return_lse=True)
    want, want_lse, tol, lse_tol = ref.attention(q, key, value, without, lengths, 64 ** -0.5)
    assert bool(torch.isnan(out[:, ::2]).all())
    assert outside(out[:, 1::2], want[:, 1::2], tol[:, 1::2]) <= 0
    assert outside(lse[:, 1::2], want_lse[:, 1::2], lse_tol[:, 1::2]) <= 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("below", [9.0, 18.0, 26.0, 40.0, 60.0])
def test_infinite_values_of_small_probability(below, dtype):
    # exp(-60) is 9e-27, far below float16's range: times infinity it is infinity all the same
    cache = mt.PagedCache.allocate(8, 16, 1, 64, dtype=dtype)
    cache.key.zero_(), cache.value.fill_(1.0)
    cache.key[0, 0, 0, 0] = below
    cache.value[3, 5, 0, 7], cache.value[5, 1, 0, 8] = float("inf"), -float("inf")
    q = torch.zeros(1, 2, 64, dtype=dtype, device="cuda")
    q[..., 0] = 1.0
    for n in (100, 128):
        out = mt.paged_attention(q, cache, torch.arange(8, dtype=torch.int32, device="cuda")[None],
                                 torch.tensor([n], dtype=torch.int32, device="cuda"), scale=1.0)[0]
        assert bool((out[:, 7] == float("inf")).all()) and bool((out[:, 8] == -float("inf")).all())
        out[:, 7:9] = 1.0
        assert bool((out == 1.0).all())


@pytest.mark.parametrize("below", [12.0, 18.0, 21.0, 24.0, 27.0])
@pytest.mark.parametrize("infinite", [False, True])
def test_small_probabilities_of_large_values_in_f16(infinite, below):
    # one token far ahead whose value is 0, 127 with 60000: exp(-21) of that counts. A probability is
    # off by 2^-24 of itself or 2^-39 of the largest, which is 1, in either form of the products
    n = 128
    cache = mt.PagedCache.allocate(8, 16, 1, 64, dtype=torch.float16)
    cache.key.zero_(), cache.value.fill_(60000.0)
    cache.key[0, 0, 0, 0] = below
    cache.value[0, 0].zero_()
    if infinite:
        cache.value[3, 5, 0, 7] = float("inf")
    q = torch.zeros(1, 2, 64, dtype=torch.float16, device="cuda")
    q[..., 0] = 1.0
    out = mt.paged_attention(q, cache, torch.arange(8, dtype=torch.int32, device="cuda")[None],
                             torch.tensor([n], dtype=torch.int32, device="cuda"), scale=1.0)[0]
    if infinite:
        assert bool((out[:, 7] == float("inf")).all())
        out[:, 7] = out[:, 8]
    p = torch.tensor(-below, dtype=torch.float64).exp()
    want = 60000.0 * (n - 1) * p / (1 + (n - 1) * p)
    # fp32 exponents and sums: 2^-20 of the result; f16's own rounding, 2^-25 below its normal numbers
    tol = (2.0 ** -11 + 2.0 ** -20) * want + 60000.0 * (n - 1) * 2.0 ** -39 + 2.0 ** -25
    assert float((out.double().cpu() - want).abs().max()) <= float(tol)


@pytest.mark.parametrize("dtype,cache_dtype", [(torch.bfloat16, torch.bfloat16),
                                               (torch.float16, torch.float16),
                                               (torch.bfloat16, torch.float8_e4m3fn),
                                               (torch.float16, torch.float8_e4m3fn)])
@pytest.mark.parametrize("lengths", LENGTHS)
def test_columns_beside_a_value_that_is_no_number(lengths, dtype, cache_dtype):
    q, cache, tables, n = attention_case(lengths, 6, 2, 64, 16, dtype=dtype, cache=cache_dtype)
    bits = (lambda t: t.view(torch.uint8) if cache_dtype == torch.float8_e4m3fn else t)
    key, value = cache.key, bits(cache.value).clone()
    table = tables.tolist()
    for r, length in enumerate(lengths):
        t = length // 2
        spot = table[r][t // 16], t % 16, 1, 11
        value[spot] = 0
        bits(cache.value)[spot] = 0x7f if cache_dtype == torch.float8_e4m3fn else float("nan")
    out = mt.paged_attention(q, cache, tables, n)
    want, _, tol, _ = ref.attention(q, key, value.view(cache_dtype), tables.cpu(), lengths,
                                    64 ** -0.5, 0, cache.key_scale, cache.value_scale)
    assert bool(torch.isnan(out[:, 3:, 11]).all())
    out[:, 3:, 11] = 0.0
    want[:, 3:, 11] = 0.0
    assert outside(out, want, tol) <= 0
