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
