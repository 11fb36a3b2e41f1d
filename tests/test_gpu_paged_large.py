"""The paged cache's operators where counts and offsets pass 32 bits or come near them."""

from __future__ import annotations

import pytest
import torch

import metile_amd as mt

pytestmark = pytest.mark.gpu


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def test_append_of_rows_past_32_bits():
    # 4.3 GB of keys and as much of values; every token to another slot, some left out
    tokens, heads, dim, page = (1 << 21) + 3, 8, 128, 64
    pages = tokens // page + 2
    cache = mt.PagedCache(*(torch.zeros(pages, page, heads, dim, dtype=torch.bfloat16, device="cuda")
                            for _ in range(2)))
    key, value = (torch.empty(tokens, heads, dim, dtype=torch.bfloat16, device="cuda").normal_()
                  for _ in range(2))
    slots = torch.arange(tokens, device="cuda").flip(0) + 5
    slots[7::1000] = -1
    mt.paged_append(key, value, cache, slots)
    left_out = slots < 0
    for rows, held in ((key, cache.key), (value, cache.value)):
        rows = rows.masked_fill(left_out[:, None, None], 0).flip(0)
        flat = held.view(-1, heads, dim)
        assert torch.equal(flat[5:5 + tokens], rows)
        assert not bool(flat[:5].any()) and not bool(flat[5 + tokens:].any())


def test_tables_of_many_tokens():
    # 5 requests, 40 million tokens: every workgroup takes some 160000 of them
    cached, new, page = [0, 7, 1000003, 16, 5], [20000001, 0, 3, 13000000, 7654321], 16
    width = -(-33000000 // page)
    have = [-(-n // page) for n in cached]
    need = [-(-(a + b) // page) - h for a, b, h in zip(cached, new, have)]
    table = torch.full((5, width), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(sum(need) + sum(have), device="cuda", dtype=torch.int32)
    at = sum(need)
    for r, n in enumerate(have):
        table[r, :n] = free[at:at + n]
        at += n
    want = table.clone()
    at = 0
    for r, (h, n) in enumerate(zip(have, need)):
        want[r, h:h + n] = free[at:at + n]
        at += n
    tokens = sum(new) + 9
    step = mt.paged_tables(i32(cached), i32(new), table, free[:sum(need)], page_size=page, tokens=tokens)
    assert torch.equal(table, want) and step.taken.tolist() == [sum(need)]
    at = 0
    for r, (a, n) in enumerate(zip(cached, new)):
        position = torch.arange(a, a + n, device="cuda")
        part = slice(at, at + n)
        assert torch.equal(step.positions[part], position.int())
        assert bool((step.requests[part] == r).all())
        slots = want[r, position // page].long() * page + position % page
        assert torch.equal(step.slots[part], slots)
        at += n
    assert step.starts.tolist() == [0, 20000001, 20000001, 20000004, 33000004, 40654325]
    assert bool((step.slots[at:] == -1).all()) and bool((step.requests[at:] == -1).all())


@pytest.mark.parametrize("window", [None, (1 << 30) + 77])
def test_attention_over_nearly_2_31_tokens(window):
    # one page of 2^20 tokens, 2047 times in the table: softmax over all is that over the page, and over
    # 2^30 + 77 tokens nearly so (77 of 2^30 have a weight 1/1024 larger)
    page, width, heads, dim = 1 << 20, 2047, 2, 64
    g = torch.Generator("cuda").manual_seed(4)
    cache = mt.PagedCache.allocate(1, page, 1, dim)
    cache.key.normal_(generator=g)
    cache.value.normal_(0.5, 1.0, generator=g)
    q = torch.randn(1, heads, dim, generator=g, device="cuda").bfloat16()
    table = torch.zeros(1, width, dtype=torch.int32, device="cuda")
    out, lse = mt.paged_attention(q, cache, table, i32([page * width]), window=window,
                                  return_lse=True)
    # (sums over the long axis, products of two operands in ordinary order)
    scores = torch.stack([(cache.key[0, :, 0].double() * q[0, h].double()).sum(-1)
                          for h in range(heads)]) * dim ** -0.5
    weights = torch.softmax(scores, -1)
    value = cache.value[0, :, 0].double()
    want = torch.stack([(weights[h, :, None] * value).sum(0) for h in range(heads)])
    seen = width if window is None else window / page
    want_lse = torch.logsumexp(scores, -1) + torch.tensor(float(seen)).log().double().cuda()
    # a wave adds up some 22000 units one after the other in fp32: 22000 * 2^-24 of the sum at most,
    # in the sum of products and in that of probabilities, of values up to 6
    drift = 22000 * 2.0 ** -24
    tol = 2.0 ** -8 * want.abs() + 6 * 2 * drift + 2.0 ** -20
    assert bool(((out[0].double() - want).abs() <= tol).all())
    assert bool(((lse[0].double() - want_lse).abs() <= drift + 2.0 ** -18).all())
