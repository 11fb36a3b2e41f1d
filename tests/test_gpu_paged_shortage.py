"""How a caller of the block tables sees that pages ran out or a table is too narrow."""

from __future__ import annotations

import pytest
import torch

import metile_amd as mt

pytestmark = pytest.mark.gpu


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def test_an_exhausted_list_shows_in_taken():
    table = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    free = i32([7, 5, 3])
    step = mt.paged_tables(i32([0, 0]), i32([9, 8]), table, free, page_size=4, tokens=17,
                           free_start=i32([1]))
    assert step.taken.tolist() == [5] and step.taken.item() > free.numel() - 1
    assert table.tolist() == [[5, 3, -1, -1], [-1, -1, -1, -1]]
    assert step.slots.tolist() == [20, 21, 22, 23, 12, 13, 14, 15] + [-1] * 9
    assert step.lengths.tolist() == [9, 8] and max(step.lengths.tolist()) <= 4 * 4


def test_a_narrow_table_shows_in_lengths_alone():
    table = i32([[6, -1], [2, 4]])
    free = i32(list(range(10, 20)))
    step = mt.paged_tables(i32([4, 7]), i32([6, 1]), table, free, page_size=4, tokens=7)
    assert step.lengths.tolist() == [10, 8]  # of 2 * 4 that the table holds
    assert step.taken.tolist() == [1] and table.tolist() == [[6, 10], [2, 4]]
    assert step.slots.tolist() == [40, 41, 42, 43, -1, -1, 19]
    # the tokens beyond are not written, and attention goes as far as the table does
    cache = mt.PagedCache.allocate(20, 4, 1, 16)
    cache.key.zero_(), cache.value.zero_()
    cache.value[6] = 1.0
    row = torch.ones(7, 1, 16, dtype=torch.bfloat16, device="cuda")
    mt.paged_append(torch.zeros_like(row), 3 * row, cache, step.slots)
    out = mt.paged_attention(row[:2], cache, table, step.lengths)
    assert torch.equal(out[0], torch.full_like(out[0], 2.0))  # 4 tokens of 1, 4 of 3
