"""Residual norms of more rows than one launch's threads can be counted in 32 bits."""

from __future__ import annotations

import pytest
import torch

import metile_amd as mt

pytestmark = pytest.mark.gpu

PART = 1 << 24


def row_values(first, count, width, dtype):
    """Rows that differ from one another, made from their numbers."""
    n = torch.arange(first, first + count, device="cuda", dtype=torch.int64)
    a = ((n * 2654435761) % 1021).float() / 512 - 1
    return (a[:, None] + torch.arange(width, device="cuda") * 0.125).to(dtype)


@pytest.mark.parametrize("rows,width", [
    ((1 << 28) + 37, 8),    # sixteen rows a workgroup of 256 threads: 2^32 threads and some
    ((1 << 31) - 1, 1),     # a row a thread, the most rows there are
    ((1 << 24) + 5, 1026),  # a row a workgroup of 256 threads
])
def test_every_row_is_normed(rows, width):
    dtype = torch.bfloat16
    x = torch.empty(rows, width, dtype=dtype, device="cuda")
    for at in range(0, rows, PART // 16):
        count = min(PART // 16, rows - at)
        x[at:at + count] = row_values(at, count, width, dtype)
    w = row_values(5, 1, width, dtype)[0]
    _, normed = mt.residual_norm(x, weight=w)
    part = min(rows, PART)
    for at in [*range(0, rows - part, part), rows - part]:
        _, want = mt.residual_norm(x[at:at + part], weight=w)
        assert torch.equal(normed[at:at + part], want), at


def test_gates_of_late_rows():
    # a gate's row for every 2^20 + 1 rows of the batch, which no number of launches divides
    dtype, per, width = torch.bfloat16, (1 << 20) + 1, 8
    rows = per * 260
    x = torch.ones(rows, width, dtype=dtype, device="cuda")
    block = row_values(0, per, width, dtype).repeat(260, 1)
    gate = row_values(0, 260, width, dtype)
    w = torch.ones(width, dtype=dtype, device="cuda")
    r, normed = mt.residual_norm(x.view(260, per, width), block.view(260, per, width), weight=w,
                                 gate=gate[:, None], residual_scale=0.5)
    for i in (0, 1, 127, 128, 200, 255, 256, 257, 258, 259):
        want = mt.residual_norm(x[:per], block[:per], weight=w, gate=gate[i], residual_scale=0.5)
        assert torch.equal(r[i], want[0]) and torch.equal(normed[i], want[1]), i
