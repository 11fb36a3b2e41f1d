"""Ranks in rows that hold NaN: counted over the values that compare, whatever kind of NaN it is."""

from __future__ import annotations

import math

import pytest
import torch

import metile_amd as mt

pytestmark = pytest.mark.gpu
# quiet and signalling, of both signs
NANS = {torch.bfloat16: (torch.int16, (0x7fc0, 0x7f81, -0x40, -0x7f)),
        torch.float16: (torch.int16, (0x7e00, 0x7c01, -0x200, -0x3ff)),
        torch.float32: (torch.int32, (0x7fc00000, 0x7f800001, -0x400000, -1))}


def rank(row, token):
    given, at = row[token], torch.arange(row.numel())
    return int(((row > given) | ((row == given) & (at < token))).sum())


@pytest.mark.parametrize("dtype", NANS)
@pytest.mark.parametrize("rows,vocab", [(2, 300), (2, 40000), (2, 300001), (300, 9001)])
def test_ranks_beside_nan(dtype, rows, vocab):
    """Tokens that are not allowed and others, with NaN before them, behind them, and in their own eight
    values: only what is larger, or as large and before it, counts."""
    kind, patterns = NANS[dtype]
    g = torch.Generator().manual_seed(vocab)
    x = (torch.randn(rows, vocab, generator=g) * 3).to(dtype)
    x[:, 5::7] = -math.inf
    x[:, 3::11] = 1.5
    odd = torch.randperm(vocab, generator=g)[:vocab // 9]
    bits = x.view(kind)
    for i, p in enumerate(patterns):
        bits[:, odd[i::4]] = p
    alive = (~torch.isnan(x[0])).nonzero()[:, 0]
    inf, same = ((x[0] == v).nonzero()[:, 0] for v in (-math.inf, 1.5))
    tokens = [int(t) for t in (inf[0], inf[-1], inf[len(inf) // 2], same[0], same[-1], alive[0], alive[-1],
                               x[0].float().nan_to_num(-1e4, neginf=-1e4).argmax())]
    tokens += alive[torch.randint(len(alive), (8,), generator=g)].tolist()
    on_gpu = x.cuda()
    for token in tokens:
        got = mt.token_logprobs(on_gpu, torch.full((rows,), token, device="cuda"))
        assert bool(torch.isnan(got.logprobs).all())
        for r in (0, rows - 1):
            assert int(got.ranks[r]) == rank(x[r].float(), token), (token, float(x[0, token]))


@pytest.mark.parametrize("dtype", NANS)
def test_a_signalling_nan_hides_no_larger_values(dtype):
    """One NaN beside the only larger value of a wave, in each place of a thread's values."""
    kind, patterns = NANS[dtype]
    for place in range(8):
        for other in range(8):
            for p in patterns:
                x = torch.full((1, 9000), -1.0, dtype=dtype)
                x[0, 17] = 1.0
                if other != place:
                    x[0, 4896 + other] = 2.0
                x.view(kind)[0, 4896 + place] = p
                got = mt.token_logprobs(x.cuda(), torch.tensor([17], device="cuda"))
                assert got.ranks.tolist() == [int(other != place)], (place, other, p)
