"""Plain 64-bit restatements of the decode-step operators, on the CPU, for their tests."""

from __future__ import annotations

import numpy as np
import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def tables(cached, new, table, free, page, tokens, free_start=0):
    """``paged_tables`` token by token: (table, slots, positions, requests, starts, lengths, taken)."""
    table = [list(map(int, row)) for row in table]
    width = len(table[0]) if table else 0
    cached, new = ([max(0, int(n)) for n in v] for v in (cached, new))
    slots, positions, owners, starts = [], [], [], [0]
    taken = 0
    for r, (had, n) in enumerate(zip(cached, new)):
        pages = -(-min(had, width * page) // page)
        for p in range(had, had + n):
            column, place = divmod(p, page)
            slot = -1
            if column < width:
                if column >= pages:  # this token opens a page
                    at = free_start + taken
                    number = int(free[at]) if 0 <= at < len(free) else -1
                    taken += 1
                    pages += 1
                    if len(slots) < tokens:
                        table[r][column] = number
                else:
                    number = table[r][column]
                if number >= 0:
                    slot = number * page + place
            slots.append(slot)
            positions.append(p)
            owners.append(r)
        starts.append(starts[-1] + n)
    pad = max(0, tokens - len(slots))
    cut = slice(0, tokens)
    return (table, slots[cut] + [-1] * pad, positions[cut] + [0] * pad, owners[cut] + [-1] * pad,
            starts, [a + b for a, b in zip(cached, new)], [taken])


def fp8_values(x):
    """e4m3 rounding (nearest even, limited to +-448) in 64 bits, from the format's definition."""
    x = np.asarray(x, np.float64)
    exponent = np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -6)))
    step = np.exp2(exponent - 3)
    return np.clip(np.rint(x / step) * step, -448, 448)


def attention(query, key, value, tables, lengths, scale, window=0, key_scale=1.0, value_scale=1.0):
    """(out, lse, tolerance of out, tolerance of lse) in 64 bits. ``key`` and ``value`` are the whole
    caches as [pages, page, heads, dim]."""
    q = query.double().cpu()
    requests, heads, dim = q.shape
    pages, page, kv_heads, _ = key.shape
    group = heads // kv_heads
    unit = UNIT[query.dtype]
    out = torch.zeros(requests, heads, dim, dtype=torch.float64)
    lse = torch.full((requests, heads), -float("inf"), dtype=torch.float64)
    out_tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
    for r in range(requests):
        length = min(max(0, int(lengths[r])), tables.shape[1] * page)
        first = max(0, length - window) if window else 0
        at = [(int(tables[r, t // page]), t % page) for t in range(first, length)]
        at = [(p, s) for p, s in at if 0 <= p < pages]
        if not at:
            continue
        p = torch.tensor([a[0] for a in at])
        s = torch.tensor([a[1] for a in at])
        k = rows(key, p, s) * key_scale
        v = rows(value, p, s) * value_scale
        for h in range(heads):
            kh, vh = k[:, h // group], v[:, h // group]
            logits = (kh * q[r, h]).sum(-1) * scale
            weights = torch.exp(logits - logits.max())
            weights = weights / weights.sum()
            out[r, h] = (weights[:, None] * vh).sum(0)
            lse[r, h] = torch.logsumexp(logits, 0)
            # fp32 sums of `dim` products, times the scale: a few units of 2^-24 of their
            # magnitudes' sum; relative in the probabilities, twice (above and below the line), and
            # 2^-16 for their two 16-bit parts. The result is rounded once.
            size = float(((kh * q[r, h]).abs().sum(-1) * abs(scale)).max())
            error = 16 * 2.0 ** -24 * (1 + size)
            lse_tol[r, h] = error + 2.0 ** -22 * abs(float(lse[r, h]))
            out_tol[r, h] = (unit * out[r, h].abs() * (1 + 2.0 ** -7)
                             + (2 * error + 2.0 ** -16) * vh.abs().max() + 2.0 ** -25)
    return out, lse, out_tol, lse_tol


def rows(cache, pages, slots):
    """Rows of a cache in 64 bits on the CPU (8-bit floats are indexed as bytes)."""
    if cache.dtype == torch.float8_e4m3fn:
        picked = cache.view(torch.uint8)[pages.to(cache.device), slots.to(cache.device)]
        return picked.view(torch.float8_e4m3fn).float().double().cpu()
    return cache[pages.to(cache.device), slots.to(cache.device)].double().cpu()


def norm(x, weight, bias, eps, kind):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double().cpu()
    return y if bias is None else y + bias.double().cpu()


def residual_norm(residual, block, *, weight, bias=None, post_weight=None, post_bias=None, gate=None,
                  residual_scale=1.0, eps=1e-6, kind="rms"):
    r = residual.double().cpu() * residual_scale
    if block is not None:
        b = block.double().cpu()
        if post_weight is not None:
            b = norm(b, post_weight, post_bias, eps, kind)
        r = r + (b if gate is None else b * gate.double().cpu())
    return r, norm(r, weight, bias, eps, kind)
