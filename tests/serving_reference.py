"""Plain 64-bit restatements of the serving operators for their tests: attention of chunks, forks, freeing
and compaction of pages, log probabilities."""

from __future__ import annotations

import math

import torch

from tests.paged_reference import UNIT, rows


def chunk_attention(query, key, value, tables, lengths, starts, scale, window=0, key_scale=1.0,
                    value_scale=1.0):
    """(out, lse, tolerance of out, tolerance of lse). ``key`` and ``value`` are the whole caches as
    [pages, page, heads, dim]."""
    q = query.double().cpu()
    tokens, heads, dim = q.shape
    pages, page, kv_heads, _ = key.shape
    group = heads // kv_heads
    unit = UNIT[query.dtype]
    out = torch.zeros(tokens, heads, dim, dtype=torch.float64)
    lse = torch.full((tokens, heads), -math.inf, dtype=torch.float64)
    out_tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
    limit = tables.shape[1] * page
    for r, length in enumerate(int(n) for n in lengths):
        begin, end = (min(max(int(s), 0), tokens) for s in starts[r:r + 2])
        new = max(0, end - begin)
        length = max(0, length)
        keys = min(length, limit)
        if not new or not keys:
            continue
        at = torch.arange(keys)
        number = torch.as_tensor(tables)[r].cpu().long()[at // page]
        known = (number >= 0) & (number < pages)
        k = rows(key, number.clamp(0, pages - 1), at % page) * key_scale
        v = rows(value, number.clamp(0, pages - 1), at % page) * value_scale
        place = length - new + torch.arange(new)[:, None]
        seen = known & (at <= place)
        if window:
            seen &= at > place - window
        for h in range(heads):
            kh, vh = k[:, h // group], v[:, h // group]
            logits = (q[begin:end, h] @ kh.T) * scale
            logits = torch.where(seen, logits, -math.inf)
            top = logits.amax(-1, keepdim=True)
            live = top[:, 0] > -math.inf
            weights = torch.where(seen, torch.exp(logits - top.clamp(min=-1e300)), 0.0)
            weights = weights / weights.sum(-1, keepdim=True).clamp(min=1e-300)
            hidden = ~seen.any(0)
            vh = torch.where(hidden[:, None], 0.0, vh)  # what no one sees does not matter
            out[begin:end, h] = product(weights, seen, vh)
            lse[begin:end, h] = torch.where(live, torch.logsumexp(logits, -1), -math.inf)
            # Scores are fp32 sums of `dim` products, times the scale: a few units of 2^-24 of their
            # magnitudes' sum; relative in the probabilities, twice (above and below the line). Each
            # probability is rounded to 16 bits as it meets its value (`unit` of it; in f16 they are
            # scaled by 2^11 to 2^15 first, so that those below its normal numbers are off by 2^-25 of
            # its 2^11: 2^-36), and the result once.
            size = float((q[begin:end, h].abs() @ torch.where(hidden[:, None], 0.0, kh).abs().T).max()
                         * abs(scale))
            error = 16 * 2.0 ** -24 * (1 + size)
            lse_tol[begin:end, h] = error + 2.0 ** -22 * lse[begin:end, h].abs()
            fine = torch.where(torch.isfinite(vh), vh, 0.0).abs()
            spread = weights @ fine
            out_tol[begin:end, h] = (unit * out[begin:end, h].abs() * (1 + 2.0 ** -7)
                                     + unit * spread * (1 + 2.0 ** -7)
                                     + (2 * error + keys * 2.0 ** -36) * fine.max() + 2.0 ** -25)
    return out, lse, out_tol, lse_tol


def product(weights, seen, v):
    """weights @ v where values that are not finite count for the rows that see them alone."""
    odd = ~torch.isfinite(v).all(-1)
    if not bool(odd.any()):
        return weights @ v
    out = weights @ torch.where(torch.isfinite(v), v, 0.0)
    for j in torch.nonzero(odd)[:, 0].tolist():
        extra = torch.where(torch.isfinite(v[j]), 0.0, v[j])
        out += torch.where(seen[:, j, None], extra, 0.0)
    return out


def columns(tokens, page, width):
    return min(-(-max(0, tokens) // page), width)


def fork(tables, lengths, sources, targets, free, page, start=0, tokens=None):
    """(tables, lengths, copies' sources, targets, taken)."""
    tables, lengths = [list(row) for row in tables], list(lengths)
    width, taken, copies = len(tables[0]), 0, []
    for i, (s, t) in enumerate(zip(sources, targets)):
        copies.append((-1, -1))
        if not (0 <= s < len(tables) and 0 <= t < len(tables)):
            continue
        n = min(max(0, lengths[s]), width * page)
        if tokens is not None:
            n = min(n, max(0, tokens[i]))
        full = n // page
        tables[t][:full] = tables[s][:full]
        if n % page:
            at = start + taken
            fresh = free[at] if 0 <= at < len(free) else -1
            taken += 1
            if fresh >= 0:
                copies[-1] = (tables[s][full], fresh)
            tables[t][full] = fresh
        lengths[t] = n
    return tables, lengths, [c[0] for c in copies], [c[1] for c in copies], [taken]


def in_use(tables, lengths, page, pages):
    width = len(tables[0]) if tables else 0
    return {p for row, n in zip(tables, lengths) for p in row[:columns(n, page, width)]
            if 0 <= p < pages}


def free(tables, lengths, kept, list_, page, pages, start):
    """(free list, freed)."""
    kept = [min(k, n) for k, n in zip(kept, lengths)]
    gone = sorted(in_use(tables, lengths, page, pages) - in_use(tables, kept, page, pages))
    out = list(list_)
    for i, p in enumerate(gone):
        at = start - len(gone) + i
        if 0 <= at < len(out):
            out[at] = p
    return out, [len(gone)]


def compact(tables, lengths, list_, page, pages, start):
    """(tables, free list, sources, targets, moves)."""
    used = in_use(tables, lengths, page, pages)
    begin = max(0, start)
    open_ = {p for p in list_[begin:] if 0 <= p < pages} - used
    ordered = sorted(used | open_)
    low = set(ordered[:len(used)])
    sources, targets = sorted(used - low, reverse=True), sorted(open_ & low)
    number = dict(zip(sources, targets))
    width = len(tables[0]) if tables else 0
    out = [[number.get(p, p) if c < columns(n, page, width) else p for c, p in enumerate(row)]
           for row, n in zip(tables, lengths)]
    rest = [p for p in ordered if p not in low]
    new = list(list_[:begin]) + (rest + [-1] * len(list_))[:max(0, len(list_) - begin)]
    most = min(pages // 2, len(tables) * width)
    pad = [-1] * (most - len(sources))
    return out, new, sources + pad, targets + pad, [len(sources)]


def logprobs(logits, tokens, top, temperature=1.0):
    """(logprobs, entropies, ranks, top_logprobs, top_tokens) of finite or -inf logits in 64 bits."""
    x = logits.double().cpu()
    logs = torch.log_softmax(x / temperature, -1)
    p = logs.exp()
    entropy = -torch.where(p > 0, p * logs, 0.0).sum(-1)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    given = rank = None
    if tokens is not None:
        t = tokens.cpu()[:, None]
        given = logs.gather(1, t)[:, 0]
        rank = (order == t).int().argmax(-1).int()
    best = order[:, :top]
    return given, entropy, rank, logs.gather(1, best), best
