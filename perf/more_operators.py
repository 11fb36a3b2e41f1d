"""The measured work of the serving operators around a decode step: prompts, pages and answers.

Each case is one pass through one operator, as a serving loop calls it:

* ``chunk``: ``paged_chunk_attention``. Several new tokens of each request (a prompt, a part of one, a
  draft to verify) over the pages of a cache, each seeing the tokens up to its own.
* ``logprobs``: ``token_logprobs``. Log probabilities and ranks of given tokens, the entropies of their
  distributions and the most likely alternatives, from a head's logits.
* ``fork``: ``paged_fork`` and ``paged_copy``. Requests that go on from another's tokens: full pages are
  shared, a page that has been begun is copied in every layer's cache.
* ``free``: ``paged_free``. Pages of finished and of shortened requests back to the free list.
* ``compact``: ``paged_compact`` and ``paged_copy``. Pages in use moved to the lowest numbers of the pool.

Shapes are the benchmark's and tests' head layouts and generic ones. With ``own`` false the operators are
computed in plain torch operations; with it true through the package's kernels.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32,
          "fp8": torch.float8_e4m3fn}
HEADS = ((12, 2, 128), (14, 2, 64), (28, 4, 128), (32, 8, 128), (40, 8, 128), (32, 32, 128),
         (16, 16, 80), (24, 3, 96), (64, 8, 64), (16, 1, 256), (20, 5, 192), (48, 1, 128))
VOCABS = (32000, 50001, 65536, 100352, 152064)
MOST_SCORES = 1 << 31          # of a chunk's padded batch
MOST_LOGITS = 2048 * 152064
MOST_CACHE = 3 << 26           # keys of all layers of a pool


def listed():
    return [
        # a draft of a few tokens of one request, verified at once, in a small model
        dict(name="chunk-draft", kind="chunk", requests=1, low=6, high=6, past=2043, hq=12, hkv=2,
             dim=128, page=16, dtype="bf16", cache="bf16", window=0, lse=False, heads_outer=True,
             padding=0),
        # a step of many requests: parts of prompts behind contexts of every length, an 8-bit cache of
        # narrow heads with a sliding window, odd pages, padding behind the last request
        dict(name="chunk-ragged", kind="chunk", requests=24, low=1, high=256, past=4000, hq=64, hkv=8,
             dim=64, page=24, dtype="f16", cache="fp8", window=1500, lse=True, heads_outer=True,
             padding=37),
        # a long prompt at once
        dict(name="chunk-prompt-8k", kind="chunk", requests=1, low=8192, high=8192, past=0, hq=32,
             hkv=8, dim=128, page=16, dtype="bf16", cache="bf16", window=0, lse=False,
             heads_outer=True, padding=0),
        # the last part of a very long prompt
        dict(name="chunk-context-128k", kind="chunk", requests=1, low=509, high=509, past=130500,
             hq=32, hkv=8, dim=128, page=64, dtype="bf16", cache="bf16", window=0, lse=False,
             heads_outer=False, padding=0),
        # one token's choice with its log probability and alternatives
        dict(name="logprobs-1row", kind="logprobs", rows=1, vocab=32000, dtype="bf16", top=5,
             temperature=1.0, banned=0.0, pad=0),
        # a prompt's tokens scored over a large vocabulary
        dict(name="logprobs-prompt", kind="logprobs", rows=2048, vocab=152064, dtype="bf16", top=20,
             temperature=1.0, banned=0.0, pad=0),
        # one request of a few layers answered twice
        dict(name="fork-1", kind="fork", requests=8, forks=1, low=700, high=700, layers=4, page=16,
             hkv=2, dim=128, cache="bf16", heads_outer=True),
        # many answers to each prompt of a batch
        dict(name="fork-256", kind="fork", requests=512, forks=256, low=1, high=900, layers=8, page=16,
             hkv=8, dim=128, cache="bf16", heads_outer=True),
        # a decode step after which a few requests end and drafts are taken back
        dict(name="free-64", kind="free", requests=64, low=1, high=4096, page=16, shared=3),
        # a large pool: thousands of requests, most of their contexts shared
        dict(name="free-4096", kind="free", requests=4096, low=1, high=8192, page=16, shared=2),
        # a small pool's pages together
        dict(name="compact-64", kind="compact", requests=64, low=1, high=700, spare=0.3, layers=4,
             page=16, hkv=2, dim=128, cache="bf16", heads_outer=True, shared=3),
        # a large one's, half empty, 8-bit
        dict(name="compact-2048", kind="compact", requests=2048, low=1, high=1500, spare=0.5, layers=2,
             page=32, hkv=2, dim=64, cache="fp8", heads_outer=False, shared=4),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    kind = rng.choice(("chunk", "chunk", "chunk", "logprobs", "logprobs", "fork", "free", "compact"))
    page = rng.choice((1, 8, 16, 16, 20, 32, 48, 64, 128, 256))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    cache = rng.choice((dtype, dtype, "fp8"))
    if kind == "logprobs":
        vocab = rng.choice(VOCABS) if rng.random() < 0.6 else _log(rng, 100, 262144)
        return dict(kind=kind, rows=_log(rng, 1, MOST_LOGITS // vocab // 2), vocab=vocab,
                    dtype=rng.choice(("bf16", "f16", "f32")), top=rng.choice((0, 1, 5, 20, 32)),
                    temperature=rng.choice((1.0, 1.0, round(rng.uniform(0.3, 1.5), 2))),
                    banned=rng.choice((0.0, 0.0, 0.5)), pad=rng.choice((0, 0, 1, 64)))
    hq, hkv, dim = rng.choice(HEADS)
    if kind == "chunk":
        while True:
            high, past = _log(rng, 1, 8192), _log(rng, 1, 131072)
            requests = _log(rng, 1, 256)
            if requests * high * (past + high) * hq * max(1, dim / 128) <= MOST_SCORES and \
                    requests * (past + high) * hkv * dim <= MOST_CACHE:
                break
        return dict(kind=kind, requests=requests, low=high if rng.random() < 0.3 else _log(rng, 1, high),
                    high=high, past=past if rng.random() < 0.8 else 0, hq=hq, hkv=hkv, dim=dim,
                    page=page, dtype=dtype, cache=cache,
                    window=_log(rng, 1, 8192) if rng.random() < 0.25 else 0, lse=rng.random() < 0.3,
                    heads_outer=rng.random() < 0.5, padding=rng.choice((0, 0, 5, 100)))
    if kind == "free":
        return dict(kind=kind, requests=_log(rng, 1, 4096), low=1, high=_log(rng, 1, 8192),
                    page=max(page, 8), shared=rng.randint(2, 5))
    most = MOST_CACHE // (hkv * dim)
    while True:
        requests, high, layers = _log(rng, 2, 2048), _log(rng, 1, 4096), rng.randint(1, 12)
        if requests * (high + 2 * page) * layers <= most // 2:
            break
    case = dict(kind=kind, requests=requests, low=1, high=high, layers=layers, page=page, hkv=hkv,
                dim=dim, cache=cache, heads_outer=rng.random() < 0.5)
    if kind == "fork":
        return dict(case, forks=rng.randint(1, requests // 2))
    return dict(case, spare=round(rng.uniform(0.05, 0.8), 2), shared=rng.randint(2, 5))


# ---- inputs --------------------------------------------------------------------------------------


def _spread(n, low, high):
    """``n`` whole numbers spread evenly over the logarithm of ``low`` .. ``high``."""
    return [int(round(low * (high / low) ** ((i + 0.5) / n))) for i in range(n)]


def _new(case):
    return _spread(case["requests"], case["low"], case["high"])


def _lengths(case):
    """Tokens of each request in the cache; of those that are forked, where some are."""
    return _spread(case["requests"] - case.get("forks", 0), case["low"], case["high"])


def _past(case):
    """Tokens before each request's chunk, in the order of its new ones; every fifth starts here."""
    if not case["past"]:
        return [0] * case["requests"]
    spread = _spread(case["requests"], 1, case["past"]) if case["requests"] > 1 else [case["past"]]
    spread = spread[1::2] + spread[::2]
    return [0 if i % 5 == 4 else n for i, n in enumerate(spread)]


def _pool(g, pages, page, hkv, dim, cache, heads_outer, device):
    """One cache tensor [pages, page, heads, dim], stored with the heads outside or inside the slots.
    Made in place, a part at a time: the largest are a gigabyte."""
    shape = (pages, hkv, page, dim) if heads_outer else (pages, page, hkv, dim)
    pool = torch.empty(shape, dtype=DTYPES[cache], device=device)
    for part in pool.view(-1).split(1 << 27):
        part.copy_(torch.randn(part.numel(), generator=g, device=device, dtype=torch.float32))
    return pool.transpose(1, 2) if heads_outer else pool


def _pools(g, case, pages, device):
    """Keys and values of every layer."""
    return [tuple(_pool(g, pages, case["page"], case["hkv"], case["dim"], case["cache"],
                        case["heads_outer"], device) for _ in range(2))
            for _ in range(case["layers"])]


def _tables(g, lengths, width, page, spare, shared, device):
    """Block tables over a pool of pages in random order, columns behind each length -1; every
    ``shared``-th request begins with the first half of the pages of the one before it (0: none
    does). Gives the pool's size, its free list ([pages], the unused ones from entry `start` on) and
    `start`."""
    lengths = torch.tensor(lengths, device=device)
    counts = (lengths + page - 1) // page
    column = torch.arange(width, device=device)
    taken = column < counts[:, None]
    total = int(counts.sum())
    pages = total + max(4, int(total * spare))
    order = torch.randperm(pages, generator=g, device=device, dtype=torch.int32)
    tables = torch.full((len(lengths), width), -1, dtype=torch.int32, device=device)
    tables[taken] = order[:total]
    if shared and len(lengths) > 1:
        heirs = torch.arange(1, len(lengths), shared, device=device)
        half = torch.minimum(counts[heirs], counts[heirs - 1]) // 2
        tables[heirs] = torch.where(column < half[:, None], tables[heirs - 1], tables[heirs])
    used = torch.zeros(pages, dtype=torch.bool, device=device)
    used[tables[taken].long()] = True
    unused = order[~used[order.long()]]
    free = torch.full((pages,), -1, dtype=torch.int32, device=device)
    free[pages - unused.numel():] = unused
    start = torch.tensor([pages - unused.numel()], dtype=torch.int32, device=device)
    return tables, pages, free, start


def _inputs(case, seed):
    device = "cuda"
    rng = random.Random(seed)
    g = torch.Generator(device).manual_seed(seed)
    kind = case["kind"]
    if kind == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        # a model's logits: the given token is likely in most rows, unlikely in some
        stored = torch.empty(rows, vocab + case["pad"], dtype=DTYPES[case["dtype"]], device=device)
        for part in stored.split(max(1, (1 << 27) // vocab)):
            part.copy_(torch.randn(part.shape, generator=g, device=device).mul_(2.5))
        logits = stored[:, :vocab]
        tokens = torch.randint(vocab, (rows,), generator=g, device=device)
        at = torch.arange(rows, device=device)
        if case["banned"]:  # tokens that a grammar does not allow
            ban = torch.rand(vocab, generator=g, device=device) < case["banned"]
            logits.masked_fill_(ban, -math.inf)
        raised = 14.0 * torch.rand(rows, generator=g, device=device)
        logits[at, tokens] = raised.to(logits.dtype)
        return dict(logits=logits, tokens=tokens)
    page = case["page"]
    # float caches hold values as they are; an 8-bit one holds them over a scale of its own
    scales = (1.0, 1.0) if case.get("cache") != "fp8" else (0.75, 1.25)
    if kind == "chunk":
        hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
        pairs = list(zip(_new(case), _past(case)))
        rng.shuffle(pairs)
        new = torch.tensor([n for n, _ in pairs], device=device)
        lengths = [n + m for n, m in pairs]
        width = -(-max(lengths) // page)
        tables, pages, _, _ = _tables(g, lengths, width, page, 0.0, 0, device)
        starts = torch.zeros(len(pairs) + 1, dtype=torch.int32, device=device)
        starts[1:] = new.cumsum(0)
        tokens = sum(n for n, _ in pairs) + case["padding"]
        fused = torch.randn(tokens, (hq + 2 * hkv) * dim, generator=g, device=device)
        query = fused.to(DTYPES[case["dtype"]])[:, :hq * dim].unflatten(1, (hq, dim))
        key, value = (_pool(g, pages, page, hkv, dim, case["cache"], case["heads_outer"], device)
                      for _ in range(2))
        return dict(query=query, tables=tables, starts=starts, scales=scales, key=key, value=value,
                    lengths=torch.tensor(lengths, dtype=torch.int32, device=device))
    lengths = _lengths(case)
    rng.shuffle(lengths)
    if kind == "fork":  # the batch's last rows are empty: forks go there
        forks, live = case["forks"], len(lengths)
        lengths += [0] * forks
        tables, pages, free, start = _tables(g, lengths, -(-case["high"] // page), page,
                                             forks / live, 0, device)
        sources = torch.randint(live, (forks,), generator=g, device=device, dtype=torch.int32)
        targets = live + torch.randperm(forks, generator=g, device=device, dtype=torch.int32)
        return dict(tables=tables, free=free, start=start, sources=sources, targets=targets,
                    lengths=torch.tensor(lengths, dtype=torch.int32, device=device), scales=scales,
                    caches=_pools(g, case, pages, device))
    tables, pages, free, start = _tables(g, lengths, -(-case["high"] // page), page,
                                         case.get("spare", 0.2), case["shared"], device)
    state = dict(tables=tables, free=free, start=start, pages=pages, scales=scales,
                 lengths=torch.tensor(lengths, dtype=torch.int32, device=device))
    if kind == "free":  # every fourth request ends, every third takes a few tokens back
        kept = [0 if i % 4 == 1 else max(0, n - rng.randint(1, 9)) if i % 3 == 0 else n
                for i, n in enumerate(lengths)]
        return dict(state, kept=torch.tensor(kept, dtype=torch.int32, device=device))
    return dict(state, caches=_pools(g, case, pages, device))


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if own:  # a serving program's handles of its caches: the tensors and scales
        import metile_amd as mt

        sides = [(state["key"], state["value"])] if "key" in state else state.get("caches", [])
        state["handles"] = [mt.PagedCache(key, value, key_scale=state["scales"][0],
                                          value_scale=state["scales"][1]) for key, value in sides]
    return state


# ---- one pass ------------------------------------------------------------------------------------


def run(state):
    kind = state["case"]["kind"]
    return (_KERNELS if own else _PLAIN)[kind](state, state["case"])


def _run_chunk(s, case):
    import metile_amd as mt

    return mt.paged_chunk_attention(s["query"], s["handles"][0], s["tables"], s["lengths"],
                                    s["starts"], window=case["window"] or None,
                                    return_lse=case["lse"])


def _run_logprobs(s, case):
    import metile_amd as mt

    return list(mt.token_logprobs(s["logits"], s["tokens"], top=case["top"],
                                  temperature=case["temperature"]))


def _run_fork(s, case):
    import metile_amd as mt

    fork = mt.paged_fork(s["tables"], s["lengths"], s["sources"], s["targets"], s["free"],
                         page_size=case["page"], free_start=s["start"])
    mt.paged_copy(s["handles"], fork.sources, fork.targets)
    return [s["tables"], s["lengths"], *fork, s["caches"]]


def _run_free(s, case):
    import metile_amd as mt

    freed = mt.paged_free(s["tables"], s["lengths"], s["kept"], s["free"], page_size=case["page"],
                          pages=s["pages"], free_start=s["start"])
    return [s["free"], freed]


def _run_compact(s, case):
    import metile_amd as mt

    moved = mt.paged_compact(s["tables"], s["lengths"], s["free"], page_size=case["page"],
                             pages=s["pages"], free_start=s["start"])
    mt.paged_copy(s["handles"], moved.sources, moved.targets)
    return [*moved, s["caches"]]


_KERNELS = {"chunk": _run_chunk, "logprobs": _run_logprobs, "fork": _run_fork, "free": _run_free,
            "compact": _run_compact}


# ---- the operators in plain torch operations -----------------------------------------------------


def _bits(cache):
    """An 8-bit cache's bytes (torch indexes no 8-bit floats); others as they are."""
    return cache.view(torch.uint8) if cache.dtype == DTYPES["fp8"] else cache


def _pages(cache, tables):
    """[requests, heads, positions, dim] of each request's pages, in 32 bits."""
    rows = _bits(cache)[tables.clamp(min=0).long()].view(cache.dtype)
    r, w, p, h, d = rows.shape
    return rows.reshape(r, w * p, h, d).transpose(1, 2).float()


def _plain_chunk(s, case):
    query, tables, lengths, starts = s["query"], s["tables"], s["lengths"], s["starts"].long()
    tokens, hq, dim = query.shape
    requests, hkv, most = tables.shape[0], s["key"].shape[2], case["high"]
    new = starts.diff()
    i = torch.arange(most, device=query.device)
    inside = i < new[:, None]
    rows = (starts[:-1, None] + i).clamp(max=tokens - 1)  # [requests, most] of the packed batch
    q = query[rows].float().reshape(requests, most, hkv, hq // hkv, dim).permute(0, 2, 3, 1, 4)
    q = q.reshape(requests, hkv, -1, dim)
    scores = (q @ _pages(s["key"], tables).transpose(2, 3)).mul_(s["scales"][0] / math.sqrt(dim))
    t = torch.arange(scores.shape[-1], device=query.device)
    last = (lengths[:, None] - new[:, None] + i)[..., None]  # the newest token that each one sees
    seen = t <= last
    if case["window"]:
        seen &= t > last - case["window"]
    scores = scores.unflatten(2, (hq // hkv, most))
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    out = weights.flatten(2, 3) @ _pages(s["value"], tables)
    out = out.unflatten(2, (hq // hkv, most)) * (s["scales"][1] / total)
    result = torch.zeros(query.shape, dtype=query.dtype, device=query.device)
    result[rows[inside]] = out.permute(0, 3, 1, 2, 4)[inside].reshape(-1, hq, dim).to(query.dtype)
    if not case["lse"]:
        return result
    lse = torch.full((tokens, hq), -math.inf, device=query.device)
    lse[rows[inside]] = (top + total.log()).permute(0, 3, 1, 2, 4)[inside].reshape(-1, hq)
    return result, lse


def _plain_logprobs(s, case):
    logits, tokens, k = s["logits"], s["tokens"], case["top"]
    x = logits.float() / case["temperature"]
    at = tokens[:, None]
    centred = x.sub_(x.amax(-1, keepdim=True))
    weights = centred.exp()
    total = weights.sum(-1, keepdim=True)
    given = centred.gather(1, at)
    # (a banned token has weight 0)
    mean = (weights.mul_(centred.clamp(min=-1e4))).sum(-1, keepdim=True) / total
    entropy = (total.log() - mean)[:, 0]
    raw = logits.gather(1, at)
    index = torch.arange(logits.shape[1], device=logits.device)
    rank = ((logits > raw) | ((logits == raw) & (index < at))).sum(-1, dtype=torch.int32)
    # values in order as whole numbers, then the lowest index first
    bits = (logits.float() + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -2147483648 - bits, bits) * (1 << 20) - index
    best = order.topk(k, dim=1).indices
    return [(given - total.log())[:, 0], entropy, rank, centred.gather(1, best) - total.log(), best]


def _copy_pages(caches, sources, targets):
    live = sources >= 0
    source, target = sources[live].long(), targets[live].long()
    for cache in (side for layer in caches for side in layer):
        _bits(cache)[target] = _bits(cache)[source]


def _plain_fork(s, case):
    tables, lengths, free, page = s["tables"], s["lengths"], s["free"], case["page"]
    source, target = s["sources"].long(), s["targets"].long()
    tokens = lengths[source]
    begun = tokens % page != 0
    last = (tokens // page).long().clamp(max=tables.shape[1] - 1)
    fresh = free[(s["start"] + begun.cumsum(0) - begun.long()).clamp(max=free.shape[0] - 1)]
    rows = tables[source]
    old = rows.gather(1, last[:, None])[:, 0]
    rows.scatter_(1, last[:, None], torch.where(begun, fresh, old)[:, None])
    column = torch.arange(tables.shape[1], device=tables.device)
    tables[target] = torch.where(column * page < tokens[:, None], rows, tables[target])
    lengths[target] = tokens
    sources, targets = torch.where(begun, old, -1), torch.where(begun, fresh, -1)
    _copy_pages(s["caches"], sources, targets)
    return [tables, lengths, sources, targets, begun.sum(0, keepdim=True).to(torch.int32),
            s["caches"]]


def _marked(pages, numbers):
    marks = torch.zeros(pages, dtype=torch.bool, device=numbers.device)
    marks[numbers.long()] = True
    return marks


def _plain_free(s, case):
    tables, page, free = s["tables"], case["page"], s["free"]
    first = torch.arange(tables.shape[1], device=tables.device) * page  # of each column
    used = first < s["lengths"][:, None]
    keeps = first < torch.minimum(s["kept"], s["lengths"])[:, None]
    freed = _marked(s["pages"], tables[used & ~keeps]) & ~_marked(s["pages"], tables[keeps])
    numbers = freed.nonzero()[:, 0].to(torch.int32)
    free[s["start"] - numbers.numel() + torch.arange(numbers.numel(), device=free.device)] = numbers
    return [free, freed.sum(0, keepdim=True).to(torch.int32)]


def _plain_compact(s, case):
    tables, page, pages, free = s["tables"], case["page"], s["pages"], s["free"]
    filled = torch.arange(tables.shape[1], device=tables.device) * page < s["lengths"][:, None]
    used = _marked(pages, tables[filled])
    listed_from = torch.arange(free.shape[0], device=free.device) >= s["start"]
    open_ = _marked(pages, free[listed_from]) & ~used
    low = (used | open_).cumsum(0) <= used.sum()
    sources, targets = (m.nonzero()[:, 0].to(torch.int32) for m in (used & ~low, open_ & low))
    sources = sources.flip(0)  # the highest page in use goes to the lowest free one
    number = torch.arange(pages, dtype=torch.int32, device=tables.device)
    number[sources.long()] = targets
    result = torch.where(filled, number[tables.clamp(min=0).long()], tables)
    left = free.clone()
    left[listed_from] = ((used | open_) & ~low).nonzero()[:, 0].to(torch.int32)
    size = min(pages // 2, tables.numel())
    padded = torch.full((2, size), -1, dtype=torch.int32, device=tables.device)
    padded[0, :sources.numel()], padded[1, :targets.numel()] = sources, targets
    _copy_pages(s["caches"], sources, targets)
    return [result, left, padded[0], padded[1], (used & ~low).sum(0, keepdim=True).to(torch.int32),
            s["caches"]]


_PLAIN = {"chunk": _plain_chunk, "logprobs": _plain_logprobs, "fork": _plain_fork,
          "free": _plain_free, "compact": _plain_compact}


# ---- what a pass cannot do without ---------------------------------------------------------------


def _seen(first, n, window):
    """Keys that ``n`` tokens see, the first at position ``first``: the sum over them, and how many
    different ones."""
    if not window:
        return n * first + n * (n + 1) // 2, first + n
    short = min(n, max(0, window - first))  # tokens that see everything before them
    total = short * first + short * (short + 1) // 2 + (n - short) * window
    return total, min(first + n, n + window - 1)


def work(case):
    kind = case["kind"]
    if kind == "logprobs":
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * size + 20 + 12 * case["top"]),
                "flops": 8 * case["rows"] * case["vocab"]}
    size = 1 if case.get("cache") == "fp8" else 2
    page = case["page"]
    if kind == "chunk":
        row = case["hkv"] * case["dim"]
        new = _new(case)
        seen = [_seen(m, n, case["window"]) for n, m in zip(new, _past(case))]
        heads = case["hq"] * case["dim"]
        tokens = sum(new) + case["padding"]
        return {"bytes": sum(n for _, n in seen) * row * 2 * size
                + sum(-(-n // page) for _, n in seen) * 4 + 8 * case["requests"]
                + sum(new) * 2 * heads + tokens * (2 * heads + (4 * case["hq"] if case["lse"] else 0)),
                "flops": 4 * sum(n for n, _ in seen) * heads}
    entries = sum(-(-n // page) for n in _lengths(case))
    both = 2 * page * case.get("hkv", 0) * case.get("dim", 0) * size * case.get("layers", 0)
    if kind == "fork":  # entries read and written, a begun page of most forks read and written
        share = case["forks"] / (case["requests"] - case["forks"])
        return {"bytes": int(8 * entries * share) + int(2 * both * case["forks"] * (1 - 1 / page)),
                "flops": 0}
    if kind == "free":
        return {"bytes": 4 * entries + 8 * case["requests"] + 4 * (entries // 4), "flops": 0}
    # pages whose numbers are not low enough: as many of those in use as the spare ones' share
    spare = case["spare"] / (1 + case["spare"])
    return {"bytes": 4 * entries + 4 * case["requests"] * -(-case["high"] // page)
            + int(2 * both * entries * spare), "flops": 0}


# ---- the definitions in 64 bits ------------------------------------------------------------------


def exact(case, seed):
    kind = case["kind"]
    if kind in ("free", "compact", "fork"):
        return None  # whole numbers, and values that are moved as they are
    s = _inputs(case, seed)
    if kind == "logprobs":
        rows = []
        for part, tokens in zip(s["logits"].split(64), s["tokens"].split(64)):
            logs = torch.log_softmax(part.double() / case["temperature"], -1)
            p = logs.exp()
            h = -torch.where(p > 0, p * logs, 0.0).sum(-1)
            top = logs.sort(-1, descending=True).values[:, :case["top"]]
            rows.append((logs[torch.arange(len(tokens)), tokens], h, top))
        lp, h, top = (torch.cat(side) for side in zip(*rows))
        return [lp, h, None, top, None]
    tokens, hq, dim = s["query"].shape
    out = torch.zeros(tokens, hq, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((tokens, hq), -math.inf, dtype=torch.float64, device="cuda")
    group, starts = hq // case["hkv"], s["starts"].tolist()
    for r, length in enumerate(s["lengths"].tolist()):
        new = starts[r + 1] - starts[r]
        at = torch.arange(length, device="cuda")
        pages, offsets = s["tables"][r].long()[at // case["page"]], at % case["page"]
        for h in range(case["hkv"]):
            k, v = (_bits(s[name])[pages, offsets, h].view(s[name].dtype).double()
                    for name in ("key", "value"))
            for i in range(0, new, 1024):
                rows = slice(starts[r] + i, min(starts[r] + i + 1024, starts[r + 1]))
                place = length - new + i + torch.arange(rows.stop - rows.start, device="cuda")[:, None]
                hidden = at > place
                if case["window"]:
                    hidden |= at <= place - case["window"]
                for head in range(h * group, (h + 1) * group):
                    logits = s["query"][rows, head].double() @ k.T.contiguous()
                    logits = (logits * s["scales"][0] * dim ** -0.5).masked_fill_(hidden, -math.inf)
                    lse[rows, head] = torch.logsumexp(logits, -1)
                    out[rows, head] = torch.softmax(logits, -1) @ v * s["scales"][1]
    return (out, lse) if case["lse"] else out
