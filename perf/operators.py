"""The measured work of the decode-step operators around a served model's projections.

Each case is one pass through one operator, as a serving loop calls it:

* ``tables``: ``paged_tables``. Block tables and slot maps of a step, from the requests' lengths.
* ``append``: ``paged_append``. A step's keys and values, heads of a fused projection's output, written
  to their slots of the paged cache (bfloat16, float16 or 8-bit floats).
* ``attention``: ``paged_attention``. One new token of each request over its pages.
* ``norm``: ``residual_norm``. A block's output through its post-norm, gate and scaled residual into
  the residual stream, and the next block's pre-norm.

Shapes are the benchmark's and tests' model widths (896, 1536, 3584, 4096, 5120 and 8192 features, heads
of 64 and 128) and generic ones between them. With ``own`` false the operators are computed in plain
torch operations in 32 bits; with it true through the package's kernels.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32,
          "fp8": torch.float8_e4m3fn}
HEADS = ((12, 2, 128), (14, 2, 64), (28, 4, 128), (32, 8, 128), (40, 8, 128), (32, 32, 128),
         (16, 16, 80), (24, 3, 96), (64, 8, 64), (16, 1, 256), (20, 5, 192), (48, 1, 128))
WIDTHS = (896, 1536, 3584, 4096, 5120, 8192)
MOST_TOKENS = 1 << 20               # of a step's tables
MOST_APPEND = 16384 * 8 * 128       # values of a step's keys
MOST_CACHE = 2 * 131072 * 8 * 128   # keys read by one attention call, and of its padded batch
MOST_NORM = 16384 * 4096            # values of the residual stream


def listed():
    return [
        # a decode step of 64 requests, every eighth of them idle
        dict(name="tables-decode-64", kind="tables", requests=64, idle=8, low=1, high=1, past=4096,
             page=16),
        # a large step of 4096 requests: prompts of 1 to 1900 tokens, some behind a cached prefix
        dict(name="tables-prompts-4096", kind="tables", requests=4096, idle=64, low=1, high=1900,
             past=1500, page=24),
        # one request's new token in a small model
        dict(name="append-1", kind="append", tokens=1, hq=12, hkv=2, dim=128, page=16, dtype="bf16",
             cache="bf16", heads_outer=True),
        # a chunk of prompts into an 8-bit cache
        dict(name="append-16k-fp8", kind="append", tokens=16384, hq=32, hkv=8, dim=128, page=64,
             dtype="bf16", cache="fp8", heads_outer=False),
        # one request of a small model, an ordinary context: the smallest attention there is
        dict(name="attention-1x2k", kind="attention", requests=1, idle=0, low=2049, high=2049, hq=12,
             hkv=2, dim=128, page=16, dtype="bf16", cache="bf16", window=0, lse=False,
             heads_outer=True),
        # a ragged batch of requests from one token to long ones, some slots of the batch empty
        dict(name="attention-ragged-64", kind="attention", requests=64, idle=4, low=1, high=8192,
             hq=32, hkv=8, dim=128, page=16, dtype="bf16", cache="bf16", window=0, lse=False,
             heads_outer=True),
        # two very long contexts
        dict(name="attention-2x128k", kind="attention", requests=2, idle=0, low=131072, high=131072,
             hq=32, hkv=8, dim=128, page=64, dtype="bf16", cache="bf16", window=0, lse=True,
             heads_outer=False),
        # an 8-bit cache of narrow heads, sliding window, odd page size, float16 queries
        dict(name="attention-fp8-window", kind="attention", requests=48, idle=0, low=1000,
             high=12001, hq=64, hkv=8, dim=64, page=24, dtype="f16", cache="fp8", window=4096,
             lse=False, heads_outer=True),
        # the norms around one token's block: sandwich norm with residual scale
        dict(name="norm-1row", kind="norm", rows=1, width=1536, norm="rms", dtype="bf16",
             residual="bf16", post=True, gate="none", scale=0.5),
        # a batch of sequences, pre-norm only, residual stream held in 32 bits
        dict(name="norm-100rows", kind="norm", rows=100, width=5120, norm="rms", dtype="bf16",
             residual="f32", post=False, gate="none", scale=1.0),
        # prompts of a wide model through gated sandwich norms
        dict(name="norm-16k", kind="norm", rows=16384, width=4096, norm="rms", dtype="bf16",
             residual="bf16", post=True, gate="row", scale=1.0),
        # layer norms with biases of an odd width, a gate a channel
        dict(name="norm-layer-odd", kind="norm", rows=2047, width=1001, norm="layer", dtype="f16",
             residual="f16", post=True, gate="channel", scale=0.7),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    kind = rng.choice(("tables", "append", "attention", "attention", "attention", "norm", "norm"))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    page = rng.choice((1, 8, 16, 16, 20, 32, 48, 64, 128, 256))
    if kind == "tables":
        while True:
            requests = _log(rng, 1, 4096)
            high = 1 if rng.random() < 0.4 else _log(rng, 2, 8192)
            case = dict(kind=kind, requests=requests, idle=rng.randint(0, requests // 4), low=1,
                        high=high, past=_log(rng, 1, 16384), page=page)
            tokens, width = sum(_new(case)), -(-(case["past"] + high) // page)
            if tokens <= MOST_TOKENS and requests * width <= 1 << 25:
                return case
    hq, hkv, dim = rng.choice(HEADS)
    cache = rng.choice((dtype, dtype, "fp8"))
    if kind == "append":
        return dict(kind=kind, tokens=_log(rng, 1, MOST_APPEND // (hkv * dim)), hq=hq, hkv=hkv,
                    dim=dim, page=page, dtype=dtype, cache=cache, heads_outer=rng.random() < 0.5)
    if kind == "attention":
        most = MOST_CACHE // (hkv * dim)
        high = _log(rng, 1, min(131072, most))
        requests = _log(rng, 1, max(1, min(512, most // high)))
        low = high if rng.random() < 0.3 else _log(rng, 1, high)
        return dict(kind=kind, requests=requests, idle=rng.randint(0, requests // 8), low=low,
                    high=high, hq=hq, hkv=hkv, dim=dim, page=page, dtype=dtype, cache=cache,
                    window=_log(rng, 1, 8192) if rng.random() < 0.25 else 0,
                    lse=rng.random() < 0.3, heads_outer=rng.random() < 0.5)
    width = rng.choice(WIDTHS) if rng.random() < 0.6 else _log(rng, 65, 16384)
    return dict(kind=kind, rows=_log(rng, 1, MOST_NORM // width), width=width,
                norm=rng.choice(("rms", "rms", "layer")), dtype=dtype,
                residual=rng.choice((dtype, dtype, "f32")), post=rng.random() < 0.6,
                gate=rng.choice(("none", "none", "channel", "row", "scalar")),
                scale=rng.choice((1.0, 1.0, round(rng.uniform(0.2, 1.4), 3))))


# ---- inputs --------------------------------------------------------------------------------------


def _spread(n, low, high):
    """``n`` whole numbers spread evenly over the logarithm of ``low`` .. ``high``."""
    return [int(round(low * (high / low) ** ((i + 0.5) / n))) for i in range(n)]


def _new(case):
    """New tokens of each request, idle ones last."""
    return _spread(case["requests"] - case["idle"], case["low"], case["high"]) + [0] * case["idle"]


def _lengths(case):
    """Tokens of each request in the cache, its new one among them; empty slots of the batch last."""
    return _new(case)


def _tables(g, lengths, most, page, device):
    """Block tables for lengths up to ``most`` over a pool of pages in random order, the pages each
    length needs assigned; the columns behind them hold -1. Gives the pool's size too (a few pages
    stay unused)."""
    counts = torch.tensor([-(-n // page) for n in lengths], device=device)
    total, width = int(counts.sum()), -(-most // page)
    order = torch.randperm(total + 3, generator=g, device=device, dtype=torch.int32)
    column = torch.arange(width, device=device)
    taken = column < counts[:, None]
    tables = torch.full((len(lengths), width), -1, dtype=torch.int32, device=device)
    tables[taken] = order[:total]
    return tables, total + 3


def _pool(g, pages, page, hkv, dim, cache, heads_outer, device):
    """One cache tensor [pages, page, heads, dim], stored with the heads outside or inside the slots.
    Made in place, a part at a time: the largest are a gigabyte."""
    shape = (pages, hkv, page, dim) if heads_outer else (pages, page, hkv, dim)
    pool = torch.empty(shape, dtype=DTYPES[cache], device=device)
    flat = pool.view(-1)
    for at in range(0, flat.numel(), 1 << 27):
        part = flat[at:at + (1 << 27)]
        part.copy_(torch.randn(part.numel(), generator=g, device=device, dtype=torch.float32))
    return pool.transpose(1, 2) if heads_outer else pool


def _inputs(case, seed):
    device = "cuda"
    rng = random.Random(seed)
    g = torch.Generator(device).manual_seed(seed)
    kind = case["kind"]

    def randn(*shape, dtype=case.get("dtype"), scale=1.0, mean=0.0):
        x = torch.randn(*shape, generator=g, device=device).mul_(scale).add_(mean)
        return x.to(DTYPES[dtype])

    if kind == "tables":
        requests, page = case["requests"], case["page"]
        new = _new(case)
        # a fifth of the requests start here, the others have up to `past` tokens in the cache
        past = [0 if i % 5 == 4 else n
                for i, n in enumerate(_spread(requests, 1, case["past"]))]
        rng.shuffle(new)
        rng.shuffle(past)
        total = [a + b for a, b in zip(past, new)]
        tables, pages = _tables(g, total, case["past"] + case["high"], page, device)
        # entries that the step has to fill: the pages behind each request's cached ones
        have = torch.tensor([-(-n // page) for n in past], device=device)
        fresh = torch.arange(tables.shape[1], device=device) >= have[:, None]
        taken = tables[fresh & (tables >= 0)]
        free = taken[torch.randperm(taken.numel(), generator=g, device=device)]
        tables[fresh] = -1
        return dict(cached=torch.tensor(past, dtype=torch.int32, device=device),
                    new=torch.tensor(new, dtype=torch.int32, device=device), tables=tables,
                    free=torch.cat([free, free.new_zeros(1)]), page=page, tokens=max(1, sum(new)))
    if kind == "norm":
        m, h = case["rows"], case["width"]
        gate = {"none": None, "channel": (h,), "row": (m, h), "scalar": (m, 1)}[case["gate"]]
        layer = case["norm"] == "layer"
        return dict(residual=randn(m, h, dtype=case["residual"], scale=2.0), block=randn(m, h),
                    weight=randn(h, scale=0.1, mean=1.0),
                    post_weight=randn(h, scale=0.1, mean=1.0) if case["post"] else None,
                    bias=randn(h, scale=0.1) if layer else None,
                    post_bias=randn(h, scale=0.1) if layer and case["post"] else None,
                    gate=None if gate is None else randn(*gate, scale=0.5))
    hq, hkv, dim, page = case["hq"], case["hkv"], case["dim"], case["page"]
    # float caches hold values as they are; an 8-bit one holds them over a scale of its own
    scales = (1.0, 1.0) if case["cache"] != "fp8" else (0.75, 1.25)
    if kind == "append":
        tokens = case["tokens"]
        pages = -(-2 * tokens // page) + 2
        slots = torch.randperm(pages * page, generator=g, device=device)[:tokens]
        slots[1::9] = -1  # tokens of padding
        fused = randn(tokens, (hq + 2 * hkv) * dim)
        _, key, value = fused.split([hq * dim, hkv * dim, hkv * dim], dim=1)
        shape = (tokens, hkv, dim)
        return dict(key=key.unflatten(1, shape[1:]), value=value.unflatten(1, shape[1:]),
                    slots=slots, scales=scales,
                    key_cache=_pool(g, pages, page, hkv, dim, case["cache"], case["heads_outer"],
                                    device),
                    value_cache=_pool(g, pages, page, hkv, dim, case["cache"],
                                      case["heads_outer"], device))
    lengths = _lengths(case)
    rng.shuffle(lengths)
    tables, pages = _tables(g, lengths, case["high"], page, device)
    return dict(query=randn(case["requests"], hq, dim), tables=tables, scales=scales,
                lengths=torch.tensor(lengths, dtype=torch.int32, device=device),
                key_cache=_pool(g, pages, page, hkv, dim, case["cache"], case["heads_outer"],
                                device),
                value_cache=_pool(g, pages, page, hkv, dim, case["cache"], case["heads_outer"],
                                  device))


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if own and "key_cache" in state:  # a serving program's handle of its cache: the tensors and scales
        import metile_amd as mt

        key_scale, value_scale = state["scales"]
        state["cache"] = mt.PagedCache(state["key_cache"], state["value_cache"],
                                       key_scale=key_scale, value_scale=value_scale)
    return state


# ---- one pass ------------------------------------------------------------------------------------


def run(state):
    kind = state["case"]["kind"]
    return (_KERNELS if own else _PLAIN)[kind](state, state["case"])


def _run_tables(s, case):
    import metile_amd as mt

    step = mt.paged_tables(s["cached"], s["new"], s["tables"], s["free"], page_size=s["page"],
                           tokens=s["tokens"])
    return [s["tables"], step.slots, step.positions, step.requests, step.starts, step.lengths,
            step.taken]


def _run_append(s, case):
    import metile_amd as mt

    mt.paged_append(s["key"], s["value"], s["cache"], s["slots"])
    return [s["key_cache"], s["value_cache"]]


def _run_attention(s, case):
    import metile_amd as mt

    return mt.paged_attention(s["query"], s["cache"], s["tables"], s["lengths"],
                              window=case["window"] or None, return_lse=case["lse"])


def _run_norm(s, case):
    import metile_amd as mt

    return mt.residual_norm(s["residual"], s["block"], weight=s["weight"], bias=s["bias"],
                            post_weight=s["post_weight"], post_bias=s["post_bias"],
                            gate=s["gate"], residual_scale=case["scale"], eps=1e-6,
                            kind=case["norm"])


_KERNELS = {"tables": _run_tables, "append": _run_append, "attention": _run_attention,
            "norm": _run_norm}


# ---- the operators in plain torch operations -----------------------------------------------------


def _plain_tables(s, case):
    cached, new, tables, free, page = s["cached"], s["new"], s["tables"], s["free"], s["page"]
    lengths = cached + new
    have = (cached + page - 1) // page
    need = (lengths + page - 1) // page - have
    ends = new.cumsum(0)
    starts = torch.cat([ends.new_zeros(1), ends]).to(torch.int32)
    first = need.cumsum(0) - need
    t = torch.arange(s["tokens"], device=cached.device)
    request = torch.searchsorted(ends, t, right=True)
    live = request < cached.numel()
    at = request.clamp(max=cached.numel() - 1)
    position = torch.where(live, t - starts[at] + cached[at], 0)
    column = position // page
    fresh = live & (column >= have[at])
    opens = fresh & (position % page == 0)
    rows, columns = at[opens], column[opens]
    tables[rows, columns] = free[first[rows] + columns - have[rows]]
    slots = torch.where(live, tables[at, column].long() * page + position % page, -1)
    return [tables, slots, position.to(torch.int32), torch.where(live, request, -1).to(torch.int32),
            starts, lengths, need.sum(0, keepdim=True).to(torch.int32)]


def _bits(cache):
    """An 8-bit cache's bytes (torch indexes no 8-bit floats); others as they are."""
    return cache.view(torch.uint8) if cache.dtype == DTYPES["fp8"] else cache


def _plain_append(s, case):
    page = s["key_cache"].shape[1]
    live = s["slots"] >= 0
    slots = s["slots"][live]
    for rows, cache, scale in ((s["key"], s["key_cache"], s["scales"][0]),
                               (s["value"], s["value_cache"], s["scales"][1])):
        rows = rows[live].float() / scale
        if case["cache"] == "fp8":
            rows = rows.clamp(-448.0, 448.0)
        _bits(cache)[slots // page, slots % page] = _bits(rows.to(cache.dtype))
    return [s["key_cache"], s["value_cache"]]


def _pages(cache, tables):
    """[requests, heads, positions, dim] of each request's pages, in 32 bits."""
    rows = _bits(cache)[tables.clamp(min=0).long()]
    if cache.dtype == DTYPES["fp8"]:
        rows = rows.view(cache.dtype)
    r, w, p, h, d = rows.shape
    return rows.reshape(r, w * p, h, d).transpose(1, 2).float()


def _plain_attention(s, case):
    query, tables, lengths = s["query"], s["tables"], s["lengths"]
    requests, hq, dim = query.shape
    hkv = s["key_cache"].shape[2]
    q = query.float().reshape(requests, hkv, hq // hkv, dim)
    keys = _pages(s["key_cache"], tables)
    scores = (q @ keys.transpose(2, 3)) * (s["scales"][0] / math.sqrt(dim))
    del keys
    t = torch.arange(scores.shape[-1], device=query.device)
    seen = t < lengths[:, None]
    if case["window"]:
        seen &= t >= lengths[:, None] - case["window"]
    seen = seen[:, None, None, :]
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    values = _pages(s["value_cache"], tables)
    out = (weights @ values) * (s["scales"][1] / total.clamp(min=torch.finfo(torch.float32).tiny))
    out = out.reshape(requests, hq, dim).to(query.dtype)
    return (out, (top + torch.log(total)).reshape(requests, hq)) if case["lse"] else out


def _plain_norm_of(x, weight, bias, kind):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()
    return x if bias is None else x + bias.float()


def _plain_norm(s, case):
    block = s["block"].float()
    if s["post_weight"] is not None:
        block = _plain_norm_of(block, s["post_weight"], s["post_bias"], case["norm"])
    if s["gate"] is not None:
        block = block * s["gate"].float()
    residual = s["residual"].float() * case["scale"] + block
    normed = _plain_norm_of(residual, s["weight"], s["bias"], case["norm"])
    return residual.to(s["residual"].dtype), normed.to(s["block"].dtype)


_PLAIN = {"tables": _plain_tables, "append": _plain_append, "attention": _plain_attention,
          "norm": _plain_norm}


# ---- what a pass cannot do without ---------------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "tables":
        # per request two lengths read, a start and a length written; per token a slot, a position
        # and a request; per new page its number read and written
        tokens = sum(_new(case))
        return {"bytes": 16 * case["requests"] + 16 * tokens + 8 * (tokens // case["page"]),
                "flops": 0}
    if kind == "norm":
        n = case["rows"] * case["width"]
        stream = 4 if case["residual"] == "f32" else 2
        gate = {"none": 0, "channel": case["width"], "row": n, "scalar": case["rows"]}[case["gate"]]
        vectors = case["width"] * (2 if case["norm"] == "layer" else 1) * (1 + case["post"])
        return {"bytes": n * (2 * stream + 4) + 2 * (gate + vectors), "flops": 10 * n}
    size = 1 if case["cache"] == "fp8" else 2
    row = case["hkv"] * case["dim"]
    if kind == "append":
        return {"bytes": case["tokens"] * (2 * row * (2 + size) + 8), "flops": 0}
    seen = [min(n, case["window"] or n) for n in _lengths(case)]
    heads = case["hq"] * case["dim"]
    return {"bytes": sum(seen) * row * 2 * size + sum(-(-n // case["page"]) for n in seen) * 4
            + case["requests"] * (4 * heads + 4 + (4 * case["hq"] if case["lse"] else 0)),
            "flops": 4 * sum(seen) * heads}


# ---- the definitions in 64 bits ------------------------------------------------------------------


def exact(case, seed):
    kind = case["kind"]
    if kind == "tables":
        return None  # whole numbers
    s = _inputs(case, seed)
    if kind == "append":
        caches = []
        for rows, cache, scale in ((s["key"], s["key_cache"], s["scales"][0]),
                                   (s["value"], s["value_cache"], s["scales"][1])):
            out = cache.double().contiguous()
            flat = out.view(-1, *out.shape[2:])
            held = rows.double() / scale
            if case["cache"] == "fp8":  # four significant bits, none below 2^-9, at most 448
                step = torch.exp2(torch.floor(torch.log2(held.abs().clamp(min=2.0 ** -6))) - 3)
                held = (torch.round(held / step) * step).clamp(-448, 448)
            where = torch.nonzero(s["slots"] >= 0)[:, 0]
            flat.index_copy_(0, s["slots"][where], held[where])
            caches.append(out)
        return caches
    if kind == "attention":
        outs, lses = [], []
        group = case["hq"] // case["hkv"]
        for r, length in enumerate(s["lengths"].tolist()):
            first = max(0, length - case["window"]) if case["window"] else 0
            at = torch.arange(first, length, device="cuda")
            pages, offsets = s["tables"][r].long()[at // case["page"]], at % case["page"]
            q = s["query"][r].double()
            out, lse = torch.zeros_like(q), torch.full_like(q[:, 0], -math.inf)
            for h in range(case["hkv"] if length else 0):
                k, v = (_bits(s[name])[pages, offsets, h].view(s[name].dtype).double()
                        for name in ("key_cache", "value_cache"))
                rows = slice(h * group, (h + 1) * group)
                logits = q[rows] @ k.T.contiguous()
                logits = logits * s["scales"][0] * case["dim"] ** -0.5
                lse[rows] = torch.logsumexp(logits, -1)
                out[rows] = torch.softmax(logits, -1) @ v * s["scales"][1]
            outs.append(out)
            lses.append(lse)
        out = torch.stack(outs)
        return (out, torch.stack(lses)) if case["lse"] else out
    layer = case["norm"] == "layer"

    def norm(x, weight, bias):
        mean = x.mean(1, keepdim=True) if layer else 0.0
        deviation = ((x - mean).square().mean(1, keepdim=True) + 1e-6).sqrt()
        return (x - mean) / deviation * weight.double() + (bias.double() if layer else 0.0)

    x = s["block"].double()
    if case["post"]:
        x = norm(x, s["post_weight"], s["post_bias"])
    x = case["scale"] * s["residual"].double() + x * (1.0 if s["gate"] is None else
                                                      s["gate"].double())
    return x, norm(x, s["weight"], s["bias"])
