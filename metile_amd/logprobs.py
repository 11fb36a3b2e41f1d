"""Log probabilities of tokens from a model's logits (a gfx950 HIP kernel via the C ABI).

The reference has no counterpart: its decode loop leaves sampling to MLX-LM.
"""

from __future__ import annotations

import functools
from typing import NamedTuple

import torch

from . import _lib
from .paged import _launch, _same_device, _scratch

_DTYPES = {torch.bfloat16: _lib.MT_BF16, torch.float16: _lib.MT_F16, torch.float32: _lib.MT_F32}


class TokenLogprobs(NamedTuple):
    """What :func:`token_logprobs` gives, for each row of logits: the given token's log probability
    (float32) and rank (int32), the entropy (float32), and the alternatives ``[..., top]`` in order
    (float32 and int64). ``logprobs`` and ``ranks`` are ``None`` without given tokens."""

    logprobs: torch.Tensor
    entropies: torch.Tensor
    ranks: torch.Tensor
    top_logprobs: torch.Tensor
    top_tokens: torch.Tensor


def token_logprobs(logits, tokens=None, *, top=0, temperature=1.0):
    """Log probabilities under ``softmax(logits / temperature)`` in one pass over the logits.

    ``logits`` ``[..., vocab]`` (bfloat16, float16 or float32; rows may be strided). ``tokens`` (int64
    ``[...]``): a token of each row, whose log probability and rank (how many are likelier, or as likely
    with a lower index: 0 is the likeliest) are wanted; one outside the vocabulary (padding) has -inf and
    rank -1. ``top``: how many of the likeliest tokens (0 to 32, at most ``vocab``), equal ones by index.
    Entropies are in nats; ``temperature`` is 1e-6 to 1e6. Logits of -inf (tokens that are not allowed)
    have no probability; a row of them alone has log probabilities of -inf and an entropy of 0. A row with
    NaN or +inf has NaN for both, and NaN is no alternative (token -1 where there are too few others).
    Returns a :class:`TokenLogprobs`; there are no gradients.
    """
    if logits.dtype not in _DTYPES:
        raise ValueError("logits must be bfloat16, float16 or float32")
    if logits.ndim < 1 or not 0 < logits.shape[-1] <= 1 << 24:
        raise ValueError("logits must be [..., vocab] with 1 to 2^24 tokens")
    vocab, shape = logits.shape[-1], logits.shape[:-1]
    if not 0 <= top <= min(vocab, 32):
        raise ValueError("top must be 0 to 32, and at most the vocabulary")
    if tokens is not None and (tokens.dtype != torch.int64 or tokens.shape != shape):
        raise ValueError("tokens must be int64, one for each row of logits")
    device = logits.device
    _same_device(device, tokens)
    flat = logits if logits.ndim == 2 else logits.reshape(-1, vocab)
    if vocab > 1 and flat.stride(1) != 1:
        flat = flat.contiguous()
    rows = flat.shape[0]
    if rows >= 1 << 31:
        raise ValueError("there must be fewer than 2^31 rows of logits")
    entropies = torch.empty(shape, dtype=torch.float32, device=device)
    logprobs = ranks = None
    if tokens is not None:
        tokens = tokens.contiguous()
        logprobs, ranks = torch.empty_like(entropies), torch.empty_like(entropies, dtype=torch.int32)
    top_logprobs = torch.empty((*shape, top), dtype=torch.float32, device=device)
    top_tokens = torch.empty((*shape, top), dtype=torch.int64, device=device)
    need = _workspace_bytes(device.index, rows, vocab, top)
    ws = _scratch(device, need) if need else None
    _launch(device, _lib.lib().mt_token_logprobs, _lib.TOKEN_LOGPROBS_ARGS.pack(
        flat.data_ptr(), flat.stride(0), 0 if tokens is None else tokens.data_ptr(),
        0 if tokens is None else logprobs.data_ptr(), entropies.data_ptr(),
        0 if tokens is None else ranks.data_ptr(), top_logprobs.data_ptr(), top_tokens.data_ptr(),
        rows, vocab, top, _DTYPES[logits.dtype], temperature), None if ws is None else ws.data_ptr(),
        need)
    return TokenLogprobs(logprobs, entropies, ranks, top_logprobs, top_tokens)


@functools.lru_cache(maxsize=256)
def _workspace_bytes(index, rows, vocab, top):
    with torch.cuda.device(index):
        return _lib.lib().mt_token_logprobs_workspace_bytes(rows, vocab, top)
