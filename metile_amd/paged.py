"""The paged key-value cache of a decode step (gfx950 HIP kernels via the C ABI).

A cache is a pool of pages of ``page_size`` tokens; each request has a row of a block table with
the numbers of its pages, in order. One step of a serving loop:

* :func:`paged_tables` turns the requests' lengths into the pages they need on top, block-table
  entries and the slot of every new token, on the GPU;
* :func:`paged_append` writes the step's keys and values to their slots;
* :func:`paged_attention` attends from one new token of each request over its pages.

The reference has no counterparts: its decode loop leaves cache and attention to MLX.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib
from .quantized import _stream_handle, workspace

_DTYPES = {torch.bfloat16: _lib.MT_BF16, torch.float16: _lib.MT_F16}
_CACHE_DTYPES = {**_DTYPES, torch.float8_e4m3fn: _lib.MT_FP8}


# torch's own getter without the check for initialisation, which a tensor on the device has done
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _launch(device, call, *args):
    """``call(*args, stream)`` on torch's current stream of ``device``, checked."""
    if device.index == _current_device():
        status = call(*args, _stream_handle(device))
    else:
        with torch.cuda.device(device):
            status = call(*args, _stream_handle(device))
    if status:
        _lib.check(status)


def _same_device(device, *tensors):
    """Refuses tensors that are not all on the ROCm device ``device``."""
    if device.type != "cuda":
        raise ValueError("metile_amd operators take ROCm device tensors")
    index = device.index
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise ValueError("metile_amd operators take tensors of one ROCm device")


def _rows16(t):
    """``(t, row stride, head stride)`` of a 16-bit ``[rows, heads, dim]`` tensor whose heads are
    contiguous and begin at whole 16-byte steps, as the kernels read them; a copy only where it is
    not so already. Strides of dimensions of one element are 0, whatever torch says they are."""
    row, head, one = t.stride()
    rows, heads, dim = t.shape
    row, head = row if rows > 1 else 0, head if heads > 1 else 0
    if one != 1 or (t.data_ptr() | 2 * row | 2 * head) & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        row, head = heads * dim, dim
    return t, row, head


class PagedCache:
    """A paged key-value cache over two tensors ``[pages, page_size, kv_heads, head_dim]``.

    ``key`` and ``value`` may have any strides as long as a head's values are contiguous and all
    strides are whole 16-byte steps; :meth:`allocate` makes them with a head's tokens of a page next
    to each other. bfloat16, float16 or float8_e4m3fn; an 8-bit cache holds ``key / key_scale`` and
    ``value / value_scale``. ``head_dim`` is a multiple of 16 up to 256. The object describes the
    tensors for the kernels and holds no other state.
    """

    def __init__(self, key, value, *, key_scale=1.0, value_scale=1.0):
        if key.ndim != 4 or key.shape != value.shape:
            raise ValueError("cache keys and values must be [pages, page_size, kv_heads, head_dim] "
                             "of one shape")
        if key.dtype not in _CACHE_DTYPES or value.dtype != key.dtype:
            raise ValueError("cache keys and values must both be bfloat16, float16 or "
                             "float8_e4m3fn")
        _same_device(key.device, value)
        pages, page_size, heads, dim = key.shape
        if min(key.shape) < 1 or pages * page_size >= 1 << 31:
            raise ValueError("a cache has at least one page, token and head, and fewer than 2^31 "
                             "tokens")
        if dim % 16 or dim > 256:
            raise ValueError("head_dim must be a multiple of 16 up to 256")
        for t in (key, value):
            if t.data_ptr() % 16 or t.stride(3) != 1 or any(
                    n > 1 and s * t.element_size() % 16 for n, s in zip(t.shape, t.stride()[:3])):
                raise ValueError("a cache's heads must be contiguous and its strides multiples of "
                                 "16 bytes")
            if any(n > 1 and s * t.element_size() >= 1 << 32
                   for n, s in zip(t.shape, t.stride()[:2])):
                raise ValueError("page and token strides of a cache must be below 4 GiB")
        if key.dtype != torch.float8_e4m3fn and (key_scale != 1.0 or value_scale != 1.0):
            raise ValueError("only 8-bit caches have scales")
        if not (0.0 < key_scale < float("inf") and 0.0 < value_scale < float("inf")):
            raise ValueError("cache scales must be positive and finite")
        self.key, self.value = key, value
        self.key_scale, self.value_scale = float(key_scale), float(value_scale)
        self.pages, self.page_size, self.kv_heads, self.head_dim = pages, page_size, heads, dim
        # strides of dimensions of one element do not matter, whatever torch says they are
        strides = [[s if n > 1 else 0 for n, s in zip(t.shape, t.stride()[:3])]
                   for t in (key, value)]
        self._desc = _lib.PagedCacheDesc(
            key.data_ptr(), value.data_ptr(), (ctypes.c_int64 * 3)(*strides[0]),
            (ctypes.c_int64 * 3)(*strides[1]), pages, page_size, heads, dim,
            _CACHE_DTYPES[key.dtype], self.key_scale, self.value_scale)
        self._ref = ctypes.byref(self._desc)
        self._device, self._dtype, self._head_shape = key.device, key.dtype, key.shape[2:]
        self._workspaces = {}  # (requests, heads, width, window) -> bytes

    @classmethod
    def allocate(cls, pages, page_size, kv_heads, head_dim, *, dtype=torch.bfloat16, device="cuda",
                 key_scale=1.0, value_scale=1.0):
        """A cache of uninitialised pages. Kept head by head within a page, so that what one
        attention workgroup reads of a page is one contiguous run."""
        shape = (pages, kv_heads, page_size, head_dim)
        key, value = (torch.empty(shape, dtype=dtype, device=device).transpose(1, 2)
                      for _ in range(2))
        return cls(key, value, key_scale=key_scale, value_scale=value_scale)

    def _workspace_bytes(self, *shape):
        need = self._workspaces.get(shape)
        if need is None:
            need = _lib.lib().mt_paged_attention_workspace_bytes(self._ref, *shape)
            if len(self._workspaces) >= 256:
                self._workspaces.clear()
            self._workspaces[shape] = need
        return need


class PagedStep(NamedTuple):
    """What :func:`paged_tables` gives: for each token of the step's packed batch ``slots`` (int64),
    ``positions`` and ``requests``; ``starts`` (``[requests + 1]``) and ``lengths`` of the requests;
    ``taken`` (``[1]``), the pages that the step needed as far as the tables reach. int32 but for the
    slots."""

    slots: torch.Tensor
    positions: torch.Tensor
    requests: torch.Tensor
    starts: torch.Tensor
    lengths: torch.Tensor
    taken: torch.Tensor


def _int32(t, what, ndim=1):
    if t.dtype != torch.int32 or t.ndim != ndim:
        raise ValueError(f"{what} must be {'a matrix' if ndim == 2 else 'a vector'} of int32")
    return t


def paged_tables(cached, new, block_tables, free_pages, *, page_size, tokens, free_start=None):
    """Pages, block-table entries and slots of a step whose lengths only the GPU knows.

    ``cached`` and ``new`` (int32 ``[requests]``): each request's tokens in the cache and in the
    step. ``block_tables`` (int32 ``[requests, width]``) is updated in place: the pages that the new
    tokens need are taken in order from ``free_pages`` (int32), beginning with entry ``free_start`` (a
    device int32 tensor of one element; ``None``: the first), request by request. ``tokens``: the
    size of the packed batch, at least the sum of ``new``; tokens behind that sum are padding (slot
    -1, request -1, position 0). Tokens without a page have slot -1. Where the list is exhausted,
    ``taken`` (the pages that the step needs and the tables have room for) is more than the list holds
    from ``free_start`` on; where a table is too narrow, ``lengths`` is more than ``width *
    page_size``, and ``taken`` does not count the pages beyond: a caller sees either shortage when it
    next looks. Returns a :class:`PagedStep`; nothing is synchronised.
    """
    device = block_tables.device
    _same_device(device, cached, new, free_pages, free_start)
    cached = _int32(cached, "cached").contiguous()
    new = _int32(new, "new").contiguous()
    free_pages = _int32(free_pages, "free_pages").contiguous()
    _int32(block_tables, "block_tables", 2)
    requests, width = block_tables.shape
    if cached.shape[0] != requests or new.shape[0] != requests:
        raise ValueError("cached, new and block_tables must describe the same requests")
    row, column = block_tables.stride()
    if width > 1 and column != 1:
        raise ValueError("block_tables must have contiguous rows")
    if free_start is not None and (free_start.dtype != torch.int32 or free_start.numel() != 1):
        raise ValueError("free_start must be an int32 tensor of one element")
    if not 0 <= tokens < 1 << 31:
        raise ValueError("tokens must not be negative, and below 2^31")
    if not 0 < page_size < 1 << 31:
        raise ValueError("page_size must be positive, and below 2^31")
    slots = torch.empty(tokens, dtype=torch.int64, device=device)
    positions, owners, starts, lengths, taken = torch.empty(
        2 * tokens + 2 * requests + 2, dtype=torch.int32, device=device).split_with_sizes(
            (tokens, tokens, requests + 1, requests, 1))
    _launch(device, _lib.lib().mt_paged_tables, _lib.PAGED_TABLES_ARGS.pack(
        cached.data_ptr(), new.data_ptr(), block_tables.data_ptr(), row, free_pages.data_ptr(),
        0 if free_start is None else free_start.data_ptr(), slots.data_ptr(), positions.data_ptr(),
        owners.data_ptr(), starts.data_ptr(), lengths.data_ptr(), taken.data_ptr(), requests, width,
        free_pages.shape[0], page_size, tokens))
    return PagedStep(slots, positions, owners, starts, lengths, taken)


def paged_append(key, value, cache, slots):
    """Write ``key`` and ``value`` (``[tokens, kv_heads, head_dim]``, bfloat16 or float16) to
    ``slots`` (int64 ``[tokens]``, as :func:`paged_tables` gives them) of ``cache``, in place. Tokens
    whose slot is negative or past the cache are left out. Rows may be strided (heads of a fused
    projection's output). An 8-bit cache gets the values over its scales, limited to what 8 bits
    hold."""
    dtype = key.dtype
    if dtype not in _DTYPES or value.dtype != dtype:
        raise ValueError("keys and values must both be bfloat16 or float16")
    if cache._dtype != dtype and cache._dtype != torch.float8_e4m3fn:
        raise ValueError("a 16-bit cache must have the keys' and values' dtype")
    shape = key.shape
    if shape != value.shape or len(shape) != 3 or shape[1:] != cache._head_shape:
        raise ValueError("keys and values must be [tokens, kv_heads, head_dim] of the cache's heads")
    if slots.dtype != torch.int64 or slots.shape != shape[:1]:
        raise ValueError("slots must be an int64 vector with one slot per token")
    _same_device(cache._device, key, value, slots)
    tokens = shape[0]
    if tokens == 0:
        return
    key, key_row, key_head = _rows16(key)
    value, value_row, value_head = _rows16(value)
    slots = slots.contiguous()
    _launch(cache._device, _lib.lib().mt_paged_append, cache._ref, _lib.PAGED_APPEND_ARGS.pack(
        key.data_ptr(), value.data_ptr(), key_row, key_head, value_row, value_head,
        slots.data_ptr(), tokens, _DTYPES[dtype]))


def paged_attention(query, cache, block_tables, lengths, *, scale=None, window=None,
                    return_lse=False):
    """Attention of one new token of each request over its pages of ``cache``.

    ``query`` ``[requests, heads, head_dim]`` (bfloat16 or float16; ``heads`` a multiple of the
    cache's: neighbouring query heads share a key-value head). ``block_tables`` int32
    ``[requests, width]``; ``lengths`` int32 ``[requests]``: tokens in the cache, the new one among
    them (what the table has no room for is cut off). ``scale``: of the scores (default ``head_dim **
    -0.5``). ``window``: attend to the last so many tokens only. Returns the output in ``query``'s shape and dtype and, with ``return_lse``, the
    log of the sum of exponentials (float32 ``[requests, heads]``). Requests without tokens give
    zeros and -inf. Table entries behind a request's last token are not read; tokens whose entry is
    no page of the cache are left out.
    """
    dtype = query.dtype
    if dtype not in _DTYPES:
        raise ValueError("queries must be bfloat16 or float16")
    if cache._dtype != dtype and cache._dtype != torch.float8_e4m3fn:
        raise ValueError("a 16-bit cache must have the queries' dtype")
    shape = query.shape
    if len(shape) != 3 or shape[2] != cache.head_dim:
        raise ValueError("queries must be [requests, heads, head_dim] of the cache's head_dim")
    requests, heads, dim = shape
    if heads == 0 or heads % cache.kv_heads:
        raise ValueError("query heads must be a positive multiple of the cache's heads")
    _int32(block_tables, "block_tables", 2)
    _int32(lengths, "lengths")
    width = block_tables.shape[1]
    if block_tables.shape[0] != requests or lengths.shape[0] != requests:
        raise ValueError("queries, block_tables and lengths must describe the same requests")
    if window is None:
        window = 0
    elif window < 1:
        raise ValueError("window must be positive")
    else:
        window = min(window, (1 << 31) - 1)
    device = cache._device
    _same_device(device, query, block_tables, lengths)
    out = (torch.empty_like(query) if query.is_contiguous()
           else torch.empty(shape, dtype=dtype, device=device))
    lse = torch.empty((requests, heads), dtype=torch.float32, device=device) if return_lse else None
    if not requests or not width:
        out.zero_()
        if lse is not None:
            lse.fill_(-float("inf"))
        return (out, lse) if return_lse else out
    query, row, head = _rows16(query)
    if width > 1 and block_tables.stride(1) != 1:
        block_tables = block_tables.contiguous()
    lengths = lengths.contiguous()
    args = _lib.PAGED_ATTENTION_ARGS.pack(
        query.data_ptr(), row, head, block_tables.data_ptr(), block_tables.stride(0),
        lengths.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(), requests, heads,
        width, window, dim ** -0.5 if scale is None else scale, _DTYPES[dtype])
    if device.index == _current_device():
        _attend(cache, args, requests, heads, width, window)
    else:
        with torch.cuda.device(device):
            _attend(cache, args, requests, heads, width, window)
    return (out, lse) if return_lse else out


def _attend(cache, args, requests, heads, width, window):
    stream = _stream_handle(cache._device)
    ws = workspace(cache._device, cache._workspace_bytes(requests, heads, width, window), stream)
    status = _lib.lib().mt_paged_attention(cache._ref, args, ws.data_ptr(), ws.numel(), stream)
    if status:
        _lib.check(status)
