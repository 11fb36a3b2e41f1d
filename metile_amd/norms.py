"""The norms around a model's blocks, fused with gate and residual (gfx950 HIP kernel via the C ABI).

:func:`residual_norm` is what stands between two blocks of a decoder layer: the block's output
through its own norm (sandwich norms) and gate into the scaled residual stream, and the norm before
the next block. The reference has no counterpart: its decode loop leaves norms to MLX.
"""

from __future__ import annotations

import torch

from . import _lib
from .paged import _launch, _same_device

_DTYPES = {torch.bfloat16: _lib.MT_BF16, torch.float16: _lib.MT_F16}
_KINDS = {"rms": _lib.MT_NORM_RMS, "layer": _lib.MT_NORM_LAYER}


def _rows(t, width):
    """``t`` as rows of ``width`` contiguous values one stride apart (a copy if it is not so), and
    that stride."""
    if t.ndim == 2 and t.stride(1) == 1:
        return t, t.stride(0)
    t = t.reshape(-1, width)
    if width > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0)


def _gate(gate, shape, width, rows):
    """``(gate, stride, rows per gate row, one value a row)`` of a gate that broadcasts to
    ``shape``."""
    if gate.is_contiguous():  # the ordinary ones: a value a channel, and one for every value
        own = gate.shape
        if own == shape:
            return gate, width, 1, False
        if len(own) == 1 and own[0] == width:
            return gate, 0, max(1, rows), False
    if gate.ndim > len(shape) or any(
            g not in (1, n) for g, n in zip(reversed(gate.shape), reversed(shape))):
        raise ValueError("the gate must broadcast to the block's shape")
    scalar = width > 1 and (gate.ndim == 0 or gate.shape[-1] == 1)
    lead = list(gate.shape[:-1])
    while lead and lead[0] == 1:
        lead.pop(0)
    # leading ones are gone: what is left names whole rows of the batch from some dimension on, with
    # trailing ones where neighbouring rows share a value
    own = len(lead)
    while own and lead[own - 1] == 1:
        own -= 1
    dims = list(shape[:-1])
    at = len(dims) - len(lead)
    per = 1
    for n in dims[at + own:]:
        per *= n
    if any(n != 1 for n in dims[:at]) and own or any(
            g != n for g, n in zip(lead[:own], dims[at:at + own])):
        # rows repeat in a way one stride does not describe
        full = gate.expand(*shape[:-1], 1 if scalar else width)
        return full.reshape(rows, -1).contiguous(), (1 if scalar else width), 1, scalar
    flat = gate.reshape(-1, 1 if scalar else width)
    if not scalar and width > 1 and flat.stride(1) != 1:
        flat = flat.contiguous()
    return flat, flat.stride(0) if own else 0, per if own else max(1, rows), scalar


def residual_norm(residual, block=None, *, weight, bias=None, post_weight=None, post_bias=None,
                  gate=None, residual_scale=1.0, eps=1e-6, kind="rms"):
    """``(r, normed)`` with ``r = residual_scale * residual + gate * post(block)`` and ``normed`` its
    norm, in one pass over ``[..., width]`` tensors.

    ``kind``: ``"rms"`` (``x / sqrt(mean(x^2) + eps) * w``) or ``"layer"`` (``(x - mean) /
    sqrt(var + eps) * w``), with an optional bias, for both norms; ``post`` is the norm with
    ``post_weight`` and ``post_bias``, or nothing without a ``post_weight``. ``gate`` broadcasts to
    ``block`` (a vector of channels, a value or a vector per row or sequence). Without a ``block``
    the residual stream is only scaled (and returned as it is where the scale is 1). ``residual`` has
    the model's 16-bit type or float32, and so has ``r``; everything else, and ``normed``, has the
    16-bit type of ``weight``. Arithmetic is fp32, ``normed`` is the norm of the unrounded ``r``, each
    output is rounded once. Widths up to 65536.
    """
    dtype = weight.dtype
    stream_dtype = residual.dtype
    if dtype not in _DTYPES:
        raise ValueError("norm weights must be bfloat16 or float16")
    if stream_dtype != dtype and stream_dtype != torch.float32:
        raise ValueError("the residual must have the weights' dtype or float32")
    code = _KINDS.get(kind)
    if code is None:
        raise ValueError("kind must be 'rms' or 'layer'")
    shape = residual.shape
    if not shape or not 1 <= shape[-1] <= 65536:
        raise ValueError("the residual's last dimension must be 1 to 65536")
    width = shape[-1]
    if block is None:
        if post_weight is not None or post_bias is not None or gate is not None:
            raise ValueError("a post-norm and a gate need a block")
    elif block.shape != shape or block.dtype != dtype:
        raise ValueError("the block must have the residual's shape and the weights' dtype")
    if post_bias is not None and post_weight is None:
        raise ValueError("a post-norm's bias needs its weight")
    if gate is not None and gate.dtype != dtype:
        raise ValueError("the gate must have the weights' dtype")
    device = residual.device
    _same_device(device, block, weight, bias, post_weight, post_bias, gate)
    weight = _vector(weight, width, dtype)
    if bias is not None:
        bias = _vector(bias, width, dtype)
    if post_weight is not None:
        post_weight = _vector(post_weight, width, dtype)
    if post_bias is not None:
        post_bias = _vector(post_bias, width, dtype)
    rows = residual.numel() // width
    if rows >= 1 << 31:
        raise ValueError("too many rows")
    whole = residual.is_contiguous()
    block_whole = block is not None and block.is_contiguous()
    keep = block is None and residual_scale == 1.0
    out = (residual if keep else torch.empty_like(residual) if whole
           else torch.empty(shape, dtype=stream_dtype, device=device))
    normed = (torch.empty_like(block) if block_whole
              else torch.empty(shape, dtype=dtype, device=device))
    if rows == 0:
        return out, normed
    x, x_stride = (residual, width) if whole else _rows(residual, width)
    b, b_stride = ((None, 0) if block is None else (block, width) if block_whole
                   else _rows(block, width))
    g, g_stride, g_rows, g_scalar = ((None, 0, 1, False) if gate is None
                                     else _gate(gate, shape, width, rows))
    code16 = _DTYPES[dtype]
    _launch(device, _lib.lib().mt_residual_norm, _lib.RESIDUAL_NORM_ARGS.pack(
        x.data_ptr(), _ptr(b), weight.data_ptr(), _ptr(bias), _ptr(post_weight), _ptr(post_bias),
        _ptr(g), 0 if keep else out.data_ptr(), normed.data_ptr(), x_stride, b_stride, g_stride,
        rows, width, g_rows, g_scalar, residual_scale, eps, code, code16,
        code16 if stream_dtype == dtype else _lib.MT_F32))
    return out, normed


def _vector(t, width, dtype):
    """A weight or bias, checked, its values next to each other."""
    if t.dtype != dtype or t.ndim != 1 or t.shape[0] != width:
        raise ValueError("norm weights and biases must be vectors of the width, of one dtype")
    return t if t.is_contiguous() else t.contiguous()


def _ptr(t):
    return 0 if t is None else t.data_ptr()
