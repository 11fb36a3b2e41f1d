"""Residual norms on the GPU against 64 bits: widths, rows, types, gates, strides and contents."""

from __future__ import annotations

import pytest
import torch

import metile_amd as mt
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu


def make(shape, dtype, seed, scale=1.0, mean=0.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale + mean).to(dtype)


def check(residual, block, **options):
    r, normed = mt.residual_norm(residual, block, **options)
    want_r, want = ref.residual_norm(residual, block, **options)
    dtype = options["weight"].dtype
    assert r.dtype == residual.dtype and normed.dtype == dtype
    assert r.shape == residual.shape == normed.shape
    # r: a norm's fp32 relative error (2^-19: sums of up to 65536 squares in a tree, root, products),
    # of its terms' size, and one rounding. normed: the same of x / deviation, whose size the weights
    # scale; a mean taken off adds 2^-20 of the largest x over the deviation.
    x = want_r
    terms = residual.double().cpu().abs() * abs(options.get("residual_scale", 1.0))
    if block is not None:  # a post-norm's bias is a term of its own: the two may cancel
        gate, bias = options.get("gate"), options.get("post_bias")
        part = block.double().cpu()
        if options.get("post_weight") is not None:
            part = ref.norm(part, options["post_weight"], None, options.get("eps", 1e-6),
                            options.get("kind", "rms")).abs()
            part = part if bias is None else part + bias.double().cpu().abs()
        terms = terms + part.abs() * (1.0 if gate is None else gate.double().cpu().abs())
    tol_r = ref.UNIT[residual.dtype] * want_r.abs() + 2.0 ** -19 * terms + 2.0 ** -25
    assert bool(((r.double().cpu() - want_r).abs() <= tol_r * 1.01).all())
    eps = options.get("eps", 1e-6)
    centre = x - x.mean(-1, keepdim=True) if options.get("kind") == "layer" else x
    deviation = torch.sqrt((centre * centre).mean(-1, keepdim=True) + eps)
    size = (terms + x.abs().mean(-1, keepdim=True)) / deviation
    weight = options["weight"].double().cpu().abs()
    bias = options.get("bias")
    tol = (ref.UNIT[dtype] * want.abs() + 2.0 ** -18 * size * weight + 2.0 ** -25
           + (0 if bias is None else 2.0 ** -22 * bias.double().cpu().abs()))
    assert bool(((normed.double().cpu() - want).abs() <= tol * 1.01).all())
    return r, normed


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dtype,stream", [(torch.bfloat16, torch.bfloat16),
                                          (torch.float16, torch.float16),
                                          (torch.bfloat16, torch.float32),
                                          (torch.float16, torch.float32)])
@pytest.mark.parametrize("width", [1, 7, 64, 513, 896, 1001, 2048, 5120, 8192, 10000, 16384, 65536])
@pytest.mark.parametrize("rows", [1, 5])
def test_widths_and_types(rows, width, dtype, stream, kind):
    w, pw = (make(width, dtype, s, 0.2, 1.0) for s in (1, 2))
    b, pb = (make(width, dtype, s, 0.2) for s in (3, 4))
    check(make((rows, width), stream, 5, 3.0), make((rows, width), dtype, 6, 2.0), weight=w,
          post_weight=pw, bias=b, post_bias=pb, residual_scale=0.6, kind=kind)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("width", [33, 896, 1537, 4096, 4100, 9000, 33000])
def test_many_rows(width, kind):
    rows = 2051
    w = make(width, torch.bfloat16, 1, 0.2, 1.0)
    check(make((rows, width), torch.bfloat16, 5), make((rows, width), torch.bfloat16, 6), weight=w,
          post_weight=w, kind=kind)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,width", [(1, 128), (17, 8), (2051, 64), (2051, 121), (2051, 128),
                                        (7, 129), (2051, 171), (2051, 256), (9, 257)])
def test_narrow_rows(rows, width, kind):  # several rows a wave, the last of them not all there
    w = make(width, torch.bfloat16, 1, 0.2, 1.0)
    check(make((rows, width), torch.bfloat16, 5), make((rows, width), torch.bfloat16, 6), weight=w,
          post_weight=w, kind=kind)


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", [(), (1,), (1, 1, 1), (96,), (3, 1, 96), (3, 1, 1), (3, 5, 1),
                                  (3, 5, 96), (5, 96), (5, 1), (1, 5, 96), (1, 1, 96)])
def test_gates(gate, post):
    dtype = torch.float16
    w = make(96, dtype, 1, 0.2, 1.0)
    check(make((3, 5, 96), dtype, 2), make((3, 5, 96), dtype, 3), weight=w,
          post_weight=w if post else None, gate=make(gate, dtype, 4), residual_scale=1.25)


def test_without_a_block():
    w = make(896, torch.bfloat16, 1, 0.2, 1.0)
    x = make((4, 896), torch.bfloat16, 2)
    r, _ = check(x, None, weight=w)
    assert r is x
    r, _ = check(x, None, weight=w, residual_scale=0.5)
    assert r is not x
    check(make((4, 896), torch.float32, 2), None, weight=w, kind="layer")


def test_strided_inputs():
    dtype = torch.bfloat16
    w = make(200, dtype, 1, 0.2, 1.0)
    wide = make((6, 555), dtype, 2)
    check(wide[:, 3:203], wide[:, 301:501], weight=w, gate=wide[:, 100:300])
    check(wide[::2, 3:203], wide[1::2, 301:501], weight=w[:200])
    flipped = make((200, 6), dtype, 3).t()
    check(flipped, flipped, weight=make((200, 2), dtype, 4, 0.2, 1.0)[:, 1])
    check(make((2, 3, 2, 400), dtype, 5)[..., 1, ::2], make((2, 3, 200), dtype, 6), weight=w)


def test_special_values():
    dtype = torch.bfloat16
    w = torch.ones(96, dtype=dtype, device="cuda")
    zero = torch.zeros(3, 96, dtype=dtype, device="cuda")
    r, normed = mt.residual_norm(zero, zero, weight=w, post_weight=w, eps=1e-6)
    assert not bool(r.any()) and not bool(normed.any())
    x = make((3, 96), dtype, 2)
    x[0, 5], x[1, 7] = float("nan"), float("inf")
    r, normed = mt.residual_norm(x, zero, weight=w)
    assert bool(torch.isnan(normed[0]).all()) and bool(torch.isnan(normed[1, 7]))
    assert bool((normed[1, :7] == 0).all()) and bool(torch.isfinite(normed[2]).all())
    # a constant row has no deviation: layer norm gives the bias
    b = make(96, dtype, 3)
    _, normed = mt.residual_norm(torch.full_like(zero, 3.0), None, weight=w, bias=b, kind="layer")
    assert torch.equal(normed, b.expand(3, 96))


def test_large_and_small_values_keep_their_precision():
    w = make(896, torch.bfloat16, 1, 0.2, 1.0)
    for scale in (1e-3, 1.0, 1e6):
        check(make((3, 896), torch.float32, 2, scale), make((3, 896), torch.bfloat16, 3, scale),
              weight=w, kind="rms")
    # deviations around a mean a thousand times as large
    check(make((3, 896), torch.float32, 2, 1.0, 1000.0), None, weight=w, kind="layer")


def test_no_rows_other_stream_and_graph():
    w = make(512, torch.float16, 1, 0.2, 1.0)
    r, normed = mt.residual_norm(make((0, 512), torch.float16, 2), None, weight=w,
                                 residual_scale=2.0)
    assert r.shape == normed.shape == (0, 512)
    x, b = make((9, 512), torch.float16, 2), make((9, 512), torch.float16, 3)
    want = mt.residual_norm(x, b, weight=w)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = mt.residual_norm(x, b, weight=w)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            held = mt.residual_norm(x, b, weight=w)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(held, want))
        x.mul_(0.5)
        want = mt.residual_norm(x, b, weight=w)


def test_refusals():
    dtype = torch.bfloat16
    x, w = make((2, 64), dtype, 1), make(64, dtype, 2)
    bad = [
        (lambda: mt.residual_norm(x, weight=w.float()), "bfloat16 or float16"),
        (lambda: mt.residual_norm(x.half(), weight=w), "residual"),
        (lambda: mt.residual_norm(x, x.float(), weight=w), "block"),
        (lambda: mt.residual_norm(x, x[:1], weight=w), "block"),
        (lambda: mt.residual_norm(x, weight=w[:32]), "vectors of the width"),
        (lambda: mt.residual_norm(x, x, weight=w, post_bias=w), "needs its weight"),
        (lambda: mt.residual_norm(x, weight=w, gate=w), "need a block"),
        (lambda: mt.residual_norm(x, x, weight=w, gate=w[:32]), "broadcast"),
        (lambda: mt.residual_norm(x, x, weight=w, gate=w.float()), "gate"),
        (lambda: mt.residual_norm(x, x, weight=w, kind="batch"), "kind"),
        (lambda: mt.residual_norm(x, x, weight=w, eps=-1.0), "eps"),
        (lambda: mt.residual_norm(x, x, weight=w, residual_scale=float("inf")), "finite"),
        (lambda: mt.residual_norm(x, x, weight=w.cpu()), "one ROCm device"),
        (lambda: mt.residual_norm(make((1, 65537), dtype, 1), weight=make(65537, dtype, 2)),
         "65536"),
    ]
    for call, message in bad:
        with pytest.raises(ValueError, match=message):
            call()
