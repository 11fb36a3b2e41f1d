"""Residual norms against 64 bits over every layout of a row (lanes, waves and vectors a thread, by width
and rows), each with biases, post-norms and gates of every form, at both ends of its widths."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_residual_norm import check, make

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
# what "many rows" is goes by the width: from 4 a CU on up to 2048 values, from 2 on beyond
FEW = [(6, w) for w in (8, 121, 128, 129, 200, 256, 257, 505, 512, 513, 896, 1001, 1024, 1025, 1133, 1536,
                        1537, 2048, 2049, 4096, 4100, 8192, 8193, 12000, 16384, 16385, 20001, 32768,
                        32769, 50001, 65536)]
MANY = [(1026, w) for w in (128, 256, 512, 513, 655, 896, 1001, 1024, 1025, 1133, 1535, 1536, 1537, 1999,
                            2048)] + [(516, w) for w in (2049, 3333, 4096, 4097, 5120, 8191, 8192)]


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("gate,dtype,stream", [("channel", BF16, BF16), ("row", F16, F16),
                                               ("scalar", BF16, F32), ("shared", F16, F32)])
@pytest.mark.parametrize("rows,width", FEW + MANY)
def test_gates_and_biases(rows, width, gate, dtype, stream, kind):
    # "shared": two batches have the gates of their rows in common
    shape = (2, rows // 2, width) if gate == "shared" else (rows, width)
    size = {"channel": (width,), "row": (rows, width), "scalar": (rows, 1),
            "shared": (1, rows // 2, width)}[gate]
    w, pw = (make(width, dtype, s, 0.2, 1.0) for s in (1, 2))
    b, pb = (make(width, dtype, s, 0.2) for s in (3, 4))
    check(make((rows, width), stream, 5, 2.0).view(shape), make((rows, width), dtype, 6).view(shape),
          weight=w, post_weight=pw, bias=b, post_bias=pb, gate=make(size, dtype, 7, 0.5),
          residual_scale=0.7, kind=kind)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,width", [(1027, 1025), (1027, 1133), (1027, 1536), (3, 16385), (3, 20001),
                                        (3, 32768), (1027, 655), (515, 4097)])
def test_without_post_norm_or_block(rows, width, kind):
    w, b = make(width, BF16, 1, 0.2, 1.0), make(width, BF16, 2, 0.2)
    x = make((rows, width), BF16, 3, 2.0)
    check(x, make((rows, width), BF16, 4), weight=w, bias=b, kind=kind)
    check(x, None, weight=w, kind=kind)
    check(x.float(), None, weight=w, bias=b, residual_scale=1.5, kind=kind)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows", [1, 255, 257, 5000])
@pytest.mark.parametrize("width", [1, 2, 5, 7])
def test_rows_of_fewer_than_eight_values(width, rows, kind):
    w, pw = (make(width, F16, s, 0.2, 1.0) for s in (1, 2))
    b = make(width, F16, 3, 0.2)
    x, block = make((rows, width), F16, 4, 2.0), make((rows, width), F16, 5)
    check(x, None, weight=w, kind=kind)
    check(x.float(), None, weight=w, bias=b, residual_scale=0.5, kind=kind)
    for size in ((width,), (rows, width), (rows, 1), ()):
        check(x, block, weight=w, bias=b, gate=make(size, F16, 6), kind=kind)
        check(x.float(), block, weight=w, post_weight=pw, post_bias=b, gate=make(size, F16, 6),
              residual_scale=0.7, kind=kind)


@pytest.mark.parametrize("width", [5, 200, 896, 1133, 4096, 20001])
def test_strided_rows_and_gates(width):
    rows = 1027 if width < 4096 else 9
    wide = make((2 * rows, 3 * width + 5), BF16, 1)
    w = make(width, BF16, 2, 0.2, 1.0)
    check(wide[::2, 3:width + 3], wide[1::2, width + 1:2 * width + 1], weight=w, post_weight=w,
          gate=wide[::2, 2 * width + 5:3 * width + 5], kind="layer")
    check(wide[:rows, 3:width + 3], wide[rows:, 1:width + 1], weight=w,
          gate=wide[5, 2:2 * width + 2:2])
