"""The check that the executors make of their kernels on the sample: roundings of the native
composition alone never refuse a kernel, wrong results always do."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

import metile_amd as mt
from metile_amd import native, quantized


def _sample(seed, n=8960):
    """Gate and up projections in fp32 as a layer of uniform weights gives them (deviation
    sqrt(1/3)), their SwiGLU rounded once and by the native composition (four roundings)."""
    g = torch.Generator().manual_seed(seed)
    gate, up = torch.randn(2, n, generator=g) * 3 ** -0.5
    once = (F.silu(gate) * up).to(torch.bfloat16)
    return once, F.silu(gate.to(torch.bfloat16)) * up.to(torch.bfloat16)


def test_results_rounded_once_are_never_refused():
    refused = 0
    for seed in range(600):
        once, composed = _sample(seed)
        refused += not mt.affine_swiglu_compatible(once, composed)
        quantized._fidelity_gate(once, composed, lambda: once, "affine SwiGLU")
    assert refused > 0  # the first comparison alone would have refused some of them


def test_neighbouring_roundings_are_not_refused():
    # fp32 sums in another order round to the neighbouring value now and then
    for seed in range(100):
        once, composed = _sample(seed)
        bits = once.view(torch.int16).clone()
        bits[seed::50] += 1
        quantized._fidelity_gate(bits.view(torch.bfloat16), composed, lambda: once, "affine SwiGLU")


@pytest.mark.parametrize("fault", ["scaled", "peak", "nan", "zero", "shifted"])
def test_wrong_results_are_refused_with_their_figures(fault):
    once, composed = _sample(1)
    bad = once.clone()
    if fault == "scaled":
        bad = (once.float() * 1.01).to(torch.bfloat16)
    elif fault == "peak":
        i = int(once.float().abs().argmax())
        bad[i] = (once[i].float() * 1.03).to(torch.bfloat16)
    elif fault == "nan":
        bad[17] = float("nan")
    elif fault == "zero":
        bad[:64] = 0
    else:
        bad = once.roll(1)
    with pytest.raises(RuntimeError, match=r"affine SwiGLU.*rms .*peak .*native.*rms .*peak"):
        quantized._fidelity_gate(bad, composed, lambda: once, "affine SwiGLU")


def test_empty_samples_pass_without_a_comparison():
    none = torch.empty(0, 8, dtype=torch.bfloat16)
    quantized._fidelity_gate(none, none, None, "affine SwiGLU")


def _constant(n, k, value):
    """MLX affine weights whose every value of column 0 counts: no codes, ``value`` as bias."""
    scales = torch.zeros(n, k // 64, dtype=torch.bfloat16, device="cuda")
    return (torch.zeros(n, k // 8, dtype=torch.int32, device="cuda"), scales,
            torch.full_like(scales, value))


@pytest.mark.gpu
def test_executors_bind_where_the_native_roundings_add_up():
    # a gate of -9.65625 rounds to -9.625: its silu, nearly proportional to exp, is off by 3%
    x = torch.zeros(1, 64, dtype=torch.bfloat16, device="cuda")
    x[0, 0] = 1.609375
    gate, up, down = (_constant(64, 64, v) for v in (-6.0, 1.0234375, 0.25))
    residual = torch.ones(1, 64, dtype=torch.bfloat16, device="cuda")
    hidden = mt.affine_swiglu(x, *gate, *up)
    assert not mt.affine_swiglu_compatible(hidden, mt.native_affine_swiglu(x, *gate, *up))
    assert torch.equal(hidden, native.exact_affine_swiglu(x, *gate, *up))
    execute = mt.mlx_affine_swiglu_executor(x, *gate, *up, autotune=False)
    assert torch.equal(execute(x), hidden)
    execute = mt.mlx_affine_mlp_executor(x, *gate, *up, *down, residual, autotune=False)
    want = native.exact_affine_residual_qmv(hidden, *down, residual)
    assert mt.affine_swiglu_compatible(execute(x, residual), want)
