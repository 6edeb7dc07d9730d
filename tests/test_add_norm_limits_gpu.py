"""Residual addition with RMS norm into 8 bits: the quotient by the scale (``csrc/addnorm.hip``)."""

from __future__ import annotations

import pytest
import torch

from conftest import stable_seed
from dattri_llm_amd.gradient import ops

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FP8 = torch.float8_e4m3fn


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("quantize", ["row", "block"])
@pytest.mark.parametrize("d", [128, 1024, 4096, 5120])
@pytest.mark.parametrize("size", [2.0**-90, 1e-3, 1.0, 1e20])
def test_entries_half_way_between_two_values(dt, quantize, d, size):
    """Rows of +-1 have a norm of 1, so that out is the weight: products of a scale with numbers
    half way between 8-bit ones.  Scale and quotient are fp32's to the last bit, and so is what
    the quotients round to."""
    gen = torch.Generator(device="cuda").manual_seed(stable_seed((d, quantize)))
    values = torch.arange(256, dtype=torch.uint8, device="cuda").view(FP8).float()
    values = values[values.isfinite() & (values >= 0)].sort().values
    half_way = (values[1:] + values[:-1]) / 2
    runs = d // 128
    w = half_way[torch.randint(0, len(half_way), (runs, 128), generator=gen, device="cuda")]
    w[:, 0] = 448.0
    scale = size * (1 + torch.rand(runs if quantize == "block" else 1, 1, generator=gen, device="cuda"))
    w = (w * scale).flatten()
    x = torch.where(torch.rand(2, 9, d, generator=gen, device="cuda") < 0.5, -1.0, 1.0)
    got = ops.add_rms_norm(x.to(DT[dt]), None, w, eps=0.0, quantize=quantize)
    most = w.view(-1, 128 if quantize == "block" else d).abs().amax(-1).cpu()
    want_scale = most / 448
    want = (x.cpu() * w.cpu()).view(2, 9, len(most), -1) / want_scale[:, None]
    scales = got.scales.cpu() if quantize == "block" else got.scales.cpu()[..., None]
    assert torch.equal(scales, want_scale.expand_as(scales))
    assert torch.equal(got.out.cpu().view(torch.uint8), want.flatten(2).to(FP8).view(torch.uint8))


@pytest.mark.parametrize("quantize", ["row", "block"])
@pytest.mark.parametrize("d", [128, 1000])
def test_zeros_and_infinities_in_8_bits(quantize, d):
    """Zeros keep their sign; beside an infinite weight its run's finite entries are zero."""
    w = torch.randn(d, device="cuda")
    w[3], w[5] = 0.0, -0.0
    x = torch.ones(1, 2, d, device="cuda")
    x[0, 1] = -1
    got = ops.add_rms_norm(x, None, w, eps=0.0, quantize=quantize).out[0, :, [3, 5]].view(torch.uint8)
    assert got.tolist() == [[0, 128], [128, 0]]
    w[7] = float("inf")
    got = ops.add_rms_norm(x, None, w, eps=0.0, quantize=quantize)
    out, scales = got.out.float()[0], got.scales[0]
    run = slice(0, d if quantize == "row" else 128)
    assert bool(out[:, 7].isnan().all()) and bool((scales[..., 0] if quantize == "block" else scales).isinf().all())
    rest = torch.arange(d, device="cuda") != 7
    assert bool((out[:, run][:, rest[run]] == 0).all()) and bool(out[:, rest].isfinite().all())
    if quantize == "block" and d > 128:
        assert bool(out[:, 128:].any())
