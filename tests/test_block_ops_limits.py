"""Limits of the decoder block operators that need no GPU: refusals on both sides of the C ABI."""

from __future__ import annotations

import pytest
import torch

from dattri_llm_amd import _native as nat
from dattri_llm_amd.gradient import ops

X, OUT = 0x10000, 0x20000  # 16-byte aligned placeholders, never dereferenced


@pytest.mark.parametrize("temperature", [float("inf"), 1e38, 1e300, 1e-31, -float("inf")])
def test_temperatures_without_an_inverse_are_refused(temperature):
    x, t, f = torch.zeros(2, 3, 8), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)
    with pytest.raises(ValueError, match="temperature"):
        ops.token_logprobs(x, t, temperature=temperature)
    with pytest.raises(ValueError, match="temperature"):
        ops.token_logprobs_grad(f, None, x, t, f, f, temperature=temperature)
    lib = nat.load()
    assert lib.da_token_logprobs(X, 2, 2, 3, 8, 24, 8, X, 3, 1, None, 0, 0, temperature, 0, OUT, OUT, OUT, None, None,
                                 None, 0, None) == nat.DA_ERR_INVALID
    assert "temperature" in lib.da_last_error().decode()


def test_ordinary_temperatures_are_taken():
    lib = nat.load()
    for temperature in (1e-29, 0.7, 5e37):
        assert lib.da_token_logprobs(X, 2, 0, 3, 8, 24, 8, X, 3, 1, None, 0, 0, temperature, 0, OUT, OUT, OUT, None, None,
                                     None, 0, None) == nat.DA_OK
