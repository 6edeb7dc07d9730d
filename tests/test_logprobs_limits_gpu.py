"""Token log probabilities of logits at the ends of their types' ranges (``csrc/logprobs.hip``)."""

from __future__ import annotations

import pytest
import torch

from conftest import stable_seed
from dattri_llm_amd.gradient import ops

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U32 = 2.0**-24


@pytest.mark.parametrize("v,rows", [(9, 2), (50, 1100), (513, 3), (3000, 1100), (5000, 3), (50257, 2), (60000, 300)])
@pytest.mark.parametrize("kept", ["first", "last", "some", "one"])
@pytest.mark.parametrize("dt", DT)
def test_vocabularies_masked_by_a_types_lowest_value(v, rows, kept, dt):
    """Most tokens are barred by their type's lowest value, a thread's, a wave's or a part's whole
    share among them: everything is that of the tokens that are left."""
    gen = torch.Generator(device="cuda").manual_seed(stable_seed((v, rows, kept)))
    x = torch.randn(1, rows, v, generator=gen, device="cuda").to(DT[dt])
    at = torch.arange(v, device="cuda")
    keep = {"first": at < max(1, v // 50), "last": at >= v - max(1, v // 50), "some": at % 97 == 5, "one": at == v // 2}[kept]
    x = x.masked_fill(~keep, torch.finfo(DT[dt]).min)
    target = keep.nonzero()[:, 0][torch.randint(0, int(keep.sum()), (1, rows), generator=gen, device="cuda")]
    got = ops.token_logprobs(x, target, top=1)
    z = x[..., keep].double()
    logs = z.log_softmax(-1)
    lse, entropy = z.logsumexp(-1), -(logs.exp() * logs).sum(-1)
    logprob = x.double().gather(-1, target[..., None])[..., 0] - lse
    # Sums of 32-bit exponentials, v / 64 + 48 of them in a row at most; exponents of up to 12.
    off = (v / 64 + 48) * U32 + 64 * U32
    for name, y, want in (("logprob", got.logprob, logprob), ("entropy", got.entropy, entropy), ("lse", got.lse, lse)):
        assert bool(((y.double() - want).abs() <= off * (2 + want.abs() + entropy)).all()), name
    up = torch.ones(1, rows, device="cuda")
    grad = ops.token_logprobs_grad(up, up, x, target, got.lse, got.entropy)
    assert bool(grad.isfinite().all()) and bool((grad[..., ~keep] == 0).all())
