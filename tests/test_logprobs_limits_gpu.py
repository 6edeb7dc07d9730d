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


def check(x, target, *, temperature=1.0, mask=None):
    """Gradients against 64 bits.  A probability is off by its exponent's rounding, 2^-24 of the
    distance |d| to the maximum a few times, by the sum's (a thread adds v / 64 terms at most) and
    by an lse below 32 as an fp32 number: none of it grows with the logits.  In 16 bits lse may be
    larger, up to a sixteenth of a half step."""
    dt = x.dtype
    u = 0.0 if dt == torch.float32 else torch.finfo(dt).eps / 2
    v = x.shape[-1]
    b, t = target.shape
    ups = [s * (1 + torch.rand(b, t, device="cuda")) for s in (0.3, 0.02, 0.1)]
    live = torch.ones(b, t, dtype=torch.bool, device="cuda") if mask is None else mask
    got = ops.token_logprobs(x, target, temperature=temperature, mask=mask)
    grad = ops.token_logprobs_grad(ups[0], ups[1], x, target, got.lse, got.entropy, up_lse=ups[2],
                                   temperature=temperature, mask=mask)
    x64 = torch.where(live[..., None], x.double(), 0.0)
    d = (x64 - x64.amax(-1, keepdim=True)) / temperature
    logs = d - d.exp().sum(-1, keepdim=True).log()
    p, logs = logs.exp(), logs.clamp(min=-1e4)
    entropy = -(p * logs).sum(-1, keepdim=True)
    one = torch.nn.functional.one_hot(target, v).double()
    a, h, e = (y.double()[..., None] for y in ups)
    want = (a * (one - p) - h * p * (logs + entropy) + e * p) / temperature
    size = (a * (one + p) + h * p * (logs.abs() + entropy) + e * p) / temperature
    mean = (p * d.abs()).sum(-1, keepdim=True)
    rel = (u / 16 + 2.0**-20 + (v / 64 + 64) * U32 + 8 * U32 * d.abs().clamp(max=1e4)) * (2 + mean)
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    # an exponential below 2^-126 becomes zero
    lost = 2.0**-126 * (a + h * (logs.abs() + entropy) + e) / temperature
    past = ((grad.double() - want).abs() - u * want.abs() - rel * size - lost - tiny)[live]
    assert past.max() <= 0, (past.max().item(), want.abs().max().item())
    assert bool((grad[~live] == 0).all())
    leaf = x.detach().clone().requires_grad_()
    auto = ops.token_logprobs(leaf, target, temperature=temperature, mask=mask)
    (auto.logprob * ups[0] + auto.entropy * ups[1] + auto.lse * ups[2]).sum().backward()
    assert torch.equal(leaf.grad, grad)


CASES = [(2, 3, 1, "fp32"), (1, 5, 7, "bf16"), (2, 9, 513, "fp32"), (1, 4, 4097, "fp16"), (1, 2, 50257, "fp32"),
         (4, 300, 1000, "fp32"), (3, 500, 33000, "fp32"), (2, 700, 40001, "bf16"), (1, 1, 262144, "fp32")]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("offset", [-3e5, 40.0, 1e4, 1e6])
def test_logits_with_a_common_offset(case, offset):
    b, t, v, dt = case
    gen = torch.Generator(device="cuda").manual_seed(stable_seed((case, offset)))
    x = 3 * torch.randn(b, t, v, generator=gen, device="cuda")
    if dt == "fp16":
        offset = max(-3e4, min(offset, 3e4))
    x = (x + offset * (1 + torch.rand(b, t, 1, generator=gen, device="cuda"))).to(DT[dt])
    target = torch.randint(0, v, (b, t), generator=gen, device="cuda")
    mask = torch.rand(b, t, generator=gen, device="cuda") < 0.9 if t > 1 else None
    check(x, target, mask=mask)


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("temperature", [0.01, 1e-4, 1e-29])
def test_small_temperatures(case, temperature):
    b, t, v, dt = case
    gen = torch.Generator(device="cuda").manual_seed(stable_seed((case, temperature)))
    x = (3 * torch.randn(b, t, v, generator=gen, device="cuda")).to(DT[dt])
    if temperature < 1e-20:  # gradients of 1e28, infinite in fp16; lse passes fp32's range
        x = x * 1e10 if dt != "fp16" else x
    target = torch.randint(0, v, (b, t), generator=gen, device="cuda")
    if dt == "fp16" and temperature < 1e-3:
        return
    # The rounding of 1 / temperature is relative in every exponent, as check() has it.
    check(x, target, temperature=temperature)


@pytest.mark.parametrize("v,rows", [(7, 3), (50, 1100), (3000, 2), (30000, 300)])
@pytest.mark.parametrize("dt", DT)
def test_rows_of_a_types_lowest_value(v, rows, dt):
    """All equal, however large: probabilities of 1 / v; and half of them infinitely far below."""
    x = torch.full((1, rows, v), torch.finfo(DT[dt]).min, dtype=DT[dt], device="cuda")
    check(x, torch.randint(0, v, (1, rows), device="cuda"))
    y = torch.full((1, rows, v), -float("inf"), dtype=DT[dt], device="cuda")
    y[..., : (v + 1) // 2] = torch.finfo(DT[dt]).min
    got = ops.token_logprobs(y, torch.zeros(1, rows, dtype=torch.int64, device="cuda"))
    one = torch.ones(1, rows, device="cuda")
    grad = ops.token_logprobs_grad(None, None, y, torch.zeros(1, rows, dtype=torch.int64, device="cuda"), got.lse,
                                   got.entropy, up_lse=one).float()
    n = (v + 1) // 2
    u = 0.0 if dt == "fp32" else torch.finfo(DT[dt]).eps / 2
    assert ((grad[..., :n] * n - 1).abs() <= u + 2.0**-20 + (2.0**-25 * n if dt == "fp16" else 0)).all()
    assert (grad[..., n:] == 0).all()


def test_rows_with_nan_and_infinities_stay_nan():
    x = torch.randn(1, 5, 3000, device="cuda") + 1e4
    x[0, 1, 100], x[0, 2, 100], x[0, 3] = float("nan"), float("inf"), -float("inf")
    target = torch.ones(1, 5, dtype=torch.int64, device="cuda")
    got = ops.token_logprobs(x, target)
    grad = ops.token_logprobs_grad(torch.ones(1, 5, device="cuda"), None, x, target, got.lse, got.entropy)
    # an entry infinitely far below +inf has no probability, whatever the others are
    assert bool(grad[0, [1, 3]].isnan().all()) and bool(grad[0, 2, 100].isnan())
    assert bool(grad[0, [0, 4]].isfinite().all())
