"""Log probabilities of given tokens against the formulas in 64 bits (``csrc/logprobs.hip``)."""

from __future__ import annotations

import math

import pytest
import torch

from conftest import stable_seed
from dattri_llm_amd.gradient import ops

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U32 = 2.0**-24


def half_step(dt):
    return torch.finfo(dt).eps / 2


def assert_near(got, want, off):
    past = (got.double() - want).abs() - off
    at = past.argmax() if past.numel() else None
    assert at is None or past.flatten()[at] <= 0, (
        f"entry {at.item()} of {tuple(got.shape)}: {got.flatten()[at].item()!r} for {want.flatten()[at].item()!r}, "
        f"{past.flatten()[at].item():.3e} past its bound")


def ordered(x, k):
    """The k largest of each row: by value, of equal ones the lower index."""
    return torch.sort(x.double() + 0.0, dim=-1, descending=True, stable=True).indices[..., :k]


def check(x, target, *, mask=None, temperature=1.0, top=0, up=(0.3, 0.02, 0.1)):
    """Everything of one call against 64 bits, gradients too."""
    dt = x.dtype
    v = x.shape[-1]
    live = torch.ones(target.shape, dtype=torch.bool, device="cuda") if mask is None else mask != 0
    got = ops.token_logprobs(x, target, mask=mask, temperature=temperature, top=top)
    clean = torch.where(live[..., None], x.double(), 0)
    z = clean / temperature
    logs = torch.log_softmax(z, -1)
    p = logs.exp()
    plogp = torch.special.xlogy(p, p)
    entropy = -plogp.sum(-1)
    lse = torch.logsumexp(z, -1)
    named = (target >= 0) & (target < v) & live
    at = target.clamp(0, v - 1)[..., None]
    logprob = torch.where(named, logs.gather(-1, at)[..., 0], 0)
    # A thread adds at most v / 64 + 32 terms (v / 512 in wide rows), then their tree of at
    # most 15: a relative error of the sum, absolute in its logarithm.  The exponents are
    # rounded by 2^-24 of their size twice, which the weighted sums feel at the mean size.
    sums = (v / (64 if v <= 4096 else 512) + 48) * U32
    mean = (p * (z - z.amax(-1, keepdim=True)).abs().clamp(max=1e4)).sum(-1)
    near = sums + 4 * U32 * mean
    scale = lambda y: 4 * U32 * torch.where(y.isfinite(), y.abs(), 0)  # noqa: E731
    assert_near(got.lse[live], lse[live], (near + scale(lse))[live])
    finite = logprob.isfinite()
    assert torch.equal(got.logprob.isfinite(), finite)
    assert_near(got.logprob[live & finite], logprob[live & finite], (near + scale(logprob))[live & finite])
    assert_near(got.entropy[live], entropy[live], (near * (2 + mean) + scale(entropy))[live])
    for y in (got.logprob, got.entropy, got.lse):
        assert y.dtype == torch.float32 and y.shape == target.shape and (y[~live] == 0).all()
    if top:
        index = ordered(clean, top)
        assert torch.equal(got.top_index, torch.where(live[..., None], index, -1))
        want = torch.where(live[..., None], logs.gather(-1, index), 0)
        ok = want.isfinite()
        assert torch.equal(got.top_logprob.isfinite(), ok)
        assert_near(got.top_logprob[ok], want[ok], (near[..., None] + scale(want))[ok])
    else:
        assert got.top_logprob is None and got.top_index is None

    ups = [None if u is None else u * (1 + torch.rand(target.shape, device="cuda")) for u in up]
    grad = ops.token_logprobs_grad(ups[0], ups[1], x, target, got.lse, got.entropy, up_lse=ups[2], mask=mask,
                                   temperature=temperature)
    u, h, e = (torch.zeros(target.shape, dtype=torch.float64, device="cuda") if y is None else y.double() for y in ups)
    u = torch.where(named, u, 0)[..., None]
    want = p * (e[..., None] - u) - h[..., None] * (plogp + p * entropy[..., None])
    size = p * (e[..., None].abs() + u.abs()) + h[..., None] * (plogp.abs() + p * entropy[..., None])
    want.scatter_add_(-1, at, u)
    size.scatter_add_(-1, at, u.abs())
    want, size = torch.where(live[..., None], want, 0) / temperature, torch.where(live[..., None], size, 0) / temperature
    # p from lse: its error (as above, and the rounding of lse and of the difference) is relative in p.
    rel = (near + scale(lse) + 16 * U32)[..., None] + 4 * U32 * (z - lse[..., None]).abs().clamp(max=1e4)
    rel = rel * (2 + mean[..., None])
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps  # half a step of the smallest values
    assert grad.dtype == dt and grad.shape == x.shape and grad.is_contiguous()
    assert_near(grad, want, half_step(dt) * want.abs() + rel * size + tiny)
    return got, grad


CASES = [  # b, t, v, dtype, top, temperature, masked
    (2, 3, 1, "fp32", 1, 1.0, False),
    (2, 3, 7, "bf16", 5, 1.0, False),
    (3, 5, 64, "fp16", 32, 0.7, True),
    (2, 9, 513, "bf16", 20, 1.0, True),
    (1, 4, 4095, "bf16", 3, 2.0, False),
    (1, 3, 4097, "bf16", 32, 1.0, False),
    (2, 2, 2049, "fp32", 32, 1.0, True),
    (1, 1, 50257, "bf16", 20, 0.7, False),
    (2, 5, 50257, "fp32", 5, 1.0, True),
    (4, 100, 32000, "bf16", 20, 1.0, True),
    (1, 300, 32003, "fp16", 7, 1.3, True),
    (1, 1, 262144, "fp32", 32, 1.0, False),
    (1, 290, 9001, "bf16", 0, 1.0, False),
    (7, 1, 151936, "bf16", 1, 1.0, False),
    # many short rows
    (4, 300, 1, "fp32", 1, 1.0, False),
    (2, 520, 7, "bf16", 5, 1.0, True),
    (3, 350, 513, "bf16", 20, 1.3, True),
    (1, 1100, 4097, "fp16", 32, 1.0, False),
    (4, 256, 8191, "fp32", 32, 0.7, True),
    (2, 600, 16385, "bf16", 0, 1.0, True),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_against_64_bits(case):
    b, t, v, dt, top, temperature, masked = case
    gen = torch.Generator(device="cuda").manual_seed(stable_seed(case))
    x = (3 * torch.randn(b, t, v, generator=gen, device="cuda")).to(DT[dt])
    target = torch.randint(0, v, (b, t), generator=gen, device="cuda")
    target[0, 0] = -100
    if t > 1:
        target[0, 1] = v  # outside too
    mask = None
    if masked:
        mask = torch.rand(b, t, generator=gen, device="cuda") < 0.8
        x = x.masked_fill(~mask[..., None], float("nan"))
    check(x, target, mask=mask, temperature=temperature, top=top)


@pytest.mark.parametrize("v", [100, 5000, 40000])
@pytest.mark.parametrize("layout", ["wide", "swapped", "strided", "flat"])
def test_strides(v, layout):
    gen = torch.Generator(device="cuda").manual_seed(v)
    b, t = 2, 6
    if layout == "wide":
        x = torch.randn(b, t, v + 5, generator=gen, device="cuda").bfloat16()[..., 3:v + 3]
    elif layout == "swapped":
        x = torch.randn(t, b, v, generator=gen, device="cuda").bfloat16().transpose(0, 1)
    elif layout == "strided":
        x = torch.randn(b, t, v, 2, generator=gen, device="cuda").bfloat16()[..., 1]
    else:
        x = torch.randn(b * t, v, generator=gen, device="cuda").bfloat16()
    target = torch.randint(0, v, (b, 2 * t), generator=gen, device="cuda")[:, ::2]
    mask = (torch.rand(b, 2 * t, generator=gen, device="cuda") < 0.8)[:, 1::2]
    if layout == "flat":
        target, mask = target.reshape(-1), mask.reshape(-1)
    check(x, target, mask=mask, top=4)


@pytest.mark.parametrize("v,rows", [(50, 4), (50, 1100), (3000, 2), (3000, 1100), (30000, 300), (60000, 3)])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "two_values", "few_finite", "lowest", "signed_zeros"])
def test_orders_that_try_the_alternatives(v, rows, kind):
    """Ties in every place, sorted rows (more entries than fit reach the bound), rows of -inf and of a type's lowest value."""
    x = torch.zeros(1, rows, v, device="cuda")
    if kind == "rising":
        x = (torch.arange(v, device="cuda") / v * 50).expand(1, rows, v)
    elif kind == "falling":
        x = (torch.arange(v, 0, -1, device="cuda") / v * 50).expand(1, rows, v)
    elif kind == "two_values":
        x = (torch.rand(1, rows, v, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) < 0.5).float()
    elif kind == "few_finite":
        x = torch.full((1, rows, v), -math.inf, device="cuda")
        x[..., v // 2::7] = 1.0
    elif kind == "lowest":
        x = torch.full((1, rows, v), torch.finfo(torch.float32).min, device="cuda")
    elif kind == "signed_zeros":
        x = torch.where(torch.arange(v, device="cuda") % 2 == 0, -0.0, 0.0).expand(1, rows, v)
    target = torch.randint(0, v, (1, rows), device="cuda")
    for dt in (torch.float32, torch.bfloat16):
        y = x.to(dt) if kind != "lowest" else torch.full(x.shape, torch.finfo(dt).min, dtype=dt, device="cuda")
        check(y.contiguous(), target, top=min(32, v))


def test_an_unlikely_and_a_certain_target():
    x = torch.full((1, 2, 1000), -40.0, device="cuda")
    x[..., 5] = 30.0
    target = torch.tensor([[5, 6]], device="cuda")
    got, _ = check(x, target, top=2)
    assert got.logprob[0, 0] == 0 and abs(got.logprob[0, 1].item() + 70) < 1e-4
    x[0, 1, 6] = -math.inf  # a target without probability
    assert check(x, target)[0].logprob[0, 1] == -math.inf


def test_nan_stays_in_its_row():
    x = torch.randn(1, 3, 9000, device="cuda")
    clean = ops.token_logprobs(x, torch.ones(1, 3, dtype=torch.int64, device="cuda"), top=3)
    x[0, 1, 100] = float("nan")
    got = ops.token_logprobs(x, torch.ones(1, 3, dtype=torch.int64, device="cuda"), top=3)
    for a, b in zip(got, clean):
        assert torch.equal(a[0, [0, 2]], b[0, [0, 2]])
    assert got.logprob[0, 1].isnan() and got.lse[0, 1].isnan()
    x[0, 1] = float("nan")
    got = ops.token_logprobs(x, torch.ones(1, 3, dtype=torch.int64, device="cuda"), top=3)
    assert got.top_logprob[0, 1].isnan().all()


def test_autograd_gives_the_plain_calls_gradients():
    x = torch.randn(2, 30, 777, device="cuda", requires_grad=True)
    target = torch.randint(-1, 777, (2, 30), device="cuda")
    mask = torch.rand(2, 30, device="cuda") < 0.9
    a, b, c = (torch.randn(2, 30, device="cuda") for _ in range(3))
    got = ops.token_logprobs(x, target, mask=mask, temperature=0.9, top=3)
    assert not got.top_logprob.requires_grad
    ((got.logprob * a).sum() + (got.entropy * b).sum() + (got.lse * c).sum()).backward()
    want = ops.token_logprobs_grad(a, b, x.detach(), target, got.lse.detach(), got.entropy.detach(), up_lse=c, mask=mask,
                                   temperature=0.9)
    assert torch.equal(x.grad, want)
    # a sum's gradient is broadcast (strides of zero); the other outputs are not used
    x.grad = None
    got = ops.token_logprobs(x, target, mask=mask)
    got.logprob.sum().backward()
    want = ops.token_logprobs_grad(torch.ones(2, 30, device="cuda"), None, x.detach(), target, got.lse.detach(),
                                   got.entropy.detach(), mask=mask)
    assert torch.equal(x.grad, want)
    # rows without samples
    x.grad = None
    flat = ops.token_logprobs(x.flatten(0, 1), target.flatten(), mask=mask.flatten())
    flat.logprob.sum().backward()
    assert torch.equal(x.grad, want)


@pytest.mark.parametrize("up", [(0.3, None, None), (None, 0.1, None), (None, None, 0.2)])
def test_single_gradients(up):
    x = torch.randn(2, 5, 600, device="cuda")
    check(x, torch.randint(0, 600, (2, 5), device="cuda"), up=up)


def test_gradient_by_differences():
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(1, 3, 40, generator=gen, device="cuda")
    target = torch.tensor([[1, 7, 39]], device="cuda")
    got = ops.token_logprobs(x, target, temperature=0.8)
    one = torch.ones(1, 3, device="cuda")
    grad = ops.token_logprobs_grad(one, 0.5 * one, x, target, got.lse, got.entropy, up_lse=2 * one, temperature=0.8)
    for i in (0, 1, 7, 20, 39):  # a step of 2^-6, its square times third derivatives of order 1, 2^-22 over the step
        d = torch.zeros(40, device="cuda")
        d[i] = 2.0**-6
        f = [ops.token_logprobs(x + s * d, target, temperature=0.8) for s in (1, -1)]
        hi, lo = (y.logprob + 0.5 * y.entropy + 2 * y.lse for y in f)
        assert torch.allclose((hi - lo) * 2.0**5, grad[..., i], atol=2e-3)


def test_captured_calls_replay_the_eager_results():
    x = torch.randn(4, 1, 70001, device="cuda").bfloat16()
    target = torch.randint(0, 70001, (4, 1), device="cuda")
    up = torch.randn(4, 1, device="cuda")

    def call():
        a = ops.token_logprobs(x, target, top=9)
        return *a, ops.token_logprobs_grad(up, up, x, target, a.lse, a.entropy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = call()
    for k in range(3):
        x.copy_(3 * torch.randn(4, 1, 70001, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, call())), k


def test_empty_inputs():
    for b, t in ((0, 4), (3, 0)):
        x = torch.zeros(b, t, 8, device="cuda")
        target = torch.zeros(b, t, dtype=torch.int64, device="cuda")
        got = ops.token_logprobs(x, target, top=2)
        assert got.top_index.shape == (b, t, 2)
        assert ops.token_logprobs_grad(got.lse, None, x, target, got.lse, got.entropy).shape == (b, t, 8)
