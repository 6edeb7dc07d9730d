"""Router balance and z losses, counts and gradients, against fp64.

Bounds.  A probability is an exponential, a sum of at most 1024 terms (16 in a
lane, 6 butterfly steps) and a division: below 40 * 2^-24 = 2.4e-6 relative, and
as much again for the logits' difference from their largest (up to 30 here).  A
mean over n tokens is a chain of at most 64 of them in a wave and the chunks'
partials, all positive: below 1e-5 in all for the sizes here (TIGHT_FP32).  A
gradient is a difference of terms of the sizes up (E/n) p (f + sum f p) and
up_z (2/n) |logsumexp| p: within 1e-5 of those, plus half a step of its type.
"""

from __future__ import annotations

import pytest
import torch

from conftest import HALF_ULP, TIGHT_FP32
from dattri_llm_amd.gradient import ops

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NAME = {torch.float32: "float32", torch.bfloat16: "bfloat16", torch.float16: "float16"}


def plain(x, index, mask):
    """(loss, z, counts, live) in fp64; x (B, T, E), index (B, T, k)."""
    e = x.shape[-1]
    n = mask.double().sum(1)
    part = (torch.nn.functional.one_hot(index.clamp(0, e - 1), e) * ((index >= 0) & (index < e))[..., None]).sum(2)
    counts = (part * mask[..., None]).sum(1)
    inv = torch.where(n > 0, 1 / n.clamp(min=1), 0.0)
    x = torch.where(mask[..., None], x, 0.0)
    mean = (torch.softmax(x, -1) * mask[..., None]).sum(1) * inv[:, None]
    loss = e * (counts.double() * inv[:, None] * mean).sum(-1)
    z = (torch.logsumexp(x, -1).square() * mask).sum(1) * inv
    return loss, z, counts, n


def check(x, index, mask, device, rows=None):
    b, t, e = x.shape
    dt = x.dtype
    gen = torch.Generator().manual_seed(9)
    up, up_z = torch.randn(b, generator=gen), torch.randn(b, generator=gen)
    live = torch.ones(b, t, dtype=torch.bool) if mask is None else mask
    dev_x = x.to(device) if rows is None else rows(x.to(device))
    dev_mask = None if mask is None else mask.to(device)
    got = ops.moe.balance_loss(dev_x, index.to(device), mask=dev_mask)
    grad = ops.moe.balance_loss_grad(up.to(device), up_z.to(device), dev_x, got.counts, got.live, mask=dev_mask)
    xd = torch.where(live[..., None], x.double(), 0.0).requires_grad_()
    loss, z, counts, n = plain(xd, index, live)
    (loss * up.double()).sum().add((z * up_z.double()).sum()).backward()
    assert torch.equal(got.counts.cpu().long(), counts) and torch.equal(got.live.cpu().double(), n)
    assert bool(((got.loss.cpu().double() - loss).abs() <= TIGHT_FP32 * loss).all())
    size = xd.detach().abs().amax(-1) + torch.logsumexp(xd.detach(), -1).abs()
    inv = torch.where(n > 0, 1 / n.clamp(min=1), 0.0)
    assert bool(((got.z_loss.cpu().double() - z).abs() <= TIGHT_FP32 * (size.square() * live).sum(1) * inv).all())
    p = torch.softmax(xd.detach(), -1)
    f = (counts * inv[:, None])[:, None]
    scale = inv[:, None, None] * p * (e * up.double().abs()[:, None, None] * (f + (f * p).sum(-1, keepdim=True))
                                      + 2 * up_z.double().abs()[:, None, None] * size[..., None])
    tol = TIGHT_FP32 * scale + HALF_ULP.get(NAME[dt], 0.0) * xd.grad.abs()
    # below the least normal value of a type the step no longer shrinks
    tol = tol + {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -140}[dt]
    assert grad.dtype == dt and grad.shape == x.shape
    off = (grad.cpu().double() - xd.grad).abs()
    assert bool((off <= tol).all()), (off / tol).max()
    assert not grad.cpu()[~live].any()
    return got, grad


def make(b, t, e, k, dt, seed=0, scale=2.0):
    gen = torch.Generator().manual_seed(seed)
    x = (scale * torch.randn(b, t, e, generator=gen)).to(dt)
    return x, torch.topk(x.float(), k, dim=-1).indices


SIZES = [(1, 1, 1, 1), (1, 1, 8, 2), (3, 1, 128, 8), (2, 7, 2, 1), (4, 64, 8, 2), (5, 65, 16, 4), (2, 300, 64, 6),
         (1, 1000, 8, 2), (2, 129, 128, 8), (1, 515, 256, 8), (3, 40, 60, 4), (2, 33, 65, 3), (1, 70, 129, 2),
         (2, 20, 257, 8), (1, 9, 1000, 16), (1, 3, 1024, 70), (64, 3, 8, 2), (1, 5000, 5, 2), (700, 1, 8, 2)]


@pytest.mark.parametrize("dt", DTYPES, ids=NAME.get)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_matches_fp64(size, dt, device):
    x, index = make(*size, dt, seed=size[1])
    check(x, index, None, device)


@pytest.mark.parametrize("dt", DTYPES, ids=NAME.get)
@pytest.mark.parametrize("size", [(4, 50, 8, 2), (5, 130, 128, 8), (4, 1, 8, 2), (4, 700, 33, 3)], ids=str)
def test_masked_tokens_take_no_part_whatever_they_hold(size, dt, device):
    x, index = make(*size, dt)
    mask = torch.rand(size[:2], generator=torch.Generator().manual_seed(4)) < 0.6
    mask[0], mask[1] = False, True
    bad = torch.tensor([float("nan"), float("inf"), float("-inf")])[torch.randint(0, 3, x.shape)].to(dt)
    x = torch.where(mask[..., None], x, bad)
    got, grad = check(x, index, mask, device)
    assert float(got.loss[0]) == 0 and float(got.z_loss[0]) == 0 and not grad[0].any()
    for m in (mask.to(torch.uint8), mask.long(), mask.t().contiguous().t()):
        again = ops.moe.balance_loss(x.to(device), index.to(device), mask=m.to(device))
        assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_closed_experts_and_extreme_logits(device):
    """-inf closes an expert; a wide spread of logits neither overflows nor loses the largest."""
    x, index = make(2, 30, 16, 2, torch.float32)
    x[0, 3] = torch.linspace(-300, 300, 16)
    x[1, 4] = 88.0
    x[..., 5] = float("-inf")
    index = torch.topk(x, 2, dim=-1).indices
    xd = x.double()
    got = ops.moe.balance_loss(x.to(device), index.to(device))
    n, part = 30, torch.nn.functional.one_hot(index, 16).sum(2).sum(1).double() / 30
    want = 16 * (part * torch.softmax(xd, -1).mean(1)).sum(-1)
    assert bool(((got.loss.cpu() - want).abs() <= TIGHT_FP32 * want).all())
    z = torch.logsumexp(xd, -1).square().mean(1)
    assert bool(((got.z_loss.cpu() - z).abs() <= TIGHT_FP32 * z).all()) and n == 30
    up = torch.ones(2, device=device)
    grad = ops.moe.balance_loss_grad(up, up, x.to(device), got.counts, got.live)
    assert bool(torch.isfinite(grad).all()) and not grad[..., 5].any()
    x[1, 0] = float("-inf")  # no expert open: no softmax, and it says so, for its sample alone
    got = ops.moe.balance_loss(x.to(device), index.to(device))
    assert bool(torch.isnan(got.loss[1])) and bool(torch.isfinite(got.loss[0]))


@pytest.mark.parametrize("dt", DTYPES, ids=NAME.get)
@pytest.mark.parametrize("experts", [8, 33])
def test_tokens_whose_logits_are_all_filled(dt, experts, device):
    """A token all of whose experts hold one large fill value, the type's lowest
    among them, is spread evenly; beside an ordinary logit a fill has no weight."""
    big = float(torch.finfo(dt).max)
    fills = [-big, big, -min(1e30, big / 2), min(1e12, big / 4), -min(1e9, big / 8)]
    for fill in fills:
        x, index = make(2, 12, experts, 2, dt)
        x[:, 3:6] = fill
        if fill < 0:
            x[0, 7, 1:] = fill
            x[1, 8, :-1] = fill
        dev_x, dev_index = x.to(device), index.to(device)
        got = ops.moe.balance_loss(dev_x, dev_index)
        up = torch.tensor([1.0, -0.5])
        grad = ops.moe.balance_loss_grad(up.to(device), None, dev_x, got.counts, got.live)
        xd = x.double().requires_grad_()
        loss, z, counts, n = plain(xd, index, torch.ones(2, 12, dtype=torch.bool))
        (loss * up.double()).sum().backward()
        assert torch.equal(got.counts.cpu(), counts) and torch.equal(got.live.cpu().double(), n)
        assert bool(((got.loss.cpu().double() - loss).abs() <= TIGHT_FP32 * loss).all()), fill
        square = (xd.detach().abs().amax(-1) ** 2).amax()
        if square < 3e38:  # else fp32 holds no such square
            assert bool(((got.z_loss.cpu().double() - z).abs() <= TIGHT_FP32 * z).all()), fill
        else:
            assert bool(torch.isinf(got.z_loss).all()), fill
        # terms up (E/n) p f: p <= 1, f <= 1
        tol = TIGHT_FP32 * experts / 12 + HALF_ULP.get(NAME[dt], 0.0) * xd.grad.abs() + 2.0 ** -25
        assert bool(((grad.cpu().double() - xd.grad).abs() <= tol).all()), fill


def test_dropped_and_repeated_choices(device):
    x, index = make(2, 40, 8, 3, torch.float32)
    index[0, :10, 0] = -1  # dropped
    index[0, 10:20, 1] = 8  # not an expert
    index[1, :5] = 6  # one expert three times
    index[1, 7, 2] = 1 << 40
    check(x, index, None, device)


@pytest.mark.parametrize("experts", [8, 128, 60])
def test_row_strides(experts, device):
    x, index = make(3, 50, experts, 2, torch.bfloat16)

    def wide(v):  # rows of a wider buffer from an odd place
        big = torch.full((*v.shape[:2], experts + 5), float("nan"), dtype=v.dtype, device=v.device)
        big[..., 1:1 + experts] = v
        return big[..., 1:1 + experts]

    plain_got, _ = check(x, index, None, device)
    got, _ = check(x, index, None, device, rows=wide)
    assert torch.equal(plain_got.counts, got.counts) and torch.equal(plain_got.live, got.live)


def test_one_loss_over_the_batch_and_even_load(device):
    x, index = make(4, 32, 8, 2, torch.float32)
    flat = ops.moe.balance_loss(x.view(-1, 8).to(device), index.view(-1, 2).to(device))
    one = ops.moe.balance_loss(x.view(1, 128, 8).to(device), index.view(1, 128, 2).to(device))
    assert flat.loss.shape == (1,) and all(torch.equal(a, b) for a, b in zip(flat, one))
    even = ops.moe.balance_loss(torch.zeros(1, 8, 8, device=device),
                                torch.arange(8, device=device).view(1, 8, 1).expand(1, 8, 2) % 8)
    assert float(even.loss) == 2.0 and even.counts.unique().tolist() == [2]


def test_router_topk_feeds_it(device):
    x, _ = make(2, 100, 128, 8, torch.float32)
    _, index = ops.moe.router_topk(x.to(device), 8)
    check(x, index.view(2, 100, 8).cpu(), None, device)


def test_empty(device):
    got = ops.moe.balance_loss(torch.zeros(2, 0, 8, device=device), torch.zeros(2, 0, 2, dtype=torch.int64, device=device))
    assert got.loss.tolist() == [0, 0] and got.z_loss.tolist() == [0, 0] and not got.counts.any() and not got.live.any()
    assert ops.moe.balance_loss_grad(None, None, torch.zeros(2, 0, 8, device=device), got.counts, got.live).shape == (2, 0, 8)
    got = ops.moe.balance_loss(torch.zeros(2, 3, 8, device=device), torch.zeros(2, 3, 0, dtype=torch.int64, device=device))
    assert got.loss.tolist() == [0, 0] and got.live.tolist() == [3, 3]


def test_autograd_and_differences(device):
    """Against central differences of the fp64 formula with the choices held (its
    own error: h^2 times a third derivative, below 1e-7 of the terms)."""
    x, index = make(3, 21, 16, 2, torch.float32)
    leaf = x.to(device).requires_grad_()
    got = ops.moe.balance_loss(leaf, index.to(device))
    up = torch.tensor([1.0, -2.0, 0.5])
    ((got.loss * up.to(device)).sum() + 0.1 * got.z_loss.sum()).backward()
    assert not got.counts.requires_grad and leaf.grad.shape == leaf.shape
    gen = torch.Generator().manual_seed(8)
    mask = torch.ones(3, 21, dtype=torch.bool)

    def total(v):
        loss, z, _, _ = plain(v, index, mask)
        return ((loss * up.double()).sum() + 0.1 * z.sum()).item()

    for _ in range(3):
        v = torch.randn(x.shape, generator=gen, dtype=torch.float64)
        h = 1e-4
        diff = (total(x.double() + h * v) - total(x.double() - h * v)) / (2 * h)
        terms = leaf.grad.cpu().double() * v
        assert abs(diff - terms.sum().item()) <= 2e-5 * terms.abs().sum().item()
    # one loss alone: the other's gradient is absent, not zero tensors the caller has to make
    leaf.grad = None
    ops.moe.balance_loss(leaf, index.to(device)).z_loss.sum().backward()
    only = leaf.grad.clone()
    want = ops.moe.balance_loss_grad(None, torch.ones(3, device=device), x.to(device), got.counts, got.live)
    assert torch.equal(only, want)


def test_two_streams_and_a_graph(device):
    x, index = make(4, 300, 128, 8, torch.bfloat16)
    x, index = x.to(device), index.to(device)
    up = torch.ones(4, device=device)

    def call():
        got = ops.moe.balance_loss(x, index)
        return (*got, ops.moe.balance_loss_grad(up, up, x, got.counts, got.live))

    want = call()
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(2)]:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(call())
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(want, r))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = call()
    for i in range(4):
        x.copy_(torch.randn_like(x))
        index.copy_(torch.topk(x.float(), 8).indices)
        graph.replay()
        torch.cuda.synchronize()
        want = call()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_transposed_logits_and_offsets_past_32_bits(device):
    x, index = make(1, 3, 16, 2, torch.bfloat16)
    want = ops.moe.balance_loss(x.to(device), index.to(device))
    across = x[0].t().contiguous().to(device).t()  # experts first in memory
    got = ops.moe.balance_loss(across, index[0].to(device))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    far = torch.empty((1 << 33) + 64, dtype=torch.bfloat16, device=device)
    rows = far.as_strided((3, 16), (1 << 32, 1))
    rows.copy_(x[0])
    got = ops.moe.balance_loss(rows, index[0].to(device))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    up = torch.ones(1, device=device)
    assert torch.equal(ops.moe.balance_loss_grad(up, up, rows, got.counts, got.live),
                       ops.moe.balance_loss_grad(up, up, x[0].to(device), got.counts, got.live))


def test_expanded_loss_gradients(device):
    x, index = make(5, 12, 8, 2, torch.float32)
    got = ops.moe.balance_loss(x.to(device), index.to(device))
    one = torch.ones(1, device=device)
    a = ops.moe.balance_loss_grad(one.expand(5), one.double().expand(5), x.to(device), got.counts, got.live)
    b = ops.moe.balance_loss_grad(one.repeat(5), one.repeat(5), x.to(device), got.counts, got.live)
    assert torch.equal(a, b)
