"""Relative position bias by buckets and its per-sample gradient, against fp64.

The forward values are copies of table entries: exact.  A gradient entry sums N
values of g in fp32 in chains of at most N roundings: within N * 2^-24 of the
sum of their sizes, and the chains here are far shorter (a diagonal of at most
q_len entries, then the offsets of a bucket in steps of at most 512).
"""

from __future__ import annotations

import ctypes

import pytest
import torch

from dattri_llm_amd import _native as nat
from dattri_llm_amd.gradient import ops
from test_attention_ops import bucket

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def ids_of(tq, tk, start, buckets, far, both):
    """(tq, tk) buckets on the CPU, one distance at a time."""
    n = buckets // 2 if both else buckets
    rel = torch.arange(tk)[None] - torch.arange(tq)[:, None] - start
    limit = int(rel.abs().max()) if rel.numel() else 0
    side = torch.tensor([bucket(r, n, far) if r <= 2 * far else n - 1 for r in range(limit + 1)])
    if both:
        return rel, side[rel.abs()] + n * (rel > 0)
    return rel, side[(-rel).clamp(min=0)]


SHAPES = [
    # h, tq, tk, start, buckets, far, both, causal
    (1, 1, 1, 0, 32, 128, True, False),
    (3, 1, 9, 8, 32, 128, False, True),
    (4, 1, 4097, 4096, 32, 128, False, True),
    (2, 7, 1, 0, 8, 16, True, False),
    (2, 5, 9, 4, 4, 3, True, False),
    (2, 64, 64, 0, 32, 128, True, False),
    (3, 65, 63, 0, 32, 128, True, False),
    (2, 63, 66, 3, 64, 100, False, True),
    (1, 130, 257, 127, 32, 128, False, True),
    (2, 257, 130, -5, 32, 128, True, False),
    (1, 40, 72, 200, 2, 5, False, False),
    (1, 40, 72, -300, 16, 40, False, True),
    (2, 300, 301, 1, 256, 300, True, False),
    (1, 600, 520, 0, 256, 200, False, False),
    (5, 31, 1031, 1000, 32, 2048, True, False),
    (1, 1100, 24, 0, 32, 128, True, False),
]


@pytest.mark.parametrize("dt", DTYPES, ids=str)
@pytest.mark.parametrize("case", SHAPES, ids=str)
def test_forward_is_exact(case, dt, device):
    h, tq, tk, start, buckets, far, both, causal = case
    table = torch.randn(buckets, h, generator=torch.Generator().manual_seed(1)).to(dt)
    got = ops.relative_bias(table.to(device), tq, tk, q_start=start, bidirectional=both, max_distance=far,
                            causal=causal)
    rel, ids = ids_of(tq, tk, start, buckets, far, both)
    want = table[ids].permute(2, 0, 1)
    if causal:
        want = want.masked_fill(rel > 0, float("-inf"))
    assert got.dtype == dt and torch.equal(got.cpu(), want)


def check_grad(got, g, case, mask=None):
    h, tq, tk, start, buckets, far, both, causal = case
    rel, ids = ids_of(tq, tk, start, buckets, far, both)
    live = torch.ones(g.shape[0], tq, tk, dtype=torch.bool)
    if causal:
        live &= rel <= 0
    if mask is not None:
        live &= mask[:, None, :] & mask[:, start:start + tq, None]
    g = torch.where(live[:, None], g.cpu().double(), 0.0).flatten(2)
    pick = torch.nn.functional.one_hot(ids.flatten(), buckets).double()
    want, size = (g @ pick).transpose(1, 2), (g.abs() @ pick).transpose(1, 2)
    bound = (tq + 512 + 8) * 2.0 ** -24 * size
    assert got.shape == want.shape and got.dtype == torch.float32
    off = (got.cpu().double() - want).abs()
    assert bool((off <= bound).all()), (off - bound).max()


def rows(g, how):
    b, h, tq, tk = g.shape
    if how == "plain":
        return g.contiguous()
    if how == "padded":  # aligned rows of a wider buffer
        big = torch.full((b, h, tq, (tk + 7) // 8 * 8 + 8), float("nan"), dtype=g.dtype, device=g.device)
        big[..., :tk] = g
        return big[..., :tk]
    if how == "odd":  # rows from an odd place, an odd number of entries apart
        big = torch.full((b, h, tq, tk // 2 * 2 + 3), float("nan"), dtype=g.dtype, device=g.device)
        big[..., 1:1 + tk] = g
        return big[..., 1:1 + tk]
    if how == "swapped":  # heads inside the queries
        return g.transpose(1, 2).contiguous().transpose(1, 2)
    if how == "apart":
        return torch.stack([g, g * float("nan")], -1)[..., 0]
    raise AssertionError(how)


@pytest.mark.parametrize("dt", DTYPES, ids=str)
@pytest.mark.parametrize("how", ["plain", "padded", "odd", "swapped", "apart"])
@pytest.mark.parametrize("case", SHAPES, ids=str)
def test_gradient_matches_fp64(case, how, dt, device):
    h, tq, tk, start, buckets, far, both, causal = case
    g = torch.randn(2, h, tq, tk, generator=torch.Generator().manual_seed(tq)).to(dt).to(device)
    if causal:  # what is not read may hold anything
        rel, _ = ids_of(tq, tk, start, buckets, far, both)
        g.masked_fill_((rel > 0).to(device), float("nan"))
    got = ops.relative_bias_grad(rows(g, how), buckets, q_start=start, bidirectional=both, max_distance=far,
                                 causal=causal)
    check_grad(got, g, case)


@pytest.mark.parametrize("extra", range(16))
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=str)
def test_every_row_length_and_offset_of_the_rows(extra, dt, device):
    """All residues of the row length and of the first entry's place."""
    tk = 73 + extra % 8
    case = (1, 70, tk, extra - 8, 32, 64, True, False)
    gen = torch.Generator().manual_seed(extra)
    for first in range(8):
        buf = torch.full((2 * 70 * tk + 16,), float("nan"), dtype=dt)
        g = torch.randn(2, 1, 70, tk, generator=gen).to(dt)
        buf[first:first + g.numel()] = g.flatten()
        view = buf.to(device)[first:first + g.numel()].view(2, 1, 70, tk)
        got = ops.relative_bias_grad(view, 32, q_start=extra - 8, max_distance=64)
        check_grad(got, g, case)


@pytest.mark.parametrize("how", ["plain", "odd"])
@pytest.mark.parametrize("case", [(2, 70, 70, 0, 32, 64, True, False), (3, 33, 80, 47, 32, 128, False, True),
                                  (1, 1, 50, 49, 32, 128, False, True), (1, 140, 300, 100, 16, 64, True, False)], ids=str)
def test_masked_positions_add_nothing_whatever_they_hold(case, how, device):
    h, tq, tk, start, buckets, far, both, causal = case
    gen = torch.Generator().manual_seed(2)
    g = torch.randn(4, h, tq, tk, generator=gen).bfloat16()
    mask = torch.rand(4, tk, generator=gen) < 0.7
    mask[1] = False
    mask[2] = True
    mask[3] = torch.arange(tk) < tk // 2 + 1  # padding at the end
    dead = ~(mask[:, None, None, :] & mask[:, None, start:start + tq, None])
    g = torch.where(dead, torch.tensor([float("nan"), float("inf"), -3.0e38])[torch.randint(0, 3, g.shape, generator=gen)].bfloat16(), g)
    for m in (mask, mask.long()):
        got = ops.relative_bias_grad(rows(g.to(device), how), buckets, q_start=start, bidirectional=both,
                                     max_distance=far, causal=causal, mask=m.to(device))
        check_grad(got, g, case, mask)
        assert not got[1].any()


def test_broadcast_and_empty(device):
    g = torch.randn(1, 1, 20, 20, device=device)
    many = g.expand(3, 4, 20, 20)
    check_grad(ops.relative_bias_grad(many, 32), many, (4, 20, 20, 0, 32, 128, True, False))
    for shape in ((0, 2, 4, 4), (2, 0, 4, 4), (2, 3, 0, 4), (2, 3, 4, 0)):
        got = ops.relative_bias_grad(torch.randn(shape, device=device), 32)
        assert got.shape == (shape[0], 32, shape[1]) and not got.any()
    table = torch.randn(32, 3, device=device)
    for tq, tk in ((0, 4), (4, 0)):
        assert ops.relative_bias(table, tq, tk).shape == (3, tq, tk)
    assert ops.relative_bias(table[:, :0], 4, 4).shape == (0, 4, 4)


def test_table_strides(device):
    table = torch.randn(3, 32, device=device).t()  # heads first in memory
    assert torch.equal(ops.relative_bias(table, 9, 12), ops.relative_bias(table.contiguous(), 9, 12))


def test_autograd_sums_and_per_sample_gradients(device):
    """The gradient against the formula, and against differences: the bias is
    linear in the table, so a difference of a linear loss has no error of its own."""
    b, h, t = 3, 2, 37
    table = torch.randn(16, h, device=device, requires_grad=True)
    weight = torch.randn(b, h, t, t, device=device)
    bias = ops.relative_bias(table, t, t, batch=b, max_distance=20)
    assert bias.shape == (b, h, t, t) and bias.stride(0) == 0
    (bias * weight).sum().backward()
    per_sample = ops.relative_bias_grad(weight, 16, max_distance=20)
    assert torch.equal(table.grad, per_sample.sum(0))
    v = torch.randn(16, h, generator=torch.Generator().manual_seed(0)).double()
    _, ids = ids_of(t, t, 0, 16, 20, True)
    line = v[ids].permute(2, 0, 1)
    want = (line * weight.cpu().double()).sum()
    terms = (line * weight.cpu().double()).abs().sum()
    assert abs((table.grad.cpu().double() * v).sum() - want) <= (t + 520) * 2.0 ** -24 * terms
    # unbatched: the samples arrive summed
    table.grad = None
    bias = ops.relative_bias(table, t, t, max_distance=20)
    assert bias.shape == (h, t, t)
    (bias * weight).sum().backward()
    size = ops.relative_bias_grad(weight.abs(), 16, max_distance=20).sum(0)
    assert bool(((table.grad - per_sample.sum(0)).abs() <= 1e-5 * size).all())
    # a gradient of zero strides (the bias summed as it is)
    table.grad = None
    ops.relative_bias(table, t, t, max_distance=20).sum().backward()
    counts = torch.bincount(ids.flatten(), minlength=16).float()
    assert torch.equal(table.grad.cpu(), counts[:, None].expand(16, h))


def test_two_streams_and_a_graph(device):
    g = torch.randn(2, 3, 200, 333, device=device).bfloat16()
    table = torch.randn(32, 3, device=device)

    def call():
        return ops.relative_bias_grad(g, 32, q_start=133), ops.relative_bias(table, 200, 333, q_start=133)

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
        g.copy_(torch.randn_like(g))
        table.add_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        want = call()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_offsets_past_32_bits(device):
    """Samples 2^32 entries apart; a plane of 70000 x 40000; an output of as many."""
    g = torch.randn(2, 2, 33, 40, device=device).bfloat16()
    far = torch.zeros((1 << 32) + 8192, dtype=torch.bfloat16, device=device)
    view = far.as_strided(g.shape, (1 << 32, *g.stride()[1:]))
    view.copy_(g)
    assert torch.equal(ops.relative_bias_grad(view, 32), ops.relative_bias_grad(g, 32))
    del view
    plane = far[: 70000 * 40000].view(1, 1, 70000, 40000).zero_()
    entries = [(0, 0), (69999, 39999), (69999, 0), (0, 39999), (50000, 39990), (40010, 39999), (54000, 123)]
    want = torch.zeros(32)
    for n, (i, j) in enumerate(entries):
        plane[0, 0, i, j] = 2.0 ** n
        _, ids = ids_of(1, 1, i - j, 32, 128, True)
        want[ids[0, 0]] += 2.0 ** n
    assert torch.equal(ops.relative_bias_grad(plane, 32)[0, :, 0].cpu(), want)
    del plane, far
    table = torch.randn(32, 2, device=device).bfloat16()
    out = ops.relative_bias(table, 50000, 50001)
    for h, i, j in ((1, 49999, 50000), (1, 49999, 0), (0, 49999, 49990), (1, 0, 50000), (1, 43000, 43002)):
        _, ids = ids_of(1, 1, i - j, 32, 128, True)
        assert out[h, i, j] == table[ids[0, 0], h]


@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("edges", [(0, 0, 3), (0, 0, 0, 2, 2, 5), (0, 0), (0, 4, 4, 9), (0,)], ids=str)
def test_c_abi_edges_that_repeat(edges, both, device):
    """An offset belongs to the last bucket whose edge is at most its distance, to
    no other: whole numbers, forward and backward, past and future offsets."""
    h, tq, tk, start = 2, 37, 41, 9
    n = len(edges)
    lib, c_edges = nat.load(), (ctypes.c_int32 * n)(*edges)
    rel = torch.arange(tk)[None] - torch.arange(tq)[:, None] - start
    r = rel.abs() if both else (-rel).clamp(min=0)
    ids = (r[..., None] >= torch.tensor(edges)).sum(-1) - 1 + n * (both & (rel > 0))
    buckets = n * (1 + both)
    table = torch.arange(buckets * h, dtype=torch.float32, device=device).view(buckets, h)
    out = torch.empty(h, tq, tk, device=device)
    stream = torch.cuda.current_stream().cuda_stream
    nat.check(lib.da_relative_bias(table.data_ptr(), 0, h, 1, h, tq, tk, start, c_edges, n, int(both), 0,
                                   out.data_ptr(), stream), "forward")
    assert torch.equal(out.cpu(), table.cpu()[ids].permute(2, 0, 1))
    g = torch.randint(-8, 9, (3, h, tq, tk), generator=torch.Generator().manual_seed(n)).float()
    dev_g = g.to(device)
    for causal in (0, 1):
        size = ctypes.c_size_t(0)
        nat.check(lib.da_relative_bias_grad_workspace(0, 3, h, tq, tk, start, buckets, causal, ctypes.byref(size)), "size")
        ws = torch.empty(max(size.value, 16), dtype=torch.uint8, device=device)
        got = torch.empty(3, buckets, h, device=device)
        nat.check(lib.da_relative_bias_grad(dev_g.data_ptr(), 0, 3, h, tq, tk, h * tq * tk, tq * tk, tk, start, c_edges, n,
                                            int(both), causal, None, 0, 0, got.data_ptr(), ws.data_ptr(), ws.numel(),
                                            stream), "backward")
        live = torch.where(rel <= 0, g, 0.0) if causal else g
        want = live.flatten(2) @ torch.nn.functional.one_hot(ids.flatten(), buckets).float()
        assert torch.equal(got.cpu(), want.transpose(1, 2)), causal
