"""Norms of queries and keys with the position rotation, against fp64.

Bounds.  A row's sum of squares is a chain of at most D/64 products in a lane
and 6 butterfly steps, the angle is fp64 up to one rounding of its fraction of a
turn (2^-25 of half a turn: 1e-7), and an output is some ten fp32 operations
after that: below 40 * 2^-24 = 2.4e-6 of the row's largest entry.  TIGHT_FP32
(1e-5) holds that with room, plus half a step of a 16-bit output.  A gradient
r (g - x r^2 mean(g x)) has the same errors in both terms, and the mean's times
x r, which stays below 16 here: within 40 * 2^-24 * 16 = 4e-5 of r max|g|.  A weight
gradient sums N terms of a sample in chains of at most N roundings: an entry is
within (N + 40) * 2^-24 of the sum of its terms' sizes.
"""

from __future__ import annotations

import math

import pytest
import torch

from conftest import HALF_ULP, TIGHT_FP32, assert_parity
from dattri_llm_amd.gradient import ops

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NAME = {torch.float32: "float32", torch.bfloat16: "bfloat16", torch.float16: "float16"}


def plain(x, w, freq, pos, eps, interleaved, scaling, mask=None):
    """One side in fp64: x (B, T, H, D), pos (B, T)."""
    x, w, rot = x.double(), w.double(), 2 * freq.shape[0]
    if mask is not None:
        x = torch.where(mask[:, :, None, None], x, 0.0)
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w
    angle = pos.double()[:, :, None, None] * freq.double()
    c, s = scaling * angle.cos(), scaling * angle.sin()
    z = y.clone()
    if interleaved:
        m, n = y[..., 0:rot:2], y[..., 1:rot:2]
        z[..., 0:rot:2], z[..., 1:rot:2] = m * c - n * s, n * c + m * s
    else:
        m, n = y[..., :rot // 2], y[..., rot // 2:rot]
        z[..., :rot // 2], z[..., rot // 2:rot] = m * c - n * s, n * c + m * s
    return z if mask is None else torch.where(mask[:, :, None, None], z, 0.0)


def check_side(got_z, got_dx, got_dw, x, gz, w, freq, pos, eps, inter, scaling, mask):
    dt = NAME[x.dtype]
    x, gz, w, freq, pos, mask = (None if v is None else v.cpu() for v in (x, gz, w, freq, pos, mask))
    xd = x.double().requires_grad_()
    wd = w.double().expand(x.shape[0], -1).clone().requires_grad_()  # one copy a sample: per-sample gradients
    z = plain(xd, wd[:, None, None, :], freq, pos, eps, inter, scaling, mask)
    live = gz.double() if mask is None else torch.where(mask[:, :, None, None], gz.double(), 0.0)
    z.backward(live)
    if got_z is not None:
        assert_parity(got_z, z, dt)
        if mask is not None:
            assert not got_z.cpu()[~mask].any()
    # a row's gradient is a difference of two terms as large as r |g|: judged by that
    rms = (xd.detach().square().mean(-1, keepdim=True) + eps).rsqrt()
    size = (rms * live.abs().amax(-1, keepdim=True) * w.double().abs().max() * abs(scaling) + xd.grad.abs()).clamp(min=1e-300)
    off = (got_dx.cpu().double() - xd.grad).abs()
    tol = TIGHT_FP32 * 4 * size + HALF_ULP.get(dt, 0.0) * xd.grad.abs()
    if x.dtype == torch.float16:
        tol = tol + 2.0 ** -25  # half a step below the least normal value
    dead = torch.zeros(x.shape[:2], dtype=torch.bool) if mask is None else ~mask
    assert not got_dx.cpu()[dead].any()
    assert bool((off <= tol)[~dead].all()), (off / tol)[~dead].max()
    terms = x.shape[1] * x.shape[2]
    y = xd.detach() * rms
    if mask is not None:
        y = torch.where(mask[:, :, None, None], y, 0.0)
    c1 = plain_back_abs(live, freq, pos, inter, scaling)
    bound = (terms + 40) * 2.0 ** -24 * (c1 * y.abs()).sum((1, 2)) + 1e-30
    assert got_dw.dtype == torch.float32
    offw = (got_dw.cpu().double() - wd.grad).abs()
    assert bool((offw <= bound).all()), (offw / bound).max()


def plain_back_abs(gz, freq, pos, inter, scaling):
    """|dy| bounded by the sizes of the two terms it is the sum of."""
    rot = 2 * freq.shape[0]
    out = gz.abs().clone()
    if rot:
        m, n = (out[..., 0:rot:2], out[..., 1:rot:2]) if inter else (out[..., :rot // 2], out[..., rot // 2:rot])
        both = (m + n) * abs(scaling)
        if inter:
            out[..., 0:rot:2], out[..., 1:rot:2] = both, both
        else:
            out[..., :rot // 2], out[..., rot // 2:rot] = both, both
    return out


def layout(x, how):
    """The same values (B, T, H, D) with other strides."""
    b, t, h, d = x.shape
    if how == "plain":
        return x.contiguous()
    if how == "heads":
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    if how == "fused":  # a slice of rows that hold more, 16-byte aligned
        big = torch.full((b, t, h + 3, d), float("nan"), dtype=x.dtype, device=x.device)
        big[:, :, 2:2 + h] = x
        return big[:, :, 2:2 + h]
    if how == "odd":  # odd strides and base: no 16-byte access fits
        big = torch.full((b, t, h, d + 3), float("nan"), dtype=x.dtype, device=x.device)
        big[..., 1:1 + d] = x
        return big[..., 1:1 + d]
    if how == "apart":  # entries not contiguous
        big = torch.full((b, t, h, d, 2), float("nan"), dtype=x.dtype, device=x.device)
        big[..., 0] = x
        return big[..., 0]
    raise AssertionError(how)


def inputs(b, t, hq, hk, d, rot, dt, seed=0, pos="index", dev="cuda"):
    gen = torch.Generator().manual_seed(seed)
    q, k = (torch.randn(b, t, h, d, generator=gen).to(dt) for h in (hq, hk))
    gq, gk = (torch.randn(b, t, h, d, generator=gen).to(dt) for h in (hq, hk))
    wq, wk = ((1 + 0.2 * torch.randn(d, generator=gen)).to(dt) for _ in range(2))
    freq = torch.tensor([10000.0 ** (-i / max(rot, 1)) for i in range(0, rot, 2)], dtype=torch.float32)
    p = torch.arange(t).expand(b, t)
    if pos == "far":
        p = p + torch.randint(0, 1_000_000, (b, 1), generator=gen)
    elif pos == "any":
        p = torch.randint(-5000, 5000, (b, t), generator=gen)
    return tuple(v.to(dev) for v in (q, k, gq, gk, wq, wk, freq, p))


CASES = [
    # b, t, hq, hk, d, rot, interleaved, layout, pos
    (1, 1, 1, 1, 2, 2, False, "plain", "index"),
    (2, 1, 32, 8, 128, 128, False, "fused", "far"),
    (3, 1, 4, 4, 64, 64, True, "plain", "far"),
    (2, 33, 8, 2, 128, 128, False, "heads", "index"),
    (2, 17, 5, 3, 128, 64, False, "fused", "any"),
    (1, 65, 3, 1, 256, 256, True, "heads", "index"),
    (2, 19, 9, 3, 80, 32, True, "heads", "index"),
    (2, 18, 4, 2, 80, 80, False, "plain", "far"),
    (1, 23, 7, 7, 96, 24, False, "plain", "index"),
    (2, 16, 2, 1, 72, 72, False, "odd", "any"),
    (1, 9, 3, 2, 100, 50, True, "odd", "index"),
    (2, 5, 2, 2, 7, 4, False, "plain", "any"),
    (2, 5, 2, 2, 7, 6, True, "apart", "any"),
    (1, 4, 2, 1, 1, 0, False, "plain", "index"),
    (1, 3, 2, 1, 64, 0, False, "plain", "index"),
    (1, 6, 3, 2, 1024, 1024, False, "plain", "index"),
    (1, 5, 2, 1, 1023, 512, False, "odd", "index"),
    (1, 7, 2, 2, 512, 130, True, "plain", "index"),
    (4, 130, 16, 16, 16, 16, False, "fused", "index"),
    (1, 300, 1, 1, 32, 32, True, "plain", "index"),
    (2, 3, 70, 9, 128, 128, False, "plain", "index"),
]


@pytest.mark.parametrize("dt", DTYPES, ids=NAME.get)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_matches_fp64(case, dt, device):
    b, t, hq, hk, d, rot, inter, how, pos = case
    q, k, gq, gk, wq, wk, freq, p = inputs(b, t, hq, hk, d, rot, dt, seed=hash((b, t, d)) % 100, pos=pos)
    q, k, gq, gk = (layout(v, how) for v in (q, k, gq, gk))
    kw = dict(eps=1e-6, interleaved=inter)
    positions = None if pos == "index" else p
    zq, zk = ops.qk_norm_rope(q, k, wq, wk, freq, positions, **kw)
    dq, dk, dwq, dwk = ops.qk_norm_rope_grad(gq, gk, q, k, wq, wk, freq, positions, **kw)
    assert zq.shape == q.shape and zk.dtype == k.dtype and dwq.shape == (b, d)
    check_side(zq, dq, dwq, q, gq, wq, freq, p, 1e-6, inter, 1.0, None)
    check_side(zk, dk, dwk, k, gk, wk, freq, p, 1e-6, inter, 1.0, None)


@pytest.mark.parametrize("t,d,how", [(37, 128, "fused"), (37, 72, "odd"), (1, 64, "plain")])
@pytest.mark.parametrize("dt", DTYPES, ids=NAME.get)
def test_masked_tokens_take_no_part_whatever_they_hold(t, d, how, dt, device):
    b = 4
    q, k, gq, gk, wq, wk, freq, p = inputs(b, t, 4, 2, d, d // 2 * 2, dt, seed=3)
    mask = torch.rand(b, t, generator=torch.Generator().manual_seed(1)) < 0.6
    mask[2] = False  # a sample without a live token
    mask = mask.to(device)
    for v, bad in ((q, float("nan")), (k, float("inf")), (gq, float("inf")), (gk, float("nan"))):
        v[~mask] = bad
    q, k, gq, gk = (layout(v, how) for v in (q, k, gq, gk))
    for m in (mask, mask.to(torch.uint8), mask.to(torch.int64), mask.to(torch.float32)):
        zq, zk = ops.qk_norm_rope(q, k, wq, wk, freq, mask=m, scaling=1.25)
        dq, dk, dwq, dwk = ops.qk_norm_rope_grad(gq, gk, q, k, wq, wk, freq, mask=m, scaling=1.25)
        check_side(zq, dq, dwq, q, gq, wq, freq, p, 1e-6, False, 1.25, mask)
        check_side(zk, dk, dwk, k, gk, wk, freq, p, 1e-6, False, 1.25, mask)
        assert not dwq[2].any() and not dwk[2].any()


def test_zero_rows_with_and_without_eps(device):
    q, k, gq, gk, wq, wk, freq, p = inputs(1, 3, 2, 1, 64, 64, torch.float32)
    q[0, 1, 0] = 0
    zq, _ = ops.qk_norm_rope(q, k, wq, wk, freq, eps=1e-6)
    assert not zq[0, 1, 0].any() and bool(torch.isfinite(zq).all())
    dq, _, dwq, _ = ops.qk_norm_rope_grad(gq, gk, q, k, wq, wk, freq, eps=1e-6)
    check_side(zq, dq, dwq, q, gq, wq, freq, p, 1e-6, False, 1.0, None)
    # without eps the formula has 0 * inf there, and nowhere else
    zq, _ = ops.qk_norm_rope(q, k, wq, wk, freq, eps=0.0)
    want = plain(q.cpu(), wq.cpu(), freq.cpu(), p.cpu(), 0.0, False, 1.0)
    assert torch.equal(torch.isnan(zq).cpu(), torch.isnan(want))


def test_a_nan_stays_in_its_row(device):
    q, k, gq, gk, wq, wk, freq, p = inputs(2, 9, 10, 2, 128, 128, torch.bfloat16)
    clean, _ = ops.qk_norm_rope(q, k, wq, wk, freq)
    q[1, 4, 3, 7] = float("nan")
    z, _ = ops.qk_norm_rope(q, k, wq, wk, freq)
    dq, _, dwq, _ = ops.qk_norm_rope_grad(gq, gk, q, k, wq, wk, freq)
    row = torch.zeros(2, 9, 10, dtype=torch.bool)
    row[1, 4, 3] = True
    assert torch.equal(torch.isnan(z).all(-1).cpu(), row) and torch.equal(torch.isnan(dq).any(-1).cpu(), row)
    assert torch.equal(z[~row.to(device)], clean[~row.to(device)])
    assert bool(torch.isnan(dwq[1]).any()) and bool(torch.isfinite(dwq[0]).all())


@pytest.mark.parametrize("dt", [torch.int32, torch.int64])
def test_position_types_and_shapes(dt, device):
    q, k, _, _, wq, wk, freq, p = inputs(3, 8, 4, 2, 64, 64, torch.float32, pos="any")
    want = ops.qk_norm_rope(q, k, wq, wk, freq, p.contiguous())
    got = ops.qk_norm_rope(q, k, wq, wk, freq, p.to(dt))
    wide = torch.stack([p, -p], -1).to(dt)[..., 0]  # every other entry
    strided = ops.qk_norm_rope(q, k, wq, wk, freq, wide)
    for a, b, c in zip(want, got, strided):
        assert torch.equal(a, b) and torch.equal(a, c)
    one = p[:1].contiguous()
    want = ops.qk_norm_rope(q, k, wq, wk, freq, one.expand(3, 8).contiguous())
    for form in (one, one[0], one.expand(3, 8), one.to(dt)):
        for a, b in zip(want, ops.qk_norm_rope(q, k, wq, wk, freq, form)):
            assert torch.equal(a, b)


def test_far_positions_keep_their_angles(device):
    """At 2^20 + t an fp32 product of position and frequency would be off by up to
    2^-4; an unrotated row of ones shows the angle itself."""
    t, d = 64, 64
    q = torch.ones(1, t, 1, d, device=device)
    w = torch.ones(d, device=device)
    freq = torch.tensor([10000.0 ** (-i / d) for i in range(0, d, 2)], device=device)
    p = (1 << 20) + torch.arange(t, device=device)
    z, none = ops.qk_norm_rope(q, None, w, None, freq, p, eps=0.0)
    assert none is None
    assert_parity(z, plain(q.cpu(), w.cpu(), freq.cpu(), p.cpu()[None], 0.0, False, 1.0), "float32", tight=1e-6)


@pytest.mark.parametrize("b,t,hq", [(0, 4, 2), (2, 0, 2), (2, 4, 0)])
def test_empty(b, t, hq, device):
    q, k, gq, gk, wq, wk, freq, _ = inputs(b, t, hq, 1, 32, 32, torch.float32)
    z, _ = ops.qk_norm_rope(q, k, wq, wk, freq)
    dq, _, dwq, dwk = ops.qk_norm_rope_grad(gq, gk, q, k, wq, wk, freq)
    assert z.shape == q.shape == dq.shape and dwq.shape == (b, 32) and not dwq.any()
    assert bool(torch.isfinite(dwk).all())


@pytest.mark.parametrize("inter", [False, True])
def test_autograd_gradients_and_differences(inter, device):
    """The summed weight gradients reach the parameters; each gradient agrees
    with a central difference of the fp64 formula along a random direction (its
    own error: h^2 times a third derivative, 1e-8 of the terms)."""
    b, t, d = 2, 11, 48
    q, k, gq, gk, wq, wk, freq, p = inputs(b, t, 3, 2, d, 32, torch.float32, pos="any")
    leaves = [v.clone().requires_grad_() for v in (q, k, wq, wk)]
    zq, zk = ops.qk_norm_rope(*leaves, freq, p, interleaved=inter, scaling=0.75)
    ((zq * gq).sum() + (zk * gk).sum()).backward()
    _, _, dwq, dwk = ops.qk_norm_rope_grad(gq, gk, q, k, wq, wk, freq, p, interleaved=inter, scaling=0.75)
    assert torch.equal(leaves[2].grad, dwq.sum(0)) and torch.equal(leaves[3].grad, dwk.sum(0))

    def loss(q, k, wq, wk):
        return sum((plain(x, w, freq.cpu(), p.cpu(), 1e-6, inter, 0.75) * g.cpu().double()).sum().item()
                   for x, w, g in ((q, wq, gq), (k, wk, gk)))

    gen = torch.Generator().manual_seed(5)
    base = [v.detach().cpu().double() for v in (q, k, wq, wk)]
    for i in range(4):
        v = torch.randn(base[i].shape, generator=gen, dtype=torch.float64)
        h = 1e-4
        up, down = (loss(*[x + s * h * v if j == i else x for j, x in enumerate(base)]) for s in (1, -1))
        terms = leaves[i].grad.cpu().double() * v
        assert abs((up - down) / (2 * h) - terms.sum().item()) <= 2e-5 * terms.abs().sum().item()


def test_one_side_alone_and_gradients_of_one_output(device):
    q, k, gq, gk, wq, wk, freq, _ = inputs(2, 7, 4, 2, 64, 64, torch.float32)
    both = ops.qk_norm_rope(q, k, wq, wk, freq)
    alone = ops.qk_norm_rope(q, None, wq, None, freq)
    assert torch.equal(both[0], alone[0]) and alone[1] is None
    q1, k1, w1 = q.clone().requires_grad_(), k.clone().requires_grad_(), wk.clone().requires_grad_()
    z, _ = ops.qk_norm_rope(q1, k1, wq, w1, freq)
    z.backward(gq)
    want = ops.qk_norm_rope_grad(gq, None, q, None, wq, None, freq)
    assert torch.equal(q1.grad, want[0]) and want[1] is None and want[3] is None
    assert not k1.grad.any() and not w1.grad.any()


def test_the_same_call_gives_the_same_bits_on_any_stream(device):
    q, k, gq, gk, wq, wk, freq, p = inputs(3, 333, 8, 2, 128, 128, torch.bfloat16, pos="far")
    want = ops.qk_norm_rope_grad(gq, gk, q, k, wq, wk, freq, p)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:  # two calls at once
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(ops.qk_norm_rope_grad(gq, gk, q, k, wq, wk, freq, p))
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(want, r))


def test_captured_and_replayed(device):
    q, k, gq, gk, wq, wk, freq, p = inputs(2, 40, 4, 2, 64, 64, torch.bfloat16, pos="any")

    def call():
        return (*ops.qk_norm_rope(q, k, wq, wk, freq, p), *ops.qk_norm_rope_grad(gq, gk, q, k, wq, wk, freq, p))

    call()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = call()
    for i in range(4):
        q.copy_(torch.randn_like(q))
        p.add_(17)
        graph.replay()
        torch.cuda.synchronize()
        want = call()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i
        assert math.isfinite(float(out[0].float().sum()))


@pytest.mark.parametrize("w_dt", DTYPES, ids=NAME.get)
@pytest.mark.parametrize("dt", DTYPES, ids=NAME.get)
def test_weights_of_another_type(dt, w_dt, device):
    q, k, gq, gk, wq, wk, freq, p = inputs(2, 9, 6, 2, 64, 32, dt)
    wq, wk = wq.to(w_dt), wk.to(w_dt)
    zq, zk = ops.qk_norm_rope(q, k, wq, wk, freq, eps=torch.tensor(1e-6))
    dq, dk, dwq, dwk = ops.qk_norm_rope_grad(gq, gk, q, k, wq, wk, freq)
    check_side(zq, dq, dwq, q, gq, wq, freq, p, 1e-6, False, 1.0, None)
    check_side(zk, dk, dwk, k, gk, wk, freq, p, 1e-6, False, 1.0, None)


def test_offsets_past_32_bits(device):
    """Samples 2^32 entries apart, in every operand."""
    q, k, gq, gk, wq, wk, freq, p = inputs(2, 5, 3, 1, 128, 128, torch.bfloat16)
    far = torch.empty((1 << 32) + 4096, dtype=torch.bfloat16, device=device)

    def apart(x, at):
        view = far.as_strided(x.shape, (1 << 32, *x.stride()[1:]), at)
        view.copy_(x)
        return view

    q2, gq2 = apart(q, 0), apart(gq, 2048)
    want = (*ops.qk_norm_rope(q, k, wq, wk, freq), *ops.qk_norm_rope_grad(gq, gk, q, k, wq, wk, freq))
    got = (*ops.qk_norm_rope(q2, k, wq, wk, freq), *ops.qk_norm_rope_grad(gq2, gk, q2, k, wq, wk, freq))
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_many_tokens_and_many_samples(device):
    """More tokens than one pass of the waves, more samples than workgroups of one."""
    for b, t in ((1, 20000), (3000, 2)):
        q, k, gq, gk, wq, wk, freq, p = inputs(b, t, 2, 1, 16, 16, torch.float32)
        zq, _ = ops.qk_norm_rope(q, k, wq, wk, freq)
        dq, _, dwq, _ = ops.qk_norm_rope_grad(gq, gk, q, k, wq, wk, freq)
        check_side(zq, dq, dwq, q, gq, wq, freq, p, 1e-6, False, 1.0, None)


@pytest.mark.parametrize("dt", DTYPES, ids=NAME.get)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("t,shift", [(9, 1), (13, 4), (40, 8), (1, 3)])
def test_rows_that_overlap_in_memory(t, shift, inter, dt, device):
    """Sliding windows over one line a sample, queries, keys and gradients alike:
    each output row has a place of its own."""
    b, d = 2, 16
    _, _, _, _, wq, wk, freq, p = inputs(b, t, 1, 1, d, d, dt)
    gen = torch.Generator().manual_seed(t)
    q, k, gq, gk = (torch.randn(b, d + shift * (t - 1), generator=gen).to(dt).to(device).unfold(1, d, shift).unsqueeze(2)
                    for _ in range(4))
    zq, zk = ops.qk_norm_rope(q, k, wq, wk, freq, interleaved=inter)
    dq, dk, dwq, dwk = ops.qk_norm_rope_grad(gq, gk, q, k, wq, wk, freq, interleaved=inter)
    check_side(zq, dq, dwq, q, gq, wq, freq, p, 1e-6, inter, 1.0, None)
    check_side(zk, dk, dwk, k, gk, wk, freq, p, 1e-6, inter, 1.0, None)


@pytest.mark.parametrize("inter,d,rot", [(False, 128, 64), (True, 128, 64), (False, 7, 4), (True, 23, 8), (False, 80, 32),
                                         (False, 300, 4)])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_entries_that_do_not_rotate_stay_apart(bad, inter, d, rot, device):
    """A weight, or a gradient, that is not finite at one entry past the rotated ones."""
    at = rot + (d - rot) // 3
    q, k, gq, gk, wq, wk, freq, p = inputs(2, 9, 3, 2, d, rot, torch.float32, pos="any")
    clean, _ = ops.qk_norm_rope(q, k, wq, wk, freq, p, interleaved=inter)
    w = wq.clone()
    w[at] = bad
    z, _ = ops.qk_norm_rope(q, k, w, wk, freq, p, interleaved=inter)
    others = torch.arange(d, device=device) != at
    assert torch.equal(z[..., others], clean[..., others]) and not bool(torch.isfinite(z[..., at]).any())
    dw = ops.qk_norm_rope_grad(gq, gk, q, k, wq, wk, freq, p, interleaved=inter)[2]
    g = gq.clone()
    g[1, 4, 1, at] = bad
    got = ops.qk_norm_rope_grad(g, gk, q, k, wq, wk, freq, p, interleaved=inter)[2]
    assert torch.equal(got[:, others], dw[:, others]) and torch.equal(got[0], dw[0])
    assert not bool(torch.isfinite(got[1, at]))


@pytest.mark.parametrize("inter,d,rot", [(False, 128, 128), (True, 80, 32), (False, 7, 4)])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_masked_rows_are_zero_whatever_the_weights_hold(bad, inter, d, rot, device):
    """Weights and frequencies that are not finite reach the live rows alone."""
    q, k, gq, gk, wq, wk, freq, p = inputs(2, 9, 3, 2, d, rot, torch.float32, pos="any")
    mask = torch.ones(2, 9, dtype=torch.bool, device=device)
    mask[0, 3:7] = mask[1] = False
    for at in ("weight", "frequency"):
        w, f = wq.clone(), freq.clone()
        if at == "weight":
            w[0] = bad
        else:
            f[0] = bad
        z, _ = ops.qk_norm_rope(q, k, w, wk, f, p, interleaved=inter, mask=mask)
        dq, _, dw, _ = ops.qk_norm_rope_grad(gq, gk, q, k, w, wk, f, p, interleaved=inter, mask=mask)
        assert not z[~mask].any() and not dq[~mask].any() and not dw[1].any()
        assert not bool(torch.isfinite(z[mask]).all()) and not bool(torch.isfinite(dq[mask]).all())


def dw_roundings(b, t, heads):
    """Roundings behind an entry of a weight gradient, at most: its term (12), a
    wave's quarter of the chunk's rows, the lanes (6), the waves (4), the chunks that
    one of eight threads adds, the eight."""
    chunk = max(1, min(1024 // heads, b * t // 512))
    chunks = -(-t // chunk)
    return 12 + chunk * heads // 4 + 1 + 6 + 4 + -(-chunks // 8) + 8


STREAMED = [
    # dt, b, t, hq, hk, d, rot, interleaved, layout: lanes of a head 8, 4, 16, 16, 32, 64 (two runs each), 64
    (torch.bfloat16, 4, 5251, 20, 5, 128, 128, False, "fused"),
    (torch.bfloat16, 13, 4051, 16, 4, 64, 64, True, "heads"),
    (torch.float32, 5, 3511, 18, 6, 80, 32, True, "heads"),
    (torch.float16, 7, 2689, 11, 3, 256, 128, False, "plain"),
    (torch.bfloat16, 3, 8741, 4, 1, 512, 512, True, "fused"),
    (torch.float32, 2, 3299, 4, 1, 1024, 1024, False, "heads"),
    (torch.float16, 1, 13127, 4, 1, 1024, 512, True, "plain"),
]


@pytest.mark.parametrize("case", STREAMED, ids=lambda c: f"{NAME[c[0]]}-{c[5]}-{c[6]}-{c[7]}-{c[8]}")
def test_rows_of_128_mib_and_more(case, device):
    """Read past the caches, by instances of their own: every row against fp64 (on
    the GPU, elementwise), padded sequences, NaN in the padding."""
    dt, b, t, hq, hk, d, rot, inter, how = case
    assert b * t * (hq + hk) * d * dt.itemsize >= 128 << 20
    gen = torch.Generator(device=device).manual_seed(d)
    mask = torch.arange(t, device=device)[None] < t - torch.randint(0, t // 4, (b, 1), generator=gen, device=device)
    freq = torch.tensor([10000.0 ** (-i / rot) for i in range(0, rot, 2)], device=device)
    p = torch.arange(t, device=device) + torch.randint(0, 100_000, (b, 1), generator=gen, device=device)
    x, g, w = [], [], []
    for h in (hq, hk):
        for side in (x, g):
            v = torch.randn(b, t, h, d, generator=gen, device=device, dtype=dt)
            v[~mask] = float("nan")
            side.append(layout(v, how))
        w.append((1 + 0.2 * torch.randn(d, generator=gen, device=device)).to(dt))
    z = ops.qk_norm_rope(*x, *w, freq, p, interleaved=inter, mask=mask)
    got = ops.qk_norm_rope_grad(*g, *x, *w, freq, p, interleaved=inter, mask=mask)
    half = HALF_ULP.get(NAME[dt], 0.0)
    least = 2.0 ** -25 if dt == torch.float16 else 0.0  # half a step below fp16's least normal value
    for i, h in enumerate((hq, hk)):
        xd = torch.where(mask[:, :, None, None], x[i].double(), 0.0).requires_grad_()
        wd = w[i].double().expand(b, -1).clone().requires_grad_()
        want = plain(xd, wd[:, None, None, :], freq, p, 1e-6, inter, 1.0, mask)
        live = torch.where(mask[:, :, None, None], g[i].double(), 0.0)
        want.backward(live)
        want, dx, dw = want.detach(), xd.grad, wd.grad
        off = (z[i].double() - want).abs()
        assert bool((off <= TIGHT_FP32 * want.abs().amax(-1, keepdim=True) + half * want.abs() + least).all())
        rms = (xd.detach().square().mean(-1, keepdim=True) + 1e-6).rsqrt()
        size = rms * live.abs().amax(-1, keepdim=True) * w[i].double().abs().max() + dx.abs()
        off = (got[i].double() - dx).abs()
        assert bool((off <= 4 * TIGHT_FP32 * size + half * dx.abs() + least).all())
        assert not z[i][~mask].any() and not got[i][~mask].any()
        terms = plain_back_abs(live, freq, p, inter, 1.0) * (xd.detach() * rms).abs()
        bound = dw_roundings(b, t, h) * 2.0 ** -24 * terms.sum((1, 2))
        assert bool(((got[2 + i].double() - dw).abs() <= bound).all())
        del want, off, dx, live, terms, xd


@pytest.mark.parametrize("b,t,hq,hk", [(1, 20000, 2, 1), (3000, 2, 2, 1), (3, 4001, 5, 1), (700, 7, 3, 3), (2, 1, 64, 8)])
@pytest.mark.parametrize("dt", DTYPES, ids=NAME.get)
def test_no_row_is_lost_from_the_weight_gradients(dt, b, t, hq, hk, device):
    """Rows and gradients of -1 and 1 at angle 0: a weight gradient is a whole number
    that each of its rows changes by 1, and rounding leaves it by less than a half."""
    d = 16
    gen = torch.Generator().manual_seed(t)
    q, k, gq, gk = (torch.randint(0, 2, (b, t, h, d), generator=gen).mul_(2).sub_(1).to(dt) for h in (hq, hk, hq, hk))
    w, freq, p = torch.ones(d, dtype=dt), torch.ones(d // 2), torch.zeros(t, dtype=torch.int64)
    got = ops.qk_norm_rope_grad(*(v.to(device) for v in (gq, gk, q, k, w, w, freq, p)), eps=0.0)
    for x, g, dx, dw in ((q, gq, got[0], got[2]), (k, gk, got[1], got[3])):
        heads = x.shape[2]
        assert dw_roundings(b, t, heads) * 2.0 ** -24 * t * heads < 0.5
        x, g = x.double(), g.double()
        assert torch.equal(dw.cpu().double().round(), (x * g).sum((1, 2)))
        want = g - x * (g * x).mean(-1, keepdim=True)
        # a root of 1 off by a step, three products of sums that are exact
        off = (dx.cpu().double() - want).abs()
        assert bool((off <= 12 * 2.0 ** -24 * 2 + HALF_ULP.get(NAME[dt], 0.0) * want.abs()).all())
