"""Difference attention where it can go wrong: scores that are not finite or very large, fp16
samples and maps of very different sizes, rows that see few keys, and every CU busy
(``csrc/diffattn.hip``, ``csrc/diffattn_grad.hip``)."""

from __future__ import annotations

import pytest
import torch

from conftest import stable_seed
from dattri_llm_amd.gradient import ops

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U32 = 2.0**-24
NAMES = ("out", "dq", "dk", "dv", "dlam")


def run(q, k, v, lam, g, **kw):
    out, state = ops.diff_attention(q, k, v, lam, return_state=True, **kw)
    return out, *ops.diff_attention_grad(g, q, k, v, lam, out, state, **kw)


def exact(q, k, v, lam, g, *, scale=None, seen=None):
    """The formulas in 64 bits, gradients by automatic differentiation; ``seen`` (b, t, s)."""
    b, t, h2, d = q.shape
    s, hk, dv = v.shape[1:]
    h = h2 // 2
    lam = lam.double().expand(h) if lam.numel() == 1 else lam.double()
    q, k, v = (x.double().contiguous().requires_grad_() for x in (q, k, v))
    lams = lam.expand(b, h).clone().requires_grad_()
    qs = q.view(b, t, h, 2, d).permute(0, 2, 3, 1, 4).contiguous()
    ks = k.view(b, s, hk, 2, d).repeat_interleave(h // hk, 2).permute(0, 2, 3, 4, 1).contiguous()
    x = torch.matmul(qs, ks) * (d ** -0.5 if scale is None else scale)
    if seen is not None:
        x = x.masked_fill(~seen[:, None, None], -torch.inf)
    p = x.softmax(-1)
    o = torch.matmul(p, v.repeat_interleave(h // hk, 2).transpose(1, 2)[:, :, None].contiguous())
    out = (o[:, :, 0] - lams[:, :, None, None] * o[:, :, 1]).transpose(1, 2)
    (out * g.double()).sum().backward()
    return tuple(y.detach() for y in (out, q.grad, k.grad, v.grad, lams.grad)), p.detach()


def normal(gen, *shape, dt=torch.float32, size=1.0):
    return (size * torch.randn(*shape, generator=gen, device="cuda")).to(dt)


def operands(seed, b, t, s, h, hk, d, dv, dt):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (normal(gen, b, t, 2 * h, d, dt=dt), normal(gen, b, s, 2 * hk, d, dt=dt), normal(gen, b, s, hk, dv, dt=dt),
            0.2 + 0.6 * torch.rand(h, generator=gen, device="cuda"), normal(gen, b, t, h, dv, dt=dt, size=0.1))


# ---------------------------------------------------------------------------
# Scores that are not finite
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dt,where", [(dt, w) for dt in DT for w in ("q0", "q1", "k0", "k1", "v", "g")
                                      if dt != "fp16" or w[0] in "qk"])
@pytest.mark.parametrize("t,s", [(40, 70), (300, 600), (1, 3000)])  # whole, and keys in splits
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_what_is_not_finite_reaches_the_gradients(dt, t, s, where, what):
    """Wherever automatic differentiation of the formula gives NaN there is NaN; the other
    sample's results do not change by a bit."""
    q, k, v, lam, g = operands(stable_seed((t, s)), 2, t, s, 4, 2, 32, 48, DT[dt])
    clean = run(q, k, v, lam, g)
    if where[0] == "q":
        q[0, t // 2, 2 + int(where[1]), 5] = what  # head 1
    elif where[0] == "k":
        k[0, s // 3, 2 + int(where[1]), 5] = what  # key head 1
    elif where == "v":
        v[0, s // 3, 1, 5] = what
    else:
        g[0, t // 2, 1, 5] = what
    got = run(q, k, v, lam, g)
    want, _ = exact(q, k, v, lam, g)
    # An infinite g: delta is g . out, +inf or -inf, where automatic differentiation sums p dp of
    # both signs to NaN; dp - delta, +inf or -inf too, then is NaN for equal signs and infinite for
    # others.  Everything else has no other order.
    lost = torch.isnan if (where, what) != ("g", float("inf")) else (lambda x: ~x.isfinite())
    for name, x, y, z in zip(NAMES, got, want, clean):
        assert bool(lost(x[y.isnan()]).all()), name
        assert torch.equal(x[1], z[1]), name
    assert torch.equal(got[0].isnan(), want[0].isnan())


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("s", [1, 33, 3000])
def test_rows_whose_scores_are_all_infinite(dt, sign, s):
    """An overflowed query: scores of +inf alone and of -inf alone give NaN, no zeros; a query
    that takes no part and a sample whose keys do not stay zero."""
    q, k, v, lam, g = operands(s, 3, 2, s, 2, 1, 32, 32, DT[dt])
    k[..., 3] = sign * (1 + k[..., 3].abs())
    q[:, 0, :, 3] = float("inf")
    mask = torch.ones(3, s, dtype=torch.bool, device="cuda")
    q_mask = torch.ones(3, 2, dtype=torch.bool, device="cuda")
    mask[1], q_mask[2, 0] = False, False
    out, dq, dk, dv, dlam = run(q, k, v, lam, g, mask=mask, q_mask=q_mask)
    assert bool(out[0, 0].isnan().all()) and bool(out[:, 1].isfinite().all())
    assert bool(dq[0, 0].isnan().all()) and bool(dk[0].isnan().any()) and bool(dv[0].isnan().all())
    assert bool(dlam[0].isnan().all())
    for x in (out, dq, dk, dv, dlam):
        assert bool((x[1] == 0).all()) and bool(x[2].isfinite().all())
    assert bool((out[2, 0] == 0).all()) and bool((dq[2, 0] == 0).all())


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_an_infinite_first_score_of_a_causal_row(dt):
    """Row 0 sees one key, whose score is -inf; the rows behind it are finite."""
    q, k, v, lam, g = operands(3, 1, 50, 50, 2, 1, 32, 32, DT[dt])
    k[0, 0, :, 7] = -1.0
    q[0, 0, :, 7] = float("inf")
    out, dq, dk, dv, _ = run(q, k, v, lam, g, causal=True)
    assert bool(out[0, 0].isnan().all()) and bool(out[0, 1:].isfinite().all())
    assert bool(dq[0, 0].isnan().all()) and bool(dq[0, 1:].isfinite().all())
    assert bool(dk[0, 0].isnan().any()) and bool(dv[0, 0].isnan().all())


# ---------------------------------------------------------------------------
# Large scores
# ---------------------------------------------------------------------------


def check_maps(q, k, v, lam, g, *, scale, rel, seen=None, grads=NAMES, **kw):
    """A call whose scores fp32 holds exactly against 64 bits.  ``rel``: how far the maps may be
    off relatively, for their exponentials' and sums' fp32 roundings; sums over n terms are off
    by n 2^-24 of their absolute terms besides, 16-bit operands and outputs by half a step."""
    dt = q.dtype
    u = 0.0 if dt == torch.float32 else torch.finfo(dt).eps / 2
    tiny = 2.0**-24 if dt == torch.float16 else 2.0**-126
    b, t, h2, d = q.shape
    s, hk, dv = v.shape[1:]
    h, group = h2 // 2, h2 // 2 // hk
    c = (s + t * group + d + dv + 64) * U32 + rel
    want, p = exact(q, k, v, lam, g, scale=scale, seen=seen)
    got = run(q, k, v, lam, g, scale=scale, **kw)
    la = lam.double().expand(h)[:, None, None]
    vs = v.double().abs().repeat_interleave(group, 2).transpose(1, 2).contiguous()  # (b, h, s, dv)
    gs = g.double().abs().transpose(1, 2).contiguous()
    a1, a2 = torch.matmul(p[:, :, 0], vs), torch.matmul(p[:, :, 1], vs)
    off = {"out": (u + c) * (a1 + la * a2).transpose(1, 2)}
    # delta = g . o_m, from outputs rounded to 16 bits of maps rounded to 16 bits
    delta = ((3 * u + c) * gs * (a1 + (1 + la) * a2)).sum(-1, keepdim=True)
    dp = torch.matmul(gs, vs.transpose(-1, -2).contiguous())
    some = (p.sum(2) > 0).double()
    # fp16: score gradients are scaled by their largest bound, whose last step is 2^-39 of it
    least = 2.0**-38 * dp.amax() if dt == torch.float16 else 2.0**-126 * dp.amax()
    ds_off = [w * p[:, :, m] * (c * dp + delta + (u + c) * (dp + delta / max(u, U32))) + least * some
              for m, w in ((0, 1.0), (1, la))]
    qs = q.double().abs().view(b, t, h, 2, d).permute(0, 2, 3, 1, 4)
    ks = k.double().abs().view(b, s, hk, 2, d).repeat_interleave(group, 2).permute(0, 2, 3, 1, 4)
    dq = torch.stack([torch.matmul(ds_off[m], ks[:, :, m].contiguous()) for m in (0, 1)], 2) * scale
    dk = torch.stack([torch.matmul(ds_off[m].transpose(-1, -2).contiguous(), qs[:, :, m].contiguous())
                      for m in (0, 1)], 2) * scale
    off["dq"] = dq.permute(0, 3, 1, 2, 4).flatten(2, 3)
    off["dk"] = dk.unflatten(1, (hk, group)).sum(2).permute(0, 3, 1, 2, 4).flatten(2, 3)
    both = p[:, :, 0] + la * p[:, :, 1]
    off["dv"] = torch.matmul(((u + c) * both + tiny * some).transpose(-1, -2).contiguous(), gs)
    off["dv"] = off["dv"].unflatten(1, (hk, group)).sum(2).transpose(1, 2)
    off["dlam"] = delta.sum((2, 3))
    for name, x, y in zip(NAMES, got, want):
        if name not in grads:
            continue
        worst = ((x.double() - y).abs() - off[name] - (0 if name == "dlam" else u) * y.abs() - tiny).max().item()
        assert worst <= 0, f"{name}: {worst:.3e} past its bound, largest value {y.abs().max().item():.3e}"
    return got


def whole(gen, most, *shape, dt):
    return torch.randint(-most, most + 1, shape, generator=gen, device="cuda").to(dt)


SHAPES = [(60, 200, False), (70, 700, True), (2, 3000, True)]  # few keys, many, in splits


def seen_by(b, t, s, causal):
    seen = torch.ones(b, t, s, dtype=torch.bool, device="cuda")
    return seen.tril(s - t) if causal else seen


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("power", [20, 30, 40, 66])
@pytest.mark.parametrize("t,s,causal", SHAPES)
def test_any_accepted_scale(dt, power, t, s, causal):
    """Whole numbers as scores, times up to 2^66: the maps are the largest scores' keys, in equal
    parts.  log2 of their number and its exponential are off by 2^-20 together."""
    gen = torch.Generator(device="cuda").manual_seed(stable_seed((t, s)))
    b, h, hk, d, dv = 2, 4, 2, 32, 48
    q, k = whole(gen, 1, b, t, 2 * h, d, dt=DT[dt]), whole(gen, 1, b, s, 2 * hk, d, dt=DT[dt])
    v, g = normal(gen, b, s, hk, dv, dt=DT[dt]), normal(gen, b, t, h, dv, dt=DT[dt], size=0.1)
    lam = 0.2 + 0.6 * torch.rand(h, generator=gen, device="cuda")
    names = NAMES if dt != "fp16" else ("out", "dv", "dlam")  # dq and dk pass fp16's range
    check_maps(q, k, v, lam, g, scale=2.0**power, rel=2.0**-20, seen=seen_by(b, t, s, causal), causal=causal, grads=names)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("size,parts", [(64, 8), (1024, 1)])
@pytest.mark.parametrize("t,s,causal", SHAPES)
def test_scores_with_a_large_common_part(dt, size, parts, t, s, causal):
    """Scores of 2^12 and 2^20 with differences of a few: multiples of 2^-6 or 1, exact in fp32.
    The exponents of what counts are below 2^6, off by 2^-19 with those of the sums."""
    gen = torch.Generator(device="cuda").manual_seed(stable_seed((size, t)))
    b, h, hk, d, dv = 2, 4, 2, 32, 48
    q = whole(gen, parts, b, t, 2 * h, d, dt=DT[dt]) / parts
    k = whole(gen, parts, b, s, 2 * hk, d, dt=DT[dt]) / parts
    q[..., -1], k[..., -1] = size, size
    v, g = normal(gen, b, s, hk, dv, dt=DT[dt]), normal(gen, b, t, h, dv, dt=DT[dt], size=0.1)
    lam = 0.2 + 0.6 * torch.rand(h, generator=gen, device="cuda")
    check_maps(q, k, v, lam, g, scale=1.0, rel=2.0**-18, seen=seen_by(b, t, s, causal), causal=causal)


# ---------------------------------------------------------------------------
# fp16
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("what,which", [*((x, y) for x in ("large", "inf", "nan") for y in "gv"), ("large", "lam")])
@pytest.mark.parametrize("t,s", [(64, 64), (300, 600), (1, 3000)])
def test_half_precision_gradients_do_not_depend_on_the_batch(what, which, t, s):
    """A sample beside one with gradients (values) of 2^20 times its own, or infinite ones, gets
    what it gets beside zeros; a key head beside another one likewise."""
    h, hk = 4, 2
    q, k, v, lam, g = operands(stable_seed((t, s, which)), 3, t, s, h, hk, 64, 64, torch.float16)
    g, v = g * 2.0**-12, v * 2.0**-6
    results = []
    for fill in (0.0, 1.0):
        q1, k1, v1, g1, lam1 = q.clone(), k.clone(), v.clone(), g.clone(), lam.clone()
        if which == "lam":  # the heads of key head 0
            lam1[:2] = 2.0**12 if fill else 0.0
        else:
            x = v1 if which == "v" else g1
            x[0] *= fill * 2.0**20 if which == "g" else fill * 2.0**14
            x[1, :, 0] *= fill * 2.0**16 if which == "g" else fill * 2.0**14
            if fill and what != "large":
                x[0, 0, 0, 3] = float(what)
                x[1, 0, 0, 3] = float(what)
        results.append(run(q1, k1, v1, lam1, g1))
    for name, x, y in zip(NAMES, *results):
        if which != "lam":
            assert torch.equal(x[2], y[2]), name
            # One query's 3000 probabilities of 2^-11.5 times gradients of 2^-15.3: dv of 2^-27 and
            # dk below that are zeros in fp16, whose last step is 2^-24.
            assert (t == 1 or bool(x[2].any())) and bool(x[2].isfinite().all())
        per = x.shape[2 if x.dim() == 4 else 1] // 2  # the second key head's
        a, b = (z[:, :, per:] if z.dim() == 4 else z[:, per:] for z in (x, y))
        assert torch.equal(a[1 if which != "lam" else slice(None)], b[1 if which != "lam" else slice(None)]), name


def test_half_precision_values_gradient_with_many_keys():
    """Probabilities of 2^-17 lie below fp16's normal range (2^-14).  Rounded to half a step each,
    where the gradients they weigh have random signs, they leave an error as large as the
    output's own rounding: sqrt 2 of it together, where steps of 2^-24 leave seven times."""
    t, s, h, hk, d, dv = 64, 131072, 4, 1, 64, 64
    q, k, v, lam, g = operands(43, 1, t, s, h, hk, d, dv, torch.float16)
    q, g = q / 4, g * 640
    want = exact(q, k, v, lam, g)[0][3]
    got = run(q, k, v, lam, g)[3].double()
    rounding = (want.half().double() - want).norm()
    assert (got - want).norm() < 1.6 * rounding, ((got - want).norm() / rounding).item()


@pytest.mark.parametrize("t,s", [(40, 60), (200, 700)])
def test_half_precision_with_factors_past_its_range(t, s):
    """|lam| p up to 10^6: the mixture of the maps passes 65504, what it gives does not."""
    q, k, v, lam, g = operands(47, 1, t, s, 4, 2, 32, 32, torch.float16)
    q, k = 3 * q, 2 * k  # maps of a few keys
    lam = torch.tensor([1e6, -1e6, 0.5, 3e5], device="cuda")
    v, g = v * 2.0**-10, g * 2.0**-10
    want, p = exact(q, k, v, lam, g)
    assert (lam.abs()[:, None, None] * p[0, :, 1]).amax() > 65504
    got = run(q, k, v, lam, g)
    u, tiny = 2.0**-11, 2.0**-24
    # Scores of up to 100 of 32 products, in fp32: exponentials off by 2^-24 (40 + 100) at most.
    both = p[:, :, 0] + lam.abs()[:, None, None] * p[:, :, 1]
    off = torch.matmul(both.transpose(-1, -2).contiguous(), g.double().abs().transpose(1, 2).contiguous())
    off = (u + 2.0**-16) * off.unflatten(1, (2, 2)).sum(2).transpose(1, 2)
    assert bool(((got[3].double() - want[3]).abs() <= off + u * want[3].abs() + tiny).all())
    assert all(bool(x.isfinite().all()) for x in got)


@pytest.mark.parametrize("dt,t", [*((dt, t) for dt in DT for t in (1, 70)), ("bf16", 40000), ("fp16", 40000)])
@pytest.mark.parametrize("below", [14.0, 18.0, 20.0])
def test_one_large_score_above_many_small_ones(dt, t, below):
    """131071 keys whose exponentials are e^-14 to e^-20 of the largest: together 11% to 3e-4 of the
    row.  The largest one's value is 0 and theirs are 1, so that out is their part, to the output's
    half step, the exponentials' own (16 bits) and the sums' 2^-24 a term (a lane adds s / 32).
    The most queries leave the keys whole, the others split them."""
    s = 131072
    q = torch.zeros(1, t, 2, 16, dtype=DT[dt], device="cuda")
    k = torch.zeros(1, s, 2, 16, dtype=DT[dt], device="cuda")
    v = torch.ones(1, s, 1, 16, dtype=DT[dt], device="cuda")
    q[..., 0], k[:, 777, :, 0], v[:, 777] = 1.0, below, 0.0
    lam = torch.tensor([0.25], device="cuda")
    mass = (s - 1) * torch.tensor(-below, dtype=torch.float64).exp().item()
    want = 0.75 * mass / (1 + mass)
    got = ops.diff_attention(q, k, v, lam, scale=1.0).double()
    u = 0.0 if dt == "fp32" else torch.finfo(DT[dt]).eps / 2
    # fp16 operands below 2^-14 have steps of 2^-24: with the largest at 2^10, half a step is 2^-35 of
    # it, of each key (at 20 below, where the exponentials are 2^-18.9, that is 2^-6 of them).
    least = 1.25 * s * 2.0**-35 if dt == "fp16" else 0.0
    off = want * (u + 1.25 / 0.75 * (u + (s / 32 + 64) * U32)) + least + 2.0**-25
    assert ((got - want).abs() <= off).all(), got.flatten()[0].item() / want


# ---------------------------------------------------------------------------
# Rows that see few keys
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("s", [40, 255, 256, 257, 1024])
@pytest.mark.parametrize("kind", ["causal", "mask", "late", "both"])
def test_the_only_key_of_a_row_has_no_score_gradient(dt, s, kind):
    """One key: its probability is 1 whatever the score is.  What is left of its gradient is fp32's,
    c terms of |g| |v| (dp and delta as sums of 64), and not the rounding of out in 16 bits."""
    b, t, h, hk, d, dv = 3, s, 4, 2, 64, 64
    q, k, v, lam, g = operands(stable_seed((s, kind)), b, t, s, h, hk, d, dv, DT[dt])
    kw, rows, key = {}, slice(0, 1), 0
    if kind in ("causal", "both"):
        kw["causal"] = True
    if kind != "causal":  # one live key in the first sample, all in the second, none in the third
        key = {"mask": s // 2, "late": s - 1, "both": 0}[kind]
        mask = torch.zeros(b, s, dtype=torch.bool, device="cuda")
        mask[0, key] = mask[1] = True
        kw["mask"] = mask
        rows = slice(0, t)
    _, dq, dk, _, dlam = run(q, k, v, lam, g, **kw)
    size = g[0, rows].double().abs().sum(-1).amax() * v[0, key].double().abs().amax()
    off = 128 * U32 * size * k[0, key].double().abs().amax() * d ** -0.5
    tiny = 2.0**-24 if dt == "fp16" else 0.0
    assert dq[0, rows].double().abs().max() <= off + tiny, (dq[0, rows].double().abs().max() / off).item()
    if kind != "causal":
        n = h // hk * t  # rows that add to the key's gradient
        assert dk[0, key].double().abs().max() <= n * 128 * U32 * size * q[0].double().abs().amax() * d ** -0.5 + tiny
        want = -(g[0].double() * v[0, key].double().repeat_interleave(h // hk, 0)).sum((0, 2))
        assert ((dlam[0] - want).abs() <= (t + 128) * U32 * t * size).all()


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("t,s,live", [(255, 255, 255), (300, 300, 40), (90, 1024, 200), (1024, 1024, 256), (2, 3000, 100)])
@pytest.mark.parametrize("causal", [False, True])
def test_score_gradients_of_few_keys(dt, t, s, live, causal):
    """dq from two 16-bit parts of ds and a repaired delta is off by its own rounding and little
    else: less than 1.15 times it in norm, where an unrepaired delta leaves 1.3 and more."""
    b, h, hk, d, dv = 2, 4, 2, 64, 64
    q, k, v, lam, g = operands(stable_seed((t, s)), b, t, s, h, hk, d, dv, DT[dt])
    mask = torch.arange(s, device="cuda")[None] < torch.tensor([[live], [s]], device="cuda")
    q_start = live - t if causal else None  # the last row sees what is live
    seen = mask[:, None].expand(b, t, s)
    if causal:
        seen = seen & (torch.arange(s, device="cuda") <= torch.arange(t, device="cuda")[:, None] + q_start)
    rows = seen[0].any(-1)
    some = seen | ~seen.any(-1, keepdim=True)  # rows without keys have no maps in 64 bits
    want = exact(q, k, v, lam, g.masked_fill(~seen.any(-1)[..., None, None], 0), seen=some)[0][1][0, rows]
    got = run(q, k, v, lam, g, mask=mask, causal=causal, q_start=q_start)[1][0, rows].double()
    rounding = (want.to(DT[dt]).double() - want).norm()
    assert (got - want).norm() < 1.15 * rounding, ((got - want).norm() / rounding).item()


# ---------------------------------------------------------------------------
# Errors as a whole, and every CU busy
# ---------------------------------------------------------------------------


def error(got, want):
    """In units of what rounding the exact result to the output's type leaves."""
    return ((got.double() - want).norm() / (want.to(got.dtype).double() - want).norm()).item()


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("t,s,fine", [(1, 90, True), (1, 5000, True), (5, 700, True), (100, 512, True), (100, 513, False),
                                      (700, 700, False)])
def test_outputs_are_rounded_once_where_keys_or_rows_are_few(dt, t, s, fine):
    """With probabilities in two parts little but the output's rounding is left.  Else theirs comes
    to it, as large where values have random signs: sqrt 2 of it together, in bf16 (whose steps
    are as coarse in both)."""
    q, k, v, lam, g = operands(stable_seed((t, s)), 2, t, s, 4, 2, 64, 64, DT[dt])
    want = exact(q, k, v, lam, g)[0][0]
    got = error(ops.diff_attention(q, k, v, lam), want)
    assert got < (1.1 if fine else 1.6), got


@pytest.mark.parametrize("masked", [False, True])
def test_every_cu_busy_against_64_bits(masked):
    """4 x 2048 causal tokens, 32 heads on 8: samples' and key heads' results at full load.  Errors in
    units of the outputs' rounding, as the roundings on the way add up to them: out and dv have
    that of the maps, dk of the score gradients, dq none but delta's."""
    b, t, h, hk, d, dv = 4, 2048, 32, 8, 64, 128
    q, k, v, lam, g = operands(53, b, t, t, h, hk, d, dv, torch.bfloat16)
    mask = torch.arange(t, device="cuda")[None] < torch.tensor([[2048], [1900], [300], [2047]], device="cuda") if masked else None
    got = run(q, k, v, lam, g, causal=True, mask=mask, q_mask=mask)
    group = h // hk
    for i, j in ((0, 0), (1, 3), (2, 6), (3, 7)):
        n = t if mask is None else int(mask[i].sum())
        heads, maps, key_maps = slice(j * group, (j + 1) * group), slice(2 * j * group, 2 * (j + 1) * group), slice(2 * j, 2 * j + 2)
        one = (q[i:i + 1, :n, maps], k[i:i + 1, :n, key_maps], v[i:i + 1, :n, j:j + 1], lam[heads], g[i:i + 1, :n, heads])
        want, _ = exact(*one, seen=torch.ones(1, n, n, dtype=torch.bool, device="cuda").tril())
        mine = (got[0][i:i + 1, :n, heads], got[1][i:i + 1, :n, maps], got[2][i:i + 1, :n, key_maps],
                got[3][i:i + 1, :n, j:j + 1])
        for name, x, y, most in zip(NAMES, mine, want, (1.6, 1.4, 1.6, 1.6)):
            assert error(x, y) < most, (i, j, name, error(x, y))
        # fp32 sums of 2^18 terms; delta from fp32 score gradients
        assert bool(((got[4][i, heads] - want[4][0]).abs() <= 1e-4 * want[4].abs().max()).all())
        for x in got[:4]:
            assert not bool(x[i, n:].any())


def test_a_state_of_other_inputs_is_refused():
    q, k, v, lam, g = operands(59, 2, 5, 7, 4, 2, 32, 32, torch.float32)
    out, state = ops.diff_attention(q, k, v, lam, return_state=True)
    for lse in (state.lse[0], state.lse[:, :1], state.lse.double(), state.lse.transpose(1, 2)[:, :, :1]):
        with pytest.raises(ValueError, match="state"):
            ops.diff_attention_grad(g, q, k, v, lam, out, state._replace(lse=lse))
