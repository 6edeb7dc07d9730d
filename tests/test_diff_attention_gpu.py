"""Attention by the difference of two softmax maps against the formulas in 64 bits
(``csrc/diffattn.hip``, ``csrc/diffattn_grad.hip``)."""

from __future__ import annotations

import pytest
import torch

from conftest import stable_seed
from dattri_llm_amd.gradient import ops

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U32 = 2.0**-24


def make(b, t, s, h, hk, d, dv, dt, gen, layout, size=1.0):
    def one(n, heads, w):
        if layout == "heads":
            return (size * torch.randn(b, heads, n, w, generator=gen, device="cuda")).to(dt).transpose(1, 2)
        if layout == "odd":  # rows at odd places inside wider ones
            return (size * torch.randn(b, n, heads, w + 3, generator=gen, device="cuda")).to(dt)[..., 1:w + 1]
        if layout == "strided":
            return (size * torch.randn(b, n, heads, w, 2, generator=gen, device="cuda")).to(dt)[..., 0]
        return (size * torch.randn(b, n, heads, w, generator=gen, device="cuda")).to(dt)
    return one(t, 2 * h, d), one(s, 2 * hk, d), one(s, hk, dv)


class Reference:
    """Outputs and gradients in 64 bits, and how far a call's may be off: ``u`` is half a
    step of a 16-bit type, which maps, score gradients and outputs are rounded by (0 in
    fp32); sums in fp32 are off by 2^-24 a term."""

    def __init__(self, q, k, v, lam, g, *, scale=None, causal=False, q_start=None, mask=None, q_mask=None):
        b, t, h2, d = q.shape
        s, hk, dv = v.shape[1:]
        h, group = h2 // 2, h2 // 2 // hk
        self.scale = scale = d ** -0.5 if scale is None else scale
        dt = q.dtype
        u = 0.0 if dt == torch.float32 else torch.finfo(dt).eps / 2
        # Below its normal range fp16 steps are 2^-24; an exponential below 2^-126 becomes zero.
        tiny = 2.0**-24 if dt == torch.float16 else 2.0**-126
        start = s - t if q_start is None else q_start
        seen = torch.ones(b, t, s, dtype=torch.bool, device="cuda")
        if causal:
            i, j = torch.arange(t, device="cuda")[:, None], torch.arange(s, device="cuda")
            seen &= j <= i + start
        if mask is not None:
            seen &= (mask != 0)[:, None]
        if q_mask is not None:
            seen &= (q_mask != 0)[..., None]
        self.seen = seen

        def clean(x, m):
            return x.double() if m is None else torch.where((m != 0)[..., None, None], x.double(), 0)

        lam = lam.double().expand(h) if lam.numel() == 1 else lam.double()
        la = lam.abs()[:, None, None]
        lam = lam[:, None, None]
        q = clean(q, q_mask).view(b, t, h, 2, d).permute(0, 2, 3, 1, 4).contiguous()
        k = clean(k, mask).view(b, s, hk, 2, d).repeat_interleave(group, 2).permute(0, 2, 3, 1, 4).contiguous()
        v = clean(v, mask).repeat_interleave(group, 2).transpose(1, 2).contiguous()
        g = clean(g, q_mask).transpose(1, 2).contiguous()  # (b, h, t, dv)
        x = torch.matmul(q, k.transpose(-1, -2)) * scale
        off = (d + 8) * U32 * torch.matmul(q.abs(), k.abs().transpose(-1, -2)) * scale
        see = seen[:, None, None]
        x = x.masked_fill(~see, -torch.inf)
        empty = ~seen.any(-1)[:, None, None, :, None]
        p = torch.softmax(x.masked_fill(empty, 0), -1).masked_fill(empty, 0)
        # A map's relative error: its scores' (twice: numerator and sum), and the sum's.
        e = 2 * off.masked_fill(~see, 0).amax(-1, keepdim=True) + (s + 64) * U32  # (b, h, 2, t, 1)
        ee = e.amax(2)
        c = (s + t + d + dv + 64) * U32
        p1, p2 = p[:, :, 0], p[:, :, 1]
        o1, o2 = torch.matmul(p1, v), torch.matmul(p2, v)
        out = o1 - lam * o2
        a2 = torch.matmul(p2, v.abs())
        a = torch.matmul(p1, v.abs()) + la * a2
        some = (p.sum(2) > 0).double()  # (b, h, t, s): pairs that count
        self.out = out.transpose(1, 2)
        out_off = (u + ee + c) * a + tiny * (1 + la) * torch.matmul(some, v.abs())
        self.out_off = (u * out.abs() + out_off).transpose(1, 2) + tiny
        dp = torch.matmul(g, v.transpose(-1, -2))
        d1, d2 = (g * o1).sum(-1, keepdim=True), (g * o2).sum(-1, keepdim=True)
        ds1, ds2 = p1 * (dp - d1), -lam * p2 * (dp - d2)
        dp_off = c * torch.matmul(g.abs(), v.abs().transpose(-1, -2))
        second_off = (2 * u + ee + c) * a2 + tiny * (torch.matmul(some, v.abs()) + 1)
        d2_off = (g.abs() * (second_off + c * o2.abs())).sum(-1, keepdim=True)
        d1_off = (g.abs() * (out_off + u * out.abs() + c * (out.abs() + la * o2.abs()) + tiny)).sum(-1, keepdim=True) + la * d2_off
        big = g.abs().amax() if g.numel() else 0.0
        f = big * tiny  # the smallest steps of scaled score gradients
        s1 = (u + ee + c) * ds1.abs() + p1 * (dp_off + d1_off + c * (dp.abs() + d1.abs())) + (f + 2.0**-126 * (dp.abs() + d1.abs())) * some
        s2 = (u + ee + c) * ds2.abs() + la * p2 * (dp_off + d2_off + c * (dp.abs() + d2.abs())) + (f + 2.0**-126 * la * (dp.abs() + d2.abs())) * some
        self.dq = torch.zeros_like(q)
        dq_off, dk, dk_off = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(k)
        for m, (ds, so) in enumerate(((ds1, s1), (ds2, s2))):
            self.dq[:, :, m] = torch.matmul(ds, k[:, :, m]) * scale
            dq_off[:, :, m] = torch.matmul(so + c * ds.abs(), k[:, :, m].abs()) * scale
            dk[:, :, m] = torch.matmul(ds.transpose(-1, -2), q[:, :, m]) * scale
            dk_off[:, :, m] = torch.matmul((so + c * ds.abs()).transpose(-1, -2), q[:, :, m].abs()) * scale
        mixed = p1 - lam * p2
        dval = torch.matmul(mixed.transpose(-1, -2), g)
        both = p1 + la * p2
        dval_off = torch.matmul(((u + ee + c * group) * both + tiny * some).transpose(-1, -2), g.abs())

        def heads(y):  # (b, h, 2, n, w) -> (b, n, 2 h, w)
            return y.permute(0, 3, 1, 2, 4).flatten(2, 3)

        def shared(y):  # sums over the heads of a key head
            return y.unflatten(1, (hk, group)).sum(2)

        self.dq, dq_off = heads(self.dq), heads(dq_off)
        self.dk, dk_off = heads(shared(dk)), heads(shared(dk_off))
        self.dv, dval_off = shared(dval).transpose(1, 2), shared(dval_off).transpose(1, 2)
        self.dq_off = dq_off + u * self.dq.abs() + tiny
        self.dk_off = dk_off + u * self.dk.abs() + tiny
        self.dv_off = dval_off + u * self.dv.abs() + tiny
        self.dlam = -(g * o2).sum((2, 3))
        self.dlam_off = d2_off.sum((2, 3)) + c * (g * o2).abs().sum((2, 3))

    def near(self, name, got):
        want, off = getattr(self, name), getattr(self, name + "_off")
        assert got.shape == want.shape, (name, got.shape, want.shape)
        worst = ((got.double() - want).abs() - off - 2.0**-149).max().item() if got.numel() else 0.0
        assert worst <= 0, f"{name}: {worst:.3e} past the bound, largest value {want.abs().max().item():.3e}"


def run(q, k, v, lam, g, **kw):
    out, state = ops.diff_attention(q, k, v, lam, return_state=True, **kw)
    assert torch.equal(out, ops.diff_attention(q, k, v, lam, **kw))
    return out, *ops.diff_attention_grad(g, q, k, v, lam, out, state, **kw)


def check(q, k, v, lam, g, **kw):
    ref = Reference(q, k, v, lam, g, **kw)
    got = run(q, k, v, lam, g, **kw)
    for name, x in zip(("out", "dq", "dk", "dv", "dlam"), got):
        assert x.is_contiguous() and x.dtype == (torch.float32 if name == "dlam" else q.dtype)
        ref.near(name, x)
    empty = ~ref.seen.any(-1)
    assert (got[0][empty] == 0).all() and (got[1][empty] == 0).all()
    dead = ~ref.seen.any(1)
    assert (got[2][dead] == 0).all() and (got[3][dead] == 0).all()
    return got


CASES = [  # b, t, s, h, hk, d, dv, dtype, layout, causal, masked, queries masked
    (1, 1, 1, 1, 1, 64, 128, "bf16", "plain", False, False, False),
    (2, 32, 32, 2, 2, 64, 128, "bf16", "plain", False, False, False),
    (2, 128, 128, 2, 1, 64, 128, "bf16", "plain", True, False, False),
    (1, 200, 200, 4, 2, 128, 256, "bf16", "plain", True, False, False),
    (2, 65, 97, 3, 3, 40, 80, "fp32", "heads", False, True, True),
    (2, 97, 97, 6, 2, 64, 64, "fp16", "heads", True, True, True),
    (1, 130, 70, 2, 2, 33, 17, "bf16", "odd", False, True, False),
    (2, 31, 33, 8, 1, 7, 9, "fp32", "odd", True, True, True),
    (1, 64, 300, 2, 1, 100, 130, "fp32", "plain", True, False, True),
    (1, 77, 300, 2, 2, 96, 200, "fp16", "strided", True, True, False),
    (3, 1, 700, 8, 2, 64, 128, "bf16", "heads", True, True, False),
    (2, 1, 5000, 4, 1, 128, 256, "bf16", "plain", True, True, False),
    (1, 2, 9000, 2, 2, 64, 64, "fp16", "plain", True, False, False),
    (1, 3, 2000, 2, 1, 64, 128, "fp32", "plain", True, True, False),
    (1, 7, 4100, 12, 2, 32, 64, "bf16", "plain", False, True, True),
    (1, 515, 515, 1, 1, 1, 1, "fp32", "plain", True, False, False),
    (1, 300, 300, 5, 5, 128, 100, "bf16", "plain", False, False, True),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_against_64_bits(case):
    b, t, s, h, hk, d, dv, dt, layout, causal, masked, q_masked = case
    gen = torch.Generator(device="cuda").manual_seed(stable_seed(case))
    q, k, v = make(b, t, s, h, hk, d, dv, DT[dt], gen, layout)
    g = (0.05 * torch.randn(b, t, h, dv, generator=gen, device="cuda")).to(DT[dt])
    lam = (0.2 + 0.6 * torch.rand(h, generator=gen, device="cuda")).to(DT[dt])
    mask = q_mask = None
    if masked:  # anything may stand at the keys that take no part
        mask = torch.rand(b, s, generator=gen, device="cuda") < 0.7
        k, v = k.masked_fill(~mask[..., None, None], float("nan")), v.masked_fill(~mask[..., None, None], float("inf"))
    if q_masked:
        q_mask = torch.rand(b, t, generator=gen, device="cuda") < 0.8
        q, g = q.masked_fill(~q_mask[..., None, None], float("nan")), g.masked_fill(~q_mask[..., None, None], float("nan"))
    check(q, k, v, lam, g, causal=causal, mask=mask, q_mask=q_mask)


@pytest.mark.parametrize("q_start", [-40, -1, 0, 5, 31, 32, 63, 64, 1000])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_causal_positions(q_start, dt):
    """Rows that see nothing, one key, whole tiles and everything."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    q, k, v = make(1, 70, 66, 2, 1, 64, 128, DT[dt], gen, "plain")
    g = torch.randn(1, 70, 2, 128, generator=gen, device="cuda").to(DT[dt])
    check(q, k, v, torch.tensor([0.4, -0.3], device="cuda"), g, causal=True, q_start=q_start)


@pytest.mark.parametrize("kind", ["none", "one", "tiles", "sample", "bytes"])
@pytest.mark.parametrize("t", [1, 50])
def test_masks(kind, t):
    gen = torch.Generator(device="cuda").manual_seed(11)
    b, s = 3, 640
    q, k, v = make(b, t, s, 4, 2, 64, 128, torch.bfloat16, gen, "plain")
    g = torch.randn(b, t, 4, 128, generator=gen, device="cuda").bfloat16()
    mask = torch.zeros(b, s, dtype=torch.bool, device="cuda")
    if kind == "one":
        mask[0, 0] = mask[1, 639] = mask[2, 321] = True
    elif kind == "tiles":  # whole tiles without a live key between others
        mask[:, 64:96] = mask[:, 300:310] = mask[:, 600:] = True
    elif kind == "sample":
        mask[1] = True
    elif kind == "bytes":
        mask = (torch.rand(b, 2 * s, generator=gen, device="cuda") < 0.5).to(torch.uint8)[:, ::2] * 7
    lam = torch.full((4,), 0.5, device="cuda")
    check(q, k, v, lam, g, mask=mask)
    check(q, k, v, lam, g, mask=mask, causal=True)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape", [(1,), (), (4,)])
def test_factor_of_any_type_and_shape(dt, shape):
    gen = torch.Generator(device="cuda").manual_seed(13)
    q, k, v = make(2, 20, 40, 4, 2, 16, 32, torch.bfloat16, gen, "plain")
    g = torch.randn(2, 20, 4, 32, generator=gen, device="cuda").bfloat16()
    lam = (torch.rand(8, generator=gen, device="cuda").to(DT[dt])[::2] if shape == (4,)
           else torch.rand(shape, generator=gen, device="cuda").to(DT[dt]))
    check(q, k, v, lam, g)


def test_scale_and_large_scores():
    """Maps that are nearly one key: maxima that grow by far more than the slack, and steep rows."""
    gen = torch.Generator(device="cuda").manual_seed(17)
    q, k, v = make(1, 90, 200, 2, 2, 64, 128, torch.float32, gen, "plain", 4.0)
    k *= torch.linspace(0.1, 2, 200, device="cuda")[:, None, None]  # the largest scores come last
    g = torch.randn(1, 90, 2, 128, generator=gen, device="cuda")
    lam = torch.tensor([0.5, 0.8], device="cuda")
    check(q, k, v, lam, g, scale=0.3)
    check(q, k.flip(1), v, lam, g, scale=0.3)


@pytest.mark.parametrize("size", [1e-4, 1e4])
def test_half_precision_gradients_of_any_size(size):
    """Upstream gradients near both ends of fp16's range keep their accuracy."""
    gen = torch.Generator(device="cuda").manual_seed(19)
    q, k, v = make(1, 128, 256, 2, 1, 64, 128, torch.float16, gen, "plain")
    g = (size * torch.randn(1, 128, 2, 128, generator=gen, device="cuda")).half()
    lam = torch.tensor([0.5, 0.8], device="cuda")
    ref = Reference(q, k, v, lam, g)
    out, dq, dk, dv, dlam = run(q, k, v, lam, g)
    for name, got in (("dq", dq), ("dk", dk), ("dv", dv)):
        want = getattr(ref, name)
        fits = want.abs() < 60000
        ref_off = getattr(ref, name + "_off")
        assert ((got.double() - want).abs() <= ref_off)[fits].all(), name


def test_autograd_gives_the_plain_calls_gradients():
    gen = torch.Generator(device="cuda").manual_seed(23)
    q, k, v = make(2, 50, 50, 4, 2, 32, 64, torch.float32, gen, "heads")
    g = torch.randn(2, 50, 4, 64, generator=gen, device="cuda")
    mask = torch.rand(2, 50, generator=gen, device="cuda") < 0.8
    for lam in (torch.rand(4, device="cuda"), torch.tensor(0.3, device="cuda")):
        leaves = [x.detach().clone().requires_grad_() for x in (q, k, v, lam)]
        ops.diff_attention(*leaves, causal=True, mask=mask, q_mask=mask).backward(g)
        _, dq, dk, dv, dlam = run(q, k, v, lam, g, causal=True, mask=mask, q_mask=mask)
        total = dlam.sum(0) if lam.dim() else dlam.sum()
        for leaf, want in zip(leaves, (dq, dk, dv, total)):
            assert torch.equal(leaf.grad, want)
    with pytest.raises(ValueError, match="return_state"):
        ops.diff_attention(*leaves, return_state=True)


def test_gradient_by_differences():
    gen = torch.Generator(device="cuda").manual_seed(29)
    q, k, v = make(1, 5, 7, 2, 1, 4, 6, torch.float32, gen, "plain")
    g = torch.randn(1, 5, 2, 6, generator=gen, device="cuda")
    lam = torch.tensor([0.4, 0.7], device="cuda")
    _, dq, dk, dv, dlam = run(q, k, v, lam, g, causal=True)
    step = 2.0**-6  # off by its square times third derivatives of order 10, and 2^-20 over the step
    for x, grad, at in ((q, dq, (0, 2, 1, 3)), (q, dq, (0, 4, 2, 0)), (k, dk, (0, 1, 0, 2)), (k, dk, (0, 5, 1, 1)),
                        (v, dv, (0, 3, 0, 5)), (lam, dlam, (1,))):
        keep = x[at].clone()
        x[at] = keep + step
        hi = (ops.diff_attention(q, k, v, lam, causal=True) * g).sum()
        x[at] = keep - step
        lo = (ops.diff_attention(q, k, v, lam, causal=True) * g).sum()
        x[at] = keep
        want = grad[at] if x is not lam else grad[0, 1]
        assert abs(((hi - lo) / (2 * step) - want).item()) < 1e-2


def test_captured_calls_replay_the_eager_results():
    gen = torch.Generator(device="cuda").manual_seed(31)
    q, k, v = make(2, 96, 96, 4, 2, 64, 128, torch.float16, gen, "plain")
    token = torch.randn(2, 1, 8, 64, generator=gen, device="cuda").half()
    cache_k, cache_v = make(2, 1, 3000, 4, 2, 64, 128, torch.float16, gen, "plain")[1:]
    g = torch.randn(2, 96, 4, 128, generator=gen, device="cuda").half()
    lam = torch.rand(4, device="cuda")

    def call():
        return *run(q, k, v, lam, g, causal=True), ops.diff_attention(token, cache_k, cache_v, lam, causal=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)

    def plain():
        out, state = ops.diff_attention(q, k, v, lam, return_state=True, causal=True)
        return (out, *ops.diff_attention_grad(g, q, k, v, lam, out, state, causal=True),
                ops.diff_attention(token, cache_k, cache_v, lam, causal=True))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = plain()
    for n in range(3):
        q.copy_(torch.randn(q.shape, device="cuda"))
        cache_k.copy_(torch.randn(cache_k.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, plain())), n


def test_results_do_not_change_from_run_to_run():
    gen = torch.Generator(device="cuda").manual_seed(37)
    q, k, v = make(2, 500, 500, 8, 2, 64, 128, torch.bfloat16, gen, "plain")
    g = torch.randn(2, 500, 8, 128, generator=gen, device="cuda").bfloat16()
    lam = torch.rand(8, device="cuda")
    first = run(q, k, v, lam, g, causal=True)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run(q, k, v, lam, g, causal=True)))


def test_empty_inputs():
    lam = torch.ones(2, device="cuda")
    for b, t, s in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        q, k, v = torch.zeros(b, t, 4, 8, device="cuda"), torch.zeros(b, s, 2, 8, device="cuda"), torch.zeros(b, s, 1, 8, device="cuda")
        out, dq, dk, dv, dlam = run(q, k, v, lam, torch.ones(b, t, 2, 8, device="cuda"))
        for x in (out, dq, dk, dv, dlam):
            assert (x == 0).all()


def test_a_cache_past_32_bits_of_offsets():
    """Keys whose offsets in elements pass 2^31 and 2^32."""
    s, gen = 70000, torch.Generator(device="cuda").manual_seed(41)
    cache = torch.zeros(s, 65536, dtype=torch.bfloat16, device="cuda")  # 9 GB: one row a position
    k = cache[:, :128].view(1, s, 2, 64)
    v = cache[:, 128:256].view(1, s, 1, 128)
    k.copy_(torch.randn(k.shape, generator=gen, device="cuda"))
    v.copy_(torch.randn(v.shape, generator=gen, device="cuda"))
    q = torch.randn(1, 1, 2, 64, generator=gen, device="cuda").bfloat16()
    lam = torch.tensor([0.5], device="cuda")
    got = ops.diff_attention(q, k, v, lam)
    assert torch.equal(got, ops.diff_attention(q, k.contiguous(), v.contiguous(), lam))
    Reference(q, k.contiguous(), v.contiguous(), lam, got).near("out", got)
