"""The residual's addition with its RMS norm against the formulas in 64 bits (``csrc/addnorm.hip``)."""

from __future__ import annotations

import pytest
import torch

from conftest import stable_seed
from dattri_llm_amd.gradient import ops

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U32 = 2.0**-24


def half_step(dt):
    return torch.finfo(dt).eps / 2


def small(dt):
    """Half a step below a type's normal range, where steps no longer shrink with the value."""
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2


def assert_near(got, want, off):
    past = (got.double() - want).abs() - off
    at = past.argmax() if past.numel() else None
    assert at is None or past.flatten()[at] <= 0, (
        f"entry {at.item()} of {tuple(got.shape)}: {got.flatten()[at].item()!r} for {want.flatten()[at].item()!r}, "
        f"{past.flatten()[at].item():.3e} past its bound")


def rows(b, t, d, dt, gen, layout):
    def one(scale=1.0):
        if layout == "wide":  # rows inside wider ones, at odd places
            return (torch.randn(b, t, 2 * d + 3, generator=gen, device="cuda") * scale).to(dt)[..., 1:d + 1]
        if layout == "swapped":
            return (torch.randn(t, b, d, generator=gen, device="cuda") * scale).to(dt).transpose(0, 1)
        if layout == "strided":  # entries apart: copied
            return (torch.randn(b, t, d, 2, generator=gen, device="cuda") * scale).to(dt)[..., 0]
        return (torch.randn(b, t, d, generator=gen, device="cuda") * scale).to(dt)
    return one


def forward64(x, r, w, eps, mask):
    """total in the rows' dtype, and out in 64 bits."""
    live = torch.ones(x.shape[:2], dtype=torch.bool, device=x.device) if mask is None else mask != 0
    total = x.float() if r is None else x.float() + r.float()
    total = torch.where(live[..., None], total, 0).to(x.dtype)  # one rounding of a sum that fp32 holds to 2^-24
    h = total.double()
    out = h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    return total, torch.where(live[..., None], out, 0), live


CASES = [  # b, t, d, dtype, weight dtype, layout, masked, residual
    (2, 3, 4096, "bf16", "bf16", "plain", False, True),
    (2, 5, 1, "fp32", "fp32", "plain", False, True),
    (3, 7, 13, "bf16", "bf16", "wide", True, True),
    (1, 9, 511, "fp16", "fp32", "swapped", True, True),
    (2, 1, 768, "bf16", "fp32", "plain", False, False),
    (2, 33, 1000, "fp32", "fp32", "wide", True, True),
    (1, 4, 2047, "fp16", "fp16", "strided", False, True),
    (2, 3, 5120, "bf16", "fp16", "plain", True, True),
    (1, 3, 8193, "bf16", "bf16", "plain", False, True),
    (1, 3, 16384, "fp32", "fp32", "plain", True, False),
    (1, 2, 32768, "fp16", "fp16", "plain", False, True),
    (5, 700, 64, "bf16", "bf16", "plain", True, True),
    (1, 3000, 1024, "bf16", "bf16", "plain", True, True),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward_and_backward(case):
    b, t, d, dt, wdt, layout, masked, with_residual = case
    dt, wdt, eps = DT[dt], DT[wdt], 1e-5
    gen = torch.Generator(device="cuda").manual_seed(stable_seed(case))
    make = rows(b, t, d, dt, gen, layout)
    x, r = make(), make(2.0) if with_residual else None
    w = (1 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(wdt)
    mask = None
    if masked:
        mask = torch.rand(b, t, generator=gen, device="cuda") < 0.7
        x = x.masked_fill(~mask[..., None], float("nan"))
    total, want, live = forward64(x, r, w, eps, mask)
    got = ops.add_rms_norm(x, r, w, eps=eps, mask=mask)
    assert got.scales is None and got.out.is_contiguous() and got.out.dtype == dt
    if with_residual:
        assert torch.equal(got.total, total)
    else:
        assert got.total is None
    # out: one rounding to its type, and in fp32 the sum of squares (a lane adds up to 32 of
    # them, joined pairwise, half of its error reaches the root), root, division, two products.
    assert_near(got.out, want, (half_step(dt) + 32 * U32) * want.abs() + small(dt))
    assert (got.out[~live] == 0).all()

    g, gt = make(0.05), make(0.05) if with_residual else None
    if masked:
        g = g.masked_fill(~live[..., None], float("inf"))
    dx, dw = ops.add_rms_norm_grad(g, gt, x if r is None else got.total, w, eps=eps, mask=mask)
    h = total.double()
    rstd = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    g64 = torch.where(live[..., None], g.double(), 0)
    gt64 = torch.zeros_like(g64) if gt is None else torch.where(live[..., None], gt.double(), 0)
    gw, xh = g64 * w.double(), h * rstd
    along = (gw * xh).mean(-1, keepdim=True)
    want = torch.where(live[..., None], rstd * (gw - xh * along) + gt64, 0)
    # Sums of up to d products in fp32 (64 a lane and their tree), products of three factors.
    size = rstd * (gw.abs() + xh.abs() * (gw * xh).abs().mean(-1, keepdim=True)) + gt64.abs()
    assert_near(dx, want, half_step(dt) * want.abs() + 96 * U32 * size + small(dt))
    assert dw.dtype == torch.float32 and dw.shape == (b, d)
    want = (g64 * xh).sum(1)
    assert_near(dw, want, (t + 48) * U32 * (g64 * xh).abs().sum(1) + small(torch.float32))
    assert dx.dtype == dt and dx.is_contiguous() and (dx[~live] == 0).all()


@pytest.mark.parametrize("d", [1, 127, 128, 129, 300, 1024, 4096, 6000])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("quantize", ["row", "block"])
def test_output_in_8_bits(d, dt, quantize):
    gen = torch.Generator(device="cuda").manual_seed(d)
    x, r = (torch.randn(2, 5, d, generator=gen, device="cuda").to(DT[dt]) for _ in range(2))
    w = 1 + 0.2 * torch.randn(d, generator=gen, device="cuda")
    mask = torch.ones(2, 5, dtype=torch.bool, device="cuda")
    mask[1, 2] = False
    x[0, 1], r[0, 1] = 0, 0  # a row of zeros: scale 1
    total, want, _ = forward64(x, r, w, 1e-6, mask)
    got = ops.add_rms_norm(x, r, w, mask=mask, quantize=quantize)
    assert got.out.dtype == torch.float8_e4m3fn and torch.equal(got.total, total)
    step = d if quantize == "row" else 128
    runs = torch.nn.functional.pad(want, (0, -d % step)).unflatten(-1, (-1, step))
    most = runs.abs().amax(-1)
    scale = torch.where(most == 0, 1.0, most / 448)
    scales = got.scales[..., None] if quantize == "row" else got.scales
    assert scales.shape == scale.shape
    assert_near(scales, scale, 34 * U32 * scale)
    # Half a step of e4m3, 2^-4 of the value or below its normal range 2^-10, times the scale.
    back = torch.nn.functional.pad(got.out.double(), (0, -d % step)).unflatten(-1, (-1, step)) * scales[..., None].double()
    near = torch.maximum(runs.abs() * 2.0**-4, scale[..., None] * 2.0**-10) + 40 * U32 * most[..., None]
    assert_near(back, runs, near)
    assert (got.out.float().abs().flatten(0, 1).amax(-1)[most.flatten(0, 1).amax(-1) > 0] == 448).all()


def test_tiny_rows_become_zeros_with_scale_one():
    x = torch.full((1, 2, 256), 1.0, device="cuda")
    w = torch.full((256,), 2.0**-120, device="cuda")
    for quantize in ("row", "block"):
        got = ops.add_rms_norm(x, None, w, quantize=quantize)
        assert (got.scales == 1).all() and (got.out.float() == 0).all()


@pytest.mark.parametrize("what", ["x", "residual", "weight"])
def test_infinite_and_nan_entries_stay_in_their_rows(what):
    x, r, w = torch.randn(1, 4, 512, device="cuda"), torch.randn(1, 4, 512, device="cuda"), torch.ones(512, device="cuda")
    clean = ops.add_rms_norm(x, r, w).out
    mask = torch.tensor([[1, 1, 0, 1]], device="cuda")
    if what == "weight":
        w[3] = float("nan")
        got = ops.add_rms_norm(x, r, w, mask=mask)
        assert (got.out[0, 2] == 0).all() and got.out[0, 0, 3].isnan()
        dx, dw = ops.add_rms_norm_grad(r, None, got.total, w, mask=mask)
        assert (dx[0, 2] == 0).all() and not dw.isnan().any()
        return
    (x if what == "x" else r)[0, 1, 7] = float("nan")
    got = ops.add_rms_norm(x, r, w, mask=mask)
    assert got.out[0, 1].isnan().all() and torch.equal(got.out[0, [0, 3]], clean[0, [0, 3]])


def test_autograd_gives_the_plain_calls_gradients():
    x, r, g, gt = (torch.randn(3, 40, 264, device="cuda") for _ in range(4))
    w = torch.randn(264, device="cuda")
    mask = torch.rand(3, 40, device="cuda") < 0.8
    for y in (x, r, w):
        y.requires_grad_()
    got = ops.add_rms_norm(x, r, w, mask=mask)
    ((got.out * g).sum() + (got.total * gt).sum()).backward()
    dx, dw = ops.add_rms_norm_grad(g, gt, got.total.detach(), w.detach(), mask=mask)
    assert torch.equal(x.grad, dx) and torch.equal(r.grad, dx) and torch.equal(w.grad, dw.sum(0))
    # one output alone; no residual; no weight gradient wanted
    x.grad = None
    ops.add_rms_norm(x, r, w, mask=mask).total.backward(gt)
    assert torch.equal(x.grad, torch.where(mask[..., None], gt, 0))
    x.grad = None
    ops.add_rms_norm(x, None, w.detach()).out.backward(g)
    dx, _ = ops.add_rms_norm_grad(g, None, x.detach(), w.detach())
    assert torch.equal(x.grad, dx)


def test_gradient_by_differences():
    gen = torch.Generator(device="cuda").manual_seed(3)
    x, r, g = (torch.randn(2, 3, 24, generator=gen, device="cuda") for _ in range(3))
    w = torch.randn(24, generator=gen, device="cuda")
    dx, dw = ops.add_rms_norm_grad(g, None, x + r, w)
    # A step of 2^-6: the differences are off by its square times third derivatives of order
    # 10, and by 2^-22 of the outputs over the step.
    step = 2.0**-6
    for i in range(0, 24, 5):
        d = torch.zeros(24, device="cuda")
        d[i] = step
        hi, lo = (ops.add_rms_norm(x + s * d, r, w).out for s in (1, -1))
        assert torch.allclose(((hi - lo) * g).sum(-1).double() / (2 * step), dx[..., i].double(), atol=1e-2)
        hi, lo = (ops.add_rms_norm(x, r, w + s * d).out for s in (1, -1))
        assert torch.allclose(((hi - lo) * g).sum((1, 2)).double() / (2 * step), dw[:, i].double(), atol=1e-2)


def test_captured_calls_replay_the_eager_results():
    x, r, g = (torch.randn(2, 300, 512, device="cuda", dtype=torch.bfloat16) for _ in range(3))
    w = torch.randn(512, device="cuda", dtype=torch.bfloat16)

    def call():
        a = ops.add_rms_norm(x, r, w)
        b = ops.add_rms_norm(x, r, w, quantize="block")
        return a.out, a.total, b.out.view(torch.uint8), b.scales, *ops.add_rms_norm_grad(g, None, a.total, w)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = call()
    for k in range(3):
        x.copy_(torch.randn(2, 300, 512, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, call())), k


def test_results_do_not_change_from_run_to_run():
    x, g = torch.randn(3, 2000, 1000, device="cuda"), torch.randn(3, 2000, 1000, device="cuda")
    w = torch.randn(1000, device="cuda")
    first = ops.add_rms_norm_grad(g, None, x, w)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, ops.add_rms_norm_grad(g, None, x, w)))


def test_empty_inputs():
    w = torch.ones(8, device="cuda")
    for b, t in ((0, 4), (3, 0)):
        x = torch.zeros(b, t, 8, device="cuda")
        assert ops.add_rms_norm(x, x, w).out.shape == (b, t, 8)
        dx, dw = ops.add_rms_norm_grad(x, x, x, w)
        assert dx.shape == (b, t, 8) and dw.shape == (b, 8) and (dw == 0).all()
