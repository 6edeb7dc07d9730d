"""Residual addition with RMS norm, difference attention and token log probabilities without a
GPU: what is refused, on which side of the C ABI, and how the capture takes their modules."""

from __future__ import annotations

import array

import pytest
import torch
from torch import nn
from torch.autograd import forward_ad

from dattri_llm_amd import _native as nat
from dattri_llm_amd import kernels
from dattri_llm_amd.gradient import AddRMSNorm, DiffAttention, FusedCapture, ops

X, OUT = 0x10000, 0x20000  # 16-byte aligned placeholders, never dereferenced


def refused(status, code, word):
    msg = nat.load().da_last_error().decode()
    assert status == code and word in msg, (status, msg)


# ---------------------------------------------------------------------------
# Python checks: before any tensor is looked for on a GPU
# ---------------------------------------------------------------------------


def test_add_rms_norm_checks():
    x, w = torch.zeros(2, 3, 8), torch.ones(8)
    for bad, word in ((dict(x=x[0]), "B, T, d"), (dict(residual=x[:, :2]), "one shape"), (dict(weight=w[:7]), "weight"),
                      (dict(mask=torch.ones(2, 2)), "mask"), (dict(quantize="column"), "quantize")):
        args = dict(x=x, residual=x, weight=w, mask=None, quantize=None) | bad
        with pytest.raises(ValueError, match=word):
            ops.add_rms_norm(args.pop("x"), args.pop("residual"), args.pop("weight"), **args)
    for bad in (x.double(), x.long()):
        with pytest.raises(NotImplementedError, match="dtype"):
            ops.add_rms_norm(bad, None, w)
    with pytest.raises(NotImplementedError, match="dtype"):
        ops.add_rms_norm(x, None, w.double())
    with pytest.raises(nat.NativeLibraryError, match="ROCm"):
        ops.add_rms_norm(x, x, w)
    with pytest.raises(NotImplementedError, match="8 bits"):
        ops.add_rms_norm(x.clone().requires_grad_(), x, w, quantize="row")
    with pytest.raises(ValueError, match="missing"):
        ops.add_rms_norm_grad(None, x, x, w)
    for g, total in ((x[:1], x), (x.half(), x)):
        with pytest.raises(ValueError, match="one shape and dtype"):
            ops.add_rms_norm_grad(g, None, total, w)


def diff(b=2, t=3, s=5, h=4, hk=2, d=8, dv=16):
    return torch.zeros(b, t, 2 * h, d), torch.zeros(b, s, 2 * hk, d), torch.zeros(b, s, hk, dv), torch.zeros(h)


def test_diff_attention_checks():
    q, k, v, lam = diff()
    for bad in ((q[0], k, v, lam), (q[:, :, :7], k, v, lam), (q, k[:, :, :2], v, lam), (q, k, v[:, :4], lam),
                (q, k[..., :4], v, lam), (q[:1], k, v, lam), (q[:, :, :6], k, v, lam[:3]), (q, k[:, :, :0], v[:, :, :0], lam)):
        with pytest.raises(ValueError):
            ops.diff_attention(*bad)
    for bad, word in (((q, k.half(), v, lam), "one dtype"), ((q, k, v, lam[:3]), "lam"), ((q, k, v, lam[None]), "lam")):
        with pytest.raises(ValueError, match=word):
            ops.diff_attention(*bad)
    for bad, word in ((dict(mask=torch.ones(2, 3)), "mask"), (dict(q_mask=torch.ones(2, 5)), "mask"),
                      (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale")):
        with pytest.raises(ValueError, match=word):
            ops.diff_attention(q, k, v, lam, **bad)
    for start in (1 << 30, -(1 << 40)):
        with pytest.raises(NotImplementedError, match="q_start"):
            ops.diff_attention(q, k, v, lam, q_start=start)
    with pytest.raises(NotImplementedError, match="dtype"):
        ops.diff_attention(q.double(), k.double(), v.double(), lam)
    with pytest.raises(NotImplementedError, match="dtype"):
        ops.diff_attention(q, k, v, lam.long())
    with pytest.raises(nat.NativeLibraryError, match="ROCm"):
        ops.diff_attention(q, k, v, lam)
    with pytest.raises(ValueError, match="return_state"):
        ops.diff_attention(q.clone().requires_grad_(), k, v, lam, return_state=True)


def test_token_logprobs_checks():
    x, t = torch.zeros(2, 3, 8), torch.zeros(2, 3, dtype=torch.int64)
    for bad, word in (((x[0, 0], t[0, 0]), "B, T, V"), ((x, t[:, :2]), "target"), ((x, t.int()), "int64")):
        with pytest.raises(ValueError, match=word):
            ops.token_logprobs(*bad)
    for bad, word in ((dict(mask=torch.ones(2, 2)), "mask"), (dict(temperature=0.0), "temperature"),
                      (dict(temperature=float("nan")), "temperature"), (dict(top=9), "top"), (dict(top=-1), "top"),
                      (dict(top=1.5), "top"), (dict(top=True), "top")):
        with pytest.raises(ValueError, match=word):
            ops.token_logprobs(x, t, **bad)
    with pytest.raises(ValueError, match="top"):
        ops.token_logprobs(torch.zeros(1, 1, 100), t[:1, :1], top=33)
    with pytest.raises(NotImplementedError, match="dtype"):
        ops.token_logprobs(x.double(), t)
    with pytest.raises(nat.NativeLibraryError, match="ROCm"):
        ops.token_logprobs(x, t)
    f = torch.zeros(2, 3)
    with pytest.raises(ValueError, match="lse and entropy"):
        ops.token_logprobs_grad(f, None, x, t, f[:, :2], f)
    with pytest.raises(ValueError, match="lse and entropy"):
        ops.token_logprobs_grad(f, None, x, t, f, f.half())
    with pytest.raises(ValueError, match="gradient"):
        ops.token_logprobs_grad(f[:1], None, x, t, f, f)


def test_forward_mode_is_refused():
    x, w = torch.zeros(2, 3, 8), torch.ones(8)
    q, k, v, lam = diff()
    t = torch.zeros(2, 3, dtype=torch.int64)
    with forward_ad.dual_level():
        dual = lambda y: forward_ad.make_dual(y, torch.ones_like(y))  # noqa: E731
        for call in (lambda: ops.add_rms_norm(dual(x), x, w), lambda: ops.add_rms_norm(x, x, dual(w)),
                     lambda: ops.diff_attention(q, dual(k), v, lam), lambda: ops.diff_attention(q, k, v, dual(lam)),
                     lambda: ops.token_logprobs(dual(x), t)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


# ---------------------------------------------------------------------------
# C ABI checks: before any launch
# ---------------------------------------------------------------------------


def test_c_abi_add_rms_norm_checks():
    lib = nat.load()

    def fwd(x=X, w=X, dt=2, wdt=2, b=2, t=3, d=64, quantize=0, out=OUT, scales=None):
        return lib.da_add_rms_norm(x, X, w, dt, wdt, b, t, d, t * d, d, t * d, d, None, 0, 0, 1e-6, quantize, out, OUT,
                                   scales, None)

    refused(fwd(dt=7), nat.DA_ERR_INVALID, "dtype")
    refused(fwd(dt=2, wdt=1), nat.DA_ERR_UNSUPPORTED, "weights")
    refused(fwd(b=-1), nat.DA_ERR_INVALID, "negative")
    refused(fwd(d=0), nat.DA_ERR_UNSUPPORTED, "entries")
    refused(fwd(d=32769), nat.DA_ERR_UNSUPPORTED, "32768")
    refused(fwd(dt=0, wdt=0, d=16385), nat.DA_ERR_UNSUPPORTED, "16384")
    refused(fwd(b=1 << 40, t=1 << 20), nat.DA_ERR_UNSUPPORTED, "too many")
    refused(fwd(quantize=3), nat.DA_ERR_INVALID, "quantize")
    for bad in (dict(x=None), dict(w=None), dict(out=None), dict(quantize=1)):
        refused(fwd(**bad), nat.DA_ERR_INVALID, "NULL")
    assert fwd(b=0) == nat.DA_OK and fwd(t=0) == nat.DA_OK

    def bwd(g=X, total=X, dx=OUT, b=2, d=64):
        return lib.da_add_rms_norm_grad(g, X, total, X, 2, 0, b, 3, d, 3 * d, d, 3 * d, d, 3 * d, d, None, 0, 0, 1e-6, dx,
                                        OUT, None, 0, None)

    for bad in (dict(g=None), dict(total=None), dict(dx=None)):
        refused(bwd(**bad), nat.DA_ERR_INVALID, "NULL")
    refused(bwd(d=40000), nat.DA_ERR_UNSUPPORTED, "entries")
    assert bwd(b=0) == nat.DA_OK
    refused(lib.da_add_rms_norm_grad_workspace(2, 1, 1, 64, None), nat.DA_ERR_INVALID, "NULL")


def test_c_abi_diff_attention_checks():
    lib = nat.load()

    def words(q=X, k=X, v=X, lam=X, lam_dtype=0, ts=64, hs=64):
        return array.array("q", (q, k, v, lam, lam_dtype, 1, 8 * ts, ts, hs, 8 * ts, ts, hs, 8 * ts, ts, hs, 0, 0, 0, 0, 0, 0))

    def fwd(rec=None, dt=2, b=2, t=3, s=5, h=4, hk=2, d=64, dv=64, scale=1.0, start=0, out=OUT, second=None, lse=None):
        rec = words() if rec is None else rec
        return lib.da_diff_attention(rec.buffer_info()[0], dt, b, t, s, h, hk, d, dv, scale, 0, start, out, second, lse,
                                     None, 0, None)

    refused(fwd(dt=9), nat.DA_ERR_INVALID, "dtype")
    refused(fwd(b=-1), nat.DA_ERR_INVALID, "negative")
    refused(fwd(h=3), nat.DA_ERR_INVALID, "share")
    refused(fwd(hk=0), nat.DA_ERR_INVALID, "share")
    refused(fwd(d=129), nat.DA_ERR_UNSUPPORTED, "entries")
    refused(fwd(dv=257), nat.DA_ERR_UNSUPPORTED, "entries")
    refused(fwd(dv=0), nat.DA_ERR_UNSUPPORTED, "entries")
    refused(fwd(s=1 << 30), nat.DA_ERR_UNSUPPORTED, "2^30")
    refused(fwd(t=1 << 29, h=8), nat.DA_ERR_UNSUPPORTED, "2^30")
    refused(fwd(start=1 << 31), nat.DA_ERR_UNSUPPORTED, "2^30")
    refused(fwd(out=None), nat.DA_ERR_INVALID, "NULL")
    refused(fwd(second=OUT), nat.DA_ERR_INVALID, "NULL")
    for bad in (dict(q=0), dict(k=0), dict(v=0), dict(lam=0)):
        refused(fwd(words(**bad)), nat.DA_ERR_INVALID, "NULL")
    refused(fwd(words(lam_dtype=5)), nat.DA_ERR_INVALID, "dtype")
    for scale in (0.0, -1.0, 1e-30, 1e30, float("inf"), float("nan")):
        refused(fwd(scale=scale), nat.DA_ERR_INVALID, "scale")
    refused(fwd(words(q=X + 8)), nat.DA_ERR_INVALID, "16-byte")
    refused(fwd(words(ts=68)), nat.DA_ERR_INVALID, "16-byte")
    refused(fwd(d=60), nat.DA_ERR_INVALID, "16-byte")
    refused(fwd(words(ts=-64)), nat.DA_ERR_INVALID, "negative")
    refused(fwd(words(ts=1 << 30), t=30), nat.DA_ERR_UNSUPPORTED, "far apart")
    assert fwd(b=0) == nat.DA_OK and fwd(t=0) == nat.DA_OK

    def bwd(g=X, lse=X, dq=OUT, dk=OUT, dlam=OUT, gs=64, b=2):
        return lib.da_diff_attention_grad(words().buffer_info()[0], g, 3 * gs, gs, 64, X, X, lse, 2, b, 3, 5, 4, 2, 64, 64,
                                          1.0, 0, 0, dq, dk, OUT, dlam, None, 0, None)

    for bad in (dict(g=None), dict(lse=None), dict(dq=None), dict(dk=None), dict(dlam=None)):
        refused(bwd(**bad), nat.DA_ERR_INVALID, "NULL")
    refused(bwd(gs=4), nat.DA_ERR_INVALID, "16-byte")
    assert bwd(b=0) == nat.DA_OK
    for query in (lib.da_diff_attention_workspace, lib.da_diff_attention_grad_workspace):
        refused(query(2, 1, 1, 1, 1, 1, 64, 64, None), nat.DA_ERR_INVALID, "NULL")


def test_c_abi_token_logprobs_checks():
    lib = nat.load()

    def fwd(logits=X, targets=X, dt=2, b=2, t=3, v=100, temperature=1.0, top=0, out=OUT, tops=None):
        return lib.da_token_logprobs(logits, dt, b, t, v, t * v, v, targets, t, 1, None, 0, 0, temperature, top, out, OUT,
                                     OUT, tops, tops, None, 0, None)

    refused(fwd(dt=4), nat.DA_ERR_INVALID, "dtype")
    refused(fwd(t=-1), nat.DA_ERR_INVALID, "negative")
    refused(fwd(v=0), nat.DA_ERR_UNSUPPORTED, "vocab")
    refused(fwd(v=1 << 31), nat.DA_ERR_UNSUPPORTED, "vocab")
    for temperature in (0.0, -1.0, float("nan"), 1e-38):
        refused(fwd(temperature=temperature), nat.DA_ERR_INVALID, "temperature")
    refused(fwd(b=1 << 20, t=1 << 20), nat.DA_ERR_UNSUPPORTED, "too many")
    for top, v in ((33, 100), (-1, 100), (5, 4)):
        refused(fwd(top=top, v=v), nat.DA_ERR_UNSUPPORTED, "alternatives")
    for bad in (dict(logits=None), dict(targets=None), dict(out=None), dict(top=3)):
        refused(fwd(**bad), nat.DA_ERR_INVALID, "NULL")
    assert fwd(b=0) == nat.DA_OK

    def bwd(lse=X, grad=OUT, up_h=None, entropy=None, t=3):
        return lib.da_token_logprobs_grad(X, 3, 1, up_h, 3, 1, None, 0, 0, X, 2, 2, t, 100, 300, 100, X, 3, 1, lse, entropy,
                                          None, 0, 0, 1.0, grad, None)

    for bad in (dict(lse=None), dict(grad=None), dict(up_h=X)):
        refused(bwd(**bad), nat.DA_ERR_INVALID, "NULL")
    assert bwd(t=0) == nat.DA_OK
    refused(lib.da_token_logprobs_workspace(2, 1, 1, 10, 0, None), nat.DA_ERR_INVALID, "NULL")


def test_the_record_has_the_struct_layout():
    import ctypes

    assert ctypes.sizeof(nat.DiffInputs) == 8 * len(nat.DiffInputs._fields_) == 8 * 21
    seen = []

    class Lib:
        def da_diff_attention_workspace(self, *a):
            return 0

        def da_diff_attention(self, record, *a):
            seen.append(nat.DiffInputs.from_buffer_copy((ctypes.c_char * 168).from_address(record)))
            return 0

    q, k, v, lam = diff()
    mask = torch.ones(2, 5, dtype=torch.bool)
    with pytest.MonkeyPatch.context() as m:
        m.setattr(nat, "load", Lib)
        m.setattr(nat, "same_device", lambda *a: torch.device("cpu"))
        m.setattr(nat, "stream_ptr", lambda d: 0)
        m.setattr(nat, "current_device", lambda: None)
        m.setattr(nat, "check", lambda status, what: None)
        kernels.diff_attention(q, k, v, lam, mask=mask)
    r = seen[0]
    assert (r.q, r.k, r.v, r.lam, r.mask, r.q_mask) == (q.data_ptr(), k.data_ptr(), v.data_ptr(), lam.data_ptr(),
                                                        mask.data_ptr(), None)
    assert (r.lam_dtype, r.lam_stride) == (nat.DA_F32, 1)
    assert (r.q_bstride, r.q_tstride, r.q_hstride) == q.stride()[:3]
    assert (r.k_bstride, r.k_tstride, r.k_hstride) == k.stride()[:3]
    assert (r.v_bstride, r.v_tstride, r.v_hstride) == v.stride()[:3]
    assert (r.mask_bstride, r.mask_kstride) == mask.stride()


# ---------------------------------------------------------------------------
# Modules under the capture
# ---------------------------------------------------------------------------


class Block(nn.Module):
    def __init__(self):
        super().__init__()
        self.norm = AddRMSNorm(8)
        self.diff = DiffAttention(4)
        self.out = nn.Linear(8, 8)


def test_capture_selects_the_modules_by_type_and_name():
    m = Block()
    factors = [f"diff.{n}" for n in ("lambda_q1", "lambda_k1", "lambda_q2", "lambda_k2")]
    assert FusedCapture(m).types == {"norm": "nn.RMSNorm", **dict.fromkeys(factors, "nn.RMSNorm"), "out": "nn.Linear"}
    assert list(FusedCapture(m, ["diff"]).slots) == factors
    assert list(FusedCapture(m.norm).slots) == [""] and list(FusedCapture(m.diff).slots) == [f[5:] for f in factors]
    cap = FusedCapture(m, batch_first=False)
    with cap:
        with pytest.raises(ValueError, match="AddRMSNorm is captured batch first"):
            m.norm(torch.zeros(2, 3, 8))
        with pytest.raises(ValueError, match="DiffAttention is captured batch first"):
            m.diff(*diff(d=4)[:3])
    assert "forward" not in m.norm.__dict__ and "forward" not in m.diff.__dict__


@pytest.fixture
def plain_kernels(monkeypatch):
    """Stand-ins for the kernels on the CPU."""
    def norm(x, residual, weight, *, eps, mask=None, quantize=None):
        total = x if residual is None else x + residual
        return total * weight, None if residual is None else total, None

    def norm_grad(g, g_total, total, weight, *, eps, mask=None, weight_grads=True):
        dx = g * weight + (0 if g_total is None else g_total)
        return dx, (g * total).sum(1) if weight_grads else None

    monkeypatch.setattr(kernels, "add_rms_norm", norm)
    monkeypatch.setattr(kernels, "add_rms_norm_grad", norm_grad)
    monkeypatch.setattr(kernels, "diff_attention", lambda q, k, v, lam, **kw: (
        q[:, :, ::2].sum(-1, keepdim=True) * lam, None, None))
    monkeypatch.setattr(kernels, "diff_attention_grad", lambda g, q, k, v, lam, out, second, lse, **kw: (
        torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v),
        (g * q[:, :, ::2].sum(-1, keepdim=True)).sum((1, 3))))


@pytest.mark.parametrize("frozen", [False, True])
def test_captured_parameters_get_per_sample_gradients(plain_kernels, frozen):
    """The chain from the factor's gradient to the four vectors, and frozen modules."""
    torch.manual_seed(0)
    norm, attend = AddRMSNorm(8), DiffAttention(4)
    x, r = torch.randn(3, 5, 8), torch.randn(3, 5, 8)
    q, k, v, _ = diff(3, 5, 5, 2, 1, 4, 1)
    q = torch.randn(q.shape)
    model = nn.ModuleDict({"norm": norm, "diff": attend}).requires_grad_(not frozen)
    cap = FusedCapture(model)
    with cap:
        out, total = norm(x, r)
        (out.square().sum() + total.sum()).backward()
        attend(q, k, v).square().sum().backward()
    got = cap.gradient()
    assert all(p.grad is None for p in model.parameters())
    model.requires_grad_()
    for i in range(3):
        model.zero_grad()
        out, total = norm(x[i:i + 1], r[i:i + 1])
        (out.square().sum() + total.sum()).backward()
        attend(q[i:i + 1], k[i:i + 1], v[i:i + 1]).square().sum().backward()
        assert torch.allclose(got.data["norm"][i], norm.weight.grad, rtol=1e-5, atol=1e-5)
        for n in ("lambda_q1", "lambda_k1", "lambda_q2", "lambda_k2"):
            assert torch.allclose(got.data[f"diff.{n}"][i], getattr(attend, n).grad, rtol=1e-4, atol=1e-5), n


def test_two_types_are_promoted(plain_kernels):
    x, r = torch.randn(2, 3, 8, dtype=torch.bfloat16), torch.randn(2, 3, 8)
    got = ops.add_rms_norm(x, r, torch.ones(8))
    assert got.out.dtype == got.total.dtype == torch.float32 and torch.equal(got.total, x.float() + r)
    assert ops.add_rms_norm(x, x.half(), torch.ones(8)).total.dtype == torch.float32


def test_the_factor_is_formed_in_fp32():
    m = DiffAttention(64, lambda_init=0.5).to(torch.bfloat16)
    a, b = (x.double() for x in (m.lambda_q1, m.lambda_k1))
    c, d = (x.double() for x in (m.lambda_q2, m.lambda_k2))
    want = (a * b).sum().exp() - (c * d).sum().exp() + 0.5
    assert m.factor().dtype == torch.float32 and abs(m.factor().item() - want.item()) < 1e-5
