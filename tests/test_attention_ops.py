"""CPU tests of the attention and router operators' host side: bucket borders,
refused arguments (Python and C ABI), the capture's layer selection."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch
from torch import nn

from dattri_llm_amd import _native as nat
from dattri_llm_amd import kernels
from dattri_llm_amd.gradient import FusedCapture, QKNormRope, RelativeBias, ops


def bucket(r: int, n: int, far: int) -> int:
    """The definition, by whole numbers: distance r on one side of n buckets."""
    m = n // 2
    if r < m:
        return r
    j = 0
    while j + 1 < n - m and r ** (n - m) * m ** (j + 1) >= far ** (j + 1) * m ** (n - m):
        j += 1
    return m + j


@pytest.mark.parametrize("buckets,far,both", [(32, 128, True), (32, 128, False), (2, 5, False), (4, 3, True),
                                              (256, 128, True), (256, 4096, False), (7, 100, False), (16, 9, False)])
def test_bucket_edges_follow_the_definition(buckets, far, both):
    edges = list(kernels._bucket_edges(buckets, far, both))
    n = buckets // 2 if both else buckets
    assert len(edges) == n and edges[0] == 0
    for r in range(2 * far + 2):
        assert max(x for x in range(n) if edges[x] <= r) == bucket(r, n, far), r


def test_bucket_edges_match_the_logarithm_off_the_borders():
    n, m, far = 16, 8, 128
    edges = list(kernels._bucket_edges(2 * n, far, True))
    for r in range(m, 4 * far):
        x = math.log(r / m) / math.log(far / m) * (n - m)
        if abs(x - round(x)) > 1e-9:
            want = min(n - 1, m + math.floor(x))
            assert max(i for i in range(n) if edges[i] <= r) == want, r


@pytest.mark.parametrize("args", [(1, 128, False), (2, 128, True), (33, 128, True), (257, 128, False), (32, 8, True),
                                  (32, 16, False), (32, (1 << 30) + 1, True)])
def test_bucket_edges_refuse(args):
    with pytest.raises(ValueError, match="relative bias"):
        kernels._bucket_edges(*args)


def qk_args(**change):
    a = dict(q=torch.zeros(2, 3, 4, 8), k=torch.zeros(2, 3, 2, 8), q_weight=torch.ones(8), k_weight=torch.ones(8),
             inv_freq=torch.ones(4), positions=None)
    opts = {k: change.pop(k) for k in ("mask",) if k in change}
    a.update(change)
    return a, opts


@pytest.mark.parametrize("change,words", [
    (dict(q=torch.zeros(2, 3, 8)), "B, T, heads, D"),
    (dict(k=torch.zeros(2, 4, 2, 8)), "disagree"),
    (dict(k=torch.zeros(2, 3, 2, 16)), "disagree"),
    (dict(q_weight=torch.ones(4)), "norm weight"),
    (dict(k_weight=None), "norm weight"),
    (dict(k=torch.zeros(2, 3, 2, 8).half()), "dtype"),
    (dict(k_weight=torch.ones(8).half()), "dtype"),
    (dict(inv_freq=torch.ones(5)), "rotate 10"),
    (dict(inv_freq=torch.ones(4).double()), "float32"),
    (dict(positions=torch.zeros(2, 3)), "int32 or int64"),
    (dict(positions=torch.zeros(4, dtype=torch.int64)), "positions must have shape"),
    (dict(mask=torch.ones(2, 4, dtype=torch.bool)), "mask must have shape"),
])
def test_qk_norm_rope_refuses(change, words):
    a, opts = qk_args(**change)
    with pytest.raises(ValueError, match=words):
        ops.qk_norm_rope(**a, **opts)
    with pytest.raises(ValueError, match=words):
        ops.qk_norm_rope_grad(a["q"], a["k"], **a, **opts)


def test_qk_norm_rope_refuses_types_gradients_and_the_cpu():
    a, _ = qk_args()
    with pytest.raises(NotImplementedError, match="float64"):
        ops.qk_norm_rope(**{k: v.double() if k in "qk" else v for k, v in a.items()})
    with pytest.raises(ValueError, match="one output gradient"):
        ops.qk_norm_rope_grad(a["q"], None, **a)
    with pytest.raises(ValueError, match="gradient of shape"):
        ops.qk_norm_rope_grad(a["k"], a["k"], **a)
    with pytest.raises(nat.NativeLibraryError, match="ROCm GPU"):
        ops.qk_norm_rope(**a)


OVERLAPPING = {  # rows of 16 that share entries, as sliding windows do: their strides leave the axes' order open
    "windows": lambda x: x.view(-1)[:48].view(2, 24).unfold(1, 16, 1).unsqueeze(2),
    "windows of heads": lambda x: x.view(-1)[:240].view(2, 5, 24).unfold(2, 16, 1),
    "one entry apart": lambda x: x.view(-1).as_strided((2, 5, 3, 16), (100, 1, 40, 1)),
    "one head": lambda x: x.view(-1).as_strided((2, 1, 3, 16), (0, 1, 0, 1)),
}


@pytest.mark.parametrize("how", [*OVERLAPPING, "expanded", "fused", "one entry"])
def test_rows_are_written_where_no_other_row_lies(how):
    """What the kernels are told of the output: entries in a row, and each row's
    place its own."""
    x = torch.zeros(4, 6, 8, 16)
    x = {**OVERLAPPING, "expanded": lambda x: x[:1, :, :1].expand(4, 6, 8, 16), "fused": lambda x: x[:, :, 2:5],
         "one entry": lambda x: x[..., 3:4]}[how](x)
    words, out, *_ = kernels._qk_side("test", x, torch.ones(x.shape[3]), None, None)
    told = dict(zip([f[0] for f in nat.QkSide._fields_], words))
    at = sum(torch.arange(n).view([-1 if i == axis else 1 for i in range(3)]) * told[f"out_{name}stride"]
             for axis, (n, name) in enumerate(zip(x.shape[:3], "bth")))
    at = at[..., None] + torch.arange(x.shape[3])
    assert told["out"] == out.data_ptr() and out.shape == x.shape
    assert at.unique().numel() == x.numel() and int(at.max()) < out.untyped_storage().nbytes() // 4
    # and the output's own strides say the same
    mine = sum(torch.arange(n).view([-1 if i == axis else 1 for i in range(4)]) * out.stride(axis)
               for axis, n in enumerate(x.shape))
    assert torch.equal(at, mine)


def test_relative_bias_refuses():
    table, g = torch.zeros(32, 4), torch.zeros(2, 4, 5, 9)
    with pytest.raises(ValueError, match="table"):
        ops.relative_bias(table[0], 5, 5)
    with pytest.raises(ValueError, match="negative"):
        ops.relative_bias(table, -1, 5)
    with pytest.raises(ValueError, match="need batch"):
        ops.relative_bias(table, 5, 5, mask=torch.ones(2, 5))
    with pytest.raises(NotImplementedError):
        ops.relative_bias(table.double(), 5, 5)
    with pytest.raises(ValueError, match="gradient"):
        ops.relative_bias_grad(g[0], 32)
    with pytest.raises(ValueError, match="mask must have shape"):
        ops.relative_bias_grad(g, 32, mask=torch.ones(2, 5))
    for start in (-1, 5):
        with pytest.raises(ValueError, match="hold the queries"):
            ops.relative_bias_grad(g, 32, q_start=start, mask=torch.ones(2, 9))
    for call in (lambda: ops.relative_bias(table, 5, 5), lambda: ops.relative_bias_grad(g, 32)):
        with pytest.raises(nat.NativeLibraryError, match="ROCm GPU"):
            call()


def test_balance_loss_refuses():
    x, i = torch.zeros(6, 4), torch.zeros(6, 2, dtype=torch.int64)
    counts, live = torch.zeros(2, 4, dtype=torch.int64), torch.zeros(2, dtype=torch.int64)
    for bad, words in ((lambda: ops.moe.balance_loss(x, i[:5]), "expert indices"),
                       (lambda: ops.moe.balance_loss(x[0], i), "expects"),
                       (lambda: ops.moe.balance_loss_grad(None, None, x[0], counts, live), "expects"),
                       (lambda: ops.moe.balance_loss(x, i.int()), "int64"),
                       (lambda: ops.moe.balance_loss(x, i, batch=4), "samples of one length"),
                       (lambda: ops.moe.balance_loss(x, i, batch=0), "samples of one length"),
                       (lambda: ops.moe.balance_loss(x.view(2, 3, 4), i, batch=3), "batch 3"),
                       (lambda: ops.moe.balance_loss(x, i, batch=2, mask=torch.ones(3, 2)), "mask must have shape"),
                       (lambda: ops.moe.balance_loss_grad(None, None, x, counts[:, :3], live), "counts"),
                       (lambda: ops.moe.balance_loss_grad(None, None, x, counts, live[:1]), "samples of one length"),
                       (lambda: ops.moe.balance_loss_grad(None, None, x, counts.int(), live), "int64"),
                       (lambda: ops.moe.balance_loss_grad(torch.ones(3), None, x, counts, live), "loss gradient")):
        with pytest.raises(ValueError, match=words):
            bad()
    with pytest.raises(NotImplementedError):
        ops.moe.balance_loss(x.double(), i)
    with pytest.raises(nat.NativeLibraryError, match="ROCm GPU"):
        ops.moe.balance_loss(x, i)


X, OUT = 0x10000, 0x20000  # aligned placeholders, never dereferenced


def refused(status, code, *words):
    msg = nat.load().da_last_error().decode()
    assert status == code and all(w in msg for w in words), (status, msg)


def test_c_abi_qk_norm_rope_checks():
    lib = nat.load()
    sides = (nat.QkSide * 2)()
    for s in sides:
        s.x = s.gz = s.out = s.weight = X
        s.weight_grad = X
        s.heads = 2

    def call(sides=sides, dt=2, wdt=0, b=2, t=3, d=8, rot=8, freq=X, pos=None, pos_bytes=0):
        return lib.da_qk_norm_rope(sides, dt, wdt, b, t, d, rot, freq, pos, pos_bytes, 0, 1, None, 0, 0, 0, 1.0, 1e-6,
                                   None)

    refused(call(dt=9), nat.DA_ERR_INVALID, "dtype")
    refused(call(sides=None), nat.DA_ERR_INVALID, "NULL sides")
    refused(call(b=-1), nat.DA_ERR_INVALID, "negative")
    refused(call(d=0, rot=0), nat.DA_ERR_UNSUPPORTED, "head width")
    refused(call(d=1025), nat.DA_ERR_UNSUPPORTED, "head width")
    refused(call(rot=3), nat.DA_ERR_INVALID, "even")
    refused(call(rot=10), nat.DA_ERR_INVALID, "at most")
    refused(call(freq=None), nat.DA_ERR_INVALID, "inv_freq")
    refused(call(pos=X, pos_bytes=2), nat.DA_ERR_INVALID, "4 or 8")
    assert call(b=0) == nat.DA_OK and call(t=0) == nat.DA_OK
    sides[1].x = None
    refused(call(), nat.DA_ERR_INVALID, "NULL pointer of side 1")
    sides[1].x = X

    def back(ws=None, n=0):
        return lib.da_qk_norm_rope_grad(sides, 2, 0, 2, 3, 8, 8, X, None, 0, 0, 1, None, 0, 0, 0, 1.0, 1e-6, ws, n,
                                        None)

    refused(back(), nat.DA_ERR_WORKSPACE, "needed")
    refused(back(X, 16), nat.DA_ERR_WORKSPACE, "needed")
    sides[0].gz = None
    refused(back(X, 1 << 20), nat.DA_ERR_INVALID, "NULL pointer of side 0")
    refused(lib.da_qk_norm_rope_grad_workspace(1, 1, 1, 1, 8, None), nat.DA_ERR_INVALID, "argument")


def test_c_abi_relative_bias_checks():
    lib = nat.load()
    edges = (ctypes.c_int32 * 4)(0, 1, 2, 9)
    down = (ctypes.c_int32 * 4)(0, 2, 1, 9)
    late = (ctypes.c_int32 * 4)(1, 2, 3, 9)

    def fwd(dt=2, h=2, tq=3, tk=3, start=0, e=edges, n=4, table=X):
        return lib.da_relative_bias(table, dt, 2, 1, h, tq, tk, start, e, n, 0, 0, OUT, None)

    refused(fwd(dt=7), nat.DA_ERR_INVALID, "dtype")
    refused(fwd(tq=-1), nat.DA_ERR_INVALID, "negative")
    refused(fwd(start=1 << 31), nat.DA_ERR_UNSUPPORTED, "lengths")
    refused(fwd(h=70000), nat.DA_ERR_UNSUPPORTED, "heads")
    refused(fwd(n=0), nat.DA_ERR_UNSUPPORTED, "buckets")
    refused(fwd(n=257), nat.DA_ERR_UNSUPPORTED, "buckets")
    refused(fwd(e=None), nat.DA_ERR_UNSUPPORTED, "buckets")
    refused(fwd(e=down), nat.DA_ERR_INVALID, "ascend")
    refused(fwd(e=late), nat.DA_ERR_INVALID, "must be 0")
    refused(fwd(table=None), nat.DA_ERR_INVALID, "NULL")
    assert fwd(tq=0) == nat.DA_OK

    def bwd(g=X, mask=None, start=0, out=OUT, ws=None, n=0, b=2, stride=999):
        return lib.da_relative_bias_grad(g, 2, b, 2, 999, 999, 2 * 999 * 999, stride * 999, stride, start, edges, 4, 0, 0,
                                         mask, 999, 1, out, ws, n, None)

    refused(bwd(), nat.DA_ERR_WORKSPACE, "needed")
    refused(bwd(g=None), nat.DA_ERR_INVALID, "NULL g")
    refused(bwd(out=None), nat.DA_ERR_INVALID, "NULL out")
    refused(bwd(stride=-8), nat.DA_ERR_INVALID, "negative stride")
    refused(bwd(mask=X, start=1), nat.DA_ERR_INVALID, "among them")
    assert bwd(b=0) == nat.DA_OK


def test_c_abi_balance_loss_checks():
    lib = nat.load()

    def fwd(dt=0, b=2, t=3, e=4, logits=X, index=X, top=2, loss=OUT, ws=None, n=0):
        return lib.da_balance_loss(logits, dt, b, t, e, 4, index, top, None, 0, 0, loss, OUT, OUT, OUT, ws, n, None)

    refused(fwd(dt=5), nat.DA_ERR_INVALID, "dtype")
    refused(fwd(b=-1), nat.DA_ERR_INVALID, "negative")
    refused(fwd(e=0), nat.DA_ERR_UNSUPPORTED, "experts")
    refused(fwd(e=1025), nat.DA_ERR_UNSUPPORTED, "experts")
    refused(fwd(top=-1), nat.DA_ERR_INVALID, "negative")
    refused(fwd(logits=None), nat.DA_ERR_INVALID, "NULL")
    refused(fwd(index=None), nat.DA_ERR_INVALID, "NULL")
    refused(fwd(loss=None), nat.DA_ERR_INVALID, "NULL")
    refused(fwd(t=100_000), nat.DA_ERR_WORKSPACE, "needed")
    assert fwd(b=0) == nat.DA_OK

    def bwd(counts=X, t=3):
        return lib.da_balance_loss_grad(X, X, X, 0, 2, t, 4, 4, counts, X, None, 0, 0, OUT, 4, None)

    refused(bwd(counts=None), nat.DA_ERR_INVALID, "NULL")
    assert bwd(t=0) == nat.DA_OK


class Block(nn.Module):
    def __init__(self):
        super().__init__()
        self.rope = QKNormRope(8)
        self.bias = RelativeBias(8, 2)
        self.out = nn.Linear(8, 8)
        self.act = nn.ReLU()


def test_capture_selects_the_modules_by_type_and_name():
    m = Block()
    cap = FusedCapture(m)
    assert cap.types == {"rope.q_weight": "nn.RMSNorm", "rope.k_weight": "nn.RMSNorm", "bias": "nn.Embedding",
                         "out": "nn.Linear"}
    assert list(FusedCapture(m, ["rope"]).slots) == ["rope.q_weight", "rope.k_weight"]
    assert list(FusedCapture(m, ["bias", "out"]).slots) == ["bias", "out"]
    with pytest.raises(ValueError, match="ReLU"):
        FusedCapture(m, ["act"])
    with pytest.raises(ValueError, match="no such layers"):
        FusedCapture(m, ["rope", "gone"])
    with pytest.raises(RuntimeError, match="no layer"):
        cap.gradient()
    with cap:
        with pytest.raises(ValueError, match="needs batch"):
            m.bias(4, 4)
    assert "forward" not in m.bias.__dict__ and "forward" not in m.rope.__dict__
    with FusedCapture(m, batch_first=False):
        with pytest.raises(ValueError, match="batch first"):
            m.rope(torch.zeros(1, 2, 1, 8), None)


def test_modules_keep_their_frequencies_in_fp32():
    m = QKNormRope(16, rotary_dim=8, base=100.0)
    want = torch.tensor([100.0 ** (-i / 8) for i in range(0, 8, 2)])
    assert torch.equal(m.inv_freq, want)
    m.to(torch.bfloat16)
    assert m.inv_freq.dtype == torch.float32 and torch.equal(m.inv_freq, want) and m.q_weight.dtype == torch.bfloat16
    for bad in (3, 18, -2):
        with pytest.raises(ValueError, match="rotary_dim"):
            QKNormRope(16, rotary_dim=bad)


@pytest.fixture
def plain_bias(monkeypatch):
    """Stand-ins for the bias kernels on the CPU: a bias that ignores the offsets,
    and a gradient of ones a sample."""
    monkeypatch.setattr(kernels, "relative_bias", lambda table, tq, tk, **kw: table[0][:, None, None].expand(-1, tq, tk).clone())
    monkeypatch.setattr(kernels, "relative_bias_grad", lambda g, n, **kw: torch.ones(g.shape[0], n, g.shape[1]))


@pytest.mark.parametrize("frozen", [False, True])
def test_a_captured_bias_is_captured_with_its_weight_frozen_too(plain_bias, frozen):
    m = Block()
    m.bias.weight.requires_grad_(not frozen)
    cap = FusedCapture(m, ["bias"])
    with cap:
        m.bias(4, 5, batch=3).sum().backward()
        with torch.no_grad():
            assert not m.bias(4, 5, batch=3).requires_grad
    got = cap.gradient()
    assert got.data["bias"].shape == (3, 16) and m.bias.weight.grad is None
    assert m.bias.weight.requires_grad != frozen
    assert m.bias(4, 5, batch=3).requires_grad != frozen  # outside the session


def test_relative_bias_refuses_a_mask_in_the_forward_call(plain_bias):
    for table in (torch.zeros(8, 2), torch.zeros(8, 2, requires_grad=True)):
        for mask, start, words in ((torch.ones(2, 5), 0, "mask must have shape"),
                                   (torch.ones(3, 4), 0, "mask must have shape"),
                                   (torch.ones(3, 5), -1, "hold the queries"),
                                   (torch.ones(3, 5), 2, "hold the queries")):
            with pytest.raises(ValueError, match=words):
                ops.relative_bias(table, 4, 5, batch=3, q_start=start, mask=mask)
        with pytest.raises(ValueError, match="different devices"):
            ops.relative_bias(table, 4, 5, batch=3, mask=torch.ones(3, 5, device="meta"))
        for start in (0, 1):
            assert ops.relative_bias(table, 4, 5, batch=3, q_start=start, mask=torch.ones(3, 5)).shape == (3, 2, 4, 5)


def test_forward_mode_derivatives_are_refused():
    """Refused, not taken for zero: with and without a graph, under functional
    transforms, for each operand that a tangent can come from."""
    from torch.autograd import forward_ad

    a, _ = qk_args()
    floats = ("q", "k", "q_weight", "k_weight", "inv_freq")
    index = torch.zeros(6, 2, dtype=torch.int64)
    calls = [(lambda v, n=n: ops.qk_norm_rope(**{**a, n: v}), a[n]) for n in floats]
    calls += [(lambda v: ops.relative_bias(v, 4, 5), torch.zeros(8, 2)),
              (lambda v: ops.relative_bias(v, 4, 5, batch=2), torch.zeros(8, 2)),
              (lambda v: ops.moe.balance_loss(v, index), torch.zeros(6, 4)),
              (lambda v: ops.moe.balance_loss(v, index.view(2, 3, 2)), torch.zeros(2, 3, 4))]
    for call, v in calls:
        for leaf in (v, v.clone().requires_grad_()):
            with forward_ad.dual_level():
                dual = forward_ad.make_dual(leaf, torch.ones_like(v))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(dual)
                with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                    call(dual)
                with torch.no_grad(), pytest.raises(nat.NativeLibraryError, match="ROCm GPU"):  # no tangent: as ever
                    call(leaf)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(call, (v,), (torch.ones_like(v),))


def test_frequencies_that_want_a_gradient_are_refused():
    """The rotation's frequencies take no gradient: refused, not left out."""
    a, _ = qk_args(inv_freq=torch.ones(4, requires_grad=True))
    for q in (a["q"], a["q"].clone().requires_grad_()):
        with pytest.raises(NotImplementedError, match="inv_freq"):
            ops.qk_norm_rope(**{**a, "q": q})
        with torch.no_grad(), pytest.raises(nat.NativeLibraryError, match="ROCm GPU"):
            ops.qk_norm_rope(**{**a, "q": q})


@pytest.mark.parametrize("used", ["loss", "z_loss", "both"])
def test_a_loss_without_a_gradient_reaches_the_backward_call_as_none(monkeypatch, used):
    """Nothing is made for an unused loss or for the counts."""
    got = []

    def backward(up, up_z, logits, counts, live, *, mask=None):
        got.append((up, up_z))
        return torch.zeros_like(logits)

    monkeypatch.setattr(kernels, "balance_loss", lambda x, i, **kw: (
        torch.zeros(2), torch.zeros(2), torch.zeros(2, 4, dtype=torch.int64), torch.zeros(2, dtype=torch.int64)))
    monkeypatch.setattr(kernels, "balance_loss_grad", backward)
    x = torch.zeros(2, 3, 4, requires_grad=True)
    res = ops.moe.balance_loss(x, torch.zeros(2, 3, 2, dtype=torch.int64))
    (res.loss.sum() if used == "loss" else res.z_loss.sum() if used == "z_loss" else res.loss.sum() + res.z_loss.sum()).backward()
    (up, up_z), = got
    assert (up is None) == (used == "z_loss") and (up_z is None) == (used == "loss") and x.grad.shape == x.shape


def test_c_abi_balance_loss_refuses_choices_past_32_bits():
    """A workgroup's choices are counted in 32 bits, four strides of its threads
    ahead of the last one."""
    lib = nat.load()

    def fwd(t, top):
        return lib.da_balance_loss(X, 0, 1, t, 4, 4, X, top, None, 0, 0, OUT, OUT, OUT, OUT, X, 1 << 40, None)

    for t, top in ((1, 0x7fffffff), (1, 0x7fffffff - 1023), (2, 0x3fffffff), (64, 33554430)):
        refused(fwd(t, top), nat.DA_ERR_UNSUPPORTED, "too many")


def test_sizes_past_the_c_types_are_refused():
    """Not cut to their low 32 or 64 bits: the tensors here are one entry, expanded."""
    x, index = torch.zeros(1, 4), torch.zeros(1, 2, dtype=torch.int64)
    wide, many = torch.zeros(1).expand(1, (1 << 32) + 4), torch.zeros(1, dtype=torch.int64).expand(1, (1 << 32) + 2)
    counts = torch.zeros(1, dtype=torch.int64).expand(1, (1 << 32) + 4)
    for bad in (lambda: ops.moe.balance_loss(wide, index), lambda: ops.moe.balance_loss(x, many),
                lambda: ops.moe.balance_loss_grad(None, None, wide, counts, torch.zeros(1, dtype=torch.int64))):
        with pytest.raises(NotImplementedError, match="32 bits"):
            bad()
    table, g = torch.zeros(8, 2), torch.zeros(2, 4, 5, 9)
    for start in (1 << 64, -(1 << 64), (1 << 26) + 1):
        for bad in (lambda: ops.relative_bias(table, 4, 4, q_start=start),
                    lambda: ops.relative_bias_grad(g, 8, q_start=start)):
            with pytest.raises(NotImplementedError, match="q_start"):
                bad()


def test_c_abi_refuses_launches_past_32_bits_of_threads():
    """A grid's threads, 256 a workgroup, are counted in 32 bits by the launch."""
    lib = nat.load()
    b = 1 << 24
    refused(lib.da_balance_loss(X, 0, b, 1, 4, 4, X, 2, None, 0, 0, OUT, OUT, OUT, OUT, X, 1 << 40, None),
            nat.DA_ERR_UNSUPPORTED, "too many")
    refused(lib.da_balance_loss_grad(X, X, X, 0, b, 1, 4, 4, X, X, None, 0, 0, OUT, 4, None), nat.DA_ERR_UNSUPPORTED,
            "too many")
    sides = (nat.QkSide * 2)()
    for side in sides:
        side.x = side.gz = side.out = side.weight = side.weight_grad = X
        side.heads = 1024
    refused(lib.da_qk_norm_rope_grad(sides, 2, 0, 8, 1 << 20, 8, 8, X, None, 0, 0, 1, None, 0, 0, 0, 1.0, 1e-6, X, 1 << 40,
                                     None), nat.DA_ERR_UNSUPPORTED, "up to")
