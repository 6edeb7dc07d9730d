"""A routed attention block captured as a whole: norms of queries and keys with
the rotation, a position bias, attention, a router with its balance loss, their
linear layers -- one batched pass under FusedCapture against one autograd pass
for each sample."""

from __future__ import annotations

import pytest
import torch
from torch import nn

from conftest import assert_parity
from dattri_llm_amd.gradient import FusedCapture, QKNormRope, RelativeBias, ops
from test_relative_bias_gpu import ids_of

pytestmark = pytest.mark.gpu
WIDTH, HEADS, KEYS, D, EXPERTS, TOP = 64, 4, 2, 16, 6, 2


class Block(nn.Module):
    def __init__(self):
        super().__init__()
        self.qkv = nn.Linear(WIDTH, (HEADS + 2 * KEYS) * D)
        self.rope = QKNormRope(D, rotary_dim=8)
        self.bias = RelativeBias(16, HEADS, max_distance=24, bidirectional=False, causal=True)
        self.out = nn.Linear(HEADS * D, WIDTH, bias=False)
        self.router = nn.Linear(WIDTH, EXPERTS, bias=False)
        self.experts = nn.ModuleList(nn.Linear(WIDTH, WIDTH, bias=False) for _ in range(EXPERTS))

    def forward(self, x, mask):
        b, t, _ = x.shape
        qkv = self.qkv(x).view(b, t, HEADS + 2 * KEYS, D)
        q, k = self.rope(qkv[:, :, :HEADS], qkv[:, :, HEADS:HEADS + KEYS], mask=mask)
        v = qkv[:, :, HEADS + KEYS:].repeat_interleave(HEADS // KEYS, 2).transpose(1, 2)
        k = k.repeat_interleave(HEADS // KEYS, 2).transpose(1, 2)
        scores = q.transpose(1, 2) @ k.transpose(2, 3).contiguous() / D ** 0.5
        scores = scores + self.bias(t, t, batch=b, mask=mask)
        scores = scores.masked_fill(~mask[:, None, None, :], -1e30)
        x = x + self.out((scores.softmax(-1) @ v).transpose(1, 2).reshape(b, t, -1))
        logits = self.router(x)
        _, index = ops.moe.router_topk(logits.detach(), TOP)
        index = index.view(b, t, TOP)
        p = logits.softmax(-1).gather(-1, index)
        y = torch.stack([e(x) for e in self.experts], 2)  # every expert on every token: the router decides the weights
        x = x + (p[..., None] * y.gather(2, index[..., None].expand(-1, -1, -1, WIDTH))).sum(2)
        return x, logits, index


def sample_losses(model, x, target, mask):
    y, logits, index = model(x, mask)
    task = ((y - target).square().mean(-1) * mask).sum(1)
    aux = ops.moe.balance_loss(logits, index, mask=mask)
    return task + 0.1 * aux.loss + 0.01 * aux.z_loss


def test_captured_block_matches_per_sample_autograd(device):
    torch.manual_seed(0)
    model = Block().to(device)
    with torch.no_grad():
        model.rope.q_weight.add_(0.1 * torch.randn(D, device=device))
        model.rope.k_weight.add_(0.1 * torch.randn(D, device=device))
    b, t = 5, 29
    x, target = torch.randn(b, t, WIDTH, device=device), torch.randn(b, t, WIDTH, device=device)
    mask = torch.arange(t, device=device)[None] < torch.tensor([29, 20, 29, 7, 1], device=device)[:, None]
    cap = FusedCapture(model)
    with cap:
        for part in (slice(0, 3), slice(3, 5)):  # two micro-batches
            sample_losses(model, x[part], target[part], mask[part]).sum().backward()
    block = cap.gradient()
    assert block.layer_types["rope.q_weight"] == "nn.RMSNorm" and block.layer_types["bias"] == "nn.Embedding"
    assert block.data["rope.k_weight"].shape == (b, D) and block.data["bias"].shape == (b, 16 * HEADS)
    dense = block.materialize()
    names = {n: n if n in ("rope.q_weight", "rope.k_weight") else f"{n}.weight" for n in block.layer_names}
    want: dict = {n: [] for n in names}
    params = dict(model.named_parameters())
    for i in range(b):
        model.zero_grad()
        sample_losses(model, x[i:i + 1], target[i:i + 1], mask[i:i + 1]).sum().backward()
        for n, pn in names.items():
            g = params[pn].grad
            bias = params.get(pn.replace("weight", "bias")) if pn == "qkv.weight" else None
            want[n].append((g if bias is None else torch.cat([g, bias.grad[:, None]], 1)).flatten())
    # Both sides are fp32 passes of the same arithmetic in other orders: the
    # attention and router between them leave a few 1e-6 of the largest entry.
    for n in names:
        assert_parity(dense.data[n], torch.stack(want[n]), "float32", tight=3e-5, label=n)
    # and its scores are the products of those gradients, all layers summed
    scores = ops.layerwise_cross_dot(block, block)
    rows = torch.cat([torch.stack(want[n]) for n in names], 1).double()
    assert_parity(scores if torch.is_tensor(scores) else sum(scores.values()), rows @ rows.T, "float32", tight=6e-5)


def test_new_tokens_one_at_a_time_equal_the_whole_prompt(device):
    """T = 1 with its position and one query row of the bias against the prompt's pass."""
    torch.manual_seed(1)
    b, t = 3, 40
    rope = QKNormRope(32, interleaved=True).to(device)
    bias = RelativeBias(32, 4, bidirectional=False, causal=True).to(device)
    q, k = torch.randn(b, t, 4, 32, device=device), torch.randn(b, t, 2, 32, device=device)
    with torch.no_grad():
        q_all, k_all = rope(q, k)
        full = bias(t, t)
        for i in (0, 1, 17, 39):
            at = torch.full((b, 1), i, device=device)
            q_one, k_one = rope(q[:, i:i + 1], k[:, i:i + 1], at)
            assert torch.equal(q_one, q_all[:, i:i + 1]) and torch.equal(k_one, k_all[:, i:i + 1])
            assert torch.equal(bias(1, t, q_start=i), full[:, i:i + 1])


def test_without_the_session_parameters_get_summed_gradients(device):
    torch.manual_seed(2)
    model = Block().to(device)
    x = torch.randn(2, 9, WIDTH, device=device)
    mask = torch.ones(2, 9, dtype=torch.bool, device=device)
    cap = FusedCapture(model, ["rope", "bias"])
    with cap:
        sample_losses(model, x, x.flip(1), mask).sum().backward()
    assert model.rope.q_weight.grad is None and model.bias.weight.grad is None and model.out.weight.grad is not None
    got = cap.gradient()
    model.zero_grad()
    sample_losses(model, x, x.flip(1), mask).sum().backward()
    assert torch.equal(got.data["rope.q_weight"].sum(0), model.rope.q_weight.grad)
    assert torch.equal(got.data["bias"].view(2, 16, HEADS).sum(0), model.bias.weight.grad)
    cap.clear()
    with pytest.raises(RuntimeError, match="no layer"):
        cap.gradient()


def test_no_second_derivatives(device):
    """A gradient of a gradient is refused, not taken for zero."""
    q, w = torch.randn(1, 3, 2, 16, device=device, requires_grad=True), torch.ones(16, device=device)
    freq = torch.ones(8, device=device)
    table = torch.randn(16, 2, device=device, requires_grad=True)
    logits = torch.randn(6, 4, device=device, requires_grad=True)
    index = torch.zeros(6, 1, dtype=torch.int64, device=device)
    for leaf, loss in ((q, ops.qk_norm_rope(q, None, w, None, freq)[0].square().sum()),
                       (table, ops.relative_bias(table, 5, 5).square().sum()),
                       (logits, ops.moe.balance_loss(logits, index).z_loss.square().sum())):
        (grad,) = torch.autograd.grad(loss, leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            grad.sum().backward()


@pytest.mark.parametrize("style", ["factorized", "materialized"])
def test_a_projected_session_keeps_these_gradients_whole(device, style):
    torch.manual_seed(3)
    model = Block().to(device)
    x = torch.randn(3, 11, WIDTH, device=device)
    mask = torch.ones(3, 11, dtype=torch.bool, device=device)
    whole, projected = FusedCapture(model), FusedCapture(model, proj_dim=8, capture_style=style)
    for cap in (whole, projected):
        with cap:
            sample_losses(model, x, x.flip(1), mask).sum().backward()
    a, b = whole.gradient(), projected.gradient()
    assert set(a.layer_names) == set(b.layer_names)
    for n in ("rope.q_weight", "rope.k_weight", "bias"):
        assert torch.equal(a.data[n], b.data[n])
    scores = ops.layerwise_cross_dot(b, b)
    want = sum((v := b.materialize().data[n].double().flatten(1)) @ v.T for n in b.layer_names)
    assert_parity(scores if torch.is_tensor(scores) else sum(scores.values()), want, "float32", tight=6e-5)


def test_a_frozen_block_is_captured_through_its_input(device):
    torch.manual_seed(4)
    model = Block().to(device)
    x = torch.randn(3, 11, WIDTH, device=device)
    mask = torch.ones(3, 11, dtype=torch.bool, device=device)
    got = []
    for frozen in (False, True):
        model.requires_grad_(not frozen)
        cap = FusedCapture(model)
        with cap:
            sample_losses(model, x.clone().requires_grad_(), x.flip(1), mask).sum().backward()
        got.append(cap.gradient().materialize())
    assert set(got[0].layer_names) == set(got[1].layer_names) and "bias" in got[1].layer_names
    for n in got[0].layer_names:
        assert_parity(got[1].data[n], got[0].data[n], "float32", label=n)
    assert all(p.grad is None for p in model.parameters())


@pytest.mark.parametrize("autocast", [False, True])
def test_captured_in_bf16(device, autocast):
    """Rotated norms and the bias in a bf16 model, and in an fp32 one under autocast.
    Whole numbers: rows and gradients of -1 and 1 at angle 0 and without an eps, so
    that the sums are exact but for the root of 1 (a step of 2^-23 of sums below
    160), and score gradients from -8 to 8, whose sums are exact."""
    torch.manual_seed(5)
    b, t, buckets = 3, 40, 8
    dt = torch.float32 if autocast else torch.bfloat16
    rope = QKNormRope(D, eps=0.0).to(device, dt)
    bias = RelativeBias(buckets, HEADS, max_distance=20).to(device, dt)
    q, k, gq, gk = (torch.randint(0, 2, (b, t, h, D), device=device).mul_(2).sub_(1).bfloat16()
                    for h in (HEADS, KEYS, HEADS, KEYS))
    gs = torch.randint(-8, 9, (b, HEADS, t, t), device=device).to(dt)
    cap = FusedCapture(nn.ModuleDict({"rope": rope, "bias": bias}))
    with cap, torch.autocast("cuda", torch.bfloat16, enabled=autocast):
        zq, zk = rope(q, k, torch.zeros(t, dtype=torch.int64, device=device))
        s = bias(t, t, batch=b)
        assert zq.dtype == zk.dtype == torch.bfloat16 and s.dtype == dt
        torch.autograd.backward([zq, zk, s], [gq, gk, gs])
    got = cap.gradient().data
    for name, x, g in (("rope.q_weight", q, gq), ("rope.k_weight", k, gk)):
        want = (x.float() * g.float()).sum((1, 2))
        assert got[name].dtype == torch.float32 and bool(((got[name] - want).abs() < 0.01).all())
    _, ids = ids_of(t, t, 0, buckets, 20, True)
    pick = nn.functional.one_hot(ids.flatten(), buckets).float().to(device)
    assert torch.equal(got["bias"].view(b, buckets, HEADS), (gs.float().flatten(2) @ pick).transpose(1, 2))
