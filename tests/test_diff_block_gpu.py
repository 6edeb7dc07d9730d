"""A decoder block and its answers as they are used together: residual additions with
their norm, difference attention with rotated maps, linear layers and the tokens' log
probabilities -- one batched pass under FusedCapture against one autograd pass for each
sample, against the formulas in 64 bits, token by token over a cache, and in graphs."""

from __future__ import annotations

import pytest
import torch
from torch import nn

from conftest import assert_parity
from dattri_llm_amd.gradient import AddRMSNorm, DiffAttention, FusedCapture, QKNormRope, ops

pytestmark = pytest.mark.gpu
WIDTH, HEADS, KEYS, D, DV, VOCAB = 64, 4, 2, 16, 32, 203


class Decoder(nn.Module):
    def __init__(self):
        super().__init__()
        self.norms = nn.ModuleList(AddRMSNorm(WIDTH) for _ in range(3))
        self.qkv = nn.Linear(WIDTH, (2 * HEADS + 2 * KEYS) * D + KEYS * DV)
        self.rope = QKNormRope(D)
        self.attend = DiffAttention(D, lambda_init=0.6, causal=True)
        self.out = nn.Linear(HEADS * DV, WIDTH, bias=False)
        self.mlp = nn.Sequential(nn.Linear(WIDTH, 2 * WIDTH), nn.GELU(), nn.Linear(2 * WIDTH, WIDTH, bias=False))
        self.head = nn.Linear(WIDTH, VOCAB, bias=False)

    def maps(self, x, mask, positions=None):
        b, t, _ = x.shape
        q, k, v = self.qkv(x).split([2 * HEADS * D, 2 * KEYS * D, KEYS * DV], -1)
        q, k = self.rope(q.reshape(b, t, 2 * HEADS, D), k.reshape(b, t, 2 * KEYS, D), positions, mask)
        return q, k, v.view(b, t, KEYS, DV)

    def tail(self, y, x, mask):
        y, x = self.norms[1](self.out(y.flatten(2)), x, mask)
        y, _ = self.norms[2](self.mlp(y), x, mask)
        return self.head(y)

    def forward(self, x, mask=None):
        q, k, v = self.maps(self.norms[0](x, mask=mask), mask)
        return self.tail(self.attend(q, k, v, mask, mask), x, mask)


def build(device, seed):
    torch.manual_seed(seed)
    model = Decoder().to(device)
    with torch.no_grad():
        for n in model.norms:
            n.weight.add_(0.1 * torch.randn(WIDTH, device=device))
    return model


def data(device, b, t, lengths=None):
    x = torch.randn(b, t, WIDTH, device=device)
    ids = torch.randint(0, VOCAB, (b, t), device=device)
    mask = None if lengths is None else torch.arange(t, device=device)[None] < torch.tensor(lengths, device=device)[:, None]
    return x, ids, mask


def losses(model, x, ids, mask):
    got = ops.token_logprobs(model(x, mask), ids, mask=mask, temperature=0.8)
    return -(got.logprob + 0.05 * got.entropy).sum(1)


def plain_losses(model, x, ids, mask):
    """The formulas in the model's dtype (64 bits), without the framework's operators."""
    live = torch.ones(x.shape[:2], dtype=torch.bool, device=x.device) if mask is None else mask
    b, t, _ = x.shape

    def norm(n, y):
        return y * (y.square().mean(-1, keepdim=True) + n.eps).rsqrt() * n.weight * live[..., None]

    def rope(y, w):
        y = y * (y.square().mean(-1, keepdim=True) + model.rope.eps).rsqrt() * w
        angle = torch.arange(t, device=x.device)[:, None] * model.rope.inv_freq.double()
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        a, e = y.chunk(2, -1)
        return torch.cat([a * c - e * s, e * c + a * s], -1)

    q, k, v = model.qkv(norm(model.norms[0], x)).split([2 * HEADS * D, 2 * KEYS * D, KEYS * DV], -1)
    q = rope(q.reshape(b, t, 2 * HEADS, D), model.rope.q_weight).view(b, t, HEADS, 2, D).permute(0, 2, 3, 1, 4)
    k = rope(k.reshape(b, t, 2 * KEYS, D), model.rope.k_weight).view(b, t, KEYS, 2, D).permute(0, 2, 3, 1, 4)
    k = k.repeat_interleave(HEADS // KEYS, 1)
    v = v.view(b, t, KEYS, DV).transpose(1, 2).repeat_interleave(HEADS // KEYS, 1)
    seen = torch.ones(t, t, dtype=torch.bool, device=x.device).tril() & live[:, None, None, None]
    p = (q @ k.transpose(-1, -2) / D ** 0.5).masked_fill(~seen, -1e300).softmax(-1)
    m = model.attend
    lam = (m.lambda_q1 @ m.lambda_k1).exp() - (m.lambda_q2 @ m.lambda_k2).exp() + m.lambda_init
    y = ((p[:, :, 0] - lam * p[:, :, 1]) @ v).transpose(1, 2) * live[..., None, None]
    x = (x + model.out(y.flatten(2))) * live[..., None]
    x = x + model.mlp(norm(model.norms[1], x))
    logp = (model.head(norm(model.norms[2], x)) / 0.8).log_softmax(-1)
    entropy = -(logp.exp() * logp).sum(-1)
    return -((logp.gather(-1, ids[..., None])[..., 0] + 0.05 * entropy) * live).sum(1)


def per_sample(model, names, call, b):
    """Gradients of each sample's loss, flattened as the capture lays them out."""
    params, rows = dict(model.named_parameters()), {n: [] for n in names}
    for i in range(b):
        model.zero_grad()
        call(slice(i, i + 1)).sum().backward()
        for n in names:
            if n in params:
                rows[n].append(params[n].grad.flatten().clone())
                continue
            g, bias = params[f"{n}.weight"].grad, params.get(f"{n}.bias")
            rows[n].append((g if bias is None else torch.cat([g, bias.grad[:, None]], 1)).flatten().clone())
    return {n: torch.stack(r) for n, r in rows.items()}


LENGTHS = [37, 20, 37, 7, 1]


def test_captured_block_matches_per_sample_autograd_and_the_formulas(device):
    model = build(device, 0)
    x, ids, mask = data(device, 5, 37, LENGTHS)
    cap = FusedCapture(model)
    with cap:
        for part in (slice(0, 3), slice(3, 5)):  # two micro-batches
            losses(model, x[part], ids[part], mask[part]).sum().backward()
    block = cap.gradient()
    vectors = [f"attend.lambda_{n}" for n in ("q1", "k1", "q2", "k2")]
    assert all(block.layer_types[n] == "nn.RMSNorm" for n in vectors + ["norms.0", "norms.1", "norms.2"])
    assert all(p.grad is None for p in model.parameters())
    dense, names = block.materialize(), block.layer_names
    assert set(vectors) < set(names) and block.data[vectors[0]].shape == (5, D)
    want = per_sample(model, names, lambda s: losses(model, x[s], ids[s], mask[s]), 5)
    # The same fp32 arithmetic in other orders, a few 1e-6 of the largest entry.
    for n in names:
        assert_parity(dense.data[n], want[n], "float32", tight=3e-5, label=n)
    scores = ops.layerwise_cross_dot(block, block)
    rows = torch.cat([want[n] for n in names], 1).double()
    assert_parity(scores if torch.is_tensor(scores) else sum(scores.values()), rows @ rows.T, "float32", tight=6e-5)
    exact = model.double()
    truth = per_sample(exact, names, lambda s: plain_losses(exact, x[s].double(), ids[s], mask[s]), 5)
    for n in names:
        assert_parity(dense.data[n], truth[n], "float32", tight=3e-5, label=f"{n} in 64 bits")


def test_without_the_session_parameters_get_summed_gradients(device):
    model = build(device, 1)
    x, ids, mask = data(device, 3, 18, [18, 5, 11])
    cap = FusedCapture(model, ["norms.0", "norms.2", "attend"])
    with cap:
        losses(model, x, ids, mask).sum().backward()
    assert model.norms[0].weight.grad is None and model.attend.lambda_k2.grad is None
    assert model.norms[1].weight.grad is not None and model.head.weight.grad is not None
    got = cap.gradient()
    model.zero_grad()
    losses(model, x, ids, mask).sum().backward()
    for n in ("norms.0", "norms.2"):
        assert torch.equal(got.data[n].sum(0), model.get_submodule(n).weight.grad)
    for n in ("q1", "k1", "q2", "k2"):
        assert_parity(got.data[f"attend.lambda_{n}"].sum(0), getattr(model.attend, f"lambda_{n}").grad, "float32")


def test_a_frozen_block_is_captured(device):
    x, ids, mask = data(device, 3, 11, [11, 4, 9])
    got = []
    for frozen in (False, True):
        model = build(device, 2).requires_grad_(not frozen)
        cap = FusedCapture(model)
        with cap:
            losses(model, x.clone().requires_grad_(), ids, mask).sum().backward()
        got.append(cap.gradient().materialize())
        assert all(p.grad is None for p in model.parameters())
    assert set(got[0].layer_names) == set(got[1].layer_names)
    for n in got[0].layer_names:
        assert_parity(got[1].data[n], got[0].data[n], "float32", label=n)


@pytest.mark.parametrize("autocast", [False, True])
def test_captured_in_bf16(device, autocast):
    """The captured gradients of a bf16 block and of an fp32 one under autocast sum to what
    the parameters get without the session, rounded to their type: the norms' by the same
    sum, the factor's vectors by another order of its sums over samples and heads."""
    model = build(device, 3).to(torch.float32 if autocast else torch.bfloat16)
    x, ids, mask = data(device, 4, 33, [33, 12, 30, 5])
    x = x.bfloat16()
    cap = FusedCapture(model, ["norms.0", "norms.1", "norms.2", "attend"])
    with torch.autocast("cuda", torch.bfloat16, enabled=autocast):
        with cap:
            losses(model, x, ids, mask).sum().backward()
        got = cap.gradient()
        model.zero_grad()
        losses(model, x, ids, mask).sum().backward()
    params = dict(model.named_parameters())
    for n in got.layer_names:
        want = params[f"{n}.weight" if n.startswith("norms") else n].grad
        assert got.data[n].dtype == torch.float32 and bool(got.data[n].abs().sum(1).all())
        if n.startswith("norms"):
            assert torch.equal(got.data[n].sum(0).to(want.dtype), want), n
        else:
            assert_parity(want, got.data[n].sum(0), "float32" if autocast else "bfloat16", label=n)


def test_no_second_derivatives(device):
    x, ids, _ = data(device, 2, 6)
    norm, attend = AddRMSNorm(WIDTH).to(device), DiffAttention(D).to(device)
    q = torch.randn(2, 6, 2, D, device=device, requires_grad=True)
    x.requires_grad_()
    logits = torch.randn(2, 6, VOCAB, device=device, requires_grad=True)
    for leaf, loss in ((x, norm(x, x)[0].square().sum()), (q, attend(q, q, x.detach()[:, :, None]).square().sum()),
                       (logits, ops.token_logprobs(logits, ids).logprob.square().sum())):
        (grad,) = torch.autograd.grad(loss, leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            grad.sum().backward()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@torch.no_grad()
def test_new_tokens_one_at_a_time_equal_the_whole_prompt(device, dt):
    """A cache longer than what is filled, its unfilled part NaN behind a mask; the norm's
    rows equal bit by bit, the attention's as near as two orders of the sums leave them:
    in bf16 half a step of the output beside half a step of each probability."""
    model = build(device, 4).to(dt)
    b, t, room = 3, 70, 130
    x, ids, _ = data(device, b, t)
    x = x.to(dt)
    y = model.norms[0](x)
    q, k, v = model.maps(y, None)
    whole = model.attend(q, k, v)
    logits = model.tail(whole, x, None)
    answers = ops.token_logprobs(logits, ids, top=5)
    cache = [torch.full((b, room, *z.shape[2:]), float("nan"), dtype=dt, device=device) for z in (k, v)]
    filled = torch.zeros(b, room, dtype=torch.bool, device=device)
    for i in range(t):
        at = torch.full((b, 1), i, device=device)
        y_one = model.norms[0](x[:, i:i + 1])
        assert torch.equal(y_one, y[:, i:i + 1])
        _, k_one, v_one = model.maps(y_one, None, at)
        cache[0][:, i], cache[1][:, i], filled[:, i] = k_one[:, 0], v_one[:, 0], True
        if i % 23 not in (0, 11) and i != t - 1:
            continue
        one = model.attend(q[:, i:i + 1], cache[0], cache[1], filled, q_start=i)
        u = torch.finfo(dt).eps / 2 if dt == torch.bfloat16 else 2e-6
        bound = 2 * u * (1 + 2 * model.attend.factor().abs()) * v.abs().amax() + 2e-6
        assert bool(((one - whole[:, i:i + 1]).abs() <= bound).all()), i
        told = ops.token_logprobs(logits[:, i:i + 1], ids[:, i:i + 1], top=5)
        assert torch.equal(told.top_index, answers.top_index[:, i:i + 1])
        assert bool(((told.logprob - answers.logprob[:, i:i + 1]).abs() < 1e-5).all())


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_rows_and_keys_that_see_nothing_may_hold_anything(device, dt):
    """Queries before the first key, queries whose keys are all masked, and keys behind the
    last query: NaN there, in the gradient that arrives too, reaches nothing else."""
    torch.manual_seed(7)
    b, t, s, h, hk, d, dv = 2, 90, 140, 4, 2, 32, 64
    start = -20  # rows 0 .. 19 see nothing, keys 70 .. 139 are seen by none
    q, k, v, g = (torch.randn(b, n, m, w, device=device).to(dt)
                  for n, m, w in ((t, 2 * h, d), (s, 2 * hk, d), (s, hk, dv), (t, h, dv)))
    lam = torch.full((h,), 0.4, device=device)
    mask = torch.ones(b, s, dtype=torch.bool, device=device)
    mask[1, :8] = False  # and in the second sample rows 20 .. 27
    rows = torch.zeros(b, t, dtype=torch.bool, device=device)
    rows[:, :20], rows[1, :28] = True, True
    keys = ~mask
    keys[:, 70:] = True
    got = []
    for fill in (0.0, float("nan")):
        q[rows], g[rows], k[keys], v[keys] = fill, fill, fill, fill
        out, state = ops.diff_attention(q, k, v, lam, causal=True, q_start=start, mask=mask, return_state=True)
        got.append((out, *ops.diff_attention_grad(g, q, k, v, lam, out, state, causal=True, q_start=start, mask=mask)))
        out, dq, dk, dval, dlam = got[-1]
        assert not out[rows].any() and not dq[rows].any() and not dk[keys].any() and not dval[keys].any()
        assert all(bool(x.isfinite().all()) for x in got[-1])
    assert all(torch.equal(x, y) for x, y in zip(*got))


@pytest.mark.parametrize("masked", [False, True])
def test_a_long_run_of_tiles_gives_the_same_results_every_time(device, masked):
    """Tiles are read ahead into LDS: with every CU busy they come late, and must be awaited."""
    torch.manual_seed(8)
    b, t, h, hk, d, dv = 2, 2048, 32, 8, 64, 128
    q, k, v, g = (torch.randn(b, t, m, w, device=device).bfloat16() for m, w in ((2 * h, d), (2 * hk, d), (hk, dv), (h, dv)))
    lam = torch.rand(h, device=device)
    mask = torch.arange(t, device=device)[None] < torch.tensor([2000, 2048], device=device)[:, None] if masked else None
    first = None
    for _ in range(6):
        out, state = ops.diff_attention(q, k, v, lam, causal=True, mask=mask, return_state=True)
        got = (out, state.lse, *ops.diff_attention_grad(g, q, k, v, lam, out, state, causal=True, mask=mask))
        assert all(bool(x.isfinite().all()) for x in got)
        first = got if first is None else first
        assert all(torch.equal(x, y) for x, y in zip(got, first))


def test_on_another_stream(device):
    model = build(device, 5)
    x, ids, mask = data(device, 3, 40, [40, 3, 25])
    want = losses(model, x, ids, mask)
    want.sum().backward()
    grads = [p.grad.clone() for p in model.parameters()]
    model.zero_grad()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = losses(model, x, ids, mask)
        got.sum().backward()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    for (n, p), g in zip(model.named_parameters(), grads):
        assert_parity(p.grad, g, "float32", label=n)


def test_two_captured_chains_replay_in_turn(device):
    """Norm, attention and log probabilities of two sizes with their backward passes, each
    in a graph of its own, replayed in turn with eager work between."""
    torch.manual_seed(6)
    w = torch.randn(WIDTH, device=device)
    lam = torch.full((2,), 0.4, device=device)

    def chain(x, r, ids):
        b, t, _ = x.shape
        out, total, _ = ops.add_rms_norm(x, r, w)
        q = out.view(b, t, 4, D)
        o, state = ops.diff_attention(q, q, total.view(b, t, 2, 2 * D), lam, causal=True, return_state=True)
        z = o.flatten(2)
        p = ops.token_logprobs(z, ids)
        up = torch.ones_like(p.logprob)
        gz = ops.token_logprobs_grad(up, None, z, ids, p.lse, p.entropy)
        dq, dk, dv, dlam = ops.diff_attention_grad(gz.view_as(o), q, q, total.view(b, t, 2, 2 * D), lam, o, state,
                                                   causal=True)
        dx, dw = ops.add_rms_norm_grad((dq + dk).flatten(2), dv.flatten(2), total, w)
        return out, total, o, p.logprob, p.entropy, gz, dq, dk, dv, dlam, dx, dw

    inputs, graphs, results = [], [], []
    for b, t in ((2, 300), (1, 1)):
        inputs.append([torch.randn(b, t, WIDTH, device=device), torch.randn(b, t, WIDTH, device=device),
                       torch.randint(0, WIDTH, (b, t), device=device)])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            chain(*inputs[-1])
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(chain(*inputs[-1]))
        graphs.append(g)
    for turn in range(4):
        for args, g, got in zip(inputs, graphs, results):
            for a in args:
                a.copy_(torch.randn_like(a) if a.is_floating_point() else torch.randint_like(a, WIDTH))
            g.replay()
            torch.cuda.synchronize()
            for n, (a, e) in enumerate(zip(got, chain(*args))):
                assert torch.equal(a, e), (turn, n)
