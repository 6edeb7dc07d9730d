"""The operators around a captured block's attention and router, and the work they are measured on.

A case is one pass through an operator over data that a program already holds
on the GPU.  Kinds:

* ``qk_forward`` / ``qk_backward``: :func:`ops.qk_norm_rope` and
  :func:`ops.qk_norm_rope_grad` -- RMS norms of the queries and keys of each
  head with the position rotation, and their gradients (the norm weights' per
  sample);
* ``bias_forward`` / ``bias_backward``: :func:`ops.relative_bias` and
  :func:`ops.relative_bias_grad` -- a learned position bias by buckets, and its
  per-sample gradient;
* ``balance``: :func:`ops.moe.balance_loss` and :func:`ops.moe.balance_loss_grad`
  -- the router's balance and z losses with per-expert counts, and the
  gradient of the logits.

With ``own`` unset, :func:`run` computes the same from elementary torch
operations in 32 bits (64 for the angles and the long sums).
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _ops():
    path = os.path.join(os.getcwd(), "dattri-llm_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from dattri_llm_amd.gradient import ops

    return ops


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------


def listed() -> list[dict]:
    return [
        # One new token of sixteen sequences, far into a long context: 32 query heads, 8 key heads of 128.
        {"name": "qk_token_bf16", "kind": "qk_forward", "b": 16, "t": 1, "hq": 32, "hk": 8, "d": 128, "rot": 128,
         "interleaved": False, "layout": "fused", "start": 100_000, "pad": 0.0, "dtype": "bf16"},
        # A train block's forward pass: eight sequences of 2048 tokens, queries and keys read out of one fused
        # projection's output.
        {"name": "qk_forward_bf16", "kind": "qk_forward", "b": 8, "t": 2048, "hq": 32, "hk": 8, "d": 128, "rot": 128,
         "interleaved": False, "layout": "fused", "start": 0, "pad": 0.0, "dtype": "bf16"},
        # The same block's backward pass with the weights' per-sample gradients.
        {"name": "qk_backward_bf16", "kind": "qk_backward", "b": 8, "t": 2048, "hq": 32, "hk": 8, "d": 128,
         "rot": 128, "interleaved": False, "layout": "fused", "start": 0, "pad": 0.0, "dtype": "bf16"},
        # A smaller fp32 model: heads of 80 of which 32 entries rotate in adjacent pairs, odd length, padded
        # sequences.
        {"name": "qk_backward_fp32", "kind": "qk_backward", "b": 6, "t": 509, "hq": 12, "hk": 12, "d": 80, "rot": 32,
         "interleaved": True, "layout": "heads", "start": 0, "pad": 0.2, "dtype": "fp32"},
        # The bias of one new token against a cache of 4097 positions.
        {"name": "bias_token_bf16", "kind": "bias_forward", "h": 32, "tq": 1, "tk": 4097, "start": 4096,
         "buckets": 32, "far": 128, "both": False, "causal": True, "dtype": "bf16"},
        # A bidirectional encoder's bias over 2048 tokens.
        {"name": "bias_forward_bf16", "kind": "bias_forward", "h": 32, "tq": 2048, "tk": 2048, "start": 0,
         "buckets": 32, "far": 128, "both": True, "causal": False, "dtype": "bf16"},
        # A train block's score gradients: sixteen sequences of 1024 tokens, sixteen heads.
        {"name": "bias_backward_bf16", "kind": "bias_backward", "b": 16, "h": 16, "tq": 1024, "tk": 1024, "start": 0,
         "buckets": 32, "far": 128, "both": True, "causal": False, "pad": 0.0, "dtype": "bf16"},
        # A decoder's in fp32: causal, odd length, padded sequences.
        {"name": "bias_backward_fp32", "kind": "bias_backward", "b": 4, "h": 12, "tq": 777, "tk": 777, "start": 0,
         "buckets": 32, "far": 128, "both": False, "causal": True, "pad": 0.2, "dtype": "fp32"},
        # A small routed layer, one loss for each sample.
        {"name": "balance_tiny_fp32", "kind": "balance", "b": 8, "t": 64, "experts": 8, "top": 2, "pad": 0.0,
         "dtype": "fp32"},
        # One side of a routed layer's scoring pass: 16 x 256 tokens, 8 experts, top-2.
        {"name": "balance_8_bf16", "kind": "balance", "b": 16, "t": 256, "experts": 8, "top": 2, "pad": 0.0,
         "dtype": "bf16"},
        # 4096 tokens over 128 experts, top-8, as one batch-level loss.
        {"name": "balance_128_fp32", "kind": "balance", "b": 1, "t": 4096, "experts": 128, "top": 8, "pad": 0.0,
         "dtype": "fp32"},
        # A long-context train block of a many-expert router, padded sequences, one loss for each.
        {"name": "balance_long_bf16", "kind": "balance", "b": 32, "t": 4096, "experts": 128, "top": 8, "pad": 0.1,
         "dtype": "bf16"},
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_one(rng: random.Random) -> dict:
    kind = rng.choice(["qk_forward", "qk_backward", "bias_forward", "bias_backward", "balance"])
    dtype = rng.choice(["bf16", "bf16", "fp32", "fp16"])
    if kind.startswith("qk"):
        d = rng.choice([64, 80, 96, 128, 128, 256, 2 * rng.randint(2, 128)])
        rot = rng.choice([d, d, d, d // 4 * 2, 2 * rng.randint(1, d // 2)])
        group = rng.choice([1, 2, 4, 8])
        hk = _log(rng, 1, 16)
        return {"kind": kind, "b": _log(rng, 1, 32), "t": 1 if rng.random() < 0.2 else _log(rng, 2, 8192),
                "hq": hk * group, "hk": hk, "d": d, "rot": rot, "interleaved": rng.random() < 0.3,
                "layout": rng.choice(["fused", "plain", "heads"]),
                "start": 0 if rng.random() < 0.5 else _log(rng, 1, 1_000_000),
                "pad": rng.choice([0.0, 0.0, 0.2]), "dtype": dtype}
    if kind.startswith("bias"):
        tq = 1 if rng.random() < 0.15 else _log(rng, 2, 2048)
        same = rng.random() < 0.6 and tq > 1
        tk = tq if same else _log(rng, max(tq, 16), 8192)
        both = rng.random() < 0.5
        buckets = rng.choice([16, 32, 32, 64, 128])
        c = {"kind": kind, "h": _log(rng, 1, 64), "tq": tq, "tk": tk, "start": tk - tq, "buckets": buckets,
             "far": max(buckets, _log(rng, 64, 2048)), "both": both, "causal": not both and rng.random() < 0.7,
             "dtype": dtype}
        if kind == "bias_backward":
            c.update(b=_log(rng, 1, 32), pad=rng.choice([0.0, 0.0, 0.2]))
        return c
    experts = rng.choice([8, 16, 64, 128, 256, rng.randint(2, 256)])
    return {"kind": kind, "b": _log(rng, 1, 64), "t": 1 if rng.random() < 0.1 else _log(rng, 2, 8192),
            "experts": experts, "top": rng.randint(1, min(8, experts)), "pad": rng.choice([0.0, 0.0, 0.2]),
            "dtype": dtype}


_MOST = {"qk": 2 * 8 * 2048 * 40 * 128, "bi": 16 * 16 * 1024 * 1024, "ba": 32 * 4096 * 128}


def _elements(c: dict) -> int:
    if c["kind"].startswith("qk"):
        return c["b"] * c["t"] * (c["hq"] + c["hk"]) * c["d"] * (BYTES[c["dtype"]] // 2) * 2
    if c["kind"].startswith("bias"):
        return c.get("b", 1) * c["h"] * c["tq"] * c["tk"] * (BYTES[c["dtype"]] // 2)
    return c["b"] * c["t"] * c["experts"] * (BYTES[c["dtype"]] // 2)


def draw(rng: random.Random) -> dict:
    """One more case of the listed ranges, no dearer than the largest of its family."""
    while True:
        c = _draw_one(rng)
        if _elements(c) <= _MOST[c["kind"][:2]]:
            return c


# ---------------------------------------------------------------------------
# What the program has in hand
# ---------------------------------------------------------------------------


def _edges(case: dict) -> list[int]:
    """The least distance of each bucket of one side: bucket ``x`` holds the
    distances from ``edges[x]`` up to the next one.  The first half are single
    distances m; above, the least r with (r/m)^(n-m) >= (far/m)^j, in integers."""
    n = case["buckets"] // (2 if case["both"] else 1)
    m, far = n // 2, case["far"]
    edges = list(range(m + 1))
    for j in range(1, n - m):
        r = edges[-1]
        while r ** (n - m) * m ** j < far ** j * m ** (n - m):
            r += 1
        edges.append(r)
    return edges


def _mask(case: dict, b: int, t: int, gen: torch.Generator, dev) -> torch.Tensor | None:
    """(b, t) live positions: each sequence ends up to ``pad`` of the length early."""
    if not case.get("pad"):
        return None
    cut = (torch.rand(b, 1, generator=gen, device=dev) * case["pad"] * t).long()
    return torch.arange(t, device=dev)[None] < t - cut


def _heads(case: dict, gen: torch.Generator, dev, dt):
    """Queries and keys (b, t, heads, d) in the case's layout."""
    b, t, hq, hk, d = case["b"], case["t"], case["hq"], case["hk"], case["d"]
    if case["layout"] == "fused":  # slices of one projection's output that holds the values too
        x = torch.randn(b, t, hq + 2 * hk, d, generator=gen, device=dev, dtype=dt)
        return x[:, :, :hq], x[:, :, hq:hq + hk]
    if case["layout"] == "heads":  # heads before tokens
        return (torch.randn(b, h, t, d, generator=gen, device=dev, dtype=dt).transpose(1, 2) for h in (hq, hk))
    return (torch.randn(b, t, h, d, generator=gen, device=dev, dtype=dt) for h in (hq, hk))


def prepare(case: dict, seed: int) -> dict:
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    s = {"case": case}

    def normal(*shape, scale=1.0, dtype=dt):
        return torch.randn(*shape, generator=gen, device=dev, dtype=dtype) * scale

    if case["kind"].startswith("qk"):
        b, t, d, rot = case["b"], case["t"], case["d"], case["rot"]
        s["q"], s["k"] = _heads(case, gen, dev, dt)
        s["wq"], s["wk"] = 1 + normal(d, scale=0.1), 1 + normal(d, scale=0.1)
        s["inv_freq"] = (10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)).float()
        first = case["start"] + torch.randint(0, 64, (b, 1), generator=gen, device=dev)
        s["positions"] = first + torch.arange(t, device=dev)
        s["mask"] = _mask(case, b, t, gen, dev)
        if case["kind"] == "qk_backward":  # what attention's backward gives: heads before tokens
            s["gq"] = normal(b, case["hq"], t, d, scale=0.02).transpose(1, 2)
            s["gk"] = normal(b, case["hk"], t, d, scale=0.02).transpose(1, 2)
        return s
    if case["kind"] == "bias_forward":
        s["table"] = normal(case["buckets"], case["h"])
        s["edges"] = torch.tensor(_edges(case), device=dev)
        return s
    if case["kind"] == "bias_backward":
        b, h, tq, tk = case["b"], case["h"], case["tq"], case["tk"]
        g = normal(b, h, tq, tk, scale=1 / 16)
        g.mul_(torch.rand(b, h, tq, 1, generator=gen, device=dev).to(dt))  # rows of different weight
        s["mask"] = _mask(case, b, tk, gen, dev)
        if s["mask"] is not None:  # what masked attention leaves: nothing
            g.mul_(s["mask"][:, None, None, :])
            g.mul_(s["mask"][:, None, case["start"]:case["start"] + tq, None])
        if case["causal"]:
            g.mul_(torch.ones(tq, tk, device=dev, dtype=dt).tril_(case["start"]))
        s["g"], s["edges"] = g, torch.tensor(_edges(case), device=dev)
        return s
    b, t, e = case["b"], case["t"], case["experts"]
    favour = torch.randn(e, generator=gen, device=dev)
    s["logits"] = (torch.randn(b * t, e, generator=gen, device=dev) + favour).to(dt)
    s["index"] = torch.topk(s["logits"].float(), case["top"], dim=-1).indices
    s["mask"] = _mask(case, b, t, gen, dev)
    s["up"] = 0.01 * (1 + torch.rand(b, generator=gen, device=dev))
    s["up_z"] = 0.001 * (1 + torch.rand(b, generator=gen, device=dev))
    return s


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------


def _angles(s: dict):
    """cos and sin (b, t, 1, rot/2), the angles in 64 bits."""
    angle = s["positions"].double()[:, :, None, None] * s["inv_freq"].double()
    return angle.cos().float(), angle.sin().float()


def _pairs(x: torch.Tensor, case: dict):
    """The two entries of each rotated pair, and the entries that stay."""
    rot = case["rot"]
    if case["interleaved"]:
        return x[..., 0:rot:2], x[..., 1:rot:2], x[..., rot:]
    return x[..., :rot // 2], x[..., rot // 2:rot], x[..., rot:]


def _unpair(a: torch.Tensor, b: torch.Tensor, rest: torch.Tensor, case: dict) -> torch.Tensor:
    if case["interleaved"]:
        return torch.cat([torch.stack([a, b], dim=-1).flatten(-2), rest], dim=-1)
    return torch.cat([a, b, rest], dim=-1)


def _live(x: torch.Tensor, mask: torch.Tensor | None) -> torch.Tensor:
    return x if mask is None else torch.where(mask[:, :, None, None], x, 0)


def _qk_one(x, w, cos, sin, s):
    case = s["case"]
    x = _live(x.float(), s["mask"])
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()
    a, b, rest = _pairs(y, case)
    return _live(_unpair(a * cos - b * sin, b * cos + a * sin, rest, case), s["mask"])


def _qk_one_grad(x, gz, w, cos, sin, s):
    case = s["case"]
    x, gz = _live(x.float(), s["mask"]), _live(gz.float(), s["mask"])
    a, b, rest = _pairs(gz, case)
    gy = _unpair(a * cos + b * sin, b * cos - a * sin, rest, case)
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
    x_hat = x * r
    g = gy * w.float()
    return r * (g - x_hat * (g * x_hat).mean(-1, keepdim=True)), (gy * x_hat).sum(2).double().sum(1).float()


def _buckets(case: dict, edges: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The offsets j - i - start of a (tq, tk) square from the least to the
    largest, and the bucket of each."""
    rel = torch.arange(1 - case["tq"] - case["start"], case["tk"] - case["start"], device=edges.device)
    away = rel.abs() if case["both"] else (-rel).clamp(min=0)
    bucket = (away[:, None] >= edges[1:]).sum(-1)
    return rel, bucket + (rel > 0) * (case["buckets"] // 2) if case["both"] else bucket


def _bias(s: dict) -> torch.Tensor:
    case = s["case"]
    rel, bucket = _buckets(case, s["edges"])
    line = s["table"].float().t()[:, bucket]  # (h, offsets)
    if case["causal"]:
        line = torch.where(rel > 0, -math.inf, line)
    at = torch.arange(case["tk"], device=rel.device) + (case["tq"] - 1 - torch.arange(case["tq"], device=rel.device))[:, None]
    return line.to(s["table"].dtype)[:, at]


def _bias_grad(s: dict) -> torch.Tensor:
    case, tq, tk = s["case"], s["case"]["tq"], s["case"]["tk"]
    rel, bucket = _buckets(case, s["edges"])
    g = s["g"].float()
    if s["mask"] is not None:
        rows = s["mask"][:, case["start"]:case["start"] + tq]
        g = torch.where(rows[:, None, :, None] & s["mask"][:, None, None, :], g, 0)
    # Rows from the last to the first, tq wide zeros after each: read with a
    # row length one less, every diagonal is a column.
    g = torch.nn.functional.pad(g.flip(-2), (0, tq)).flatten(-2)[..., :tq * (tk + tq - 1)]
    line = g.unflatten(-1, (tq, tk + tq - 1)).sum(-2)  # (b, h, offsets)
    if case["causal"]:
        line = torch.where(rel > 0, 0, line)
    chosen = (bucket[:, None] == torch.arange(case["buckets"], device=rel.device)).double()
    return (line.double() @ chosen).transpose(1, 2).float()  # (b, buckets, h)


def _balance(s: dict):
    case = s["case"]
    b, t, e = case["b"], case["t"], case["experts"]
    x = s["logits"].float().view(b, t, e)
    mask = s["mask"] if s["mask"] is not None else torch.ones(b, t, dtype=torch.bool, device=x.device)
    live = mask.sum(1)
    n = live.clamp(min=1).float()
    lse = x.max(-1).values
    ex = (x - lse[..., None]).exp()
    total = ex.sum(-1)
    p, lse = ex / total[..., None], lse + total.log()
    p, lse = torch.where(mask[..., None], p, 0), torch.where(mask, lse, 0)
    chosen = (s["index"].view(b, t, -1)[..., None] == torch.arange(e, device=x.device)) & mask[..., None, None]
    counts = chosen.sum((1, 2))
    f = counts.float() / n[:, None]
    loss = e * (f * (p.double().sum(1).float() / n[:, None])).sum(-1)
    z = lse.square().double().sum(1).float() / n
    up, up_z = (s["up"] * e / n)[:, None, None], (2 * s["up_z"] / n)[:, None, None]
    f = f[:, None]
    grad = up * p * (f - (f * p).sum(-1, keepdim=True)) + up_z * lse[..., None] * p
    return loss, z, counts, grad.view(b * t, e).to(s["logits"].dtype)


def run(s: dict):
    case = s["case"]
    kind = case["kind"]
    if own:
        ops = _ops()
        if kind == "qk_forward":
            return ops.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["inv_freq"], s["positions"], eps=1e-6,
                                    interleaved=case["interleaved"], mask=s["mask"])
        if kind == "qk_backward":
            return ops.qk_norm_rope_grad(s["gq"], s["gk"], s["q"], s["k"], s["wq"], s["wk"], s["inv_freq"],
                                         s["positions"], eps=1e-6, interleaved=case["interleaved"], mask=s["mask"])
        if kind == "bias_forward":
            return ops.relative_bias(s["table"], case["tq"], case["tk"], q_start=case["start"],
                                     bidirectional=case["both"], max_distance=case["far"], causal=case["causal"])
        if kind == "bias_backward":
            return ops.relative_bias_grad(s["g"], case["buckets"], q_start=case["start"],
                                          bidirectional=case["both"], max_distance=case["far"],
                                          causal=case["causal"], mask=s["mask"])
        got = ops.moe.balance_loss(s["logits"], s["index"], batch=case["b"], mask=s["mask"])
        grad = ops.moe.balance_loss_grad(s["up"], s["up_z"], s["logits"], got.counts, got.live, mask=s["mask"])
        return got.loss, got.z_loss, got.counts.long(), grad
    if kind.startswith("qk"):
        cos, sin = _angles(s)
        if kind == "qk_forward":
            return (_qk_one(s["q"], s["wq"], cos, sin, s).to(s["q"].dtype),
                    _qk_one(s["k"], s["wk"], cos, sin, s).to(s["k"].dtype))
        dq, dwq = _qk_one_grad(s["q"], s["gq"], s["wq"], cos, sin, s)
        dk, dwk = _qk_one_grad(s["k"], s["gk"], s["wk"], cos, sin, s)
        return dq.to(s["q"].dtype), dk.to(s["k"].dtype), dwq, dwk
    if kind == "bias_forward":
        return _bias(s)
    if kind == "bias_backward":
        return _bias_grad(s)
    return _balance(s)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------


def work(case: dict) -> dict:
    es = BYTES[case["dtype"]]
    kind = case["kind"]
    if kind.startswith("qk"):
        n = case["b"] * case["t"] * (case["hq"] + case["hk"]) * case["d"]
        extra = case["b"] * case["t"] * 8 + case["rot"] * 2 + 2 * case["d"] * es
        if kind == "qk_forward":
            return {"bytes": 2 * n * es + extra, "flops": 8 * n}
        return {"bytes": 3 * n * es + extra + 8 * case["b"] * case["d"], "flops": 16 * n}
    if kind.startswith("bias"):
        n = case.get("b", 1) * case["h"] * case["tq"] * case["tk"]
        table = case["buckets"] * case["h"]
        if kind == "bias_forward":
            return {"bytes": n * es + table * es, "flops": n}
        if case["causal"]:  # the live triangle (the rows of a square end at their own position)
            n = case["b"] * case["h"] * (case["tq"] * case["start"] + case["tq"] * (case["tq"] + 1) // 2)
        return {"bytes": n * es + 4 * case["b"] * table, "flops": n}
    n = case["b"] * case["t"]
    return {"bytes": 2 * n * case["experts"] * es + 8 * n * case["top"] + 4 * case["b"] * (case["experts"] + 4),
            "flops": 16 * n * case["experts"]}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------


def _exact_qk(x, w, s, gz=None):
    """One side from the definition: each pair as one complex number that the
    position turns, each row divided by its root mean square."""
    case = s["case"]
    rot, d = case["rot"], case["d"]
    order = list(range(0, rot, 2)) + list(range(1, rot, 2)) if case["interleaved"] else list(range(rot))
    order = torch.tensor(order + list(range(rot, d)), device=x.device)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                       s["positions"].double()[..., None, None] * s["inv_freq"].double())
    dead = torch.zeros_like(s["positions"], dtype=torch.bool) if s["mask"] is None else ~s["mask"]
    x = x.double().masked_fill(dead[..., None, None], 0.0)
    rms = ((x * x).sum(-1, keepdim=True) / d + 1e-6).sqrt()
    norm, w = x / rms, w.double()

    def turned(v, by):
        v = v[..., order]
        c = torch.complex(v[..., :rot // 2], v[..., rot // 2:rot]) * by
        return torch.empty_like(v).index_copy_(-1, order, torch.cat([c.real, c.imag, v[..., rot:]], -1))

    if gz is None:
        return turned(norm * w, turn).masked_fill(dead[..., None, None], 0.0)
    gy = turned(gz.double().masked_fill(dead[..., None, None], 0.0), turn.conj())
    along = (gy * w * norm).sum(-1, keepdim=True) / d
    return (gy * w - norm * along) / rms, (gy * norm).sum((1, 2))


def _exact_bucket(rel: int, case: dict) -> int:
    n = case["buckets"]
    add = 0
    if case["both"]:
        n //= 2
        add = n if rel > 0 else 0
        r = abs(rel)
    else:
        r = max(-rel, 0)
    m = n // 2
    if r < m:
        return add + r
    j = 0  # the largest j below n - m with (r / m) ** (n - m) >= (far / m) ** j
    while j + 1 < n - m and r ** (n - m) * m ** (j + 1) >= case["far"] ** (j + 1) * m ** (n - m):
        j += 1
    return add + m + j


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "qk_forward":
        return _exact_qk(s["q"], s["wq"], s), _exact_qk(s["k"], s["wk"], s)
    if kind == "qk_backward":
        dq, dwq = _exact_qk(s["q"], s["wq"], s, s["gq"])
        dk, dwk = _exact_qk(s["k"], s["wk"], s, s["gk"])
        return dq, dk, dwq, dwk
    if kind.startswith("bias"):
        tq, tk, start = case["tq"], case["tk"], case["start"]
        limit = 2 * max(case["far"], case["buckets"])  # everything further is in the last bucket
        near = torch.tensor([_exact_bucket(r, case) for r in range(-limit, limit + 1)], device="cuda")
        rel = torch.arange(tk, device="cuda") - torch.arange(tq, device="cuda")[:, None] - start
        ids = near[rel.clamp(-limit, limit) + limit]
        if kind == "bias_forward":
            out = s["table"].double()[ids].permute(2, 0, 1).contiguous()
            return out.masked_fill_(rel > 0, -math.inf) if case["causal"] else out
        g = s["g"].double()
        if s["mask"] is not None:
            g = g * (s["mask"][:, None, None, :] * s["mask"][:, None, start:start + tq, None])
        if case["causal"]:
            g = g * (rel <= 0)
        return torch.stack([(g * (ids == v)).sum((2, 3)) for v in range(case["buckets"])], dim=1)
    b, t, e = case["b"], case["t"], case["experts"]
    x = s["logits"].double().view(b, t, e).requires_grad_()
    live = torch.ones(b, t, dtype=torch.float64, device="cuda") if s["mask"] is None else s["mask"].double()
    n = live.sum(1).clamp(min=1)
    chosen = torch.zeros(b, t, e, dtype=torch.float64, device="cuda")
    chosen.scatter_(2, s["index"].view(b, t, -1), 1.0)
    part = torch.einsum("bte,bt->be", chosen, live) / n[:, None]
    mean = (torch.softmax(x, -1) * live[..., None]).sum(1) / n[:, None]
    loss, z = e * (part * mean).sum(-1), (torch.logsumexp(x, -1).square() * live).sum(1) / n
    ((loss * s["up"].double()).sum() + (z * s["up_z"].double()).sum()).backward()
    return loss.detach(), z.detach(), None, x.grad.view(b * t, e)
