"""The learned parts of attention beside its linear layers: the norms of queries
and keys with the position rotation, the relative position bias, and attention
by the difference of two softmax maps.

They hold parameters whose per-sample gradient cannot be formed from the
layer's own input and output, as the reference does for its norm and embedding
layers (``dattri_llm/gradient/ops/materialize.py:22-48``, ``:96-98``): the
norms' output gradient is known only behind the rotation, and a bias table is
looked up once for the whole batch, so that the gradient which reaches it is
already summed over the samples, as is that of the factor between two maps.
Here the backward pass of each operator gives the per-sample gradient itself:

* :func:`qk_norm_rope` / :func:`qk_norm_rope_grad` (``da_qk_norm_rope``);
* :func:`relative_bias` / :func:`relative_bias_grad` (``da_relative_bias``);
* :func:`diff_attention` / :func:`diff_attention_grad` (``da_diff_attention``).

The unsuffixed functions are differentiable; the ``_grad`` functions are the
same backward passes as plain calls, which can be captured into a HIP graph.
Second and forward-mode derivatives are refused.
They work in the dtypes they are given and hold sums, norms and angles in 32
bits or more (no compute-dtype policy applies).
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from dattri_llm_amd import kernels


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, inv_freq, positions, mask, cfg, slots):
        ctx.save_for_backward(q, k, q_weight, k_weight, inv_freq, positions, mask)
        ctx.cfg, ctx.slots = cfg, slots
        return kernels.qk_norm_rope(q, k, q_weight, k_weight, inv_freq, positions, mask=mask, **cfg)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, q_weight, k_weight, inv_freq, positions, mask = ctx.saved_tensors
        # An output that no gradient reached has zeros; gk is None where k is.
        wanted = ctx.slots is not None or ctx.needs_input_grad[2] or ctx.needs_input_grad[3]
        dq, dk, wq, wk = kernels.qk_norm_rope_grad(gq, gk, q, k, q_weight, k_weight, inv_freq, positions, mask=mask,
                                                   weight_grads=wanted, **ctx.cfg)
        if ctx.slots is not None:
            for slot, w in zip(ctx.slots, (wq, wk)):
                if w is not None:
                    slot.put(w)
            wq = wk = None
        need = ctx.needs_input_grad
        return (dq if need[0] else None, dk if need[1] else None,
                wq.sum(0).to(q_weight.dtype) if need[2] and wq is not None else None,
                wk.sum(0).to(k_weight.dtype) if need[3] and wk is not None else None,
                None, None, None, None, None)


def qk_norm_rope(q, k, q_weight, k_weight, inv_freq, positions=None, *, eps: float = 1e-6, interleaved: bool = False,
                 scaling: float = 1.0, mask=None, slots=None):
    """RMS-normalise each head of ``q (B, T, Hq, D)`` and ``k (B, T, Hk, D)`` with
    weights ``(D,)``, then rotate its first ``R = 2 * len(inv_freq)`` entries by
    ``position * inv_freq``: ``(q_out, k_out)``, differentiable.

    Pairs are ``(i, i + R/2)``, or ``(2i, 2i+1)`` with ``interleaved``; cosine and
    sine are multiplied by ``scaling``.  ``positions``: int32/int64 ``(T,)`` or
    ``(B, T)``, by default the token's index; ``inv_freq`` float32, without a
    gradient.  ``mask`` (B, T): a token with a zero gets zero rows, whatever its
    input holds, and takes no part in any gradient.  ``k`` may be None.  Inputs of
    any strides; outputs keep their layout (contiguous where rows overlap in
    memory).  A single new token is ``T = 1`` with its position.

    ``slots``: a ``(q, k)`` pair that takes the weights' per-sample gradients in
    the backward pass, in place of their summed ones (``FusedCapture``)."""
    if getattr(forward_ad, "_current_level", 0) >= 0:
        kernels.refuse_tangents("qk_norm_rope", q, k, q_weight, k_weight, inv_freq)
    if inv_freq.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("qk_norm_rope: inv_freq takes no gradient; pass it detached")
    cfg = {"eps": eps, "interleaved": interleaved, "scaling": scaling}
    if torch.is_grad_enabled() and (q.requires_grad or q_weight.requires_grad or (
            k is not None and k_weight is not None and (k.requires_grad or k_weight.requires_grad))):
        return _QkNormRope.apply(q, k, q_weight, k_weight, inv_freq, positions, mask, cfg, slots)
    return kernels.qk_norm_rope(q, k, q_weight, k_weight, inv_freq, positions, mask=mask, **cfg)


def qk_norm_rope_grad(gq, gk, q, k, q_weight, k_weight, inv_freq, positions=None, *, eps: float = 1e-6,
                      interleaved: bool = False, scaling: float = 1.0, mask=None):
    """The backward pass of :func:`qk_norm_rope` for its outputs' gradients:
    ``(dq, dk, dq_weight, dk_weight)`` with the weights' gradients per sample,
    fp32 ``(B, D)`` (a layer of type ``"nn.RMSNorm"``, materialized)."""
    return kernels.qk_norm_rope_grad(gq, gk, q, k, q_weight, k_weight, inv_freq, positions, eps=eps,
                                     interleaved=interleaved, scaling=scaling, mask=mask)


class _RelativeBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, q_len, k_len, batch, mask, cfg, slot):
        ctx.save_for_backward(mask)
        ctx.cfg, ctx.slot, ctx.table = cfg, slot, (table.shape[0], table.dtype)
        bias = kernels.relative_bias(table, q_len, k_len, **cfg)
        return bias if batch is None else bias.expand(batch, -1, -1, -1)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        (mask,) = ctx.saved_tensors
        buckets, dtype = ctx.table
        per_sample = kernels.relative_bias_grad(g if g.dim() == 4 else g.unsqueeze(0), buckets, mask=mask, **ctx.cfg)
        if ctx.slot is not None:
            ctx.slot.put(per_sample.flatten(1))
            return (None,) * 7
        return per_sample.sum(0).to(dtype), None, None, None, None, None, None


def relative_bias(table, q_len: int, k_len: int, *, batch: int | None = None, q_start: int = 0,
                  bidirectional: bool = True, max_distance: int = 128, causal: bool = False, mask=None, slot=None):
    """Attention bias from a learned ``(num_buckets, H)`` table, differentiable:
    ``bias[h, i, j] = table[bucket(j - i - q_start), h]``, shape ``(H, q_len,
    k_len)``.

    Of one side's ``n`` buckets (``num_buckets / 2`` for each direction with
    ``bidirectional``, else all for the past) the first half hold one distance
    each, the others ranges that widen by a constant factor up to
    ``max_distance``; a range starts at the least whole distance that reaches
    its border exactly.  ``causal``: ``-inf`` where the key follows the query.
    One new token against a cache is ``q_len = 1`` with ``q_start`` its position.

    ``batch``: the bias as a ``(batch, H, q_len, k_len)`` view without copies of
    it; its gradient then arrives with the samples apart, which a per-sample
    gradient needs.  ``mask`` (batch, k_len) names the live positions of each
    sample: gradients of the others' scores are not counted.  ``slot`` takes the
    per-sample gradient in place of the summed one, a frozen table's too
    (``FusedCapture``)."""
    if getattr(forward_ad, "_current_level", 0) >= 0:
        kernels.refuse_tangents("relative_bias", table)
    if batch is None and (mask is not None or slot is not None):
        raise ValueError("relative_bias: mask and slot need batch, the samples apart")
    if mask is not None:  # read by the backward pass alone, checked here
        kernels.check_bias_mask("relative_bias", mask, batch, q_len, k_len, q_start)
        if mask.device != table.device:
            raise ValueError(f"relative_bias: tensors on different devices: {table.device} and {mask.device}")
    cfg = {"q_start": q_start, "bidirectional": bidirectional, "max_distance": max_distance, "causal": causal}
    if slot is not None and torch.is_grad_enabled() and not table.requires_grad:
        table = table.detach().requires_grad_()  # a frozen table has no input to carry the gradient to its slot
    if torch.is_grad_enabled() and table.requires_grad:
        return _RelativeBias.apply(table, q_len, k_len, batch, mask, cfg, slot)
    bias = kernels.relative_bias(table, q_len, k_len, **cfg)
    return bias if batch is None else bias.expand(batch, -1, -1, -1)


def relative_bias_grad(g, num_buckets: int, *, q_start: int = 0, bidirectional: bool = True, max_distance: int = 128,
                       causal: bool = False, mask=None):
    """Per-sample gradient ``(B, num_buckets, H)``, fp32, of a bias table from the
    gradient ``g (B, H, q_len, k_len)`` of the scores it was added to; flattened
    past the batch it is a layer of type ``"nn.Embedding"``, materialized."""
    return kernels.relative_bias_grad(g, num_buckets, q_start=q_start, bidirectional=bidirectional,
                                      max_distance=max_distance, causal=causal, mask=mask)


class DiffAttentionState(NamedTuple):
    """What :func:`diff_attention_grad` needs of the forward call beside its output: the
    second map's values, and each row's log of its sum and largest score in either map."""

    second: torch.Tensor
    lse: torch.Tensor


class _DiffAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, mask, q_mask, cfg, slot):
        out, second, lse = kernels.diff_attention(q, k, v, lam, mask=mask, q_mask=q_mask, state=True, **cfg)
        ctx.save_for_backward(q, k, v, lam, mask, q_mask, out, second, lse)
        ctx.cfg, ctx.slot = cfg, slot
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        q, k, v, lam, mask, q_mask, out, second, lse = ctx.saved_tensors
        dq, dk, dv, per_sample = kernels.diff_attention_grad(g, q, k, v, lam, out, second, lse, mask=mask,
                                                             q_mask=q_mask, **ctx.cfg)
        need = ctx.needs_input_grad
        dlam = None
        if ctx.slot is not None:
            ctx.slot.put(per_sample)
        elif need[3]:
            dlam = per_sample.sum(0) if lam.numel() > 1 else per_sample.sum()
            dlam = dlam.reshape(lam.shape).to(lam.dtype)
        return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, dlam,
                None, None, None, None)


def diff_attention(q, k, v, lam, *, scale: float | None = None, causal: bool = False, q_start: int | None = None,
                   mask=None, q_mask=None, return_state: bool = False, slot=None):
    """Attention by the difference of two softmax maps, differentiable:
    ``out_h = softmax(scale q_2h k^T) v - lam_h softmax(scale q_2h+1 k^T) v``.

    ``q (B, T, 2 H, D)`` holds head ``h``'s two query maps at ``2h`` and ``2h +
    1``, ``k (B, S, 2 Hk, D)`` a key head's two key maps likewise, ``v (B, S, Hk,
    Dv)``; head ``h`` reads key head ``h // (H // Hk)``.  ``out (B, T, H, Dv)``,
    contiguous.  ``lam``: ``(H,)``, or one entry for all heads.  ``D`` up to 128,
    ``Dv`` up to 256; ``scale`` is ``D ** -0.5`` by default.  Inputs of any
    strides (a copy is made where entries are not contiguous).

    ``causal``: query ``i`` sees the keys up to ``i + q_start``, by default ``S -
    T`` (the queries are the last positions; one new token against a cache is
    ``T = 1``).  ``mask`` (B, S): a zero hides the key from every query;
    ``q_mask`` (B, T): a zero takes the query out.  Both may hold anything there.
    A query that sees no key has a zero row and no gradient; one with a NaN or
    infinite score has NaN in its row, and in the gradients of what it sees.

    ``return_state``: ``(out, state)`` for :func:`diff_attention_grad`; not
    differentiable.  ``slot`` takes ``lam``'s per-sample gradient ``(B, H)`` in the
    backward pass, in place of its summed one (``FusedCapture``).  It is formed from
    the maps in 32 bits (in 16 bits that of a factor below 2^-60 from the second map's
    rounded values)."""
    if getattr(forward_ad, "_current_level", 0) >= 0:
        kernels.refuse_tangents("diff_attention", q, k, v, lam)
    cfg = {"scale": scale, "causal": causal, "q_start": q_start}
    if torch.is_grad_enabled() and (slot is not None or q.requires_grad or k.requires_grad or v.requires_grad or
                                    lam.requires_grad):
        if return_state:
            raise ValueError("diff_attention: return_state is for plain calls; call it under no_grad")
        if slot is not None and not lam.requires_grad:
            lam = lam.detach().requires_grad_()  # a frozen factor is captured too
        return _DiffAttention.apply(q, k, v, lam, mask, q_mask, cfg, slot)
    out, second, lse = kernels.diff_attention(q, k, v, lam, mask=mask, q_mask=q_mask, state=return_state, **cfg)
    return (out, DiffAttentionState(second, lse)) if return_state else out


def diff_attention_grad(g, q, k, v, lam, out, state: DiffAttentionState, *, scale: float | None = None,
                        causal: bool = False, q_start: int | None = None, mask=None, q_mask=None):
    """The backward pass of :func:`diff_attention` for the gradient ``g`` of
    ``out``, with what it returned under ``return_state`` and the same settings:
    ``(dq, dk, dv, dlam)``, ``dlam`` per sample, fp32 ``(B, H)``."""
    return kernels.diff_attention_grad(g, q, k, v, lam, out, state.second, state.lse, scale=scale, causal=causal,
                                       q_start=q_start, mask=mask, q_mask=q_mask)


__all__ = ["DiffAttentionState", "diff_attention", "diff_attention_grad", "qk_norm_rope", "qk_norm_rope_grad",
           "relative_bias", "relative_bias_grad"]
