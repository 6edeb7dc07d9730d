"""Log probabilities of given tokens: the losses that a block's gradients start from.

Each sample's loss is a sum of its tokens' log probabilities, so the samples'
gradients (and a query's, that of a given answer) come from one backward pass
over logits whose tokens stay apart.  :func:`token_logprobs` gives them with the
entropy and the most likely alternatives in one pass over the logits, and is
differentiable; :func:`token_logprobs_grad` is the same backward pass as a plain
call, which can be captured into a HIP graph.  Second and forward-mode
derivatives are refused.  Sums are held in 32 bits, of differences from a row's
largest logit: a common offset or a small temperature costs no accuracy.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from dattri_llm_amd import kernels


class TokenLogprobs(NamedTuple):
    """Per token, fp32: ``logprob`` of its target (0 where it has none),
    ``entropy`` and ``lse`` (the logits' logsumexp); with ``top`` the most likely
    tokens' ``top_logprob`` and int64 ``top_index``, in order (else None)."""

    logprob: torch.Tensor
    entropy: torch.Tensor
    lse: torch.Tensor
    top_logprob: torch.Tensor | None
    top_index: torch.Tensor | None


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, mask, temperature, top):
        got = kernels.token_logprobs(logits, targets, mask=mask, temperature=temperature, top=top)
        ctx.save_for_backward(logits, targets, mask, got[2], got[1])
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        if not top:
            return got[:3]
        ctx.mark_non_differentiable(*got[3:])
        return got

    @staticmethod
    @once_differentiable
    def backward(ctx, up, up_entropy, up_lse, *_top):
        if up is None and up_entropy is None and up_lse is None:
            return (None,) * 5
        logits, targets, mask, lse, entropy = ctx.saved_tensors
        grad = kernels.token_logprobs_grad(up, up_entropy, logits, targets, lse, entropy, up_lse=up_lse, mask=mask,
                                           temperature=ctx.temperature)
        return grad, None, None, None, None


def token_logprobs(logits, targets, *, mask=None, temperature: float = 1.0, top: int = 0) -> TokenLogprobs:
    """Log probabilities of ``targets`` under ``softmax(logits / temperature)``,
    differentiable in ``logprob``, ``entropy`` and ``lse``.

    ``logits`` ``(B, T, V)`` or ``(N, V)`` of any strides, ``targets`` int64 in
    the leading shape; one outside the vocabulary (-100, say) names no token.
    ``mask`` in the same shape: a token with a zero gets zeros (indices -1),
    whatever its logits hold, and takes no part in any gradient.  ``top``: how
    many of the most likely tokens (at most 32) to return; of equal logits the
    lower index comes first.  A logit of ``-inf`` (or of its type's lowest value
    beside others) has no probability; a row with NaN gives NaN.  ``temperature``
    lies between 1e-30 and 8e37."""
    if getattr(forward_ad, "_current_level", 0) >= 0:
        kernels.refuse_tangents("token_logprobs", logits)
    if torch.is_grad_enabled() and logits.requires_grad:
        got = _TokenLogprobs.apply(logits, targets, mask, temperature, top)
        return TokenLogprobs(*got) if top else TokenLogprobs(*got, None, None)
    return TokenLogprobs(*kernels.token_logprobs(logits, targets, mask=mask, temperature=temperature, top=top))


def token_logprobs_grad(up, up_entropy, logits, targets, lse, entropy, *, up_lse=None, mask=None,
                        temperature: float = 1.0):
    """The backward pass of :func:`token_logprobs` for the gradients of
    ``logprob``, ``entropy`` and ``lse`` (the targets' shape, any strides; None:
    zero), with ``lse`` and ``entropy`` as it returned them: the logits'
    gradient, in their dtype."""
    return kernels.token_logprobs_grad(up, up_entropy, logits, targets, lse, entropy, up_lse=up_lse, mask=mask,
                                       temperature=temperature)


__all__ = ["TokenLogprobs", "token_logprobs", "token_logprobs_grad"]
