"""The residual's addition with the RMS norm that follows it.

A block's norm reads the residual stream's sum and nothing else does between the
two, so one pass forms both.  The backward pass gives the norm weight's
per-sample gradient beside the input's in one pass too, where a hook's capture
(``dattri_llm/gradient/ops/materialize.py:96-98``) reads the input and the
output gradient once more.

:func:`add_rms_norm` is differentiable; :func:`add_rms_norm_grad` is the same
backward pass as a plain call, which can be captured into a HIP graph.  Second
and forward-mode derivatives are refused.  Sums are held in 32 bits.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from dattri_llm_amd import kernels


class AddNorm(NamedTuple):
    """``out``: the normalised rows; ``total``: ``x + residual`` (None without a
    residual); ``scales``: what ``out`` is to be multiplied by where it is in 8
    bits (else None)."""

    out: torch.Tensor
    total: torch.Tensor | None
    scales: torch.Tensor | None


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, mask, eps, slot):
        out, total, _ = kernels.add_rms_norm(x, residual, weight, eps=eps, mask=mask)
        ctx.save_for_backward(x if total is None else total, weight, mask)
        ctx.eps, ctx.slot = eps, slot
        ctx.set_materialize_grads(False)
        return out if total is None else (out, total)

    @staticmethod
    @once_differentiable
    def backward(ctx, g, g_total=None):
        total, weight, mask = ctx.saved_tensors
        if g is None and g_total is None:
            return (None,) * 6
        g = torch.zeros_like(total) if g is None else g
        wanted = ctx.slot is not None or ctx.needs_input_grad[2]
        dx, dw = kernels.add_rms_norm_grad(g, g_total, total, weight, eps=ctx.eps, mask=mask, weight_grads=wanted)
        if ctx.slot is not None:
            ctx.slot.put(dw)
            dw = None
        need = ctx.needs_input_grad
        return (dx if need[0] else None, dx if need[1] else None,
                dw.sum(0).to(weight.dtype) if need[2] and dw is not None else None, None, None, None)


def add_rms_norm(x, residual, weight, *, eps: float = 1e-6, mask=None, quantize: str | None = None,
                 slot=None) -> AddNorm:
    """``total = x + residual`` of ``(B, T, d)`` rows and its RMS norm
    ``total * rsqrt(mean(total^2) + eps) * weight``, differentiable.

    The norm is that of ``total`` as it is returned, in the rows' dtype.
    ``residual`` may be None (``total`` is None then); two dtypes are promoted as an
    addition promotes them; ``weight`` ``(d,)``, in any dtype.  ``mask`` (B, T): a
    token with a zero gets zero rows, whatever its input holds, and takes no part
    in any gradient.  Inputs of any strides; outputs are contiguous.  A single new
    token is ``T = 1``.

    ``quantize``: ``out`` in 8 bits (``torch.float8_e4m3fn``) with fp32
    ``scales``, ``"row"`` ``(B, T)``, or ``"block"`` one for each 128 entries
    ``(B, T, ceil(d / 128))``: the largest absolute value / 448.  Not
    differentiable.

    ``slot`` takes the weight's per-sample gradient in the backward pass, in
    place of its summed one (``FusedCapture``)."""
    if getattr(forward_ad, "_current_level", 0) >= 0:
        kernels.refuse_tangents("add_rms_norm", x, residual, weight)
    if residual is not None and residual.dtype != x.dtype:
        wide = torch.promote_types(x.dtype, residual.dtype)
        x, residual = x.to(wide), residual.to(wide)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (
            residual is not None and residual.requires_grad) or (slot is not None)):
        if quantize is not None:
            raise NotImplementedError("add_rms_norm: an output in 8 bits has no gradient; call it under no_grad")
        if slot is not None and not weight.requires_grad:
            weight = weight.detach().requires_grad_()  # a frozen weight is captured too
        got = _AddRmsNorm.apply(x, residual, weight, mask, eps, slot)
        return AddNorm(got, None, None) if residual is None else AddNorm(*got, None)
    return AddNorm(*kernels.add_rms_norm(x, residual, weight, eps=eps, mask=mask, quantize=quantize))


def add_rms_norm_grad(g, g_total, total, weight, *, eps: float = 1e-6, mask=None):
    """The backward pass of :func:`add_rms_norm` for the gradients ``g`` of
    ``out`` and ``g_total`` of ``total`` (None: zero), from ``total`` (``x``
    where there was no residual): ``(dx, dweight)``, the gradient of ``x`` and of
    ``residual`` alike, and the weight's per sample, fp32 ``(B, d)`` (a layer of
    type ``"nn.RMSNorm"``, materialized)."""
    return kernels.add_rms_norm_grad(g, g_total, total, weight, eps=eps, mask=mask)


__all__ = ["AddNorm", "add_rms_norm", "add_rms_norm_grad"]
