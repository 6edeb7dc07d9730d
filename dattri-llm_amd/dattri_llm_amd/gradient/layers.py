"""Modules over the differentiable operators whose parameters
:class:`~dattri_llm_amd.gradient.capture.FusedCapture` captures.

A hook on these layers sees no usable pair of input and output gradient (the
norms' output gradient lies behind the rotation, the bias is shared by the
batch; the reference's hooks have no counterpart), so they are captured in
their own backward pass, as per-sample weight gradients.
"""

from __future__ import annotations

import torch
from torch import nn

from dattri_llm_amd.gradient import ops


class QKNormRope(nn.Module):
    """RMS norms of each head's queries and keys, then the position rotation
    (:func:`ops.qk_norm_rope`).

    Parameters ``q_weight`` and ``k_weight`` ``(head_dim,)``; ``rotary_dim``
    entries rotate (default all) with frequencies ``base ** (-2i / rotary_dim)``,
    or the given ``inv_freq``."""

    def __init__(self, head_dim: int, *, rotary_dim: int | None = None, base: float = 10000.0,
                 inv_freq: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = False,
                 scaling: float = 1.0, device=None, dtype=None) -> None:
        super().__init__()
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if inv_freq is None:
            if rotary_dim % 2 or not 0 <= rotary_dim <= head_dim:
                raise ValueError(f"rotary_dim must be even and at most head_dim {head_dim}, got {rotary_dim}")
            half = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
            inv_freq = base ** (-half / max(rotary_dim, 1))
        self.register_buffer("inv_freq", inv_freq.to(device=device, dtype=torch.float32), persistent=False)
        self.q_weight = nn.Parameter(torch.ones(head_dim, device=device, dtype=dtype))
        self.k_weight = nn.Parameter(torch.ones(head_dim, device=device, dtype=dtype))
        self.eps, self.interleaved, self.scaling = eps, interleaved, scaling

    def _apply(self, fn, recurse=True):
        # A cast of the model keeps the frequencies in fp32: angles of far
        # positions need them.
        freq = self.inv_freq
        super()._apply(fn, recurse)
        if self.inv_freq.dtype != torch.float32:
            self.inv_freq = freq.to(self.inv_freq.device)
        return self

    def forward(self, q, k, positions=None, mask=None, *, _slots=None):
        return ops.qk_norm_rope(q, k, self.q_weight, self.k_weight, self.inv_freq, positions, eps=self.eps,
                                interleaved=self.interleaved, scaling=self.scaling, mask=mask, slots=_slots)


class RelativeBias(nn.Module):
    """Learned relative position bias by buckets (:func:`ops.relative_bias`).

    Parameter ``weight`` ``(num_buckets, heads)``, an embedding table's layout.
    Pass ``batch`` in the forward call where per-sample gradients are wanted."""

    def __init__(self, num_buckets: int, heads: int, *, max_distance: int = 128, bidirectional: bool = True,
                 causal: bool = False, device=None, dtype=None) -> None:
        super().__init__()
        self.weight = nn.Parameter(torch.randn(num_buckets, heads, device=device, dtype=dtype))
        self.max_distance, self.bidirectional, self.causal = max_distance, bidirectional, causal

    def forward(self, q_len: int, k_len: int, *, batch: int | None = None, q_start: int = 0, mask=None, _slot=None):
        return ops.relative_bias(self.weight, q_len, k_len, batch=batch, q_start=q_start,
                                 bidirectional=self.bidirectional, max_distance=self.max_distance,
                                 causal=self.causal, mask=mask, slot=_slot)


__all__ = ["QKNormRope", "RelativeBias"]
