"""Norms of queries and keys for each head with the rotary embedding in the same pass, differentiable.

No counterpart in the reference, whose heads are rotated as projected (``apply_rotary_emb``,
``dsalt/kernels/window_utils.py:73-90``): a root-mean-square norm with a weight per channel before
that rotation, ``ops.qk_norm_rope`` forward and ``ops.qk_norm_rope_backward`` for the gradients of
q, k and both weights.  The rotation's tables get no gradient; the inputs are kept for the backward
pass, their norms computed again there.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import ops


class QkNormRopeFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, cu_seqlens, pos, max_seqlen, eps):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, cu_seqlens, pos)
        ctx.at = dict(max_seqlen=max_seqlen, eps=eps)
        return ops.qk_norm_rope(q, k, q_weight, k_weight, cos, sin, cu_seqlens=cu_seqlens, pos=pos, **ctx.at)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        q, k, q_weight, k_weight, cos, sin, cu_seqlens, pos = ctx.saved_tensors
        dq, dk, dqw, dkw = ops.qk_norm_rope_backward(dq, dk, q, k, q_weight, k_weight, cos, sin, cu_seqlens=cu_seqlens, pos=pos, **ctx.at)
        dqw, dkw = (d if d is None else d.to(w.dtype) for d, w in ((dqw, q_weight), (dkw, k_weight)))
        return dq, dk, dqw, dkw, None, None, None, None, None, None


def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, *, cu_seqlens=None, pos=None, max_seqlen=None, eps=1e-6):
    """(q, k) of ``ops.qk_norm_rope``, differentiable in q, k and the weights (once)."""
    if cu_seqlens is not None and max_seqlen is None:
        max_seqlen = ops._max_seqlen(cu_seqlens)  # one device-to-host copy for both passes
    return QkNormRopeFunction.apply(q, k, q_weight, k_weight, cos, sin, cu_seqlens, pos, max_seqlen, eps)
