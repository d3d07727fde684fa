"""Norms of query and key heads with the rotation after them, and their gradients, in float64 numpy.  No counterpart in
the reference (its rotation alone: ``apply_rotary_emb``, ``dsalt/kernels/window_utils.py:74-89``)."""
from __future__ import annotations

import numpy as np


def positions(T, cu):
    pos = np.full(T, -1)
    for a, b in zip(cu, cu[1:]):
        pos[a:b] = np.arange(b - a)
    return pos


def _tables(pos, cos, sin):
    on = (pos >= 0) & (pos < len(cos))
    at = np.where(on, pos, 0)
    return on[:, None, None], cos[at][:, None], sin[at][:, None]


def forward(x, w, pos, cos, sin, eps):
    """(y, reach): reach = |n1 cos| + |n2 sin|, the size of what is summed."""
    on, c, s = _tables(pos, cos, sin)
    half = x.shape[-1] // 2
    n = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    rot = np.concatenate([-n[..., half:], n[..., :half]], -1)
    return np.where(on, n * c + rot * s, 0.0), np.where(on, np.abs(n * c) + np.abs(rot * s), 0.0)


def backward(d, x, w, pos, cos, sin, eps):
    """(dx, dw, reach of dx, reach of dw)."""
    on, c, s = _tables(pos, cos, sin)
    half = x.shape[-1] // 2
    ds = d * s
    dn = d * c + np.concatenate([ds[..., half:], -ds[..., :half]], -1)
    an = np.abs(d * c) + np.abs(np.concatenate([ds[..., half:], ds[..., :half]], -1))
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    dx = r * (w * dn - x * r * r * (w * dn * x).mean(-1, keepdims=True))
    ax = r * (np.abs(w) * an + np.abs(x) * r * r * (np.abs(w * x) * an).mean(-1, keepdims=True))
    dn, an = np.where(on, dn, 0.0), np.where(on, an, 0.0)
    return np.where(on, dx, 0.0), (dn * x * r).sum((0, 1)), np.where(on, ax, 0.0), (an * np.abs(x) * r).sum((0, 1))
