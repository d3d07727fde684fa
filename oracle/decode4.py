"""The 4-bit cache and the verification of drafted tokens in float64 numpy.  No counterpart in the reference;
written from the definitions stated in ``include/dsalt_amd.h``.

``Pages4`` holds values (what codes and scales stand for) and exponents; ``decode.attention`` reads it like the
8-bit pages.
"""
from __future__ import annotations

import numpy as np

from . import decode as OD

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def exponent_of(x):
    """Exponent of the least power of two in [2^-126, 2^125] with every element of x (finite) within 7 of it."""
    top, e = float(np.abs(np.asarray(x, dtype=np.float64)).max(initial=0.0)), -126
    while e < 125 and top > 7.0 * 2.0 ** e:
        e += 1
    return e


def e2m1(x):
    """x rounded to the nearest of the grid, ties to the even code, past 6 to 6."""
    a = np.minimum(np.abs(np.asarray(x, dtype=np.float64)), 6.0)
    d = np.abs(a[..., None] - GRID)
    best = d.min(-1, keepdims=True)
    near = d == best
    code = np.where(near & (np.arange(8) % 2 == 0), 1, 0).argmax(-1)   # the even one of two
    code = np.where(near.sum(-1) == 2, code, near.argmax(-1))
    return np.copysign(GRID[code], x)


def block(x):
    """(values held, exponent byte) of 32 elements."""
    x = np.asarray(x, dtype=np.float64)
    if not np.isfinite(x).all():
        return np.full(x.shape, np.nan), 255
    e = exponent_of(x)
    return e2m1(x / 2.0 ** e) * 2.0 ** e, e + 127


class Pages4:
    def __init__(self, n_blocks, n_kv, block_tokens, head_dim):
        self.k, self.v = (np.zeros((n_blocks, n_kv, block_tokens, head_dim)) for _ in range(2))

    def write(self, k, v, pieces):
        n_blocks, G, bt, D = self.k.shape
        for row0, rows, page, off in np.asarray(pieces).tolist():
            if rows <= 0 or row0 < 0 or row0 + rows > len(k) or not 0 <= page < n_blocks or off < 0 or off + rows > bt:
                continue
            for x, held in ((k, self.k), (v, self.v)):
                for i in range(rows):
                    for g in range(G):
                        for c in range(0, D, 32):
                            held[page, g, off + i, c:c + 32] = block(x[row0 + i, g, c:c + 32])[0]

    def token(self, row, pos):
        bt = self.k.shape[2]
        if pos < 0 or pos // bt >= len(row) or not 0 <= row[pos // bt] < len(self.k):
            return None
        return self.k[row[pos // bt], :, pos % bt], self.v[row[pos // bt], :, pos % bt]

    read = OD.Pages.read


# ------------------------------------------------------------------------ verification
def weights(x, temperature):
    """Whole weights of one row of logits."""
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, dtype=np.float64))
    top = x.max()
    w = np.zeros(x.shape, dtype=np.int64)
    if top == -np.inf:
        return w
    if not temperature > 0:
        w[int(np.argmax(x))] = int(OD.UNIT)
        return w
    if top == np.inf:
        return np.where(x == np.inf, OD.UNIT, 0.0).astype(np.int64)
    ok = x > -np.inf
    z = np.where(ok, np.where(ok, x - top, 0.0) / temperature, -np.inf)
    return np.rint(np.exp(z) * OD.UNIT).astype(np.int64)


def verify(logits, tokens, cu, u, v, draft_logits, temperature, draft_temperature):
    """(accepted [R], tokens [T]); temperatures [R]."""
    T, V = logits.shape
    accepted, out = [], [-1] * T
    for r in range(len(cu) - 1):
        n = 0
        for t in range(cu[r], cu[r + 1]):
            a = weights(logits[t], temperature[r])
            total = int(a.sum())
            if t + 1 == cu[r + 1]:
                break
            x = int(tokens[t + 1])
            if draft_logits is None:
                b = np.zeros(V)
                if 0 <= x < V:
                    b[x] = 1.0
            else:
                b = weights(draft_logits[t], draft_temperature[r])
            bs = float(b.sum())
            p = a[x] / total if total and 0 <= x < V else 0.0
            q = b[x] / bs if bs and 0 <= x < V else 0.0
            uu = u[t] if u[t] >= 0 else 0.0
            if uu * q < p:
                out[t], n = x, n + 1
                continue
            left = np.rint(np.maximum(a * (2.0 ** 52 / total if total else 0.0) - b * (2.0 ** 52 / bs if bs else 0.0), 0.0)).astype(np.int64)
            if left.any():
                a = left
            break
        else:
            accepted.append(0)
            continue
        accepted.append(n)
        cum = np.cumsum(a)
        if cum[-1]:
            goal = (v[r] if v[r] >= 0 else 0.0) * float(cum[-1])
            hit = np.flatnonzero(cum > goal)
            out[t] = int(hit[0]) if len(hit) else int(np.flatnonzero(a)[-1])
    return accepted, out
