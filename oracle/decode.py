"""A decoding step over a paged 8-bit key/value cache in float64 numpy: row maps, the cache's write and
read-back, attention of single tokens over it and sampling.  No counterpart in the reference; written from
the definitions stated in ``include/dsalt_amd.h``.

The cache here is ``Pages``: unscaled values (what the e4m3 codes stand for) and scales, per block and head.
"""
from __future__ import annotations

import math

import numpy as np

UNIT = 2.0 ** 42


# ------------------------------------------------------------------------ e4m3 and scales
def e4m3(x):
    """x rounded to the nearest e4m3 number, ties to even, past 448 to 448, what is not finite to NaN."""
    x = np.asarray(x, dtype=np.float64)
    ok = np.isfinite(x)
    a = np.minimum(np.abs(np.where(ok, x, 0.0)), 448.0)
    step = np.exp2(np.floor(np.log2(np.maximum(a, 2.0 ** -6))) - 3)
    return np.where(ok, np.copysign(np.rint(a / step) * step, x), np.nan)


def scale_of(x):
    """The least power of two in [2^-126, 2^119] that keeps every finite element of x within 448 of it."""
    x = np.asarray(x, dtype=np.float64)
    top = float(np.abs(x[np.isfinite(x)]).max(initial=0.0))
    e = -126
    while e < 119 and top > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


class Pages:
    def __init__(self, n_blocks, n_kv, block_tokens, head_dim):
        shape = (n_blocks, n_kv, block_tokens, head_dim)
        self.k, self.v = np.zeros(shape), np.zeros(shape)
        self.ks, self.vs = np.zeros(shape[:2]), np.zeros(shape[:2])

    def write(self, k, v, pieces):
        """k, v [T, G, D]; pieces of (first row, rows, page, first token in the page)."""
        n_blocks, G, bt, _ = self.k.shape
        for row0, rows, page, off in np.asarray(pieces).tolist():
            if rows <= 0 or row0 < 0 or row0 + rows > len(k) or not 0 <= page < n_blocks or off < 0 or off + rows > bt:
                continue
            for x, codes, scale in ((k, self.k, self.ks), (v, self.v, self.vs)):
                for g in range(G):
                    new = np.asarray(x[row0:row0 + rows, g], dtype=np.float64)
                    was = scale[page, g] if off > 0 else 0.0
                    now = max(scale_of(new), was)
                    codes[page, g, :off] = e4m3(codes[page, g, :off] * (was / now))
                    codes[page, g, off:off + rows] = e4m3(new / now)
                    scale[page, g] = now

    def read(self, table, cu, start, n_rows):
        k = np.zeros((n_rows, self.k.shape[1], self.k.shape[3]))
        v = np.zeros_like(k)
        for r in range(len(table)):
            for t in range(cu[r], min(cu[r + 1], n_rows)):
                got = self.token(table[r], start[r] + t - cu[r])
                if got is not None:
                    k[t], v[t] = got
        return k, v

    def token(self, row, pos):
        """(k [G, D], v [G, D]) of the token at pos of a table row, None where it names no page."""
        bt = self.k.shape[2]
        if pos < 0 or pos // bt >= len(row) or not 0 <= row[pos // bt] < len(self.k):
            return None
        b, o = row[pos // bt], pos % bt
        return self.k[b, :, o] * self.ks[b][:, None], self.v[b, :, o] * self.vs[b][:, None]


# ------------------------------------------------------------------------ row maps
def rows(seq_len, new_len, table, ring, span, n_rows, bt):
    """Updates table and ring (lists or arrays) in place; returns a dict of the step's maps."""
    R, M = table.shape
    N = len(ring)
    head, tail = (int(x) for x in span)
    need = upto = give = row = 0
    seq, granted, cu = list(seq_len), [0] * R, [0]
    req, pos, slot = [-1] * n_rows, [-1] * n_rows, [-1] * n_rows
    pieces, taken = [], 0
    back = []
    for r in range(R):
        L, n = int(seq_len[r]), int(new_len[r])
        held = min(max(-(-L // bt), 0), M)
        first, row = row, row + max(n, 0)
        cu.append(row)
        for t in range(first, min(row, n_rows)):
            req[t] = r
        if n < 0:
            if L >= 0:
                back += [int(x) for x in table[r, :held]]
                seq[r], granted[r] = 0, 1
            continue
        if L < 0 or L + n > M * bt or row > n_rows:
            continue
        need = max(-(-(L + n) // bt) - held, 0)
        upto += need
        if need and upto > tail - head:
            continue
        granted[r], seq[r] = 1, L + n
        if need:
            taken = upto
            for j in range(need):
                table[r, held + j] = ring[(head + upto - need + j) % N]
        for i in range(n):
            p, t = L + i, first + i
            pos[t], slot[t] = p, int(table[r, p // bt]) * bt + p % bt
            if i == 0 or p % bt == 0:
                pieces.append([t, min(bt - p % bt, n - i), int(table[r, p // bt]), p % bt])
    for i, page in enumerate(back):
        if tail + i - head < N:
            ring[(tail + i) % N] = page
    P = min(n_rows, n_rows // bt + 2 * R)
    pieces += [[0, 0, 0, 0]] * (P - len(pieces))
    return dict(seq_len=seq, span=[head + taken, min(tail + len(back), head + N)], granted=granted, cu=cu, req=req, pos=pos,
                slot=slot, pieces=np.array(pieces, dtype=np.int64).reshape(P, 4))


# ------------------------------------------------------------------------ attention
def attention(q, pages, table, req, pos, w, lmk, bias, scale):
    """(out [T, H, D], lse [T, H], mass [T, H, D], reach [T, H], keys [T, H]): mass = sum p |v|, reach the largest
    sum of |scale q k| over a row's keys and keys their number (what error bounds are made of)."""
    T, H, D = q.shape
    G = pages.k.shape[1]
    out, lse, mass = np.zeros((T, H, D)), np.full((T, H), -np.inf), np.zeros((T, H, D))
    reach, keys = np.zeros((T, H)), np.zeros((T, H), dtype=np.int64)
    for t in range(T):
        r, i = int(req[t]), int(pos[t])
        if not 0 <= r < len(table) or i < 0:
            continue
        low = max(i - max(int(w[t]), 1) + 1, 0)
        cached = {}

        def token(p):
            if p not in cached:
                cached[p] = pages.token(table[r], p)
            return cached[p]
        window = [(p, 0.0) for p in range(low, i + 1) if token(p) is not None]
        for h in range(H):
            g = h // (H // G)
            mine = list(window)
            for s in range(lmk.shape[3]):
                p = int(lmk[h, r, 0, s])
                b = float(bias[h, r, 0, s]) if bias is not None else 0.0
                if 0 <= p < low and b > -np.inf and token(p) is not None:
                    mine.append((p, b))
            if not mine:
                continue
            K = np.stack([token(p)[0][g] for p, _ in mine])
            V = np.stack([token(p)[1][g] for p, _ in mine])
            s = (K @ q[t, h]) * scale + np.array([b for _, b in mine])
            m = s.max()
            if m == -np.inf:
                continue
            e = np.exp(s - m)
            out[t, h], lse[t, h] = e @ V / e.sum(), m + math.log(e.sum())
            mass[t, h] = e @ np.abs(V) / e.sum()
            reach[t, h], keys[t, h] = (np.abs(K) @ np.abs(q[t, h])).max() * scale, len(mine)
    return out, lse, mass, reach, keys


# ------------------------------------------------------------------------ sampling
def sample(x, u, temperature, top_k, top_p, min_p):
    """(token, logp) of one row of float64 logits."""
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, dtype=np.float64))
    order = np.argsort(-x, kind="stable")
    top = x[order[0]]
    if top == -np.inf:
        return -1, -np.inf
    if not temperature > 0:
        return int(order[0]), 0.0
    if top == np.inf:
        w = np.where(x == np.inf, UNIT, 0.0).astype(np.int64)
    else:
        ok = x > -np.inf
        z = np.where(ok, np.where(ok, x - top, 0.0) * (1.0 / temperature), -np.inf)
        w = np.rint(np.exp(z) * UNIT).astype(np.int64)
    if 0 < top_k < len(x):
        order = order[:top_k]
    before = np.concatenate([[0], np.cumsum(w[order])])
    stay = w[order] >= min_p * UNIT
    if not top_p >= 1:
        stay &= before[:-1] < top_p * float(before[-1])
    stay[0] = True
    kept = np.zeros_like(w)
    kept[order[stay]] = w[order[stay]]
    cum = np.cumsum(kept)
    u = u if u >= 0 else 0.0
    hit = np.flatnonzero(cum > u * float(cum[-1]))
    j = int(hit[0]) if len(hit) else int(np.flatnonzero(kept)[-1])
    return j, math.log(kept[j] / cum[-1])
