"""The operators of a decoding step over a paged 8-bit key/value cache, in their plain form and
through the framework, with the cases they are timed on.

Kinds of case (the ``kind`` of a case's dict):
  rows    block tables, slot maps and row positions of a step from the requests' lengths
          (``ops.cache_rows_``): admission, growth and release of pages
  store   a step's keys and values written into the cache as e4m3 with a scale for each block of
          tokens and head (``ops.cache_write_``), and the written blocks read back as values
          (``ops.cache_read``)
  attend  attention of single query tokens over the cache: the causal window and the landmarks of
          each row (``ops.cache_attention``)
  sample  one token a row of logits from given random numbers, with temperature, top-k, top-p and
          min-p (``ops.sample_rows``)

The cache: pages of ``bt`` tokens, ``k`` and ``v`` [blocks, kv_heads, bt, D] in e4m3 (largest 448, no
infinities), ``k_scale`` and ``v_scale`` [blocks, kv_heads] float32 powers of two; a code stands for
code * scale.  The scale of a block is the least power of two (2^-126 .. 2^119) that keeps every finite
element written to it within 448; where a later token needs a larger one, the codes held are rounded to
it.  Values that are not finite are held as NaN.

Sampling weighs a logit x of a row with largest m as round(2^42 exp((x - m) / temperature)), a whole
number, so that sums do not depend on their order.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_DEV = "cuda"
_FP8 = torch.float8_e4m3fn
_UNIT = 2.0 ** 42


# ------------------------------------------------------------------------ the cases
def listed():
    return [
        # a small decoding step: 64 requests, a token each, a few entering a new page
        dict(name="rows_decode_r64", kind="rows", reqs=64, rows=64, max_len=8192, bt=64, mix="decode"),
        # a large serving step: prompts in chunks, tokens of running requests, requests that end
        dict(name="rows_mixed_r1500", kind="rows", reqs=1500, rows=32768, max_len=16384, bt=64, mix="mixed"),
        # decoding at batch 256 of the 16/2-head shape: one token a request, most pages part full
        dict(name="store_decode_r256_g2_d128", kind="store", reqs=256, rows=256, max_len=4096, bt=64, kv_heads=2, head_dim=128,
             dtype="bf16"),
        # prompts of odd lengths entering the cache in float32, heads of 64, pages of 32
        dict(name="store_prefill_f32_g8_d64", kind="store", reqs=23, rows=16001, max_len=4096, bt=32, kv_heads=8, head_dim=64,
             dtype="f32"),
        # the next token of one long sequence: latency
        dict(name="attend_r1_h16kv2_l32768", kind="attend", reqs=1, max_len=32768, lens="even", bt=64, heads=16, kv_heads=2,
             head_dim=128, w_max=512, k_lmk=128, dtype="bf16"),
        # batch 256 of the same shape, ragged lengths
        dict(name="attend_r256_h16kv2_l8192", kind="attend", reqs=256, max_len=8192, lens="ragged", bt=64, heads=16, kv_heads=2,
             head_dim=128, w_max=512, k_lmk=128, dtype="bf16"),
        # a key/value head a query head, fp16, pages of 16, lengths from one token
        dict(name="attend_r33_h16_d64_f16", kind="attend", reqs=33, max_len=2049, lens="ragged", bt=16, heads=16, kv_heads=16,
             head_dim=64, w_max=256, k_lmk=64, dtype="f16"),
        # float32 rows, grouped heads, an odd batch
        dict(name="attend_r17_h8kv2_f32", kind="attend", reqs=17, max_len=2048, lens="ragged", bt=32, heads=8, kv_heads=2,
             head_dim=64, w_max=128, k_lmk=32, dtype="f32"),
        # windows as long as the sequence (dense attention of a few long requests)
        dict(name="attend_r4_h16kv2_w131072", kind="attend", reqs=4, max_len=131072, lens="even", bt=64, heads=16, kv_heads=2,
             head_dim=128, w_max=131072, k_lmk=256, dtype="bf16"),
        # one row of a 152K vocabulary, the usual filters: latency
        dict(name="sample_r1_v151936", kind="sample", rows=1, vocab=151936, dtype="bf16", mix="filters"),
        # a served batch, each row with settings of its own
        dict(name="sample_r256_v151936", kind="sample", rows=256, vocab=151936, dtype="bf16", mix="each"),
        # float32 logits of an odd vocabulary, temperature alone
        dict(name="sample_r37_v50257_f32", kind="sample", rows=37, vocab=50257, dtype="f32", mix="temperature"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["rows", "store", "store", "attend", "attend", "attend", "sample", "sample"])
    bt = rng.choice([16, 32, 64, 128])
    if kind == "rows":
        reqs = _log_int(rng, 1, 1500)
        mix = rng.choice(["decode", "mixed"])
        top = _log_int(rng, 600, 16384)
        return dict(kind=kind, reqs=reqs, rows=reqs if mix == "decode" else reqs + _log_int(rng, 64, min(32768, 64 + reqs * top // 32)),
                    max_len=top, bt=max(bt, 32), mix=mix)
    if kind == "store":
        reqs = _log_int(rng, 1, 256)
        top = _log_int(rng, 600, 4096)
        return dict(kind=kind, reqs=reqs, rows=reqs if rng.random() < 0.5 else _log_int(rng, reqs + 1, min(16001, reqs * top // 4)),
                    max_len=top, bt=bt, kv_heads=rng.choice([1, 2, 4, 8]), head_dim=rng.choice([64, 128]),
                    dtype=rng.choice(["bf16", "f16", "f32"]))
    if kind == "attend":
        heads = rng.choice([4, 8, 16, 32])
        c = dict(kind=kind, reqs=_log_int(rng, 1, 200), max_len=_log_int(rng, 130, 16384), lens=rng.choice(["even", "ragged", "ragged"]), bt=bt,
                 heads=heads, kv_heads=max(1, heads // rng.choice([1, 4, 8])), head_dim=rng.choice([64, 128]),
                 w_max=rng.choice([64, 128, 384, 512]), k_lmk=rng.choice([0, 16, 100, 128]), dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
        if rng.random() < 0.25:  # long windows of a few requests
            c.update(reqs=rng.randint(1, 4), max_len=_log_int(rng, 4096, 65536), w_max=65536)
        while c["reqs"] * c["max_len"] * c["kv_heads"] * c["head_dim"] > 1 << 29:
            c["reqs"] = c["reqs"] // 2
        while c["reqs"] * heads * c["head_dim"] * c["k_lmk"] > 1 << 27:
            c["reqs"] = c["reqs"] // 2
        return c
    return dict(kind=kind, rows=_log_int(rng, 1, 200), vocab=rng.choice([997, 32000, 50257, 128256, 151936]), dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                mix=rng.choice(["filters", "each", "temperature", "greedy"]))


# ------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=_DEV).manual_seed(int(seed) * 7919 + 29)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=_DEV)


def _batch(c, seed):
    """Host lists of a step: tokens held, new tokens, and the pages of the requests in a shuffled pool."""
    r = random.Random(int(seed) * 31 + c["reqs"])
    R, bt, top = c["reqs"], c["bt"], c["max_len"]
    mix = c.get("mix", "decode" if c["rows"] == R else "prefill")
    if mix == "decode":
        new = [1] * R
    else:  # most rows belong to a few prompts; the running requests take one each
        new = [-1 if mix == "mixed" and r.random() < 0.05 else 1 if mix == "mixed" else 0 for _ in range(R)]
        left = c["rows"] - sum(max(n, 0) for n in new)
        prompts = [i for i in range(R) if new[i] >= 0 and (mix != "mixed" or r.random() < 0.1)] or [max(range(R), key=lambda i: new[i])]
        cuts = sorted(r.randint(0, left) for _ in range(len(prompts) - 1))
        for i, a, b in zip(prompts, [0] + cuts, cuts + [left]):
            if new[i] >= 0:
                new[i] = new[i] + min(b - a, top // 2)
    old = [r.randint(0, max(0, top - max(n, 0))) if n >= 0 and (n <= 1 or r.random() < 0.5) else r.randint(1, top) if n < 0 else 0
           for n in new]
    return old, new


def _pool(c, old, new, seed):
    """table [R, M] with the pages held, the ring of free pages, and its (head, tail) counters."""
    bt, M = c["bt"], -(-c["max_len"] // c["bt"]) + 1
    held = [-(-n // bt) for n in old]
    need = [max(0, -(-(a + max(b, 0)) // bt) - h) for a, b, h in zip(old, new, held)]
    N = len(old) * M if c["kind"] == "rows" else sum(held) + sum(need) + 64
    ids = torch.randperm(N, generator=_gen(seed + 5), device=_DEV).to(torch.int32)
    h = torch.tensor(held, device=_DEV)
    j = torch.arange(M, device=_DEV)
    at = (torch.cumsum(h, 0) - h)[:, None] + j
    table = torch.where(j < h[:, None], ids[at.clamp(max=N - 1)], torch.full((), -1, dtype=torch.int32, device=_DEV))
    ring = torch.full((N,), -1, dtype=torch.int32, device=_DEV)
    first = 7  # the ring has turned before
    ring[(torch.arange(N - sum(held), device=_DEV) + first) % N] = ids[sum(held):]
    return table, ring, torch.tensor([first, first + N - sum(held)], dtype=torch.int64, device=_DEV), N


def _codes(x, scale):
    return (x / scale).clamp(-448.0, 448.0).to(_FP8)


def _filled(g, N, G, bt, D):
    """A page tensor holding N(0, 1) values with a few large channels, and its scales."""
    codes = torch.empty((N, G, bt, D), dtype=_FP8, device=_DEV)
    scale = torch.empty((N, G), device=_DEV)
    chan = torch.exp(0.7 * torch.randn(G, 1, D, generator=g, device=_DEV))
    step = max(1, (1 << 26) // (G * bt * D))
    for a in range(0, N, step):
        x = torch.randn(min(step, N - a), G, bt, D, generator=g, device=_DEV) * chan
        s = _scale_of(x.abs().amax(dim=(2, 3)))
        scale[a:a + step] = s
        codes[a:a + step] = _codes(x, s[..., None, None])
    return codes, scale


def _scale_of(amax):
    """The least power of two s with amax <= 448 s: amax = f 2^e, f in [1/2, 1), and 448 = 7/8 2^9."""
    f, e = torch.frexp(amax)
    e = torch.where(amax > 0, e - 9 + (f > 0.875).to(e.dtype), torch.full_like(e, -126)).clamp(-126, 119)
    return torch.exp2(e.double()).float()


def prepare(case, seed):
    c, g = dict(case), _gen(seed)
    kind, st = c["kind"], dict(c=c)
    if kind == "sample":
        R, V = c["rows"], c["vocab"]
        x = torch.randn(R, V, generator=g, device=_DEV) * 2.2
        lift = torch.randint(0, V, (R, 48), generator=g, device=_DEV)  # the few tokens that fit
        x.scatter_add_(1, lift, -3.0 * torch.log(torch.rand(R, 48, generator=g, device=_DEV).clamp(min=1e-3)) + 4)
        st["x"] = x.to(_DT[c["dtype"]])
        st["u"] = torch.rand(R, generator=g, device=_DEV)
        r = torch.rand(4, R, generator=g, device=_DEV)
        one, zero = torch.ones(R, device=_DEV), torch.zeros(R, dtype=torch.int32, device=_DEV)
        st.update(t=0.5 + r[0], k=zero, p=one, m=one * 0)
        if c["mix"] == "filters":
            st.update(k=zero + 50, p=one * 0.95, m=one * 0.02)
        elif c["mix"] == "greedy":
            st.update(t=one * 0)
        elif c["mix"] == "each":
            st.update(t=torch.where(r[0] < 0.1, one * 0, st["t"]), k=torch.where(r[1] < 0.5, zero, (r[1] * 400).int()),
                      p=torch.where(r[2] < 0.4, one, 0.5 + 0.5 * r[2]), m=torch.where(r[3] < 0.6, one * 0, 0.1 * r[3]))
        return st
    if kind in ("rows", "store"):
        old, new = _batch(c, seed if kind == "rows" else 0)  # what is read back of a store has the shape of the batch
        table, ring, span, N = _pool(c, old, new, seed)
        st.update(old=_i32(old), new=_i32(new), table=table, ring=ring, span=span)
        if kind == "rows":
            return st
        G, D, bt = c["kv_heads"], c["head_dim"], c["bt"]
        st["rows"] = _plain_rows(st["old"], st["new"], table, ring, span, c["rows"], bt)  # a step's rows serve all its layers
        k, ks = _filled(g, N, G, bt, D)
        v, vs = _filled(g, N, G, bt, D)
        st["cache"] = (k, v, ks, vs)
        qkv = torch.randn(c["rows"], 3 * G * D, generator=g, device=_DEV) * torch.exp(torch.randn(c["rows"], 1, generator=g, device=_DEV))
        qkv = qkv.to(_DT[c["dtype"]])  # columns of one projection
        st["k"], st["v"] = qkv[:, G * D:2 * G * D].view(-1, G, D), qkv[:, 2 * G * D:].view(-1, G, D)
        first = [n // bt * bt for n in old]  # what is read back: the blocks of the step's rows, whole
        lens = [(a + n - f) if n > 0 else 0 for a, n, f in zip(old, new, first)]
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        st.update(first=_i32(first), cu=_i32(cu), back=cu[-1])
        return st
    R, H, G, D, bt, K = (c[n] for n in ("reqs", "heads", "kv_heads", "head_dim", "bt", "k_lmk"))
    r = random.Random(int(seed) * 17 + R)
    lens = [c["max_len"] if c["lens"] == "even" or i == 0 else r.randint(1, c["max_len"]) for i in range(R)]
    held = [-(-n // bt) for n in lens]
    N, M = sum(held), max(held)
    ids = torch.randperm(N, generator=g, device=_DEV).to(torch.int32)
    h, j = torch.tensor(held, device=_DEV), torch.arange(M, device=_DEV)
    at = ((torch.cumsum(h, 0) - h)[:, None] + j).clamp(max=N - 1)
    st["table"] = torch.where(j < h[:, None], ids[at], torch.full((), -1, dtype=torch.int32, device=_DEV))
    k, ks = _filled(g, N, G, bt, D)
    v, vs = _filled(g, N, G, bt, D)
    st["cache"] = (k, v, ks, vs)
    st["q"] = torch.randn(R, H, D, generator=g, device=_DEV).to(_DT[c["dtype"]])
    n = torch.tensor(lens, device=_DEV)
    st["req"], st["pos"] = torch.arange(R, dtype=torch.int32, device=_DEV), (n - 1).to(torch.int32)
    if c["w_max"] > 512:
        w = torch.full((R,), c["w_max"], device=_DEV)
    else:
        w = torch.round((torch.sigmoid(torch.randn(R, generator=g, device=_DEV)) * c["w_max"]).clamp(min(16, c["w_max"])))
    st["w"] = w.to(torch.int32)
    lmk = (torch.rand(H, R, 1, K, generator=g, device=_DEV) * n[:, None, None]).long().sort(dim=-1).values
    dup = torch.zeros_like(lmk, dtype=torch.bool)
    dup[..., 1:] = lmk[..., 1:] == lmk[..., :-1]
    lmk = torch.where(dup, torch.full_like(lmk, 1 << 40), lmk).sort(dim=-1).values  # positions once, -1 last
    st["lmk"] = torch.where(lmk < (1 << 40), lmk, torch.full_like(lmk, -1)).to(torch.int32)
    return st


# ------------------------------------------------------------------------ plain forms
def _plain_rows(old, new, table, ring, span, n_rows, bt):
    """The step's rows: updates table and ring, returns (seq_len, span, granted, cu, req, pos, slot, pieces)."""
    R, M = table.shape
    N = ring.numel()
    dev = table.device
    old, new = old.long(), new.long()
    release = (new < 0) & (old >= 0)
    held = (-(-old // bt)).clamp(0, M)
    n = new.clamp(min=0)
    end = torch.cumsum(n, 0)
    fits = (new >= 0) & (old >= 0) & (old + n <= M * bt) & (end <= n_rows)
    need = torch.where(fits, (-(-(old + n) // bt)) - held, torch.zeros_like(n)).clamp(min=0)
    upto = torch.cumsum(need, 0)
    ok = fits & ((need == 0) | (upto <= span[1] - span[0]))
    off = upto - need
    back = torch.where(release, held, torch.zeros_like(held))
    boff = torch.cumsum(back, 0) - back
    # pages in and out, over the whole table
    j = torch.arange(M, device=dev)
    k = off[:, None] + j - held[:, None]
    grow = ok[:, None] & (j >= held[:, None]) & (j < (held + need)[:, None])
    at = span[1] + boff[:, None] + j
    give = release[:, None] & (j < held[:, None]) & (at - span[0] < N)
    grown = torch.where(grow, ring[((span[0] + k) % N)], table)
    ext = torch.cat([ring, ring.new_zeros(1)])
    ext.scatter_(0, torch.where(give, at % N, torch.full_like(at, N)).view(-1), table.reshape(-1))
    ring.copy_(ext[:N])
    table.copy_(grown)
    taken = torch.where(ok, upto * (need > 0), torch.zeros_like(upto)).max()
    tail = torch.minimum(span[1] + back.sum(), span[0] + N)
    seq = torch.where(ok, old + n, torch.where(release, torch.zeros_like(old), old)).to(torch.int32)
    cu = torch.cat([end.new_zeros(1), end])
    t = torch.arange(n_rows, device=dev)
    req = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    inside = req < R
    rc = req.clamp(max=R - 1)
    live = inside & ok[rc]
    pos = torch.where(live, old[rc] + t - cu[rc], torch.full_like(t, -1))
    page = table[rc, (pos // bt).clamp(0, M - 1)].long()
    slot = torch.where(live, page * bt + pos % bt, torch.full_like(t, -1))
    # pieces: runs of a request's rows within one block
    P = min(n_rows, n_rows // bt + 2 * R)
    lead = live & ((t == cu[rc]) | (pos % bt == 0))
    rank = torch.where(lead, torch.cumsum(lead, 0) - 1, torch.full_like(t, P))
    rows = torch.minimum(bt - pos % bt, cu[rc + 1] - t)
    pieces = torch.zeros((P + 1, 4), dtype=torch.int32, device=dev)
    pieces.scatter_(0, rank[:, None].expand(-1, 4), torch.stack([t, rows, page, pos % bt], 1).to(torch.int32))
    return (seq, torch.stack([span[0] + taken, tail]), (ok | release).to(torch.int32), cu.to(torch.int32),
            torch.where(inside, req, torch.full_like(req, -1)).to(torch.int32), pos.to(torch.int32), slot, pieces[:P].contiguous())


def _plain_write(x, codes, scale, pieces, req_rows):
    """x [T, G, D] into the blocks of `pieces`; req_rows: the piece of each row (P for a row without)."""
    T, G, D = x.shape
    bt = codes.shape[2]
    P = pieces.shape[0]
    x = x.float()
    x = torch.where(torch.isfinite(x), x, torch.full_like(x, float("nan")))
    amax = torch.zeros((P + 1, G), device=x.device)
    amax.scatter_reduce_(0, req_rows[:, None].expand(-1, G), x.abs().nan_to_num(0.0).amax(dim=2), "amax")
    # pieces past the last one repeat it: the same values are written twice
    last = (pieces[:, 1] > 0).sum() - 1
    at = torch.minimum(torch.arange(P, device=x.device), last).clamp(min=0)
    row0, rows, page, off = pieces[at].long().unbind(1)
    held = torch.where(off[:, None] > 0, scale[page], torch.zeros_like(scale[page]))
    s = torch.maximum(_scale_of(amax[at]), held)
    j = torch.arange(bt, device=x.device)
    vals = codes.view(torch.uint8)[page].view(_FP8).float()
    keep = (j < off[:, None])[:, None, :, None]
    vals = torch.where(keep, vals * (held / s)[..., None, None], vals)
    fresh = (j >= off[:, None]) & (j < (off + rows)[:, None])
    src = (row0[:, None] + j - off[:, None]).clamp(0, T - 1)
    put = (x[src] / s[:, None, :, None]).clamp(-448.0, 448.0).transpose(1, 2)
    vals = torch.where(fresh[:, None, :, None], put, vals)
    codes.view(torch.uint8)[page] = vals.to(_FP8).view(torch.uint8)
    scale[page] = s


def _plain_read(codes, scale, table, cu, first, n_rows, dt):
    bt, M = codes.shape[2], table.shape[1]
    t = torch.arange(n_rows, device=codes.device)
    cu = cu.long()
    r = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=table.shape[0] - 1)
    pos = t - cu[r] + first.long()[r]
    page = table[r, (pos // bt).clamp(0, M - 1)].long()
    return (codes.view(torch.uint8)[page, :, pos % bt].view(_FP8).float() * scale[page][..., None]).to(dt)


def _taken(codes, scale, table, req, head, pos):
    """Values at positions `pos` (any shape; the request and head broadcast with it), float32 [..., D]."""
    bt = codes.shape[2]
    pos = pos.clamp(min=0)
    page = table[req, (pos // bt).clamp(max=table.shape[1] - 1)].long().clamp(min=0)
    return codes.view(torch.uint8)[page, head, pos % bt].view(_FP8).float() * scale[page, head][..., None]


def _plain_attend(q, cache, table, req, pos, w, lmk, w_max):
    k, v, ks, vs = cache
    T, H, D = q.shape
    G, K = k.shape[1], lmk.shape[-1]
    dev = q.device
    qf = q.float() / math.sqrt(D)
    req, pos, w = req.long(), pos.long(), w.long().clamp(min=1)
    low = (pos - w + 1).clamp(min=0)
    j = low[:, None] + torch.arange(min(w_max, table.shape[1] * k.shape[2]), device=dev)      # [T, W]
    seen = (j <= pos[:, None])[:, None]                                                       # [T, 1, W]
    at = (table, req[:, None, None], torch.arange(G, device=dev)[None, :, None], j[:, None])
    s1 = torch.matmul(qf.view(T, G, H // G, D), _taken(k, ks, *at).transpose(2, 3)).view(T, H, -1)
    s1 = torch.where(seen, s1, torch.full_like(s1, float("-inf")))
    p = lmk[:, :, 0].transpose(0, 1)[req].long()                                              # [T, H, K]
    has = (p >= 0) & (p < (pos - w + 1)[:, None, None])
    al = (table, req[:, None, None], (torch.arange(H, device=dev) // (H // G))[None, :, None], p)
    s2 = (qf[:, :, None] * _taken(k, ks, *al)).sum(-1)
    s2 = torch.where(has, s2, torch.full_like(s2, float("-inf")))
    m = torch.maximum(s1.amax(-1), s2.amax(-1)) if K else s1.amax(-1)
    m0 = torch.where(torch.isinf(m), torch.zeros_like(m), m)[..., None]
    p1, p2 = torch.exp(s1 - m0), torch.exp(s2 - m0)
    l = p1.sum(-1) + p2.sum(-1)
    vw = torch.where(seen[..., None], _taken(v, vs, *at), torch.zeros((), device=dev))
    o = torch.matmul(p1.view(T, G, H // G, -1), vw).view(T, H, D)
    o = o + (p2[..., None] * torch.where(has[..., None], _taken(v, vs, *al), torch.zeros((), device=dev))).sum(2)
    o = torch.where(l[..., None] > 0, o / l[..., None], torch.zeros_like(o))
    return o.to(q.dtype), m0[..., 0] + torch.log(l)


def _plain_sample(x, u, temp, top_k, top_p, min_p):
    R, V = x.shape
    xs, ids = torch.sort(x.float().nan_to_num(nan=float("-inf"), posinf=float("inf"), neginf=float("-inf")), dim=1, descending=True,
                         stable=True)
    greedy = ~(temp > 0)
    t = torch.where(greedy, torch.ones_like(temp), temp).double()[:, None]
    w = torch.round(torch.exp((xs.double() - xs[:, :1].double()) / t) * _UNIT).long()
    n = torch.arange(V, device=x.device)
    kk = torch.where((top_k <= 0) | (top_k > V), torch.full_like(top_k, V), top_k)
    kk = torch.where(greedy, torch.ones_like(kk), kk)
    w = torch.where(n < kk[:, None], w, torch.zeros_like(w))
    cum = torch.cumsum(w, 1)
    keep = (cum - w).double() < top_p.double()[:, None] * cum[:, -1:].double()
    keep = keep & (w.double() >= min_p.double()[:, None] * _UNIT)
    keep[:, 0] = True
    kept = torch.zeros_like(w).scatter_(1, ids, torch.where(keep, w, torch.zeros_like(w)))  # in the order of the vocabulary
    cum = torch.cumsum(kept, 1)
    total = cum[:, -1:]
    hit = cum.double() > u.double()[:, None] * total.double()
    token = torch.argmax(hit.to(torch.uint8), dim=1)
    wt = kept.gather(1, token[:, None])
    return token, torch.log(wt.double() / total.double())[:, 0].float()


# ------------------------------------------------------------------------ one pass
def run(s):
    c = s["c"]
    kind = c["kind"]
    if kind == "sample":
        a = (s["x"], s["u"], s["t"], s["k"], s["p"], s["m"])
        if own:
            from dsalt_amd import ops
            return list(ops.sample_rows(a[0], a[1], temperature=a[2], top_k=a[3], top_p=a[4], min_p=a[5]))
        return list(_plain_sample(*a))
    if kind == "rows":
        if own:
            from dsalt_amd import ops
            rows = ops.cache_rows_(s["old"], s["new"], s["table"], s["ring"], s["span"], c["rows"], block_tokens=c["bt"])
        else:
            rows = _plain_rows(s["old"], s["new"], s["table"], s["ring"], s["span"], c["rows"], c["bt"])
        return [*rows, s["table"], s["ring"]]
    if kind == "store":
        dt = s["k"].dtype
        if own:
            from dsalt_amd import ops
            cache = ops.Cache8(*s["cache"])
            ops.cache_write_(s["k"], s["v"], cache, s["rows"][-1])
            return list(ops.cache_read(cache, s["table"], s["cu"], start=s["first"], n_rows=s["back"], dtype=dt))
        pieces = s["rows"][-1]
        piece = torch.searchsorted(torch.where(pieces[:, 1] > 0, pieces[:, 0], torch.full_like(pieces[:, 0], c["rows"])).contiguous(),
                                   torch.arange(c["rows"], dtype=torch.int32, device=_DEV), right=True) - 1
        piece = torch.where((s["rows"][5] >= 0) & (piece >= 0), piece, torch.full_like(piece, pieces.shape[0]))
        k, v, ks, vs = s["cache"]
        _plain_write(s["k"], k, ks, pieces, piece)
        _plain_write(s["v"], v, vs, pieces, piece)
        return [_plain_read(*y, s["table"], s["cu"], s["first"], s["back"], dt) for y in ((k, ks), (v, vs))]
    a = (s["table"], s["req"], s["pos"], s["w"], s["lmk"])
    if own:
        from dsalt_amd import ops
        return list(ops.cache_attention(s["q"], ops.Cache8(*s["cache"]), *a, w_max=c["w_max"]))
    return list(_plain_attend(s["q"], s["cache"], *a, c["w_max"]))


# ------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = dict(case)
    kind = c["kind"]
    if kind == "sample":
        es = 4 if c["dtype"] == "f32" else 2
        return {"bytes": c["rows"] * (c["vocab"] * es + 32), "flops": 4.0 * c["rows"] * c["vocab"]}
    if kind == "rows":
        R, T, M = c["reqs"], c["rows"], -(-c["max_len"] // c["bt"]) + 1
        P = min(T, T // c["bt"] + 2 * R)
        # lengths in and out, row maps, pieces, and the table entries that rows or releases look up
        return {"bytes": R * 4 * 5 + T * (4 + 4 + 8) + P * 20, "flops": 8.0 * (R + T)}
    if kind == "store":
        T, G, D, R, bt = c["rows"], c["kv_heads"], c["head_dim"], c["reqs"], c["bt"]
        es = 4 if c["dtype"] == "f32" else 2
        back = T + (bt // 2) * R  # rows read back: the step's own and those before them in their first block
        return {"bytes": 2.0 * G * D * (T * (es + 1) + back * (1 + es)) + 16.0 * G * (T // bt + R), "flops": 4.0 * G * D * (T + back)}
    R, H, G, D, K = c["reqs"], c["heads"], c["kv_heads"], c["head_dim"], c["k_lmk"]
    es = 4 if c["dtype"] == "f32" else 2
    mean = c["max_len"] if c["lens"] == "even" else (c["max_len"] + 1) / 2
    win = min(c["w_max"] / 2 if c["w_max"] <= 512 else c["w_max"], mean)
    lm = min(K, max(0.0, mean - win))
    tokens = min(mean, win + lm * (H // G))  # of a key/value head: the window, and its query heads' landmarks
    return {"bytes": R * (2.0 * G * D * tokens + 2.0 * H * D * es + 4 * H * (K + 1)), "flops": 4.0 * R * H * D * (win + lm)}


# ------------------------------------------------------------------------ the definitions in 64 bits
def _e4m3(x):
    """x rounded to the nearest e4m3 number (ties to even), float64."""
    a = np.minimum(np.abs(x), 448.0)
    e = np.floor(np.log2(np.maximum(a, 2.0 ** -6)))
    step = np.exp2(e - 3)
    return np.copysign(np.rint(a / step) * step, x)


def _host(t):
    return t.detach().cpu().double().numpy() if t.is_floating_point() or t.dtype == _FP8 else t.cpu().numpy()


def _exact_store(s):
    out = []
    pieces, table, cu, first = (_host(t) for t in (s["rows"][-1], s["table"], s["cu"], s["first"]))
    for x, codes, scale in ((s["k"], s["cache"][0], s["cache"][2]), (s["v"], s["cache"][1], s["cache"][3])):
        x, scale = _host(x.float()), _host(scale)
        bt = codes.shape[2]
        pages = sorted(set(int(p) for p in pieces[pieces[:, 1] > 0, 2]))
        at = {p: i for i, p in enumerate(pages)}
        c = _host(codes.view(torch.uint8)[torch.tensor(pages, device=_DEV)].view(_FP8).float())
        sc = scale[pages]
        for row0, rows, page, off in pieces:
            if rows == 0:
                continue
            i = at[int(page)]
            new = x[row0:row0 + rows].transpose(1, 0, 2)
            top = np.where(np.isfinite(new), np.abs(new), 0.0).max(axis=(1, 2))
            need = np.exp2(np.clip(np.ceil(np.log2(np.maximum(top, 1e-300) / 448.0)), -126, 119))
            was = sc[i] if off > 0 else np.zeros_like(need)
            now = np.maximum(need, was)
            c[i][:, :off] = _e4m3(c[i][:, :off] * (was / now)[:, None, None])
            c[i][:, off:off + rows] = np.where(np.isfinite(new), _e4m3(new / now[:, None, None]), np.nan)
            sc[i] = now
        vals = c * sc[..., None, None]
        got = np.zeros((s["back"],) + x.shape[1:])
        for r in range(len(cu) - 1):
            p = np.arange(cu[r + 1] - cu[r]) + first[r]
            if p.size:
                got[cu[r]:cu[r + 1]] = vals[[at[int(b)] for b in table[r, p // bt]], :, p % bt]
        out.append(torch.from_numpy(got))
    return out


def _exact_attend(s):
    q = s["q"].double() / math.sqrt(s["q"].shape[-1])
    k, v, ks, vs = s["cache"]
    T, H, D = q.shape
    G, bt = k.shape[1], k.shape[2]
    k8, v8 = k.view(torch.uint8), v.view(torch.uint8)
    out, lse = torch.zeros(T, H, D, dtype=torch.float64, device=_DEV), torch.zeros(T, H, dtype=torch.float64, device=_DEV)
    pos, w, lens = s["pos"].tolist(), s["w"].tolist(), s["lmk"].shape[-1]
    for t in range(T):
        i, low = pos[t], max(0, pos[t] - max(w[t], 1) + 1)
        tab = s["table"][t].long()

        def values(codes, scale, heads, p):  # [heads, n, D]
            page = tab[p // bt]
            return codes[page, heads, p % bt].view(_FP8).double() * scale[page, heads].double()[..., None]
        j = torch.arange(low, i + 1, device=_DEV)[None]
        g = torch.arange(G, device=_DEV)[:, None]
        kw, vw = values(k8, ks, g, j), values(v8, vs, g, j)
        sw = torch.bmm(q[t].view(G, H // G, D), kw.transpose(1, 2).contiguous()).view(H, -1)
        p = s["lmk"][:, t, 0].long()
        ok = (p >= 0) & (p < low)
        hg = (torch.arange(H, device=_DEV) // (H // G))[:, None]
        pc = p.clamp(min=0)
        sl = (values(k8, ks, hg, pc) * q[t][:, None]).sum(-1).masked_fill(~ok, float("-inf"))
        a = torch.softmax(torch.cat([sw, sl], 1), 1)
        n = sw.shape[1]
        out[t] = torch.bmm(a[:, :n].reshape(G, H // G, n), vw).view(H, D)
        if lens:
            out[t] += (a[:, n:, None] * values(v8, vs, hg, pc)).sum(1)
        lse[t] = torch.logsumexp(torch.cat([sw, sl], 1), 1)
    return [out, lse]


def _exact_sample(s):
    x = _host(s["x"])
    u, t, k, p, m = (_host(s[n]).tolist() for n in ("u", "t", "k", "p", "m"))
    tok, lp = np.zeros(len(u), dtype=np.int64), np.zeros(len(u))
    for r in range(len(u)):
        order = np.argsort(-x[r], kind="stable")
        top = x[r][order[0]]
        w = np.rint(np.exp((x[r] - top) / t[r]) * _UNIT).astype(np.int64) if t[r] > 0 else (np.arange(x.shape[1]) == order[0]).astype(np.int64)
        if 0 < k[r] < len(order):
            order = order[:k[r]]
        before = np.concatenate([[0], np.cumsum(w[order])])
        stay = (before[:-1] < p[r] * float(before[-1])) & ((w[order] >= m[r] * _UNIT) | (t[r] <= 0))
        stay[0] = True
        kept = np.zeros_like(w)
        kept[order[stay]] = w[order[stay]]
        cum = np.cumsum(kept)
        tok[r] = np.flatnonzero(cum > u[r] * float(cum[-1]))[0]
        lp[r] = math.log(kept[tok[r]] / cum[-1])
    return [torch.from_numpy(tok), torch.from_numpy(lp)]


def exact(case, seed):
    kind = case["kind"]
    if kind == "rows":
        return None  # whole numbers alone
    s = prepare(case, seed)
    return {"store": _exact_store, "attend": _exact_attend, "sample": _exact_sample}[kind](s)
