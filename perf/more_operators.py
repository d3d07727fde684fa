"""The operators of a step of speculative decoding over a paged 4-bit key/value cache, in their plain
form and through the framework, with the cases they are timed on.

Kinds of case (the ``kind`` of a case's dict):
  qk      a norm of every query and key head and the rotation after it, in one pass
          (``ops.qk_norm_rope``), by sequence or by position, and its gradients
          (``ops.qk_norm_rope_backward``)
  store   a step's keys and values written into a 4-bit cache (``ops.cache_write_``) and read back as
          values (``ops.cache_read``)
  attend  attention of single query tokens and of runs of drafted tokens over the 4-bit cache: the
          causal window and the landmarks of each row (``ops.cache_attention``)
  verify  drafted tokens taken or refused against the target's probabilities, from given random
          numbers, and the token that follows them (``ops.verify_rows``)

The norm: n = x / sqrt(mean(x^2) + eps) * weight over a head; the rotation of its halves n1, n2 at
position p: n1 cos[p, :D/2] - n2 sin[p, :D/2] and n2 cos[p, D/2:] + n1 sin[p, D/2:].

The cache: pages of ``bt`` tokens, ``kv`` [blocks, kv_heads, bt, 2, D/2] bytes of two e2m1 codes each
(0, 1/2, 1, 3/2, 2, 3, 4, 6 and a sign; the first element in the lower half), a token's key before its
value, and ``scale`` [blocks, kv_heads, bt, 2, D/32], the exponent of a power of two above -127 for
each 32 elements.  That is the least power of two s, from 2^-126 to 2^125, with all 32 within 7 s;
elements are rounded to the nearest code, ties to the even one, past 6 s to 6 s.  32 elements of which
one is not finite are held as NaN (exponent 255).

Verification weighs a logit x of a row with largest m as round(2^42 exp((x - m) / temperature)), a
whole number, a probability being a weight over the row's total; what is left of a refused row's
probabilities, max(p - q, 0), is weighed in whole multiples of 2^-52.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_DEV = "cuda"
_EPS = 1e-6
_LUT = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------------ the cases
def listed():
    return [
        # queries and keys of a 32K prompt, 16/2 heads of 128: an inference pass
        dict(name="qk_fwd_l32768_h16kv2_d128", kind="qk", way="fwd", seqs=1, rows=32768, heads=16, kv_heads=2, head_dim=128,
             dtype="bf16"),
        # the gradients of a packed training batch, as many key/value heads as query heads, odd lengths
        dict(name="qk_bwd_s5_t16001_h16_d64", kind="qk", way="bwd", seqs=5, rows=16001, heads=16, kv_heads=16, head_dim=64,
             dtype="bf16"),
        # the next token of one sequence: latency
        dict(name="qk_decode_r1_h16kv2_d128", kind="qk", way="pos", seqs=1, rows=1, heads=16, kv_heads=2, head_dim=128,
             dtype="bf16"),
        # decoding at batch 256 of the 16/2-head shape: a token a request
        dict(name="store_decode_r256_g2_d128", kind="store", reqs=256, rows=256, max_len=4096, bt=64, kv_heads=2, head_dim=128,
             dtype="bf16"),
        # prompts of odd lengths entering the cache in float32, heads of 64, pages of 32
        dict(name="store_prefill_f32_g8_d64", kind="store", reqs=23, rows=16001, max_len=4096, bt=32, kv_heads=8, head_dim=64,
             dtype="f32"),
        # the next token of one long sequence: latency
        dict(name="attend_r1_h16kv2_l32768", kind="attend", reqs=1, per=1, max_len=32768, lens="even", bt=64, heads=16, kv_heads=2,
             head_dim=128, w_max=512, k_lmk=128, dtype="bf16"),
        # a served batch, a token a request, ragged lengths
        dict(name="attend_r256_h16kv2_l8192", kind="attend", reqs=256, per=1, max_len=8192, lens="ragged", bt=64, heads=16,
             kv_heads=2, head_dim=128, w_max=512, k_lmk=128, dtype="bf16"),
        # four drafted tokens and one more of 64 requests, fp16, pages of 16
        dict(name="attend_r64x5_h16kv4_f16", kind="attend", reqs=64, per=5, max_len=8192, lens="ragged", bt=16, heads=16,
             kv_heads=4, head_dim=64, w_max=512, k_lmk=128, dtype="f16"),
        # windows as long as the sequence (dense attention of a few long requests)
        dict(name="attend_r4_h16kv2_w131072", kind="attend", reqs=4, per=1, max_len=131072, lens="even", bt=64, heads=16,
             kv_heads=2, head_dim=128, w_max=131072, k_lmk=256, dtype="bf16"),
        # four drafts of one request against a 152K vocabulary: latency
        dict(name="verify_r1x5_v151936", kind="verify", reqs=1, most=4, vocab=151936, dtype="bf16", lens="even", draft="logits"),
        # a served batch, up to four drafts a request, each with a temperature of its own, some greedy
        dict(name="verify_r64x5_v151936", kind="verify", reqs=64, most=4, vocab=151936, dtype="bf16", lens="ragged", draft="logits"),
        # drafts looked up in the text (certain of themselves), float32 logits of an odd vocabulary
        dict(name="verify_r37x9_v50257_f32", kind="verify", reqs=37, most=8, vocab=50257, dtype="f32", lens="ragged", draft="none"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["qk", "qk", "store", "attend", "attend", "attend", "verify", "verify"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    heads = rng.choice([4, 8, 16, 32])
    kv = max(1, heads // rng.choice([1, 4, 8]))
    if kind == "qk":
        way = rng.choice(["fwd", "bwd", "pos"])
        c = dict(kind=kind, way=way, seqs=1, rows=_log_int(rng, 1, 512 if way == "pos" else 32768), heads=heads, kv_heads=kv,
                 head_dim=rng.choice([32, 64, 96, 128]), dtype=dtype)
        while c["rows"] * (heads + kv) * c["head_dim"] > 1 << 26:
            c["rows"] = c["rows"] // 2
        c["seqs"] = rng.randint(1, min(c["rows"], 9))
        return c
    bt = rng.choice([16, 32, 64, 128])
    if kind == "store":
        reqs = _log_int(rng, 1, 256)
        top = _log_int(rng, 600, 4096)
        return dict(kind=kind, reqs=reqs, rows=reqs if rng.random() < 0.5 else _log_int(rng, reqs + 1, min(16001, reqs * top // 4)),
                    max_len=top, bt=bt, kv_heads=rng.choice([1, 2, 4, 8]), head_dim=rng.choice([64, 128]), dtype=dtype)
    if kind == "attend":
        c = dict(kind=kind, reqs=_log_int(rng, 1, 200), per=rng.choice([1, 1, 2, 4, 5, 8]), max_len=_log_int(rng, 130, 16384),
                 lens=rng.choice(["even", "ragged", "ragged"]), bt=bt, heads=heads, kv_heads=kv, head_dim=rng.choice([64, 128]),
                 w_max=rng.choice([64, 128, 384, 512]), k_lmk=rng.choice([0, 16, 100, 128]), dtype=dtype)
        if rng.random() < 0.25:  # long windows of a few requests
            c.update(reqs=rng.randint(1, 4), per=rng.choice([1, 3]), max_len=_log_int(rng, 4096, 32768), w_max=65536)
        while c["reqs"] > 1 and c["reqs"] * c["per"] * min(c["max_len"], c["w_max"]) * kv * c["head_dim"] > 1 << 27:
            c["reqs"] = c["reqs"] // 2
        while c["reqs"] > 1 and c["reqs"] * c["per"] * heads * c["head_dim"] * c["k_lmk"] > 1 << 27:
            c["reqs"] = c["reqs"] // 2
        return c
    c = dict(kind=kind, reqs=_log_int(rng, 1, 64), most=rng.choice([1, 3, 4, 8]), vocab=rng.choice([997, 32000, 50257, 128256, 151936]),
             dtype=dtype, lens=rng.choice(["even", "ragged"]), draft=rng.choice(["logits", "logits", "none"]))
    while c["reqs"] > 1 and c["reqs"] * (c["most"] + 1) * c["vocab"] * (2 if dtype == "f32" else 1) > 320 * 151936:
        c["reqs"] = c["reqs"] // 2
    return c


# ------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=_DEV).manual_seed(int(seed) * 7919 + 31)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=_DEV)


def _cuts(r, total, parts):
    """Offsets of `parts` non-empty runs of `total` rows."""
    return [0] + sorted(r.sample(range(1, total), parts - 1)) + [total]


def _tables(rows, D):
    """cos and sin [rows, D] of the rotation (base 10^6), both halves alike."""
    theta = 1e6 ** (-torch.arange(0, D, 2, device=_DEV, dtype=torch.float64) / D)
    ang = torch.arange(rows, device=_DEV, dtype=torch.float64)[:, None] * theta
    ang = torch.cat([ang, ang], 1)
    return ang.cos().float(), ang.sin().float()


def _encode(x):
    """Codes (uint8 [..., D/2]) and exponents (uint8 [..., D/32]) of float32 x [..., D]."""
    b = x.unflatten(-1, (-1, 32))
    ok = torch.isfinite(b).all(-1, keepdim=True)
    b = torch.where(ok, b, torch.zeros_like(b))
    f, e = torch.frexp(b.abs().amax(-1, keepdim=True))  # f 2^e, f in [1/2, 1); 7 = 7/8 2^3
    e = torch.where(f > 0, e - 3 + (f > 0.875).to(e.dtype), torch.full_like(e, -126)).clamp(-126, 125)
    y = torch.ldexp(b, -e)
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)).to(torch.uint8)
    code = (code + 8 * (y < 0).to(torch.uint8)).flatten(-2)
    return code[..., 0::2] + 16 * code[..., 1::2], torch.where(ok, e + 127, torch.full_like(e, 255))[..., 0].to(torch.uint8)


def _decode(codes, exps):
    """Values (float32 [..., D]) of codes [..., D/2] and exponents [..., D/32]."""
    lut = torch.tensor(_LUT + tuple(-v for v in _LUT), device=codes.device)
    c = codes.int()
    x = torch.stack([lut[c & 15], lut[c >> 4]], -1).flatten(-2).unflatten(-1, (-1, 32))
    s = torch.exp2(exps.float() - 127.0)
    s = torch.where(exps == 255, torch.full_like(s, float("nan")), s)
    return (x * s[..., None]).flatten(-2)


def _filled(g, N, G, bt, D):
    """Pages holding keys and values: N(0, 1) with a few large channels."""
    kv = torch.empty((N, G, bt, 2, D // 2), dtype=torch.uint8, device=_DEV)
    scale = torch.empty((N, G, bt, 2, D // 32), dtype=torch.uint8, device=_DEV)
    chan = torch.exp(0.7 * torch.randn(G, 1, 2, D, generator=g, device=_DEV))
    step = max(1, (1 << 25) // (G * bt * D))
    for a in range(0, N, step):
        kv[a:a + step], scale[a:a + step] = _encode(torch.randn(min(step, N - a), G, bt, 2, D, generator=g, device=_DEV) * chan)
    return kv, scale


def _pages(g, held):
    """table [R, pages] of shuffled pages, -1 behind those held, and the number of pages."""
    N, M = sum(held), max(held) + 1
    ids = torch.randperm(N, generator=g, device=_DEV).to(torch.int32)
    h, j = torch.tensor(held, device=_DEV), torch.arange(M, device=_DEV)
    at = ((torch.cumsum(h, 0) - h)[:, None] + j).clamp(max=N - 1)
    return torch.where(j < h[:, None], ids[at], torch.full((), -1, dtype=torch.int32, device=_DEV)), N


def prepare(case, seed):
    c, g = dict(case), _gen(seed)
    kind, st = c["kind"], dict(c=c)
    if kind == "qk":
        T, H, G, D = c["rows"], c["heads"], c["kv_heads"], c["head_dim"]
        r = random.Random(int(seed) * 13 + T)
        dt = _DT[c["dtype"]]
        qkv = torch.randn(T, (H + 2 * G) * D, generator=g, device=_DEV) * torch.exp(0.5 * torch.randn(T, 1, generator=g, device=_DEV))
        qkv = qkv.to(dt)  # one projection's columns
        st["q"], st["k"] = qkv[:, :H * D].view(T, H, D), qkv[:, H * D:(H + G) * D].view(T, G, D)
        st["qw"], st["kw"] = (1.0 + 0.2 * torch.randn(D, generator=g, device=_DEV) for _ in range(2))
        if c["way"] == "pos":  # the tables of a served model, rows anywhere in it
            st["cos"], st["sin"] = _tables(32768, D)
            st["pos"] = torch.randint(0, 32768, (T,), generator=g, device=_DEV, dtype=torch.int32)
            return st
        cu = _cuts(r, T, c["seqs"])
        st["max_len"] = max(b - a for a, b in zip(cu, cu[1:]))
        st["cu"] = _i32(cu)
        st["cos"], st["sin"] = _tables(st["max_len"], D)
        if c["way"] == "bwd":
            st["dq"] = torch.randn(T, H, D, generator=g, device=_DEV).to(dt)
            st["dk"] = torch.randn(T, G, D, generator=g, device=_DEV).to(dt)
        return st
    if kind == "store":
        R, T, G, D, bt, top = (c[n] for n in ("reqs", "rows", "kv_heads", "head_dim", "bt", "max_len"))
        r = random.Random(R * 31 + T)  # the batch's shape is the case's
        new = [1] * R
        if T > R:  # prompts share the rows
            cuts = sorted(r.randint(0, T - R) for _ in range(R - 1))
            new = [1 + min(b - a, top - 1) for a, b in zip([0] + cuts, cuts + [T - R])]
        old = [r.randint(0, top - n) if T == R or r.random() < 0.5 else 0 for n in new]
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        T = cu[-1]
        st["table"], N = _pages(g, [-(-(a + n) // bt) for a, n in zip(old, new)])
        tab = st["table"].tolist()
        pieces = []
        for q, (a, n) in enumerate(zip(old, new)):
            p = a
            while p < a + n:
                k = min(bt - p % bt, a + n - p)
                pieces.append([cu[q] + p - a, k, tab[q][p // bt], p % bt])
                p += k
        st["pieces"], st["cu"], st["start"], st["rows"] = _i32(pieces), _i32(cu), _i32(old), T
        st["cache"] = _filled(g, N, G, bt, D)
        qkv = torch.randn(T, 3 * G * D, generator=g, device=_DEV) * torch.exp(torch.randn(T, 1, generator=g, device=_DEV))
        qkv = qkv.to(_DT[c["dtype"]])
        st["k"], st["v"] = qkv[:, G * D:2 * G * D].view(-1, G, D), qkv[:, 2 * G * D:].view(-1, G, D)
        return st
    if kind == "attend":
        R, n, H, G, D, bt, K = (c[x] for x in ("reqs", "per", "heads", "kv_heads", "head_dim", "bt", "k_lmk"))
        r = random.Random(int(seed) * 17 + R)
        lens = [c["max_len"] if c["lens"] == "even" or i == 0 else r.randint(n, c["max_len"]) for i in range(R)]
        st["table"], N = _pages(g, [-(-x // bt) for x in lens])
        st["cache"] = _filled(g, N, G, bt, D)
        st["q"] = torch.randn(R * n, H, D, generator=g, device=_DEV).to(_DT[c["dtype"]])
        ln = torch.tensor(lens, device=_DEV)
        st["req"] = torch.arange(R, dtype=torch.int32, device=_DEV).repeat_interleave(n)
        st["pos"] = (ln[:, None] - n + torch.arange(n, device=_DEV)).view(-1).to(torch.int32)
        if c["w_max"] > 512:
            w = torch.full((R * n,), c["w_max"], device=_DEV)
        else:
            w = torch.round((torch.sigmoid(torch.randn(R * n, generator=g, device=_DEV)) * c["w_max"]).clamp(min(16, c["w_max"])))
        st["w"] = w.to(torch.int32)
        lmk = (torch.rand(H, R, 1, K, generator=g, device=_DEV) * ln[:, None, None]).long().sort(dim=-1).values
        dup = torch.zeros_like(lmk, dtype=torch.bool)
        dup[..., 1:] = lmk[..., 1:] == lmk[..., :-1]
        lmk = torch.where(dup, torch.full_like(lmk, 1 << 40), lmk).sort(dim=-1).values  # positions once, -1 last
        st["lmk"] = torch.where(lmk < (1 << 40), lmk, torch.full_like(lmk, -1)).to(torch.int32)
        return st
    R, V = c["reqs"], c["vocab"]
    r = random.Random(R * 19 + c["most"])  # the batch's shape is the case's
    cu = [0]
    for i in range(R):
        cu.append(cu[-1] + 1 + (c["most"] if c["lens"] == "even" or i == 0 else r.randint(0, c["most"])))
    T = cu[-1]
    st["cu"] = _i32(cu)
    x = torch.randn(T, V, generator=g, device=_DEV) * 2.2
    lift = torch.randint(0, V, (T, 48), generator=g, device=_DEV)  # the few tokens that fit
    x.scatter_add_(1, lift, -3.0 * torch.log(torch.rand(T, 48, generator=g, device=_DEV).clamp(min=1e-3)) + 4)
    temp = 0.5 + torch.rand(R, generator=g, device=_DEV)
    if R > 8:
        temp = torch.where(torch.rand(R, generator=g, device=_DEV) < 0.1, torch.zeros_like(temp), temp)  # some greedy
    st["temp"] = temp
    trow = temp[torch.repeat_interleave(torch.arange(R, device=_DEV), st["cu"].diff().long())].clamp(min=0.05)[:, None]
    y = x + 0.7 * torch.randn(T, V, generator=g, device=_DEV)  # a draft model that mostly agrees
    st["x"], st["y"] = x.to(_DT[c["dtype"]]), None
    if c["draft"] == "logits":
        st["y"] = y.to(_DT[c["dtype"]])
    gumbel = -torch.log(-torch.log(torch.rand(T, V, generator=g, device=_DEV).clamp(1e-9, 1 - 1e-7)))
    tok = torch.argmax((st["y"].float() if st["y"] is not None else x) / trow + gumbel, 1)
    st["tok"] = torch.cat([torch.zeros_like(tok[:1]), tok[:-1]])  # a row's draft is the token fed to the next row
    st["u"], st["v"] = torch.rand(T, generator=g, device=_DEV), torch.rand(R, generator=g, device=_DEV)
    return st


# ------------------------------------------------------------------------ plain forms
def _plain_positions(s):
    if "pos" in s:
        return s["pos"].long()
    t = torch.arange(s["q"].shape[0], device=_DEV)
    cu = s["cu"].long()
    return t - cu[torch.searchsorted(cu, t, right=True) - 1]


def _plain_qk(x, w, cos, sin):
    x, half = x.float(), x.shape[-1] // 2
    n = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * w
    n1, n2 = n[..., :half], n[..., half:]
    return torch.cat([n1 * cos[..., :half] - n2 * sin[..., :half], n2 * cos[..., half:] + n1 * sin[..., half:]], -1)


def _plain_qk_grad(d, x, w, cos, sin):
    d, x, half = d.float(), x.float(), x.shape[-1] // 2
    d1, d2 = d[..., :half], d[..., half:]
    dn = torch.cat([d1 * cos[..., :half] + d2 * sin[..., half:], d2 * cos[..., half:] - d1 * sin[..., :half]], -1)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
    xh, g = x * r, dn * w
    return r * (g - xh * (g * xh).mean(-1, keepdim=True)), (dn * xh).sum((0, 1))


def _plain_write(x, kv, scale, at, which):
    """x [T, G, D] into the tokens `at` (page and place of each row)."""
    codes, exps = _encode(x.float())
    kv[at[0], :, at[1], which] = codes
    scale[at[0], :, at[1], which] = exps


def _plain_slots(pieces, n_rows, bt):
    t = torch.arange(n_rows, device=_DEV)
    p = pieces.long()
    i = torch.searchsorted(p[:, 0].contiguous(), t, right=True) - 1
    return p[i, 2], p[i, 3] + t - p[i, 0]


def _taken(cache, table, req, head, pos, which):
    """Values at positions `pos` (any shape; the request and head broadcast with it), float32 [..., D]."""
    kv, scale = cache
    bt = kv.shape[2]
    pos = pos.clamp(min=0)
    page = table[req, (pos // bt).clamp(max=table.shape[1] - 1)].long().clamp(min=0)
    return _decode(kv[page, head, pos % bt, which], scale[page, head, pos % bt, which])


def _plain_attend(q, cache, table, req, pos, w, lmk, w_max):
    T, H, D = q.shape
    G, K = cache[0].shape[1], lmk.shape[-1]
    qf = q.float() / math.sqrt(D)
    req, pos, w = req.long(), pos.long(), w.long().clamp(min=1)
    low = (pos - w + 1).clamp(min=0)
    j = low[:, None] + torch.arange(min(w_max, table.shape[1] * cache[0].shape[2]), device=_DEV)     # [T, W]
    seen = (j <= pos[:, None])[:, None]                                                              # [T, 1, W]
    at = (cache, table, req[:, None, None], torch.arange(G, device=_DEV)[None, :, None], j[:, None])
    s1 = torch.matmul(qf.view(T, G, H // G, D), _taken(*at, 0).transpose(2, 3).contiguous()).view(T, H, -1)
    s1 = torch.where(seen, s1, torch.full_like(s1, float("-inf")))
    p = lmk[:, :, 0].transpose(0, 1)[req].long()                                                     # [T, H, K]
    has = (p >= 0) & (p < (pos - w + 1)[:, None, None])
    al = (cache, table, req[:, None, None], (torch.arange(H, device=_DEV) // (H // G))[None, :, None], p)
    s2 = (qf[:, :, None] * _taken(*al, 0)).sum(-1)
    s2 = torch.where(has, s2, torch.full_like(s2, float("-inf")))
    m = torch.maximum(s1.amax(-1), s2.amax(-1)) if K else s1.amax(-1)
    m0 = torch.where(torch.isinf(m), torch.zeros_like(m), m)[..., None]
    p1, p2 = torch.exp(s1 - m0), torch.exp(s2 - m0)
    l = p1.sum(-1) + p2.sum(-1)
    vw = torch.where(seen[..., None], _taken(*at, 1), torch.zeros((), device=_DEV))
    o = torch.matmul(p1.view(T, G, H // G, -1), vw).view(T, H, D)
    o = o + (p2[..., None] * torch.where(has[..., None], _taken(*al, 1), torch.zeros((), device=_DEV))).sum(2)
    o = torch.where(l[..., None] > 0, o / l[..., None], torch.zeros_like(o))
    return o.to(q.dtype), m0[..., 0] + torch.log(l)


def _plain_weights(x, temp):
    """Whole weights (float64) of the rows of x and their totals; temperature 0 and below: the first largest alone."""
    xd = x.double().nan_to_num(nan=float("-inf"), posinf=1e39, neginf=float("-inf"))
    m = xd.amax(1, keepdim=True)
    w = torch.round(torch.exp((xd - m) / torch.where(temp > 0, temp, torch.ones_like(temp)).double()[:, None]) * 2.0 ** 42)
    first = torch.arange(x.shape[1], device=x.device) == torch.argmax(xd, 1, keepdim=True)
    w = torch.where((temp > 0)[:, None], w, first * 2.0 ** 42)
    w = torch.where(torch.isneginf(m), torch.zeros_like(w), w)
    return w, w.sum(1)


def _plain_verify(x, tok, cu, u, v, y, temp):
    """(drafts taken [R], tokens of the rows [T]): the taken drafts, the token that follows, -1 behind it."""
    T, V = x.shape
    R = cu.numel() - 1
    cu = cu.long()
    t = torch.arange(T, device=x.device)
    req = torch.searchsorted(cu, t, right=True) - 1
    trow = temp[req]
    last = t == cu[req + 1] - 1
    draft = torch.where(last, torch.zeros_like(tok), torch.cat([tok[1:], tok[:1]]))
    a, total = _plain_weights(x, trow)
    p = a.gather(1, draft[:, None])[:, 0] / total
    if y is not None:
        b, btotal = _plain_weights(y, trow)
        q = b.gather(1, draft[:, None])[:, 0] / btotal
    else:
        q = torch.ones_like(p)
    refused = (u.double() * q >= p) | last
    taken = torch.full((R,), T, device=x.device).scatter_reduce_(0, req, torch.where(refused, t - cu[req], torch.full_like(t, T)), "amin")
    row = cu[:-1] + taken
    a, total = a[row], total[row]
    if y is not None:
        gone = b[row] * (2.0 ** 52 / btotal[row])[:, None]
    else:
        gone = (torch.arange(V, device=x.device) == draft[row][:, None]) * 2.0 ** 52
    left = torch.round((a * (2.0 ** 52 / total)[:, None] - gone).clamp(min=0))
    a = torch.where((last[row] | (left.sum(1) == 0))[:, None], a, left)
    cum = torch.cumsum(a.long(), 1)
    token = torch.argmax((cum.double() > (v.double() * cum[:, -1].double())[:, None]).to(torch.uint8), 1)
    at = t - cu[req]
    out = torch.where(at < taken[req], draft, torch.where(at == taken[req], token[req], torch.full_like(tok, -1)))
    return taken.to(torch.int32), out


# ------------------------------------------------------------------------ one pass
def run(s):
    c = s["c"]
    kind = c["kind"]
    if kind == "qk":
        if own:
            from dsalt_amd import ops
            where = dict(pos=s["pos"]) if c["way"] == "pos" else dict(cu_seqlens=s["cu"], max_seqlen=s["max_len"])
            a = (s["q"], s["k"], s["qw"], s["kw"], s["cos"], s["sin"])
            if c["way"] == "bwd":
                return list(ops.qk_norm_rope_backward(s["dq"], s["dk"], *a, eps=_EPS, **where))
            return list(ops.qk_norm_rope(*a, eps=_EPS, **where))
        pos = _plain_positions(s)
        cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
        dt = s["q"].dtype
        if c["way"] == "bwd":
            dq, dqw = _plain_qk_grad(s["dq"], s["q"], s["qw"], cos, sin)
            dk, dkw = _plain_qk_grad(s["dk"], s["k"], s["kw"], cos, sin)
            return [dq.to(dt), dk.to(dt), dqw, dkw]
        return [_plain_qk(s["q"], s["qw"], cos, sin).to(dt), _plain_qk(s["k"], s["kw"], cos, sin).to(dt)]
    if kind == "store":
        dt = s["k"].dtype
        if own:
            from dsalt_amd import ops
            cache = ops.Cache4(*s["cache"])
            ops.cache_write_(s["k"], s["v"], cache, s["pieces"])
            return list(ops.cache_read(cache, s["table"], s["cu"], start=s["start"], n_rows=s["rows"], dtype=dt))
        at = _plain_slots(s["pieces"], s["rows"], c["bt"])
        for i, x in enumerate((s["k"], s["v"])):
            _plain_write(x, *s["cache"], at, i)
        t = torch.arange(s["rows"], device=_DEV)
        cu = s["cu"].long()
        r = torch.searchsorted(cu, t, right=True) - 1
        pos = s["start"].long()[r] + t - cu[r]
        heads = torch.arange(c["kv_heads"], device=_DEV)
        return [_taken(s["cache"], s["table"], r[:, None], heads, pos[:, None], i).to(dt) for i in range(2)]
    if kind == "attend":
        a = (s["table"], s["req"], s["pos"], s["w"], s["lmk"])
        if own:
            from dsalt_amd import ops
            return list(ops.cache_attention(s["q"], ops.Cache4(*s["cache"]), *a, w_max=c["w_max"], rows_per_req=c["per"]))
        return list(_plain_attend(s["q"], s["cache"], *a, c["w_max"]))
    a = (s["x"], s["tok"], s["cu"], s["u"], s["v"])
    if own:
        from dsalt_amd import ops
        return list(ops.verify_rows(*a, draft_logits=s["y"], temperature=s["temp"]))
    return list(_plain_verify(*a, s["y"], s["temp"]))


# ------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = dict(case)
    kind = c["kind"]
    es = 4 if c["dtype"] == "f32" else 2
    if kind == "qk":
        n = 1.0 * c["rows"] * (c["heads"] + c["kv_heads"]) * c["head_dim"]
        # the tables' rows of each position, once (both halves alike, but given apart)
        tab = 8.0 * c["head_dim"] * (c["rows"] if c["way"] == "pos" else min(c["rows"], 2 * c["rows"] / (c["seqs"] + 1)))
        return {"bytes": n * es * (3 if c["way"] == "bwd" else 2) + tab, "flops": n * (18 if c["way"] == "bwd" else 9)}
    if kind == "store":
        n = 2.0 * c["rows"] * c["kv_heads"] * c["head_dim"]
        return {"bytes": 2 * n * (es + 17 / 32), "flops": 6 * n}
    if kind == "attend":
        R, n, H, G, D, K = c["reqs"], c["per"], c["heads"], c["kv_heads"], c["head_dim"], c["k_lmk"]
        mean = c["max_len"] if c["lens"] == "even" else (c["max_len"] + n) / 2
        win = min(c["w_max"] / 2 if c["w_max"] <= 512 else c["w_max"], mean)
        lm = min(K, max(0.0, mean - win))
        tokens = min(mean, win + n - 1 + lm * (H // G))  # of a key/value head: the window, and its query heads' landmarks
        return {"bytes": R * (G * D * (17 / 16) * tokens + 2.0 * n * H * D * es + 4 * H * K + 4.0 * n * H),
                "flops": 4.0 * R * n * H * D * (win + lm)}
    rows = c["reqs"] * (1 + (c["most"] if c["lens"] == "even" else c["most"] / 2))
    drafts = rows - c["reqs"] if c["draft"] == "logits" else 0
    return {"bytes": (rows + drafts) * c["vocab"] * es + 32.0 * rows, "flops": 4.0 * (rows + drafts) * c["vocab"]}


# ------------------------------------------------------------------------ the definitions in 64 bits
def _exact_qk(s):
    way = s["c"]["way"]
    if way == "pos":
        pos = s["pos"].long()
    else:
        pos = torch.cat([torch.arange(int(n), device=_DEV) for n in s["cu"].diff()])
    out, grads = [], []
    for x, w, d in ((s["q"], s["qw"], s.get("dq")), (s["k"], s["kw"], s.get("dk"))):
        x, w = x.double(), w.double()
        T, heads, D = x.shape
        c = s["cos"].double()[pos].view(T, 1, 2, D // 2)
        sn = s["sin"].double()[pos].view(T, 1, 2, D // 2)
        size = (x.pow(2).sum(-1, keepdim=True) / D + _EPS).sqrt()
        if way != "bwd":
            n = (x / size * w).view(T, heads, 2, D // 2)
            out.append((n * c + torch.stack([-n[:, :, 1], n[:, :, 0]], 2) * sn).view(T, heads, D))
            continue
        d = d.double().view(T, heads, 2, D // 2)
        ds = d * sn
        dn = (d * c + torch.stack([ds[:, :, 1], -ds[:, :, 0]], 2)).view(T, heads, D)
        grads.append((dn * x / size).sum(0).sum(0))
        g = dn * w
        out.append(g / size - x * (g * x).sum(-1, keepdim=True) / (D * size.pow(3)))
    return out + grads


def _values(code, exp):
    """float64 values of codes and exponents, by the format's arithmetic: 2^e (1 + m/2), 2^0 (m/2) for e = 0."""
    c = torch.stack([code & 15, code >> 4], -1).flatten(-2).long()
    e, m = (c >> 1) & 3, c & 1
    x = torch.where(e > 0, torch.exp2((e - 1).double()) * (1 + 0.5 * m), 0.5 * m.double()) * (1 - 2 * (c >> 3)).double()
    sc = torch.where(exp == 255, torch.full(exp.shape, math.nan, dtype=torch.float64, device=exp.device), torch.exp2(exp.double() - 127))
    return x * sc.repeat_interleave(32, -1)


def _exact_store(s):
    out = []
    grid = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    for x in (s["k"], s["v"]):
        x = x.detach().cpu().double().numpy()
        b = x.reshape(*x.shape[:-1], -1, 32)
        top = np.abs(b).max(-1, keepdims=True)
        sc = np.exp2(np.clip(np.ceil(np.log2(np.maximum(top, 1e-300) / 7)), -126, 125))
        y = np.minimum(np.abs(b) / sc, 6.0)
        up = np.searchsorted(grid, y)  # the first grid value not below y
        lo = np.maximum(up - 1, 0)
        mid = (grid[up] + grid[lo]) / 2
        code = np.where(y > mid, up, np.where(y < mid, lo, np.where(up % 2 == 0, up, lo)))
        out.append(torch.from_numpy((np.sign(b) * grid[code] * sc).reshape(x.shape)))
    return out


def _exact_attend(s):
    q = s["q"].double() / math.sqrt(s["q"].shape[-1])
    kv, scale = s["cache"]
    T, H, D = q.shape
    G, bt = kv.shape[1], kv.shape[2]
    out, lse = torch.zeros(T, H, D, dtype=torch.float64, device=_DEV), torch.zeros(T, H, dtype=torch.float64, device=_DEV)
    pos, w, req = s["pos"].tolist(), s["w"].tolist(), s["req"].tolist()
    g = torch.arange(G, device=_DEV)[:, None]
    hg = (torch.arange(H, device=_DEV) // (H // G))[:, None]
    for t in range(T):
        low = max(0, pos[t] - max(w[t], 1) + 1)
        tab = s["table"][req[t]].long()

        def values(which, heads, p):  # [heads, n, D]
            page = tab[p // bt]
            return _values(kv[page, heads, p % bt, which], scale[page, heads, p % bt, which])
        j = torch.arange(low, pos[t] + 1, device=_DEV)[None]
        sw = torch.bmm(q[t].view(G, H // G, D), values(0, g, j).transpose(1, 2).contiguous()).view(H, -1)
        p = s["lmk"][:, req[t], 0].long()
        ok, pc = (p >= 0) & (p < low), p.clamp(min=0)
        sl = (values(0, hg, pc) * q[t][:, None]).sum(-1).masked_fill(~ok, float("-inf"))
        a, n = torch.softmax(torch.cat([sw, sl], 1), 1), sw.shape[1]
        out[t] = torch.bmm(a[:, :n].reshape(G, H // G, n), values(1, g, j)).view(H, D) + (a[:, n:, None] * values(1, hg, pc)).sum(1)
        lse[t] = torch.logsumexp(torch.cat([sw, sl], 1), 1)
    return [out, lse]


def _exact_verify(s):
    cu, tok = s["cu"].tolist(), s["tok"].tolist()
    u, v, temp = (s[n].double().tolist() for n in ("u", "v", "temp"))
    taken, out = [], [-1] * cu[-1]

    def weights(row, t):
        x = row.double().cpu().numpy()
        if t > 0:
            return np.rint(np.exp((x - x.max()) / t) * 2.0 ** 42)
        w = np.zeros(x.shape)
        w[int(np.argmax(x))] = 2.0 ** 42
        return w
    for r in range(len(cu) - 1):
        for t in range(cu[r], cu[r + 1]):
            a = weights(s["x"][t], temp[r])
            if t + 1 == cu[r + 1]:
                break
            x = tok[t + 1]
            if s["y"] is None:
                b = np.zeros(a.shape)
                b[x] = 1.0
            else:
                b = weights(s["y"][t], temp[r])
            if u[t] * (b[x] / b.sum()) < a[x] / a.sum():
                out[t] = x
                continue
            a = np.rint(np.maximum(a * (2.0 ** 52 / a.sum()) - b * (2.0 ** 52 / b.sum()), 0.0))
            break
        cum = np.cumsum(a.astype(np.int64))
        out[t] = int(np.flatnonzero(cum > v[r] * float(cum[-1]))[0])
        taken.append(t - cu[r])
    return [torch.tensor(taken, dtype=torch.int32), torch.tensor(out)]


def exact(case, seed):
    s = prepare(case, seed)
    return {"qk": _exact_qk, "store": _exact_store, "attend": _exact_attend, "verify": _exact_verify}[case["kind"]](s)
