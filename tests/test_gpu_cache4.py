"""The paged 4-bit cache on the GPU against the float64 oracle: write, read-back and attention, pages kept for tokens taken
back, and a run of speculative steps.

Tolerances, from the arithmetic.  Codes and scales are exact.  Attention: keys and values are exact in bfloat16, so that the
errors are those of the sums and weights.  A weight's relative error is at most twice its logit's absolute error; a logit is a
float32 dot product of D terms in any order and tree, (D + 8) 2^-24 of the largest sum |scale q k| of its row (``reach``); sums
over n keys add n 2^-24, weights of 16-bit types are granted 2^-16 (they are handed to the matrix products whole: see the test of
weights in 32 bits, which grants none); the output is rounded once to its type, half a step being 2^-8 (bfloat16), 2^-11 (float16) or 2^-24.  Errors of weights act on sum p |v|
(``mass``)."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from dsalt_amd import ops
from oracle import decode as OD
from oracle import decode4 as O4

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def f64(t):
    return t.detach().cpu().double().numpy()


# ------------------------------------------------------------------------ write and read
def _host_pages(cache):
    n, g, bt, _, half = cache.kv.shape
    c = cache.kv.cpu().numpy().astype(np.int64)
    code = np.stack([c & 15, c >> 4], -1).reshape(n, g, bt, 2, 2 * half)
    e = cache.scale.cpu().numpy().astype(np.float64)
    s = np.where(e == 255, np.nan, np.exp2(e - 127)).repeat(32, -1)
    x = np.where(code & 8, -1.0, 1.0) * O4.GRID[code & 7] * s
    p = O4.Pages4(n, g, bt, 2 * half)
    p.k, p.v = x[:, :, :, 0], x[:, :, :, 1]
    return p


def _same_pages(cache, pages):
    got = _host_pages(cache)
    assert np.array_equal(got.k, pages.k, equal_nan=True) and np.array_equal(got.v, pages.v, equal_nan=True)


def _random_cache(n_blocks, G, bt, D, seed):
    g = torch.Generator().manual_seed(seed)
    c = ops.new_cache(n_blocks, G, D, block_tokens=bt, device=DEV, bits=4)
    c.kv.copy_(torch.randint(0, 256, c.kv.shape, generator=g, dtype=torch.uint8))
    c.scale.copy_(torch.randint(123, 128, c.scale.shape, generator=g, dtype=torch.uint8))
    return c


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("bt,D,G", [(16, 64, 3), (32, 128, 1), (64, 64, 1), (128, 128, 2)])
def test_write_follows_the_oracle(dt, bt, D, G):
    """Whole prompts, single tokens and runs that end and begin inside pages; what the pages held before stays."""
    R, M = 5, 6
    cache = _random_cache(R * M + 4, G, bt, D, bt + D)
    pages = _host_pages(cache)
    table = torch.full((R, M), -1, dtype=torch.int32, device=DEV)
    ring = torch.randperm(R * M + 4).to(torch.int32).to(DEV)
    span = torch.tensor([0, R * M + 4], device=DEV)
    seq = torch.zeros(R, dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(3)
    for new, size in (([bt, 1, 2 * bt + 5, 0, 2 * bt - 1], 1.0), ([1] * R, 30.0), ([1, 2, 1, 7, 1], 1e-3), ([1] * R, 1000.0)):
        T = sum(new) + 2  # padded rows
        rows = ops.cache_rows_(seq, _i32(new), table, ring, span, T, block_tokens=bt)
        x = (torch.randn(T, 3 * G * D, generator=g) * size * torch.exp2(torch.randn(T, 1, generator=g) * 3)).to(dt).to(DEV)
        k, v = x[:, :G * D].view(T, G, D), x[:, 2 * G * D:].view(T, G, D)
        assert ops.cache_write_(k, v, cache, rows.pieces) is cache
        pages.write(f64(k), f64(v), rows.pieces.cpu().numpy())
        _same_pages(cache, pages)
        seq, span = rows.seq_len, rows.span
    n = seq.tolist()
    cu = np.concatenate([[0], np.cumsum(n)])
    for od in (torch.float32, dt):
        got = ops.cache_read(cache, table, _i32(cu), n_rows=int(cu[-1]) + 3, dtype=od)
        for a, b in zip(got, pages.read(table.cpu().numpy(), cu, [0] * R, int(cu[-1]) + 3)):
            assert torch.equal(a.cpu(), torch.from_numpy(b).to(od))


def test_write_extremes():
    """Zeros, subnormals, the types' largest, infinities and NaN, magnitudes on both sides of a scale, every tie."""
    x = torch.zeros(12, 1, 64)
    x[1, 0, :5] = torch.tensor([1e-45, -1e-40, 2.0 ** -126, -2.0 ** -120, 0.0])
    x[2, 0, :4] = torch.tensor([3.4e38, -3.3e38, 1.0, 1e-38])
    x[3, 0, :5] = torch.tensor([float("inf"), 1.0, 2.0, 3.0, -0.0])   # the second half of the head stays finite
    x[3, 0, 40] = 5.0
    x[4, 0, 33], x[5, 0, 7] = float("nan"), float("-inf")
    x[6, 0, :32] = torch.tensor([6.0] + [s * t for t in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.2500001, 0.7499999, 1.2500001,
                                                           1.7499999, 2.5000002, 3.4999998, 5.0000005) for s in (1, -1)] + [0.0, -0.0, 6.9])
    x[7, 0, 0], x[7, 0, 32] = 7.0, 7.0000005
    x[8, 0, 0], x[8, 0, 32] = 3.5, 3.4999998
    x[9, 0] = 2.0 ** -126
    x[10, 0] = torch.arange(64) - 32.0
    x[11] = float("nan")
    for dt in (torch.float32, torch.bfloat16):
        cache = _random_cache(2, 1, 16, 64, 1)
        pages = _host_pages(cache)
        y = x.to(dt).to(DEV)
        ops.cache_write_(y, y, cache, _i32([[0, 12, 1, 2]]))
        pages.write(f64(y), f64(y), [[0, 12, 1, 2]])
        _same_pages(cache, pages)
        k, v = ops.cache_read(cache, _i32([[1]]), _i32([0, 12]), start=_i32([2]), n_rows=12, dtype=torch.float32)
        assert np.array_equal(f64(k), pages.k[1, 0, 2:14][:, None], equal_nan=True) and torch.equal(k.isnan(), v.isnan())


def test_write_skips_pieces_that_lie_outside():
    cache = _random_cache(4, 2, 16, 64, 9)
    before = [t.clone() for t in cache]
    x = torch.randn(8, 2, 64, device=DEV)
    bad = [[0, 1, 4, 0], [0, 1, -1, 0], [7, 2, 0, 0], [-1, 1, 0, 0], [0, 3, 0, 14], [0, 1, 0, -1], [0, -4, 0, 0], [0, 0, 2, 0],
           [2 ** 31 - 1, 2, 0, 0], [0, 2 ** 31 - 1, 0, 1]]
    ops.cache_write_(x, x, cache, _i32(bad))
    assert all(torch.equal(a, b) for a, b in zip(cache, before))


def test_write_of_rows_in_other_layouts():
    """Heads first, a token stride of one element too many, an offset off 16 bytes: the same codes; a page in two pieces."""
    x = torch.randn(20, 2, 64, device=DEV).to(torch.bfloat16)
    pieces = _i32([[0, 9, 0, 0], [9, 7, 0, 9], [16, 4, 1, 3]])
    ref = ops.cache_write_(x, x, ops.new_cache(2, 2, 64, block_tokens=16, bits=4), pieces)
    flat = torch.zeros(20 * 129 + 1, device=DEV, dtype=torch.bfloat16)
    odd = flat[1:1 + 20 * 128].view(20, 2, 64)
    odd.copy_(x)
    gap = torch.zeros(20, 129, device=DEV, dtype=torch.bfloat16)
    gap[:, :128] = x.view(20, 128)
    for y in (x.transpose(0, 1).contiguous().transpose(0, 1), odd, gap[:, :128].unflatten(1, (2, 64)),
              x.transpose(1, 2).contiguous().transpose(1, 2)):
        got = ops.cache_write_(y, y, ops.new_cache(2, 2, 64, block_tokens=16, bits=4), pieces)
        assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_read_outside_is_zero():
    cache = _random_cache(4, 1, 16, 64, 2)
    table = _i32([[0, 9, -1], [3, 2, 1]])
    cu, start = [2, 30, 40], [4, 45]  # the first rows belong to no request
    k, v = ops.cache_read(cache, table, _i32(cu), start=_i32(start), n_rows=50, dtype=torch.float32)
    wk, wv = _host_pages(cache).read(table.cpu().numpy(), cu, start, 50)
    assert np.array_equal(f64(k), wk) and np.array_equal(f64(v), wv) and not wk[:2].any() and not wk[14:30].any()


# ------------------------------------------------------------------------ attention
def _attend_case(R, H, G, D, bt, K, dt, seed, max_len, w_max, per=1, lens=None):
    """`per` rows of each request side by side, at its last positions."""
    g = torch.Generator().manual_seed(seed)
    r = np.random.RandomState(seed)
    lens = lens or [int(x) for x in r.randint(1, max_len + 1, R)]
    held = [-(-n // bt) for n in lens]
    M, N = max(held) + 1, sum(held) + 2
    cache = _random_cache(N, G, bt, D, seed)
    ids, at = r.permutation(N), 0
    table = np.full((R, M), -1)
    for i, h in enumerate(held):
        table[i, :h] = ids[at:at + h]
        at += h
    req = [i for i in range(R) for _ in range(per)]
    pos = [max(0, lens[i] - per + j) for i in range(R) for j in range(per)]
    T = len(req)
    q = torch.randn(T, H, D, generator=g).to(dt)
    w = [int(x) for x in r.randint(0, w_max + 1, T)]
    lmk = np.full((H, R, 1, K), -1)
    for i in range(R):
        for h in range(H):
            p = r.randint(0, lens[i], K)  # any order, repeats, inside the window too
            lmk[h, i, 0] = np.where(r.rand(K) < 0.2, -1 - r.randint(0, 9, K), p)
    return q, cache, table, req, pos, w, lmk


def _check_attend(q, cache, table, req, pos, w, lmk, bias=None, scale=None, w_max=None, pages=None, dev_q=None, per=1):
    T, H, D = q.shape
    pages = pages or _host_pages(cache)
    args = (_i32(table), _i32(req), _i32(pos), _i32(w), _i32(lmk).view(*np.shape(lmk)))
    b = torch.from_numpy(bias).float().to(DEV) if bias is not None else None
    out, lse = ops.cache_attention(q.to(DEV) if dev_q is None else dev_q, cache, *args, b, scale=scale, w_max=w_max, rows_per_req=per)
    ref, rl, mass, reach, keys = OD.attention(f64(q), pages, table, req, pos, w, lmk, bias, scale or 1 / math.sqrt(D))
    assert out.dtype == q.dtype and out.shape == q.shape and lse.shape == (T, H)
    out, lse = f64(out), f64(lse)
    nan = np.isnan(ref)
    assert np.array_equal(np.isnan(out), nan)
    logit = (D + 8) * 2.0 ** -24 * reach + 2.0 ** -23 * (0 if bias is None else 40)
    tol = (2 * logit + (keys + 64) * 2.0 ** -24 + (0 if q.dtype == torch.float32 else 2.0 ** -16))[..., None] * mass
    tol = tol + U[q.dtype] * np.abs(ref) + (2.0 ** -25 if q.dtype == torch.float16 else 0)
    assert (np.abs(out - ref) <= tol)[~nan].all(), float((np.abs(out - ref) / np.maximum(tol, 1e-300))[~nan].max())
    empty = np.isneginf(rl)
    assert np.array_equal(np.isneginf(lse), empty) and not out[empty].any()
    ok = np.isfinite(rl)
    ltol = logit + (keys + 64) * 2.0 ** -24 + 2.0 ** -23 * np.abs(np.where(ok, rl, 0))
    assert (np.abs(lse[ok] - rl[ok]) <= ltol[ok]).all()
    return out, lse


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("R,H,G,D,bt,K,max_len,w_max,per", [
    (1, 1, 1, 64, 16, 0, 1, 1, 1), (1, 16, 2, 128, 64, 33, 700, 512, 1), (7, 4, 4, 64, 16, 5, 90, 40, 3), (3, 8, 1, 128, 32, 16, 300, 128, 2),
    (4, 32, 1, 64, 128, 9, 400, 70, 1), (2, 34, 2, 64, 16, 3, 200, 200, 2), (5, 6, 2, 128, 128, 64, 257, 1, 4), (2, 2, 1, 64, 32, 130, 1500, 1500, 9),
    (40, 3, 3, 128, 16, 7, 60, 33, 1), (3, 2, 2, 64, 64, 70, 500, 300, 21), (9, 4, 1, 128, 64, 20, 250, 64, 5)])
def test_attention_follows_the_oracle(dt, R, H, G, D, bt, K, max_len, w_max, per):
    c = _attend_case(R, H, G, D, bt, K, dt, R * 7 + H, max_len, w_max, per)
    _check_attend(*c, w_max=w_max, per=per)
    _check_attend(*c, per=per + 2)  # runs that hold rows of several requests; the bound on the windows not given
    bias = np.random.RandomState(1).randn(*c[-1].shape)
    bias[..., ::3] = -np.inf
    _check_attend(*c, bias=bias, scale=0.3, w_max=max(1, w_max // 3), per=per)  # and given too small
    _check_attend(*c, bias=bias, per=1 << 40)


@pytest.mark.parametrize("bt", [16, 64, 128])
@pytest.mark.parametrize("G", [1, 4])
def test_attention_at_every_page_place(bt, G):
    """Positions around the ends of pages and of the kernels' runs of keys, windows from one key to all."""
    lens = [1, 2, bt - 1, bt, bt + 1, 31, 32, 33, 63, 64, 65, 2 * bt, 2 * bt + 1, 127, 128, 129, 255, 257]
    for wide in (1, 2, 16, 17, 10 ** 6):
        c = list(_attend_case(len(lens), 4, G, 64, bt, 6, torch.bfloat16, bt + G, 0, 1, per=2, lens=lens))
        c[5] = [wide] * len(c[3])
        _check_attend(*c, w_max=wide, per=2)


@pytest.mark.parametrize("per", [1, 2, 4, 15])
def test_attention_of_rows_in_any_order(per):
    """Rows of a request side by side or not, at positions far apart, with windows of their own."""
    q, cache, table, req, pos, w, lmk = _attend_case(3, 8, 2, 64, 32, 12, torch.bfloat16, 5, 150, 60, per=5, lens=[150, 90, 33])
    pos[1], pos[3], pos[7] = 3, 70, 0
    w[0], w[2] = 1, 200
    order = np.random.RandomState(0).permutation(15)
    _check_attend(q, cache, table, req, pos, w, lmk, w_max=60, per=per)
    _check_attend(q[order], cache, table, [req[i] for i in order], [pos[i] for i in order], [w[i] for i in order], lmk, w_max=60, per=per)


@pytest.mark.parametrize("per", [1, 3])
def test_attention_inert_rows_and_absent_pages(per):
    q, cache, table, req, pos, w, lmk = _attend_case(6, 4, 2, 64, 16, 8, torch.float32, 11, 100, 50, lens=[100, 3, 50, 77, 64, 20], per=per)
    first = [i * per for i in range(6)]
    for i in range(first[0], first[1]):
        req[i] = -1                                # no request
    pos[first[1]], req[first[2]] = -1, 6          # no position, a request past the table
    table[3] = -1                                 # no page at all
    table[4, 1], table[4, 3] = -3, len(cache.kv)  # pages below and past the cache
    pos[first[5]] = 10 ** 6                       # past the table: only landmarks are there
    w[first[5]] = 5
    out, lse = _check_attend(q, cache, table, req, pos, w, lmk, w_max=50, per=per)
    assert np.isneginf(lse[[first[0], first[1], first[2], first[3]]]).all() and np.isfinite(lse[[first[4], first[5]]]).all()


def _widened(table, bt, tokens):
    """The table with empty columns up to `tokens` tokens a request: without a bound on them the windows may be that long."""
    return np.pad(table, ((0, 0), (0, max(0, tokens // bt - table.shape[1]))), constant_values=-1)


# what the size rules choose between, and a shape each (R, H, G, D, bt, K, lens or the longest, largest window, bound given, rows of a request)
RULES = {
    "one head a block": (2, 4, 4, 128, 64, 40, 900, 700, 700, 1),
    "heads of a group apart": (1, 16, 2, 128, 64, 40, 900, 700, 700, 1),
    "split": (1, 2, 2, 128, 64, 70, [5001], 4900, 4900, 1),
    "split, heads of a group": (1, 8, 2, 64, 16, 9, [4500], 4500, 4500, 1),
    "split, most splits empty": (3, 8, 2, 64, 16, 130, [300, 33, 1], 290, 1 << 15, 1),
    "split, rows of a request": (2, 8, 2, 128, 64, 200, [2500, 40], 2400, 1 << 13, 3),
    "many requests, heads of a group apart": (110, 8, 2, 64, 64, 17, 90, 60, 300, 1),
    "many requests": (280, 8, 2, 128, 32, 33, 90, 60, 300, 1),
    "many requests, rows of a request": (150, 4, 2, 64, 32, 33, 90, 60, 300, 4),
    "five rows, heads in threes": (130, 8, 1, 64, 16, 9, 60, 40, 150, 5),
    "five rows, heads in pairs": (70, 8, 1, 128, 16, 9, 60, 40, 150, 5),
    "groups of 17 heads": (140, 34, 2, 64, 16, 5, 70, 40, 150, 1),
    "groups of 16 heads of 128": (80, 32, 2, 128, 64, 6, 150, 100, 256, 2),
}


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rule", RULES)
def test_attention_on_each_side_of_the_size_rules(rule, dt):
    R, H, G, D, bt, K, lens, w, bound, per = RULES[rule]
    given = lens if isinstance(lens, list) else None
    c = list(_attend_case(R, H, G, D, bt, K, dt, R + H, max(given) if given else lens, w, per, given))
    if given:
        c[5] = [x for x in [w, w // 2, 5][:R] for _ in range(per)]
    c[2] = _widened(c[2], bt, bound)
    _check_attend(*c, w_max=bound, per=per)
    bias = np.random.RandomState(3).randn(*c[-1].shape)
    _check_attend(*c, bias=bias, w_max=bound, per=per)


@pytest.mark.parametrize("per", [1, 2])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("G", [2, 8])
def test_attention_reads_nothing_masked(dt, G, per):
    """NaN in every token that no row of a head's group attends: results as without them.  Then NaN values in one token of the
    window of the last row alone, and in one landmark of one head: they reach the rows and heads that attend them, no other."""
    H, D, bt = 8, 64, 16
    q, cache, table, req, pos, w, lmk = _attend_case(3, H, G, D, bt, 9, dt, 21, 200, 30, lens=[200, 45, 3], per=per)
    w = [x for x in (30, 7, 3) for _ in range(per)]
    clean = _host_pages(cache)
    seen = np.zeros((len(cache.kv), G, bt), dtype=bool)
    for t in range(len(req)):
        i, low = req[t], max(pos[t] - w[t] + 1, 0)
        for h in range(H):
            for p in list(range(low, pos[t] + 1)) + [int(x) for x in lmk[h, i, 0] if 0 <= x < low]:
                seen[table[i, p // bt], h // (H // G), p % bt] = True
    cache.scale[torch.from_numpy(~seen).to(DEV)] = 255
    a, _ = _check_attend(q, cache, table, req, pos, w, lmk, pages=clean, w_max=30, per=per)
    assert np.isfinite(a).all()
    # the newest token of request 0: the earlier rows of the request do not see it
    last = pos[per - 1]
    cache.scale[table[0, last // bt], :, last % bt, 1, 1] = 255
    bad = _host_pages(cache)
    b, _ = _check_attend(q, cache, table, req, pos, w, lmk, pages=bad, w_max=30, per=per)
    assert np.isnan(b[per - 1, :, 32:]).all() and np.isfinite(b[per - 1, :, :32]).all() and np.array_equal(b[:per - 1], a[:per - 1])
    assert np.array_equal(b[per:], a[per:])
    # one landmark of head 3 of request 0
    only = int(next(p for p in lmk[3, 0, 0] if 0 <= p < pos[0] - 29))
    cache.scale[table[0, only // bt], 3 // (H // G), only % bt, 1, 0] = 255
    c, _ = _check_attend(q, cache, table, req, pos, w, lmk, pages=_host_pages(cache), w_max=30, per=per)
    for h in range(H):
        user = h // (H // G) == 3 // (H // G) and only in lmk[h, 0, 0]
        assert np.isnan(c[:per, h, :32]).all() if user else np.array_equal(c[:per, h], b[:per, h], equal_nan=True)


def test_attention_landmark_that_only_some_rows_see():
    """A landmark with NaN that lies inside the window of one row and before that of another."""
    q, cache, table, req, pos, w, lmk = _attend_case(1, 2, 1, 64, 16, 4, torch.bfloat16, 3, 0, 1, lens=[120], per=3)
    w = [50, 5, 50]
    lmk[:] = np.array([100, 3, -1, 9])
    a, _ = _check_attend(q, cache, table, req, pos, w, lmk, w_max=64, per=3)
    lmk[:] = np.array([100, 3, 110, 9])
    cache.scale[table[0, 6], 0, 4, 1, 0] = 255  # token 100
    b, _ = _check_attend(q, cache, table, req, pos, w, lmk, w_max=64, per=3)
    assert np.isnan(b[:, :, :32]).all() and np.isfinite(b[:, :, 32:]).all()  # row 1 as its landmark, the others in their window
    w = [5, 5, 5]
    lmk[:] = np.array([70, 116, -1, 9])
    cache.scale[table[0, 6], 0, 4, 1, 0] = 127
    cache.scale[table[0, 116 // 16], 0, 116 % 16, 1, 0] = 255  # in the windows of rows 0 to 2: positions 113..119
    c, _ = _check_attend(q, cache, table, req, pos, w, lmk, w_max=64, per=3)
    assert np.isnan(c[:, :, :32]).all()
    w = [2, 1, 1]
    d, _ = _check_attend(q, cache, table, req, pos, w, lmk, w_max=64, per=3)  # row 0 sees it in its window, 1 and 2 as a landmark
    assert np.isnan(d[:, :, :32]).all()


def test_attention_empty_by_bias():
    """Landmarks of weight -inf and a window whose page is absent: nothing is attended."""
    q, cache, table, req, pos, w, lmk = _attend_case(2, 2, 1, 64, 16, 4, torch.float32, 2, 60, 4, lens=[60, 60])
    w, table[0, 3] = [4, 4], -1
    bias = np.zeros(lmk.shape)
    bias[:, 0] = -np.inf
    out, lse = _check_attend(q, cache, table, req, pos, w, lmk, bias=bias)
    assert np.isneginf(lse[0]).all() and np.isfinite(lse[1]).all()


@pytest.mark.parametrize("lowest", [-1e4, -3.4e38])
def test_attention_masks_of_the_lowest_value(lowest):
    """Landmarks masked by a type's lowest value count where nothing else does, and weigh nothing beside others."""
    q, cache, table, req, pos, w, lmk = _attend_case(2, 2, 1, 64, 16, 4, torch.float32, 2, 60, 4, lens=[60, 60])
    w, table[0, 3] = [4, 4], -1
    lmk[:] = np.array([1, 9, 20, 33])
    bias = np.full(lmk.shape, lowest)
    args = [_i32(x) for x in (table, req, pos, w, lmk)]
    out, lse = ops.cache_attention(q.to(DEV), cache, *args, torch.from_numpy(bias).float().to(DEV))
    none = ops.cache_attention(q.to(DEV), cache, *args[:4], torch.full_like(args[4], -1))
    assert torch.equal(out[1], none[0][1]) and torch.isfinite(out).all() and torch.isfinite(lse[1]).all() and not torch.isnan(lse).any()
    free = ops.cache_attention(q.to(DEV), cache, *args)[0]
    if lowest == -1e4:  # the shift costs its rounding, 2^-11 of a logit
        assert torch.allclose(out[0], free[0], atol=2e-2)


def test_attention_strides_and_layouts():
    c = _attend_case(5, 4, 2, 64, 32, 6, torch.bfloat16, 8, 120, 30)
    x = torch.randn(5, 3, 4, 64).to(torch.bfloat16)
    x[:, 1] = c[0]
    for dq in (x.to(DEV)[:, 1], c[0].to(DEV).transpose(0, 1).contiguous().transpose(0, 1),
               c[0].to(DEV).transpose(1, 2).contiguous().transpose(1, 2)):
        _check_attend(*c, dev_q=dq)
    q, cache, table, req, pos, w, lmk = c
    a = ops.cache_attention(q.to(DEV), cache, _i32(table), _i32(req), _i32(pos), _i32(w), _i32(lmk))
    b = ops.cache_attention(q.to(DEV), cache, _i32(np.pad(table, ((0, 0), (0, 4)), constant_values=0))[:, :table.shape[1]],
                            _i32(req).long(), _i32(pos).long(), _i32(w).float(), _i32(lmk).long())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("w", [300, 40])
def test_attention_long_caches(w):
    """Pages whose bytes lie past 2^32, and a position of some hundred thousand tokens."""
    G, bt, D = 8, 128, 128
    n = (1 << 32) // (G * bt * D) + 40
    cache = ops.new_cache(n, G, D, block_tokens=bt, device=DEV, bits=4)
    use = [n - 1, n - 3, 5, n - 2]
    small = _random_cache(4, G, bt, D, 6)
    for i, b in enumerate(use):
        cache.kv[b], cache.scale[b] = small.kv[i], small.scale[i]
    M = 3000
    table, ref_table = np.full((1, M), -1), np.full((1, M), -1)
    at = [0, M - 3, M - 2, M - 1]
    table[0, at], ref_table[0, at] = use, [0, 1, 2, 3]
    lmk = np.full((16, 1, 1, 5), -1)
    lmk[:, 0, 0, :3] = [5, 127, (M - 3) * bt + 1]
    q = torch.randn(1, 16, D, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    p = _host_pages(small)
    out, lse = ops.cache_attention(q.to(DEV), cache, _i32(table), _i32([0]), _i32([M * bt - 2]), _i32([w]), _i32(lmk), w_max=w)
    ref, rl, mass, reach, keys = OD.attention(f64(q), p, ref_table, [0], [M * bt - 2], [w], lmk, None, 1 / math.sqrt(D))
    tol = (2 * (D + 8) * 2.0 ** -24 * reach + 2.0 ** -15)[..., None] * mass + U[torch.bfloat16] * np.abs(ref)
    assert (np.abs(f64(out) - ref) <= tol).all()
    x = torch.randn(1, G, D, device=DEV)
    ops.cache_write_(x, x, cache, _i32([[0, 1, n - 2, 127]]))
    p.write(f64(x), f64(x), [[0, 1, 3, 127]])
    k, v = ops.cache_read(cache, _i32(table), _i32([0, 4]), start=_i32([M * bt - 4]), n_rows=4, dtype=torch.float32)
    wk, wv = p.read(ref_table, [0, 4], [M * bt - 4], 4)
    assert np.array_equal(f64(k), wk) and np.array_equal(f64(v), wv)


@pytest.mark.parametrize("per", [1, 2])
def test_attention_of_long_windows(per):
    """Windows of 40000 keys split over the chip against float64 torch on the same values."""
    n, H, G, D, bt = 40001, 8, 2, 128, 64
    cache = _random_cache(-(-n // bt), G, bt, D, 1)
    table = torch.arange(-(-n // bt), dtype=torch.int32).flip(0)[None]
    q = torch.randn(per, H, D).to(torch.bfloat16)
    lmk = torch.full((H, 1, 1, 0), -1, dtype=torch.int32)
    k, v = (x.double().cpu() for x in ops.cache_read(cache, table.to(DEV), _i32([0, n]), n_rows=n, dtype=torch.float32))
    for w in (n, n - 1, 20000):
        out, lse = ops.cache_attention(q.to(DEV), cache, table.to(DEV), _i32([0] * per), _i32([n - 1] * per), _i32([w] * per), lmk.to(DEV),
                                       w_max=w, rows_per_req=per)
        for t in range(per):
            s = torch.einsum("hd,nhd->hn", q[t].double(), k[n - w:].repeat_interleave(H // G, 1)) / math.sqrt(D)
            p = torch.softmax(s, 1)
            ref = torch.einsum("hn,nhd->hd", p, v[n - w:].repeat_interleave(H // G, 1))
            mass = torch.einsum("hn,nhd->hd", p, v[n - w:].abs().repeat_interleave(H // G, 1))
            reach = torch.einsum("hd,nhd->hn", q[t].double().abs(), k.abs().repeat_interleave(H // G, 1)).amax(1) / math.sqrt(D)
            # sums over lanes, waves and splits: chains of at most n / 256 keys and joins of 64 and 1024 parts
            tol = (2 * (D + 8) * 2.0 ** -24 * reach + 2000 * 2.0 ** -24 + 2.0 ** -16)[:, None] * mass + 2.0 ** -8 * ref.abs()
            assert ((out[t].cpu().double() - ref).abs() <= tol).all()
            ltol = (D + 8) * 2.0 ** -24 * reach + 2000 * 2.0 ** -24 + 2.0 ** -23 * torch.logsumexp(s, 1).abs()
            assert ((lse[t].cpu().double() - torch.logsumexp(s, 1)).abs() <= ltol).all()


def test_attention_of_more_rows_than_a_launch_holds():
    for per, T in ((1, (1 << 20) + 77), (4, (1 << 21) + 78)):
        q, cache, table, req, pos, w, lmk = _attend_case(16, 16, 16, 64, 16, 2, torch.bfloat16, 1, 40, 5, per=4)
        args = [_i32(x) for x in (req, pos, w)]
        out, lse = ops.cache_attention(q.to(DEV), cache, _i32(table), *args, _i32(lmk), w_max=5, rows_per_req=per)
        turn = torch.arange(T, device=DEV) % 64
        big, bl = ops.cache_attention(q.to(DEV)[turn], cache, _i32(table), *(x[turn] for x in args), _i32(lmk), w_max=5, rows_per_req=per)
        whole = T // 64 * 64
        for x, y in ((big, out), (bl, lse)):
            assert bool((x[:whole].view(-1, *y.shape) == y).all()) and torch.equal(x[whole:], y[:T - whole])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,G", [(2, 2), (8, 2)])
def test_calls_without_rows(D, H, G):
    bt = 64
    cache = _random_cache(4, G, bt, D, 3)
    before = _host_pages(cache)
    none, x = _i32([]), torch.zeros(0, H, D, dtype=torch.bfloat16, device=DEV)
    for M in (2, 4096):
        table, lmk = torch.zeros(3, M, dtype=torch.int32, device=DEV), torch.zeros(H, 3, 1, 8, dtype=torch.int32, device=DEV)
        for w_max in (None, 1, M * bt, 1 << 40):
            for sets in (lmk, lmk[..., :0]):
                out, lse = ops.cache_attention(x, cache, table, none, none, none, sets, w_max=w_max, rows_per_req=5)
                assert out.shape == (0, H, D) and out.dtype == x.dtype and lse.shape == (0, H)
        k, v = ops.cache_read(cache, table, _i32([0, 0, 0, 0]), n_rows=0)
        assert k.shape == v.shape == (0, G, D)
    ops.cache_write_(x[:, :G], x[:, :G], cache, torch.zeros(0, 4, dtype=torch.int32, device=DEV))
    ops.cache_write_(x[:, :G], x[:, :G], cache, _i32([[0, 1, 1, 0]]))
    _same_pages(cache, before)


def test_windows_past_32_bits_attend_all():
    q, cache, table, req, pos, _, lmk = _attend_case(3, 4, 2, 64, 16, 5, torch.bfloat16, 4, 90, 1)
    args = [_i32(x) for x in (table, req, pos)]
    ref = ops.cache_attention(q.to(DEV), cache, *args, _i32([1 << 20] * 3), _i32(lmk))
    got = ops.cache_attention(q.to(DEV), cache, *args, torch.tensor([1 << 31, (1 << 32) + 1, 1 << 40], device=DEV), _i32(lmk))
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


def test_the_8_bit_cache_takes_the_hint():
    """rows_per_req over a Cache8 changes nothing."""
    c8 = ops.new_cache(4, 2, 64, block_tokens=16)
    x = torch.randn(40, 2, 64, device=DEV).to(torch.bfloat16)
    ops.cache_write_(x, x, c8, _i32([[0, 16, 0, 0], [16, 16, 2, 0], [32, 8, 1, 0]]))
    a = (torch.randn(4, 4, 64, device=DEV).to(torch.bfloat16), c8, _i32([[0, 2, 1]]), _i32([0] * 4), _i32([36, 37, 38, 39]), _i32([9] * 4),
         _i32(np.arange(4).reshape(1, 1, 1, 4).repeat(4, 0)))
    for p, q in zip(ops.cache_attention(*a), ops.cache_attention(*a, rows_per_req=4)):
        assert torch.equal(p, q)


# ------------------------------------------------------------------------ pages of tokens taken back
@pytest.mark.parametrize("R", [1, 37, 1025, 4097])
def test_rows_keep_the_pages_they_hold(R):
    """Requests that hold pages for more tokens than they have take none twice, use the ones they hold in their order and give
    all of them back; a `held` of the tokens themselves, or fewer, changes nothing."""
    r = np.random.RandomState(R)
    bt, M = 16, 7
    seq = r.randint(0, bt * (M - 1), R)
    held = np.minimum(seq + np.where(r.rand(R) < 0.5, r.randint(0, 3 * bt, R), -r.randint(0, 99, R)), bt * M)
    new = np.where(r.rand(R) < 0.2, -1, np.where(r.rand(R) < 0.5, 1, r.randint(0, 2 * bt, R)))
    has = -(-np.maximum(seq, held) // bt)
    N = int(has.sum()) + 2 * R
    ids = r.permutation(N)
    table, ring, at = np.full((R, M), -1), np.full(N, -7), 0
    for i, h in enumerate(has):
        table[i, :h] = ids[at:at + h]
        at += h
    ring[:N - at] = ids[at:]
    T = int(np.maximum(new, 0).sum()) + 5
    dt, dr, span = _i32(table), _i32(ring), torch.tensor([0, N - at], device=DEV)
    got = ops.cache_rows_(_i32(seq), _i32(new), dt, dr, span, T, block_tokens=bt, held=_i32(held))
    # the same step of requests whose tokens fill the pages held, moved back
    fits = seq + new <= bt * M
    need = np.where((new >= 0) & fits, np.maximum(-(-(seq + new) // bt) - has, 0), 0)
    ok = (new < 0) | (fits & ((need == 0) | (np.cumsum(need) <= N - at)))
    assert np.array_equal(got.granted.cpu().numpy(), ok) and np.array_equal(got.seq_len.cpu().numpy(), np.where(new < 0, 0, np.where(ok, seq + new, seq)))
    after, ring2 = dt.cpu().numpy(), dr.cpu().numpy()
    slot, pos, req = (getattr(got, n).cpu().numpy() for n in ("slot", "pos", "req"))
    first = np.cumsum(need) - need
    back = []
    for i in range(R):
        assert np.array_equal(after[i, :has[i]], table[i, :has[i]])
        if ok[i] and new[i] >= 0:
            assert np.array_equal(after[i, has[i]:has[i] + need[i]], ring[first[i]:first[i] + need[i]])
        elif new[i] < 0:
            back += table[i, :has[i]].tolist()
    assert ring2[N - at:N - at + len(back)].tolist() == back[:N - (N - at)] and got.span.tolist()[1] == min(N - at + len(back), N + 0)
    live = pos >= 0
    assert np.array_equal(slot[live], after[req[live], pos[live] // bt].astype(np.int64) * bt + pos[live] % bt)
    assert live.sum() == int(np.where(ok & (new > 0), new, 0).sum())
    a = ops.cache_rows_(_i32(seq), _i32(new), _i32(table), _i32(ring), span, T, block_tokens=bt)
    b = ops.cache_rows_(_i32(seq), _i32(new), _i32(table), _i32(ring), span, T, block_tokens=bt, held=_i32(np.minimum(held, seq)))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


# ------------------------------------------------------------------------ a run of speculative steps
class Run:
    """Requests decoded with drafts: one layer, random projections of the token's embedding."""

    def __init__(self, R, H, G, D, bt, V, n, dt, seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.R, self.H, self.G, self.D, self.bt, self.V, self.n, self.dt = R, H, G, D, bt, V, n, dt
        pages = 3 * R
        self.emb = torch.randn(V, (H + 2 * G) * D, generator=g, device=DEV).to(dt)
        self.head = (torch.randn(V, H * D, generator=g, device=DEV) * 0.3).to(dt)
        self.qw, self.kw = (1 + 0.1 * torch.randn(D, generator=g, device=DEV) for _ in range(2))
        ang = torch.arange(256, device=DEV)[:, None] * 1e4 ** (-torch.arange(0, D, 2, device=DEV) / D)
        self.cos, self.sin = (torch.cat([f(ang)] * 2, 1).float() for f in (torch.cos, torch.sin))
        self.lmk = torch.arange(4, dtype=torch.int32, device=DEV).expand(H, R, 1, 4).contiguous()
        self.state = dict(cache=ops.new_cache(pages, G, D, block_tokens=bt, device=DEV, bits=4),
                          table=torch.full((R, 256 // bt), -1, dtype=torch.int32, device=DEV),
                          ring=torch.randperm(pages, generator=g, device=DEV).to(torch.int32), span=torch.tensor([0, pages], device=DEV),
                          seq=torch.zeros(R, dtype=torch.int32, device=DEV), held=torch.zeros(R, dtype=torch.int32, device=DEV))

    def copy(self, s):
        return {k: ops.Cache4(*(t.clone() for t in v)) if k == "cache" else v.clone() for k, v in s.items()}

    def step(self, s, tokens, new, u, v, draft, w_max=20):
        """One step of n + 1 rows a request, in place on s; returns everything it computed."""
        R, H, G, D, n = self.R, self.H, self.G, self.D, self.n
        T = R * (n + 1)
        rows = ops.cache_rows_(s["seq"], new, s["table"], s["ring"], s["span"], T, block_tokens=self.bt, held=s["held"])
        x = self.emb[tokens]
        q, k = ops.qk_norm_rope(x[:, :H * D].view(T, H, D), x[:, H * D:(H + G) * D].view(T, G, D), self.qw, self.kw, self.cos, self.sin, pos=rows.pos)
        vv = x[:, (H + G) * D:].view(T, G, D)
        ops.cache_write_(k, vv, s["cache"], rows.pieces)
        w = torch.full((T,), w_max, dtype=torch.int32, device=DEV)
        out, lse = ops.cache_attention(q, s["cache"], s["table"], rows.req, rows.pos, w, self.lmk, w_max=w_max, rows_per_req=n + 1)
        logits = out.view(T, -1) @ self.head.T
        got = ops.verify_rows(logits, tokens, rows.cu, u, v, draft_logits=draft, temperature=0.9)
        s["held"].copy_(torch.where(new < 0, torch.zeros_like(s["held"]), torch.maximum(s["held"], rows.seq_len)))
        s["seq"].copy_(torch.where(new > 0, rows.seq_len - new + 1 + got.accepted, rows.seq_len))
        s["span"].copy_(rows.span)
        return [rows.granted, rows.pos, q, k, out, lse, logits, *got], vv, logits


def test_speculative_steps_against_the_oracle():
    """Steps whose drafts are partly refused, over page ends: attention and tokens follow the oracle at every step, no page
    belongs to two requests, and all come back when the requests end."""
    a = Run(5, 8, 2, 64, 16, 211, 3, torch.bfloat16, 0)
    s, g = a.state, torch.Generator(device=DEV).manual_seed(1)
    R, n, T = a.R, a.n, a.R * 4
    pages = O4.Pages4(3 * R, a.G, a.bt, a.D)
    last = torch.randint(0, a.V, (R,), generator=g, device=DEV)
    new = torch.full((R,), n + 1, dtype=torch.int32, device=DEV)
    taken = []
    for _ in range(9):
        before = a.copy(s)
        # tokens of the next positions drafted from logits near the target's (those of a pass without drafts)
        tokens = torch.cat([last[:, None], torch.randint(0, a.V, (R, n), generator=g, device=DEV)], 1)
        for i in range(n):
            logits = a.step(a.copy(s), tokens.view(-1), new, torch.zeros(T, device=DEV), torch.zeros(R, device=DEV), None)[2].view(R, n + 1, -1)
            tokens[:, i + 1] = torch.multinomial(torch.softmax(logits[:, i].float() / 0.9 + 0.5, 1), 1, generator=g)[:, 0]
        draft = (logits.float() + 0.5 * torch.randn(logits.shape, generator=g, device=DEV)).to(a.dt).view(T, -1)
        u, v = torch.rand(T, generator=g, device=DEV), torch.rand(R, generator=g, device=DEV)
        (granted, pos, q, k, out, lse, logits, accepted, toks), vv, _ = a.step(s, tokens.view(-1), new, u, v, draft)
        assert granted.all()
        seq, table = before["seq"].tolist(), s["table"].cpu().numpy()
        assert pos.view(R, -1).tolist() == [[x + i for i in range(n + 1)] for x in seq]
        want = [[r * (n + 1) + i, 1, int(table[r, (seq[r] + i) // a.bt]), (seq[r] + i) % a.bt] for r in range(R) for i in range(n + 1)]
        pages.write(f64(k), f64(vv), want)
        req = [r for r in range(R) for _ in range(n + 1)]
        ref, _, mass, reach, keys = OD.attention(f64(q), pages, table, req, pos.tolist(), [20] * T, a.lmk.cpu().numpy(), None, 1 / math.sqrt(a.D))
        tol = (2 * (a.D + 8) * 2.0 ** -24 * reach + (keys + 64) * 2.0 ** -24 + 2.0 ** -16)[..., None] * mass + 2.0 ** -8 * np.abs(ref)
        assert (np.abs(f64(out) - ref) <= tol).all()
        cu = list(range(0, T + 1, n + 1))
        ra, rt = O4.verify(f64(logits), tokens.view(-1).tolist(), cu, u.tolist(), v.tolist(), f64(draft), [0.9] * R, [0.9] * R)
        assert accepted.tolist() == ra and toks.tolist() == rt
        assert s["seq"].tolist() == [x + 1 + y for x, y in zip(seq, ra)]
        taken += ra
        last = toks.view(R, -1).gather(1, accepted.long()[:, None])[:, 0]
        used = table[table >= 0].tolist()
        assert len(set(used)) == len(used) == int(s["span"][0]) == sum(-(-x // a.bt) for x in s["held"].tolist())
    assert 0 < sum(taken) < n * len(taken) and int(s["span"][0]) > R
    a.step(s, tokens.view(-1), torch.full_like(new, -1), u, v, None)
    h, t = s["span"].tolist()
    assert t - h == 3 * R and sorted(s["ring"].tolist()) == list(range(3 * R)) and not s["seq"].any() and not s["held"].any()


def test_speculative_step_captured_and_replayed():
    """A whole step in one graph whose inputs advance in place: each replay, with eager steps and synchronisations between, equals
    the eager step on a copy of its state."""
    a = Run(6, 8, 2, 128, 16, 1003, 4, torch.bfloat16, 2)
    R, n, T = a.R, a.n, a.R * 5
    g = torch.Generator(device=DEV).manual_seed(0)
    tokens = torch.randint(0, a.V, (T,), generator=g, device=DEV)
    new, u, v = torch.full((R,), n + 1, dtype=torch.int32, device=DEV), torch.rand(T, device=DEV), torch.rand(R, device=DEV)
    draft = torch.randn(T, a.V, generator=g, device=DEV).to(a.dt)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.step(a.copy(a.state), tokens, new, u, v, draft)
    torch.cuda.current_stream().wait_stream(side)
    live, start = a.copy(a.state), a.copy(a.state)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = a.step(live, tokens, new, u, v, draft)[0]
    for k in ("table", "ring", "span", "seq", "held"):
        live[k].copy_(start[k])
    for rep in range(25):
        tokens.copy_(torch.randint(0, a.V, (T,), generator=g, device=DEV))
        draft.copy_(torch.randn(T, a.V, generator=g, device=DEV) * 0.1)
        u.copy_(torch.rand(T, generator=g, device=DEV) * (0.2 if rep % 2 else 1.0))
        v.copy_(torch.rand(R, generator=g, device=DEV))
        new.fill_(n + 1)
        if rep % 7 == 6:
            new[rep % R] = -1
        eager = a.copy(live)
        ref = a.step(eager, tokens, new, u, v, draft)[0]
        torch.cuda.synchronize()
        for t in outs:
            t.fill_(-3)
        graph.replay()
        torch.cuda.synchronize()
        for i, (x, y) in enumerate(zip(outs, ref)):
            assert torch.equal(x, y), (rep, i)
        for k in ("table", "ring", "span", "seq", "held"):
            assert torch.equal(live[k], eager[k]), (rep, k)
        assert all(torch.equal(x, y) for x, y in zip(live["cache"], eager["cache"]))
    assert live["span"][1] > 3 * R


def test_split_windows_on_two_streams_at_once(monkeypatch):
    """Windows split over blocks and joined from a workspace, with inputs of their own on each of two streams in turn: equal to
    the same calls one after the other."""
    need = []
    place = ops._set_workspace
    monkeypatch.setattr(ops, "_set_workspace", lambda a, n, dev: need.append(n) or place(a, n, dev))
    cases = []
    for i in range(2):
        c = _attend_case(1, 32, 2, 128, 64, 20, torch.bfloat16, 10 * i, 0, 1, lens=[12000 + i], per=1 + i)
        cases.append((c[0].to(DEV), c[1], *(_i32(x) for x in c[2:5]), _i32([9000] * (1 + i)), _i32(c[6])))

    def work(i):
        return ops.cache_attention(*cases[i], w_max=9000, rows_per_req=1 + i)
    ref = [work(i) for i in range(2)]
    assert all(n > 0 for n in need) and len(need) == 2
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    res = [[], []]
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                res[i].append(work(i))
    torch.cuda.synchronize()
    for i in range(2):
        for got in res[i]:
            assert all(torch.equal(x, y) for x, y in zip(got, ref[i]))


def test_two_graphs_of_split_windows_replayed_in_turn():
    g = torch.Generator(device=DEV).manual_seed(8)
    cases = []
    for i in range(2):
        c = _attend_case(1, 32, 2, 128, 64, 20, torch.bfloat16, 20 + i, 0, 1, lens=[12000])
        cases.append((c[0].to(DEV), c[1], *(_i32(x) for x in c[2:5]), _i32([9000 - i]), _i32(c[6])))
    ops.cache_attention(*cases[0], w_max=9000)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for c, gr in zip(cases, graphs):
        torch.cuda.synchronize()
        with torch.cuda.graph(gr):
            outs.append(ops.cache_attention(*c, w_max=9000))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(4):
        for c in cases:
            c[0].copy_(torch.randn(c[0].shape, generator=g, device=DEV))
        ref = [ops.cache_attention(*c, w_max=9000) for c in cases]
        for o in outs:
            for t in o:
                t.fill_(-3)
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for x, y in zip(outs, ref):
            assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1]), rep


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("place", ["window", "landmarks"])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_keeps_weights_in_32_bits(dt, place, D):
    """Two keys of nearly equal weight whose values cancel, so that an output is a hundredth of its ``mass`` and shows what the
    weights lose.  A logit is at most ``reach`` = 2^-4 here and off by (D + 8) 2^-24 of it; a weight by twice that and 3 2^-24 for its
    exponent and power; the sum of two values in three parts each by 6 2^-24, that of the weights by 2 2^-24, joins and quotient by
    3 2^-24: 16 2^-24 of the mass in all beside the logits'.  (Weights of 16 bits are off by up to 2^-16, 256 2^-24.)"""
    R, H, G, bt = 64, 4, 2, 16
    g = torch.Generator().manual_seed(D)
    k = torch.randint(-4, 5, (2 * R, G, D), generator=g) / 2.0
    v = torch.tensor([0.5, 1.0, 1.5, 2.0, 3.0])[torch.randint(0, 5, (R, 1, G, D), generator=g)]
    k[..., ::32], v[..., ::32] = 2.0, 3.0  # every 32 elements have the scale 1/2: all of these are codes of it
    v = (v * torch.tensor([1.0, -1.0])[None, :, None, None]).reshape(2 * R, G, D)
    cache = ops.new_cache(R, G, D, block_tokens=bt, device=DEV, bits=4)
    ops.cache_write_(k.to(DEV), v.to(DEV), cache, _i32([[2 * i, 2, i, 0] for i in range(R)]))
    got = ops.cache_read(cache, torch.arange(R, device=DEV, dtype=torch.int32)[:, None], _i32(range(0, 2 * R + 1, 2)), n_rows=2 * R,
                         dtype=torch.float32)
    assert torch.equal(got[0].cpu(), k) and torch.equal(got[1].cpu(), v)
    q = torch.randn(R, H, D, generator=g)
    q = (q / (q[:, :, None].abs() * k.view(R, 2, G, D).abs().repeat_interleave(H // G, 2).transpose(1, 2)).sum(-1).amax(-1, keepdim=True)).to(dt)
    table = np.arange(R)[:, None]
    if place == "window":
        pos, w, lmk = [1] * R, [2] * R, np.full((H, R, 1, 0), -1)
    else:  # both lie before a window without a page, side by side in a set (a part of it that holds one key weighs it 1)
        table = np.concatenate([table, np.full((R, 1), -1)], 1)
        pos, w, lmk = [bt] * R, [1] * R, np.full((H, R, 1, 128), -1)
        lmk[..., :2] = [1, 0]
    scale = 2.0 ** -4
    out, _ = ops.cache_attention(q.to(DEV), cache, *(_i32(x) for x in (table, range(R), pos, w)), _i32(lmk).view(*lmk.shape), scale=scale,
                                 w_max=16)
    ref, _, mass, reach, keys = OD.attention(f64(q), _host_pages(cache), table, list(range(R)), pos, w, lmk, None, scale)
    assert (keys == 2).all() and (reach <= 2.0 ** -4 * 1.01).all() and (np.abs(ref) < mass / 30).mean() > 0.9
    tol = (2 * (D + 8) * reach + 16)[..., None] * 2.0 ** -24 * mass + U[dt] * np.abs(ref) + (2.0 ** -25 if dt == torch.float16 else 0)
    assert (np.abs(f64(out) - ref) <= tol).all(), float((np.abs(f64(out) - ref) / tol).max())


def test_speculative_step_of_refused_requests():
    """Requests without pages are answered from inert rows; what a caller keeps, masked by ``granted`` and ``pos``, is that of the
    others alone, as where all found their pages, and the refused ones' tokens come again in the next step."""
    a = Run(6, 4, 2, 64, 16, 97, 3, torch.bfloat16, 4)
    R, n, T = a.R, a.n, a.R * 4
    g = torch.Generator(device=DEV).manual_seed(3)
    tokens, new = torch.randint(0, a.V, (T,), generator=g, device=DEV), torch.full((R,), n + 1, dtype=torch.int32, device=DEV)
    u, v = 0.3 * torch.rand(T, generator=g, device=DEV), torch.rand(R, generator=g, device=DEV)
    draft = 0.1 * torch.randn(T, a.V, generator=g, device=DEV).to(a.dt)
    s, full = a.copy(a.state), a.copy(a.state)
    s["span"][1] = 4  # a page each for four of six
    accepted_all, tokens_all = a.step(full, tokens, new, u, v, draft)[0][-2:]
    granted, pos, *_, accepted, toks = a.step(s, tokens, new, u, v, draft)[0]
    assert granted.tolist() == [1, 1, 1, 1, 0, 0] and (pos.view(R, -1)[4:] == -1).all()
    ran = (granted > 0) & (new > 0)
    accepted, answer = torch.where(ran, accepted, 0), torch.where(pos >= 0, toks, -1)
    assert torch.equal(accepted[:4], accepted_all[:4]) and torch.equal(answer.view(R, -1)[:4], tokens_all.view(R, -1)[:4])
    assert not accepted[4:].any() and (answer.view(R, -1)[4:] == -1).all()
    s["seq"].copy_(torch.where(ran, s["seq"], 0))  # (nothing of theirs is held)
    s["held"].copy_(torch.where(ran, s["held"], 0))
    s["span"][1] = 3 * R
    only = torch.where(ran, 0, new)
    t = torch.cat([tokens[16:], tokens[:16]])  # their rows come first
    uu, dd = torch.cat([u[16:], u[:16]]), torch.cat([draft[16:], draft[:16]])
    granted, pos, *_, accepted, toks = a.step(s, t, only, uu, v, dd)[0]
    assert granted.all() and torch.equal(accepted[4:], accepted_all[4:]) and torch.equal(toks[:8], tokens_all[16:])


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("G,per,split", [(2, 1, False), (8, 1, False), (2, 3, False), (2, 1, True), (1, 2, True)])
def test_attention_of_keys_that_are_nan(dt, G, per, split):
    """Keys held as NaN where they are attended: through scores, maximum, sums and joins they make the outputs and logarithms of the rows
    and heads that attend them NaN, and leave the others' as they were.  One in the newest token (the last row's alone), in each
    wave's part of the windows, in a landmark of one head, and in every key, where no maximum is found."""
    H, D, bt = 8, 64, 16
    lens, wide = ([3000, 45, 3], 2900) if split else ([400, 45, 3], 200)
    q, cache, table, req, pos, w, lmk = _attend_case(3, H, G, D, bt, 40, dt, 31, max(lens), 30, lens=lens, per=per)
    w = [x for x in (wide, 7, 3) for _ in range(per)]
    lmk[..., 0] = 1  # of every head; before the windows of requests 0 and 1
    kw = dict(w_max=1 << 15 if split else wide, per=per)
    if split:
        table = _widened(table, bt, 1 << 15)
    a, al = _check_attend(q, cache, table, req, pos, w, lmk, **kw)
    assert np.isfinite(a).all() and np.isfinite(al).all()
    clean = cache.scale.clone()

    def put(spots):
        cache.scale.copy_(clean)
        for i, p, g in spots:
            cache.scale[int(table[i, p // bt]), g, p % bt, 0, -1] = 255
        out, lse = _check_attend(q, cache, table, req, pos, w, lmk, **kw)
        hit = np.zeros(out.shape[:2], dtype=bool)
        for t in range(len(req)):
            low = max(pos[t] - w[t] + 1, 0)
            for h in range(H):
                mine = {x for x in lmk[h, req[t], 0] if 0 <= x < low}
                hit[t, h] = any(i == req[t] and g == h // (H // G) and (low <= p <= pos[t] or p in mine) for i, p, g in spots)
        assert np.isnan(out[hit]).all() and np.isnan(lse[hit]).all() and np.array_equal(out[~hit], a[~hit]) and np.array_equal(lse[~hit], al[~hit])
        return hit
    newest = put([(0, pos[per - 1], 0)])
    assert newest.any() and newest[:per - 1].sum() == 0
    for back in (40, 70, 100, 130):  # of each wave of the block
        assert put([(0, pos[0] - back, G - 1)])[0, -1]
    assert put([(0, 1, 0), (1, 1, G - 1)]).any()
    only = max(int(p) for p in lmk[3, 0, 0] if p < pos[0] - wide + 1)  # (1, or one that few heads have)
    assert put([(0, only, 3 // (H // G))])[0, 3]
    assert put([(2, p, g) for p in range(3) for g in range(G)])[2 * per:].all()
    cache.scale[:] = 255
    out, lse = ops.cache_attention(q.to(DEV), cache, *(_i32(x) for x in (table, req, pos, w, lmk)), w_max=kw["w_max"], rows_per_req=per)
    assert out.isnan().all() and lse.isnan().all()
