"""The paged 8-bit cache on the GPU against the float64 oracle: row maps, write, read-back and attention.

Tolerances, from the arithmetic.  Row maps, codes and scales are exact.  Attention: a weight's relative error is
at most twice its logit's absolute error; a logit is a float32 dot product of D terms in any order and tree,
(D + 8) 2^-24 of the largest sum |scale q k| of its row (``reach``); sums over n keys add n 2^-24, weights handed
to the matrix products of 16-bit types in two bfloat16 parts 2^-16; the output is rounded once to its type, half a
step being 2^-8 (bfloat16), 2^-11 (float16) or 2^-24.  Errors of weights act on sum p |v| (``mass``)."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from dsalt_amd import ops
from oracle import decode as OD

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def f64(t):
    return t.detach().cpu().double().numpy()


# ------------------------------------------------------------------------ row maps
def _rows_case(seq, new, M, bt, n_rows, n_free=None, first=3, seed=0):
    """A pool with the pages of `seq` in a shuffled table and the others in a ring that has turned."""
    r = np.random.RandomState(seed)
    held = [min(max(-(-n // bt), 0), M) for n in seq]
    need = sum(max(0, -(-(a + max(b, 0)) // bt) - h) for a, b, h in zip(seq, new, held))
    n_free = need if n_free is None else n_free
    N = sum(held) + n_free + 5
    ids = r.permutation(N)
    table, ring, at = np.full((len(seq), M), -1), np.full(N, -7), 0
    for i, h in enumerate(held):
        table[i, :h] = ids[at:at + h]
        at += h
    for i in range(n_free):
        ring[(first + i) % N] = ids[at + i]
    return table, ring, [first, first + n_free]


def _check_rows(seq, new, M, bt, n_rows, **kw):
    table, ring, span = _rows_case(seq, new, M, bt, n_rows, **kw)
    wide = torch.full((len(seq), M + 3), 77, dtype=torch.int32, device=DEV)  # a table that is a view of a wider one
    wide[:, :M] = _i32(table)
    dt, dr, ds = wide[:, :M], _i32(ring), torch.tensor(span, dtype=torch.int64, device=DEV)
    want = OD.rows(seq, new, table, ring, span, n_rows, bt)
    a, b = _i32(seq), _i32(new)
    for rep in range(2):  # inputs stay: a second call on the same ones writes the same
        got = ops.cache_rows_(a, b, dt, dr, ds, n_rows, block_tokens=bt)
        for name in OD.rows([1], [1], np.zeros((1, 1), dtype=int), [0], (0, 0), 1, 16):
            assert np.array_equal(getattr(got, name).cpu().numpy(), np.asarray(want[name])), (name, rep)
        assert np.array_equal(dt.cpu().numpy(), table) and np.array_equal(dr.cpu().numpy(), ring)
    assert (wide[:, M:] == 77).all() and ds.tolist() == span and a.tolist() == list(seq)
    return want


@pytest.mark.parametrize("bt", [16, 32, 64, 128])
def test_rows_of_a_decoding_step(bt):
    """One token each, at every place of a page, with a page held or not, and a full table."""
    seq = [0, 1, bt - 1, bt, bt + 1, 4 * bt - 1, 4 * bt, 2 * bt - 1, 17]
    w = _check_rows(seq, [1] * len(seq), 4, bt, len(seq))
    assert w["granted"] == [1, 1, 1, 1, 1, 1, 0, 1, 1]
    _check_rows(seq, [1] * len(seq), 4, bt, len(seq) + 40)  # rows past the last request


@pytest.mark.parametrize("seed", range(8))
def test_rows_of_mixed_steps(seed):
    """Request counts on both sides of a thread each, and of one launch (4096)."""
    r = np.random.RandomState(seed)
    R, bt, M = [1, 5, 70, 1024, 1025, 3001, 4096, 4097][seed], [16, 64, 32, 128, 64, 16, 16, 32][seed], 9 if seed < 6 else 3
    seq = r.randint(0, bt * M + 1, R).tolist()
    new = [int(x) for x in np.where(r.rand(R) < 0.2, -r.randint(1, 4, R), np.where(r.rand(R) < 0.4, 1, r.randint(0, bt * 4, R)))]
    total = sum(max(n, 0) for n in new)
    for n_rows, free in ((total, None), (total + 13, 2), (total // 2, R)):
        _check_rows(seq, new, M, bt, n_rows, n_free=free, seed=seed)


def test_rows_without_rows_pages_or_requests():
    _check_rows([40, 0, 7], [-1, 0, -2], 4, 16, 0)                  # requests that end, no rows at all
    _check_rows([0], [0], 1, 64, 5)
    w = _check_rows([0, 16, 3], [16, 1, 1], 4, 16, 18, n_free=0)    # nothing is free: a page held still serves
    assert w["granted"] == [0, 0, 1]
    w = _check_rows([-5, 3, 200], [1, 1, -1], 4, 16, 2, n_free=4)   # a negative length, one past the table
    assert w["granted"] == [0, 1, 1]
    w = _check_rows([0, 0], [30, 3], 4, 16, 31)                      # the last request's rows do not fit
    assert w["granted"] == [1, 0]


def test_rows_ring_without_room_drops():
    """A ring that holds as much as it can keeps its pages: pages given back beyond it are dropped."""
    table, ring = np.array([[4, 5, 6]]), np.array([0, 1, 2, 3])
    want_t, want_r = table.copy(), ring.copy()
    OD.rows([48], [-1], want_t, want_r, (2, 5), 0, 16)
    dr = _i32(ring)
    got = ops.cache_rows_(_i32([48]), _i32([-1]), _i32(table), dr, torch.tensor([2, 5], device=DEV), 0, block_tokens=16)
    assert np.array_equal(dr.cpu().numpy(), want_r) and got.span.tolist() == [2, 6] and want_r[1] == 4


# ------------------------------------------------------------------------ write and read
def _host_pages(cache):
    n, g, bt, d = cache.k.shape
    p = OD.Pages(n, g, bt, d)
    p.k, p.v = (f64(c.view(torch.uint8).view(torch.float8_e4m3fn).float()) for c in cache[:2])
    p.ks, p.vs = f64(cache.k_scale), f64(cache.v_scale)
    return p


def _same_pages(cache, pages):
    got = _host_pages(cache)
    for n in ("k", "v", "ks", "vs"):
        assert np.array_equal(getattr(got, n), getattr(pages, n), equal_nan=True), n


def _random_cache(n_blocks, G, bt, D, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    c = ops.new_cache(n_blocks, G, D, block_tokens=bt, device=DEV)
    for codes, scale in ((c.k, c.k_scale), (c.v, c.v_scale)):
        scale.copy_(torch.exp2(torch.randint(-12, -4, scale.shape, generator=g).float()))
        codes.view(torch.uint8).copy_((torch.randn(codes.shape, generator=g) * 60).clamp(-448, 448).to(torch.float8_e4m3fn)
                                      .view(torch.uint8))
    return c


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bt,D,G", [(16, 64, 3), (32, 128, 1), (64, 64, 1), (128, 128, 2)])
def test_write_follows_the_oracle(dt, bt, D, G):
    """Steps of whole prompts, single tokens and runs that end and begin inside pages, with magnitudes from step
    to step up and down so that scales grow under held codes; other pages stay bit for bit."""
    R, M = 5, 6
    cache = _random_cache(R * M + 4, G, bt, D, bt + D)
    pages = _host_pages(cache)
    table = torch.full((R, M), -1, dtype=torch.int32, device=DEV)
    ring = torch.randperm(R * M + 4).to(torch.int32).to(DEV)
    span = torch.tensor([0, R * M + 4], device=DEV)
    seq = torch.zeros(R, dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(3)
    steps = [([bt, 1, 3 * bt + 5, 0, 2 * bt - 1], 1.0), ([1] * R, 30.0), ([1, 2, 1, 7, 1], 0.01), ([1] * R, 1000.0),
             ([bt // 2, 1, 1, bt, 3], 1e-6)]
    for new, size in steps:
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
        kr, vr = ops.cache_read(cache, table, _i32(cu), n_rows=int(cu[-1]) + 3, dtype=od)
        wk, wv = pages.read(table.cpu().numpy(), cu, [0] * R, int(cu[-1]) + 3)
        for got, want in ((kr, wk), (vr, wv)):
            assert torch.equal(got.cpu(), torch.from_numpy(want).to(od))


def test_write_extremes():
    """Zeros, subnormals, values near the types' largest, infinities and NaN; codes on the rounding ties."""
    rows = torch.zeros(12, 1, 64)
    rows[1, 0, :5] = torch.tensor([1e-45, -1e-40, 2.0 ** -126, -2.0 ** -120, 0.0])
    rows[2, 0, :4] = torch.tensor([3.4e38, -3.3e38, 1.0, 1e-38])
    rows[3, 0, :5] = torch.tensor([float("inf"), float("-inf"), float("nan"), 3.0, -0.0])
    rows[4] = float("nan")
    rows[5, 0] = torch.arange(64) * 0.5 + 200  # ties between codes 16 and 32 apart
    rows[6, 0] = (torch.arange(64) - 32) * 2.0 ** -10  # ties among the subnormals beside one of 448
    rows[6, 0, 63] = 448.0
    rows[7, 0, 0], rows[8, 0, 0], rows[9, 0, 0] = 448.0, 448.00003, 447.99997
    for lo in range(0, 12):
        cache = _random_cache(3, 1, 16, 64, lo)
        pages = _host_pages(cache)
        pieces = _i32([[lo, 1, 1, 0], [0, 0, 0, 0]])
        x = rows.to(DEV)
        ops.cache_write_(x, x, cache, pieces)
        pages.write(f64(x), f64(x), pieces.cpu().numpy())
        _same_pages(cache, pages)
        after = _i32([[(lo + 5) % 12, 3 if lo + 5 < 10 else 1, 1, 1]])  # then rows beside it: the scale may grow
        ops.cache_write_(x, x, cache, after)
        pages.write(f64(x), f64(x), after.cpu().numpy())
        _same_pages(cache, pages)


def test_write_skips_pieces_that_lie_outside():
    cache = _random_cache(4, 2, 16, 64, 9)
    before = [t.clone() for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)]
    x = torch.randn(8, 2, 64, device=DEV)
    bad = [[0, 1, 4, 0], [0, 1, -1, 0], [7, 2, 0, 0], [-1, 1, 0, 0], [0, 3, 0, 14], [0, 1, 0, -1], [0, -4, 0, 0], [0, 0, 2, 0],
           [2 ** 31 - 1, 2, 0, 0], [0, 2 ** 31 - 1, 0, 1]]
    ops.cache_write_(x, x, cache, _i32(bad))
    for a, b in zip((cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale), before):
        assert torch.equal(a, b)


def test_write_of_rows_in_other_layouts():
    """Heads first, a token stride of one element too many, an offset off 16 bytes: the same codes."""
    x = torch.randn(20, 2, 64, device=DEV).to(torch.bfloat16)
    pieces = _i32([[0, 16, 0, 0], [16, 4, 1, 3]])
    ref = ops.cache_write_(x, x, ops.new_cache(2, 2, 64, block_tokens=16), pieces)
    flat = torch.zeros(20 * 129 + 1, device=DEV, dtype=torch.bfloat16)
    odd = flat[1:1 + 20 * 128].view(20, 2, 64)
    odd.copy_(x)
    gap = torch.zeros(20, 129, device=DEV, dtype=torch.bfloat16)
    gap[:, :128] = x.view(20, 128)
    for y in (x.transpose(0, 1).contiguous().transpose(0, 1), odd, gap[:, :128].unflatten(1, (2, 64)),
              x.transpose(1, 2).contiguous().transpose(1, 2)):
        got = ops.cache_write_(y, y, ops.new_cache(2, 2, 64, block_tokens=16), pieces)
        for a, b in zip(got, ref):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_read_outside_is_zero():
    cache = _random_cache(4, 1, 16, 64, 2)
    table = _i32([[0, 9, -1], [3, 2, 1]])
    cu = [2, 30, 40]  # the first rows belong to no request
    start = [4, 45]
    k, v = ops.cache_read(cache, table, _i32(cu), start=_i32(start), n_rows=50, dtype=torch.float32)
    wk, wv = _host_pages(cache).read(table.cpu().numpy(), cu, start, 50)
    assert np.array_equal(f64(k), wk) and np.array_equal(f64(v), wv) and not wk[:2].any() and not wk[14:30].any()


# ------------------------------------------------------------------------ attention
def _attend_case(R, H, G, D, bt, K, dt, seed, max_len, w_max, rows_per=1, lens=None):
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
    req = [i for i in range(R) for _ in range(rows_per)]
    pos = [max(0, lens[i] - 1 - j) for i in range(R) for j in range(rows_per)]
    T = len(req)
    q = torch.randn(T, H, D, generator=g).to(dt)
    w = [int(x) for x in r.randint(0, w_max + 1, T)]
    lmk = np.full((H, R, 1, K), -1)
    for i in range(R):
        for h in range(H):
            p = r.randint(0, lens[i], K)  # any order, repeats, inside the window too
            lmk[h, i, 0] = np.where(r.rand(K) < 0.2, -1 - r.randint(0, 9, K), p)
    return q, cache, table, req, pos, w, lmk


def _check_attend(q, cache, table, req, pos, w, lmk, bias=None, scale=None, w_max=None, pages=None, dev_q=None):
    T, H, D = q.shape
    pages = pages or _host_pages(cache)
    args = (_i32(table), _i32(req), _i32(pos), _i32(w), _i32(lmk).view(*np.shape(lmk)))
    b = torch.from_numpy(bias).float().to(DEV) if bias is not None else None
    out, lse = ops.cache_attention(q.to(DEV) if dev_q is None else dev_q, cache, *args, b, scale=scale, w_max=w_max)
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


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,H,G,D,bt,K,max_len,w_max", [
    (1, 1, 1, 64, 16, 0, 1, 1), (1, 16, 2, 128, 64, 33, 700, 512), (7, 4, 4, 64, 16, 5, 90, 40), (3, 8, 1, 128, 32, 16, 300, 128),
    (4, 32, 1, 64, 128, 9, 400, 70), (2, 34, 2, 64, 16, 3, 200, 200), (5, 6, 2, 128, 128, 64, 257, 1), (2, 2, 1, 64, 32, 130, 1500, 1500),
    (40, 3, 3, 128, 16, 7, 60, 33)])
def test_attention_follows_the_oracle(dt, R, H, G, D, bt, K, max_len, w_max):
    c = _attend_case(R, H, G, D, bt, K, dt, R * 7 + H, max_len, w_max)
    a = _check_attend(*c, w_max=w_max)
    b = _check_attend(*c)  # the bound on the windows not given
    bias = np.random.RandomState(1).randn(*c[-1].shape)
    bias[..., ::3] = -np.inf
    _check_attend(*c, bias=bias, scale=0.3, w_max=max(1, w_max // 3))  # and given too small


@pytest.mark.parametrize("bt", [16, 64, 128])
@pytest.mark.parametrize("G", [1, 4])
def test_attention_at_every_page_place(bt, G):
    """Positions around the ends of pages and of the kernels' runs of keys, windows from one key to all."""
    lens = [1, 2, bt - 1, bt, bt + 1, 31, 32, 33, 63, 64, 65, 2 * bt, 2 * bt + 1, 127, 128, 129, 255, 257]
    for wide in (1, 2, 16, 17, 10 ** 6):
        c = list(_attend_case(len(lens), 4, G, 64, bt, 6, torch.bfloat16, bt + G, 0, 1, lens=lens))
        c[5] = [wide] * len(lens)
        _check_attend(*c, w_max=wide)


def test_attention_several_rows_of_a_request():
    c = _attend_case(3, 8, 2, 64, 32, 12, torch.bfloat16, 5, 150, 60, rows_per=5)
    order = np.random.RandomState(0).permutation(15)  # rows in any order
    q, cache, table, req, pos, w, lmk = c
    _check_attend(q[order], cache, table, [req[i] for i in order], [pos[i] for i in order], [w[i] for i in order], lmk, w_max=60)


@pytest.mark.parametrize("wide", [False, True])
def test_attention_inert_rows_and_absent_pages(wide):
    q, cache, table, req, pos, w, lmk = _attend_case(6, 4, 2, 64, 16, 8, torch.float32, 11, 100, 50, lens=[100, 3, 50, 77, 64, 20])
    req[0], pos[1], req[2] = -1, -1, 6           # no request, no position, a request past the table
    table[3] = -1                                 # no page at all
    table[4, 1], table[4, 3] = -3, len(cache.k)   # pages below and past the cache
    pos[5] = 10 ** 6                              # past the table: only landmarks are there
    w[5] = 5
    if wide:
        table, pos[5] = _widened(table, 16, 1 << 15), 1 << 20
    out, lse = _check_attend(q, cache, table, req, pos, w, lmk, w_max=None if wide else 50)
    assert np.isneginf(lse[:4]).all() and np.isfinite(lse[4:]).all()


def _widened(table, bt, tokens):
    """The table with empty columns up to `tokens` tokens a request: with the bound on the windows not given, the
    kernels are chosen for windows that long."""
    return np.pad(table, ((0, 0), (0, max(0, tokens // bt - table.shape[1]))), constant_values=-1)


# what the size rules choose between, and a shape each (R, H, G, D, bt, K, lens or the longest, largest window, bound given)
RULES = {
    "heads, four waves": (9, 4, 4, 64, 32, 20, 300, 200, 200),
    "heads, eight waves": (2, 4, 4, 128, 64, 40, 900, 700, 700),
    "heads, split": (1, 2, 2, 128, 64, 70, [3001], 2900, 2900),
    "heads of a group, split": (1, 8, 2, 64, 16, 9, [2500], 2500, 2500),
    "groups, split, most splits empty": (3, 8, 2, 64, 16, 130, [300, 33, 1], 290, 1 << 15),
    "groups, split, float rows full": (2, 12, 4, 128, 128, 70, [4100, 2000], 4100, 1 << 14),
    "groups, eight waves": (128, 8, 2, 64, 64, 17, 90, 60, 300),
    "groups, four waves": (140, 8, 2, 128, 32, 33, 90, 60, 300),
    "groups of 17 heads": (70, 34, 2, 64, 16, 5, 70, 40, 150),
    "groups of 16 heads of 128": (40, 32, 2, 128, 64, 6, 150, 100, 256),
}


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rule", RULES)
def test_attention_on_each_side_of_the_size_rules(rule, dt):
    R, H, G, D, bt, K, lens, w, bound = RULES[rule]
    c = list(_attend_case(R, H, G, D, bt, K, dt, R + H, lens if isinstance(lens, int) else max(lens), w, lens=None if isinstance(lens, int) else lens))
    if isinstance(lens, list):
        c[5] = [w, w // 2, 5][:R]
    c[2] = _widened(c[2], bt, bound)
    _check_attend(*c, w_max=bound)
    bias = np.random.RandomState(3).randn(*c[-1].shape)
    _check_attend(*c, bias=bias, w_max=bound)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("G", [2, 8])
def test_attention_reads_nothing_masked(dt, G, wide):
    """NaN codes in every token that a row does not attend (behind the last, before the window, landmarks of
    other heads, pages of nobody, scales of pages without a key): results as without them.  A NaN that a
    row attends reaches its own heads alone."""
    H, D, bt = 8, 64, 16
    q, cache, table, req, pos, w, lmk = _attend_case(3, H, G, D, bt, 9, dt, 21, 200, 30, lens=[200, 45, 1])
    w = [30, 7, 3]
    clean = _host_pages(cache)
    seen = np.zeros((len(cache.k), G, bt), dtype=bool)
    for i in range(3):
        low = max(pos[i] - w[i] + 1, 0)
        for h in range(H):
            for p in list(range(low, pos[i] + 1)) + [int(x) for x in lmk[h, i, 0] if 0 <= x < low]:
                seen[table[i, p // bt], h // (H // G), p % bt] = True
    hide = torch.from_numpy(~seen).to(DEV)
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        codes.view(torch.uint8)[hide] = 0x7f
        scale[~torch.from_numpy(seen.any(-1)).to(DEV)] = float("nan")
    bound = (1 << 15) + 31 if wide else 30  # (a key/value head's query heads as a group, or one by one)
    table = _widened(table, bt, bound)
    a, _ = _check_attend(q, cache, table, req, pos, w, lmk, pages=clean, w_max=bound)
    assert np.isfinite(a).all()
    # one landmark of head 3 of request 0 now holds NaN values: rows of the other heads stay
    only = int(next(p for p in lmk[3, 0, 0] if 0 <= p < pos[0] - 29))
    users = [h for h in range(H) if h // (H // G) == 3 // (H // G) and only in lmk[h, 0, 0]]
    cache.v.view(torch.uint8)[table[0, only // bt], 3 // (H // G), only % bt] = 0x7f
    b = f64(ops.cache_attention(q.to(DEV), cache, _i32(table), _i32(req), _i32(pos), _i32(w), _i32(lmk), w_max=bound)[0])
    for h in range(H):
        assert np.isnan(b[0, h]).all() if h in users else np.array_equal(a[0, h], b[0, h])
    assert np.array_equal(a[1:], b[1:])


def test_attention_empty_by_bias():
    """Landmarks of weight -inf and a window whose page is absent: nothing is attended."""
    q, cache, table, req, pos, w, lmk = _attend_case(2, 2, 1, 64, 16, 4, torch.float32, 2, 60, 4, lens=[60, 60])
    w, table[0, 3] = [4, 4], -1
    bias = np.zeros(lmk.shape)
    bias[:, 0] = -np.inf
    out, lse = _check_attend(q, cache, table, req, pos, w, lmk, bias=bias)
    assert np.isneginf(lse[0]).all() and np.isfinite(lse[1]).all()


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_attention_reads_nothing_behind_a_bias_of_minus_infinity(dt, wide):
    """Landmarks masked by their bias hold NaN (keys, values or scales): results as without them."""
    H, G, bt = 8, 2, 16
    q, cache, table, req, pos, w, lmk = _attend_case(3, H, G, 64, bt, 6, dt, 5, 200, 9, lens=[200, 150, 90])
    w = [9, 9, 9]
    lmk[:] = np.array([0, 17, 33, 40, 49, 64])
    bias = np.random.RandomState(0).randn(*lmk.shape)
    bias[..., [1, 2, 4]] = -np.inf
    clean = _host_pages(cache)
    for r in range(3):
        cache.k.view(torch.uint8)[table[r, 1], :, 1] = 0x7f
        cache.v.view(torch.uint8)[table[r, 2], :, 1] = 0xff
        cache.k_scale[table[r, 3]] = cache.v_scale[table[r, 3]] = float("nan")
    bound = (1 << 15) + 31 if wide else 30
    out, lse = _check_attend(q, cache, _widened(table, bt, bound), req, pos, w, lmk, bias=bias, pages=clean, w_max=bound)
    assert np.isfinite(out).all() and np.isfinite(lse).all()


@pytest.mark.parametrize("lowest", [-1e4, -3.4e38])
def test_attention_masks_of_the_lowest_value(lowest):
    """Landmarks masked by a large negative bias weigh nothing beside others, and share the weight where they are all
    that a row attends."""
    q, cache, table, req, pos, w, lmk = _attend_case(2, 2, 1, 64, 16, 8, torch.float32, 2, 60, 4, lens=[60, 60])
    w, table[0, 3] = [4, 4], -1
    lmk[:] = np.arange(8) * 4
    bias = np.zeros(lmk.shape)
    bias[:, 0] = lowest
    bias[:, 1, :, ::2] = lowest
    out, _ = ops.cache_attention(q.to(DEV), cache, _i32(table), _i32(req), _i32(pos), _i32(w), _i32(lmk),
                                 torch.from_numpy(bias).float().to(DEV))
    pages = _host_pages(cache)
    same = np.zeros(lmk.shape)  # a bias common to all that is attended changes no weight
    if lowest == -1e4:
        ref, *_ = OD.attention(f64(q), pages, table, req, pos, w, lmk, same, 0.125)
        assert np.allclose(f64(out)[0], ref[0], rtol=0, atol=2e-3 * np.abs(ref[0]).max())  # logits beside 1e4 keep 2^-10 of a unit
    else:  # beside 3.4e38 logits do not count: the mean of the values
        v = np.stack([pages.token(table[0], int(p))[1][0] for p in lmk[0, 0, 0]])
        assert np.allclose(f64(out)[0], v.mean(0), rtol=0, atol=1e-5 * np.abs(v).max())
    keep = np.where(bias[:, 1:2] < 0, -1, lmk[:, 1:2])
    ref, *_ = OD.attention(f64(q)[1:], pages, table[1:], [0], pos[1:], w[1:], keep, None, 0.125)
    assert np.allclose(f64(out)[1], ref[0], rtol=0, atol=1e-5 * np.abs(ref).max())


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
    cache = ops.new_cache(n, G, D, block_tokens=bt, device=DEV)
    g = torch.Generator().manual_seed(4)
    last = 4 * bt
    use = [n - 1, n - 3, 5, n - 2]
    small = _random_cache(4, G, bt, D, 6)
    for i, b in enumerate(use):
        for a, s in zip(cache, small):
            if a.dim() == 4:
                a.view(torch.uint8)[b] = s.view(torch.uint8)[i]
            else:
                a[b] = s[i]
    M = 3000
    table = np.full((1, M), -1)
    at = [0, M - 3, M - 2, M - 1]
    table[0, at] = use
    lmk = np.full((16, 1, 1, 5), -1)
    lmk[:, 0, 0, :3] = [5, 127, (M - 3) * bt + 1]
    q = torch.randn(1, 16, D, generator=g).to(torch.bfloat16)
    p = _host_pages(small)
    ref_table = np.full((1, M), -1)
    ref_table[0, at] = [0, 1, 2, 3]
    out, lse = ops.cache_attention(q.to(DEV), cache, _i32(table), _i32([0]), _i32([M * bt - 2]), _i32([w]), _i32(lmk), w_max=w)
    ref, rl, mass, reach, keys = OD.attention(f64(q), p, ref_table, [0], [M * bt - 2], [w], lmk, None, 1 / math.sqrt(D))
    tol = (2 * (D + 8) * 2.0 ** -24 * reach + 2.0 ** -15)[..., None] * mass + U[torch.bfloat16] * np.abs(ref)
    assert (np.abs(f64(out) - ref) <= tol).all()
    k, v = ops.cache_read(cache, _i32(table), _i32([0, 4]), start=_i32([M * bt - 4]), n_rows=4, dtype=torch.float32)
    wk, wv = p.read(ref_table, [0, 4], [M * bt - 4], 4)
    assert np.array_equal(f64(k), wk) and np.array_equal(f64(v), wv)


def test_attention_of_long_windows():
    """A window of 40000 keys split over the chip against float64 torch on the same values."""
    n, H, G, D, bt = 40001, 8, 2, 128, 64
    cache = _random_cache(-(-n // bt), G, bt, D, 1)
    table = torch.arange(-(-n // bt), dtype=torch.int32).flip(0)[None]
    q = torch.randn(1, H, D).to(torch.bfloat16)
    lmk = torch.full((H, 1, 1, 0), -1, dtype=torch.int32)
    k, v = (x.double().cpu() for x in ops.cache_read(cache, table.to(DEV), _i32([0, n]), n_rows=n, dtype=torch.float32))
    for w in (n, n - 1, 20000):
        out, lse = ops.cache_attention(q.to(DEV), cache, table.to(DEV), _i32([0]), _i32([n - 1]), _i32([w]), lmk.to(DEV), w_max=w)
        s = torch.einsum("hd,nhd->hn", q[0].double(), k[n - w:].repeat_interleave(H // G, 1)) / math.sqrt(D)
        p = torch.softmax(s, 1)
        ref = torch.einsum("hn,nhd->hd", p, v[n - w:].repeat_interleave(H // G, 1))
        mass = torch.einsum("hn,nhd->hd", p, v[n - w:].abs().repeat_interleave(H // G, 1))
        reach = torch.einsum("hd,nhd->hn", q[0].double().abs(), k.abs().repeat_interleave(H // G, 1)).amax(1) / math.sqrt(D)
        # sums over lanes, waves and splits: chains of at most n / 256 keys and joins of 64 and 1024 parts
        tol = (2 * (D + 8) * 2.0 ** -24 * reach + 2000 * 2.0 ** -24 + 2.0 ** -16)[:, None] * mass + 2.0 ** -8 * ref.abs()
        assert ((out[0].cpu().double() - ref).abs() <= tol).all()
        assert torch.allclose(lse[0].cpu().double(), torch.logsumexp(s, 1), atol=3e-4, rtol=1e-6)


# ------------------------------------------------------------------------ a decoding run
def _decode_state(R, G, D, bt, M, n, dt, seed):
    g = torch.Generator().manual_seed(seed)
    cache = ops.new_cache(n, G, D, block_tokens=bt, device=DEV)
    return dict(cache=cache, table=torch.full((R, M), -1, dtype=torch.int32, device=DEV),
                ring=torch.randperm(n, generator=g).to(torch.int32).to(DEV), span=torch.tensor([0, n], device=DEV),
                seq=torch.zeros(R, dtype=torch.int32, device=DEV))


def test_prompt_then_tokens_as_the_prompt_forward():
    """A prompt written in two parts and tokens added one at a time: every row of attention over the cache equals
    attention_forward over the cache's own values (exact in bfloat16), with the selection's landmarks."""
    R, H, G, D, bt, K = 3, 8, 2, 64, 32, 9
    s = _decode_state(R, G, D, bt, 12, 40, torch.bfloat16, 0)
    g = torch.Generator().manual_seed(1)
    lmk = None
    for step, new in enumerate(([70, 1, 33], [30, 64, 0], [1, 1, 1], [1, 1, 1], [1, 0, 1], [1, 1, -1])):
        T = sum(max(x, 0) for x in new)
        rows = ops.cache_rows_(s["seq"], _i32(new), s["table"], s["ring"], s["span"], T, block_tokens=bt)
        s["seq"], s["span"] = rows.seq_len, rows.span
        assert rows.granted.all()
        x = torch.randn(T, (H + 2 * G) * D, generator=g).to(torch.bfloat16).to(DEV)
        q = x[:, :H * D].view(T, H, D)
        ops.cache_write_(x[:, H * D:(H + G) * D].view(T, G, D), x[:, (H + G) * D:].view(T, G, D), s["cache"], rows.pieces)
        n = s["seq"].tolist()
        cu = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        k, v = ops.cache_read(s["cache"], s["table"], _i32(cu), n_rows=int(cu[-1]), dtype=torch.bfloat16)
        w_all = torch.randint(1, 40, (int(cu[-1]),), generator=g).to(torch.int32).to(DEV)
        if step == 1:  # sets chosen once the prompts are there
            lmk = ops.select_landmarks(torch.randn(int(cu[-1]), 64, generator=g).to(torch.bfloat16).to(DEV), v,
                                       torch.full((H,), 0.5, device=DEV), w_all, _i32(cu), K, max_seqlen=max(n))
        if step < 2:
            continue
        at = [int(cu[r]) + int(p) for r, p in zip(rows.req.tolist(), rows.pos.tolist())]
        full_q = torch.zeros((int(cu[-1]), H, D), dtype=torch.bfloat16, device=DEV)
        full_q[at] = q
        out, lse = ops.cache_attention(q, s["cache"], s["table"], rows.req, rows.pos, w_all[at], lmk, w_max=40)
        ref, rl = ops.attention_forward(full_q, k, v, w_all, _i32(cu), lmk, None, max_seqlen=max(n))
        assert (out.float() - ref[at].float()).norm() <= 2 * 2.0 ** -8 * ref[at].float().norm()
        # the forward sums the weights it rounded to bfloat16, each off by at most 2^-8 of itself, so the log of its
        # sum is off by at most -log(1 - 2^-8) = 2^-8 (1 + 2^-9 + ..); 1e-4 is left for float32
        assert (lse - rl[at]).abs().max() <= 2.0 ** -8 * (1 + 2.0 ** -8) + 1e-4


def test_step_captured_and_replayed():
    """Row maps, write, attention and sampling of a step in one graph whose inputs advance in place: each replay,
    with eager steps and synchronisations between, equals the eager step on a copy of its state."""
    R, H, G, D, bt, V = 9, 8, 2, 128, 16, 1003
    g = torch.Generator(device=DEV).manual_seed(0)
    s = _decode_state(R, G, D, bt, 8, 80, torch.bfloat16, 0)
    x = torch.zeros(R, (H + 2 * G) * D, dtype=torch.bfloat16, device=DEV)
    u, w = torch.zeros(R, device=DEV), torch.full((R,), 30, dtype=torch.int32, device=DEV)
    new = torch.ones(R, dtype=torch.int32, device=DEV)
    lmk = torch.arange(4, dtype=torch.int32, device=DEV).expand(H, R, 1, 4).contiguous()
    head = torch.randn(V, H * D, generator=g, device=DEV).to(torch.bfloat16) * 0.1

    def step(s, x, u, new):
        rows = ops.cache_rows_(s["seq"], new, s["table"], s["ring"], s["span"], R, block_tokens=bt)
        ops.cache_write_(x[:, H * D:(H + G) * D].view(R, G, D), x[:, (H + G) * D:].view(R, G, D), s["cache"], rows.pieces)
        out, lse = ops.cache_attention(x[:, :H * D].view(R, H, D), s["cache"], s["table"], rows.req, rows.pos, w, lmk, w_max=30)
        token, logp = ops.sample_rows(out.view(R, -1) @ head.T, u, temperature=0.8, top_k=40, top_p=0.9)
        s["seq"].copy_(rows.seq_len)
        s["span"].copy_(rows.span)
        return [out, lse, token, logp, rows.slot]

    def copy(s):
        return {k: ops.Cache8(*(t.clone() for t in v)) if k == "cache" else v.clone() for k, v in s.items()}

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(copy(s), x, u, new)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    live = copy(s)
    with torch.cuda.graph(graph):
        outs = step(live, x, u, new)
    for k in ("table", "ring", "span", "seq"):
        live[k].copy_(s[k])
    for rep in range(40):
        x.copy_(torch.randn(x.shape, generator=g, device=DEV) * (1 + rep % 5))
        u.copy_(torch.rand(R, generator=g, device=DEV))
        new.fill_(1)
        if rep % 7 == 6:
            new[rep % R] = -1
        eager = copy(live)
        ref = step(eager, x, u, new)
        torch.cuda.synchronize()
        for t in outs:
            t.fill_(-3)
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(outs, ref)):
            assert torch.equal(a, b), (rep, i)
        for k in ("table", "ring", "span", "seq"):
            assert torch.equal(live[k], eager[k]), (rep, k)
        for a, b in zip(live["cache"], eager["cache"]):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert live["span"][0] > 9 and live["span"][1] > 80  # pages were taken and given back


def test_large_calls_captured_and_replayed():
    """A call whose window is split and joined, one with more than 64 KB of LDS, and a row whose weights are by value: each
    replay equals the eager call on the inputs of the moment."""
    g = torch.Generator(device=DEV).manual_seed(3)
    a = _attend_case(1, 32, 2, 128, 64, 20, torch.bfloat16, 3, 12000, 9000, lens=[12000])
    b = _attend_case(140, 32, 2, 128, 64, 20, torch.bfloat16, 4, 200, 120)
    cases = [(q.to(DEV), cache, *(_i32(x) for x in rest[:4]), _i32(rest[4])) for q, cache, *rest in (a, b)]
    x, u = torch.zeros(5, 9001, device=DEV, dtype=torch.bfloat16), torch.zeros(5, device=DEV)

    def step():
        return [*ops.cache_attention(*cases[0], w_max=9000), *ops.cache_attention(*cases[1], w_max=200), *ops.sample_rows(x, u, top_p=0.9),
                *ops.sample_rows(x, u, top_k=20)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for rep in range(4):
        x.copy_(torch.randn(x.shape, generator=g, device=DEV) * 3)
        u.copy_(torch.rand(5, generator=g, device=DEV))
        for c in cases:
            c[0].copy_(torch.randn(c[0].shape, generator=g, device=DEV))
        ref = step()
        torch.cuda.synchronize()
        for t in outs:
            t.fill_(-3)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(outs, ref)), rep


def test_two_streams_at_once():
    """Two independent attentions and samplings enqueued on two streams equal the same ones in turn."""
    cases = [_attend_case(20, 16, 2, 128, 64, 30, torch.bfloat16, i, 3000, 512) for i in range(2)]
    cases = [(c[0].to(DEV), c[1], *(_i32(x) for x in c[2:6]), _i32(c[6])) for c in cases]
    logits = [torch.randn(20, 30011, device=DEV) * 3 for _ in range(2)]
    u = torch.rand(20, device=DEV)

    def work(i):
        res = []
        for _ in range(3):
            res += [*ops.cache_attention(*cases[i], w_max=512), *ops.sample_rows(logits[i], u, top_p=0.8)]
        return res
    ref = [work(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    res = []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for i, st in enumerate(streams):
        with torch.cuda.stream(st):
            res.append(work(i))
    torch.cuda.synchronize()
    for a, b in zip(res, ref):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


# ------------------------------------------------------------------------ more than one launch holds
def _repeats(x, ref):
    """x [T, ...] is ref [n, ...] over and over."""
    n, whole = len(ref), len(x) // len(ref) * len(ref)
    return torch.equal(x[whole:], ref[:len(x) - whole]) and bool((x[:whole].view(-1, *ref.shape) == ref).all())


def test_attention_of_more_rows_than_a_launch_holds():
    q, cache, table, req, pos, w, lmk = _attend_case(64, 16, 16, 64, 16, 2, torch.bfloat16, 1, 40, 5)
    args = [_i32(x) for x in (req, pos, w)]
    out, lse = ops.cache_attention(q.to(DEV), cache, _i32(table), *args, _i32(lmk), w_max=5)
    T = (1 << 20) + 77
    turn = torch.arange(T, device=DEV) % 64
    big, bl = ops.cache_attention(q.to(DEV)[turn], cache, _i32(table), *(x[turn] for x in args), _i32(lmk), w_max=5)
    assert _repeats(big, out) and _repeats(bl, lse)


def test_read_of_more_rows_than_a_launch_holds():
    cache = _random_cache(5, 4, 16, 64, 2)
    R = (1 << 17) + 3  # requests of 64 tokens in the same four pages, the last one cut short
    table = _i32([[3, 0, 4, 1]]).expand(R, 4).contiguous()
    n = 64 * R - 5
    k, v = ops.cache_read(cache, table, torch.arange(R + 1, dtype=torch.int32, device=DEV) * 64, n_rows=n)
    rk, rv = ops.cache_read(cache, table[:1], _i32([0, 64]), n_rows=64)
    assert rk.any() and _repeats(k, rk) and _repeats(v, rv)


def test_write_of_more_pieces_than_a_launch_holds():
    """Most pieces hold no rows; those that do lie on both sides of where a launch ends."""
    P, x = (1 << 24) + 9, torch.randn(40, 2, 64).to(torch.bfloat16).to(DEV)
    few = _i32([[4 * i, 4, i, i] for i in range(10)])
    at = torch.tensor([0, 1, 77, (1 << 24) - 3, (1 << 24) - 2, (1 << 24) - 1, 1 << 24, (1 << 24) + 1, P - 2, P - 1], device=DEV)
    pieces = torch.zeros((P, 4), dtype=torch.int32, device=DEV)
    pieces[at] = few
    a, b = (ops.cache_write_(x, x + 1, ops.new_cache(10, 2, 64, block_tokens=16), p) for p in (few, pieces))
    assert a.k_scale.all() and all(torch.equal(s.view(torch.uint8), t.view(torch.uint8)) for s, t in zip(a, b))


def test_sizes_past_32_bits_are_refused():
    c = ops.new_cache(4, 2, 64, block_tokens=16)
    t, i = _i32([[0, 1]]), _i32([0])
    span, ring = torch.tensor([0, 4], device=DEV), _i32([0, 1, 2, 3])
    for n in ((1 << 30) + 1, (1 << 32) + 1):
        with pytest.raises(ValueError, match="n_rows"):
            ops.cache_rows_(i, i, t, ring, span, n)
    for n in (1 << 31, (1 << 32) + 1):
        with pytest.raises(ValueError, match="n_rows"):
            ops.cache_read(c, t, _i32([0, 4]), n_rows=n)
    with pytest.raises(ValueError, match="logits"):
        ops.sample_rows(torch.zeros(1, 4, device=DEV).expand((1 << 32) + 1, 4), torch.zeros(1, device=DEV))
    lmk = _i32(np.zeros((2, 1, 1, 2)))
    q = torch.zeros(1, 2, 64, device=DEV)
    a = ops.cache_attention(q, c, t, i, i, i, lmk)
    b = ops.cache_attention(q, c, t, i, i, i, lmk, w_max=1 << 40)  # (no window is longer than the table either)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_argument_checks():
    c = ops.new_cache(4, 2, 64, block_tokens=16)
    x = torch.zeros(3, 2, 64, device=DEV)
    q = torch.zeros(3, 4, 64, device=DEV)
    t, i = _i32([[0, 1]] * 3), _i32([0, 1, 2])
    lmk = _i32(np.zeros((4, 3, 1, 2)))
    pieces = _i32(np.zeros((3, 4)))
    good = dict(q=q, cache=c, table=t, req=i, pos=i, w=i, lmk_idx=lmk)
    ops.cache_attention(**good)
    for bad in (dict(q=torch.zeros(3, 4, 128, device=DEV)), dict(q=torch.zeros(3, 3, 64, device=DEV)), dict(table=t.long()),
                dict(table=t.t()), dict(req=i[:2]), dict(pos=i[None]), dict(w=i[:1]), dict(lmk_idx=lmk[:2]), dict(lmk_idx=lmk[:, :2]),
                dict(lmk_bias=torch.zeros(1, device=DEV)), dict(cache=c._replace(k=c.k.view(torch.uint8))),
                dict(cache=c._replace(v_scale=c.v_scale[:2])), dict(cache=c._replace(v=c.v.transpose(0, 1)))):
        with pytest.raises(ValueError):
            ops.cache_attention(**{**good, **bad})
    with pytest.raises(TypeError):
        ops.cache_attention(**{**good, "q": q.double()})
    with pytest.raises(RuntimeError):
        ops.cache_attention(**good, scale=-1.0)
    for k, v, p in ((x, x[:2], pieces), (x, x.half(), pieces), (x[:, :1], x[:, :1], pieces), (x, x, pieces[:, :3]), (x, x, pieces.long())):
        with pytest.raises(ValueError):
            ops.cache_write_(k, v, c, p)
    span, ring = torch.tensor([0, 4], device=DEV), _i32([0, 1, 2, 3])
    for a in ((i[:2], i, t, ring, span, 3), (i, i, t.long(), ring, span, 3), (i, i, t, ring.long(), span, 3), (i, i, t, ring, span[:1], 3),
              (i, i, t, ring, span.int(), 3), (i, i, t, ring, span, -1)):
        with pytest.raises(ValueError):
            ops.cache_rows_(*a, block_tokens=16)
    with pytest.raises(ValueError):
        ops.cache_rows_(i, i, t, ring, span, 3, block_tokens=20)
    with pytest.raises(ValueError):
        ops.cache_read(c, t, i, n_rows=2)
    with pytest.raises(TypeError):
        ops.cache_read(c, t, _i32([0, 1, 2, 3]), n_rows=2, dtype=torch.float64)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,G", [(2, 2), (8, 2)])
def test_calls_without_rows(D, H, G):
    """No query tokens, none written, none read, whatever the table and the windows hold: outputs without rows, pages as
    they were."""
    bt = 64
    cache = _random_cache(4, G, bt, D, 3)
    before = _host_pages(cache)
    none, x = _i32([]), torch.zeros(0, H, D, dtype=torch.bfloat16, device=DEV)
    for M in (2, 40, 4096):
        table, lmk = torch.zeros(3, M, dtype=torch.int32, device=DEV), torch.zeros(H, 3, 1, 8, dtype=torch.int32, device=DEV)
        for w_max in (None, 1, 512, M * bt, 1 << 40):
            for sets in (lmk, lmk[..., :0]):
                out, lse = ops.cache_attention(x, cache, table, none, none, none, sets, w_max=w_max)
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


def test_split_windows_on_two_streams_at_once(monkeypatch):
    """Windows split over blocks and joined from a workspace (key/value heads with their query heads, and heads one by one),
    with inputs of their own on each of two streams in turn: equal to the same calls one after the other."""
    need = []
    place = ops._set_workspace
    monkeypatch.setattr(ops, "_set_workspace", lambda a, n, dev: need.append(n) or place(a, n, dev))

    def case(seed, H, G, n, w):
        c = _attend_case(1, H, G, 128, 64, 20, torch.bfloat16, seed, 0, 1, lens=[n])
        return c[0].to(DEV), c[1], *(_i32(x) for x in c[2:5]), _i32([w]), _i32(c[6])
    cases = [[case(10 * i, 32, 2, 12000 + i, 9000), case(10 * i + 1, 2, 2, 3001 + i, 2900)] for i in range(2)]

    def work(i):
        return [t for c, w in zip(cases[i], (9000, 2900)) for t in ops.cache_attention(*c, w_max=w)]
    ref = [work(i) for i in range(2)]
    assert all(n > 0 for n in need) and len(need) == 4
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
    """Two captured calls whose windows are split, replayed in turn on two streams with inputs of the moment: each equals its
    eager call every time."""
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
        for a, b in zip(outs, ref):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]), rep
