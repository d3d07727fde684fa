"""Verification of drafted tokens on the GPU against the float64 oracle: tokens and counts are whole numbers and equal."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from dsalt_amd import ops
from oracle import decode4 as O4

pytestmark = pytest.mark.gpu
DEV = "cuda"


def f64(t):
    return t.detach().cpu().double().numpy()


def _case(lens, V, dt, seed, noise=0.7, size=2.2):
    """Rows of requests of lens[r] rows each, drafts drawn from the draft's logits."""
    g = torch.Generator().manual_seed(seed)
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    T, R = cu[-1], len(lens)
    x = torch.randn(T, V, generator=g) * size
    y = (x + noise * torch.randn(T, V, generator=g)).to(dt)
    x = x.to(dt)
    drawn = torch.multinomial(torch.softmax(y.float(), 1), 1, generator=g)[:, 0] if T else torch.zeros(0, dtype=torch.int64)
    tok = torch.cat([torch.zeros(1, dtype=torch.int64), drawn[:-1]]) if T else drawn
    return x, tok, cu, torch.rand(T, generator=g), torch.rand(R, generator=g), y


def _check(x, tok, cu, u, v, y, temperature=1.0, draft_temperature=None, pad=0):
    R, T = len(cu) - 1, x.shape[0]
    per = [t if t is None or not isinstance(t, (list, np.ndarray)) else torch.tensor(t, dtype=torch.float32, device=DEV)
           for t in (temperature, draft_temperature)]
    got = ops.verify_rows(x.to(DEV), tok.to(DEV), torch.tensor(cu, device=DEV), u.to(DEV), v.to(DEV),
                          draft_logits=y if y is None else y.to(DEV), temperature=per[0], draft_temperature=per[1])
    t = f64(torch.as_tensor(temperature, dtype=torch.float32).expand(R))
    d = t if draft_temperature is None else f64(torch.as_tensor(draft_temperature, dtype=torch.float32).expand(R))
    ra, rt = O4.verify(f64(x), tok.tolist(), cu, u.tolist(), v.tolist(), None if y is None else f64(y), t, d)
    assert got.accepted.dtype == torch.int32 and got.tokens.dtype == torch.int64
    assert got.accepted.tolist() == ra and got.tokens.tolist() == rt
    return ra, rt


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [1, 2, 7, 64, 1000, 1003, 4096, 50257])
def test_follows_the_oracle(dt, V):
    lens = [5, 1, 2, 9, 1, 4, 3, 6]
    x, tok, cu, u, v, y = _case(lens, V, dt, V)
    temps = [1.0, 0.7, 0.0, 1.5, 2.0, 0.4, -1.0, 1.0]
    for draft in (y, None):
        a, _ = _check(x, tok, cu, u, v, draft, temps)
        _check(x, tok, cu, u, v, draft)
        _check(x, tok, cu, u.double(), v.double(), draft, 0.8, temps[::-1])
    if V > 1:
        assert 0 < sum(_check(x, tok, cu, u * 0.2, v, y)[0])


@pytest.mark.parametrize("n", [1, 2, 3, 300, 1100])
def test_runs_of_many_drafts(n):
    """A request of many drafts, all of them taken, and one refused at each end."""
    V = 257
    x, tok, cu, u, v, y = _case([n, n], V, torch.float32, n)
    assert _check(x, tok, cu, torch.zeros_like(u), v, y)[0] == [n - 1, n - 1]
    u = torch.zeros_like(u)
    if n > 1:
        u[0], u[cu[2] - 2] = 0.999999, 0.999999
    _check(x, tok, cu, u, v, y * 0.1)
    _check(x, tok, cu, u, v, None)


def test_one_row_split_over_many_blocks():
    for V, dt in ((151936, torch.bfloat16), (200003, torch.float32), (1 << 20, torch.float16)):
        x, tok, cu, u, v, y = _case([3], V, dt, 5)
        _check(x, tok, cu, u, v, y, 0.9)
        _check(x, tok, cu, u * 1e-9, v, y, 0.9)
        _check(x, tok, cu, u, v, None, 0.9)


@pytest.mark.parametrize("rows", [8, 15, 16, 20])
def test_largest_vocabulary_in_few_rows(rows):
    """Rows in as many parts as they are ever cut into, with most of the weight behind the first parts."""
    V = 1 << 20
    x, tok, cu, u, v, _ = _case([rows // 2, rows - rows // 2 - 1, 1], V, torch.bfloat16, rows)
    x[:, V - V // 8:] += 4
    tok[1] = V - 3
    _check(x, tok, cu, u * 1e-7, v, None)
    _check(x, tok, cu, u, torch.full_like(v, 0.03), None)


def test_infinities_nan_and_empty_rows():
    V = 40
    x, tok, cu, u, v, y = _case([2] * 10, V, torch.float32, 3)
    inf, nan = float("inf"), float("nan")
    x[0, 3] = x[0, 9] = inf                 # the two largest weigh alike, the rest nothing
    x[2, :] = -inf                          # no probability at all: the draft is refused, no token follows
    x[4, :] = nan
    x[4, 7] = 1.0                           # one token alone
    y[6, :] = -inf                          # a draft without probabilities
    y[8, 5] = inf
    y[8, 6] = nan
    x[10] = -inf
    x[10, 11] = -3.4e38                     # the lowest value is a logit
    x[12] = -3.4e38                         # and weighs like its equals
    x[15] = -inf                            # the last row of a request
    tok[1], tok[9], tok[17], tok[19] = 9, 5, -5, V  # two drafts outside the vocabulary
    u[14] = 0
    for draft in (y, None):
        for temps in (1.0, 0.0):
            a, t = _check(x, tok, cu, u, v, draft, temps)
            assert t[2] == -1 and a[1] == 0
    _check(x, tok, cu, torch.full_like(u, nan), torch.full_like(v, nan), y)
    _check(x, tok, cu, u - 2, v - 2, y)
    _check(x, tok, cu, u + 1, v + 1, y)
    _check(x, tok, cu, u, v, y, inf)
    _check(x, tok, cu, u, v, y, 1e-30)


def test_draft_equal_to_the_target():
    """q = p: every draft is taken; one it cannot hold is refused, and the token then comes from p, of which nothing is left."""
    x, tok, cu, u, v, _ = _case([6, 6], 500, torch.bfloat16, 9, noise=0.0)
    assert _check(x, tok, cu, u, v, x)[0] == [5, 5]
    x[2, 17] = float("-inf")
    tok[3] = 17
    assert _check(x, tok, cu, u, v, x)[0] == [2, 5]


def test_greedy_takes_the_largest():
    x, tok, cu, u, v, y = _case([4, 4, 4], 300, torch.bfloat16, 2)
    x[:, 100] = x[:, 20] = 60.0  # two largest: the first
    tok[1], tok[2], tok[3] = 20, 20, 100
    a, t = _check(x, tok, cu, u, v, y, 0.0, 1.0)
    assert a[0] == 2 and t[:4] == [20, 20, 20, -1]
    a, t = _check(x, tok, cu, u, v, None, 0.0)
    assert a[0] == 2 and t[:4] == [20, 20, 20, -1]


def test_offsets_that_leave_rows_out():
    """Rows before the first request, behind the last and of requests without any, offsets past the rows."""
    x, tok, _, u, v, y = _case([10, 1], 33, torch.float32, 4)
    x, tok, u, y = x[:10], tok[:10], u[:10], y[:10]
    for cu in ([2, 5], [0, 0, 0, 4, 4, 9], [10, 10], [0, 3, 10]):
        _check(x, tok, cu, u, torch.rand(len(cu) - 1), y)
    wide = ops.verify_rows(x.to(DEV), tok.to(DEV), torch.tensor([0, 4, 25], device=DEV), u.to(DEV), v.to(DEV), draft_logits=y.to(DEV))
    ref = ops.verify_rows(x.to(DEV), tok.to(DEV), torch.tensor([0, 4, 10], device=DEV), u.to(DEV), v.to(DEV), draft_logits=y.to(DEV))
    assert torch.equal(wide.accepted, ref.accepted) and torch.equal(wide.tokens, ref.tokens)
    for T, cu in ((0, [0]), (0, [0, 0, 0]), (4, [0])):
        got = ops.verify_rows(x[:T].to(DEV), tok[:T].to(DEV), torch.tensor(cu, device=DEV), u[:T].to(DEV), torch.zeros(len(cu) - 1, device=DEV))
        assert got.accepted.tolist() == [0] * (len(cu) - 1) and got.tokens.tolist() == [-1] * T


def test_strides_and_alignments():
    """Rows off 16-byte boundaries, the draft's elsewhere than the target's, columns of a wider tensor, column-major logits."""
    for dt in (torch.bfloat16, torch.float32):
        x, tok, cu, u, v, y = _case([4, 3, 5], 1001, dt, 6)
        ref = _check(x, tok, cu, u, v, y, 0.9)
        a = (tok.to(DEV), torch.tensor(cu, device=DEV), u.to(DEV), v.to(DEV))
        for off, pad in ((0, 7), (1, 0), (3, 5)):
            for off2 in (0, 1, 2):
                bx, by = (torch.full((12, 1001 + 8 + pad), float("inf"), dtype=dt, device=DEV) for _ in range(2))
                bx[:, off:off + 1001], by[:, off2:off2 + 1001] = x.to(DEV), y.to(DEV)
                got = ops.verify_rows(bx[:, off:off + 1001], *a, draft_logits=by[:, off2:off2 + 1001], temperature=0.9)
                assert (got.accepted.tolist(), got.tokens.tolist()) == ref
        got = ops.verify_rows(x.to(DEV).T.contiguous().T, a[0].int(), a[1].long(), *a[2:], draft_logits=y.to(DEV).T.contiguous().T, temperature=0.9)
        assert (got.accepted.tolist(), got.tokens.tolist()) == ref


def test_two_streams_and_graphs():
    """Calls on two streams at once, and two captured ones replayed in turn, each with a workspace of its own."""
    cases = []
    for i in range(2):
        x, tok, cu, u, v, y = _case([5, 3, 4 + i], 30011, torch.bfloat16, i)
        cases.append([x.to(DEV), tok.to(DEV), torch.tensor(cu, device=DEV, dtype=torch.int32), u.to(DEV), v.to(DEV), y.to(DEV)])

    def work(i):
        *a, y = cases[i]
        return ops.verify_rows(*a, draft_logits=y, temperature=0.8)
    ref = [work(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    res = [[], []]
    for _ in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                res[i].append(work(i))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in range(2) for got in res[i] for a, b in zip(got, ref[i]))
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for i in range(2):
        with torch.cuda.graph(graphs[i]):
            outs.append(work(i))
    for rep in range(4):
        for c in cases:
            c[3].copy_(torch.rand_like(c[3]))
            c[4].copy_(torch.rand_like(c[4]))
        ref = [work(i) for i in range(2)]
        for o in outs:
            for t in o:
                t.fill_(-9)
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for o, r in zip(outs, ref) for a, b in zip(o, r)), rep
