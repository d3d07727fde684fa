"""Sampling of rows of logits on the GPU against the float64 oracle: tokens are equal, log probabilities within a
float32 rounding of sums that are exact."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from dsalt_amd import ops
from oracle import decode as OD

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _check(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """x [R, V] on the device; the settings numbers or lists [R]."""
    R = x.shape[0]

    def dev(v, dt):
        return torch.tensor(v, dtype=dt, device=DEV) if isinstance(v, (list, np.ndarray)) else v
    tok, lp = ops.sample_rows(x, u, temperature=dev(temperature, torch.float32), top_k=dev(top_k, torch.int32),
                              top_p=dev(top_p, torch.float32), min_p=dev(min_p, torch.float32))
    assert tok.dtype == torch.int64 and lp.dtype == torch.float32 and tok.shape == lp.shape == (R,)
    xs, us = x.detach().cpu().double().numpy(), u.cpu().double().numpy()

    def at(v, r):
        v = v[r] if isinstance(v, (list, np.ndarray)) else v
        return float(np.float32(v))
    want = [OD.sample(xs[r], us[r], at(temperature, r), int(at(top_k, r)), at(top_p, r), at(min_p, r)) for r in range(R)]
    assert tok.tolist() == [w[0] for w in want]
    wl = np.array([w[1] for w in want])
    got = lp.cpu().double().numpy()
    fin = np.isfinite(wl)
    assert np.array_equal(np.isneginf(got), ~fin) and (np.abs(got[fin] - wl[fin]) <= 2.0 ** -23 * np.abs(wl[fin]) + 1e-11).all()
    return tok


def _logits(R, V, dt, seed, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, V, generator=g) * spread
    x.scatter_add_(1, torch.randint(0, V, (R, 20), generator=g), torch.rand(R, 20, generator=g) * 12)
    return x.to(dt).to(DEV), torch.rand(R, generator=g).to(DEV)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("V", [1, 2, 7, 64, 513, 1003, 8192, 50257])
def test_settings_over_vocabularies(dt, V):
    x, u = _logits(5, V, dt, V)
    for kw in (dict(), dict(top_k=1), dict(top_k=5), dict(top_k=max(1, V - 1)), dict(top_k=V), dict(top_k=V + 9), dict(top_k=-3),
               dict(top_p=0.9), dict(top_p=0.3), dict(top_p=1e-9), dict(min_p=0.1), dict(top_k=40, top_p=0.9, min_p=0.05),
               dict(temperature=0.2, top_p=0.99), dict(temperature=7.0, top_p=0.95), dict(temperature=0.0), dict(top_k=1500, top_p=0.5)):
        _check(x, u, **kw)


@pytest.mark.parametrize("dt", TYPES)
def test_settings_of_each_row(dt):
    R, V = 64, 20011
    x, u = _logits(R, V, dt, 4)
    r = np.random.RandomState(0)
    _check(x, u, temperature=list(r.choice([0.0, -1.0, 0.3, 1.0, 2.5, float("nan"), float("inf")], R)),
           top_k=[int(k) for k in r.choice([0, 1, 2, 50, 1000, 5000, 30000, -1], R)],
           top_p=list(r.choice([1.0, 0.95, 0.5, 0.0, 2.0, float("nan")], R)), min_p=list(r.choice([0.0, 0.02, 0.5, 1.0, 1.5, float("nan")], R)))


@pytest.mark.parametrize("dt", TYPES)
def test_ties_go_to_the_lowest_index(dt):
    """All logits equal, few distinct values, and a tie across the end of each prefix."""
    V = 4099
    same = torch.zeros(4, V, dtype=dt, device=DEV)
    u = torch.tensor([0.0, 0.25, 0.5, 0.999], device=DEV)
    for kw in (dict(), dict(top_k=3), dict(top_k=1000), dict(top_p=0.5), dict(top_p=0.1, top_k=2000), dict(min_p=1.0)):
        _check(same, u, **kw)
    g = torch.Generator().manual_seed(0)
    few = torch.randint(-2, 3, (6, V), generator=g).to(dt).to(DEV)
    few[:, 11] = -0.0
    u = torch.rand(6, generator=g).to(DEV)
    for kw in (dict(top_k=10), dict(top_k=900), dict(top_k=2900), dict(top_p=0.7), dict(top_p=0.5, top_k=900), dict(top_p=0.93),
               dict(min_p=0.3), dict(top_p=0.2, min_p=0.9)):
        _check(few, u, **kw)


@pytest.mark.parametrize("dt", TYPES)
def test_masks_infinities_and_nan(dt):
    V = 777
    x, _ = _logits(8, V, dt, 2)
    low = torch.finfo(dt).min
    x[0] = float("-inf")
    x[1] = float("nan")
    x[2, 5:] = float("-inf")
    x[3, ::2] = low
    x[4, ::3] = float("nan")
    x[5] = low
    x[6, 40], x[6, 50] = float("inf"), float("inf")
    x[7, 1:] = float("-inf")
    u = torch.tensor([0.5, 0.5, 0.9, 0.7, 0.2, 0.6, 0.8, 0.99], device=DEV)
    for kw in (dict(), dict(top_k=3), dict(top_k=600), dict(top_p=0.8), dict(min_p=0.2), dict(temperature=0.0), dict(temperature=1e-30),
               dict(temperature=float("inf")), dict(top_k=700, top_p=0.9, min_p=0.01)):
        tok = _check(x, u, **kw)
        assert tok[0] == -1 and tok[1] == -1 and tok[6] in (40, 50) and tok[7] == 0


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("V", [2500, 16383, 16384])
def test_masked_rows_of_longer_vocabularies(dt, V):
    """Most of a row masked, by -inf, NaN or the type's lowest value, or beside infinite logits; rows past a list's length and
    on both sides of the weights by value."""
    x, u = _logits(6, V, dt, V)
    x[0, 5:] = float("-inf")
    x[1, ::2] = torch.finfo(dt).min
    x[2, 7:] = float("nan")
    x[3, ::3] = float("inf")
    x[4] = torch.finfo(dt).min
    for kw in (dict(), dict(top_p=0.8), dict(top_k=1500), dict(top_k=1500, top_p=0.6), dict(min_p=0.1), dict(top_k=30, top_p=0.9),
               dict(temperature=3.0, top_p=0.95), dict(temperature=float("inf"), top_p=0.3)):
        _check(x, u, **kw)


def test_random_numbers_at_the_ends():
    x, _ = _logits(9, 3001, torch.float32, 3)
    for dt in (torch.float32, torch.float64):
        u = torch.tensor([0.0, 1e-300, 1 - 2.0 ** -24, 1 - 2.0 ** -53, 1.0, 1.5, -0.5, float("nan"), 0.5], dtype=torch.float64).to(dt).to(DEV)
        for kw in (dict(), dict(top_k=7), dict(top_p=0.9), dict(min_p=0.05)):
            _check(x, u, **kw)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("V", [2005, 9001])
def test_layouts(dt, V):
    """Rows off 16-byte boundaries, columns of a wider buffer, a transposed buffer, rows that repeat."""
    x, u = _logits(6, V, dt, 9)
    ref = _check(x, u, top_p=0.9)
    wide = torch.zeros(6, V + 72, dtype=dt, device=DEV)
    for off in range(1, 9):
        y = wide[:, off:off + V]
        y.copy_(x)
        wide[:, :off], wide[:, off + V:] = 1e4, 1e4  # what lies beside a row is not its own
        assert torch.equal(_check(y, u, top_p=0.9), ref)
        _check(y, u)
        _check(y, u, top_k=30, min_p=0.01)
    assert torch.equal(_check(x.t().contiguous().t(), u, top_p=0.9), ref)
    _check(x[:1].expand(6, -1), u, top_k=50)


@pytest.mark.parametrize("dt", TYPES)
def test_largest_logit_off_16_byte_boundaries(dt):
    """The largest logit first, last, in the first few places and several times, rows from every offset."""
    for V in (1, 3, 9, 700, 5003):
        for off in range(1, 9):
            buf = torch.full((7, V + 16), 9.0, dtype=dt, device=DEV)
            x = buf[:, off:off + V]
            x.copy_(torch.randn(7, V).to(dt))
            x[1, 0] = x[2, V - 1] = x[3, min(2, V - 1)] = 8.0
            x[4, V // 2], x[4, V - 1] = 7.0, 7.0
            x[5] = -0.0
            x[5, V // 3:] = 0.0
            u = torch.full((7,), 0.5, device=DEV)
            _check(x, u, temperature=0.0)
            _check(x, u, top_k=1)
            _check(x, u, top_k=2, top_p=0.5)


@pytest.mark.parametrize("dt,V", [(torch.float32, 1 << 20), (torch.bfloat16, 1 << 20), (torch.bfloat16, 151936), (torch.float16, 262144)])
def test_large_vocabularies(dt, V):
    x, u = _logits(3, V, dt, 1)
    x[2] = 1.0  # sums as large as they get
    for kw in (dict(), dict(top_k=50, top_p=0.95), dict(top_p=0.95), dict(top_k=V // 2), dict(min_p=1e-4), dict(temperature=30.0, top_p=0.9)):
        _check(x, u, **kw)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("V", [2047, 2048, 2049, 8191, 8193, 20011])
def test_each_side_of_the_size_rules(dt, V):
    """Rows that are listed whole, searched, and (bfloat16 from 8192 on) weighed by value; lists of up to 256, 1024 and
    2048 tokens, and more than they hold; flat and peaked rows."""
    for spread in (0.02, 2.5, 12.0):
        x, u = _logits(4, V, dt, V, spread)
        for kw in (dict(), dict(top_p=0.9), dict(top_p=0.5, min_p=0.001), dict(top_k=200), dict(top_k=700, top_p=0.999), dict(top_k=1024),
                   dict(top_k=1025, top_p=0.7), dict(temperature=0.1, top_p=0.95), dict(temperature=20.0, top_p=0.3)):
            _check(x, u, **kw)


def test_bfloat16_values_on_both_sides_of_zero():
    """What the weights by value treat apart: zeros of both signs, subnormals and small magnitudes (most of the
    row, and where a prefix ends), all logits negative, all positive, magnitudes up to the largest."""
    V = 10007
    g = torch.Generator().manual_seed(0)
    tiny = torch.randn(V, generator=g) * 1e-30
    rows = [torch.zeros(V), tiny, torch.where(torch.rand(V, generator=g) < 0.7, torch.zeros(V), torch.randn(V, generator=g)),
            -torch.rand(V, generator=g) * 20 - 3, torch.rand(V, generator=g) * 5 + 40, torch.randn(V, generator=g) * 1e-3,
            torch.randn(V, generator=g) * 1e37, torch.full((V,), -0.0), torch.randn(V, generator=g).abs() * 1e-6 - 25]
    x = torch.stack(rows).to(torch.bfloat16)
    x[:, ::997] = torch.finfo(torch.bfloat16).min
    x[5, 13], x[8, 77], x[2, 5] = 0.0, 3e-7, float("nan")
    x = x.to(DEV)
    u = torch.rand(len(rows), generator=g).to(DEV)
    for kw in (dict(), dict(top_p=0.6), dict(top_p=0.97), dict(top_k=3000), dict(top_k=5000, top_p=0.5), dict(top_k=9999), dict(min_p=0.5),
               dict(temperature=1e-4, top_p=0.9), dict(temperature=1e30, top_p=0.9), dict(temperature=1e-38), dict(top_k=64, top_p=0.9)):
        _check(x, u, **kw)


@pytest.mark.parametrize("dt", TYPES)
def test_prefixes_that_end_near_zero(dt):
    """Logits even over [-1000, 1000] at temperature 1000: prefixes end at logits about 0, where those are closest to each
    other beside the largest."""
    V = 30011
    g = torch.Generator().manual_seed(2)
    x = (torch.rand(24, V, generator=g) * 2000 - 1000).to(dt).to(DEV)
    x[::2, ::3] *= 1e-5
    u = torch.rand(24, generator=g).to(DEV)
    for p in (np.linspace(0.725, 0.737, 24), np.linspace(0.62, 0.83, 24)):
        _check(x, u, temperature=1000.0, top_p=list(p))
    _check(x, u, temperature=1000.0, top_k=[int(k) for k in np.linspace(9000, 21000, 24)])
    _check(x, u, temperature=1000.0, top_k=[int(k) for k in np.linspace(1025, 2100, 24)], top_p=0.95, min_p=0.3)


def test_draws_follow_the_probabilities():
    """65536 rows of one distribution, u an even grid: counts are the probabilities to one part of the grid a token."""
    n = 1 << 16
    x = torch.tensor([[0.3, -1.0, 2.0, 0.0, -40.0, 1.1, 0.9]]).to(DEV)
    u = (torch.arange(n, device=DEV, dtype=torch.float64) + 0.5) / n
    tok, lp = ops.sample_rows(x.expand(n, -1), u, temperature=0.7)
    p = torch.softmax(x[0].double() / 0.7, 0)
    assert (torch.bincount(tok, minlength=7).double() / n - p).abs().max() <= 1.01 / n
    assert torch.allclose(lp.double(), torch.log(p)[tok], atol=1e-6)


def test_more_rows_than_a_launch_holds():
    """Rows that repeat, each with settings of its own."""
    n, R = 64, (1 << 22) + 70
    x, u = _logits(n, 5, torch.float32, 6)
    r = np.random.RandomState(1)
    s = [torch.tensor(v, dtype=dt, device=DEV) for v, dt in ((r.rand(n) * 2, torch.float32), (r.randint(0, 6, n), torch.int32),
                                                             (r.rand(n) * 1.2, torch.float32), (r.rand(n) * 0.4, torch.float32))]
    turn = torch.arange(R, device=DEV) % n
    for un in (u, u.double()):
        ref = ops.sample_rows(x, un, temperature=s[0], top_k=s[1], top_p=s[2], min_p=s[3])
        got = ops.sample_rows(x[turn], un[turn], **dict(zip(("temperature", "top_k", "top_p", "min_p"), (v[turn] for v in s))))
        assert all(torch.equal(a, b[turn]) for a, b in zip(got, ref))


def test_argument_checks():
    x, u = torch.zeros(3, 5, device=DEV), torch.zeros(3, device=DEV)
    for a in ((x[0], u), (x, u[:2]), (x[:, :0], u)):
        with pytest.raises(ValueError):
            ops.sample_rows(*a)
    for kw in (dict(temperature=u[:2]), dict(top_k=torch.zeros(1, dtype=torch.int32, device=DEV)), dict(top_p=u[None])):
        with pytest.raises(ValueError):
            ops.sample_rows(x, u, **kw)
    for a in ((x.double(), u), (x, u.half()), (x, u.long())):
        with pytest.raises(TypeError):
            ops.sample_rows(*a)
    tok, lp = ops.sample_rows(x[:0], u[:0])
    assert tok.shape == lp.shape == (0,)
    big = torch.tensor([1 << 40] * 3, device=DEV)
    assert torch.equal(ops.sample_rows(x, u, top_k=big)[0], ops.sample_rows(x, u, top_k=1 << 40)[0])


@pytest.mark.parametrize("dt", [torch.uint8, torch.int8, torch.int16, torch.uint16, torch.int64, torch.float16, torch.float32, torch.bool])
def test_counts_of_every_type(dt):
    """top_k as a tensor of another type than int32 draws what the same numbers draw in it."""
    x, u = _logits(6, 3001, torch.bfloat16, 12)
    k = torch.tensor([1, 0, 1, 1, 0, 1] if dt == torch.bool else [1, 0, 3, 50, 100, 127], dtype=torch.int32, device=DEV)
    ref = ops.sample_rows(x, u, top_k=k)
    got = ops.sample_rows(x, u, top_k=k.to(dt))
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("V", [2049, 2500, 16383, 16384, 16385])
def test_weights_by_value_on_each_side_of_their_rule(dt, V):
    """bfloat16 rows are weighed by value from 16384 columns on, and with filters from where a row is longer than a list
    (2048): flat and peaked rows of lengths beside both, with settings that reach the one and the other."""
    for spread in (0.02, 2.5, 12.0):
        x, u = _logits(4, V, dt, V, spread)
        for kw in (dict(), dict(temperature=0.3), dict(min_p=0.01), dict(top_p=0.9), dict(top_k=1025), dict(top_k=2000, top_p=0.7),
                   dict(temperature=20.0, top_p=0.3, min_p=0.2)):
            _check(x, u, **kw)
