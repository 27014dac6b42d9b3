"""The weights of attention over the paged cache: what their rounding to 16 bits may cost, and bounds for every element that see
a piece of the work left out."""
import numpy as np
import pytest

from paged_ref import EPS, attention, attention_bounds, rounded, to_bits
from tang_amd import capi
from test_gpu_paged import NAMES, TYPES, Model, _normal

pytestmark = pytest.mark.gpu

F32, F16, BF16 = capi.F32, capi.F16, capi.BF16


def _store(m, s, k, v):
    """Sequence s grows by these rows (values of the cache's type)."""
    m.begin([s], [len(k)])
    m.batch.append(0, None, m.dev.upload(to_bits(k, m.dt), m.dt), m.dev.upload(to_bits(v, m.dt), m.dt), None)
    m.rows[s] = np.concatenate((m.rows[s], np.stack((k, v))[None]), 2)


def _scores(n, hd, first, others, rng, dt):
    """q [1][1][hd] and keys whose scores (times 1 / sqrt(hd)) are `first` for key 0 and `others` (n - 1 of them) for the rest."""
    q = np.zeros((1, 1, hd), np.float32)
    q[0, 0, 0] = np.sqrt(hd)
    k = rounded(_normal(rng, n, 1, hd), dt)  # the other dims do not matter
    k[:, 0, 0] = rounded(np.r_[first, others].astype(np.float32), dt)
    return q, k


@pytest.mark.parametrize("new,G", [(1, 1), (1, 16), (40, 1), (3, 8)])
@pytest.mark.parametrize("n,nats", [(8192, 17.0), (30000, 16.0), (30000, 17.0), (30000, 20.0)])
def test_many_small_weights_beside_a_large_one(dev, new, G, n, nats):
    """One key has most of the weight and a value of zero, thousands have a weight of e^-16 to e^-20 each, below f16's normal range
    and its last bit: the result is made up of theirs."""
    rng = np.random.default_rng(int(nats) + new)
    m = Model(dev, 1, 64, 16, n // 16 + 8, 1, 1, n + 64, F16, heads=G, rows=n)
    s = m.create()
    q, k = _scores(n, 64, 8.0, 8.0 - nats + 0.25 * rng.random(n - 1), rng, F16)
    v = rounded(0.5 + rng.random((n, 1, 64), np.float32), F16)
    v[0] = 0.0
    _store(m, s, k[:n - new], v[:n - new])
    _store(m, s, k[n - new:], v[n - new:])
    q = np.broadcast_to(q, (new, G, 64)) * np.float32(1.0)
    _, got = m.attend(rng, F16, F16, q=q, check=False)
    args = (q, k, v, np.arange(n - new, n))
    want = attention(*args)
    assert 0 < want.max() < 0.01
    assert (np.abs(got - want) <= attention_bounds(*args, F16, F16, F16, tiles=new * G > 16)).all()
    # and in one plain number: the result's rounding, that of weights that are subnormal beside 2^9 (2^-25 of at least 2^(9 - 29)), sums
    assert (np.abs(got - want) <= want * (EPS[F16] + 2.0 ** -5 if nats == 20.0 else 3 * EPS[F16] + 2.0 ** -8)).all()


@pytest.mark.parametrize("dt", [F16, BF16], ids=lambda t: NAMES[t])
@pytest.mark.parametrize("new,G,prefix", [(1, 1, 0), (1, 8, 0), (33, 1, 0), (200, 2, 0), (1, 1, 1), (1, 4, 1)])
def test_equal_values_give_that_value(dev, dt, new, G, prefix):
    """Weights that are all rounded down (a score whose weight lies just under the middle of two values) still add up to one.
    (prefix: 40 forks whose rows make up a tile)"""
    rng = np.random.default_rng(new)
    n, forks = 2000, 40 if prefix else 1
    m = Model(dev, 1, 64, 16, 600, 48, 1, 2600, dt, heads=G, rows=2048)
    s = m.create()
    w = 0.5 * (1.0 + 0.96 * EPS[dt])
    assert rounded(np.float32(w), dt) == 0.5
    q = np.zeros((1, 1, 64), np.float32)
    q[0, 0, 0] = 1.0
    k = rounded(_normal(rng, n, 1, 64), dt)
    k[:, 0, 0] = np.where(np.arange(n) % 32 == 0, 0.0, -1.0)  # a largest one in every block, all others of weight w
    one = np.ones((n, 1, 64), np.float32)
    _store(m, s, k[:n - new], one[:n - new])
    seqs = [s]
    if prefix:
        seqs = m.cache.seq_fork(s, forks)
        for c in seqs:
            m.rows[c] = m.rows[s].copy()
    m.begin(seqs, [new] * forks)
    d = [dev.upload(to_bits(np.concatenate([t[n - new:]] * forks), dt), dt) for t in (k, one)]
    m.batch.append(0, None, *d, None)
    q = np.broadcast_to(q, (new * forks, G, 64)) * np.float32(1.0)
    _, got = m.attend(rng, dt, dt, q=q, check=False, scale=-np.log(w))
    assert (got == 1.0).all(), (got.min(), got.max())


def _check(m, rng, qdt, odt, window=0, sinks=0):
    q, got = m.attend(rng, qdt, odt, window, sinks, check=False)
    at = 0
    for s, n in m.step:
        if n:
            k, v = m.rows[s][0]
            args = (q[at:at + n], k, v, np.arange(len(k) - n, len(k)))
            off = np.abs(got[at:at + n] - attention(*args, window, sinks))
            tol = attention_bounds(*args, qdt, m.dt, odt, window, sinks)
            assert (off <= tol).all(), (s, n, window, (off / tol).max())
        at += n


@pytest.mark.parametrize("qdt,cdt,odt", TYPES, ids=lambda t: NAMES[t])
@pytest.mark.parametrize("kh,G,hd,starts,news", [(1, 1, 64, [9000, 10], [1, 2]), (2, 4, 128, [5000, 300], [1, 1]), (1, 2, 256, [2500], [3]),
                                                 (1, 8, 128, [3500, 0], [70, 9]), (2, 4, 96, [700, 33, 90], [1, 150, 20])])
def test_every_element(dev, qdt, cdt, odt, kh, G, hd, starts, news):
    rng = np.random.default_rng(sum(starts))
    m = Model(dev, kh, hd, 16, 700, 4, 1, 10000, cdt, heads=kh * G, rows=9100)
    seqs = [m.create() for _ in starts]
    m.fill(rng, seqs, starts)
    m.fill(rng, seqs, news)
    for window, sinks in [(0, 0), (2000, 4), (300, 0)]:
        _check(m, rng, qdt, odt, window, sinks)


@pytest.mark.parametrize("qdt,cdt", [(F16, F16), (BF16, BF16), (F32, F16)], ids=lambda t: NAMES[t])
@pytest.mark.parametrize("G,prefix,n", [(4, 512, 7), (2, 3000, 24)])
def test_every_element_of_forks(dev, qdt, cdt, G, prefix, n):
    rng = np.random.default_rng(prefix)
    m = Model(dev, 1, 64, 16, 600, 30, 1, 4000, cdt, heads=G)
    first = m.create()
    m.fill(rng, [first], [prefix])
    seqs = m.cache.seq_fork(first, n)
    for s in seqs:
        m.rows[s] = m.rows[first].copy()
    m.fill(rng, seqs, [11 * i % 60 for i in range(n)])
    m.fill(rng, seqs, [1 + i % 3 for i in range(n)])
    _check(m, rng, qdt, qdt)
    _check(m, rng, qdt, qdt, 700, 5)


def test_sums_of_long_items_do_not_drift(dev):
    """20000 keys in one item, values between one and two: the mean of the signed errors of 67000 results. A sum that loses half a step of
    its 24 bits at each of 1250 steps of 16 keys is off by 2.7e-5. The f16 roundings of the results (2^-11 / sqrt(3) at
    most each) have a mean of 1.1e-6 in either direction, six times which is allowed, and 2^-20 for plain f32 sums."""
    rng = np.random.default_rng(3)
    m = Model(dev, 1, 64, 64, 400, 1, 1, 24000, F16, heads=2, rows=16000)
    s = m.create()
    for n in (16000, 4200):
        k, v = rounded(0.5 * _normal(rng, n, 1, 64), F16), rounded(1.0 + np.linspace(0.0, 0.9, 64, dtype=np.float32) + 0.125 * _normal(rng, n, 1, 64), F16)
        _store(m, s, k, v)
    q, got = m.attend(rng, F16, F16, check=False)
    k, v = m.rows[s][0]
    rows = np.arange(3, 4200, 8)
    want = attention(q[rows], k, v, 16000 + rows)
    off = (got[rows] - want) / want
    assert off.size > 67000 and abs(off.mean()) <= 6 * 1.1e-6 + 2.0 ** -20, off.mean()
