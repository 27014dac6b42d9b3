"""The weights of attention over the paged cache: what their rounding to 16 bits may cost."""
import numpy as np
import pytest

from paged_ref import EPS, attention, attention_bounds, rounded, to_bits
from tang_amd import capi
from test_gpu_paged import NAMES, Model, _normal

pytestmark = pytest.mark.gpu

F16, BF16 = capi.F16, capi.BF16


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
