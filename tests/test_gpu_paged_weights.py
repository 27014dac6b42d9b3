"""The weights of attention over the paged cache: what their rounding to 16 bits may cost."""
import numpy as np
import pytest

from paged_ref import EPS, rounded, to_bits
from tang_amd import capi
from test_gpu_paged import NAMES, Model, _normal

pytestmark = pytest.mark.gpu

F16, BF16 = capi.F16, capi.BF16


def _store(m, s, k, v):
    """Sequence s grows by these rows (values of the cache's type)."""
    m.begin([s], [len(k)])
    m.batch.append(0, None, m.dev.upload(to_bits(k, m.dt), m.dt), m.dev.upload(to_bits(v, m.dt), m.dt), None)
    m.rows[s] = np.concatenate((m.rows[s], np.stack((k, v))[None]), 2)


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
