"""Moves of more pages than one launch has threads for."""
import numpy as np
import pytest

from paged_ref import to_bits
from tang_amd import capi

pytestmark = pytest.mark.gpu

F16 = capi.F16


def _rows(cache, s, start, n):
    return [b.to_numpy().reshape(n, 8) for b in cache.seq_read(s, 0, start, n)]


def test_two_to_the_24_pages(dev):
    """The longest sequence, 2^28 positions in 2^24 pages behind as many vacant ones: compaction copies all its pages, a selection in
    reverse order gathers all its rows (2^32 threads each in one launch would be too many)."""
    own = capi.HipComputeDevice(0)  # its workspaces go with it
    n = 1 << 28
    cache = own.kv_cache(1, 1, 8, 16, 2 << 24, 2, n, F16)
    batch = cache.batch(1, 40, 1)
    gap, s = cache.seq_create(2)
    cache.seq_resize(gap, n)
    rng = np.random.default_rng(24)
    parts = {}
    for at, m in ((0, 40), ((1 << 27) - 9, 23), (n - 37, 37)):  # the start, around the middle (where the second slice begins), the end
        cache.seq_resize(s, at)
        batch.begin([s], [m])
        k, v = (to_bits(rng.standard_normal((m, 8), dtype=np.float32), F16) for _ in range(2))
        batch.append(0, None, own.upload(k, F16), own.upload(v, F16), None)
        parts[at] = k, v

    def check(reverse):
        for at, rows in parts.items():
            m = len(rows[0])
            got = _rows(cache, s, n - at - m if reverse else at, m)
            for x, y in zip(got, rows):
                assert np.array_equal(x[::-1] if reverse else x, y), (at, reverse)

    check(False)
    cache.seq_free([gap])
    assert cache.compact() == 1 << 24
    check(False)
    cache.seq_select(s, np.arange(n - 1, -1, -1, dtype=np.uint32))
    check(True)
    assert cache.info() == (1 << 24, 1)
    batch.free()
    cache.free()
    own.close()
