"""The bounds that the paged attention's results are held to see work that is left out: on the statement itself, in 64 bits."""
import numpy as np
import pytest

from paged_ref import attention, attention_bounds, rounded
from tang_amd import capi

F32, F16, BF16 = capi.F32, capi.F16, capi.BF16


def _inputs(KH, G, D, n, rows, qdt, cdt):
    rng = np.random.default_rng(n)
    q = rounded(rng.standard_normal((rows, KH * G, D), dtype=np.float32), qdt)
    k, v = (rounded(rng.standard_normal((n, KH, D), dtype=np.float32), cdt) for _ in range(2))
    return q, k, v, np.arange(n - rows, n)


def _without(q, k, v, pos, drop, window=0, sinks=0):
    """The statement with the keys of a range left out of every row."""
    keep = np.ones(len(k), bool)
    keep[drop] = False
    out = []
    for i, p in enumerate(pos):
        j = np.arange(len(k))
        ok = keep & (j <= p) & ((j > p - window) | (j < sinks) if window else True)
        out.append(attention(q[i:i + 1], k[ok], v[ok], [len(k)]))
    return np.concatenate(out)


@pytest.mark.parametrize("qdt,cdt,odt", [(F32, F16, F32), (F16, F16, F16), (BF16, BF16, BF16), (F32, BF16, F32), (BF16, F16, BF16)])
@pytest.mark.parametrize("KH,G,D,n", [(1, 1, 64, 9001), (2, 4, 128, 5001), (1, 2, 256, 2503), (1, 8, 128, 3570)])
def test_missing_work_is_seen(qdt, cdt, odt, KH, G, D, n):
    args = _inputs(KH, G, D, n, 3, qdt, cdt)

    def seen(off, window=0, sinks=0):
        return (np.abs(off - attention(*args, window, sinks)) > attention_bounds(*args, qdt, cdt, odt, window, sinks)).any()

    assert not seen(rounded(attention(*args), odt))
    for at in (0, n // 2, n - 300):
        assert seen(_without(*args, slice(at, at + 256)))          # a piece of 256 keys
        assert seen(_without(*args, slice(at, at + 16)))           # and one of 16
    assert seen(0.0 * attention(*args))
    assert seen(attention(*args, 2000, 0), 2000, 4)                # the sinks are forgotten
    for window in (1984, 2016):                                    # a window that is too short or too long
        assert seen(attention(*args, window, 4), 2000, 4)
    assert seen(attention(*args, 2000, 4))                         # or not looked at
