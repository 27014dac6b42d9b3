"""The choice of tokens from given random numbers, against its definition in 64
bits and against the host's sampler."""
import numpy as np
import pytest

from paged_ref import rounded, to_bits
from tang_amd import capi

pytestmark = pytest.mark.gpu

F32, F16, BF16 = capi.F32, capi.F16, capi.BF16


def kept(row, temp, k, p, low):
    """(indexes, weights) of the kept tokens of one row, by index."""
    row = np.where(np.isnan(row), -np.inf, row.astype(np.float64))
    seen = np.flatnonzero(row > -np.inf)
    seen = seen[np.lexsort((seen, -row[seen]))]
    top = row[seen[0]]
    if 0 < k < len(seen):
        seen = seen[row[seen] >= row[seen[k - 1]]]
    with np.errstate(all="ignore"):
        w = np.where(row[seen] == top, 1.0, np.exp((row[seen] - top) / temp))
    if p < 1:
        cum = np.cumsum(w)
        n = int(np.searchsorted(cum, p * cum[-1])) + 1 if p > 0 else 1
        seen, w = seen[:n], w[:n]
    if low > 0:
        seen, w = seen[w >= min(low, 1.0)], w[w >= min(low, 1.0)]
    at = np.argsort(seen)
    return seen[at], w[at]


def choose(row, u, temp, k, p, low):
    """(token, its share, how far u is from a border that would choose another)"""
    row = np.where(np.isnan(row), -np.inf, row)
    if not row.max() > -np.inf:
        return 0, 0.0, 1.0
    if not temp > 0:
        return int(np.flatnonzero(row == row.max())[0]), 1.0, 1.0
    seen, w = kept(row, temp, k, p, low)
    share = np.cumsum(w) / w.sum()
    at = min(int(np.searchsorted(share, u, side="right")), len(seen) - 1)
    return int(seen[at]), w[at] / w.sum(), np.abs(share[:-1] - u).min() if len(seen) > 1 else 1.0


def _run(dev, x, dt, u, temp=None, k=None, p=None, low=None):
    n, V = x.shape
    f = lambda v: None if v is None else dev.upload(np.asarray(v, np.float32))  # noqa: E731
    prob = dev.alloc(n)
    tokens = dev.sample_rows(dev.upload(to_bits(x, dt), dt), n, V, f(u), f(temp), None if k is None else dev.upload_u32(k), f(p), f(low), prob=prob)
    return tokens.to_numpy(), prob.to_numpy()


def _check(dev, x, dt, u, temp=None, k=None, p=None, low=None):
    """Tokens are equal; shares are within the f32 rounding of the result and of the sums (weights are held to
    2^-43 of the largest, 2^20 of them to 2^-23 of the sum at the very worst: 2^-22 in all)."""
    x = rounded(x, dt)
    got, prob = _run(dev, x, dt, u, temp, k, p, low)
    pick = lambda v, r, off: off if v is None else np.float32(v[r]).astype(np.float64)  # noqa: E731
    for r in range(len(x)):
        args = (float(np.float32(u[r])), float(pick(temp, r, 1.0)), 0 if k is None else int(k[r]), float(pick(p, r, 1.0)), float(pick(low, r, 0.0)))
        want, share, border = choose(x[r], *args)
        assert border > 1e-9, "the row's random number lies on a border"
        assert got[r] == want, (r, got[r], want, args, border)
        assert abs(prob[r] - share) <= share * 2.0 ** -22, (r, prob[r], share)
    return got


def _logits(rng, n, V, spread=2.0):
    x = rng.standard_normal((n, V)).astype(np.float32) * np.float32(spread)
    for r in x:
        r[rng.integers(0, V, min(V, 30))] += rng.uniform(0, 10, min(V, 30))
    return x


VOCABS = [1, 2, 7, 64, 65, 1000, 8192, 8193, 32000, 50001]


@pytest.mark.parametrize("V", VOCABS + [131072, 200003, 1 << 20])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_settings(dev, V, dt):
    """Rows of every mixture of settings."""
    rng = np.random.default_rng(V)
    n = 48 if V < 100000 else 16
    temp = np.where(rng.random(n) < 0.15, 0.0, rng.uniform(0.2, 2.5, n))
    k = np.where(rng.random(n) < 0.4, 0, np.exp(rng.uniform(0, np.log(V + 5), n))).astype(np.uint32)
    p = np.where(rng.random(n) < 0.4, 1.0, rng.uniform(0, 1, n))
    low = np.where(rng.random(n) < 0.5, 0.0, np.exp(rng.uniform(-9, 0, n)))
    _check(dev, _logits(rng, n, V), dt, rng.random(n, np.float32), temp, k, p, low)


@pytest.mark.parametrize("V", [1000, 32000, 50001])
@pytest.mark.parametrize("which", ["none", "temp", "k", "p", "low"])
def test_one_setting(dev, V, which):
    rng = np.random.default_rng(V + 1)
    n = 12
    over = dict(temp=dict(temp=rng.uniform(0.1, 3, n)), k=dict(k=np.array([1, 2, 5, 50, 63, 64, 65, 300, 900, V - 1, V, V + 1], np.uint32)),
                p=dict(p=np.linspace(0.01, 0.999, n)), low=dict(low=np.exp(np.linspace(-12, 0, n)))).get(which, {})
    _check(dev, _logits(rng, n, V), F32, rng.random(n, np.float32), **over)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("V", [511, 513, 8191, 16385, 32000])
def test_runs(dev, V, dt):
    """Top-p alone and with min-p, from runs of one to runs of nearly all: their ends and shares over every wave's part of a row."""
    rng = np.random.default_rng(V)
    n = 40
    u, temp, p = rng.random(n, dtype=np.float32), rng.uniform(0.3, 2.5, n), rng.uniform(0.3, 1, n)
    _check(dev, _logits(rng, n, V), dt, u, temp, None, p, np.where(rng.random(n) < 0.5, 0, rng.uniform(0, 0.05, n)))


@pytest.mark.parametrize("spread", [0.0, 1e-6, 1e-3, 0.05])
def test_rows_that_are_nearly_flat(dev, spread):
    """All weights in one bin: values a few steps of f32 apart, at a large and a small base."""
    rng = np.random.default_rng(7)
    n, V = 12, 40000
    for base in (0.0, 17.0):
        x = (base + spread * rng.standard_normal((n, V))).astype(np.float32)
        k = np.array([1, 40, 64, 65, 2000, 2049, 5000, 20000, 39999, 0, 0, 0], np.uint32)
        p = np.array([1, 1, 0.5, 0.9, 0.3, 1, 0.77, 0.51, 1, 0.013, 0.5001, 0.9999])
        _check(dev, x, F32, rng.random(n, np.float32), k=k, p=p)


@pytest.mark.parametrize("V", [100, 9000, 50000])
def test_equal_logits(dev, V):
    """A few distinct values: top-k keeps the equal ones, top-p the ones of lowest index."""
    rng = np.random.default_rng(V)
    n = 24
    x = rng.integers(0, 4, (n, V)).astype(np.float32)
    k = rng.integers(0, V, n).astype(np.uint32)
    p = np.where(rng.random(n) < 0.2, 1.0, rng.uniform(0.05, 1, n))
    got = _check(dev, x, BF16, rng.random(n, np.float32), k=k, p=p)
    assert len(set(got)) > n // 3
    # every half of a row of equal ones is the one in front
    got, _ = _run(dev, np.zeros((n, V), np.float32), F32, np.full(n, 0.999, np.float32), p=np.full(n, 0.5))
    assert np.all(got == int(0.999 * np.ceil(V / 2)))
    x = np.zeros((4, V), np.float32)
    x[:, ::2] = -0.0  # equal to 0
    got, _ = _run(dev, x, F32, [0.0, 0.3, 0.6, 0.999], temp=[0.0, 1.0, 1.0, 1.0], k=np.array([1, 1, 1, 1], np.uint32))
    assert list(got) == [0] + [int(np.float32(v) * V) for v in (0.3, 0.6, 0.999)]


def test_min_p_that_leaves_fewer_than_k(dev):
    """A k far beyond what min-p keeps, with and without top-p; a k in the middle of them."""
    rng = np.random.default_rng(13)
    n, V = 9, 40000
    x = _logits(rng, n, V, 1.0)
    for k in (3, 50, 5000, 39000):
        for low in (1.0, 0.5, 1e-3):
            for p in (None, np.full(n, 0.95)):
                _check(dev, x, F32, rng.random(n, np.float32), k=np.full(n, k, np.uint32), low=np.full(n, low), p=p)


@pytest.mark.parametrize("V", [5000, 33000, 70000])
def test_lists_that_are_full(dev, V):
    """Candidates about as many as a list holds (4096), one fewer, one more: by k, by p over equal ones, by min-p."""
    rng = np.random.default_rng(V)
    for m in (4095, 4096, 4097):
        x = np.full((3, V), -30.0, np.float32)
        for r in x:
            r[rng.permutation(V)[:m]] = rng.uniform(0, 0.001, m)
        u = rng.random(3, np.float32)
        _check(dev, x, F32, u, k=np.full(3, m, np.uint32))
        _check(dev, x, F32, u, k=np.full(3, 4000, np.uint32), p=np.full(3, 0.7))
        _check(dev, x, F32, u, p=np.full(3, 0.99))
        _check(dev, x, F32, u, low=np.full(3, 0.9))


def test_masked_and_infinite(dev):
    rng = np.random.default_rng(9)
    V = 9001
    x = np.full((12, V), -np.inf, np.float32)
    x[1, 77] = -5.0
    x[2, [3, 8000]] = 1.0
    x[3] = rng.standard_normal(V)
    x[3, rng.random(V) < 0.9] = -np.inf
    x[4] = np.nan
    x[5] = rng.standard_normal(V)
    x[5, ::3] = np.nan
    x[6] = rng.standard_normal(V)
    x[6, [5, 17]] = np.inf
    x[7] = -3e38
    x[7, 9] = 3e38
    x[8] = rng.standard_normal(V) * 1e-42
    x[9, 50] = np.finfo(np.float32).min  # the type's lowest beside what is masked
    x[10] = np.finfo(np.float32).min
    x[11] = rng.standard_normal(V)
    x[11, 1:] = np.nan
    u = np.array([0.5, 0.9, 0.7, 0.3, 0.2, 0.8, 0.6, 0.5, 0.4, 0.1, 0.25, 0.5], np.float32)
    for settings in (dict(), dict(k=np.full(12, 3, np.uint32)), dict(p=np.full(12, 0.9)), dict(low=np.full(12, 0.1)),
                     dict(temp=np.zeros(12)), dict(temp=np.full(12, 0.7), k=np.full(12, 100, np.uint32), p=np.full(12, 0.8), low=np.full(12, 0.01))):
        got = _check(dev, x, F32, u, **settings)
        assert got[0] == 0 and got[4] == 0 and got[1] == 77 and got[6] in (5, 17) and got[9] == 50 and got[7] == 9


def test_settings_at_their_ends(dev):
    rng = np.random.default_rng(10)
    V, n = 5000, 10
    x = _logits(rng, n, V)
    u = rng.random(n, np.float32)
    top = x.argmax(1)
    for t in (0.0, -1.0, np.nan, 1e-40, 1e-30):
        assert np.array_equal(_run(dev, x, F32, u, temp=np.full(n, t))[0], top)
    for settings in (dict(p=np.full(n, 0.0)), dict(p=np.full(n, -1.0)), dict(low=np.full(n, 1.0)), dict(low=np.full(n, 7.0)),
                     dict(k=np.ones(n, np.uint32))):
        assert np.array_equal(_run(dev, x, F32, u, **settings)[0], top)
    for t in (1e10, np.inf):  # all alike
        assert np.array_equal(_run(dev, x, F32, np.full(n, 0.3), temp=np.full(n, t))[0], np.full(n, int(np.float32(0.3) * V)))
    for settings in (dict(p=np.full(n, np.nan)), dict(p=np.full(n, 2.0)), dict(low=np.full(n, np.nan)), dict(low=np.full(n, -1.0)),
                     dict(k=np.full(n, 4294967295, np.uint32)), dict(k=np.zeros(n, np.uint32))):
        assert np.array_equal(_run(dev, x, F32, u, **settings)[0], _run(dev, x, F32, u)[0])
    # u at its ends and outside of them: the first and the last of the kept
    for k in (7, 4000):
        seen = [kept(r, 1.0, k, 1.0, 0.0)[0] for r in x]
        for v, at in ((0.0, 0), (-1.0, 0), (np.nan, 0), (1.0, -1), (5.0, -1), (np.inf, -1)):
            got = _run(dev, x, F32, np.full(n, v), k=np.full(n, k, np.uint32), low=np.full(n, 1e-12))[0]
            assert np.array_equal(got, [kept(r, 1.0, k, 1.0, 1e-12)[0][at] for r in x]), (k, v)


@pytest.mark.parametrize("V", [700, 9001])
def test_temperatures_below_the_normal_range(dev, V):
    """Logits and temperatures that are subnormal: bins are all one then, and the weights alone decide."""
    rng = np.random.default_rng(V)
    n = 20
    x, u = rng.standard_normal((n, V)).astype(np.float32) * np.float32(3e-42), rng.random(n, dtype=np.float32)
    temp = rng.uniform(1e-42, 3e-42, n)
    for settings in (dict(), dict(k=rng.integers(1, 300, n).astype(np.uint32)), dict(p=rng.uniform(0.3, 1, n)), dict(low=rng.uniform(0.01, 0.3, n)),
                     dict(k=rng.integers(1, 300, n).astype(np.uint32), p=rng.uniform(0.3, 1, n), low=rng.uniform(0, 0.1, n))):
        _check(dev, x, F32, u, temp=temp, **settings)


def test_no_rows(dev):
    tokens = dev.upload(np.array([9], np.uint32), capi.U32)
    dev.sample_rows(dev.alloc(1), 0, 5, dev.alloc(1), tokens=tokens)
    assert tokens.to_numpy()[0] == 9


@pytest.mark.parametrize("cfg", [dict(), dict(top_k=40), dict(top_p=0.9), dict(temperature=0.7, top_k=50, top_p=0.95), dict(temperature=0.0),
                                 dict(temperature=1.5, top_p=0.99)])
def test_as_the_host_samples(dev, cfg):
    """The tokens of th_sampler_sample (no min-p there) for the random numbers that its generator gives."""
    rng = np.random.default_rng(11)
    V, n = 3000, 40
    x = _logits(rng, n, V, 1.5)
    seeds = rng.integers(0, 1 << 62, n)
    r = [((int(s) * 6364136223846793005 + 1442695040888963407) % 2 ** 64 >> 11) / 2.0 ** 53 for s in seeds]
    u = np.array(r, np.float32)
    cfg = {k: float(np.float32(v)) if isinstance(v, float) else v for k, v in cfg.items()}
    host = [capi.Sampler(capi.SamplingConfig(**cfg), int(s)).sample(row) for s, row in zip(seeds, x)]
    got, _ = _run(dev, x, F32, u, np.full(n, cfg.get("temperature", 1.0)), np.full(n, cfg.get("top_k", 0), np.uint32), np.full(n, cfg.get("top_p", 1.0)))
    settings = (cfg.get("temperature", 1.0), cfg.get("top_k", 0), cfg.get("top_p", 1.0), 0.0)
    sure = [choose(row, float(a), *settings)[0] == choose(row, b, *settings)[0] for row, a, b in zip(x, u, r)]  # u is r in f32
    assert sum(sure) >= n - 1 and all(a == b for a, b, ok in zip(got, host, sure) if ok)


def test_captured(dev):
    """Replays on new logits and settings give the eager bits, with eager work between."""
    rng = np.random.default_rng(12)
    n, V = 6, 20000
    x, u, temp, p, prob = (dev.alloc(m) for m in (n * V, n, n, n, n))
    k, tokens = dev.alloc(n, capi.U32), dev.alloc(n, capi.U32)
    call = lambda: dev.sample_rows(x, n, V, u, temp, k, p, None, tokens, prob)  # noqa: E731

    def fill():
        x.upload(_logits(rng, n, V))
        for b, v in ((u, rng.random(n)), (temp, rng.uniform(0, 2, n)), (p, rng.uniform(0.5, 1.1, n)), (k, rng.integers(0, 3000, n))):
            b.upload(v)
    fill()
    call()
    graph = dev.capture(call)
    seen = []
    for _ in range(4):
        fill()
        call()
        want = tokens.to_numpy(), prob.to_numpy()
        dev.zero_buffer(prob)
        graph.launch()
        assert np.array_equal(tokens.to_numpy(), want[0]) and np.array_equal(prob.to_numpy(), want[1])
        seen.append(tuple(want[0]))
    assert len(set(seen)) == 4
    graph.free()


@pytest.mark.parametrize("V", [1000, 32000, 131072, 1 << 20])
@pytest.mark.parametrize("part", [1.2, 0.8, 0.0])
def test_small_weights_that_all_round_alike(dev, V, part):
    """One large weight and V - 1 of which each is 2^-part of the last place that weights are held to: all become none (1.2), twice
    as much as they nearly are (0.8), or what they are (0).  Running sums are off by half a last place for each weight, and by 2^-45 of
    themselves (a weight's exponent has three roundings of up to 53 bits, 2^-46.2 of the weight; its series 2^-48; the table and the products 2^-50).
    So each token's part of the sum, from border to border, reaches to u times the sum within twice that; its share is off by as much of the
    sum and its rounding."""
    last = 62 - (V - 1).bit_length() if V > 2048 else 51
    off = V * 2.0 ** -(last + 1)
    rng = np.random.default_rng(V)
    u = np.concatenate((1 - 2.0 ** -np.arange(1, 25), rng.random(8))).astype(np.float32)
    n = len(u)
    small = np.float32(-(last + part) * np.log(2))
    x = np.full((n, V), small, np.float32)
    at = rng.integers(0, V, n)
    x[np.arange(n), at] = 0
    w = np.exp(float(small))
    total = 1 + (V - 1) * w
    off += total * 2.0 ** -45
    for settings in (dict(), dict(k=np.full(n, V - 1, np.uint32)), dict(low=np.full(n, 1e-30))):
        got, prob = _run(dev, x, F32, u, **settings)
        for r in range(n):
            before = got[r] * w + (1 - w if got[r] > at[r] else 0)
            mine = 1.0 if got[r] == at[r] else w
            target = float(u[r]) * total
            assert before - 2 * off <= target <= before + mine + 2 * off, (r, got[r], at[r])
            assert abs(prob[r] - mine / total) <= mine / total * (off + 2.0 ** -24)


def test_rows_in_slices(dev):
    """2^21 rows and three more, which a launch of its own takes, each with its settings: of two logits (all rows checked), and of one."""
    rng = np.random.default_rng(31)
    n = (1 << 21) + 3
    x = rng.standard_normal((n, 2)).astype(np.float32)
    u, temp = rng.random(n, np.float32), np.where(rng.random(n) < 0.1, 0.0, rng.uniform(0.3, 2, n)).astype(np.float32)
    k = rng.integers(0, 4, n).astype(np.uint32)
    p, low = (np.where(rng.random(n) < 0.5, off, rng.random(n)).astype(np.float32) for off in (1.0, 0.0))
    with np.errstate(divide="ignore"):
        w = np.exp(-np.abs(x[:, 0].astype(np.float64) - x[:, 1]) / temp)  # of the smaller one
    first = (x[:, 1] > x[:, 0]).astype(np.int64)
    share = np.where(first == 0, 1 / (1 + w), w / (1 + w))  # of the logit at 0
    u[np.abs(u - share) < 1e-5] = 0  # (none on a border)
    p[np.abs(1 - p * (1 + w)) < 1e-5] = 1
    low[np.abs(w - low) < 1e-5] = 0
    both = (temp > 0) & (k != 1) & ((p >= 1) | (p * (1 + w) > 1)) & ((low <= 0) | (w >= low))
    want = np.where(both, (u >= share).astype(np.int64), first)
    part = np.where(both, np.where(want == 0, share, 1 - share), 1.0)
    got, prob = _run(dev, x, F32, u, temp, k, p, low)
    bad = np.flatnonzero(got != want)
    assert not len(bad), (len(bad), bad[0], u[bad[0]], share[bad[0]])
    assert np.all(np.abs(prob - part) <= part * 2.0 ** -22)
    x[::7] = -np.inf
    got, prob = _run(dev, x[:, :1], BF16, u, temp, k, p, low)
    assert not got.any() and np.array_equal(prob, np.isfinite(x[:, 0]).astype(np.float32))
