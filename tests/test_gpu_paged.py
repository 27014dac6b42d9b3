"""The paged key/value cache: rotary positions into its pages, attention over
them, and the moves of pages, against plain 64-bit statements (paged_ref)."""
import ctypes
import gc

import numpy as np
import pytest

import oracle
from paged_ref import EPS, attention, attention_bound, from_bits, rotate, rounded, to_bits
from tang_amd import capi

pytestmark = pytest.mark.gpu

F32, F16, BF16 = capi.F32, capi.F16, capi.BF16
NAMES = {F32: "f32", F16: "f16", BF16: "bf16"}


def _normal(rng, *shape):
    return rng.standard_normal(shape, dtype=np.float32)


class Model:
    """A cache with one layer (or more) and, beside it, what its sequences hold."""

    def __init__(self, dev, kh=2, hd=64, page=16, pages=64, seqs=8, layers=1, max_len=4096, dt=F16, heads=None, rows=4096):
        self.dev, self.kh, self.hd, self.dt, self.layers, self.heads = dev, kh, hd, dt, layers, heads or kh
        self.cache = dev.kv_cache(layers, kh, hd, page, pages, seqs, max_len, dt)
        self.batch = self.cache.batch(seqs, rows, self.heads)
        self.rows = {}  # sequence -> [layers][2][len][kh][hd]

    def create(self):
        s = self.cache.seq_create()[0]
        self.rows[s] = np.zeros((self.layers, 2, 0, self.kh, self.hd), np.float32)
        return s

    def begin(self, seqs, news):
        self.batch.begin(seqs, news)
        self.step = list(zip(seqs, news))

    def fill(self, rng, seqs, news):
        """The sequences grow by new random rows, as they are (no rotation)."""
        self.begin(seqs, news)
        n = sum(news)
        for l in range(self.layers):
            k, v = (rounded(_normal(rng, n, self.kh, self.hd), self.dt) for _ in range(2))
            self.batch.append(l, None, self.dev.upload(to_bits(k, self.dt), self.dt), self.dev.upload(to_bits(v, self.dt), self.dt), None)
            at = 0
            for s, m in zip(seqs, news):
                if l == 0:
                    pad = np.zeros((self.layers, 2, m, self.kh, self.hd), np.float32)
                    self.rows[s] = np.concatenate((self.rows[s], pad), 2)
                if m:
                    self.rows[s][l, 0, -m:], self.rows[s][l, 1, -m:] = k[at:at + m], v[at:at + m]
                at += m

    def check(self):
        for s, want in self.rows.items():
            assert self.cache.seq_len(s) == want.shape[2], s
            for l in range(self.layers):
                for w, b in enumerate(self.cache.seq_read(s, l)):
                    got = from_bits(b.to_numpy(), self.dt).reshape(-1, self.kh, self.hd)
                    assert np.array_equal(got, want[l, w]), (s, l, w)

    def attend(self, rng, qdt=F32, odt=F32, window=0, sinks=0, scale=0.0, layer=0, q=None, check=True):
        """Attention of the begun step's rows; compared with the statement unless check is false."""
        n = sum(m for _, m in self.step)
        if q is None:
            q = rounded(_normal(rng, n, self.heads, self.hd), qdt)
        out = self.dev.upload(to_bits(np.full(q.shape, 7.0, np.float32), odt), odt)
        self.batch.attention(layer, self.dev.upload(to_bits(q, qdt), qdt), out, window, sinks, scale)
        got = from_bits(out.to_numpy(), odt).reshape(q.shape)
        at = 0
        for s, m in self.step if check else ():
            k, v = self.rows[s][layer]
            if m:
                pos = np.arange(k.shape[0] - m, k.shape[0])
                args = (q[at:at + m], k, v, pos)
                with np.errstate(invalid="ignore"):
                    want = attention(*args, window, sinks, scale or None)
                tol = attention_bound(*args, qdt, self.dt, odt, window, sinks, scale or None)
                err = np.abs(got[at:at + m] - want).max()
                assert err <= tol, (s, m, err, tol)
            at += m
        return q, got


# ---------------------------------------------------------------------------
# Rotary positions
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("hd,rot", [(64, 64), (64, 32), (80, 48), (128, 128), (96, 20), (256, 96), (8, 2), (64, 0)])
@pytest.mark.parametrize("xdt,cdt,odt", [(F32, F16, F32), (BF16, BF16, BF16), (F32, BF16, BF16), (F16, F16, F32)])
def test_append(dev, half, hd, rot, xdt, cdt, odt):
    """Ragged rows of four sequences (one with none), some behind what is cached: the
    products and sums in f32, one rounding to the output's type, bit for bit."""
    rng = np.random.default_rng(hd * 1000 + rot + half)
    m = Model(dev, 2, hd, 16, 40, 4, 2, 400, cdt, heads=6)
    seqs = [m.create() for _ in range(4)]
    m.fill(rng, seqs, [5, 0, 33, 16])
    news = [1, 0, 40, 17]
    m.begin([seqs[i] for i in (2, 0, 1, 3)], [news[i] for i in (2, 0, 1, 3)])
    pos = np.concatenate([np.arange(33, 73), np.arange(5, 6), np.arange(16, 33)])
    n = len(pos)
    cos, sin = capi.rope_tables_scaled(rot, 100, 10000.0) if rot else (np.zeros((1, 1), np.float32),) * 2
    dc, ds = (dev.upload(cos), dev.upload(sin)) if rot else (None, None)
    for l in range(2):
        q, k, v = (rounded(_normal(rng, n, h, hd), xdt) for h in (6, 2, 2))
        qo = dev.alloc(n * 6 * hd, odt)
        m.batch.append(l, *(dev.upload(to_bits(t, xdt), xdt) for t in (q, k, v)), qo, dc, ds, rot, half)
        want = rounded(rotate(q, cos, sin, pos, rot, half), odt)
        assert np.array_equal(from_bits(qo.to_numpy(), odt).reshape(q.shape), want)
        k, v, at = rounded(rotate(k, cos, sin, pos, rot, half), cdt), rounded(v, cdt), 0
        for s, cnt in m.step:
            if l == 0:
                m.rows[s] = np.concatenate((m.rows[s], np.zeros((2, 2, cnt, 2, hd), np.float32)), 2)
            if cnt:
                m.rows[s][l, 0, -cnt:], m.rows[s][l, 1, -cnt:] = k[at:at + cnt], v[at:at + cnt]
            at += cnt
    m.check()


def test_append_positions_and_in_place(dev):
    """Positions of the caller's own, one of them behind the tables: that row's pairs are
    NaN, its other dims and the other rows are not. The rotated queries take the place of q."""
    rng = np.random.default_rng(3)
    m = Model(dev, 2, 64, 16, 8, 1, 1, 64, F16, heads=4)
    s = m.create()
    m.begin([s], [5])
    pos = np.array([7, 3, 20, 0, 7], np.uint32)
    cos, sin = capi.rope_tables_scaled(48, 20, 10000.0)
    q, k, v = (_normal(rng, 5, h, 64) for h in (4, 2, 2))
    dq = dev.upload(q)
    m.batch.append(0, dq, dev.upload(k), dev.upload(v), dq, dev.upload(cos), dev.upload(sin), 48, 1, dev.upload_u32(pos))
    got = dq.to_numpy().reshape(q.shape)
    ok = [0, 1, 3, 4]
    assert np.array_equal(got[ok], rotate(q[ok], cos, sin, pos[ok], 48, 1))
    assert np.isnan(got[2, :, :48]).all() and np.array_equal(got[2, :, 48:], q[2, :, 48:])
    kk = from_bits(m.cache.seq_read(s, 0)[0].to_numpy(), F16).reshape(k.shape)
    assert np.array_equal(kk[ok], rounded(rotate(k[ok], cos, sin, pos[ok], 48, 1), F16)) and np.isnan(kk[2, :, :48]).all()


@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("rows,heads,hd,rot,xdt,odt", [(1, 1, 2, 2, F32, F32), (3, 5, 64, 64, BF16, F32), (129, 4, 80, 20, F16, F16),
                                                       (700, 3, 128, 96, F32, BF16), (2, 3, 7, 4, F32, F32), (0, 4, 64, 64, F32, F32)])
def test_rope_rows(dev, half, rows, heads, hd, rot, xdt, odt):
    rng = np.random.default_rng(rows + hd)
    cos, sin = capi.rope_tables_scaled(rot, 1000, 5000.0, kind="linear", factor=3.0)
    x = rounded(_normal(rng, rows, heads, hd), xdt)
    dx, dc, ds = dev.upload(to_bits(x, xdt), xdt), dev.upload(cos), dev.upload(sin)
    out = dev.alloc(rows * heads * hd, odt)
    got = from_bits(dev.rope_rows(dx, dc, ds, rows, heads, hd, rot, half, start_pos=11, out=out).to_numpy(), odt).reshape(x.shape)
    assert np.array_equal(got, rounded(rotate(x, cos, sin, np.arange(11, 11 + rows), rot, half), odt))
    pos = rng.integers(0, 1000, rows).astype(np.uint32)
    got = from_bits(dev.rope_rows(dx, dc, ds, rows, heads, hd, rot, half, positions=dev.upload_u32(pos), out=dx if xdt == odt else out).to_numpy(), odt)
    assert np.array_equal(got.reshape(x.shape), rounded(rotate(x, cos, sin, pos, rot, half), odt))


def test_rope_rows_is_rope_forward_on_whole_interleaved_heads(dev):
    rng = np.random.default_rng(8)
    x, (c, s) = dev.upload(_normal(rng, 9, 4, 128)), capi.rope_tables(128, 64, 10000.0)
    dc, ds = dev.upload(c), dev.upload(s)
    a = dev.rope_forward_cached(x, dc, ds, 9, 4, 128, 33).to_numpy()
    assert np.array_equal(a, dev.rope_rows(x, dc, ds, 9, 4, 128, 128, start_pos=33).to_numpy())


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------

TYPES = [(F32, F16, F32), (F16, F16, F16), (BF16, BF16, BF16), (F32, BF16, F32), (BF16, F16, BF16)]


@pytest.mark.parametrize("qdt,cdt,odt", TYPES, ids=lambda t: NAMES[t])
@pytest.mark.parametrize("kh,G,hd,page,starts,news", [
    (2, 1, 64, 16, [0], [1]),                                  # the first position
    (1, 4, 128, 32, [0, 31, 32, 33, 127, 300], [1] * 6),        # block and page ends
    (2, 7, 128, 16, [15, 500, 0, 90], [2, 1, 3, 0]),           # a few new ones, none
    (3, 3, 80, 32, [100, 3], [5, 1]),                          # 80 of 128 dims
    (2, 1, 256, 16, [70, 260], [1, 16]),
    (1, 16, 64, 64, [1000], [1]),
    (1, 24, 64, 16, [50, 700], [1, 2]),                        # more query heads than a tile of 16
    (2, 4, 128, 16, [0], [130]),                               # a prompt
    (2, 2, 64, 16, [37, 0, 200], [61, 200, 9]),                # chunks behind what is cached
    (1, 3, 200, 16, [20], [64]),
    (4, 1, 40, 16, [0, 64], [65, 40]),
    (1, 128, 64, 16, [9], [3]),
])
def test_attention(dev, qdt, cdt, odt, kh, G, hd, page, starts, news):
    rng = np.random.default_rng(hd + sum(starts))
    m = Model(dev, kh, hd, page, 400, 8, 1, 1500, cdt, heads=kh * G)
    seqs = [m.create() for _ in starts]
    m.fill(rng, seqs, starts)
    m.fill(rng, seqs, news)
    for window, sinks in [(0, 0), (40, 0), (33, 5), (1, 0), (64, 70), (1, 1)]:
        m.attend(rng, qdt, odt, window, sinks)
    m.attend(rng, qdt, odt, scale=0.31)


@pytest.mark.parametrize("qdt,cdt", [(F32, F16), (BF16, BF16)], ids=lambda t: NAMES[t])
@pytest.mark.parametrize("kh,G,hd,start,new", [(1, 1, 64, 9000, 1), (2, 4, 128, 5000, 1), (1, 8, 128, 3500, 70), (1, 2, 256, 2500, 3)])
def test_attention_split_over_long_sequences(dev, qdt, cdt, kh, G, hd, start, new):
    """Long rows are cut into pieces whose records are merged."""
    rng = np.random.default_rng(start)
    m = Model(dev, kh, hd, 16, 700, 2, 1, 10000, cdt, heads=kh * G, rows=9100)
    s, t = m.create(), m.create()
    m.fill(rng, [s, t], [start, 10])
    m.fill(rng, [s, t], [new, 2])
    m.attend(rng, qdt, qdt)
    m.attend(rng, qdt, qdt, 2000, 4)


@pytest.mark.parametrize("qdt,cdt", [(F16, F16), (BF16, BF16), (F32, F16)])
@pytest.mark.parametrize("other", [0, 1])
def test_long_prompt_without_splits(dev, qdt, cdt, other):
    """So many rows that records for pieces run out: items of more keys than the MFMAs' own sums are for. Values about
    one would show sums that drift. (other: a second sequence's decode step in the same launch)"""
    rng = np.random.default_rng(other)
    m = Model(dev, 1, 64, 64, 400, 2, 1, 24000, cdt, heads=2, rows=16000)
    s, t = m.create(), m.create()
    for step in ([s, t], [16000, 0]), ([s, t], [4200, other]):
        m.begin(*step)
        n = sum(step[1])
        k, v = rounded(_normal(rng, n, 1, 64), cdt), rounded(1.0 + 0.125 * _normal(rng, n, 1, 64), cdt)
        m.batch.append(0, None, dev.upload(to_bits(k, cdt), cdt), dev.upload(to_bits(v, cdt), cdt), None)
        m.rows[s] = np.concatenate((m.rows[s], np.stack((k, v))[None, :, :step[1][0]]), 2)
        m.rows[t] = np.concatenate((m.rows[t], np.stack((k, v))[None, :, step[1][0]:]), 2)
    q, got = m.attend(rng, qdt, qdt, check=False)
    k, v = m.rows[s][0]
    rows = [0, 1, 63, 64, 2000, 4111, 4199]
    args = (q[rows], k, v, 16000 + np.array(rows))
    assert np.abs(got[rows] - attention(*args)).max() <= attention_bound(*args, qdt, cdt, qdt)
    if other:
        assert np.abs(got[4200] - m.rows[t][0, 1, 0]).max() <= 2 * EPS[qdt] * 2.0
    # replayed, with buffers for all 16000 rows that the batch may have
    wide = np.zeros((16000, 2, 64), np.float32)
    wide[:len(q)] = q
    qb, out = dev.upload(to_bits(wide, qdt), qdt), dev.upload(to_bits(wide, qdt), qdt)
    g = dev.capture(lambda: m.batch.attention(0, qb, out))
    for _ in range(2):
        g.launch()
        dev.sync()
        again = from_bits(out.to_numpy(), qdt).reshape(wide.shape)
        assert np.abs(again[rows] - attention(*args)).max() <= attention_bound(*args, qdt, cdt, qdt)
        assert not again[len(q):].any()  # rows behind the last stay as they were
    g.free()
    with pytest.raises(ValueError):
        m.batch.begin([s, t], [1])


def test_f32_queries_keep_their_precision(dev):
    """An f16 rounding of queries and probabilities (2^-12 of each on the average)
    shows in the results; parts that leave 2^-24 must show at most a 64th of that."""
    rng = np.random.default_rng(77)
    m = Model(dev, 2, 128, 16, 200, 2, 1, 1500, F16, heads=8)
    s, t = m.create(), m.create()
    m.fill(rng, [s, t], [700, 0])
    m.fill(rng, [s, t], [1, 150])
    q, got = m.attend(rng)
    off = rough = 0.0
    at = 0
    for sq, n in m.step:
        k, v = m.rows[sq][0]
        pos = np.arange(k.shape[0] - n, k.shape[0])
        want = attention(q[at:at + n], k, v, pos)
        off += np.square(got[at:at + n] - want).sum()
        rough += np.square(attention(rounded(q[at:at + n], F16), k, v, pos) - want).sum()
        at += n
    assert off < rough / 64 ** 2, (off, rough)


@pytest.mark.parametrize("qdt,cdt", [(F32, F16), (BF16, BF16)], ids=lambda t: NAMES[t])
@pytest.mark.parametrize("kh,G,hd,prefix,own,news,window", [
    (2, 4, 64, 256, [0, 5, 30, 17], [1, 1, 1, 1], 0),            # rows of four sequences in one tile of 16
    (1, 4, 128, 512, [3, 0, 60, 200, 1, 9, 33], [1] * 7, 0),     # more than 16 rows
    (1, 2, 128, 384, [0, 50, 7], [40, 1, 9], 0),
    (2, 2, 64, 384, [4, 90, 7], [2, 1, 3], 200),                 # the window leaves part of the prefix
    (2, 2, 64, 384, [4, 90, 7], [2, 1, 3], 30),                  # and none of it but the sinks
    (1, 4, 128, 128, [0] * 40, [1] * 40, 0),
    (1, 1, 64, 100, [30, 40], [1, 1], 0),                        # a shared page that is not full
])
def test_shared_prefix(dev, qdt, cdt, kh, G, hd, prefix, own, news, window):
    """Forks' shared pages are read once for all: the same results as the statement."""
    rng = np.random.default_rng(prefix + len(own))
    m = Model(dev, kh, hd, 16, 500, 48, 1, 1500, cdt, heads=kh * G)
    first, other = m.create(), m.create()
    m.fill(rng, [first, other], [prefix, 150])
    seqs = m.cache.seq_fork(first, len(own))
    for s in seqs:
        m.rows[s] = m.rows[first].copy()
    m.fill(rng, seqs, own)
    order = [seqs[0], other] + seqs[1:]  # the others of the group are not next to each other
    m.fill(rng, order, [news[0], 2] + news[1:])
    m.attend(rng, qdt, qdt, window, 3 if window else 0)
    m.attend(rng, qdt, qdt)
    m.check()


def test_prefix_of_unequal_lengths(dev):
    """Children of a child: all share the first pages, some share more."""
    rng = np.random.default_rng(5)
    m = Model(dev, 1, 64, 16, 200, 12, 1, 1500, F16, heads=4)
    a = m.create()
    m.fill(rng, [a], [400])
    b = m.cache.seq_fork(a, 1, 320)[0]
    m.rows[b] = m.rows[a][:, :, :320].copy()
    m.fill(rng, [b], [200])
    c = m.cache.seq_fork(b, 3)
    for s in c:
        m.rows[s] = m.rows[b].copy()
    m.fill(rng, [a, b] + c, [1, 2, 1, 0, 3])
    m.attend(rng)
    m.attend(rng, window=100, sinks=2)
    m.check()


@pytest.mark.parametrize("qdt,cdt", [(F32, F16), (BF16, BF16)], ids=lambda t: NAMES[t])
def test_what_others_left_in_pages_is_not_seen(dev, qdt, cdt):
    """NaN and infinities behind a sequence's end (another had the page) and in hidden keys."""
    rng = np.random.default_rng(9)
    m = Model(dev, 2, 64, 16, 40, 4, 1, 600, cdt, heads=4)
    bad = m.create()
    n = 600
    m.begin([bad], [n])
    junk = rng.choice(np.array([np.nan, np.inf, -np.inf, 1.0], np.float32), (n, 2, 64))
    d = dev.upload(to_bits(junk, cdt), cdt)
    m.batch.append(0, None, d, d, None)
    m.cache.seq_free([bad])
    del m.rows[bad]
    s, t = m.create(), m.create()
    m.fill(rng, [s, t], [50, 0])
    m.fill(rng, [s, t], [1, 77])
    for window, sinks in [(0, 0), (20, 3)]:
        m.attend(rng, qdt, qdt, window, sinks)


@pytest.mark.parametrize("qdt,cdt", [(F32, F16), (BF16, BF16)], ids=lambda t: NAMES[t])
@pytest.mark.parametrize("start,new", [(60, 1), (0, 60), (700, 3), (64, 100)])
def test_infinities_and_nan_reach_only_rows_that_see_them(dev, qdt, cdt, start, new):
    """An infinite V, a NaN V and an infinite K at some keys: rows that see them get what the
    statement gives (infinities and NaN included), the others what they would without."""
    rng = np.random.default_rng(start + new)
    m = Model(dev, 1, 64, 16, 120, 2, 1, 1200, cdt, heads=2)
    s = m.create()
    m.fill(rng, [s], [start + new])
    end = start + new
    k, v = (b.to_numpy().reshape(end, 1, 64) for b in m.cache.seq_read(s, 0))
    k, v = from_bits(k, cdt).copy(), from_bits(v, cdt).copy()
    v[end - 1, 0, 3] = np.inf
    v[end // 2, 0, 5] = np.nan
    v[end // 3, 0, 7] = -np.inf
    k[2, 0, :] = np.inf
    m.batch.trim([0])
    m.begin([s], [start] if start else [0])
    kd, vd = to_bits(k, cdt), to_bits(v, cdt)
    if start:
        m.batch.append(0, None, dev.upload(kd[:start], cdt), dev.upload(vd[:start], cdt), None)
    m.begin([s], [new])
    m.batch.append(0, None, dev.upload(kd[start:], cdt), dev.upload(vd[start:], cdt), None)
    for window, sinks in [(0, 0), (9, 0), (9, 2), (9, 4)]:
        q, got = m.attend(rng, qdt, qdt, window, sinks, check=False)
        pos = np.arange(start, end)
        with np.errstate(invalid="ignore", over="ignore"):
            # 0 * inf where a key is not seen is not part of the statement: hidden rows are zeroed for each row
            want = np.concatenate([attention(q[i:i + 1], *(np.where(sees[:, None, None], t, 0.0) for t in (k, v)), [p], window, sinks)
                                   for i, p in enumerate(pos) for sees in [_sees(p, end, window, sinks)]])
        fin = np.isfinite(want)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
        clean = np.where(np.isfinite(k), k, 0.0), np.where(np.isfinite(v), v, 0.0)
        tol = attention_bound(q, *clean, pos, qdt, cdt, qdt, window, sinks)
        assert np.abs(got[fin] - want[fin]).max(initial=0.0) <= tol


def _sees(p, n, window, sinks):
    j = np.arange(n)
    return (j <= p) & ((j > p - window) | (j < sinks) if window else True)


def test_queries_that_are_not_finite(dev):
    rng = np.random.default_rng(4)
    m = Model(dev, 1, 64, 16, 40, 2, 1, 500, F16, heads=2)
    s = m.create()
    m.fill(rng, [s], [70])
    m.fill(rng, [s], [40])
    q = _normal(rng, 40, 2, 64)
    q[3, 0, 1], q[17, 1, 0], q[20, 0, :], q[21] = np.nan, np.inf, 0.0, q[21] * 1e-30
    _, got = m.attend(rng, q=q, check=False)
    k, v = m.rows[s][0]
    with np.errstate(invalid="ignore"):
        want = attention(q, k, v, np.arange(70, 110))
    bad = np.isnan(want)
    assert bad[3, 0].all() and np.array_equal(np.isnan(got), bad)
    fine = ~bad.any(-1)
    tol = attention_bound(np.where(np.isfinite(q), q, 0.0), k, v, np.arange(70, 110), F32, F16, F32)
    assert np.abs(got[fine] - want[fine]).max() <= tol


def test_kv_attention_agrees_on_rows_read_out(dev):
    """The pages' rows read out are what th_kv_attention takes."""
    rng = np.random.default_rng(12)
    m = Model(dev, 2, 128, 16, 60, 1, 1, 900, F16, heads=8)
    s = m.create()
    m.fill(rng, [s], [800])
    m.fill(rng, [s], [3])
    q, got = m.attend(rng)
    k, v = m.cache.seq_read(s, 0)
    want = dev.kv_attention(dev.upload(q), k, v, 800, 3, 8, 2, 128).to_numpy().reshape(q.shape)
    kk, vv = m.rows[s][0]
    tol = 2 * attention_bound(q, kk, vv, np.arange(800, 803), F32, F16, F32)
    assert np.abs(got - want).max() <= tol


@pytest.mark.parametrize("qdt,cdt", [(F32, F16), (F16, F16), (F32, BF16), (BF16, BF16)], ids=lambda t: NAMES[t])
@pytest.mark.parametrize("start,new", [(50, 1), (10, 90)])
def test_small_and_large_values(dev, qdt, cdt, start, new):
    """Keys and values among the smallest of the cache's type (f16's below its normal range), queries that make up for
    it, and rows of tiny and of huge queries."""
    rng = np.random.default_rng(start + new)
    m = Model(dev, 1, 64, 16, 20, 1, 1, 200, cdt, heads=2)
    s = m.create()
    small = 2.0 ** -17
    for n in (start, new):
        m.begin([s], [n])
        k, v = (rounded(_normal(rng, n, 1, 64) * small, cdt) for _ in range(2))
        m.batch.append(0, None, dev.upload(to_bits(k, cdt), cdt), dev.upload(to_bits(v, cdt), cdt), None)
        m.rows[s] = np.concatenate((m.rows[s], np.stack((k, v))[None]), 2)
    q = rounded(_normal(rng, new, 2, 64) * np.float32(2.0 ** 13), qdt)
    m.attend(rng, qdt, F32 if qdt == F32 else qdt, q=q)
    if qdt == F32:
        q[0] *= np.float32(2.0 ** -100)
        q[new // 2] = np.float32(2.0 ** 90) * np.sign(q[new // 2])
        _, got = m.attend(rng, q=q, check=False)
        kk, vv = m.rows[s][0]
        want = attention(q, kk, vv, np.arange(start, start + new))
        row = [i for i in range(new) if i != new // 2]
        if row:
            tol = attention_bound(q[row], kk, vv, np.arange(start, start + new)[row], qdt, cdt, qdt)
            assert np.abs(got[row] - want[row]).max() <= tol
        # scores of 2^80 and more: all weight on the largest, which f32 sums of 64 products (2^-17 of the terms' sum) must tell
        # from the second
        p = np.sort(np.einsum("hd,nd->hn", q[new // 2].astype(np.float64), kk[:start + new // 2 + 1, 0].astype(np.float64)), -1)
        scale = np.abs(q[new // 2]).astype(np.float64) @ np.abs(kk[:, 0]).max(0)
        clear = (p[:, -1] - p[:, -2]) > scale * 2.0 ** -17
        assert clear.any()
        assert np.array_equal(got[new // 2][clear], want[new // 2][clear].astype(np.float32))


def test_beyond_four_gibibytes(dev):
    """Pages behind 2^32 bytes of a layer's keys: attention, append, copies, gathers and reads."""
    rng = np.random.default_rng(2)
    pages = 140100  # of 32 KiB: 4.6 GB of keys, as much of values
    m = Model(dev, 8, 128, 16, pages, 8, 1, 140000 * 16, F16, heads=16, rows=300)
    first = m.cache.seq_create()[0]
    m.cache.seq_resize(first, 139950 * 16)
    a, b = m.create(), m.create()
    m.fill(rng, [a, b], [70, 3])
    m.fill(rng, [a, b], [1, 40])
    m.attend(rng)
    c = m.cache.seq_fork(a, 2)
    for s in c:
        m.rows[s] = m.rows[a].copy()
    m.fill(rng, c, [1, 30])
    m.attend(rng)
    m.cache.seq_select(c[0], np.arange(50, 10, -1))
    m.rows[c[0]] = m.rows[c[0]][:, :, 50:10:-1].copy()
    m.check()
    m.cache.seq_free([first])
    assert m.cache.compact() > 0
    m.check()
    m.batch.free()
    m.cache.free()


# ---------------------------------------------------------------------------
# Pages
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("page,hd,dt", [(16, 8, F16), (16, 128, BF16), (64, 40, F16)])
def test_moves_of_pages(dev, page, hd, dt):
    """Random growth, forks, cuts, selections, frees and compactions: every sequence
    keeps its own rows, and no page is lost."""
    rng = np.random.default_rng(page)
    m = Model(dev, 2, hd, page, 40, 10, 2, 30 * page, dt)
    for turn in range(120):
        live = list(m.rows)
        vacant, free_seqs = m.cache.info()
        assert free_seqs == 10 - len(live)
        what = rng.integers(0, 7)
        if what == 0 and free_seqs:
            m.create()
        elif what == 1 and live:
            some = [int(s) for s in rng.permutation(live)[:rng.integers(1, len(live) + 1)]]
            news = [int(x) for x in rng.integers(0, 2 * page, len(some))]
            if vacant >= 3 * len(some) and all(m.rows[s].shape[2] + n <= 30 * page for s, n in zip(some, news)):
                m.fill(rng, some, news)
        elif what == 2 and live and free_seqs >= 2:
            s = int(rng.choice(live))
            n = int(rng.integers(0, m.rows[s].shape[2] + 1))
            for c in m.cache.seq_fork(s, 2, n):
                m.rows[c] = m.rows[s][:, :, :n].copy()
        elif what == 3 and live:
            s = int(rng.choice(live))
            n = int(rng.integers(0, m.rows[s].shape[2] + 1))
            m.cache.seq_resize(s, n)
            m.rows[s] = m.rows[s][:, :, :n]
        elif what == 4 and live:
            s = int(rng.choice(live))
            n = m.rows[s].shape[2]
            pos = rng.integers(0, max(n, 1), int(rng.integers(0, n + 1)))
            if vacant >= -(-len(pos) // page):
                m.cache.seq_select(s, pos)
                m.rows[s] = m.rows[s][:, :, pos].copy()
        elif what == 5 and live:
            s = int(rng.choice(live))
            m.cache.seq_free([s])
            del m.rows[s]
        else:
            m.cache.compact()
            assert m.cache.compact() == 0
        if turn % 10 == 0:
            m.check()
    m.check()
    m.cache.seq_free(list(m.rows))
    assert m.cache.info() == (40, 10)


def test_many_moves_at_once(dev):
    """More pages than a launch's arguments hold: forks that all write, a compaction of all."""
    rng = np.random.default_rng(1)
    m = Model(dev, 1, 64, 16, 900, 300, 1, 800, F16)
    a, gap = m.create(), m.create()
    m.fill(rng, [a], [13])
    m.cache.seq_resize(gap, 799)
    m.rows[gap] = None
    children = m.cache.seq_fork(a, 200)
    for s in children:
        m.rows[s] = m.rows[a].copy()
    m.batch.free()
    m.batch = m.cache.batch(300, 4096, 1)
    m.fill(rng, children, [2] * 200)
    m.cache.seq_free([gap])
    del m.rows[gap]
    m.check()
    assert m.cache.compact() == 50
    m.check()
    m.cache.seq_select(children[0], np.arange(14, -1, -1))
    m.rows[children[0]] = m.rows[children[0]][:, :, ::-1].copy()
    m.check()


def test_forks_that_go_again_before_a_step(dev):
    """Thousands of forks, resizes and frees without a step between: what is left of them is all that the next one uploads."""
    rng = np.random.default_rng(9)
    m = Model(dev, 1, 8, 16, 60, 6, 1, 500, F16)
    s = m.create()
    m.fill(rng, [s], [300])
    for i in range(3000):
        kids = m.cache.seq_fork(s, 3, 16 * (1 + i % 18))
        m.cache.seq_resize(kids[0], 16 * (i % 5))
        m.cache.seq_resize(kids[1], 400)
        m.cache.seq_free(kids)
    kid = m.cache.seq_fork(s, 1, 100)[0]
    m.rows[kid] = m.rows[s][:, :, :100].copy()
    other = m.create()
    m.cache.seq_resize(kid, 50)
    m.rows[kid] = m.rows[kid][:, :, :50]
    m.fill(rng, [other, kid, s], [33, 70, 1])
    m.check()


@pytest.mark.parametrize("seed", range(6))
def test_any_order_of_forks_and_changes(dev, seed):
    """Forks of forks, parents that shrink, go, or come again as something else, before anything of it is uploaded."""
    rng = np.random.default_rng(seed)
    m = Model(dev, 1, 8, 16, 150, 12, 1, 600, F16)
    m.fill(rng, [m.create()], [400])
    for i in range(250):
        live = list(m.rows)
        s = live[rng.integers(len(live))]
        have = m.rows[s].shape[2]
        kind = rng.integers(6)
        if kind == 0 and len(live) > 2:
            m.cache.seq_free([s])
            del m.rows[s]
        elif kind == 1 and len(live) < 11:
            n = int(rng.integers(0, have + 1))
            for c in m.cache.seq_fork(s, int(rng.integers(1, 13 - len(live))), n):
                m.rows[c] = m.rows[s][:, :, :n].copy()
        elif kind == 2 and rng.random() < 0.3:
            n = int(rng.integers(have // 2, have + 1))
            m.cache.seq_resize(s, n)
            m.rows[s] = m.rows[s][:, :, :n]
        elif kind == 3 and rng.random() < 0.3 and have and m.cache.info()[0] > 40:
            at = rng.integers(0, have, int(rng.integers(1, min(have, 100) + 1)))
            m.cache.seq_select(s, at)
            m.rows[s] = m.rows[s][:, :, at]
        elif kind == 4 and rng.random() < 0.2:
            m.cache.compact()
        elif kind == 5 and m.cache.info()[0] > 30:
            some = [x for x in live if m.rows[x].shape[2] < 500][:3]
            m.fill(rng, some, [int(rng.integers(0, 40)) for _ in some])
        if i % 9 == 8:
            m.check()
    m.check()


def test_uploads_ahead_of_the_stream(dev):
    """200 forks of a long sequence, 1.6 MB of table entries, behind work that keeps the stream busy: every child's row
    goes to its own page, whatever of the uploads' memory is reused by then."""
    rng = np.random.default_rng(8)
    m = Model(dev, 1, 64, 16, 1300, 201, 1, 17000, F16, rows=16008)
    s = m.create()
    m.fill(rng, [s], [16008])
    q = dev.alloc(16008 * 64, F16)
    out = dev.alloc(16008 * 64, F16)
    for _ in range(60):
        m.batch.attention(0, q, out)
    kids = []
    rows = [[dev.upload(to_bits(np.full((1, 1, 64), x, np.float32), F16), F16) for x in (i + 1, -i - 1)] for i in range(200)]
    for k, v in rows:
        kids += m.cache.seq_fork(s, 1)
        m.begin(kids[-1:], [1])
        m.batch.append(0, None, k, v, None)
    for i, c in enumerate(kids):
        for w, b in enumerate(m.cache.seq_read(c, 0, 16000)):
            got = from_bits(b.to_numpy(), F16).reshape(9, 64)
            assert np.array_equal(got[:8], m.rows[s][0, w, 16000:, 0]), (i, w)
            assert (got[8] == (i + 1 if w == 0 else -i - 1)).all(), (i, w)


def test_pages_are_handed_out_lowest_first_and_addressed(dev):
    m = Model(dev, 2, 64, 16, 10, 4, 2, 160, F16)
    k0, v0 = m.cache.page_pointers(0)
    k1, _ = m.cache.page_pointers(1)
    plane = 10 * 2 * 16 * 64 * 2
    assert v0 - k0 == plane and k1 - k0 == 2 * plane
    a, b = m.create(), m.create()
    m.cache.seq_resize(a, 33)
    m.cache.seq_resize(b, 160 - 48)
    assert m.cache.info()[0] == 0
    with pytest.raises(capi.TangHipError) as e:
        m.cache.seq_resize(a, 49)
    assert e.value.code == capi.TH_ERR_OOM
    assert m.cache.seq_len(a) == 33


# ---------------------------------------------------------------------------
# Together, captured, interleaved
# ---------------------------------------------------------------------------


def _step(rng, m, seqs, news, cos, sin, dc, ds, rot, half, window=0, sinks=0):
    """One step through all layers as a serving program makes it; the statement beside it."""
    m.begin(seqs, news)
    n = sum(news)
    lens = {s: m.rows[s].shape[2] for s in seqs}
    pos = np.concatenate([np.arange(lens[s], lens[s] + c) for s, c in zip(seqs, news)]).astype(int)
    for s, c in zip(seqs, news):
        m.rows[s] = np.concatenate((m.rows[s], np.zeros((m.layers, 2, c, m.kh, m.hd), np.float32)), 2)
    for l in range(m.layers):
        q, k, v = (_normal(rng, n, h, m.hd) for h in (m.heads, m.kh, m.kh))
        dq = m.dev.upload(q)
        m.batch.append(l, dq, m.dev.upload(k), m.dev.upload(v), dq, dc, ds, rot, half)
        out = m.dev.alloc(n * m.heads * m.hd)
        m.batch.attention(l, dq, out, window if l % 2 else 0, sinks if l % 2 else 0)
        got = out.to_numpy().reshape(q.shape)
        q = rotate(q, cos, sin, pos, rot, half)
        k, v, at = rounded(rotate(k, cos, sin, pos, rot, half), m.dt), rounded(v, m.dt), 0
        for s, c in zip(seqs, news):
            if c:
                m.rows[s][l, 0, -c:], m.rows[s][l, 1, -c:] = k[at:at + c], v[at:at + c]
                kk, vv = m.rows[s][l]
                w = (window, sinks) if l % 2 else (0, 0)
                args = (q[at:at + c], kk, vv, pos[at:at + c])
                err = np.abs(got[at:at + c] - attention(*args, *w)).max()
                assert err <= attention_bound(*args, F32, m.dt, F32, *w), (l, s, err)
            at += c


def test_serving_run(dev):
    """Prompts, forks with a shared prefix, decode steps with rejected drafts, a
    selection, a compaction: rotary positions, window and full layers in turns."""
    rng = np.random.default_rng(21)
    m = Model(dev, 2, 64, 16, 300, 12, 2, 1200, F16, heads=6)
    cos, sin = capi.rope_tables_scaled(32, 1200, 10000.0, kind="bands", factor=4.0, original_len=256)
    dc, ds = dev.upload(cos), dev.upload(sin)
    args = (cos, sin, dc, ds, 32, 1, 100, 3)
    a, b = m.create(), m.create()
    _step(rng, m, [a, b], [300, 45], *args)
    kids = m.cache.seq_fork(a, 4)
    for s in kids:
        m.rows[s] = m.rows[a].copy()
    for i in range(3):
        _step(rng, m, [b] + kids, [3, 1, 1, 2, 1], *args)
        m.batch.trim([1, 1, 1, 1, 1])
        m.rows[b] = m.rows[b][:, :, :-2]
        m.rows[kids[2]] = m.rows[kids[2]][:, :, :-1]
        m.check()
    keep = np.r_[0:4, 50:m.rows[b].shape[2]]
    m.cache.seq_select(b, keep)
    m.rows[b] = m.rows[b][:, :, keep].copy()
    m.cache.seq_free([a, kids[0]])
    del m.rows[a], m.rows[kids[0]]
    m.cache.compact()
    m.check()
    _step(rng, m, kids[1:] + [b], [1, 60, 1, 1], *args)
    m.check()


@pytest.mark.parametrize("cdt,qdt", [(F16, F32), (BF16, BF16)])
def test_captured_steps(dev, cdt, qdt):
    """A captured step (append and attention of two layers) replayed over begun steps whose
    sequences grow, join and leave, whose plans change from one kernel to another, with
    eager work between: every replay gives the eager call's bits."""
    rng = np.random.default_rng(31)
    m = Model(dev, 2, 64, 16, 300, 10, 2, 1500, cdt, heads=4, rows=96)
    seqs = [m.create() for _ in range(4)]
    m.fill(rng, seqs, [70, 3, 20, 1])
    big = m.cache.batch(4, 1200, 4)
    cap, kv = 96, 96 * 2 * 64
    cos, sin = capi.rope_tables_scaled(64, 1500, 10000.0)
    dc, ds = dev.upload(cos), dev.upload(sin)
    q, k, v = (dev.alloc(cap * h * 64, qdt) for h in (4, 2, 2))
    qr, out = dev.alloc(cap * 256, qdt), [dev.alloc(cap * 256, qdt) for _ in range(2)]

    def step():
        for l in range(2):
            m.batch.append(l, q, k, v, qr, dc, ds, 64, 1)
            m.batch.attention(l, qr, out[l], 50 * l, 2 * l)

    m.batch.begin(seqs, [1, 1, 1, 1])
    step()
    dev.sync()
    graph = dev.capture(step)
    for news in ([1, 1, 1, 1], [1, 0, 2, 1], [20, 30, 1, 1], [0, 0, 0, 1], [1, 1, 1, 1], [90, 1, 1, 1]):
        m.batch.trim([0] * len(seqs)) if news == [1, 1, 1, 1] else None
        m.batch.begin(seqs, news)
        n = sum(news)
        for buf, h in ((q, 4), (k, 2), (v, 2)):
            buf.upload(np.concatenate((to_bits(_normal(rng, n, h, 64), qdt).ravel(), buf.to_numpy()[n * h * 64:])))
        for o in out:
            dev.zero_buffer(o)
        graph.launch()
        dev.sync()
        got = [o.to_numpy() for o in out] + [b.to_numpy() for s in seqs for l in range(2) for b in m.cache.seq_read(s, l)]
        for o in out:
            dev.zero_buffer(o)
        step()
        want = [o.to_numpy() for o in out] + [b.to_numpy() for s in seqs for l in range(2) for b in m.cache.seq_read(s, l)]
        assert all(np.array_equal(x, y) for x, y in zip(got, want)), news
        assert not any(o.to_numpy()[n * 256:].any() for o in out)  # rows behind the last are left as they were
        if sum(news) == 4:  # another batch on the cache between, with a long sequence
            extra = m.cache.seq_create()
            big.begin(extra, [700])
            kk = dev.upload(to_bits(_normal(rng, 700, 2, 64), cdt), cdt)
            for l in range(2):
                big.append(l, None, kk, kk, None)
            m.cache.seq_free(extra)
    graph.free()


def test_many_windows(dev):
    """More windows than a batch keeps plans for, in turns over steps; one is captured and stays."""
    rng = np.random.default_rng(61)
    m = Model(dev, 1, 64, 16, 60, 2, 1, 600, F16, heads=2, rows=4)
    s = m.create()
    for _ in range(100):
        m.fill(rng, [s], [4])
    m.fill(rng, [s], [1])
    q, out = dev.alloc(4 * 128), dev.alloc(4 * 128)
    m.batch.attention(0, q, out, 50, 1)
    graph = dev.capture(lambda: m.batch.attention(0, q, out, 50, 1))
    for step in range(3):
        for window in range(1, 60, 2):
            m.attend(rng, window=window, sinks=window % 3)
        m.fill(rng, [s], [2 + step])
        x = _normal(rng, 4, 2, 64)
        q.upload(x)
        graph.launch()
        dev.sync()
        n = 2 + step
        k, v = m.rows[s][0]
        args = (x[:n], k, v, np.arange(k.shape[0] - n, k.shape[0]))
        err = np.abs(out.to_numpy().reshape(x.shape)[:n] - attention(*args, 50, 1)).max()
        assert err <= attention_bound(*args, F32, F16, F32, 50, 1)
    graph.free()


def test_out_of_memory_leaves_no_trace(dev):
    """A cache that does not fit is refused, and the calls behind it work."""
    _refused(capi.TH_ERR_OOM, dev.kv_cache, 1024, 8, 256, 1024, 4096, 1, 64)  # 33 TB
    m = Model(dev, 1, 64, 16, 10, 2, 1, 100, F16)
    s = m.create()
    m.fill(np.random.default_rng(1), [s], [20])
    m.check()


def test_two_batches_and_two_handles(dev):
    """Batches of disjoint sequences may both have begun; a buffer of another handle is refused."""
    rng = np.random.default_rng(41)
    m = Model(dev, 1, 64, 16, 60, 4, 1, 300, F16, heads=2)
    a, b = m.create(), m.create()
    m.fill(rng, [a, b], [50, 90])
    first, second = m.batch, m.cache.batch(2, 100, 2)
    m.fill(rng, [a], [2])
    step_a = m.step
    m.batch = second
    m.fill(rng, [b], [40])
    m.attend(rng)
    m.batch, m.step = first, step_a
    m.attend(rng)
    other = capi.HipComputeDevice(0)
    x = other.upload(_normal(rng, 2, 2, 64))
    with pytest.raises(capi.TangHipError):
        m.batch.attention(0, x, dev.alloc(256))
    m2 = Model(other, 1, 64, 16, 30, 2, 1, 300, F16, heads=2)
    s = m2.create()
    m2.fill(rng, [s], [33])
    m2.fill(rng, [s], [1])
    m2.attend(rng)
    m.attend(rng)
    m2.batch.free()
    m2.cache.free()
    other.close()


def test_results_repeat_bit_for_bit(dev):
    """No order of arrival decides a sum."""
    rng = np.random.default_rng(51)
    m = Model(dev, 2, 128, 16, 600, 6, 1, 4000, F16, heads=8, rows=4500)
    seqs = [m.create() for _ in range(3)]
    m.fill(rng, seqs, [3500, 900, 40])
    m.fill(rng, seqs, [1, 70, 1])
    q, want = m.attend(rng)
    for _ in range(5):
        assert np.array_equal(m.attend(rng, q=q, check=False)[1], want)


# ---------------------------------------------------------------------------
# Refusals
# ---------------------------------------------------------------------------


def _refused(code, fn, *args, **kw):
    with pytest.raises(capi.TangHipError) as e:
        fn(*args, **kw)
    assert e.value.code == code, e.value


def test_refusals(dev):
    bad, oom, uns = capi.TH_ERR_INVALID, capi.TH_ERR_OOM, capi.TH_ERR_UNSUPPORTED
    _refused(uns, dev.kv_cache, 1, 1, 64, 16, 4, 1, 64, F32)
    _refused(uns, dev.kv_cache, 1, 1, 12, 16, 4, 1, 64)
    _refused(uns, dev.kv_cache, 1, 1, 264, 16, 4, 1, 64)
    for args in [(0, 1, 64, 16, 4, 1, 64), (1, 0, 64, 16, 4, 1, 64), (1, 1, 64, 24, 4, 1, 64), (1, 1, 64, 8, 4, 1, 64), (1, 1, 64, 16, 0, 1, 64),
                 (1, 1, 64, 16, 4, 0, 64), (1, 1, 64, 16, 4, 1, 0), (1, 1, 64, 16, 1 << 28, 1, 64), (1, 1, 64, 16, 4, 1, 1 << 29)]:
        _refused(bad, dev.kv_cache, *args)
    c = dev.kv_cache(2, 2, 64, 16, 8, 3, 100)
    _refused(bad, c.batch, 4, 10, 2)
    _refused(bad, c.batch, 1, 10, 3)
    _refused(bad, c.batch, 1, 0, 2)
    _refused(bad, c.batch, 1, 10, 258)
    b = c.batch(2, 40, 4)
    x, kv = dev.alloc(40 * 4 * 64), dev.alloc(40 * 2 * 64)
    y = dev.alloc(40 * 4 * 64)
    _refused(bad, b.attention, 0, x, y)  # not begun
    s, t = c.seq_create(2)
    _refused(oom, c.seq_create, 2)
    for fn in (c.seq_len, lambda i: c.seq_resize(i, 1), lambda i: c.seq_fork(i, 1, 0), lambda i: c.seq_select(i, [0]), lambda i: c.seq_free([i])):
        for i in (-1, 2, 3, 1 << 20):
            _refused(bad, fn, i)
    _refused(bad, c.seq_resize, s, 101)
    _refused(bad, c.seq_free, [s, s])
    _refused(bad, b.begin, [s, s], [1, 1])
    _refused(bad, b.begin, [s, 2], [1, 1])
    _refused(bad, b.begin, [s], [41])
    _refused(bad, b.begin, [s, t, s], [1, 1, 1])
    _refused(bad, c.seq_fork, s, 1, 1)
    c.seq_resize(t, 90)
    _refused(oom, b.begin, [s, t], [30, 9])
    assert c.seq_len(s) == 0 and c.seq_len(t) == 90 and c.info() == (2, 1)
    _refused(bad, b.begin, [t], [11])
    _refused(bad, c.seq_select, t, [0, 90])
    _refused(oom, c.seq_select, t, np.arange(40))
    b.begin([s, t], [20, 3])
    n = 23
    _refused(bad, b.attention, 2, x, y)
    _refused(bad, b.attention, 0, x, x)
    _refused(bad, b.attention, 0, dev.alloc(n * 256 - 1), y)
    _refused(bad, b.attention, 0, x, dev.alloc(n * 256 - 1))
    _refused(bad, b.attention, 0, dev.alloc(n * 256, capi.I32), y)
    for scale in (-1.0, float("nan"), float("inf")):
        _refused(bad, b.attention, 0, x, y, scale=scale)
    tab = dev.alloc(92 * 32)
    _refused(bad, b.append, 0, x, kv, kv, y, tab, tab, 64, 0)  # positions up to 92
    tab = dev.alloc(93 * 32)
    _refused(bad, b.append, 0, x, kv, kv, y, tab, tab, 63, 0)
    _refused(bad, b.append, 0, x, kv, kv, y, tab, tab, 66, 0)
    _refused(bad, b.append, 0, x, kv, kv, y, tab, tab, 64, 2)
    _refused(bad, b.append, 0, x, kv, kv, y, None, tab, 64, 0)
    _refused(bad, b.append, 0, x, kv, dev.alloc(n * 128, F16), y, tab, tab, 64, 0)
    _refused(bad, b.append, 0, x, kv, kv, None, tab, tab, 64, 0)
    _refused(bad, b.append, 0, x, kv, dev.alloc(n * 128 - 1), y, tab, tab, 64, 0)
    _refused(bad, b.append, 0, x, kv, kv, y, tab, tab, 64, 0, dev.alloc(22, capi.U32))
    _refused(bad, b.append, 2, x, kv, kv, y, tab, tab, 64, 0)
    b.append(0, x, kv, kv, y, tab, tab, 64, 0)
    _refused(bad, b.trim, [1])
    _refused(bad, b.trim, [1, 4])
    k16 = dev.alloc(20 * 128, F16)
    for layer, start, cnt in [(2, 0, 1), (0, 21, 0), (0, 20, 1), (0, 0, 21)]:
        rc = capi.lib().th_kv_seq_read(c.handle, s, layer, start, cnt, k16.handle, dev.alloc(20 * 128, F16).handle)
        assert rc == bad
    assert capi.lib().th_kv_seq_read(c.handle, s, 0, 0, 1, k16.handle, k16.handle) == bad
    # the batch's sequences changed: it has to begin again
    c.seq_resize(s, 19)
    _refused(bad, b.attention, 0, x, y)
    _refused(bad, b.append, 0, x, kv, kv, y)
    b.begin([t], [1])
    c.seq_free([t])
    _refused(bad, b.attention, 0, x, y)
    _refused(bad, b.trim, [0])
    _refused(bad, dev.rope_rows, x, tab, tab, 3, 4, 64, 65)
    _refused(bad, dev.rope_rows, x, tab, tab, 3, 4, 64, 66)
    _refused(bad, dev.rope_rows, x, tab, tab, 3, 4, 64, 64, 0, 91)
    _refused(bad, dev.rope_rows, x, tab, None, 3, 4, 64, 64)
    _refused(bad, dev.rope_rows, x, tab, tab, 41, 4, 64, 64)
    _refused(bad, dev.rope_rows, x, tab, tab, 3, 4, 64, 64, out=dev.alloc(100))


def test_what_cannot_be_captured(dev):
    c = dev.kv_cache(1, 1, 64, 16, 8, 2, 100)
    b = c.batch(2, 8, 2)
    s = c.seq_create()[0]
    c.seq_resize(s, 10)
    b.begin([s], [1])
    x, y = dev.alloc(8 * 128), dev.alloc(8 * 128)
    b.attention(0, x, y, 5)

    def inside():
        _refused(capi.TH_ERR_INVALID, b.begin, [s], [1])
        _refused(capi.TH_ERR_INVALID, c.seq_resize, s, 20)
        _refused(capi.TH_ERR_INVALID, c.seq_select, s, [0])
        _refused(capi.TH_ERR_INVALID, c.compact)
        _refused(capi.TH_ERR_INVALID, dev.kv_cache, 1, 1, 64, 16, 8, 2, 100)
        _refused(capi.TH_ERR_INVALID, c.batch, 2, 8, 2)
        _refused(capi.TH_ERR_INVALID, b.attention, 0, x, y, 6)  # a window that has no plan yet
        _refused(capi.TH_ERR_INVALID, b.attention, 0, dev_small, y, 5)  # fewer than max_rows rows
        b.attention(0, x, y, 5)

    dev_small = dev.alloc(128)
    g = dev.capture(inside)
    g.launch()
    dev.sync()
    g.free()


def test_garbage_does_not_end_a_capture(dev):
    """Buffers in a cycle of references, which the collector frees when so many objects have been made."""
    x, y = dev.upload(np.ones(8, np.float32)), dev.upload(np.full(8, 2.0, np.float32))

    def inside():
        for _ in range(2):
            dev.add_assign(x, y)
            objects = [[i] for i in range(100000)]  # the collector's thresholds are passed
            assert objects

    cycle = [dev.alloc(64)]
    cycle.append(cycle)
    del cycle
    assert gc.isenabled()
    g = dev.capture(inside)
    assert gc.isenabled()
    g.launch()
    assert np.array_equal(x.to_numpy(), np.full(8, 5.0, np.float32))
    g.free()


def test_handles_go_in_any_order(dev):
    """A batch may outlive its cache; captured graphs keep what they name."""
    c = dev.kv_cache(1, 1, 64, 16, 8, 2, 100)
    b = c.batch(2, 8, 2)
    s = c.seq_create()[0]
    c.seq_resize(s, 10)
    b.begin([s], [1])
    x, y = dev.upload(np.ones(8 * 128, np.float32)), dev.alloc(8 * 128)
    b.attention(0, x, y)
    g = dev.capture(lambda: b.attention(0, x, y))
    c.free()
    _refused(capi.TH_ERR_INVALID, b.attention, 0, x, y)
    b.free()
    g.launch()  # reads the pages as they were
    dev.sync()
    assert np.isfinite(y.to_numpy()[:128]).all()
    g.free()
    L = capi.lib()
    assert L.th_kv_cache_destroy(None) == 0 and L.th_kv_batch_destroy(None) == 0
    for fn, n in (("th_kv_cache_info", 2), ("th_kv_cache_compact", 1)):
        assert getattr(L, fn)(None, *[None] * n) == capi.TH_ERR_INVALID
    assert L.th_kv_batch_begin(None, None, None, 0) == capi.TH_ERR_INVALID
    assert L.th_kv_batch_attention(None, 0, None, 0, 0, ctypes.c_float(0.0), None) == capi.TH_ERR_INVALID
