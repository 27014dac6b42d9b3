"""Norms of query and key heads with their rotation, into rows and into a
cache's pages, against the formula in 64 bits."""
import numpy as np
import pytest

from paged_ref import EPS, LEAST, from_bits, rounded, to_bits
from tang_amd import capi

pytestmark = pytest.mark.gpu

F32, F16, BF16 = capi.F32, capi.F16, capi.BF16


def _normal(rng, *shape):
    return rng.standard_normal(shape, dtype=np.float32)


def _formula(x, w, eps, cos, sin, pos, rot, half):
    """(results, bounds without the result's own rounding) of x [rows][heads][hd].

    In f32 a sum of squares is off by at most (16 + 6) half steps u of itself (sixteen in a lane, six joins), its mean, eps, root and
    reciprocal add four: 15 u for the reciprocal root. With the products by it and the weight a value is off by 17 u, a product with
    the table's value by 18 u, and the pair's sum by 1 u more: 20 u of |a c| + |b s| covers them and their products."""
    x = np.asarray(x, np.float64)
    with np.errstate(all="ignore"):
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
        if w is not None:
            y = y * np.asarray(w, np.float64)
        size = np.abs(y)
        if rot:
            pos = np.asarray(pos)
            known = pos < len(cos)
            c, s = (np.where(known[:, None], t[np.where(known, pos, 0)].astype(np.float64), np.nan)[:, None] for t in (cos, sin))
            i = np.arange(rot // 2)
            u, v = (i, i + rot // 2) if half else (2 * i, 2 * i + 1)
            a, b = y[..., u].copy(), y[..., v].copy()
            y[..., u], y[..., v] = a * c - b * s, a * s + b * c
            size[..., u], size[..., v] = np.abs(a * c) + np.abs(b * s), np.abs(a * s) + np.abs(b * c)
    return y, 20 * 2.0 ** -24 * size


def _check(got, want, dt):
    y, bound = want
    fine = np.isfinite(y)
    assert np.array_equal(np.isnan(got), np.isnan(y))
    with np.errstate(all="ignore"):
        tol = bound * (1 + EPS[dt]) + np.maximum(EPS[dt] * np.abs(y), LEAST[dt])
        err = np.abs(got - y)
    bad = fine & ~(err <= tol)
    assert not bad.any(), (np.argwhere(bad)[0], got[bad][0], y[bad][0])
    assert np.array_equal(got[~fine & ~np.isnan(y)], y[~fine & ~np.isnan(y)])


def _tables(dev, rot, n, base=10000.0):
    if not rot:
        return np.zeros((1, 1), np.float32), np.zeros((1, 1), np.float32), None, None
    cos, sin = capi.rope_tables_scaled(rot, n, base)
    return cos, sin, dev.upload(cos), dev.upload(sin)


def _weights(dev, rng, hd, dt):
    w = [rounded(1 + 0.3 * _normal(rng, hd), dt) for _ in range(2)]
    return w, [dev.upload(to_bits(v, dt), dt) for v in w]


SHAPES = [(64, 64), (128, 128), (128, 32), (80, 48), (96, 96), (256, 256), (8, 0), (40, 16), (24, 24), (96, 20), (6, 2), (1, 0), (65, 34), (512, 128),
          (1032, 16), (1024, 1024)]


@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("hd,rot", SHAPES)
@pytest.mark.parametrize("xdt,odt,wdt", [(F32, F32, F32), (BF16, BF16, BF16), (F16, F32, BF16), (F32, F16, None)])
def test_rows(dev, half, hd, rot, xdt, odt, wdt):
    """Queries and keys of their own, scattered positions."""
    rng = np.random.default_rng(hd * 1000 + rot + half)
    n, H, K = 7, 5, 2
    cos, sin, dc, ds = _tables(dev, rot, 50)
    w, dw = _weights(dev, rng, hd, wdt) if wdt is not None else ([None, None], [None, None])
    pos = rng.integers(0, 50, n).astype(np.uint32)
    x = [rounded(3 * _normal(rng, n, h, hd), xdt) for h in (H, K)]
    out = [dev.upload(to_bits(np.full(t.shape, 7.0, np.float32), odt), odt) for t in x]
    dx = [dev.upload(to_bits(t, xdt), xdt) for t in x]
    dev.qk_norm_rope(*dx, *dw, 1e-5, dc, ds, n, H, K, hd, rot, half, positions=dev.upload_u32(pos), q_out=out[0], k_out=out[1])
    for t, o, v, d in zip(x, out, w, dx):
        _check(from_bits(o.to_numpy(), odt).reshape(t.shape), _formula(t, v, 1e-5, cos, sin, pos, rot, half), odt)
        assert np.array_equal(d.to_numpy(), to_bits(t, xdt).reshape(-1))


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("hd,rot,extra", [(64, 64, 0), (128, 64, 8), (128, 128, 3), (20, 6, 1)])
@pytest.mark.parametrize("form", ["apart", "together", "inplace", "queries"])
def test_packed_rows(dev, dt, hd, rot, extra, form):
    """Rows that hold q, k, v and `extra` elements more: results in buffers of their own, in one, in
    place (values and the rest stay), or of the queries alone; positions from a start."""
    rng = np.random.default_rng(hd + rot + extra)
    n, H, K = 37, 6, 2
    stride = (H + 2 * K) * hd + extra
    cos, sin, dc, ds = _tables(dev, rot, 60)
    w, dw = _weights(dev, rng, hd, F32)
    x = rounded(2 * _normal(rng, n * stride - extra), dt)  # the last row ends with its values
    dx = dev.upload(to_bits(x, dt), dt)
    full = np.concatenate((x, np.zeros(extra, np.float32))).reshape(n, stride)
    heads = full[:, :(H + 2 * K) * hd].reshape(n, H + 2 * K, hd)
    pos = np.arange(n) + 20
    args = (1e-6, dc, ds, n, H, 0 if form == "queries" else K, hd, rot, 1)
    want_q, want_k = (_formula(t, v, 1e-6, cos, sin, pos, rot, 1) for t, v in ((heads[:, :H], w[0]), (heads[:, H:H + K], w[1])))
    if form == "inplace":
        dev.qk_norm_rope(dx, None, *dw, *args, start_pos=20, q_stride=stride, q_out=dx)
        got = np.concatenate((from_bits(dx.to_numpy(), dt), np.zeros(extra, np.float32))).reshape(n, stride)
        assert np.array_equal(got[:, (H + K) * hd:], full[:, (H + K) * hd:])
        got = got[:, :(H + K) * hd].reshape(n, H + K, hd)
    elif form == "together":
        out = dev.alloc(n * (H + K) * hd, dt)
        dev.qk_norm_rope(dx, None, *dw, *args, start_pos=20, q_stride=stride, q_out=out)
        got = from_bits(out.to_numpy(), dt).reshape(n, H + K, hd)
    else:
        q, k = dev.qk_norm_rope(dx, None, *dw, *args, start_pos=20, q_stride=stride)
        got = from_bits(q.to_numpy(), dt).reshape(n, H, hd)
        if form == "queries":
            assert k is None
            return _check(got, want_q, dt)
        got = np.concatenate((got, from_bits(k.to_numpy(), dt).reshape(n, K, hd)), 1)
    _check(got[:, :H], want_q, dt)
    _check(got[:, H:], want_k, dt)


@pytest.mark.parametrize("hd", [64, 20])
def test_values_at_the_ends_of_f32(dev, hd):
    """Heads whose squares overflow or vanish, heads of zeros, infinities and NaN; positions behind the tables."""
    rng = np.random.default_rng(5)
    x = _normal(rng, 9, 2, hd)
    x[0] *= 1e30
    x[1] *= 1e-30
    x[2] = 0.0
    x[3, 0, 3] = np.inf
    x[4, 1, 5] = np.nan
    x[5] = 3e38
    x[6] = 2.0 ** -149
    x[7, 0, :4] = 0.0
    cos, sin, dc, ds = _tables(dev, 16, 10)
    pos = np.array([0, 1, 2, 3, 4, 5, 6, 10, 4000000000], np.uint32)
    for eps in (0.0, 1e-6):
        out, _ = dev.qk_norm_rope(dev.upload(x), None, None, None, eps, dc, ds, 9, 2, 0, hd, 16, 1, positions=dev.upload_u32(pos))
        y, bound = _formula(x, None, eps, cos, sin, pos, 16, 1)
        # An infinity makes its head's other dims zero; a value that the division makes NaN, and its pair, are NaN.
        _check(out.to_numpy().reshape(x.shape), (y, bound + 2.0 ** -148), F32)


def test_no_rows_and_many(dev):
    """No rows write nothing; 70000 rows of one head go through a grid that walks."""
    rng = np.random.default_rng(6)
    cos, sin, dc, ds = _tables(dev, 64, 70000)
    x = dev.upload(np.full(64, 5.0, np.float32))
    dev.qk_norm_rope(x, None, None, None, 1e-6, dc, ds, 0, 1, 0, 64, 64, 1, q_out=x)
    assert np.all(x.to_numpy() == 5.0)
    t = rounded(_normal(rng, 70000, 1, 64), BF16)
    out, _ = dev.qk_norm_rope(dev.upload(to_bits(t, BF16), BF16), None, None, None, 1e-6, dc, ds, 70000, 1, 0, 64, 64, 1)
    _check(from_bits(out.to_numpy(), BF16).reshape(t.shape), _formula(t, None, 1e-6, cos, sin, np.arange(70000), 64, 1), BF16)


@pytest.mark.parametrize("half", [0, 1])
def test_many_heads_a_group(dev, half):
    """So many rows that lanes take several heads of a row, whose number is no multiple of theirs; in place too, and into pages."""
    rng = np.random.default_rng(7 + half)
    n, H, K, hd = 30000, 7, 2, 64
    cos, sin, dc, ds = _tables(dev, 48, n)
    w, dw = _weights(dev, rng, hd, F32)
    x = rounded(2 * _normal(rng, n, H + K, hd), BF16)
    dx = dev.upload(to_bits(x, BF16), BF16)
    args = (dx, None, *dw, 1e-6, dc, ds, n, H, K, hd, 48, half)
    q, k = dev.qk_norm_rope(*args)
    want = [_formula(t, v, 1e-6, cos, sin, np.arange(n), 48, half) for t, v in ((x[:, :H], w[0]), (x[:, H:], w[1]))]
    _check(from_bits(q.to_numpy(), BF16).reshape(n, H, hd), want[0], BF16)
    _check(from_bits(k.to_numpy(), BF16).reshape(n, K, hd), want[1], BF16)
    dev.qk_norm_rope(*args, q_out=dx)
    got = dx.to_numpy().reshape(n, H + K, hd)
    assert np.array_equal(got[:, :H].reshape(-1), q.to_numpy()) and np.array_equal(got[:, H:].reshape(-1), k.to_numpy())
    # 30000 rows of 6 + 2 + 2 heads into pages
    cache = dev.kv_cache(1, K, hd, 64, 480, 1, n, F16)
    batch, seqs = cache.batch(1, n, 6), cache.seq_create(1)
    batch.begin(seqs, [n])
    x = rounded(2 * _normal(rng, n, 6 + 2 * K, hd), F16)
    out = dev.alloc(n * 6 * hd, F16)
    batch.append_norm(0, dev.upload(to_bits(x, F16), F16), None, None, out, *dw, 1e-6, dc, ds, 48, half)
    _check(from_bits(out.to_numpy(), F16).reshape(n, 6, hd), _formula(x[:, :6], w[0], 1e-6, cos, sin, np.arange(n), 48, half), F16)
    gk, gv = (from_bits(b.to_numpy(), F16).reshape(n, K, hd) for b in cache.seq_read(seqs[0], 0))
    _check(gk, _formula(x[:, 6:8], w[1], 1e-6, cos, sin, np.arange(n), 48, half), F16)
    assert np.array_equal(gv, x[:, 8:])


@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("hd,rot,heads", [(64, 64, 4), (128, 128, 6), (80, 48, 2), (96, 20, 2), (256, 96, 8)])
@pytest.mark.parametrize("xdt,cdt,odt", [(F32, F16, F32), (BF16, BF16, BF16), (F16, BF16, F32)])
@pytest.mark.parametrize("packed", [False, True])
def test_append(dev, half, hd, rot, heads, xdt, cdt, odt, packed):
    """Ragged rows of three sequences, one of them with none, into pages that hold rows already; other rows of the pages stay."""
    rng = np.random.default_rng(hd + rot + half)
    K, layers, news, had = 2, 2, [33, 0, 1], [5, 20, 16]
    cache = dev.kv_cache(layers, K, hd, 16, 20, 3, 200, cdt)
    batch, seqs = cache.batch(3, 64, heads), cache.seq_create(3)
    cos, sin, dc, ds = _tables(dev, rot, 200)
    old = [rounded(_normal(rng, 2, sum(had), K, hd), cdt) for _ in range(layers)]
    batch.begin(seqs, had)
    for l in range(layers):
        batch.append(l, None, *[dev.upload(to_bits(t, cdt), cdt) for t in old[l]], None)
    order = [2, 0, 1]
    batch.begin([seqs[i] for i in order], [news[i] for i in order])
    pos = np.concatenate([np.arange(had[i], had[i] + news[i]) for i in order])
    n = len(pos)
    for l in range(layers):
        w, dw = _weights(dev, rng, hd, F32)
        x = rounded(2 * _normal(rng, n, heads + 2 * K, hd), xdt)
        q, k, v = x[:, :heads], x[:, heads:heads + K], x[:, heads + K:]
        out = dev.alloc(n * heads * hd, odt)
        bufs = (dev.upload(to_bits(x, xdt), xdt), None, None) if packed else [dev.upload(to_bits(t, xdt), xdt) for t in (q, k, v)]
        batch.append_norm(l, *bufs, out, *dw, 1e-6, dc, ds, rot, half)
        _check(from_bits(out.to_numpy(), odt).reshape(q.shape), _formula(q, w[0], 1e-6, cos, sin, pos, rot, half), odt)
        want = _formula(k, w[1], 1e-6, cos, sin, pos, rot, half)
        at = 0
        for i in order:
            gk, gv = (from_bits(b.to_numpy(), cdt).reshape(-1, K, hd) for b in cache.seq_read(seqs[i], l))
            first = sum(had[:i])
            assert np.array_equal(gk[:had[i]], old[l][0][first:first + had[i]]) and np.array_equal(gv[:had[i]], old[l][1][first:first + had[i]])
            _check(gk[had[i]:], [t[at:at + news[i]] for t in want], cdt)
            assert np.array_equal(gv[had[i]:], rounded(v[at:at + news[i]], cdt))
            at += news[i]


def test_append_keys_alone_and_in_place(dev):
    """Keys and values without queries; queries in place; positions from a buffer."""
    rng = np.random.default_rng(8)
    K, hd, n = 2, 64, 9
    cache = dev.kv_cache(1, K, hd, 16, 4, 1, 64, F16)
    batch, seqs = cache.batch(1, 16, 4), cache.seq_create(1)
    cos, sin, dc, ds = _tables(dev, hd, 64)
    w, dw = _weights(dev, rng, hd, BF16)
    pos = rng.integers(0, 64, n).astype(np.uint32)
    q, k, v = (_normal(rng, n, h, hd) for h in (4, K, K))
    dq, dk, dv = (dev.upload(t) for t in (q, k, v))
    batch.begin(seqs, [n])
    batch.append_norm(0, None, dk, dv, None, dw[0], dw[1], 1e-6, dc, ds, hd, 1, positions=dev.upload_u32(pos))
    got = from_bits(cache.seq_read(seqs[0], 0)[0].to_numpy(), F16).reshape(n, K, hd)
    _check(got, _formula(k, w[1], 1e-6, cos, sin, pos, hd, 1), F16)
    batch.append_norm(0, dq, dk, dv, dq, dw[0], dw[1], 1e-6, dc, ds, hd, 1)
    _check(dq.to_numpy().reshape(q.shape), _formula(q, w[0], 1e-6, cos, sin, np.arange(n), hd, 1), F32)


def test_replays_give_the_eager_bits(dev):
    """A step captured once, replayed on what the batch begins with later (fewer rows: what lies behind stays)."""
    rng = np.random.default_rng(9)
    K, H, hd, top = 2, 4, 64, 24
    cache = dev.kv_cache(1, K, hd, 16, 12, 3, 64, BF16)
    batch, seqs = cache.batch(3, top, H), cache.seq_create(3)
    _, _, dc, ds = _tables(dev, hd, 64)
    _, dw = _weights(dev, rng, hd, F32)
    x, out = dev.alloc(top * (H + 2 * K) * hd, BF16), dev.alloc(top * H * hd, BF16)
    call = lambda: batch.append_norm(0, x, None, None, out, *dw, 1e-6, dc, ds, hd, 1)  # noqa: E731
    batch.begin(seqs, [1, 1, 1])
    graph = dev.capture(call)
    batch.trim([0, 0, 0])
    for news in ([3, 0, 5], [8, 8, 8], [1, 1, 1]):
        n = sum(news)
        rows = to_bits(_normal(rng, top, H + 2 * K, hd), BF16)
        x.upload(rows)
        batch.begin(seqs, news)
        got = []
        for go in (call, graph.launch):
            out.upload(np.full(top * H * hd, 0x4321, np.uint16))
            go()
            got.append([out.to_numpy()] + [b.to_numpy() for s in seqs for b in cache.seq_read(s, 0)])
        assert all(np.array_equal(a, b) for a, b in zip(*got))
        assert np.all(got[0][0][n * H * hd:] == 0x4321) and not np.any(got[0][0][:n * H * hd] == 0x4321)
    graph.free()


@pytest.mark.parametrize("hd,rot", [(64, 64), (96, 20), (6, 2)])
@pytest.mark.parametrize("xdt,qdt,kdt", [(F32, BF16, F16), (BF16, F32, F16), (F16, BF16, F32), (BF16, BF16, F32), (F16, F32, F16)])
def test_results_of_two_types(dev, hd, rot, xdt, qdt, kdt):
    """Queries and keys that leave in types of their own, from rows of their own and from packed ones."""
    rng = np.random.default_rng(hd + rot + xdt)
    n, H, K = 9, 3, 2
    cos, sin, dc, ds = _tables(dev, rot, 20)
    w, dw = _weights(dev, rng, hd, F32)
    x = rounded(2 * _normal(rng, n, H + K, hd), xdt)
    want = [_formula(t, v, 1e-6, cos, sin, np.arange(n) + 4, rot, 1) for t, v in ((x[:, :H], w[0]), (x[:, H:], w[1]))]
    for packed in (False, True):
        q, k = dev.alloc(n * H * hd, qdt), dev.alloc(n * K * hd, kdt)
        up = lambda t: dev.upload(to_bits(np.ascontiguousarray(t), xdt), xdt)  # noqa: E731
        ins = (up(x), None) if packed else (up(x[:, :H]), up(x[:, H:]))
        dev.qk_norm_rope(*ins, *dw, 1e-6, dc, ds, n, H, K, hd, rot, 1, start_pos=4, q_out=q, k_out=k)
        _check(from_bits(q.to_numpy(), qdt).reshape(n, H, hd), want[0], qdt)
        _check(from_bits(k.to_numpy(), kdt).reshape(n, K, hd), want[1], kdt)


def test_replays_of_a_long_batch_on_few_rows(dev):
    """A step captured for so many rows that lanes take several heads each, replayed on one row, a few and all: the eager bits, and
    what lies behind the rows stays."""
    rng = np.random.default_rng(17)
    K, H, hd, top = 2, 6, 64, 30000
    cache = dev.kv_cache(1, K, hd, 64, 480, 2, top, F16)
    batch, seqs = cache.batch(2, top, H), cache.seq_create(2)
    cos, sin, dc, ds = _tables(dev, 48, top)
    w, dw = _weights(dev, rng, hd, F32)
    x, out = dev.alloc(top * (H + 2 * K) * hd, F16), dev.alloc(top * H * hd, F16)
    call = lambda: batch.append_norm(0, x, None, None, out, *dw, 1e-6, dc, ds, 48, 1)  # noqa: E731
    batch.begin(seqs, [1, 0])
    graph = dev.capture(call)
    batch.trim([0, 0])
    had = np.zeros(2, int)
    for news in ([1, 0], [30, 31], [1, 1], [0, 61], [25000, 4875]):
        n = sum(news)
        rows = rounded(2 * _normal(rng, n, H + 2 * K, hd), F16)
        full = np.zeros(top * (H + 2 * K) * hd, np.uint16)
        full[:rows.size] = to_bits(rows, F16).reshape(-1)
        x.upload(full)
        batch.begin(seqs, news)
        got = []
        for go in (call, graph.launch):
            out.upload(np.full(top * H * hd, 0x4321, np.uint16))
            go()
            got.append([out.to_numpy()] + [b.to_numpy() for i, s in enumerate(seqs) if had[i] + news[i] for b in cache.seq_read(s, 0)])
        assert all(np.array_equal(a, b) for a, b in zip(*got, strict=True))
        assert np.all(got[0][0][n * H * hd:] == 0x4321)
        pos = np.concatenate([np.arange(had[i], had[i] + news[i]) for i in range(2)])
        _check(from_bits(got[0][0][:n * H * hd], F16).reshape(n, H, hd), _formula(rows[:, :H], w[0], 1e-6, cos, sin, pos, 48, 1), F16)
        had += news
    graph.free()
