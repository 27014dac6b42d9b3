"""Rows to 8-bit integers and their products, against the formulas in 64 bits:
every integer, every f32 result to the bit, 16-bit ones to their rounding."""
import numpy as np
import pytest

from paged_ref import EPS, LEAST, from_bits, rounded, to_bits
from tang_amd import capi

pytestmark = pytest.mark.gpu

F32, F16, BF16, I8 = capi.F32, capi.F16, capi.BF16, capi.I8


def _kp(k):
    return -(-k // 64) * 64


def _places(m, k):
    """Where value (i, k) lies in quantized rows."""
    i, kk = np.arange(m)[:, None], np.arange(k)[None]
    first = i - i % 16
    return first * _kp(k) + (kk - kk % 16) * np.minimum(16, m - first) + i % 16 * 16 + kk % 16


def _quantized(x):
    """(q, scale) of f32 rows. In 64 bits x / s is off by 2^-46 at most, and x / s that is not on a half is at least 2^-26 from it."""
    top = np.abs(x).max(1)
    fine = np.isfinite(x).all(1)
    s = np.where(fine, np.where(fine, top, 0) / np.float32(127), np.nan).astype(np.float32)
    with np.errstate(all="ignore"):
        q = np.rint(x.astype(np.float64) / s.astype(np.float64)[:, None])
    return np.clip(np.where((s > 0)[:, None], q, 0), -127, 127).astype(np.int8), s


def _quantize(dev, x, dt):
    m, k = x.shape
    q, s = dev.alloc(m * _kp(k) + 5, I8), dev.alloc(m + 1)
    q.upload(np.full(q.n, 99, np.int8))
    s.upload(np.full(s.n, 99, np.float32))
    dev.quantize_rows(dev.upload(to_bits(x, dt), dt), m, k, q, s)
    gq, gs = q.to_numpy(), s.to_numpy()
    assert np.all(gq[m * _kp(k):] == 99) and gs[m] == 99
    gq = gq[_places(m, _kp(k))]
    assert not gq[:, k:].any()
    return gq[:, :k], gs[:m]


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("m,k", [(1, 1), (3, 2), (5, 63), (2, 64), (7, 65), (4, 2047), (3, 2048), (2, 4095), (3, 4097), (2, 8192), (2, 11008), (3, 16385),
                                 (2, 131071), (300, 130), (16, 640), (17, 4097), (1024, 33), (1030, 4096), (1040, 5000), (1025, 16400)])
def test_quantize(dev, dt, m, k):
    rng = np.random.default_rng(m * 100 + k)
    x = rng.standard_normal((m, k)) * np.exp(rng.uniform(-8, 8, (m, 1)))
    x = rounded(x.astype(np.float32), dt)
    q, s = _quantized(x)
    gq, gs = _quantize(dev, x, dt)
    assert np.array_equal(gs, s)
    assert np.array_equal(gq, q)


def test_quantize_ties_and_ends(dev):
    """Values on a half, next to it, in rows of any size; rows of zeros, of the smallest numbers, with infinities and NaN."""
    rng = np.random.default_rng(3)
    k = 300
    rows = []
    for e in (-120, -100, -99, -60, -3, 0, 5, 100, 120):  # the scale is 2^e
        r = (rng.integers(-127, 127, k) + 0.5).astype(np.float32) * np.float32(2.0) ** e
        r[0] = np.float32(127.0) * np.float32(2.0) ** e
        rows += [r, np.nextafter(r, np.float32(np.inf)), np.nextafter(r, np.float32(-np.inf))]
        rows[-1][0] = rows[-2][0] = r[0]
    for top in (1.0, 0.3, 7e-39, 2e-42, 1e-40, 3.4e38):  # halves of scales that are no powers of two, as near as they come
        s = np.float32(top) / np.float32(127)
        r = ((rng.integers(-127, 127, k) + 0.5) * float(s)).astype(np.float32)
        r[0] = top
        rows.append(r)
    for tiny in (1, 60, 63, 64, 90, 127, 190, 191):  # multiples of the smallest number
        r = (rng.integers(-tiny, tiny + 1, k) * 2.0 ** -149).astype(np.float32)
        r[0] = tiny * 2.0 ** -149
        rows.append(r)
    rows.append(np.zeros(k, np.float32))
    bad = rng.standard_normal((3, k)).astype(np.float32)
    bad[0, 5], bad[1, 299], bad[2, 0] = np.inf, np.nan, -np.inf
    x = np.concatenate((np.stack(rows), bad))
    q, s = _quantized(x)
    gq, gs = _quantize(dev, x, F32)
    assert np.array_equal(gs, s, equal_nan=True)
    bad = np.argwhere(gq != q)
    assert not len(bad), (bad[0], x[tuple(bad[0])], s[bad[0][0]])


def _product(q, s, w, t, b):
    y = (q.astype(np.int64) @ w.astype(np.int64).T).astype(np.float64)
    with np.errstate(all="ignore"):
        y = y * s.astype(np.float64)[:, None] * t.astype(np.float64)
        return (y if b is None else y + b.astype(np.float64)).astype(np.float32)


def _run(dev, rng, m, k, n, dt=F32, bias=False, w=None):
    """A product whose rows hold noise behind k and whose results have room behind them."""
    q, wq = (rng.integers(-128, 128, (r, k)).astype(np.int8) for r in (m, n))
    s, t = (np.exp(rng.uniform(-9, 3, r)).astype(np.float32) for r in (m, n))
    b = rng.standard_normal(n).astype(np.float32) if bias else None
    rows = rng.integers(-128, 128, m * _kp(k)).astype(np.int8)
    rows[_places(m, _kp(k))[:, :k]] = q
    w = dev.q8_upload_rowwise(wq, t, n, k)
    y = dev.upload(np.full(m * n + 7, 9.0, np.float32) if dt == F32 else np.full(m * n + 7, 0x1234, np.uint16), dt)
    dev.gemm_i8(dev.upload(rows, I8), dev.upload(s), m, w, y, None if b is None else dev.upload(b))
    got = y.to_numpy()
    assert np.all(got[m * n:] == (9.0 if dt == F32 else 0x1234))
    got = got[:m * n].reshape(m, n)
    if dt == F32:
        want = _product(q, s, wq, t, b)
        bad = np.argwhere(got != want)
        assert not len(bad), (len(bad), bad[0], got[tuple(bad[0])], want[tuple(bad[0])])
        return
    # In f32: the sum's, the scales' and their product's rounding (3 half steps of it), the bias' addition (one of the result), then the result's own.
    p = (q.astype(np.int64) @ wq.astype(np.int64).T) * s.astype(np.float64)[:, None] * t.astype(np.float64)
    y = p if b is None else p + b
    tol = (3 * 2.0 ** -24 * np.abs(p) + 2.0 ** -24 * np.abs(y)) * (1 + 2.0 ** -8) + np.maximum(EPS[dt] * np.abs(y), LEAST[dt])
    top = {F16: 65520.0, BF16: 3.39e38}[dt]  # what rounds to infinity
    got = from_bits(got, dt)
    fine = np.abs(y) < top * (1 - 2.0 ** -10)
    bad = np.argwhere(fine & ~(np.abs(got - y) <= tol))
    assert not len(bad), (len(bad), bad[0], got[tuple(bad[0])], y[tuple(bad[0])])
    over = np.abs(y) > top * (1 + 2.0 ** -10)
    assert np.array_equal(got[over], np.sign(y[over]) * np.inf)


SIZES = [(1, 1, 1), (1, 64, 16), (1, 4096, 250), (3, 65, 17), (2, 11008, 40), (16, 130, 33), (17, 2047, 100), (31, 320, 64), (33, 64, 15), (61, 4096, 300),
         (64, 1000, 48), (65, 192, 130), (100, 2048, 1000), (128, 128, 128), (129, 257, 255), (200, 513, 400), (256, 256, 256), (300, 4100, 700),
         (509, 2047, 631), (1030, 640, 1100)]


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("dt,bias", [(F32, False), (BF16, True), (F16, False), (F32, True)])
def test_product(dev, m, k, n, dt, bias):
    _run(dev, np.random.default_rng(m + k + n), m, k, n, dt, bias)


def test_product_of_the_largest(dev):
    """Sums next to 2^31, all terms of one sign; scales whose products with a sum or with each other leave f32's range."""
    k = 131071
    for m in (2, 40, 300):
        q, w = np.full((m, k), -128, np.int8), np.full((5, k), -128, np.int8)
        rows = np.zeros(m * _kp(k), np.int8)
        rows[_places(m, _kp(k))[:, :k]] = q
        s = np.where(np.arange(m) % 2 == 0, 1e-30, 2e36).astype(np.float32)
        t = np.array([1e-30, 1e-10, 1.0, 0.0, 1e30], np.float32)
        y = dev.gemm_i8(dev.upload(rows, I8), dev.upload(s), m, dev.q8_upload_rowwise(w, t, 5, k))
        with np.errstate(over="ignore"):
            want = _product(q[:2], s[:2], w, t, None)
        got = y.to_numpy().reshape(m, 5)
        assert np.array_equal(got, want[np.arange(m) % 2])
        assert np.isinf(got[1, 4]) and got[0, 4] != 0 and got[1, 3] == 0
        y16 = dev.alloc(m * 5, BF16)
        dev.gemm_i8(dev.upload(rows, I8), dev.upload(s), m, dev.q8_upload_rowwise(w, t, 5, k), y16)
        got16 = from_bits(y16.to_numpy(), BF16).reshape(m, 5)
        fine = np.isfinite(got)
        assert np.array_equal(np.isfinite(got16), fine)
        assert np.all(np.abs(got16[fine].astype(np.float64) - got[fine]) <= (EPS[BF16] + 2.0 ** -22) * np.abs(got[fine]) + LEAST[BF16])


def test_rows_without_a_scale(dev):
    """A row with a NaN has a NaN scale: its products are NaN, the others' are not."""
    x = np.random.default_rng(1).standard_normal((20, 100)).astype(np.float32)
    x[7, 3] = np.nan
    x[9, 4] = np.inf
    x[11] = 0
    w = np.random.default_rng(2).integers(-127, 128, (30, 100)).astype(np.int8)
    q, s = dev.quantize_rows(dev.upload(x), 20, 100)
    y = dev.gemm_i8(q, s, 20, dev.q8_upload_rowwise(w, np.ones(30, np.float32), 30, 100)).to_numpy().reshape(20, 30)
    bad = np.isnan(y).all(1)
    assert list(np.flatnonzero(bad)) == [7, 9] and np.isfinite(y[~bad]).all() and not y[11].any()


@pytest.mark.parametrize("rows,cols", [(1, 1), (16, 64), (17, 65), (250, 1000), (100, 4096)])
def test_packed_weights(dev, rows, cols):
    """A weight packed on the device is the one that the host packs: the same bits from both products that take it. Columns behind its end do not count."""
    rng = np.random.default_rng(rows + cols)
    wq = rng.integers(-127, 128, (rows, cols)).astype(np.int8)
    t = rng.uniform(0.001, 0.01, rows).astype(np.float32)
    noisy = rng.integers(-127, 128, (rows, _kp(cols))).astype(np.int8)
    noisy[:, :cols] = wq
    a, b = dev.q8_upload_rowwise(wq, t, rows, cols), dev.q8_pack_rows(dev.upload(noisy, I8), dev.upload(t), rows, cols)
    x = dev.upload(rng.standard_normal((5, cols)).astype(np.float32))
    q, s = dev.quantize_rows(x, 5, cols)
    behind = q.to_numpy()
    behind[_places(5, _kp(cols))[:, cols:]] = 77
    q.upload(behind)
    assert np.array_equal(dev.gemv_q8(x, 5, a).to_numpy(), dev.gemv_q8(x, 5, b).to_numpy())
    assert np.array_equal(dev.gemm_i8(q, s, 5, a).to_numpy(), dev.gemm_i8(q, s, 5, b).to_numpy())


def test_weights_quantized_on_the_device(dev):
    """A float matrix quantized and packed on the device, and its product with quantized rows against the exact one of the floats.

    Both operands are off by half a step of their scale at most: |y - x.w| <= sum |x| t/2 + |w| s/2 + s t/4 a term."""
    rng = np.random.default_rng(4)
    m, k, n = 70, 900, 130
    x, w = rng.standard_normal((m, k)).astype(np.float32), rng.standard_normal((n, k)).astype(np.float32)
    qx, sx = dev.quantize_rows(dev.upload(x), m, k)
    y = dev.gemm_i8(qx, sx, m, dev.q8_quantize(dev.upload(w), n, k)).to_numpy().reshape(m, n)
    qw, tw = _quantized(w)
    assert np.array_equal(y, _product(_quantized(x)[0], _quantized(x)[1], qw, tw, None))
    s, t = sx.to_numpy().astype(np.float64)[:, None], tw.astype(np.float64)
    bound = np.abs(x).sum(1, dtype=np.float64)[:, None] * t / 2 + np.abs(w).sum(1, dtype=np.float64) * s / 2 + k * s * t / 4
    want = x.astype(np.float64) @ w.astype(np.float64).T
    assert np.all(np.abs(y - want) <= bound * (1 + 2.0 ** -20))


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (15, 64), (16, 100), (33, 4097), (1100, 130), (1030, 4200), (2, 20000)])
def test_weight_of_a_matrix(dev, dt, rows, cols):
    """th_q8_quantize's weight is the one that the quantized rows make: rows behind the last in its tiles are zeros."""
    rng = np.random.default_rng(rows + cols)
    w = rounded(rng.standard_normal((rows, cols)).astype(np.float32), dt)
    q, s = _quantized(w)
    x = dev.upload(rng.standard_normal((3, cols)).astype(np.float32))
    qx, sx = dev.quantize_rows(x, 3, cols)
    a, b = dev.q8_quantize(dev.upload(to_bits(w, dt), dt), rows, cols), dev.q8_upload_rowwise(q, s, rows, cols)
    assert np.array_equal(dev.gemm_i8(qx, sx, 3, a).to_numpy(), dev.gemm_i8(qx, sx, 3, b).to_numpy())
    if cols < 5000:
        assert np.array_equal(dev.gemv_q8(x, 3, a).to_numpy(), dev.gemv_q8(x, 3, b).to_numpy())


def test_captured(dev):
    """Quantization and products captured into one graph, replayed on new rows with eager work between: the eager bits."""
    rng = np.random.default_rng(5)
    for m, k, n in ((1, 4096, 512), (40, 1000, 300), (300, 2048, 600)):
        w = dev.q8_upload_rowwise(rng.integers(-127, 128, (n, k)).astype(np.int8), np.ones(n, np.float32), n, k)
        x, y = dev.alloc(m * k), dev.alloc(m * n)
        q, s = dev.alloc(m * _kp(k), I8), dev.alloc(m)

        def call():
            dev.quantize_rows(x, m, k, q, s)
            dev.gemm_i8(q, s, m, w, y)
        call()
        graph = dev.capture(call)
        for _ in range(3):
            x.upload(rng.standard_normal(m * k).astype(np.float32))
            call()
            want = y.to_numpy()
            dev.zero_buffer(y)
            graph.launch()
            assert np.array_equal(y.to_numpy(), want)
        graph.free()


def test_results_beyond_32_bits_of_places(dev):
    """More than 2^31 results, and rows of quantized values that begin beyond 2^31 bytes of the results."""
    m, k, n = 67200, 64, 32000
    rng = np.random.default_rng(6)
    x = rng.integers(-128, 128, m * k).astype(np.int8)
    w, s, t = rng.integers(-128, 128, (n, k)).astype(np.int8), rng.uniform(1, 2, m).astype(np.float32), rng.uniform(1, 2, n).astype(np.float32)
    y = dev.alloc(m * n, BF16)
    dev.gemm_i8(dev.upload(x, I8), dev.upload(s), m, dev.q8_upload_rowwise(w, t, n, k), y)
    got = y.to_numpy().reshape(m, n)
    y.free()
    for rows in (range(0, 20), range(67100, 67121), range(67184, 67200)):
        q = x[_places(m, k)[list(rows)]]
        p = (q.astype(np.int64) @ w.astype(np.int64).T) * s[list(rows)].astype(np.float64)[:, None] * t.astype(np.float64)
        tol = 3 * 2.0 ** -24 * np.abs(p) * (1 + 2.0 ** -8) + np.maximum(EPS[BF16] * np.abs(p), LEAST[BF16])
        assert np.all(np.abs(from_bits(got[list(rows)], BF16) - p) <= tol)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("bias", [False, True])
def test_rows_have_their_bits_in_any_batch(dev, dt, bias):
    """A row's results are the same bits alone, among few rows and among many."""
    rng = np.random.default_rng(21)
    m, k, n = 300, 1000, 2000
    x = rng.standard_normal((m, k)).astype(np.float32) * np.exp(rng.uniform(-3, 3, (m, 1))).astype(np.float32)
    w = dev.q8_quantize(dev.upload(rng.standard_normal((n, k)).astype(np.float32)), n, k)
    b = dev.upload(rng.standard_normal(n).astype(np.float32)) if bias else None

    def rows(first, count):
        q, s = dev.quantize_rows(dev.upload(x[first:first + count]), count, k)
        return dev.gemm_i8(q, s, count, w, dev.alloc(count * n, dt), b).to_numpy().reshape(count, n)
    want = rows(0, m)
    assert len(set(want.reshape(-1).tolist())) > 1000
    for first, count in ((0, 1), (7, 16), (20, 31), (100, 64), (40, 65), (3, 200)):
        got = rows(first, count)
        bad = np.argwhere(got != want[first:first + count])
        assert not len(bad), (count, len(bad), bad[0])
