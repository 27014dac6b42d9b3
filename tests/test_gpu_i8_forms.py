"""Products that take every form of th_gemm_i8 (i8_sizes.py), and batches that go to
the device in slices, against the formulas in 64 bits."""
import numpy as np
import pytest

from i8_sizes import SIZES
from paged_ref import EPS, LEAST, from_bits
from tang_amd import capi
from test_gpu_i8 import _kp, _places, _quantized

pytestmark = pytest.mark.gpu

F32, F16, BF16, I8 = capi.F32, capi.F16, capi.BF16, capi.I8


def _tolerance(p, y, dt):
    """Of a 16-bit result: three half steps of the product in f32, one of the sum, then the result's own rounding."""
    return (3 * 2.0 ** -24 * np.abs(p) + 2.0 ** -24 * np.abs(y)) * (1 + 2.0 ** -8) + np.maximum(EPS[dt] * np.abs(y), LEAST[dt])


@pytest.mark.parametrize("form,m,k,n", SIZES)
def test_form(dev, form, m, k, n):
    """Every type of results, with and without a bias. Rows hold noise behind k, results have room behind them."""
    rng = np.random.default_rng(m + k + n)
    q, wq = (rng.integers(-128, 128, (r, k)).astype(np.int8) for r in (m, n))
    # results of 16 bits stay within f16's range: sums are below 2^14 k
    s, t = np.exp(rng.uniform(-3, 0, m)).astype(np.float32), (np.exp(rng.uniform(-3, 0, n)) / k).astype(np.float32)
    b = rng.standard_normal(n).astype(np.float32)
    rows = rng.integers(-128, 128, m * _kp(k)).astype(np.int8)
    rows[_places(m, _kp(k))[:, :k]] = q
    w, dq, ds, db = dev.q8_upload_rowwise(wq, t, n, k), dev.upload(rows, I8), dev.upload(s), dev.upload(b)
    # sums are below 2^31, so f64 has them exactly
    p = (q.astype(np.float64) @ wq.T.astype(np.float64)) * s.astype(np.float64)[:, None] * t.astype(np.float64)
    for dt, bias in ((F32, None), (F32, db), (BF16, db), (F16, None), (BF16, None)):
        out = dev.upload(np.full(m * n + 7, 9.0, np.float32) if dt == F32 else np.full(m * n + 7, 0x1234, np.uint16), dt)
        dev.gemm_i8(dq, ds, m, w, out, bias)
        got = out.to_numpy()
        assert np.all(got[m * n:] == (9.0 if dt == F32 else 0x1234))
        got = got[:m * n].reshape(m, n)
        y = p if bias is None else p + b.astype(np.float64)
        bad = got != y.astype(np.float32) if dt == F32 else ~(np.abs(from_bits(got, dt) - y) <= _tolerance(p, y, dt))
        assert not bad.any(), (dt, bias is not None, bad.sum(), np.argwhere(bad)[0], got[bad][0], y[bad][0])
        out.free()


@pytest.mark.parametrize("more", [17, 100])
def test_products_in_slices(dev, more):
    """2^21 rows and some more, which a launch of its own takes: few of them, and many."""
    rng = np.random.default_rng(more)
    m, k, n = (1 << 21) + more, 3, 5
    x = rng.integers(-128, 128, m * 64).astype(np.int8)
    w, s, t, b = (rng.integers(-128, 128, (n, k)).astype(np.int8), rng.uniform(1, 2, m).astype(np.float32), rng.uniform(1, 2, n).astype(np.float32),
                  rng.standard_normal(n).astype(np.float32))
    y = dev.gemm_i8(dev.upload(x, I8), dev.upload(s), m, dev.q8_upload_rowwise(w, t, n, k), bias=dev.upload(b)).to_numpy().reshape(m, n)
    p = (x[_places(m, k)].astype(np.float64) @ w.T.astype(np.float64)) * s.astype(np.float64)[:, None] * t.astype(np.float64)
    assert np.array_equal(y, (p + b.astype(np.float64)).astype(np.float32))


def test_rows_quantized_in_slices(dev):
    """2^22 rows and 17 more of one element, as activations and as a weight."""
    rng = np.random.default_rng(3)
    m = (1 << 22) + 17
    x = rng.standard_normal((m, 1)).astype(np.float32)
    q, s = _quantized(x)
    dx = dev.upload(x)
    gq, gs = dev.quantize_rows(dx, m, 1)
    assert np.array_equal(gs.to_numpy(), s)
    got = gq.to_numpy()
    at = _places(m, 1)
    assert np.array_equal(got[at], q)
    got[at] = 0
    assert not got.any()
    gq.free()
    one, unit = dev.upload(np.concatenate((np.array([3], np.int8), np.zeros(63, np.int8))), I8), dev.upload(np.array([0.5], np.float32))
    y = dev.gemm_i8(one, unit, 1, dev.q8_quantize(dx, m, 1)).to_numpy()
    assert np.array_equal(y, (3.0 * q[:, 0].astype(np.float64) * 0.5 * s.astype(np.float64)).astype(np.float32))


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("m", [3, 40, 90])
def test_scales_at_the_ends_of_f32(dev, m, dt):
    """Subnormal scales beside large ones, zeros, infinities and NaN, whose products are ordinary numbers, none, infinite or NaN."""
    rng = np.random.default_rng(m)
    k, n = 70, 36
    q, wq = (rng.integers(-128, 128, (r, k)).astype(np.int8) for r in (m, n))
    wq[:, 0] = 0
    q[:, 1:][0] = 0  # sums of zero
    rows = np.zeros(m * _kp(k), np.int8)
    rows[_places(m, _kp(k))[:, :k]] = q
    ends = np.array([1e-45, 3e-42, 1e-39, 1.2e-38, 1e-30, 1.0, 1e30, 3e38, 0.0, np.inf, np.nan], np.float32)
    s, t = ends[np.arange(m) % len(ends)], ends[rng.permutation(np.arange(n) % len(ends))]
    y = dev.alloc(m * n, dt)
    dev.gemm_i8(dev.upload(rows, I8), dev.upload(s), m, dev.q8_upload_rowwise(wq, t, n, k), y)
    got = y.to_numpy().reshape(m, n)
    with np.errstate(all="ignore"):
        p = (q.astype(np.float64) @ wq.T.astype(np.float64)) * s.astype(np.float64)[:, None] * t.astype(np.float64)
        if dt == F32:
            return np.testing.assert_array_equal(got, p.astype(np.float32))
        got = from_bits(got, dt).astype(np.float64)
        assert np.array_equal(np.isnan(got), np.isnan(p))
        top = {F16: 65520.0, BF16: 3.39e38}[dt]
        over, fine = np.abs(p) > top * (1 + 2.0 ** -7), np.abs(p) < top * (1 - 2.0 ** -7)
        assert np.array_equal(got[over], np.sign(p[over]) * np.inf)
        assert np.all(np.abs(got - p)[fine] <= _tolerance(p, p, dt)[fine] + 2.0 ** -150)
