"""Host side of the paged cache's operators: scaled rotary tables, and null arguments."""
import ctypes

import numpy as np
import pytest

import oracle
from tang_amd import capi


def _freqs(rot, base, kind, factor, low, high, original):
    i = np.arange(rot // 2, dtype=np.float64)
    if kind == "base":
        base = base * factor ** (rot / (rot - 2.0))
    f = 1.0 / base ** (2.0 * i / rot)
    if kind == "linear":
        return f / factor
    if kind == "bands":
        wave = 2 * np.pi / f
        out = np.where(wave > original / low, f / factor, f)
        mid = (wave <= original / low) & (wave >= original / high)
        s = (original / wave - low) / (high - low)
        return np.where(mid, (1 - s) * f / factor + s * f, out)
    if kind == "ramp":
        def index(turns):
            return rot * np.log(original / (turns * 2 * np.pi)) / (2 * np.log(base))
        lo, hi = max(np.floor(index(high)), 0), min(np.ceil(index(low)), rot - 1)
        r = np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
        return f / factor * r + f * (1 - r)
    return f


@pytest.mark.parametrize("rot,base", [(128, 10000.0), (64, 500000.0), (20, 10000.0), (4, 100.0)])
@pytest.mark.parametrize("kind,factor,low,high", [("plain", 1.0, 1.0, 4.0), ("linear", 4.0, 1.0, 4.0), ("base", 2.5, 1.0, 4.0),
                                                  ("bands", 8.0, 1.0, 4.0), ("ramp", 16.0, 1.0, 32.0), ("ramp", 1.0, 1.0, 32.0)])
def test_scaled_tables(rot, base, kind, factor, low, high):
    """Angles in 64 bits on both sides: frequencies are off by some 2^-52 of themselves (a
    power and a few products, 8 steps), an angle below 2^14 so by 2^-35 at most, and the table by
    that and half a step of f32 (values up to 1.3)."""
    n, original = 9000, 2048
    c, s = capi.rope_tables_scaled(rot, n, base, kind=kind, factor=factor, low=low, high=high, original_len=original)
    a = np.arange(n, dtype=np.float64)[:, None] * _freqs(rot, base, kind, factor, low, high, original)
    warm = 0.1 * np.log(factor) + 1.0 if kind == "ramp" else 1.0
    assert c.shape == s.shape == (n, rot // 2)
    tol = 2.0 ** -35 + 2.0 ** -24 * 1.3
    assert np.abs(c - np.cos(a) * warm).max() <= tol and np.abs(s - np.sin(a) * warm).max() <= tol


def test_plain_tables_are_rope_tables():
    """The same angles up to the last step of a frequency: at positions below 300 2^-43, next to f32's 2^-24."""
    c, s = capi.rope_tables_scaled(128, 300, 10000.0)
    oc, os_ = oracle.rope_tables(128, 300, 10000.0)
    assert np.abs(c.ravel() - oc).max() <= 2.0 ** -23 and np.abs(s.ravel() - os_).max() <= 2.0 ** -23


def test_warmth_is_taken_as_given():
    c, _ = capi.rope_tables_scaled(64, 10, 10000.0, kind="ramp", factor=8.0, low=1.0, high=32.0, original_len=4096, warmth=2.0)
    assert np.array_equal(c[0], np.full(32, 2.0, np.float32))


def test_refused_scalings():
    ok = dict(kind="ramp", factor=4.0, low=1.0, high=32.0, original_len=4096)
    for bad in (dict(ok, factor=0.5), dict(ok, factor=float("nan")), dict(ok, low=0.0), dict(ok, low=33.0), dict(ok, original_len=0),
                dict(ok, kind="bands", original_len=0), dict(kind="linear", factor=0.0), dict(kind="base", factor=float("inf"))):
        with pytest.raises(capi.TangHipError):
            capi.rope_tables_scaled(64, 4, 10000.0, **bad)
    for rot, base in ((63, 1e4), (0, 1e4), (64, 1.0), (64, float("nan"))):
        with pytest.raises(capi.TangHipError):
            capi.rope_tables_scaled(rot, 4, base)
    with pytest.raises(capi.TangHipError):
        capi.rope_tables_scaled(2, 4, 1e4, kind="base", factor=2.0)
    s = capi.RopeScaling(7, 1.0, 1.0, 4.0, 0.0, 0)
    t = np.empty(128, np.float32)
    assert capi.lib().th_rope_tables_scaled(64, 4, 1e4, ctypes.byref(s), capi.ptr(t), capi.ptr(t)) == capi.TH_ERR_INVALID


def test_null_arguments_are_errors():
    L, bad = capi.lib(), capi.TH_ERR_INVALID
    assert L.th_kv_cache_create(None, None, None) == bad and b"null" in L.th_last_error()
    assert L.th_kv_cache_destroy(None) == 0 and L.th_kv_batch_destroy(None) == 0
    assert L.th_kv_cache_info(None, None, None) == bad
    assert L.th_kv_cache_pages(None, 0, None, None) == bad
    assert L.th_kv_cache_compact(None, None) == bad
    assert L.th_kv_seq_create(None, 1, None) == bad
    assert L.th_kv_seq_free(None, None, 0) == bad
    assert L.th_kv_seq_len(None, 0, None) == bad
    assert L.th_kv_seq_resize(None, 0, 0) == bad
    assert L.th_kv_seq_fork(None, 0, 0, 0, None) == bad
    assert L.th_kv_seq_select(None, 0, None, 0) == bad
    assert L.th_kv_seq_read(None, 0, 0, 0, 0, None, None) == bad
    assert L.th_kv_batch_create(None, 1, 1, 1, None) == bad
    assert L.th_kv_batch_begin(None, None, None, 0) == bad
    assert L.th_kv_batch_trim(None, None, 0) == bad
    assert L.th_kv_append(None, 0, None, None, None, None, None, None, 0, 0, None) == bad
    assert L.th_kv_batch_attention(None, 0, None, 0, 0, 0.0, None) == bad
    assert L.th_rope_rows(None, None, None, None, None, 0, 0, 1, 8, 0, 0, None) == bad
    assert L.th_buffer_ptr(None, None) == bad
