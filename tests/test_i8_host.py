"""What the 8-bit products' calls refuse, on the host (no GPU)."""
import ctypes
import os

import pytest

import i8_sizes
from host_operators import CLANG, Cache, Refusals, Refused, build
from tang_amd import capi

pytestmark = pytest.mark.skipif(not os.path.exists(CLANG), reason="needs ROCm's clang++")

F32, F16, I8, U8 = capi.F32, capi.F16, capi.I8, capi.U8


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    return build(tmp_path_factory.mktemp("host"))


def test_quantize_rows(lib):
    c, other = Cache(lib), Cache(lib)
    f = Refusals(c, "th_quantize_rows", dev=c.dev, x=c.buffer(3 * 65, F32), m=3, k=65, q=c.buffer(3 * 128, I8), scale=c.buffer(3, F32))
    f.call()
    f.call(m=0)
    f.call(x=c.buffer(3 * 65, F16))
    for name in ("dev", "x", "q", "scale"):
        f.refused("null", **{name: None})
    f.refused("f32, f16 or bf16", x=c.buffer(3 * 65, I8))
    f.refused("k must", k=0)
    f.refused("k must", k=1 << 17)
    f.refused("too many rows", m=1 << 31)
    f.refused("buffer x .*too small", x=c.buffer(3 * 65 - 1, F32))
    f.refused("buffer q .*too small", q=c.buffer(3 * 128 - 1, I8))
    f.refused("dtype", q=c.buffer(3 * 128, U8))
    f.refused("dtype", scale=c.buffer(3, F16))
    f.refused("buffer scale .*too small", scale=c.buffer(2, F32))
    for name, n, dt in (("x", 195, F32), ("q", 384, I8), ("scale", 3, F32)):
        f.refused("another device", **{name: other.buffer(n, dt)})
    x = c.buffer(195, F32)
    f.refused("must not be x", x=x, scale=x)


def test_pack_and_product(lib):
    c, other = Cache(lib), Cache(lib)
    q, s = c.buffer(20 * 128, I8), c.buffer(20, F32)
    out = ctypes.c_void_p()
    f = Refusals(c, "th_q8_pack_rows", dev=c.dev, q=q, scale=s, rows=20, cols=70, out=ctypes.byref(out))
    f.call()
    w = ctypes.c_void_p(out.value)
    for name in ("dev", "q", "scale", "out"):
        f.refused("null", **{name: None})
    f.refused("empty", rows=0)
    f.refused("empty", cols=0)
    f.refused("out of range", cols=1 << 17)
    f.refused("out of range", rows=1 << 27)
    f.refused("another device", q=other.buffer(20 * 128, I8))
    f.refused("buffer q .*too small", q=c.buffer(20 * 128 - 1, I8))
    f.refused("buffer scale .*too small", scale=c.buffer(19, F32))
    # a failed allocation leaves nothing behind
    for n in range(2):
        lib.host_fail(n)
        f.refused("hipMalloc", code=capi.TH_ERR_OOM)
    lib.host_fail(-1)

    x = c.buffer(20 * 70, F32)
    z = Refusals(c, "th_q8_quantize", dev=c.dev, x=x, rows=20, cols=70, out=ctypes.byref(out))
    z.call()
    c.call("th_qweight_free", ctypes.c_void_p(out.value))
    z.refused("null", x=None)
    z.refused("null", out=None)
    z.refused("empty", rows=0)
    z.refused("out of range", cols=1 << 17)
    z.refused("another device", x=other.buffer(20 * 70, F32))
    z.refused("buffer x .*too small", x=c.buffer(20 * 70 - 1, F32))
    z.refused("f32, f16 or bf16", x=c.buffer(20 * 70, I8))

    y = c.buffer(3 * 20, F32)
    g = Refusals(c, "th_gemm_i8", dev=c.dev, xq=c.buffer(3 * 128, I8), xs=c.buffer(3, F32), m=3, w=w, bias=None, y=y)
    g.call()
    g.call(m=0)
    g.call(bias=c.buffer(20, F32), y=c.buffer(60, F16))
    for name in ("dev", "xq", "xs", "w", "y"):
        g.refused("null", **{name: None})
    g.refused("buffer xq .*too small", xq=c.buffer(3 * 128 - 1, I8))
    g.refused("dtype", xq=c.buffer(3 * 128, U8))
    g.refused("buffer x_scale .*too small", xs=c.buffer(2, F32))
    g.refused("buffer bias .*too small", bias=c.buffer(19, F32))
    g.refused("dtype", bias=c.buffer(20, F16))
    g.refused("buffer y .*too small", y=c.buffer(59, F32))
    g.refused("f32, f16 or bf16", y=c.buffer(60, I8))
    g.refused("out of range", m=1 << 31)
    g.refused("must not be an input", xs=y)
    g.refused("must not be an input", bias=y)
    g.refused("another device", y=other.buffer(60, F32))
    lib.host_rows(w, ctypes.c_size_t(1 << 27))
    g.refused("out of range")
    lib.host_rows(w, ctypes.c_size_t(20))
    lib.host_grouped(w, 8, 0)
    g.refused("each group", code=capi.TH_ERR_UNSUPPORTED)
    lib.host_grouped(w, 4, 1)
    g.refused("not q8")
    lib.host_grouped(w, 8, 1)
    g.call()
    c.call("th_qweight_free", w)
    c.call("th_capture_begin", c.dev)
    f.refused("capture")
    z.refused("capture")


def test_as_many_rows_as_a_launch_takes(lib):
    """A launch has 32 threads for each weight row at most (512 for 16 of them), and below 2^32 of them in all: weights of up to 2^27 - 16 rows,
    as more are 2^27 in whole tiles of 16."""
    c = Cache(lib)
    out = ctypes.c_void_p()
    q, s, x = c.buffer(64, I8), c.buffer(1, F32), c.buffer(1, F32)
    pack = Refusals(c, "th_q8_pack_rows", dev=c.dev, q=q, scale=s, rows=1, cols=1, out=ctypes.byref(out))
    make = Refusals(c, "th_q8_quantize", dev=c.dev, x=x, rows=1, cols=1, out=ctypes.byref(out))
    pack.call()
    w = ctypes.c_void_p(out.value)
    g = Refusals(c, "th_gemm_i8", dev=c.dev, xq=q, xs=s, m=0, w=w, bias=None, y=x)
    for rows in ((1 << 27) - 15, (1 << 27) - 1):
        pack.refused("out of range", rows=rows)
        make.refused("out of range", rows=rows)
        lib.host_rows(w, ctypes.c_size_t(rows))
        g.refused("out of range")
    # one tile fewer is taken (the buffers are too small for such weights)
    pack.refused("too small", rows=(1 << 27) - 16)
    make.refused("too small", rows=(1 << 27) - 16)
    lib.host_rows(w, ctypes.c_size_t((1 << 27) - 16))
    g.call()
    lib.host_rows(w, ctypes.c_size_t(1))
    c.call("th_qweight_free", w)


def test_every_form_of_a_product_is_run(lib):
    """The sizes that the GPU tests run take, by the rule on a card of 256 CUs, the forms that stand beside them: each of them, with rows and channels
    that are no whole tiles and a k of no whole chunks."""
    lib.host_i8_form.argtypes = [ctypes.c_size_t] * 4
    names = [i8_sizes.FORMS[lib.host_i8_form(m, n, k, 256)] for _, m, k, n in i8_sizes.SIZES]
    assert names == [s[0] for s in i8_sizes.SIZES]
    for f in i8_sizes.FORMS:
        mine = [s for s in i8_sizes.SIZES if s[0] == f]
        assert any(m % 16 and n % 16 for _, m, k, n in mine) and any(k % 64 for _, m, k, n in mine) and any(-(-k // 64) % 4 > 0 for _, m, k, n in mine), f


def test_launches_of_a_product(lib):
    """Slices of rows are whole blocks of 16; a launch has below 2^32 threads and 2^16 tiles of rows."""
    lib.host_i8_rows.argtypes, lib.host_i8_rows.restype = [ctypes.c_size_t], ctypes.c_size_t
    lib.host_i8_form.argtypes = [ctypes.c_size_t] * 4
    threads = {"tile 64x64": 256, "tile 64x128, two groups": 512, "tile 64x128": 256, "tile 128x128": 256, "tile 128x256": 256, "tile 256x256": 256}
    for n in (1, 16, 17, 4096, 32000, (1 << 20) + 5, 1 << 24, (1 << 27) - 16):
        rows = lib.host_i8_rows(n)
        assert rows % 16 == 0 and 16 <= rows <= 1 << 21
        for m in (1, 17, 33, 65, 129, rows):
            if m > rows:
                continue
            form = i8_sizes.FORMS[lib.host_i8_form(m, n, 64, 256)]
            kind, size = form.split(",")[0].split()
            a, b = (int(v) for v in size.split("x"))
            if kind == "rows":
                assert -(-n // 16 // a) * 512 < 1 << 32 and -(-m // 16) <= b
            else:
                assert -(-m // a) * -(-n // b) * threads[form] < 1 << 32 and -(-m // a) < 1 << 16
