"""What the calls that bring heads to their norm refuse, on the host (no GPU)."""
import os

import pytest

from host_cache import CLANG, Cache, Refused, build
from tang_amd import capi

pytestmark = pytest.mark.skipif(not os.path.exists(CLANG), reason="needs ROCm's clang++")

F32, F16, BF16, U32, I8 = capi.F32, capi.F16, capi.BF16, capi.U32, capi.I8


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    return build(tmp_path_factory.mktemp("host"))


def test_rows_refusals(lib):
    c, other = Cache(lib), Cache(lib)
    q, k, qo, ko, w, cos, sin = (c.buffer(n, F32) for n in (4 * 3 * 8, 4 * 2 * 8, 4 * 3 * 8, 4 * 2 * 8, 8, 40, 40))
    good = dict(dev=c.dev, q=q, q_stride=0, k=k, k_stride=0, qw=w, kw=w, eps=1e-6, cos=cos, sin=sin, pos=None, start=0, rows=4, heads=3, kv=2, hd=8,
                rot=8, layout=1, q_out=qo, k_out=ko)

    def call(**over):
        c.call("th_qk_norm_rope", *{**good, **over}.values())

    def refused(match, **over):
        with pytest.raises(Refused, match=match) as e:
            call(**over)
        assert e.value.code == capi.TH_ERR_INVALID

    call()
    call(q_out=q, k_out=k)  # in place
    call(qw=None, kw=None, cos=None, sin=None, rot=0)
    call(rows=0, q=c.buffer(1, F32), k=c.buffer(1, F32))
    packed = c.buffer(4 * 7 * 8, F32)
    call(q=packed, k=None, q_stride=56)
    call(q=packed, k=None, q_stride=56, q_out=packed, k_out=None)
    call(q=packed, k=None, q_stride=56, q_out=packed)
    call(q=c.buffer(3 * 56 + 40, F32), k=None, q_stride=56)  # the last row ends with its keys
    for name in ("dev", "q", "q_out"):
        refused("null", **{name: None})
    refused("f32, f16 or bf16", q=c.buffer(96, U32))
    refused("of this device", q_out=other.buffer(96, F32))
    refused("of one type", k=c.buffer(64, F16))
    refused("too small", q=c.buffer(95, F32))
    refused("too small", k=c.buffer(63, F32))
    refused("too small", q_out=c.buffer(95, F32))
    refused("too small", k_out=c.buffer(63, F32))
    refused("too small", q=c.buffer(3 * 56 + 39, F32), k=None, q_stride=56)
    refused("too small", q_out=qo, k_out=None)  # the keys behind the queries
    refused("shorter than its row", q_stride=23)
    refused("shorter than its row", k_stride=15)
    refused("shorter than its row", q=packed, k=None, q_stride=39)
    refused("a stride of no keys", q=packed, k=None, k_stride=16)
    refused("no room for the keys", q_out=q, k_out=None)
    refused("keys without key heads", kv=0)
    refused("no queries", heads=0)
    refused("no queries", hd=0)
    for over in (dict(heads=1 << 17), dict(kv=1 << 17), dict(hd=1 << 17), dict(rows=1 << 31), dict(q_stride=1 << 32), dict(start=2 ** 64 - 2)):
        refused("out of range", **over)
    refused("buffers of their own", k=q)
    refused("buffers of their own", k_out=qo)
    big = c.buffer(96, F32)
    refused("others read", k=big, q_out=big)
    refused("others read", k_out=q)
    refused("others read", qw=big, q_out=big)
    refused("others read", kw=big, k_out=big)
    refused("table", cos=qo, q=q)
    refused("table", sin=ko)
    refused("tables end", start=7)
    refused("null table", cos=None)
    refused("even", rot=7)
    refused("even", rot=10)
    refused("layout", layout=2)
    refused("weight", qw=c.buffer(7, F32))
    refused("weights must be", kw=c.buffer(8, F16))
    refused("weight is on another", kw=other.buffer(8, F32))
    refused("positions", pos=c.buffer(3, U32))
    refused("positions", pos=c.buffer(4, F32))
    for eps in (-1e-6, float("nan"), float("inf")):
        refused("eps", eps=eps)


def test_append_refusals(lib):
    c, other = Cache(lib, kh=2, pages=4, seqs=1), Cache(lib)
    b, s = c.batch(1, 4, 4), c.create()
    q, k, v, qo = (c.buffer(n, F16) for n in (128, 64, 64, 128))
    w, cos, sin = (c.buffer(n, F32) for n in (8, 16, 16))
    packed = c.buffer(4 * 8 * 8, F16)
    good = dict(b=b, layer=0, q=q, k=k, v=v, qw=w, kw=w, eps=1e-6, cos=cos, sin=sin, pos=None, rot=8, layout=1, q_out=qo)

    def refused(match, **over):
        with pytest.raises(Refused, match=match) as e:
            c.call("th_kv_append_norm", *{**good, **over}.values())
        assert e.value.code == capi.TH_ERR_INVALID

    refused("not begun")
    c.begin(b, [s], [4])
    refused("null batch", b=None)
    refused("no layer", layer=1)
    refused("k and v go together", v=None)
    refused("q and q_out go together", q_out=None)
    refused("q and q_out go together", q=None)
    refused("null", q=None, q_out=None, k=None, v=None)
    refused("too small", k=None, v=None)  # q alone holds no keys
    refused("packed rows", q=packed, k=None, v=None, q_out=packed)
    big = c.buffer(128, F16)
    refused("others read", k=big, q_out=big)
    refused("others read", v=big, q_out=big)
    refused("of one type", k=c.buffer(64, F32))
    refused("too small", q_out=c.buffer(127, F16))
    refused("f32, f16 or bf16", q_out=c.buffer(128, I8))
    refused("another device", q_out=other.buffer(128, F16))
    refused("tables end", cos=c.buffer(15, F32))
    refused("eps", eps=-1.0)
    refused("weights must be", qw=c.buffer(8, F16))
