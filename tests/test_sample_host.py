"""What th_sample_rows refuses, on the host (no GPU)."""
import os

import pytest

from host_operators import CLANG, Cache, Refusals, build
from tang_amd import capi

pytestmark = pytest.mark.skipif(not os.path.exists(CLANG), reason="needs ROCm's clang++")

F32, F16, U32, I32, I8 = capi.F32, capi.F16, capi.U32, capi.I32, capi.I8


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    return build(tmp_path_factory.mktemp("host"))


def test_sample_rows(lib):
    c, other = Cache(lib), Cache(lib)
    r = lambda dt=F32: c.buffer(3, dt)  # noqa: E731
    f = Refusals(c, "th_sample_rows", dev=c.dev, logits=c.buffer(30, F32), rows=3, vocab=10, u=r(), temp=r(), k=r(U32), p=r(), low=r(), tokens=r(U32),
                 prob=r())
    f.call()
    f.call(rows=0)
    f.call(temp=None, k=None, p=None, low=None, prob=None)
    f.call(logits=c.buffer(30, F16), k=r(I32), tokens=r(I32))
    for name in ("dev", "logits", "u", "tokens"):
        f.refused("null", **{name: None})
    f.refused("empty row", vocab=0)
    f.refused("out of range", vocab=(1 << 20) + 1)
    f.refused("out of range", rows=1 << 31)
    f.refused("f32, f16 or bf16", logits=c.buffer(30, I8))
    f.refused("logits .*too small", logits=c.buffer(29, F32))
    for name in ("u", "temp", "p", "low", "prob"):
        f.refused("too small", **{name: c.buffer(2, F32)})
        f.refused("dtype", **{name: r(F16)})
        f.refused("another device", **{name: other.buffer(3, F32)})
    for name in ("k", "tokens"):
        f.refused("too small", **{name: c.buffer(2, U32)})
        f.refused("must be u32", **{name: r()})
        f.refused("another device", **{name: other.buffer(3, U32)})
    x = c.buffer(30, F32)
    f.refused("must not be an input", logits=x, prob=x)
    for name in ("u", "temp", "p", "low"):
        b = r()
        f.refused("must not be an input", prob=b, **{name: b})
    b = r(U32)
    f.refused("must not be an input", k=b, tokens=b)
