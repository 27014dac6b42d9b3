"""The paged cache's bookkeeping without a GPU: calls that find no memory leave everything as it was."""
import ctypes
import os

import numpy as np
import pytest

from host_cache import CLANG, Cache, Refused, build
from tang_amd import capi

pytestmark = pytest.mark.skipif(not os.path.exists(CLANG), reason="needs ROCm's clang++")


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    return build(tmp_path_factory.mktemp("host"))


class _Setup:
    """A long sequence, 150 forks of it that end inside a shared page, one that has been written behind, a batch that has begun (and whose
    attention a graph has), vacant pages before live ones."""

    def __init__(self, L):
        rng = self.rng = np.random.default_rng(1)
        c = self.c = Cache(L, layers=2, pages=24000, seqs=170, max_len=160000)
        self.b = c.batch(160, 12000)
        gap, self.a = c.created(2)
        c.resize(gap, 160000)
        c.grow(rng, self.b, [self.a], [10005])
        c.grow(rng, self.b, [self.a], [11000])
        self.kids = c.fork(self.a, 150, 21003)
        self.other, self.begun = c.created(2)
        c.grow(rng, self.b, [self.other], [30])
        c.free([gap])
        self.b2 = c.batch(160, 12000)
        c.begin(self.b2, [self.begun], [20])
        c.attend(self.b2, 20)
        # another batch, with a plan that a graph reads
        self.c.begin(self.b, [], [])
        c.attend(self.b, 0)
        q = c.buffer(12000 * 8), c.buffer(12000 * 8)
        c.call("th_capture_begin", c.dev)
        c.call("th_kv_batch_attention", self.b, 0, q[0], 0, 0, 0.0, q[1])
        c.new("th_capture_end", c.dev)
        c.fill(rng, self.b2, [self.begun], [20])


def _begin_forks(S):
    news = [1] * len(S.kids) + [9000]
    S.c.begin(S.b, S.kids + [S.other], news)
    return lambda: S.c.fill(S.rng, S.b, S.kids + [S.other], news)


def _begin_few(S):
    S.c.begin(S.b, [S.kids[3], S.a, S.other], [40, 11000, 0])
    return lambda: S.c.fill(S.rng, S.b, [S.kids[3], S.a, S.other], [40, 11000, 0])


def _resize(S):
    S.c.resize(S.kids[5], 160000)
    S.c.resize(S.kids[5], 21003)
    return lambda: None


def _select(S):
    keep = S.rng.permutation(21005)[:20500]
    S.c.select(S.a, keep)
    S.c.rows[S.a] = S.c.rows[S.a][:, :, keep]
    return lambda: None


def _compact(S):
    assert S.c.compact() > 1000
    return lambda: None


@pytest.mark.parametrize("act,least", [(_begin_forks, 3), (_begin_few, 1), (_resize, 1), (_select, 2), (_compact, 2)])
def test_calls_that_find_no_memory_change_nothing(lib, act, least):
    """Every allocation of a call fails in turn: the call is refused, lengths, pages, rows, the books and begun batches are as they were, and
    the same call works afterwards."""
    for fail in range(50):
        S = _Setup(lib)
        c, before = S.c, S.c.info()
        rows = dict(c.rows)
        lib.host_fail(fail)
        try:
            act(S)
            refused = False
        except Refused as e:
            assert e.code == capi.TH_ERR_OOM
            refused = True
        finally:
            lib.host_fail(-1)
        if not refused:
            break
        assert c.info() == before, fail
        c.rows = rows
        c.attend(S.b2, 20)  # still begun
        c.check((act.__name__, fail, "refused"))
        act(S)()
        c.check((act.__name__, fail, "again"))
        c.call("th_kv_batch_destroy", S.b)
        c.call("th_kv_batch_destroy", S.b2)
        c.close()
    assert fail >= least, "too few allocations to have been looked at"


def test_plans_of_graphs_that_are_gone(lib):
    """A step rebuilds the plans that captured graphs read, and no others: not those of a graph that was destroyed. Their memory is used for
    other windows."""
    c = Cache(lib, pages=40, seqs=2, max_len=600)
    b = c.batch(2, 4)
    s = c.create()
    c.resize(s, 300)
    c.begin(b, [s], [1])
    q, o = c.buffer(4 * 8), c.buffer(4 * 8)

    def step():
        n = lib.host_launches()
        c.begin(b, [s], [1])
        return lib.host_launches() - n

    graphs = []
    for windows in (range(10, 20), range(20, 30), range(10, 13)):
        for w in windows:
            c.attend(b, 1, window=w)
        c.call("th_capture_begin", c.dev)
        for w in windows:
            for _ in range(2):
                c.call("th_kv_batch_attention", b, 0, q, w, 0, 0.0, o)
        graphs.append(c.new("th_capture_end", c.dev))
    assert step() == 1 + 20
    c.call("th_graph_destroy", graphs[0])
    assert step() == 1 + 13
    c.call("th_graph_destroy", graphs[1])
    assert step() == 1 + 3
    asked = lib.host_bytes()
    for w in range(30, 60):
        c.attend(b, 1, window=w)
    assert lib.host_bytes() == asked  # no memory for new plans
    assert step() == 1 + 3
    c.call("th_graph_destroy", graphs[2])
    assert step() == 1
    c.call("th_kv_batch_destroy", b)
    c.close()


def test_rows_of_rotary_positions_that_pass_32_bits(lib):
    """2^20 heads of 2^14 dims make 2^31 threads of a row, which the kernel counts in 32 bits: refused, before the buffers are looked at."""
    c = Cache(lib)
    x, t = c.buffer(64), c.buffer(64, capi.F32)
    for heads, hd in ((1 << 20, 1 << 14), (1 << 20, 1 << 16), (1 << 18, 1 << 16)):
        with pytest.raises(Refused, match="sizes out of range") as e:
            c.call("th_rope_rows", c.dev, x, t, t, None, 0, 1, heads, hd, 2, 0, x)
        assert e.value.code == capi.TH_ERR_INVALID
    with pytest.raises(Refused, match="too small"):
        c.call("th_rope_rows", c.dev, x, t, t, None, 0, 1, (1 << 18) - 1, 1 << 16, 2, 0, x)
    c.call("th_rope_rows", c.dev, x, t, t, None, 0, 1, 1, 64, 2, 0, x)
    c.close()


def test_rotated_rows_over_the_tables_they_read(lib):
    """A result in the place of a table that other rows still read."""
    c = Cache(lib, pages=4, seqs=1)
    b, s = c.batch(1, 4, 2), c.create()
    c.begin(b, [s], [4])
    x, kv, t, u = (c.buffer(256, capi.F32) for _ in range(4))
    for cos, sin, out in ((t, u, t), (t, u, u), (t, t, t)):
        for name, args in (("th_rope_rows", (c.dev, x, cos, sin, None, 0, 4, 2, 8, 8, 0, out)),
                           ("th_kv_append", (b, 0, x, kv, kv, cos, sin, None, 8, 0, out))):
            with pytest.raises(Refused, match="table") as e:
                c.call(name, *args)
            assert e.value.code == capi.TH_ERR_INVALID
    c.call("th_rope_rows", c.dev, x, t, u, None, 0, 4, 2, 8, 8, 0, x)
    c.call("th_kv_batch_destroy", b)
    c.close()


def test_scales_that_overflow(lib):
    """3e38 is finite, 3e38 log2(e) is not: every row would be NaN."""
    c = Cache(lib, pages=4, seqs=1)
    b, s = c.batch(1, 4), c.create()
    c.begin(b, [s], [4])
    q, o = c.buffer(256), c.buffer(256)
    for scale in (3e38, float("inf"), float("nan"), -1.0):
        with pytest.raises(Refused, match="scale"):
            c.call("th_kv_batch_attention", b, 0, q, 0, 0, scale, o)
    c.call("th_kv_batch_attention", b, 0, q, 0, 0, 2e38, o)
    c.call("th_kv_batch_destroy", b)
    c.close()


def _fails_in_turn(lib, call, undo=lambda x: None):
    """call() with each of its allocations failing in turn, until none does; how many there were."""
    for fail in range(50):
        lib.host_fail(fail)
        try:
            x = call()
        except Refused as e:
            assert e.code == capi.TH_ERR_OOM
            continue
        finally:
            lib.host_fail(-1)
        undo(x)
        return fail
    raise AssertionError("refused for good")


def test_handles_plans_and_reads_that_find_no_memory(lib):
    """The calls that change no sequence: refused, and the next one works."""
    rng = np.random.default_rng(2)
    c = Cache(lib, pages=4000, seqs=4, max_len=30000)
    cfg = capi.KvCacheConfig(capi.F16, 1, 1, 8, 16, 10, 2, 100)
    assert _fails_in_turn(lib, lambda: c.new("th_kv_cache_create", c.dev, ctypes.byref(cfg)), lambda h: c.call("th_kv_cache_destroy", h)) >= 10
    assert _fails_in_turn(lib, lambda: c.batch(2, 100), lambda h: c.call("th_kv_batch_destroy", h)) == 3
    b, s = c.batch(2, 20000), c.create()
    c.grow(rng, b, [s], [20000])
    assert _fails_in_turn(lib, lambda: c.attend(b, 20000)) >= 2  # the plan's block, its upload
    assert _fails_in_turn(lib, lambda: c.attend(b, 20000, window=50)) >= 1
    kid = c.fork(s, 1, 20000)[0]
    c.select(s, np.arange(20000))  # (the child's table row goes up as entries now)
    c.check()
    c.fork(kid, 1, 20000)
    c.check()
    c.call("th_kv_batch_destroy", b)
    c.close()
