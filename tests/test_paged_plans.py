"""Plans of attention over the paged cache, made without a GPU: what their items cover, and how the work is cut."""
import os

import numpy as np
import pytest

from host_cache import CLANG, Cache, build

pytestmark = pytest.mark.skipif(not os.path.exists(CLANG), reason="needs ROCm's clang++")

OWN = 1 << 30


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    return build(tmp_path_factory.mktemp("host"))


def _plan(c, b, seqs, news, heads, window=0, sinks=0):
    """A step's plan, checked: every key that a token sees is in one of its items, every item has keys of its sequence, every record of
    a token is written once. Returns (rows items, tile items)."""
    c.attend(b, sum(news), heads, window, sinks)
    toks, rows, tiles, joins = c.plan(sum(news))
    G = heads // c.kh
    starts = {s: c.length(s) - n for s, n in zip(seqs, news)}
    at = [(s, starts[s] + j) for s, n in zip(seqs, news) for j in range(n)]
    assert sorted(toks[:, 0]) == list(range(len(at)))
    assert all(at[t[0]][1] == t[1] for t in toks)
    seen, recs = [[] for _ in toks], [[] for _ in toks]
    for items, most in ((rows, 16), (tiles, 128)):
        for tok0, ntok, seq, j0, j1, sink_end, gap, rec in items.tolist():
            assert ntok > 0 and ntok * G <= most
            assert j0 < j1, "an item without keys"
            last = j1 - 1 + (gap if j1 - 1 >= sink_end else 0)
            assert last < c.length(seq) and j0 % 16 == 0
            for t in range(tok0, tok0 + ntok):
                for lo, hi, g in ((j0, min(j1, sink_end), 0), (max(j0, sink_end), j1, gap)):
                    if lo < hi:
                        seen[t].append((lo + g, hi + g))
                if rec < 0:
                    recs[t].append(None)
                else:
                    recs[t].append((rec & ~OWN) + (toks[t, 3] & 0xFFFF if rec & OWN else 0))
    joined = {tuple(j) for j in joins.tolist()}
    for t, (row, pos, first, own_n) in enumerate(toks.tolist()):
        ranges = sorted(seen[t])
        assert all(a[1] <= b[0] for a, b in zip(ranges, ranges[1:]))
        cover = np.zeros(pos + 1, bool)
        for a, z in ranges:
            cover[a:z] = True
        j = np.arange(pos + 1)
        need = (j > pos - window) | (j < sinks) if window else j >= 0
        assert (cover | ~need).all(), (row, pos)
        if (row, pos, first, own_n) in joined:
            assert sorted(recs[t]) == list(range(own_n >> 16))
        else:
            assert recs[t] == [None]
    spans = sorted((j[2], j[2] + (j[3] >> 16)) for j in joined)
    assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))
    return rows, tiles


def test_pieces_of_a_very_long_sequence_have_keys(lib):
    """5.2 million keys in pieces of 13107 that begin at multiples of 64: 400 of 13120 were all, and the 401st began behind the sequence's end,
    where the kernel looks up a page before it sees that there is nothing to do."""
    n = 400 * 13107 + 100
    c = Cache(lib, pages=n // 16 + 2, seqs=1, max_len=n)
    b = c.batch(1, 17)
    s = c.create()
    c.resize(s, n - 17)
    c.begin(b, [s], [17])
    _plan(c, b, [s], [17], 1)
    c.call("th_kv_batch_destroy", b)
    c.close()


@pytest.mark.parametrize("seed", range(30))
def test_plans_cover_what_rows_see(lib, seed):
    rng = np.random.default_rng(seed)
    kh, G = int(rng.choice([1, 2])), int(rng.choice([1, 2, 3, 7, 16, 40]))
    page = int(rng.choice([16, 64, 256]))
    c = Cache(lib, kh=kh, page=page, pages=40000 // page + 400, seqs=40, max_len=9000)
    b = c.batch(40, 3000, kh * G)
    first = c.created(int(rng.integers(1, 4)))
    for s in first:
        c.resize(s, int(rng.integers(1, 4000)))
    seqs = list(first)
    for s in first:
        if rng.random() < 0.6:
            seqs += c.fork(s, int(rng.integers(1, 9)), int(rng.integers(0, c.length(s) + 1)))
    for s in seqs:
        if rng.random() < 0.5:
            c.resize(s, c.length(s) + int(rng.integers(0, 300)))
    seqs = [seqs[i] for i in rng.permutation(len(seqs))]
    news = [int(rng.choice([0, 1, 1, 2, 5, int(rng.integers(1, 120))])) for _ in seqs]
    c.begin(b, seqs, news)
    for window, sinks in [(0, 0), (1, 0), (300, 4), (50, 70), (1000, 0)]:
        if sum(news):
            _plan(c, b, seqs, news, kh * G, window, sinks)
    c.call("th_kv_batch_destroy", b)
    c.close()


def _longest(items):
    return int((items[:, 4] - items[:, 3]).max(initial=0))


@pytest.mark.parametrize("new,shared", [(400, 1), (600, 0)])
def test_long_prompts_on_a_prefix_leave_decode_steps_split(lib, new, shared):
    """Eight forks of 2000 positions with 400 or 600 new ones each, more than records are there for with the longer, next to a decode step at
    100000: its keys are cut into pieces all the same. As many of the forks as fit share the prefix."""
    c = Cache(lib, pages=8000, seqs=12, max_len=131072)
    b = c.batch(12, 6000, 4)
    a, far = c.created(2)
    c.resize(a, 2000)
    c.resize(far, 100000)
    kids = c.fork(a, 8, 2000)
    news = [new] * 8 + [1]
    c.begin(b, kids + [far], news)
    rows, tiles = _plan(c, b, kids + [far], news, 4)
    assert _longest(rows) <= 2048
    prefix = tiles[tiles[:, 4] <= 2000]
    assert len(prefix) and (shared or prefix[:, 1].sum() < 2 * 8 * new)
    c.call("th_kv_batch_destroy", b)
    c.close()


def test_thousands_of_rows_on_a_prefix(lib):
    """More forks than records are there for: those that fit share the prefix, whatever came first."""
    c = Cache(lib, pages=3000, seqs=1100, max_len=4096)
    b = c.batch(1100, 6000, 2)
    a = c.create()
    c.resize(a, 1600)
    kids = c.fork(a, 1001, 1600)
    news = [1500] + [4] * 1000
    c.begin(b, kids, news)
    rows, tiles = _plan(c, b, kids, news, 2)
    prefix = tiles[(tiles[:, 3] < 1600) & (tiles[:, 4] <= 1600)]
    assert prefix[:, 1].sum() >= 3000
    c.call("th_kv_batch_destroy", b)
    c.close()


@pytest.mark.parametrize("page", [16, 64])
def test_documents_behind_a_short_common_start(lib, page):
    """Two documents behind the same 64 positions, four answers to each: each document is read once."""
    c = Cache(lib, page=page, pages=4000 // page + 60, seqs=12, max_len=2048)
    b = c.batch(12, 100, 2)
    start = c.create()
    c.resize(start, 64)
    docs = c.fork(start, 2, 64)
    seqs = []
    for d in docs:
        c.resize(d, 1280)
        seqs += c.fork(d, 4, 1280)
    seqs = seqs[::2] + seqs[1::2]
    c.begin(b, seqs, [1] * 8)
    rows, tiles = _plan(c, b, seqs, [1] * 8, 2)
    keys = sum(int((t[:, 4] - t[:, 3]).sum()) for t in (rows, tiles))
    assert keys == 2 * 1280 + 8
    c.call("th_kv_batch_destroy", b)
    c.close()


@pytest.mark.parametrize("rows,max_len,most", [(1, 4096, 1 << 20), (1, 131072, 10 << 20), (64, 1024, 10 << 20), (8192, 131072, 300 << 20)])
def test_memory_of_a_batch(lib, rows, max_len, most):
    """Records for what its rows can have, not for what any batch could."""
    c = Cache(lib, kh=8, hd=128, pages=8, seqs=4, max_len=max_len)
    before = lib.host_bytes()
    b = c.batch(4, rows, 32)
    assert lib.host_bytes() - before <= most
    c.call("th_kv_batch_destroy", b)
    c.close()


@pytest.mark.parametrize("news", [[1], [1, 1, 1, 1], [30], [3, 1]])
@pytest.mark.parametrize("n,window", [(256 * 40 + 1, 0), (3000, 0), (10000, 5000), (300, 0)])
def test_small_batches_are_cut_as_large_ones(lib, news, n, window):
    """A batch with room for just these rows has the plan of one with room for thousands."""
    c = Cache(lib, pages=4000, seqs=9, max_len=256 * 42)
    plans = []
    for most in (sum(news), 4000):
        b = c.batch(len(news), most, 2)
        a = c.create()
        c.resize(a, n)
        seqs = c.fork(a, len(news), n - n % 16)
        c.begin(b, seqs, news)
        c.attend(b, sum(news), 2, window, 4)
        plans.append(c.plan(sum(news)))
        c.free(seqs + [a])
        c.call("th_kv_batch_destroy", b)
    assert all(np.array_equal(x, y) for x, y in zip(*plans))
    c.close()
