"""Replays of captured attention give the eager calls' bits, however long the cache's sequences may get."""
import numpy as np
import pytest

from paged_ref import rounded, to_bits
from tang_amd import capi
from test_gpu_paged import NAMES, Model, _normal

pytestmark = pytest.mark.gpu

F32, F16, BF16 = capi.F32, capi.F16, capi.BF16


@pytest.mark.parametrize("qdt,cdt", [(F16, F16), (BF16, BF16), (F32, F16)], ids=lambda t: NAMES[t])
@pytest.mark.parametrize("hd", [64, 80])
@pytest.mark.parametrize("max_len", [4096, 40000])
def test_bits_of_replays(dev, qdt, cdt, hd, max_len):
    """Steps of prompts, of decode rows and of both, and one whose items are longer than sums in the MFMAs are for (where the cache
    has room for it), eagerly and replayed."""
    rng = np.random.default_rng(hd)
    m = Model(dev, 2, hd, 16, 3000, 3, 1, max_len, cdt, heads=4, rows=4000)
    seqs = [m.create() for _ in range(3)]
    m.fill(rng, seqs, [700, 3000, 40])
    q, out = dev.alloc(4000 * 4 * hd, qdt), dev.alloc(4000 * 4 * hd, qdt)

    def call():
        m.batch.attention(0, q, out)

    m.batch.begin(seqs, [1, 1, 1])
    call()
    graph = dev.capture(call)
    steps = [[300, 1, 0], [1, 1, 1], [0, 500, 70]]
    if max_len > 20000:
        m.cache.seq_resize(seqs[1], 21000)
        steps.append([0, 3500, 1])
    for news in steps:
        m.batch.begin(seqs, news)
        n = sum(news)
        q.upload(to_bits(rounded(_normal(rng, 4000, 4, hd), qdt), qdt).ravel())
        got = []
        for run in (call, graph.launch):
            dev.zero_buffer(out)
            run()
            dev.sync()
            got.append(out.to_numpy())
        assert got[0][:n * 4 * hd].any() and not got[0][n * 4 * hd:].any()
        assert np.array_equal(*got), (news, int((got[0] != got[1]).sum()))
    graph.free()
