"""A decoder's step as a program strings it together: 8-bit products, head norms
with rotation into a paged cache, attention from it, logits and a token for each row.

Every link is checked against its formula in 64 bits on what the link before
left on the device, so that each has the tolerance of its own; the captured
step gives the eager one's bits on every replay."""
import numpy as np
import pytest

import test_gpu_heads as heads
import test_gpu_i8 as i8
import test_gpu_sample as sample
from paged_ref import EPS, LEAST, attention, attention_bounds, from_bits, rounded, to_bits
from tang_amd import capi

pytestmark = pytest.mark.gpu

F32, BF16 = capi.F32, capi.BF16
HEADS, KV, HD, DIM, VOCAB, PAGE, LAYERS, ROWS = 6, 2, 64, 320, 1000, 16, 2, 96
QKV = (HEADS + 2 * KV) * HD


class Step:
    """Buffers of a program for up to ROWS rows, and its calls."""

    def __init__(self, dev, rng, batch, cos, sin):
        self.dev, self.batch, self.cos, self.sin = dev, batch, cos, sin
        normal = lambda *s: rng.standard_normal(s, dtype=np.float32)  # noqa: E731
        self.table = normal(VOCAB, DIM)
        self.matrix = {}
        for l in range(LAYERS):
            self.matrix[l, "in"] = rounded(normal(QKV, DIM) * DIM ** -0.5, BF16)
            self.matrix[l, "out"] = rounded(normal(DIM, HEADS * HD) * (HEADS * HD) ** -0.5, BF16)
        self.matrix["top"] = rounded(normal(VOCAB, DIM) * 3 * DIM ** -0.5, BF16)
        self.w = {key: dev.q8_quantize(dev.upload(to_bits(m, BF16), BF16), *m.shape) for key, m in self.matrix.items()}
        self.bias = normal(QKV) * np.float32(0.1)
        self.norm = [[rounded(1 + 0.3 * normal(HD), F32) for _ in range(2)] for _ in range(LAYERS)]
        up = dev.upload
        self.d_table, self.d_bias, self.d_norm = up(self.table), up(self.bias), [[up(t) for t in n] for n in self.norm]
        self.ids, self.token = dev.alloc(ROWS, capi.U32), dev.alloc(ROWS, capi.U32)
        self.u, self.temp, self.p = dev.alloc(ROWS), dev.alloc(ROWS), dev.alloc(ROWS)
        self.k = dev.alloc(ROWS, capi.U32)
        f = lambda n, t=F32: dev.alloc(ROWS * n, t)  # noqa: E731
        self.x = [f(DIM) for _ in range(LAYERS + 1)]
        self.qkv, self.q, self.att = ([f(n, BF16) for _ in range(LAYERS)] for n in (QKV, HEADS * HD, HEADS * HD))
        self.add = [f(DIM) for _ in range(LAYERS)]
        self.i8, self.scale = f(HEADS * HD, capi.I8), dev.alloc(ROWS)  # (one of each: every product's rows in turn)
        self.logits, self.share = f(VOCAB), dev.alloc(ROWS)

    def linear(self, x, n, w, y, bias=None):
        self.dev.quantize_rows(x, n, w.cols, self.i8, self.scale)
        self.dev.gemm_i8(self.i8, self.scale, n, w, y, bias)

    def embed(self, ids):
        """(Looks at the ids, so it waits for the device and is not captured.)"""
        self.ids.upload(ids)
        n = len(ids)
        capi.check(capi.lib().th_embedding(self.dev.handle, self.d_table.handle, self.ids.handle, n, DIM, self.x[0].handle))

    def run(self, n):
        L, dev = capi.lib(), self.dev
        for l in range(LAYERS):
            self.linear(self.x[l], n, self.w[l, "in"], self.qkv[l], self.d_bias)
            self.batch.append_norm(l, self.qkv[l], None, None, self.q[l], *self.d_norm[l], 1e-6, self.cos[1], self.sin[1], HD, 1)
            self.batch.attention(l, self.q[l], self.att[l])
            self.linear(self.att[l], n, self.w[l, "out"], self.add[l])
            capi.check(L.th_add(dev.handle, self.x[l].handle, self.add[l].handle, n * DIM, self.x[l + 1].handle))
        self.linear(self.x[LAYERS], n, self.w["top"], self.logits)
        dev.sample_rows(self.logits, n, VOCAB, self.u, self.temp, self.k, self.p, None, self.token, self.share)

    def bits(self, n):
        """What a step of n rows leaves."""
        left = [(self.token, 1), (self.share, 1), (self.logits, VOCAB)] + [(b, b.n // ROWS) for g in (self.qkv, self.q, self.att, self.add, self.x[1:]) for b in g]
        return [b.to_numpy()[:n * each] for b, each in left]

    def check(self, n, ids, settings, positions, rows_of):
        """rows_of: for each sequence its rows of the step."""
        get = lambda b, each: (b.to_numpy() if b.dtype == F32 else from_bits(b.to_numpy(), b.dtype))[:n * each].reshape(n, each)  # noqa: E731
        assert np.array_equal(get(self.x[0], DIM), self.table[ids])
        for l in range(LAYERS):
            x = get(self.x[l], DIM)
            qkv = get(self.qkv[l], QKV)
            self.check_linear(x, (l, "in"), qkv, BF16, self.bias)
            t = qkv.reshape(n, HEADS + 2 * KV, HD)
            q = get(self.q[l], HEADS * HD).reshape(n, HEADS, HD)
            heads._check(q, heads._formula(t[:, :HEADS], self.norm[l][0], 1e-6, self.cos[0], self.sin[0], positions, HD, 1), BF16)
            keys = heads._formula(t[:, HEADS:HEADS + KV], self.norm[l][1], 1e-6, self.cos[0], self.sin[0], positions, HD, 1)
            att = get(self.att[l], HEADS * HD).reshape(n, HEADS, HD)
            for seq, rows in rows_of.items():
                gk, gv = (from_bits(b.to_numpy(), BF16).reshape(-1, KV, HD) for b in self.batch.cache.seq_read(seq, l))
                pos = positions[rows]
                heads._check(gk[pos], [v[rows] for v in keys], BF16)
                assert np.array_equal(gv[pos], t[rows, HEADS + KV:])
                want = attention(q[rows], gk, gv, pos)
                bound = attention_bounds(q[rows], gk, gv, pos, BF16, BF16, BF16)
                assert np.all(np.abs(att[rows] - want) <= bound)
            add = get(self.add[l], DIM)
            self.check_linear(att.reshape(n, -1), (l, "out"), add, F32)
            assert np.array_equal(get(self.x[l + 1], DIM), x + add)
        logits = get(self.logits, VOCAB)
        self.check_linear(get(self.x[LAYERS], DIM), "top", logits, F32)
        token, share = self.token.to_numpy(), self.share.to_numpy()
        for r in range(n):
            want, part, border = sample.choose(logits[r], *[float(s[r]) if i != 2 else int(s[r]) for i, s in enumerate(settings)], 0.0)
            assert border > 1e-9 and token[r] == want
            assert abs(share[r] - part) <= part * 2.0 ** -22

    def check_linear(self, x, key, y, dt, bias=None):
        (q, s), (w, t) = i8._quantized(x), i8._quantized(self.matrix[key])
        if dt == F32:
            assert np.array_equal(y, i8._product(q, s, w, t, bias))
            return
        p = (q.astype(np.int64) @ w.astype(np.int64).T) * s.astype(np.float64)[:, None] * t.astype(np.float64)
        want = p if bias is None else p + bias
        # three roundings of the product in f32, one of the sum, the result's own
        tol = (3 * 2.0 ** -24 * np.abs(p) + 2.0 ** -24 * np.abs(want)) * (1 + 2.0 ** -8) + np.maximum(EPS[dt] * np.abs(want), LEAST[dt])
        assert np.all(np.abs(y - want) <= tol)


def test_steps(dev):
    """Ragged prompts of three sequences, then steps of one token each: eager, and a graph that was captured before the first of them."""
    rng = np.random.default_rng(11)
    cache = dev.kv_cache(LAYERS, KV, HD, PAGE, 24, 3, 120, BF16)
    batch, seqs = cache.batch(3, ROWS, HEADS), cache.seq_create(3)
    cos, sin = capi.rope_tables_scaled(HD, 120, 10000.0)
    step = Step(dev, rng, batch, (cos, dev.upload(cos)), (sin, dev.upload(sin)))

    def settings():
        u, temp = rng.random(ROWS, dtype=np.float32), rng.uniform(0.5, 1.5, ROWS).astype(np.float32)
        k, p = rng.integers(0, 60, ROWS).astype(np.uint32), rng.uniform(0.5, 1.1, ROWS).astype(np.float32)
        temp[::5] = 0
        for b, v in ((step.u, u), (step.temp, temp), (step.k, k), (step.p, p)):
            b.upload(v)
        return u, temp, k, p

    lengths = [37, 1, 33]
    n = sum(lengths)
    ids = rng.integers(0, VOCAB, n).astype(np.uint32)
    step.embed(ids)
    batch.begin(seqs, lengths)
    chosen = settings()
    step.run(n)
    ends = np.cumsum(lengths)
    rows_of = {s: np.arange(e - c, e) for s, c, e in zip(seqs, lengths, ends)}
    step.check(n, ids, chosen, np.concatenate([np.arange(c) for c in lengths]), rows_of)
    ids = step.token.to_numpy()[ends - 1]

    batch.begin(seqs, [1, 1, 1])
    step.run(3)  # (what attention needs is made by a first call)
    graph = dev.capture(lambda: step.run(3))
    batch.trim([0, 0, 0])
    for more in range(4):
        step.embed(ids)
        batch.begin(seqs, [1, 1, 1])
        chosen = settings()
        step.run(3)
        step.check(3, ids, chosen, np.array([c + more for c in lengths]), {s: np.array([i]) for i, s in enumerate(seqs)})
        eager = step.bits(3) + [b.to_numpy() for s in seqs for l in range(LAYERS) for b in cache.seq_read(s, l)]
        for b in step.q + step.qkv + step.att + step.add + step.x[1:] + [step.logits, step.token, step.share]:
            dev.zero_buffer(b)
        graph.launch()
        replay = step.bits(3) + [b.to_numpy() for s in seqs for l in range(LAYERS) for b in cache.seq_read(s, l)]
        assert all(np.array_equal(a, b) for a, b in zip(eager, replay, strict=True))
        ids = step.token.to_numpy()[:3]
    graph.free()
