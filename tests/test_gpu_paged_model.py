"""A decoder composed of the library's operators around the paged cache (embedding, norms, int4 linears, rotary append, attention over
pages, SwiGLU, argmax), serving several sequences at a time, against the CPU oracle's decode and the library's own engine."""
import numpy as np
import pytest

import oracle
from conftest import max_abs_rel
from llama_ref import CONFIG_SMALL, OracleLlama, device_generate, device_llama
from oracle.models import T_KCACHE, T_LM_HEAD, T_VCACHE, T_WD, T_WG, T_WK, T_WO, T_WQ, T_WU, T_WV
from tang_amd import capi

pytestmark = pytest.mark.gpu

F16, BF16 = capi.F16, capi.BF16

# How far logits may be from the oracle's, of the largest. A linear's input that lies near the middle of two bf16 values goes either way: 2^-8 of one of
# 256 terms, 2^-12 of the sum. Once two sides are 1e-4 apart that befalls 1e-4 / 2^-8, some 8 of 256, at each of nine stages (four a layer, the
# head): sqrt(72) 2^-12 = 2e-3 in all; and as much through the cached rows of the steps before.
LOGITS = 4e-3


class Served:
    """CONFIG_SMALL's model with th_llama_init_synthetic's weights, its layers as a program would call them."""

    def __init__(self, dev, cfg, seed, ref, max_seqs):
        self.dev, self.cfg = dev, cfg
        L, d, ff, kvd = cfg["n_layers"], cfg["d_model"], cfg["d_ff"], cfg["n_kv_heads"] * cfg["head_dim"]
        f32 = oracle.bf16_to_f32

        def linear(l, tid, rows, cols):
            nib, sc = capi.synth_q4(capi.synth_seed(seed, l, tid), rows, cols)
            return dev.q4_upload_packed(nib, sc, rows, cols, F16)

        self.w = [{n: linear(l, t, r, c) for n, t, r, c in (("q", T_WQ, d, d), ("k", T_WK, kvd, d), ("v", T_WV, kvd, d), ("o", T_WO, d, d),
                                                            ("g", T_WG, ff, d), ("u", T_WU, ff, d), ("d", T_WD, d, ff))} for l in range(L)]
        self.head = linear(L, T_LM_HEAD, cfg["vocab"], d)
        self.embed = dev.upload(f32(ref.embed))
        self.norms = [[dev.upload(f32(w[l * d:(l + 1) * d])) for l in range(L)] for w in (ref.attn_norm, ref.ffn_norm)]
        self.last_norm = dev.upload(f32(ref.final_norm))
        self.cos, self.sin = (dev.upload(t) for t in capi.rope_tables(cfg["head_dim"], cfg["max_seq"], cfg["rope_theta"]))
        self.cache = dev.kv_cache(L, cfg["n_kv_heads"], cfg["head_dim"], 16, 64, max_seqs, cfg["max_seq"], F16)
        self.batch = self.cache.batch(max_seqs, 256, cfg["n_heads"])

    def prefill(self, s, n, kv_seed):
        """The rows of th_llama_fill_kv_synthetic, already rotated."""
        cfg = self.cfg
        self.batch.begin([s], [n])
        for l in range(cfg["n_layers"]):
            m = n * cfg["n_kv_heads"] * cfg["head_dim"]
            k, v = (self.dev.upload(capi.synth_normal(capi.synth_seed(kv_seed, l, t), m, 1.0, F16), F16) for t in (T_KCACHE, T_VCACHE))
            self.batch.append(l, None, k, v, None)

    def step(self, seqs, ids):
        """One token of each sequence: the next ones, and the logits."""
        dev, cfg, m, d = self.dev, self.cfg, len(seqs), self.cfg["d_model"]

        def norm(x, w):
            return dev.convert(dev.rms_norm(x, w, m, d, cfg["eps"]), BF16)

        self.batch.begin(seqs, [1] * m)
        x = dev.embedding(self.embed, dev.upload_u32(np.asarray(ids, np.uint32)), m, d)
        for l, w in enumerate(self.w):
            h = norm(x, self.norms[0][l])
            q, k, v = (dev.gemm_q4(h, m, w[n]) for n in "qkv")
            self.batch.append(l, q, k, v, q, self.cos, self.sin, cfg["head_dim"], capi.ROPE_INTERLEAVED)
            att = dev.alloc(m * d)
            self.batch.attention(l, q, att)
            x = dev.add_tensors_buf(x, dev.gemm_q4(dev.convert(att, BF16), m, w["o"]), m * d)
            h = norm(x, self.norms[1][l])
            a = dev.swiglu_fused_buf(dev.gemm_q4(h, m, w["g"]), dev.gemm_q4(h, m, w["u"]), m * cfg["d_ff"])
            x = dev.add_tensors_buf(x, dev.gemm_q4(dev.convert(a, BF16), m, w["d"]), m * d)
        logits = dev.gemm_q4(norm(x, self.last_norm), m, self.head).to_numpy().reshape(m, -1)
        return logits.argmax(-1), logits


def test_decode_of_several_sequences(dev):
    """Three prefixes of different lengths, 24 tokens of each, against the oracle one sequence at a time; then two continuations of
    the first one that share its pages, one of them the engine's own."""
    cfg, seed, kv_seed = CONFIG_SMALL, 7, 8
    lens, first = [100, 63, 16], [1, 5, 9]
    refs = [OracleLlama(cfg, seed, kv_seed + i, n) for i, n in enumerate(lens)]
    model = Served(dev, cfg, seed, refs[0], 6)
    seqs = model.cache.seq_create(3)
    for i, s in enumerate(seqs):
        model.prefill(s, lens[i], kv_seed + i)
    base = model.cache.seq_fork(seqs[0], 2)

    def run(seqs, ids, refs, lens, n):
        out = []
        for i in range(n):
            want = [r.step(t, p + i) for r, t, p in zip(refs, ids, lens)]
            ids, logits = model.step(seqs, ids)
            for j, (tok, ref) in enumerate(want):
                assert max_abs_rel(logits[j], ref) < LOGITS, (i, j)
                top = np.sort(ref)[-2:]
                if top[1] - top[0] > 2 * LOGITS * np.abs(ref).max():  # the choice is determined
                    assert ids[j] == tok, (i, j)
            ids = [tok for tok, _ in want]
            out.append(ids)
        return np.array(out).T

    toks = run(seqs, first, refs, lens, 24)
    refs = [OracleLlama(cfg, seed, kv_seed, 100) for _ in range(2)]
    again = run(base, [1, 77], refs, [100, 100], 12)
    assert list(again[0]) == list(toks[0][:12])
    engine = device_llama(dev, cfg, seed, kv_seed, 100)
    try:
        own, logits = device_generate(engine, cfg, 77, 100, 12)
    finally:
        capi.lib().th_llama_destroy(engine)
    assert list(own) == list(again[1])
