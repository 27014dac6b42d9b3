// Attention over a paged cache for tiles of up to 128 rows (new tokens x query
// heads of one kv head): prompts, and shared prefixes whose sequences' rows make
// up one tile.
//
// Workgroup = (item, kv head); its four waves have 32 rows each and share blocks
// of keys in LDS, the next block's loads in flight meanwhile.  The products are
// transposed as in kvattn_rows.hpp, on the 32x32x16 MFMA: S^T = K.Q^T leaves lane (h, c) of
// row c the keys 8i + 4h .. + 3 of each 32, and the numbering of the
// contraction in O^T += V^T.P^T follows that (slots 8h .. 8h + 7 of a step of 16 keys are
// keys 4h .. 4h + 3 and 8 + 4h ..), so probabilities never leave their lane.
//
// Bound by the SIMDs' issue: the MFMAs' time and the softmax's vector instructions (four for a score, six with two parts) add up.
// A prompt of 8192 (bf16, 32 heads of 128 on 8): 600 to 620 us by box, 890 to 915 TFLOP/s of what rows see, where a large matrix product
// reaches 1231.  Eight waves in two phases, wave priorities, two chains of MFMAs and blocks of 32 keys
// with three workgroups a CU gave nothing more.  f32 queries on an f16 cache take twice the MFMAs.
#pragma once

#include "kvattn.hpp"

namespace th {

template <int D, int NP>
struct KvTiles {
    static constexpr int KB = D <= 64 || (D <= 128 && NP == 1) ? 64 : 32;  // what the registers hold
    // LDS rows of K end in 16 bytes (16-byte reads of 16 rows then meet all banks),
    // those of V in 64 (the transposing reads take 32 bytes of each of four rows).
    // Two blocks: one is filled while the other is read.
    static constexpr int LK = D + 8, LV = D + 32;
    static constexpr size_t LDS = (size_t)2 * KB * (LK + LV) * 2;
};

// One item by a workgroup.  ADD: a block's sum of values is added to the sums so far in plain additions, since an
// MFMA may drop bits of what it adds to a larger sum.  Results of 16 bits do not see that over the KV_LONG_ITEM keys that an item
// without ADD has at most: 1024 steps of 16 keys lose less than 2^-23 of the sum so far each, 1.2e-4 together, next to a
// rounding of 5e-4 (f16) or 4e-3 (bf16).  (Over 20000 keys with values of one sign the mean error of f16 results was -7e-7 without ADD and -6e-7
// with it.  Without ADD the sums cost no vector instruction.)
template <int D, typename E, int NP, bool PAD, bool ADD>
__device__ __forceinline__ void kv_tiles_item(const KvAttnArgs& a, const KvItem& it, int hk, char* lds_) {
    typedef KvTiles<D, NP> T;
    typedef typename KvVec<E>::x8 x8;
    constexpr int KB = T::KB, LK = T::LK, LV = T::LV, KT = KB / 32, NS = D / 16, NDT = D / 32, CPR = D / 8;
    constexpr int NL = KB * CPR / 256, DE = D / 64;
    E(*lds)[KB * (LK + LV)] = (E(*)[KB * (LK + LV)])lds_;
    const KvTok* toks = a.toks;
    const int G = a.n_heads / a.pages.n_kv_heads, hd = PAD ? a.pages.hd : D, nch = hd / 8;
    const int tid = kv_fresh(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = lane >> 5, c = lane & 31;
    KvGroups groups(a.pages, it);
    const int R = it.ntok * G;
    // token and query head of a row
    auto tok_of = [&](int row) { return toks[it.tok0 + row / G]; };
    auto head_of = [&](int row) { return hk * G + row % G; };
    const KvTok tok = tok_of(min(wave * 32 + c, R - 1));
    // piece i of this thread: 16 bytes of row (tid + 256 i) / CPR
    kv_u4_t kr[NL], vr[NL];
    constexpr int RPI = 256 / CPR;  // rows a load of the workgroup covers
    const uint32_t off = (uint32_t)(tid / CPR % 16 * hd + (PAD ? min(tid % CPR, nch - 1) : tid % CPR) * 8) * 2;
    auto load = [&](int j0) {
        groups.reach(a.pages, it, j0 >> 4);
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int group = RPI * i / 16 + (RPI > 16 ? wave * RPI / 64 : 0);
            const size_t at = groups.at(a.pages, it, hk, hd, (j0 >> 4) + group);
            const uint32_t o = off + (uint32_t)(RPI < 16 ? RPI * i % 16 * hd * 2 : 0);
            kr[i] = kv_load16<E>(a.pages.k, at, o);
            vr[i] = kv_load16<E>(a.pages.v, at, o);
        }
    };
    load(it.j0);

    // which blocks need no mask, and which no work, for this wave's rows
    const KvSeen see(it, tok.pos, a.window, a.sinks);
    int hi_lo = see.hi, hi_hi = see.hi, to_lo = see.to, to_hi = see.to;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) {
        hi_lo = min(hi_lo, __shfl_xor(hi_lo, x, 64));
        hi_hi = max(hi_hi, __shfl_xor(hi_hi, x, 64));
        to_lo = min(to_lo, __shfl_xor(to_lo, x, 64));
        to_hi = max(to_hi, __shfl_xor(to_hi, x, 64));
    }
    hi_lo = __builtin_amdgcn_readfirstlane(hi_lo);
    hi_hi = __builtin_amdgcn_readfirstlane(hi_hi);
    to_lo = __builtin_amdgcn_readfirstlane(to_lo);
    to_hi = __builtin_amdgcn_readfirstlane(to_hi);
    const int hidden = __builtin_amdgcn_readfirstlane(see.from);  // the same for all rows

    // the queries: B operand, lane (h, c) dims 16s + 8h.. of row c
    x8 q[NP][NS];
    int qe = 0;
    const size_t q_at = ((size_t)tok.row * a.n_heads + head_of(min(wave * 32 + c, R - 1))) * hd;
    if constexpr (NP == 1) {
#pragma unroll
        for (int s = 0; s < NS; s++) {
            q[0][s] = *(const x8*)((const E*)a.q + q_at + (PAD ? min(2 * s + h, nch - 1) : 2 * s + h) * 8);
            if (PAD && 2 * s + h >= nch) q[0][s] = x8{};
        }
    } else {
        float x[NS][8], mx = 0.0f;
        kv_load_row<NS>(a.q, a.qdt, q_at, [&](int s) { return PAD ? min(2 * s + h, nch - 1) : 2 * s + h; }, x);
#pragma unroll
        for (int s = 0; s < NS; s++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (PAD && 2 * s + h >= nch) x[s][i] = 0.0f;
                mx = fmaxf(mx, fabsf(x[s][i]));
            }
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        qe = range_exp(mx, KV_Q_TOP);
#pragma unroll
        for (int s = 0; s < NS; s++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                E part[NP];
                kv_split<E, NP>(__builtin_amdgcn_ldexpf(x[s][i], -qe), part);
#pragma unroll
                for (int u = 0; u < NP; u++) q[u][s][i] = part[u];
            }
    }
    const float scale = NP == 1 ? a.scale : __builtin_amdgcn_ldexpf(a.scale, qe);
    float m = -INFINITY, l = 0.0f;
    kv_f32x16_t o[NDT];
#pragma unroll
    for (int t = 0; t < NDT; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[t][i] = 0.0f;

    auto block = [&](const E* ks, const E* vs, int j) {
        if (j > hi_hi || (j >= hidden && j + KB - 1 <= to_lo)) return;  // wave-uniform: no row sees any of it
        const int ln = kv_fresh(lane);
        // S^T.  The operands of a step are read while the step before it is in the MFMAs.
        kv_f32x16_t s[KT];
        {
            constexpr int XS = NS < 2 ? 1 : 2, STEPS = KT * NS / XS;
            const E* kp = ks + (ln & 31) * LK + 8 * (ln >> 5);
            x8 ka[2][XS];
            auto read = [&](int i) {
#pragma unroll
                for (int y = 0; y < XS; y++) ka[i & 1][y] = *(const x8*)(kp + (i * XS / NS) * 32 * LK + (i * XS % NS + y) * 16);
            };
            read(0);
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int e = 0; e < 16; e++) s[t][e] = 0.0f;
#pragma unroll
            for (int i = 0; i < STEPS; i++) {
                if (i + 1 < STEPS) read(i + 1);
                __builtin_amdgcn_sched_barrier(0);
                const int t = i * XS / NS;
#pragma unroll
                for (int y = 0; y < XS; y++)
#pragma unroll
                    for (int u = NP - 1; u >= 0; u--) s[t] = kv_mfma32(ka[i & 1][y], q[u][i * XS % NS + y], s[t]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        kv_mfma_wait();
        if (j + KB - 1 > hi_lo || (j <= to_hi && j + KB - 1 >= hidden)) {
            const int hi = see.hi - j - 4 * h, from = see.from - j - 4 * h, to = see.to - j - 4 * h;
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int x = t * 32 + 8 * (i >> 2) + (i & 3);
                    s[t][i] = (x <= hi) & ((x < from) | (x > to)) ? s[t][i] : -INFINITY;
                }
        }
        float bm = kv_max3(s[0][0], s[0][1], s[0][2]);
#pragma unroll
        for (int i = 3; i < KT * 16 - 1; i += 2) bm = kv_max3(bm, s[i >> 4][i & 15], s[(i + 1) >> 4][(i + 1) & 15]);
        bm = kv_max3(bm, s[KT - 1][15], __shfl_xor(kv_max3(bm, bm, s[KT - 1][15]), 32, 64)) * scale;
        float f = 1.0f;
        if constexpr (NP == 1) {
            // The sums' reference follows the maximum only when that has risen by 2^6: weights up to
            // 64 have the same relative rounding, and the sums are seldom rescaled.
            bm -= kv_tiles_low<E>();
            if (__any(bm > m + KV_LAG)) {
                const float mn = fmaxf(m, bm);
                f = kv_exp2(m - (mn == -INFINITY ? 0.0f : mn));
                m = mn;
#pragma unroll
                for (int t = 0; t < NDT; t++)
#pragma unroll
                    for (int i = 0; i < 16; i++) o[t][i] *= f;
                l *= f;
            }
        } else {
            const float mn = fmaxf(m, bm);
            f = kv_exp2(m - (mn == -INFINITY ? 0.0f : mn));
            m = mn;
            l *= f;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        float ps = 0.0f;
        x8 p[NP][KT * 2];
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float e0 = kv_exp2(__builtin_fmaf(s[t][i], scale, -ref)), e1 = kv_exp2(__builtin_fmaf(s[t][i + 1], scale, -ref));
                typename KvVec<E>::x2 part[NP];
                kv_split_pair<E, NP>(e0, e1, NP == 1 ? 1.0f : KV_P_UP, part);
                if constexpr (NP == 1) {
                    ps = kv_add_pair(part[0], ps);
                } else {
                    ps += e0;
                    ps += e1;
                }
#pragma unroll
                for (int u = 0; u < NP; u++) {
                    p[u][2 * t + (i >> 3)][i & 7] = part[u][0];
                    p[u][2 * t + (i >> 3)][(i & 7) + 1] = part[u][1];
                }
            }
        l += ps;  // this lane's keys; the row's two lanes meet at the end
        {
            typedef short s8 __attribute__((ext_vector_type(8)));
            constexpr int XS = 2, PER = KT * 2 / XS, STEPS = NDT * PER;
            // lane 4k + i of sixteen addresses four dims of key k and gets its dim of four keys
            kv_lds_s4_t* vp = (kv_lds_s4_t*)(vs + (4 * (ln >> 5) + ((ln & 15) >> 2)) * LV + (ln & 16) + 4 * (ln & 3));
            s8 va[2][XS];
            auto read = [&](int i) {
#pragma unroll
                for (int y = 0; y < XS; y++) {
                    kv_s4_t w[2];
#pragma unroll
                    for (int z = 0; z < 2; z++)
                        w[z] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(vp + ((16 * (i % PER * XS + y) + 8 * z) * LV + i / PER * 32) / 4);
                    va[i & 1][y] = s8{w[0][0], w[0][1], w[0][2], w[0][3], w[1][0], w[1][1], w[1][2], w[1][3]};
                }
            };
            read(0);
            kv_f32x16_t d;
#pragma unroll
            for (int i = 0; i < STEPS; i++) {
                const int dt = i / PER, x0 = i % PER * XS;
                if (x0 == 0) {
#pragma unroll
                    for (int e = 0; e < 16; e++) d[e] = ADD ? 0.0f : o[dt][e];
                }
                if (i + 1 < STEPS) read(i + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int y = 0; y < XS; y++)
#pragma unroll
                    for (int u = NP - 1; u >= 0; u--) d = kv_mfma32(__builtin_bit_cast(x8, va[i & 1][y]), p[u][x0 + y], d);
                if (x0 + XS == KT * 2) {
#pragma unroll
                    for (int e = 0; e < 16; e++) o[dt][e] = !ADD ? d[e] : NP == 1 ? o[dt][e] + d[e] : __builtin_fmaf(o[dt][e], f, d[e]);
                }
                if (i + 1 < STEPS) __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    for (int j = it.j0, b = 0; j < it.j1; j += KB, b ^= 1) {
        E *ks = lds[b], *vs = ks + KB * LK;
        const int ti = kv_fresh(tid);
#pragma unroll
        for (int i = 0; i < NL; i++) {
            *(kv_u4_t*)(ks + ti / CPR * LK + ti % CPR * 8 + i * RPI * LK) = kr[i];
            *(kv_u4_t*)(vs + ti / CPR * LV + ti % CPR * 8 + i * RPI * LV) = vr[i];
        }
        // behind the barrier the block is whole, and the other buffer's reads (a block ago) are done
        __syncthreads();
        load(j + KB);  // past the last: its last group again
        block(ks, vs, j);
    }
    kv_mfma_wait();
    l += __shfl_xor(l, 32, 64);
    bool fine = kv_fine(m, l);
#pragma unroll
    for (int t = 0; t < NDT; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
            if constexpr (NP > 1) o[t][i] *= 1.0f / KV_P_UP;
            fine &= fabsf(o[t][i]) <= 3.402823466e38f;
        }
    const bool live = wave * 32 + c < R;
    if (live) {
        const int row = wave * 32 + kv_fresh(c), hq = head_of(row);
        const KvTok t = tok_of(row);
        const size_t at = ((size_t)t.row * a.n_heads + hq) * hd, rec = it.rec < 0 ? 0 : kv_record(it, t, a.n_heads, hq);
        const float inv = it.rec < 0 ? 1.0f / l : 1.0f;
#pragma unroll
        for (int t = 0; t < NDT; t++)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int d = t * 32 + 2 * i + 4 * h;
                if (PAD && d >= hd) continue;
                const kv_f32x4_t x = {o[t][i] * inv, o[t][i + 1] * inv, o[t][i + 2] * inv, o[t][i + 3] * inv};
                if (it.rec < 0) kv_store_out4(a.out, a.odt, at + d, x);
                else *(kv_f32x4_t*)(a.rec_o + rec * hd + d) = x;
            }
        if (it.rec >= 0 && h == 0) a.rec_ml[rec] = make_float2(m, l);
    }
    uint64_t todo = __ballot(live && !fine);
    todo = (todo | (todo >> 32)) & 0xFFFFFFFFull;
    for (; todo; todo &= todo - 1) {
        const int rw = wave * 32 + (int)__builtin_ctzll(todo);
        const KvTok t = tok_of(rw);
        const int hx = head_of(rw);
        const size_t at = ((size_t)t.row * a.n_heads + hx) * hd;
        float pm, pl, acc[DE];
        kv_row_plain<E, DE>(a, it, groups.table, hk, at, t.pos, it.j0, KB, KB, pm, pl, acc);
        const size_t rx = it.rec < 0 ? 0 : kv_record(it, t, a.n_heads, hx);
#pragma unroll
        for (int e = 0; e < DE; e++) {
            if (lane + 64 * e >= hd) continue;
            if (it.rec < 0) kv_store_out(a.out, a.odt, at + lane + 64 * e, acc[e] / pl);
            else a.rec_o[rx * hd + lane + 64 * e] = acc[e];
        }
        if (it.rec >= 0 && lane == 0) a.rec_ml[rx] = make_float2(pm, pl);
    }
}

}  // namespace th
