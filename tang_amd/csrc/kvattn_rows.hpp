// Attention over a paged cache for at most 16 rows (new tokens x query heads of
// one kv head): decode steps.
//
//   o = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m),  s_j = q.k_j * scale * log2(e)
//
// over the keys that the row sees, in one pass with the running maximum m.
// Workgroup = (item, kv head); its four waves take 32-key blocks in turn, each
// with a softmax state of its own.  Both products are transposed: S^T = K.Q^T
// takes K as it lies in memory as the first operand and leaves lane (g, r) the
// scores of row r for keys 4g..4g+3 of each 16, which is the operand that
// O^T += V^T.P^T wants; V^T comes out of row-major LDS by transposing reads.
//
// A step over long caches is bound by the reads of K and V: 48 sequences of 100 to 16000 positions (bf16, 32 heads of
// 128 on 8) take 120 us, 5.4 TB/s, with a block of loads in flight for each wave and two workgroups a CU.
// Eight waves to a workgroup read slower (143 us).  One sequence of 8192 positions is bound by latency: item,
// pages, first rows, two blocks, the waves' join take 11 us, the records' join 4.5 us.
#pragma once

#include "kvattn.hpp"

namespace th {

template <int D>
struct KvRows {
    static constexpr int NK = D / 32, NDT = D / 16, LD = D + 8, KB = 32, CPR = D / 8, VL = KB * CPR / 64;
    // a wave's V rows, then its 16 rows of sums
    static constexpr size_t REGION = (size_t)KB * LD * 2 > (size_t)16 * D * 4 ? (size_t)KB * LD * 2 : (size_t)16 * D * 4;
    static constexpr size_t LDS = 4 * REGION + 9 * 16 * 4;  // and the waves' maxima and sums
};

// One item by a workgroup.
template <int D, typename E, int NP, bool PAD>
__device__ __forceinline__ void kv_rows_item(const KvAttnArgs& a, const KvItem& it, int h, char* lds) {
    typedef KvRows<D> W;
    typedef typename KvVec<E>::x8 x8;
    constexpr int NK = W::NK, NDT = W::NDT, LD = W::LD, KB = W::KB, CPR = W::CPR, VL = W::VL, DE = D / 64;
    constexpr int PP = NP == 1 ? 2 : NP;  // parts of a weight (kvattn.hpp)
    constexpr size_t REGION = W::REGION;
    float(*sm)[16] = (float(*)[16])(lds + 4 * REGION), (*sl)[16] = sm + 4, *sM = sl[4];
    const KvTok* toks = a.toks;
    const int G = a.n_heads / a.pages.n_kv_heads, hd = PAD ? a.pages.hd : D, nch = hd / 8;
    const int tid = kv_fresh(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, r = lane & 15;
    E* vs = (E*)(lds + wave * REGION);
    const int R = it.ntok * G, row = min(r, R - 1);
    const KvTok tok = toks[it.tok0 + row / G];
    KvGroups groups(a.pages, it);
    auto q_at = [&](const KvTok& t, int rw) { return ((size_t)t.row * a.n_heads + h * G + rw % G) * hd; };

    // K: lane (g, r) has row r of each group, pieces 4c + g.  V: piece lane + 64 i of the block.
    kv_u4_t k[2][NK], v[VL];
    size_t at[2];
    auto place = [&](int j0) {
        groups.reach(a.pages, it, j0 >> 4);
#pragma unroll
        for (int t = 0; t < 2; t++) at[t] = groups.at(a.pages, it, h, hd, (j0 >> 4) + t);
    };
    auto load_k = [&]() {
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int c = 0; c < NK; c++)
                k[t][c] = kv_load16<E>(a.pages.k, at[t], (uint32_t)(r * hd + (PAD ? min(4 * c + g, nch - 1) : 4 * c + g) * 8) * 2);
    };
    auto load_v = [&]() {
#pragma unroll
        for (int i = 0; i < VL; i++) {
            constexpr int RPI = 64 / CPR;  // rows a load covers
            const int c = lane % CPR, row = lane / CPR + RPI * i % 16;
            v[i] = kv_load16<E>(a.pages.v, at[RPI * i / 16], (uint32_t)(row * hd + (PAD ? min(c, nch - 1) : c) * 8) * 2);
        }
    };
    int j = it.j0 + wave * KB;
    place(j);
    load_k();
    load_v();

    // the queries: B operand, lane (g, r) dims 32c + 8g.. of row r
    x8 q[NP][NK];
    int qe = 0;
    if constexpr (NP == 1) {
#pragma unroll
        for (int c = 0; c < NK; c++) {
            q[0][c] = *(const x8*)((const E*)a.q + q_at(tok, row) + (PAD ? min(4 * c + g, nch - 1) : 4 * c + g) * 8);
            if (PAD && 4 * c + g >= nch) q[0][c] = x8{};
        }
    } else {
        float x[NK][8], mx = 0.0f;
        kv_load_row<NK>(a.q, a.qdt, q_at(tok, row), [&](int c) { return PAD ? min(4 * c + g, nch - 1) : 4 * c + g; }, x);
#pragma unroll
        for (int c = 0; c < NK; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (PAD && 4 * c + g >= nch) x[c][i] = 0.0f;
                mx = fmaxf(mx, fabsf(x[c][i]));
            }
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        qe = range_exp(mx, KV_Q_TOP);
#pragma unroll
        for (int c = 0; c < NK; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                E part[NP];
                kv_split<E, NP>(__builtin_amdgcn_ldexpf(x[c][i], -qe), part);
#pragma unroll
                for (int u = 0; u < NP; u++) q[u][c][i] = part[u];
            }
    }
    const float scale = NP == 1 ? a.scale : __builtin_amdgcn_ldexpf(a.scale, qe);
    const KvSeen see(it, tok.pos, a.window, a.sinks);
    float m = -INFINITY, l = 0.0f;
    kv_f32x4_t o[NDT];
#pragma unroll
    for (int t = 0; t < NDT; t++) o[t] = kv_f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

    for (; j < it.j1; j += 4 * KB) {
        kv_f32x4_t s[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            s[t] = kv_f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int u = NP - 1; u >= 0; u--)  // the small parts first
#pragma unroll
                for (int c = 0; c < NK; c++) s[t] = kv_mfma16(__builtin_bit_cast(x8, k[t][c]), q[u][c], s[t]);
        }
        // the next block (past the last: its last group again)
        place(j + 4 * KB);
        load_k();
        float bm = -INFINITY;
        const int hi = see.hi - j - 4 * g, from = see.from - j - 4 * g, to = see.to - j - 4 * g;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int x = 16 * t + i;
                s[t][i] = (x <= hi) & ((x < from) | (x > to)) ? s[t][i] : -INFINITY;
                bm = fmaxf(bm, s[t][i]);
            }
        bm = fmaxf(bm, __shfl_xor(bm, 16, 64));
        bm = fmaxf(bm, __shfl_xor(bm, 32, 64)) * scale;
        if constexpr (NP == 1) bm -= kv_rows_low<E>();
        const float mn = fmaxf(m, bm), ref = mn == -INFINITY ? 0.0f : mn, f = kv_exp2(m - ref);
        float ps = 0.0f;
        x8 p[PP];
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const float e0 = kv_exp2(__builtin_fmaf(s[t][i], scale, -ref)), e1 = kv_exp2(__builtin_fmaf(s[t][i + 1], scale, -ref));
                ps += e0;
                ps += e1;
                typename KvVec<E>::x2 part[PP];
                kv_split_pair<E, PP>(e0, e1, NP == 1 ? 1.0f : KV_P_UP, part);
#pragma unroll
                for (int u = 0; u < PP; u++) {
                    p[u][4 * t + i] = part[u][0];
                    p[u][4 * t + i + 1] = part[u][1];
                }
            }
        l = l * f + ps;  // this lane's keys; the row's lanes meet at the end
        m = mn;
#pragma unroll
        for (int i = 0; i < VL; i++)
            *(kv_u4_t*)(vs + (lane + 64 * i) / CPR * LD + lane % CPR * 8) = v[i];
        wave_lds_fence();
        load_v();
        kv_lds_s4_t* vp = (kv_lds_s4_t*)(vs + (4 * g + (r >> 2)) * LD + 4 * (r & 3));
#pragma unroll
        for (int dt = 0; dt < NDT; dt++) {
            // lane r addresses four dims of key r >> 2 of its group's four, and gets its dim of all four
            kv_s4_t w[2];
#pragma unroll
            for (int t = 0; t < 2; t++)
                w[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(vp + (16 * t * LD + dt * 16) / 4);
            typedef short s8 __attribute__((ext_vector_type(8)));
            const x8 va = __builtin_bit_cast(x8, (s8){w[0][0], w[0][1], w[0][2], w[0][3], w[1][0], w[1][1], w[1][2], w[1][3]});
            kv_f32x4_t d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int u = PP - 1; u >= 0; u--) d = kv_mfma16(va, p[u], d);
#pragma unroll
            for (int i = 0; i < 4; i++) o[dt][i] = __builtin_fmaf(o[dt][i], f, d[i]);
        }
        wave_lds_fence();  // the rows are rewritten by the next block
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    bool fine = kv_fine(m, l);
#pragma unroll
    for (int t = 0; t < NDT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (NP > 1) o[t][i] *= 1.0f / KV_P_UP;
            fine &= fabsf(o[t][i]) <= 3.402823466e38f;
        }
    float* mo = (float*)vs;  // [16][D]
#pragma unroll
    for (int t = 0; t < NDT; t++) *(kv_f32x4_t*)(mo + r * D + t * 16 + 4 * g) = o[t];
    if (g == 0) { sm[wave][r] = m; sl[wave][r] = l; }
    if (__any(!fine)) {
        wave_lds_fence();
        for (int rw = 0; rw < R; rw++) {
            const KvTok t = toks[it.tok0 + rw / G];
            float pm, pl, acc[DE];
            kv_row_plain<E, DE>(a, it, groups.table, h, q_at(t, rw), t.pos, it.j0 + wave * KB, KB, 4 * KB, pm, pl, acc);
#pragma unroll
            for (int e = 0; e < DE; e++) mo[rw * D + lane + 64 * e] = acc[e];
            if (lane == 0) { sm[wave][rw] = pm; sl[wave][rw] = pl; }
        }
    }
    __syncthreads();
    if (tid < 16) {  // row tid: the waves' weights relative to the workgroup's maximum, and their sum
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int x = 0; x < 4; x++) M = fmaxf(M, sm[x][tid]);
#pragma unroll
        for (int x = 0; x < 4; x++) {
            const float f = sm[x][tid] == -INFINITY && sl[x][tid] == 0.0f ? 0.0f : kv_exp2(sm[x][tid] - M);
            L = __builtin_fmaf(f, sl[x][tid], L);
            sm[x][tid] = f;
        }
        sM[tid] = M;
        sl[0][tid] = L;
    }
    __syncthreads();
    for (int i = tid; i < R * D; i += 256) {
        const int rw = i / D, d = i % D;
        if (PAD && d >= hd) continue;
        float A = 0.0f;
#pragma unroll
        for (int x = 0; x < 4; x++) A = __builtin_fmaf(sm[x][rw], ((const float*)(lds + x * REGION))[rw * D + d], A);
        const KvTok t = toks[it.tok0 + rw / G];
        const int hq = h * G + rw % G;
        if (it.rec < 0) {
            kv_store_out(a.out, a.odt, ((size_t)t.row * a.n_heads + hq) * hd + d, A / sl[0][rw]);
        } else {
            const size_t rec = kv_record(it, t, a.n_heads, hq);
            a.rec_o[rec * hd + d] = A;
            if (d == 0) a.rec_ml[rec] = make_float2(sM[rw], sl[0][rw]);
        }
    }
}

}  // namespace th
