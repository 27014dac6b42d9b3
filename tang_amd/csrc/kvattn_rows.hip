// Attention over a paged cache for at most 16 rows (new tokens x query heads of
// one kv head): decode steps, and the merge of split work.
//
//   o = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m),  s_j = q.k_j * scale * log2(e)
//
// over the keys that the row sees, in one pass with the running maximum m.
// Workgroup = (item, kv head); its four waves take 32-key blocks in turn, each
// with a softmax state of its own.  Both products are transposed: S^T = K.Q^T
// takes K as it lies in memory as the first operand and leaves lane (g, r) the
// scores of row r for keys 4g..4g+3 of each 16, which is the operand that
// O^T += V^T.P^T wants; V^T comes out of row-major LDS by transposing reads.
#include <algorithm>
#include <type_traits>

#include "kvattn.hpp"

namespace th {

template <int D, typename E, int NP, bool PAD>
struct KvRowsWave {
    typedef typename KvVec<E>::x8 x8;
    static constexpr int NK = D / 32, NDT = D / 16, LD = D + 8, KB = 32, CPR = D / 8, VL = KB * CPR / 64;
};

template <int D, typename E, int NP, bool PAD>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void kv_attn_rows_kernel(KvAttnArgs a) {
    typedef KvRowsWave<D, E, NP, PAD> W;
    typedef typename W::x8 x8;
    constexpr int NK = W::NK, NDT = W::NDT, LD = W::LD, KB = W::KB, CPR = W::CPR, VL = W::VL, DE = D / 64;
    constexpr size_t REGION = std::max((size_t)KB * LD * 2, (size_t)16 * D * 4);
    __shared__ __align__(16) char lds[4 * REGION];
    __shared__ float sm[4][16], sl[4][16], sM[16];
    const KvPlanHead& head = *(const KvPlanHead*)a.plan;
    const KvTok* toks = (const KvTok*)(a.plan + KV_HEAD_WORDS);
    const KvItem* items = (const KvItem*)(a.plan + head.rows_items);
    const int kvh = a.pages.n_kv_heads, h = blockIdx.x % kvh, G = a.n_heads / kvh, hd = PAD ? a.pages.hd : D, nch = hd / 8;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, r = lane & 15;
    E* vs = (E*)(lds + wave * REGION);
    for (int n = blockIdx.x / kvh; n < head.n_rows_items; n += gridDim.x / kvh) {
        const KvItem it = items[n];
        const int R = it.ntok * G, row = min(r, R - 1);
        const KvTok tok = toks[it.tok0 + row / G];
        const int* table = a.pages.table + (size_t)it.seq * a.pages.pages_per_seq;
        auto q_at = [&](const KvTok& t, int rw) { return ((size_t)t.row * a.n_heads + h * G + rw % G) * hd; };

        // this block's K and V rows: lane (g, r) finds keys r and 16 + r
        uint32_t rn[2];
        auto find = [&](int j0) {
#pragma unroll
            for (int t = 0; t < 2; t++) rn[t] = kv_row(a.pages, table, h, kv_key(it, min(j0 + 16 * t + r, it.j1 - 1)));
        };
        kv_u4_t k[2][NK], v[VL];
        auto load_k = [&]() {
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const E* p = (const E*)a.pages.k + (size_t)rn[t] * hd;
#pragma unroll
                for (int c = 0; c < NK; c++) k[t][c] = *(const kv_u4_t*)(p + (PAD ? min(4 * c + g, nch - 1) : 4 * c + g) * 8);
            }
        };
        auto load_v = [&]() {
#pragma unroll
            for (int i = 0; i < VL; i++) {  // 16-byte piece lane + 64 i of the block
                const int key = (lane + 64 * i) / CPR, c = lane % CPR;
                const uint32_t rw = __shfl(rn[(64 * i / CPR) >> 4], key & 15, 64);
                v[i] = *(const kv_u4_t*)((const E*)a.pages.v + (size_t)rw * hd + (PAD ? min(c, nch - 1) : c) * 8);
            }
        };
        int j = it.j0 + wave * KB;
        find(j);
        load_k();
        load_v();
        find(j + 4 * KB);

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
#pragma unroll
            for (int c = 0; c < NK; c++) {
                kv_load_q8(a.q, a.qdt, q_at(tok, row) + (PAD ? min(4 * c + g, nch - 1) : 4 * c + g) * 8, x[c]);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (PAD && 4 * c + g >= nch) x[c][i] = 0.0f;
                    mx = fmaxf(mx, fabsf(x[c][i]));
                }
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
            load_k();  // of the next block (past the last: its last row again)
            float bm = -INFINITY;
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int jj = j + 16 * t + 4 * g + i;
                    const bool seen = jj < it.j1 && kv_sees(kv_key(it, jj), tok.pos, a.window, a.sinks);
                    s[t][i] = seen ? s[t][i] * scale : -INFINITY;
                    bm = fmaxf(bm, s[t][i]);
                }
            bm = fmaxf(bm, __shfl_xor(bm, 16, 64));
            bm = fmaxf(bm, __shfl_xor(bm, 32, 64));
            const float mn = fmaxf(m, bm), ref = mn == -INFINITY ? 0.0f : mn, f = kv_exp2(m - ref);
            float ps = 0.0f;
            x8 p[NP];
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float e = kv_exp2(s[t][i] - ref);
                    ps += e;
                    E part[NP];
                    kv_split<E, NP>(NP == 1 ? e : e * KV_P_UP, part);
#pragma unroll
                    for (int u = 0; u < NP; u++) p[u][4 * t + i] = part[u];
                }
            l = l * f + ps;  // this lane's keys; the row's lanes meet at the end
            m = mn;
#pragma unroll
            for (int i = 0; i < VL; i++)
                *(kv_u4_t*)(vs + (lane + 64 * i) / CPR * LD + lane % CPR * 8) = v[i];
            wave_lds_fence();
            load_v();
            find(j + 8 * KB);
#pragma unroll
            for (int dt = 0; dt < NDT; dt++) {
                // lane r addresses four dims of key r >> 2 of its group's four, and gets its dim of all four
                kv_s4_t w[2];
#pragma unroll
                for (int t = 0; t < 2; t++)
                    w[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (kv_lds_s4_t*)(vs + (16 * t + 4 * g + (r >> 2)) * LD + dt * 16 + 4 * (r & 3)));
                typedef short s8 __attribute__((ext_vector_type(8)));
                const x8 va = __builtin_bit_cast(x8, (s8){w[0][0], w[0][1], w[0][2], w[0][3], w[1][0], w[1][1], w[1][2], w[1][3]});
                kv_f32x4_t d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int u = NP - 1; u >= 0; u--) d = kv_mfma16(va, p[u], d);
#pragma unroll
                for (int i = 0; i < 4; i++) o[dt][i] = __builtin_fmaf(o[dt][i], f, d[i]);
            }
            wave_lds_fence();  // the rows are rewritten by the next block
        }
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        bool fine = l == l;
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
                kv_row_plain<E, DE>(a, it, table, h, q_at(t, rw), t.pos, it.j0 + wave * KB, KB, 4 * KB, pm, pl, acc);
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
        __syncthreads();  // the next item writes these rows
    }
}

// One wave per (token, query head): the records of its pieces joined in order.
template <int DE>
__global__ __launch_bounds__(256) void kv_attn_merge_kernel(KvAttnArgs a) {
    const KvPlanHead& head = *(const KvPlanHead*)a.plan;
    const KvTok* toks = (const KvTok*)(a.plan + KV_HEAD_WORDS);
    const int* list = a.plan + head.merge;
    const int lane = threadIdx.x & 63, hd = a.pages.hd;
    const int total = head.n_merge * a.n_heads;
    for (int x = blockIdx.x * 4 + (threadIdx.x >> 6); x < total; x += gridDim.x * 4) {
        const KvTok t = toks[list[x / a.n_heads]];
        const int hq = x % a.n_heads, n = t.own_n >> 16;
        const float2* ml = a.rec_ml + (size_t)t.rec * a.n_heads + hq;
        const float* po = a.rec_o + ((size_t)t.rec * a.n_heads + hq) * hd;
        const size_t step = (size_t)a.n_heads * hd;
        // lane s looks at records s, s + 64, ...
        float M = -INFINITY, L = 0.0f, A[DE];
        for (int s = lane; s < n; s += 64) M = fmaxf(M, ml[(size_t)s * a.n_heads].x);
        M = wave_max(M);
#pragma unroll
        for (int e = 0; e < DE; e++) A[e] = 0.0f;
        for (int s0 = 0; s0 < n; s0 += 64) {
            float2 w = make_float2(0.0f, 0.0f);
            if (s0 + lane < n) w = ml[(size_t)(s0 + lane) * a.n_heads];
            const float f = w.x == -INFINITY && w.y == 0.0f ? 0.0f : kv_exp2(w.x - M);
            L += f * w.y;
            const int here = min(64, n - s0);
            for (int u0 = 0; u0 < here; u0 += 8) {
                float v[8][DE];
#pragma unroll
                for (int u = 0; u < 8; u++)
#pragma unroll
                    for (int e = 0; e < DE; e++)
                        v[u][e] = lane + 64 * e < hd ? po[(size_t)(s0 + min(u0 + u, here - 1)) * step + lane + 64 * e] : 0.0f;
#pragma unroll
                for (int u = 0; u < 8; u++) {
                    const float fu = __shfl(f, u0 + u < here ? u0 + u : 0, 64);
                    if (u0 + u < here) {
#pragma unroll
                        for (int e = 0; e < DE; e++) A[e] = __builtin_fmaf(fu, v[u][e], A[e]);
                    }
                }
            }
        }
        L = wave_sum(L);
#pragma unroll
        for (int e = 0; e < DE; e++)
            if (lane + 64 * e < hd) kv_store_out(a.out, a.odt, ((size_t)t.row * a.n_heads + hq) * hd + lane + 64 * e, A[e] / L);
    }
}

template <int D, typename E>
static void rows_launch(const KvAttnArgs& a, unsigned grid, hipStream_t s) {
    constexpr int WIDE = kv_wide_parts<E>();
    const th_dtype own = std::is_same<E, __bf16>::value ? TH_BF16 : TH_F16;
    const bool one = a.qdt == own && a.odt == own, pad = a.pages.hd != D;
    if (one && pad) TH_LAUNCH((kv_attn_rows_kernel<D, E, 1, true>), dim3(grid), dim3(256), 0, s, a);
    else if (one) TH_LAUNCH((kv_attn_rows_kernel<D, E, 1, false>), dim3(grid), dim3(256), 0, s, a);
    else if (pad) TH_LAUNCH((kv_attn_rows_kernel<D, E, WIDE, true>), dim3(grid), dim3(256), 0, s, a);
    else TH_LAUNCH((kv_attn_rows_kernel<D, E, WIDE, false>), dim3(grid), dim3(256), 0, s, a);
    TH_LAUNCH_CHECK();
}

void launch_kv_attn_rows(const KvAttnArgs& a, th_dtype cache, size_t grid, hipStream_t s) {
    if (grid == 0) return;
    const unsigned g = (unsigned)(grid * a.pages.n_kv_heads);
    auto with = [&](auto e) {
        typedef decltype(e) E;
        if (a.pages.hd <= 64) rows_launch<64, E>(a, g, s);
        else if (a.pages.hd <= 128) rows_launch<128, E>(a, g, s);
        else rows_launch<256, E>(a, g, s);
    };
    if (cache == TH_F16) with((_Float16)0);
    else with((__bf16)0.0f);
}

void launch_kv_attn_merge(const KvAttnArgs& a, size_t grid, hipStream_t s) {
    if (grid == 0) return;
    const unsigned g = (unsigned)ceil_div(grid * a.n_heads, (size_t)4);
    if (a.pages.hd <= 64) TH_LAUNCH(kv_attn_merge_kernel<1>, dim3(g), dim3(256), 0, s, a);
    else if (a.pages.hd <= 128) TH_LAUNCH(kv_attn_merge_kernel<2>, dim3(g), dim3(256), 0, s, a);
    else TH_LAUNCH(kv_attn_merge_kernel<4>, dim3(g), dim3(256), 0, s, a);
    TH_LAUNCH_CHECK();
}

}  // namespace th
