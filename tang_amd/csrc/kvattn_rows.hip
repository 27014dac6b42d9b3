// Attention over a paged cache for at most 16 rows (new tokens x query heads of
// one kv head): decode steps; and the join of split work.
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
    const KvTok* toks = a.toks;
    const int kvh = a.pages.n_kv_heads, h = blockIdx.x % kvh, G = a.n_heads / kvh, hd = PAD ? a.pages.hd : D, nch = hd / 8;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, r = lane & 15;
    E* vs = (E*)(lds + wave * REGION);
    // the first item is read before it is known to be there (the list has room for the grid)
    const int count = __builtin_amdgcn_readfirstlane(*a.n_items);
    int n = blockIdx.x / kvh;
    KvItem it = kv_item(a.items, n);
    for (; n < count; it = kv_item(a.items, n)) {
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
            const float mn = fmaxf(m, bm), ref = mn == -INFINITY ? 0.0f : mn, f = kv_exp2(m - ref);
            float ps = 0.0f;
            x8 p[NP];
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float e = kv_exp2(__builtin_fmaf(s[t][i], scale, -ref));
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
        n += gridDim.x / kvh;
        if (n >= count) break;
        __syncthreads();  // the next item writes these rows
    }
}

// Records joined: WR waves for each (token, query head), wave w the records w, w + WR, ...
// with lane l on dims DE l .. ; the waves meet in LDS.  Few rows take all four waves of a
// workgroup (latency: one round of loads for 64 records), many one wave each.
template <int DE, int WR>
__global__ __launch_bounds__(256) void kv_attn_join_kernel(KvAttnArgs a, const int* __restrict__ list) {
    constexpr int U = DE == 4 ? 8 : 16, RPB = 4 / WR;
    __shared__ float sA[WR > 1 ? 4 : 1][64 * DE], sM[4], sL[4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hd = a.pages.hd, d0 = lane * DE;
    const int total = *a.n_items * a.n_heads, part = wave % WR;
    const size_t step = (size_t)a.n_heads * hd;
    for (int x0 = blockIdx.x * RPB; x0 < total; x0 += gridDim.x * RPB) {
        const int x = min(x0 + wave / WR, total - 1), hq = x % a.n_heads;
        const KvTok t = a.toks[list[x / a.n_heads]];
        const int n = t.own_n >> 16, mine = (n - part + WR - 1) / WR;  // this wave's records
        const float2* ml = a.rec_ml + (size_t)t.rec * a.n_heads + hq;
        const float* po = a.rec_o + ((size_t)t.rec * a.n_heads + hq) * hd + (d0 < hd ? d0 : 0);
        float M = -INFINITY, L = 0.0f, A[DE];
#pragma unroll
        for (int e = 0; e < DE; e++) A[e] = 0.0f;
        for (int s0 = 0; s0 < mine; s0 += U) {
            typedef float vec __attribute__((ext_vector_type(DE == 1 ? 2 : DE)));
            float v[U][DE];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const float* p = po + (size_t)(min(s0 + u, mine - 1) * WR + part) * step;
                if constexpr (DE == 1) v[u][0] = *p;
                else {
                    const vec w = *(const vec*)p;
#pragma unroll
                    for (int e = 0; e < DE; e++) v[u][e] = w[e];
                }
            }
            const int sl = s0 + (lane & (U - 1));
            const float2 w = ml[(size_t)(min(sl, mine - 1) * WR + part) * a.n_heads];
            const bool none = sl >= mine || (w.x == -INFINITY && w.y == 0.0f);  // no record, or one without a key that the row sees
            const float mn = fmaxf(M, group_max<16>(none ? -INFINITY : w.x)), ref = mn == -INFINITY ? 0.0f : mn;
            const float f = none ? 0.0f : kv_exp2(w.x - ref), back = kv_exp2(M - ref);
            L = L * back + (lane < U ? f * w.y : 0.0f);
#pragma unroll
            for (int e = 0; e < DE; e++) A[e] *= back;
            M = mn;
#pragma unroll
            for (int u = 0; u < U; u++) {
                const float fu = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), u));
                if (s0 + u < mine) {
#pragma unroll
                    for (int e = 0; e < DE; e++) A[e] = __builtin_fmaf(fu, v[u][e], A[e]);
                }
            }
        }
        L = wave_sum(L);
        if constexpr (WR > 1) {
            __syncthreads();  // the last row's sums have been read
#pragma unroll
            for (int e = 0; e < DE; e++) sA[wave][d0 + e] = A[e];
            if (lane == 0) { sM[wave] = M; sL[wave] = L; }
            __syncthreads();
            if (wave > 0) continue;
            M = fmaxf(fmaxf(sM[0], sM[1]), fmaxf(sM[2], sM[3]));
            L = 0.0f;
#pragma unroll
            for (int e = 0; e < DE; e++) A[e] = 0.0f;
#pragma unroll
            for (int w = 0; w < WR; w++) {
                const float f = sM[w] == -INFINITY && sL[w] == 0.0f ? 0.0f : kv_exp2(sM[w] - M);
                L = __builtin_fmaf(f, sL[w], L);
#pragma unroll
                for (int e = 0; e < DE; e++) A[e] = f == 0.0f ? A[e] : __builtin_fmaf(f, sA[w][d0 + e], A[e]);
            }
        }
        if (d0 < hd && x == x0 + wave / WR) {
#pragma unroll
            for (int e = 0; e < DE; e++) kv_store_out(a.out, a.odt, ((size_t)t.row * a.n_heads + hq) * hd + d0 + e, A[e] / L);
        }
    }
}

void launch_kv_attn_join(const KvAttnArgs& a, const int* list, size_t grid, hipStream_t s) {
    if (grid == 0) return;
    const size_t rows = grid * a.n_heads;
    auto with = [&](auto de) {
        constexpr int DE = decltype(de)::value;
        if (rows <= 1024) TH_LAUNCH((kv_attn_join_kernel<DE, 4>), dim3((unsigned)rows), dim3(256), 0, s, a, list);
        else TH_LAUNCH((kv_attn_join_kernel<DE, 1>), dim3((unsigned)ceil_div(rows, (size_t)4)), dim3(256), 0, s, a, list);
    };
    if (a.pages.hd <= 64) with(std::integral_constant<int, 1>{});
    else if (a.pages.hd <= 128) with(std::integral_constant<int, 2>{});
    else with(std::integral_constant<int, 4>{});
    TH_LAUNCH_CHECK();
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

}  // namespace th
