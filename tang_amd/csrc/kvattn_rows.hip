// The launch of rows items (kvattn_rows.hpp), and the join of split work.
#include <algorithm>
#include <type_traits>

#include "kvattn_rows.hpp"

namespace th {

template <int D, typename E, int NP, bool PAD>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void kv_attn_rows_kernel(KvAttnArgs a) {
    __shared__ __align__(16) char lds[KvRows<D>::LDS];
    const int kvh = a.pages.n_kv_heads, h = blockIdx.x % kvh, count = a.head->n_rows_items;
    int n = blockIdx.x / kvh;
    // the first item is read before it is known to be there (the list has room for the grid)
    KvItem it = kv_item(a.rows_items, n);
    for (; n < count; it = kv_item(a.rows_items, n)) {
        kv_rows_item<D, E, NP, PAD>(a, it, h, lds);
        n += gridDim.x / kvh;
        if (n >= count) break;
        __syncthreads();  // the next item writes these rows
    }
}

// Records joined, few rows (a row: token and query head): four waves for each, wave w the
// records w, w + 4, ... with lane l on dims DE l ..; the waves meet in LDS.  One round of loads covers
// 64 records: latency is what it costs.
template <int DE>
__device__ __forceinline__ void kv_join_few(const KvAttnArgs& a, const KvTok* __restrict__ list, int room) {
    constexpr int U = DE == 4 ? 8 : 16;
    typedef float vec __attribute__((ext_vector_type(DE == 1 ? 2 : DE)));
    __shared__ float sA[4][64 * DE], sM[4], sL[4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hd = a.pages.hd, d0 = lane * DE;
    const int total = a.head->n_joins * a.n_heads;
    const size_t step = (size_t)a.n_heads * hd;
    int x = blockIdx.x;
    KvTok t = list[min(x / a.n_heads, room - 1)];  // (read with the count, before it is known to be there)
    for (; x < total; x += gridDim.x, t = list[min(x, total - 1) / a.n_heads]) {
        const int hq = x % a.n_heads;
        const int n = t.own_n >> 16, mine = (n - wave + 3) / 4;  // this wave's records
        const float2* ml = a.rec_ml + (size_t)t.rec * a.n_heads + hq;
        const float* po = a.rec_o + ((size_t)t.rec * a.n_heads + hq) * hd + (d0 < hd ? d0 : 0);
        float M = -INFINITY, L = 0.0f, A[DE];
#pragma unroll
        for (int e = 0; e < DE; e++) A[e] = 0.0f;
        for (int s0 = 0; s0 < mine; s0 += U) {
            float v[U][DE];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const float* p = po + (size_t)(min(s0 + u, mine - 1) * 4 + wave) * step;
                if constexpr (DE == 1) v[u][0] = *p;
                else {
                    const vec w = *(const vec*)p;
#pragma unroll
                    for (int e = 0; e < DE; e++) v[u][e] = w[e];
                }
            }
            const int sl = s0 + (lane & (U - 1));
            const float2 w = ml[(size_t)(min(sl, mine - 1) * 4 + wave) * a.n_heads];
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
        for (int w = 0; w < 4; w++) {
            const bool none = sM[w] == -INFINITY && sL[w] == 0.0f;
            const float f = none ? 0.0f : kv_exp2(sM[w] - M);
            L = __builtin_fmaf(f, sL[w], L);
#pragma unroll
            for (int e = 0; e < DE; e++) A[e] = none ? A[e] : __builtin_fmaf(f, sA[w][d0 + e], A[e]);
        }
        if (d0 < hd) {
#pragma unroll
            for (int e = 0; e < DE; e++) kv_store_out(a.out, a.odt, ((size_t)t.row * a.n_heads + hq) * hd + d0 + e, A[e] / L);
        }
    }
}

// Many rows of few records: LPR lanes for each, eight dims a lane, two records in flight.
template <int LPR>
__device__ __forceinline__ void kv_join_many(const KvAttnArgs& a, const KvTok* __restrict__ list, int room) {
    const int hd = a.pages.hd, part = threadIdx.x % LPR, d0 = part * 8;
    const int total = a.head->n_joins * a.n_heads;
    const size_t step = (size_t)a.n_heads * hd;
    int x = blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
    KvTok t = list[min(x / a.n_heads, room - 1)];
    for (; x < total; x += gridDim.x * (256 / LPR), t = list[min(x, total - 1) / a.n_heads]) {
        const int hq = x % a.n_heads;
        const int n = t.own_n >> 16;
        const float2* ml = a.rec_ml + (size_t)t.rec * a.n_heads + hq;
        const float* po = a.rec_o + ((size_t)t.rec * a.n_heads + hq) * hd + (d0 < hd ? d0 : 0);
        float M = -INFINITY, L = 0.0f, A[8];
#pragma unroll
        for (int e = 0; e < 8; e++) A[e] = 0.0f;
        for (int s0 = 0; s0 < n; s0 += 2) {
            kv_f32x4_t v[2][2];
            float2 w[2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int s = min(s0 + u, n - 1);
                w[u] = ml[(size_t)s * a.n_heads];
#pragma unroll
                for (int y = 0; y < 2; y++) v[u][y] = *(const kv_f32x4_t*)(po + (size_t)s * step + 4 * y);
            }
            const bool none0 = w[0].x == -INFINITY && w[0].y == 0.0f, none1 = s0 + 1 >= n || (w[1].x == -INFINITY && w[1].y == 0.0f);
            const float mn = fmaxf(M, fmaxf(none0 ? -INFINITY : w[0].x, none1 ? -INFINITY : w[1].x)), ref = mn == -INFINITY ? 0.0f : mn;
            const float f0 = none0 ? 0.0f : kv_exp2(w[0].x - ref), f1 = none1 ? 0.0f : kv_exp2(w[1].x - ref), back = kv_exp2(M - ref);
            L = L * back + f0 * (none0 ? 0.0f : w[0].y) + f1 * (none1 ? 0.0f : w[1].y);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                A[e] *= back;
                A[e] = none0 ? A[e] : __builtin_fmaf(f0, v[0][e >> 2][e & 3], A[e]);
                A[e] = none1 ? A[e] : __builtin_fmaf(f1, v[1][e >> 2][e & 3], A[e]);
            }
            M = mn;
        }
        if (d0 < hd) {
            const size_t at = ((size_t)t.row * a.n_heads + hq) * hd + d0;
            kv_store_out4(a.out, a.odt, at, kv_f32x4_t{A[0] / L, A[1] / L, A[2] / L, A[3] / L});
            kv_store_out4(a.out, a.odt, at + 4, kv_f32x4_t{A[4] / L, A[5] / L, A[6] / L, A[7] / L});
        }
    }
}

template <int DE>
__global__ __launch_bounds__(256) void kv_attn_join_few_kernel(KvAttnArgs a, const KvTok* __restrict__ list, int room) {
    kv_join_few<DE>(a, list, room);
}
template <int DE>
__global__ __launch_bounds__(256) void kv_attn_join_many_kernel(KvAttnArgs a, const KvTok* __restrict__ list, int room) {
    kv_join_many<8 * DE>(a, list, room);
}
// As the plan says (captured calls).
template <int DE>
__global__ __launch_bounds__(256) void kv_attn_join_kernel(KvAttnArgs a, const KvTok* __restrict__ list, int room) {
    if (a.head->flags & KV_PLAN_MANY) kv_join_many<8 * DE>(a, list, room);
    else kv_join_few<DE>(a, list, room);
}

// 33 records a row: few 9.4 us, many 12.1; about 3 records for each of 3000 rows: many 11, one wave a row 19
bool kv_join_many(size_t n, size_t n_recs, size_t n_heads) { return n * n_heads > 1024 && n_recs < 8 * n; }

void launch_kv_attn_join(const KvAttnArgs& a, const KvTok* list, size_t n, size_t room, int flags, hipStream_t s) {
    if (n == 0) return;
    const size_t rows = n * a.n_heads;
    auto with = [&](auto de) {
        constexpr int DE = decltype(de)::value, LPR = 8 * DE;
        const dim3 few((unsigned)std::min(rows, KV_MAX_BLOCKS)), many((unsigned)std::min(ceil_div(rows, (size_t)(256 / LPR)), KV_MAX_BLOCKS));
        if (flags == KV_BY_PLAN) TH_LAUNCH((kv_attn_join_kernel<DE>), few, dim3(256), 0, s, a, list, (int)room);
        else if (flags & KV_PLAN_MANY) TH_LAUNCH((kv_attn_join_many_kernel<DE>), many, dim3(256), 0, s, a, list, (int)room);
        else TH_LAUNCH((kv_attn_join_few_kernel<DE>), few, dim3(256), 0, s, a, list, (int)room);
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
    const unsigned g = (unsigned)(std::min(grid, KV_MAX_BLOCKS / a.pages.n_kv_heads) * a.pages.n_kv_heads);
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
