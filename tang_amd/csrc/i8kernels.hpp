// Kernels of the 8-bit products (i8gemm.hpp).
#pragma once

#include "i8gemm.hpp"
#include "ops.hpp"
#include "qlinear.hpp"

namespace th {

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x16_t __attribute__((ext_vector_type(16)));

// (sum s) t + b.  For f32 results in f64, rounded once (no order of the scales leaves
// its range); for 16-bit ones in f32 from the scales' mantissas and the sum of their exponents: off
// by 3 2^-24 of the product, far below their own rounding, at a third of the time.  Both
// kernels do the same, so that a row has the same bits in any batch.
__device__ __forceinline__ float i8_wide(int sum, float s, float t, float b) { return (float)((double)sum * (double)s * (double)t + (double)b); }
__device__ __forceinline__ float i8_narrow(int sum, float s, float t, int exponent, float b) {
    return __builtin_amdgcn_ldexpf((float)sum * (s * t), exponent) + b;
}
__device__ __forceinline__ void i8_store(const I8Out& o, size_t m, int n, float v) {
    const size_t at = m * o.N + n;
    if (o.dt == TH_F32) ((float*)o.y)[at] = v;
    else if (o.dt == TH_F16) ((_Float16*)o.y)[at] = (_Float16)v;
    else ((__bf16*)o.y)[at] = (__bf16)v;
}

// Four channels from n on, those of them that there are (rows may start at any element).
template <typename Y>
__device__ __forceinline__ void i8_store4(Y* to, size_t m, int n, int N, const float (&y)[4]) {
    typedef Y y4_t __attribute__((ext_vector_type(4), aligned(sizeof(Y))));
    to += m * N + n;
    if (n + 4 <= N) {
        *(y4_t*)to = (y4_t){(Y)y[0], (Y)y[1], (Y)y[2], (Y)y[3]};
    } else {
#pragma unroll
        for (int i = 0; i < 3; i++)
            if (n + i < N) to[i] = (Y)y[i];
    }
}

// A few rows, bound by the stream of the weights: a workgroup has RT tiles of 16
// channels and all rows, CB tiles of 16, its NW waves take chunks of 64 k in turn (eight
// waves read 8 KiB of a tile row at a time), operands come from global memory
// straight into registers, and the waves' sums meet in LDS.  Integer sums: any split gives the same bits.
template <int RT, int CB, int U, int NW>
__global__ __launch_bounds__(64 * NW) void i8_rows_kernel(const uint4* __restrict__ wt, const int8_t* __restrict__ xq, I8Out out, int M, int Kp) {
    extern __shared__ i32x4_t red[];  // [NW][RT * CB][64]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q = lane >> 4, r = lane & 15;
    const int bx = blockIdx.x, NCH = Kp >> 6, NT = (out.N + 15) >> 4;
    const i32x4_t* w[RT];
    const i32x4_t* x[CB];
    int xstep[CB];
#pragma unroll
    for (int a = 0; a < RT; a++) w[a] = (const i32x4_t*)wt + (size_t)min(bx * RT + a, NT - 1) * NCH * 64 + lane;
#pragma unroll
    for (int b = 0; b < CB; b++) {  // rows past the end re-read the last one
        const int first = min(b, (M - 1) >> 4) * 16, h = min(16, M - first);
        x[b] = (const i32x4_t*)(xq + (size_t)first * Kp) + q * h + min(r, h - 1);
        xstep[b] = 4 * h;
    }
    i32x4_t acc[RT][CB];
#pragma unroll
    for (int a = 0; a < RT; a++)
#pragma unroll
        for (int b = 0; b < CB; b++) acc[a][b] = (i32x4_t){0, 0, 0, 0};
    for (int c0 = wave; c0 < NCH; c0 += NW * U) {
        i32x4_t wv[U][RT], xv[U][CB];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int c = c0 + u * NW;
            if (c < NCH) {  // (the same for the whole wave)
#pragma unroll
                for (int a = 0; a < RT; a++) wv[u][a] = __builtin_nontemporal_load(w[a] + (size_t)c * 64);
#pragma unroll
                for (int b = 0; b < CB; b++) xv[u][b] = x[b][(size_t)c * xstep[b]];
            } else {
#pragma unroll
                for (int a = 0; a < RT; a++) wv[u][a] = (i32x4_t){0, 0, 0, 0};
#pragma unroll
                for (int b = 0; b < CB; b++) xv[u][b] = (i32x4_t){0, 0, 0, 0};
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int a = 0; a < RT; a++)
#pragma unroll
                for (int b = 0; b < CB; b++) acc[a][b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xv[u][b], wv[u][a], acc[a][b], 0, 0, 0);
    }
    mfma_settle(acc);
#pragma unroll
    for (int a = 0; a < RT; a++)
#pragma unroll
        for (int b = 0; b < CB; b++) red[(wave * RT * CB + a * CB + b) * 64 + lane] = acc[a][b];
    __syncthreads();
    for (int i = threadIdx.x; i < RT * CB * 64; i += 64 * NW) {
        i32x4_t s = red[i];
#pragma unroll
        for (int v = 1; v < NW; v++) s += red[v * RT * CB * 64 + i];
        const int t = i >> 6, a = t / CB, b = t % CB, ln = i & 63;
        const int n = (bx * RT + a) * 16 + (ln & 15), m = b * 16 + (ln >> 4) * 4;
        if (n >= out.N) continue;
        const float wsc = out.ws[n], bias = out.bias ? out.bias[n] : 0.0f;
        int we = 0;
        const float wf = __builtin_frexpf(wsc, &we);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (m + e >= M) continue;
            const float xsc = out.xs[m + e];
            int xe = 0;
            const float xf = __builtin_frexpf(xsc, &xe);
            i8_store(out, m + e, n, out.dt == TH_F32 ? i8_wide(s[e], xsc, wsc, bias) : i8_narrow(s[e], xf, wf, xe + we, bias));
        }
    }
}

// Many rows: 64 TM x 64 TN results a workgroup, 32 TM x 32 TN a wave (2 x 2
// waves) on the 32x32x32 MFMA, 64 k a step.  LDS holds three steps: one is read,
// the next is there (its first operands are read ahead), the one after is
// written, so one barrier a step orders all and no wave waits for LDS behind
// it.  Rows come through registers, ST steps ahead of their place in LDS.  Both operands lie
// in LDS as they are read: 1 KiB blocks of 16 rows x 64 k, lane by lane.
// KW: groups of four waves, each with every KW-th step of k and LDS of its own, whose
// sums meet at the end, for tiles that are alone on their CU.
// Measured: 8192 x 8192 x 8192 2308 TOP/s (the library's product there: 2456), 8192 x 4096 x 11008 1914 (2186), where
// the matrix operations take half of the cycles at the 1.75 GHz that the chip then runs at (5.4 rounds of tiles take six, and no other
// tile of its CU works while one fills its pipe or leaves); 512 x 4096 x 4096 1000 (837), 128 x 4096 x 11008 648 (488).
// Tried: weights from memory straight into registers (each wave its own, 1846 and 1639:
// they are loaded twice), more steps ahead (the same).
// LDS in bytes: the stages, or the strips that results leave through; then the tile's scales and bias.
template <int TM, int TN, int KW>
struct I8TileLds {
    static constexpr int STAGES = 3 * KW * 4 * (TM + TN) * 1024, STRIPS = KW * 4 * 32 * (32 * TN + 4) * 4;
    static constexpr int SCALES = STAGES > STRIPS ? STAGES : STRIPS, BYTES = SCALES + 64 * (2 * TM + 3 * TN) * 4;
};
template <int TM, int TN, int KW, int ST, int WPE>
__global__ __launch_bounds__(256 * KW) __attribute__((amdgpu_waves_per_eu(WPE, WPE))) void i8_tile_kernel(
    const uint4* __restrict__ wt, const int8_t* __restrict__ xq, I8Out out, int M, int Kp) {
    constexpr int NA = 4 * TM, NB = 4 * TN, SZ = (NA + NB) * 64;
    extern __shared__ i32x4_t tile[];  // [3][KW][NA + NB][64], then the scales and the bias of the tile
    float* const scales = (float*)((char*)tile + I8TileLds<TM, TN, KW>::SCALES);
    const int tid = threadIdx.x, lane = tid & 63, wave8 = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wave = wave8 & 3, group = wave8 >> 2;
    int bx = blockIdx.x, by = blockIdx.y, bz = 0;
    gemm_xcd_tile(bx, by, bz);
    const int NCH = Kp >> 6, NT = (out.N + 15) >> 4;
    const int m0 = by * 64 * TM, n0 = bx * 64 * TN;
    // this wave's blocks: those past the end re-read the last one
    uint32_t xo[TM], wo[TN];
    int xstep[TM];
    const int mlast = (M - 1 - m0) >> 4, tlast = NT - 1 - n0 / 16;
#pragma unroll
    for (int i = 0; i < TM; i++) {
        const int blk = min(wave * TM + i, mlast), h = min(16, M - m0 - blk * 16);
        xo[i] = (uint32_t)blk * 16u * (uint32_t)Kp + ((lane >> 4) * h + min(lane & 15, h - 1)) * 16;
        xstep[i] = 64 * h;
    }
#pragma unroll
    for (int i = 0; i < TN; i++) wo[i] = (uint32_t)min(wave * TN + i, tlast) * (uint32_t)NCH * 1024u + lane * 16;
    const __amdgpu_buffer_rsrc_t xb = buffer_rsrc(xq + (size_t)m0 * Kp, (uint32_t)(min(M - m0, 64 * TM) * Kp));
    const __amdgpu_buffer_rsrc_t wb = buffer_rsrc(wt + (size_t)(n0 / 16) * NCH * 64, (uint32_t)(min(NT - n0 / 16, 4 * TN) * NCH * 1024));
    // Steps come in turns of ST by KW: chunks before the first of k fill them up, as zeros.
    const int steps = (NCH + KW * ST - 1) / (KW * ST) * ST, lead = steps * KW - NCH;
    i32x4_t g[ST][TM + TN];
    auto chunk = [&](int s) { return max(0, min(s * KW + group - lead, NCH - 1)); };
    auto gload = [&](int set, int c, int i) {
        const auto v = i < TM ? __builtin_amdgcn_raw_buffer_load_b128(xb, (int)xo[i < TM ? i : 0], c * xstep[i < TM ? i : 0], 0)
                              : __builtin_amdgcn_raw_buffer_load_b128(wb, (int)wo[i < TM ? 0 : i - TM], c * 1024, 0);
        g[set][i] = __builtin_bit_cast(i32x4_t, v);
    };
    auto lwrite = [&](int set, i32x4_t* to, int i) { to[(i < TM ? wave * TM + i : NA + wave * TN + i - TM) * 64 + lane] = g[set][i]; };
    auto load_all = [&](int set, int s) {
#pragma unroll
        for (int i = 0; i < TM + TN; i++) gload(set, chunk(s), i);
    };
    auto write_all = [&](int set, i32x4_t* to) {
#pragma unroll
        for (int i = 0; i < TM + TN; i++) lwrite(set, to, i);
    };
    auto zeros_before = [&](int set, int s) {
        if (s * KW + group < lead)
#pragma unroll
            for (int i = 0; i < TM; i++) g[set][i] = (i32x4_t){0, 0, 0, 0};
    };
    // operand of 32 rows and 32 k: lanes 0..31 have its first 16 k
    const int wm = wave >> 1, wn = wave & 1;
    const int at = ((lane >> 4) & 1) * 64 + (lane >> 5) * 16 + (lane & 15);
    i32x4_t op[2][TM + TN];
    auto lread = [&](const i32x4_t* from, int half, int i) {
        op[half][i] = from[(i < TM ? (wm * TM + i) * 128 : NA * 64 + (wn * TN + i - TM) * 128) + half * 32 + at];
    };
    i32x16_t acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = 0;
    i32x4_t *now = tile + group * SZ, *next = now + KW * SZ, *after = next + KW * SZ;
#pragma unroll
    for (int i = 0; i < ST; i++) load_all(i, i);
    float *const rs = scales, *const cs = rs + 64 * TM, *const cb = cs + 64 * TN;
    int *const re = (int*)(cb + 64 * TN), *const ce = re + 64 * TM;
    const bool wide = out.dt == TH_F32;
    for (int i = tid; i < 64 * (TM + TN); i += 256 * KW) {
        const int n = min(n0 + i - 64 * TM, out.N - 1);
        const float v = i < 64 * TM ? out.xs[min(m0 + i, M - 1)] : out.ws[n];
        int e = 0;
        const float f = __builtin_frexpf(v, &e);
        rs[i] = wide ? v : f;  // (rows, then columns)
        if (i >= 64 * TM) cb[i - 64 * TM] = out.bias ? out.bias[n] : 0.0f;
        re[i] = e;
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        zeros_before(i, i);
        write_all(i, i ? next : now);
        load_all(i, ST + i);
    }
    lds_barrier();
#pragma unroll
    for (int i = 0; i < TM + TN; i++) lread(now, 0, i);
    // The order is the source's: a step's LDS accesses lie evenly between its
    // matrix operations (four waves' reads or writes behind every one of them are
    // more than LDS takes: 2011 against 2167 TOP/s at 8192 x 8192 x 8192), operands
    // are read in the order of their use, half a step ahead.
    constexpr int NM = TM * TN, NR = TM + TN;
    auto operand = [&](int r) { return r == 0 ? 0 : r <= TN ? TM + r - 1 : r - TN; };
    auto half_step = [&](int half, int set, int c) {
#pragma unroll
        for (int q = 0; q < NM; q++) {
            acc[q / TN][q % TN] =
                __builtin_amdgcn_mfma_i32_32x32x32_i8(op[half][q / TN], op[half][TM + q % TN], acc[q / TN][q % TN], 0, 0, 0);
#pragma unroll
            for (int r = 0; r < NR; r++) {
                if (r * NM / NR == q) lread(half ? next : now, 1 - half, operand(r));
                const int write = (4 * r + 1) * NM / (2 * NR), load = (4 * r + 3) * NM / (2 * NR);  // of the step's 2 NM places
                if (write == half * NM + q) lwrite(set, after, r);
                if (load == half * NM + q) gload(set, c, r);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto step = [&](int set, int s) {  // writes step s + 2, which `set` holds, and loads step s + 2 + ST into it
        const int c = chunk(s + 2 + ST);
        if (ST * KW > 2) zeros_before(set, s + 2);
        half_step(0, set, c);
        half_step(1, set, c);
        lds_barrier();
        i32x4_t* t = now;
        now = next;
        next = after;
        after = t;
    };
    for (int s = 0; s < steps; s += ST) {
#pragma unroll
        for (int i = 0; i < ST; i++) step((2 + i) % ST, s + i);
    }
    // Strips of 32 rows go through LDS (each wave's own part), where the groups'
    // sums meet, and leave as whole rows, four channels a lane and four rows at a
    // time, in code of their type's own (K = 64, 256 x 256 tiles: with a branch
    // for each value 25.9 us a launch).
    asm volatile("s_nop 15\n\ts_nop 3");  // (the last MFMA's passes, see mfma_settle)
    constexpr int W = 32 * TN, LW = W + 4, LPR = W / 4, RPI = 64 / LPR;  // lanes of a row, rows a wave reads at once
    constexpr int ITS = 32 / RPI / KW, AT_ONCE = ITS < 4 ? ITS : 4;
    int* const strip = (int*)tile + wave * 32 * LW;
    const int c = lane % LPR * 4, n = n0 + wn * W + c;
    const float4 ws = *(const float4*)&cs[wn * W + c], bs = *(const float4*)&cb[wn * W + c];
    const int4 we = *(const int4*)&ce[wn * W + c];
    const float t[4] = {ws.x, ws.y, ws.z, ws.w}, b[4] = {bs.x, bs.y, bs.z, bs.w};
    const int te[4] = {we.x, we.y, we.z, we.w};
    auto leave = [&](auto as) {
        using Y = decltype(as);
#pragma unroll
        for (int i = 0; i < TM; i++) {
            int* const to = strip + group * 4 * 32 * LW + (lane >> 5) * 4 * LW + (lane & 31);
#pragma unroll
            for (int j = 0; j < TN; j++)
#pragma unroll
                for (int e = 0; e < 16; e++) to[((e >> 2) * 8 + (e & 3)) * LW + j * 32] = acc[i][j][e];
            if constexpr (KW > 1) __syncthreads();
            else wave_lds_fence();
            const int ml = (wm * TM + i) * 32;
#pragma unroll 1
            for (int it = 0; it < ITS; it += AT_ONCE) {
                i32x4_t v[AT_ONCE];
                float s[AT_ONCE];
                int se[AT_ONCE];
#pragma unroll
                for (int x = 0; x < AT_ONCE; x++) {
                    const int r = ((it + x) * KW + group) * RPI + lane / LPR;
                    v[x] = *(const i32x4_t*)&strip[r * LW + c];
#pragma unroll
                    for (int k = 1; k < KW; k++) v[x] += *(const i32x4_t*)&strip[k * 4 * 32 * LW + r * LW + c];
                    s[x] = rs[ml + r];
                    se[x] = re[ml + r];
                }
#pragma unroll
                for (int x = 0; x < AT_ONCE; x++) {
                    float y[4];
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        y[e] = sizeof(Y) == 4 ? i8_wide(v[x][e], s[x], t[e], b[e]) : i8_narrow(v[x][e], s[x], t[e], se[x] + te[e], b[e]);
                    const int m = m0 + ml + ((it + x) * KW + group) * RPI + lane / LPR;
                    if (m < M && n < out.N) i8_store4((Y*)out.y, m, n, out.N, y);
                }
            }
            if constexpr (KW > 1) __syncthreads();
            else wave_lds_fence();
        }
    };
    if (out.dt == TH_F32) leave(float{});
    else if (out.dt == TH_F16) leave((_Float16)0);
    else leave((__bf16)0.0f);
}

}  // namespace th
