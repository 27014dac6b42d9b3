// Kernels of the 8-bit products (i8gemm.hpp).
#pragma once

#include "i8gemm.hpp"
#include "ops.hpp"
#include "qlinear.hpp"

namespace th {

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x16_t __attribute__((ext_vector_type(16)));

__device__ __forceinline__ float i8_value(const I8Out& o, int sum, double s, double t, int n) {
    double v = (double)sum * s * t;
    if (o.bias) v += (double)o.bias[n];
    return (float)v;
}
__device__ __forceinline__ void i8_store(const I8Out& o, size_t m, int n, float v) {
    const size_t at = m * o.N + n;
    if (o.dt == TH_F32) ((float*)o.y)[at] = v;
    else if (o.dt == TH_F16) ((_Float16*)o.y)[at] = (_Float16)v;
    else ((__bf16*)o.y)[at] = (__bf16)v;
}

__device__ __forceinline__ void i8_store4(const I8Out& o, size_t m, int n, float a, float b, float c, float d) {
    const size_t at = m * o.N + n;
    typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
    typedef __bf16 b4_t __attribute__((ext_vector_type(4)));
    if (o.dt == TH_F32) *(float4*)((float*)o.y + at) = make_float4(a, b, c, d);
    else if (o.dt == TH_F16) *(h4_t*)((_Float16*)o.y + at) = (h4_t){(_Float16)a, (_Float16)b, (_Float16)c, (_Float16)d};
    else *(b4_t*)((__bf16*)o.y + at) = (b4_t){(__bf16)a, (__bf16)b, (__bf16)c, (__bf16)d};
}

// A few rows, bound by the stream of the weights: a workgroup has RT tiles of 16
// channels and CB of 16 rows, its NW waves take chunks of 64 k in turn (eight
// waves read 8 KiB of a tile row at a time), operands come from global memory
// straight into registers, and the waves' sums meet in LDS.  Integer sums: any split gives the same bits.
template <int RT, int CB, int U, int NW>
__global__ __launch_bounds__(64 * NW) void i8_rows_kernel(const uint4* __restrict__ wt, const int8_t* __restrict__ xq, I8Out out, int M, int Kp,
                                                          int nbx) {
    extern __shared__ i32x4_t red[];  // [NW][RT * CB][64]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q = lane >> 4, r = lane & 15;
    const int bx = blockIdx.x % nbx, by = blockIdx.x / nbx;
    const int NCH = Kp >> 6, NT = (out.N + 15) >> 4;
    const int m0 = by * CB * 16;
    const i32x4_t* w[RT];
    const i32x4_t* x[CB];
#pragma unroll
    for (int a = 0; a < RT; a++) w[a] = (const i32x4_t*)wt + (size_t)min(bx * RT + a, NT - 1) * NCH * 64 + lane;
#pragma unroll
    for (int b = 0; b < CB; b++) x[b] = (const i32x4_t*)(xq + (size_t)min(m0 + b * 16 + r, M - 1) * Kp) + q;
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
                for (int b = 0; b < CB; b++) xv[u][b] = x[b][(size_t)c * 4];
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
        const int n = (bx * RT + a) * 16 + (ln & 15), m = m0 + b * 16 + (ln >> 4) * 4;
        if (n >= out.N) continue;
        const double wsc = (double)out.ws[n];
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (m + e < M) i8_store(out, m + e, n, i8_value(out, s[e], (double)out.xs[m + e], wsc, n));
    }
}

// Many rows: 64 TM x 64 TN results a workgroup, 32 TM x 32 TN a wave (2 x 2
// waves) on the 32x32x32 MFMA, 64 k a step.  LDS holds three steps: one is read,
// the next is there (its first operands are read ahead), the one after is
// written, so one barrier a step orders all and no wave waits for LDS behind
// it.  Rows come through registers, two steps ahead of their place in LDS.  Both operands lie
// in LDS as they are read: 1 KiB blocks of 16 rows x 64 k, lane by lane.
// part: the sums of a K split instead of results, [split][M][N].
template <int TM, int TN, int WPE>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(WPE, WPE))) void i8_tile_kernel(
    const uint4* __restrict__ wt, const int8_t* __restrict__ xq, I8Out out, int M, int Kp, int chunks_per_split, int* __restrict__ part) {
    constexpr int NA = 4 * TM, NB = 4 * TN, SZ = (NA + NB) * 64;
    extern __shared__ i32x4_t tile[];  // [3][NA + NB][64], then the scales and the bias of the tile
    float* const scales = (float*)(tile + 3 * SZ);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int bx = blockIdx.x, by = blockIdx.y, split = blockIdx.z;
    gemm_xcd_tile(bx, by, split);
    const int NCH = Kp >> 6, NT = (out.N + 15) >> 4;
    const int c0 = split * chunks_per_split, steps = min(NCH - c0, chunks_per_split);
    const int m0 = by * 64 * TM, n0 = bx * 64 * TN;
    // this wave's blocks: rows past the end re-read the last one
    uint32_t xo[TM], wo[TN];
    const int mlast = M - 1 - m0, tlast = NT - 1 - n0 / 16;
#pragma unroll
    for (int i = 0; i < TM; i++) xo[i] = (uint32_t)min((wave * TM + i) * 16 + (lane & 15), mlast) * (uint32_t)Kp + (lane >> 4) * 16;
#pragma unroll
    for (int i = 0; i < TN; i++) wo[i] = (uint32_t)min(wave * TN + i, tlast) * (uint32_t)NCH * 1024u + lane * 16;
    const __amdgpu_buffer_rsrc_t xb = buffer_rsrc(xq + (size_t)m0 * Kp + (size_t)c0 * 64, (uint32_t)(min(M - m0, 64 * TM) * Kp - c0 * 64));
    const __amdgpu_buffer_rsrc_t wb =
        buffer_rsrc(wt + ((size_t)(n0 / 16) * NCH + c0) * 64, (uint32_t)((min(NT - n0 / 16, 4 * TN) * NCH - c0) * 1024));
    for (int i = tid; i < 64 * TM; i += 256) scales[i] = out.xs[min(m0 + i, M - 1)];
    for (int i = tid; i < 64 * TN; i += 256) {
        const int n = min(n0 + i, out.N - 1);
        scales[64 * TM + i] = out.ws[n];
        scales[64 * (TM + TN) + i] = out.bias ? out.bias[n] : 0.0f;
    }
    i32x4_t g[2][TM + TN];
    auto gload = [&](int set, int c, int i) {
        const auto v = i < TM ? __builtin_amdgcn_raw_buffer_load_b128(xb, (int)xo[i < TM ? i : 0], c * 64, 0)
                              : __builtin_amdgcn_raw_buffer_load_b128(wb, (int)wo[i < TM ? 0 : i - TM], c * 1024, 0);
        g[set][i] = __builtin_bit_cast(i32x4_t, v);
    };
    auto chunk = [&](int s) { return max(0, min(s, steps - 1)); };
    auto lwrite = [&](int set, i32x4_t* to, int i) { to[(i < TM ? wave * TM + i : NA + wave * TN + i - TM) * 64 + lane] = g[set][i]; };
    auto load_all = [&](int set, int s) {
#pragma unroll
        for (int i = 0; i < TM + TN; i++) gload(set, chunk(s), i);
    };
    auto write_all = [&](int set, i32x4_t* to) {
#pragma unroll
        for (int i = 0; i < TM + TN; i++) lwrite(set, to, i);
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
    // steps come in pairs: the first of an odd number of them has zeros before it
    const int first = -(steps & 1);
    load_all(0, first);
    load_all(1, first + 1);
    if (first < 0)
#pragma unroll
        for (int i = 0; i < TM; i++) g[0][i] = (i32x4_t){0, 0, 0, 0};
    write_all(0, tile);
    load_all(0, first + 2);
    write_all(1, tile + SZ);
    load_all(1, first + 3);
    lds_barrier();
#pragma unroll
    for (int i = 0; i < TM + TN; i++) lread(tile, 0, i);
    i32x4_t *now = tile, *next = tile + SZ, *after = tile + 2 * SZ;
    // The order is the source's: a step's LDS accesses lie evenly between its
    // matrix operations (four waves' reads or writes behind every one of them are
    // more than LDS takes: 2011 against N TOP/s at 8192 x 8192 x 8192), operands
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
                if (r * 2 * NM / NR + NM / NR / 2 == half * NM + q) lwrite(set, after, r);
                if (r * 2 * NM / NR + NM / NR + NM / NR / 2 == half * NM + q) gload(set, c, r);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto step = [&](int set, int s) {
        const int c = chunk(s + 4);
        half_step(0, set, c);
        half_step(1, set, c);
        lds_barrier();
        i32x4_t* t = now;
        now = next;
        next = after;
        after = t;
    };
    for (int s = first; s < steps; s += 2) {
        step(0, s);
        step(1, s + 1);
    }
    // Strips of 32 rows go through LDS (each wave's own part) and leave as whole
    // rows: four channels a lane, or one where rows do not start on four.
    asm volatile("s_nop 15\n\ts_nop 3");  // (the last MFMA's 16 passes, see mfma_settle)
    constexpr int W = 32 * TN, LW = W + 4;
    int* const strip = (int*)tile + wave * 32 * LW;
    const int nw = n0 + wn * W;
#pragma unroll
    for (int i = 0; i < TM; i++) {
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) strip[((e >> 2) * 8 + (lane >> 5) * 4 + (e & 3)) * LW + j * 32 + (lane & 31)] = acc[i][j][e];
        wave_lds_fence();
        const int ml = (wm * TM + i) * 32;
        if (part) {
            for (int x = lane; x < 32 * W; x += 64) {
                const int r = x / W, c = x % W, m = m0 + ml + r, n = nw + c;
                if (m < M && n < out.N) part[((size_t)split * M + m) * out.N + n] = strip[r * LW + c];
            }
        } else if ((out.N & 3) == 0) {
            constexpr int LPR = W / 4;  // lanes of a row
            const int c = lane % LPR * 4, n = nw + c;
            const float4 ws = *(const float4*)&scales[64 * TM + wn * W + c], bs = *(const float4*)&scales[64 * (TM + TN) + wn * W + c];
            if (n < out.N)
#pragma unroll 4
                for (int r = lane / LPR; r < 32; r += 64 / LPR) {
                    const int m = m0 + ml + r;
                    if (m >= M) break;
                    const i32x4_t v = *(const i32x4_t*)&strip[r * LW + c];
                    const double s = (double)scales[ml + r];
                    i8_store4(out, m, n, (float)((double)v[0] * s * (double)ws.x + (double)bs.x), (float)((double)v[1] * s * (double)ws.y + (double)bs.y),
                              (float)((double)v[2] * s * (double)ws.z + (double)bs.z), (float)((double)v[3] * s * (double)ws.w + (double)bs.w));
                }
        } else {
            for (int x = lane; x < 32 * W; x += 64) {
                const int r = x / W, c = x % W, m = m0 + ml + r, n = nw + c;
                if (m < M && n < out.N)
                    i8_store(out, m, n, (float)((double)strip[r * LW + c] * (double)scales[ml + r] * (double)scales[64 * TM + wn * W + c] +
                                                (double)scales[64 * (TM + TN) + wn * W + c]));
            }
        }
        wave_lds_fence();
    }
}

// The splits' sums, and what is done to them.
__global__ __launch_bounds__(256) void i8_join_kernel(const int* __restrict__ part, I8Out out, int M, int splits) {
    const size_t total = (size_t)M * out.N;
    for (size_t i = blockIdx.x * (size_t)256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
        int v = 0;
        for (int s = 0; s < splits; s++) v += part[(size_t)s * total + i];
        const size_t m = i / out.N;
        const int n = (int)(i - m * out.N);
        i8_store(out, m, n, i8_value(out, v, (double)out.xs[m], (double)out.ws[n], n));
    }
}

}  // namespace th
