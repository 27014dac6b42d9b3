// Kernels of the 8-bit products (i8gemm.hpp).
#pragma once

#include "i8gemm.hpp"
#include "ops.hpp"

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

}  // namespace th
