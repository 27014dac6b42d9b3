// Rows to 8-bit integers, and their product with 8-bit weights (i8gemm.hpp).
#include <algorithm>

#include "capi_util.hpp"
#include "i8kernels.hpp"

namespace th {

// ---------------------------------------------------------------------------
// Rows to integers
// ---------------------------------------------------------------------------

// Eight consecutive elements at any element's alignment, as f32.
template <typename X>
__device__ __forceinline__ void load8_any(const X* p, float (&v)[8]) {
    typedef X x8 __attribute__((ext_vector_type(8), aligned(sizeof(X))));
    const x8 t = *(const x8*)p;
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = (float)t[i];
}

// x / s to the nearest integer, ties to even, exactly: the rounded product with
// the reciprocal is off by one at most, and the rest x - q s has no rounding
// (it is a multiple of the smaller operand's last bit and not above s).
__device__ __forceinline__ int quantized(float x, float s, float rs) {
    float q = rintf(x * rs);
    const float rest2 = 2.0f * __builtin_fmaf(-q, s, x);
    const bool odd = ((int)q & 1) != 0;
    if (rest2 > s || (rest2 == s && odd)) q += 1.0f;
    else if (rest2 < -s || (rest2 == -s && odd)) q -= 1.0f;
    return (int)fminf(fmaxf(q, -127.0f), 127.0f);
}

// A row's scale from the largest |x| as bits (those of infinities and NaN are the largest of all).
struct RowScale {
    float s, rs, up;  // scale; reciprocal of s * up; what x and s are multiplied with first
    __device__ __forceinline__ explicit RowScale(uint32_t top) {
        s = top < 0x7F800000u ? __uint_as_float(top) / 127.0f : __builtin_nanf("");
        // a reciprocal has to be finite: scales of the smallest rows go up by 2^64 with their x
        up = s < 0x1p-100f ? 0x1p64f : 1.0f;
        rs = 1.0f / (s * up);
    }
    __device__ __forceinline__ uint32_t four(const float* x) const {
        uint32_t w = 0;
        if (s > 0.0f)  // (neither zero nor NaN)
#pragma unroll
            for (int i = 0; i < 4; i++) w |= (uint32_t)(quantized(x[i] * up, s * up, rs) & 255) << (8 * i);
        return w;
    }
};

// One workgroup a row; C chunks of eight elements stay in a thread's registers
// between the search for the largest and the rounding, so x is read once (0: any
// length, read twice).
template <typename X, int C>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const X* __restrict__ x, size_t m, int K, int Kp, int8_t* __restrict__ q,
                                                            float* __restrict__ scale) {
    __shared__ uint32_t red[4];
    const int tid = threadIdx.x;
    for (size_t row = blockIdx.x; row < m; row += gridDim.x) {
        const X* xr = x + row * K;
        uint2* qr = (uint2*)(q + row * Kp);
        auto load = [&](int c, float (&v)[8]) {
            const int k = c * 8;
            if (k + 8 <= K) {
                load8_any(xr + k, v);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = k + i < K ? (float)xr[k + i] : 0.0f;
            }
        };
        float v[C ? C : 1][8];
        uint32_t top = 0;
        auto look = [&](const float (&t)[8]) {
#pragma unroll
            for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(t[i]) & 0x7FFFFFFFu);
        };
        if constexpr (C > 0) {
#pragma unroll
            for (int c = 0; c < C; c++) load(c * 256 + tid, v[c]);
#pragma unroll
            for (int c = 0; c < C; c++) look(v[c]);
        } else {
            for (int c = tid; c * 8 < K; c += 256) {
                load(c, v[0]);
                look(v[0]);
            }
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
        if ((tid & 63) == 0) red[tid >> 6] = top;
        __syncthreads();
        const RowScale rs(max(max(red[0], red[1]), max(red[2], red[3])));
        __syncthreads();
        if (tid == 0) scale[row] = rs.s;
        if constexpr (C > 0) {
#pragma unroll
            for (int c = 0; c < C; c++)
                if ((c * 256 + tid) * 8 < Kp) qr[c * 256 + tid] = make_uint2(rs.four(v[c]), rs.four(v[c] + 4));
        } else {
            for (int c = tid; c * 8 < Kp; c += 256) {
                load(c, v[0]);
                qr[c] = make_uint2(rs.four(v[0]), rs.four(v[0] + 4));
            }
        }
    }
}

template <typename X>
static void quantize_types(const void* x, size_t m, size_t K, size_t Kp, int8_t* q, float* scale, hipStream_t s) {
    const dim3 grid((unsigned)std::min<size_t>(m, (size_t)1 << 20));
    auto go = [&](auto c) {
        TH_LAUNCH((quantize_rows_kernel<X, decltype(c)::value>), grid, dim3(256), 0, s, (const X*)x, m, (int)K, (int)Kp, q, scale);
    };
    if (Kp <= 2048) go(std::integral_constant<int, 1>{});
    else if (Kp <= 4096) go(std::integral_constant<int, 2>{});
    else if (Kp <= 8192) go(std::integral_constant<int, 4>{});
    else if (Kp <= 16384) go(std::integral_constant<int, 8>{});
    else go(std::integral_constant<int, 0>{});
    TH_LAUNCH_CHECK();
}

void launch_quantize_rows(const void* x, th_dtype xdt, size_t m, size_t K, int8_t* q, float* scale, hipStream_t s) {
    if (m == 0) return;
    const size_t Kp = round_up(K, 64);
    if (xdt == TH_F32) quantize_types<float>(x, m, K, Kp, q, scale, s);
    else if (xdt == TH_F16) quantize_types<_Float16>(x, m, K, Kp, q, scale, s);
    else quantize_types<__bf16>(x, m, K, Kp, q, scale, s);
}

// Rows of int8 into the tiles of th_qweight, and their scales: zeros behind K and the last row.
__global__ __launch_bounds__(256) void q8_pack_kernel(const int8_t* __restrict__ q, const float* __restrict__ scale, int rows, int Np, int K,
                                                      int Kp, uint4* __restrict__ tiles, float* __restrict__ scales, size_t n) {
    for (int i = blockIdx.x * 256 + threadIdx.x; i < Np; i += gridDim.x * 256) scales[i] = i < rows ? scale[i] : 0.0f;
    for (size_t i = blockIdx.x * (size_t)256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        const int lane = (int)(i & 63), NCH = Kp >> 6;
        const size_t t = i >> 6, row = t / NCH * 16 + (lane & 15);
        const int k = (int)(t % NCH) * 64 + (lane >> 4) * 16;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row < (size_t)rows && k < K) {
            v = *(const uint4*)(q + row * Kp + k);
            if (K - k < 16) {
                uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int have = K - k - 4 * j;
                    if (have < 4) w[j] &= have <= 0 ? 0u : (1u << (8 * have)) - 1u;
                }
                v = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        tiles[i] = v;
    }
}

void launch_q8_pack(const int8_t* q, const float* scale, const th_qweight* w, hipStream_t s) {
    const size_t n = w->data_bytes / 16;
    TH_LAUNCH(q8_pack_kernel, dim3((unsigned)std::min<size_t>(ceil_div(n, 256), 8192)), dim3(256), 0, s, q, scale, (int)w->rows, (int)w->Np,
              (int)w->cols, (int)w->Kp, (uint4*)w->data, (float*)w->scales, n);
    TH_LAUNCH_CHECK();
}

// ---------------------------------------------------------------------------
// Products
// ---------------------------------------------------------------------------

template <int RT, int CB, int U>
static void i8_rows_launch(const th_qweight* w, const int8_t* xq, const I8Out& out, size_t m, hipStream_t s) {
    constexpr int NW = 8;
    constexpr size_t smem = (size_t)NW * RT * CB * 1024;
    auto k = i8_rows_kernel<RT, CB, U, NW>;
    (void)hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    const size_t nbx = ceil_div(w->Np / 16, (size_t)RT), nby = ceil_div(m, (size_t)(16 * CB));
    TH_LAUNCH(k, dim3((unsigned)(nbx * nby)), dim3(64 * NW), smem, s, (const uint4*)w->data, xq, out, (int)m, (int)w->Kp, (int)nbx);
    TH_LAUNCH_CHECK();
}

template <int TM, int TN, int WPE>
static void i8_tile_launch(th_device* dev, const th_qweight* w, const int8_t* xq, const I8Out& out, size_t m, size_t ks) {
    constexpr size_t smem = (size_t)3 * 4 * (TM + TN) * 1024 + 64 * (TM + 2 * TN) * 4;
    auto k = i8_tile_kernel<TM, TN, WPE>;
    (void)hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    const size_t NCH = w->Kp / 64, cps = ceil_div(NCH, ks);
    ks = ceil_div(NCH, cps);
    int* part = ks > 1 ? (int*)device_scratch(dev, ks * m * w->rows * 4) : nullptr;
    const dim3 grid((unsigned)ceil_div(w->rows, (size_t)(64 * TN)), (unsigned)ceil_div(m, (size_t)(64 * TM)), (unsigned)ks);
    TH_LAUNCH(k, grid, dim3(256), smem, dev->stream, (const uint4*)w->data, xq, out, (int)m, (int)w->Kp, (int)cps, part);
    TH_LAUNCH_CHECK();
    if (part) {
        TH_LAUNCH(i8_join_kernel, dim3((unsigned)std::min<size_t>(ceil_div(m * w->rows, 256), 8192)), dim3(256), 0, dev->stream, part, out, (int)m,
                  (int)ks);
        TH_LAUNCH_CHECK();
    }
}

static void i8_linear(th_device* dev, const th_qweight* w, const int8_t* xq, const I8Out& out, size_t m) {
    const hipStream_t s = dev->stream;
    if (m <= 16) i8_rows_launch<1, 1, 8>(w, xq, out, m, s);
    else if (m <= 64) i8_rows_launch<2, 4, 2>(w, xq, out, m, s);
    else if (m <= 1024) i8_tile_launch<2, 2, 2>(dev, w, xq, out, m, 1);
    else i8_tile_launch<4, 4, 1>(dev, w, xq, out, m, 1);
}

void launch_i8_linear(th_device* dev, const th_qweight* w, const int8_t* xq, const I8Out& out, size_t m) {
    // a launch has below 2^32 threads: at most 8 for each 16 x 16 results
    const size_t rows = std::max<size_t>(16, ((size_t)1 << 28) / (w->Np / 16) / 16 * 16);
    for (size_t m0 = 0; m0 < m; m0 += rows) {
        I8Out o = out;
        o.y = (char*)out.y + m0 * w->rows * dtype_size(out.dt);
        o.xs = out.xs + m0;
        i8_linear(dev, w, xq + m0 * w->Kp, o, std::min(rows, m - m0));
    }
}

}  // namespace th
