// Rows to 8-bit integers, and their product with 8-bit weights (i8gemm.hpp).
#include <algorithm>

#include "capi_util.hpp"
#include "i8kernels.hpp"

namespace th {

// ---------------------------------------------------------------------------
// Rows to integers
// ---------------------------------------------------------------------------

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
#pragma unroll
        for (int i = 0; i < 4; i++) w |= (uint32_t)(quantized(x[i] * up, s * up, rs) & 255) << (8 * i);
        return w;
    }
    // Sixteen of a row: the integer is what an addition of 1.5 2^23 leaves in the low byte. x rs is off by 2^-17, so
    // only where one lies as near to a half, for one in 25000, the sixteen are rounded as above (8192 rows of 4096 in bf16:
    // 26 us; with all of them so it took 41, bound by instructions).
    __device__ __forceinline__ uint4 sixteen(const float (&x)[16]) const {
        if (!(s > 0.0f)) return make_uint4(0, 0, 0, 0);  // (zero or NaN)
        uint32_t y[16], w[4];
        float most = up > 1.0f ? 1.0f : 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float v = __builtin_fmaf(x[i], rs, 0x1.8p23f);
            most = fmaxf(most, fabsf(__builtin_fmaf(x[i], rs, 0x1.8p23f - v)));
            y[i] = __float_as_uint(v);
        }
        if (most > 0.49998f) return make_uint4(four(x), four(x + 4), four(x + 8), four(x + 12));
#pragma unroll
        for (int i = 0; i < 4; i++)
            w[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(y[4 * i + 3], y[4 * i + 2], 0x0C0C0400u),
                                         __builtin_amdgcn_perm(y[4 * i + 1], y[4 * i], 0x0C0C0400u), 0x05040100u);
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// The largest |x| of sixteen, as the bits of a float, over what `top` has; 16-bit values two at a time.
template <typename X>
struct RowTop {
    typedef X r16_t __attribute__((ext_vector_type(16)));
    typedef uint16_t h2_t __attribute__((ext_vector_type(2)));
    typedef uint32_t u8_t __attribute__((ext_vector_type(8)));
    uint32_t top = 0;
    h2_t top2 = {0, 0};
    __device__ __forceinline__ void look(const r16_t& r) {
        if constexpr (sizeof(X) == 4) {
#pragma unroll
            for (int i = 0; i < 16; i++) top = max(top, __float_as_uint((float)r[i]) & 0x7FFFFFFFu);
        } else {
            const u8_t v = __builtin_bit_cast(u8_t, r);
#pragma unroll
            for (int i = 0; i < 8; i++) top2 = __builtin_elementwise_max(top2, __builtin_bit_cast(h2_t, v[i] & 0x7FFF7FFFu));
        }
    }
    __device__ __forceinline__ uint32_t bits() const {
        if constexpr (sizeof(X) == 4) return top;
        else return __float_as_uint((float)__builtin_bit_cast(X, (uint16_t)max(top2.x, top2.y)));
    }
};

// WPR waves a row, ROWS rows a workgroup; a lane has 16 consecutive elements, one
// piece of a block, and up to IT pieces stay in its registers between the search
// for the largest and the rounding (0: any length, read twice).  Few rows: four
// waves each, for the latency of one.  Many: four rows a workgroup, which leave their
// blocks together, of two waves or four (8192 x 4096 in bf16, waves by rows: 2 x 4 26 us, 2 x 8 27, 2 x 2 28, 4 x 4 31,
// 1 x 16, which the chip holds all at once, so that reading and writing take turns, 32).
template <typename X, int WPR, int ROWS, int IT>
__global__ __launch_bounds__(64 * WPR * ROWS) void quantize_rows_kernel(const X* __restrict__ x, int m, int K, int Kp, int8_t* __restrict__ q,
                                                                        float* __restrict__ scale, int whole) {
    typedef X x16_t __attribute__((ext_vector_type(16), aligned(sizeof(X))));
    typedef X r16_t __attribute__((ext_vector_type(16)));
    __shared__ uint32_t red[WPR * ROWS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = (wave % WPR) * 64 + lane;
    const int row = blockIdx.x * ROWS + wave / WPR;
    const bool there = row < m;
    const X* xr = x + (size_t)(there ? row : 0) * K;
    auto load = [&](int c) -> r16_t {
        const int k = c * 16;
        if (there && k + 16 <= K) return *(const x16_t*)(xr + k);
        r16_t r;
#pragma unroll
        for (int i = 0; i < 16; i++) r[i] = there && k + i < K ? xr[k + i] : (X)0.0f;
        return r;
    };
    RowTop<X> of_lane;
    r16_t held[IT ? IT : 1];
    if constexpr (IT > 0) {
#pragma unroll
        for (int i = 0; i < IT; i++) held[i] = load(i * 64 * WPR + t);
#pragma unroll
        for (int i = 0; i < IT; i++) of_lane.look(held[i]);
    } else {
        for (int c = t; c * 16 < K; c += 64 * WPR) of_lane.look(load(c));
    }
    uint32_t top = of_lane.bits();
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    if constexpr (WPR > 1) {
        if (lane == 0) red[wave] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WPR; i++) top = max(top, red[wave / WPR * WPR + i]);
    }
    const int first = row & ~15, h = whole ? 16 : min(16, m - first);
    if (!there && !(whole && first < m)) return;
    const RowScale rs(top);
    if (t == 0) scale[row] = rs.s;
    uint4* const to = (uint4*)(q + (size_t)first * Kp) + (row & 15);
    auto put = [&](int c, const r16_t& r) {
        if (c * 16 >= Kp) return;
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = (float)r[i];
        to[(size_t)c * h] = rs.sixteen(v);
    };
    if constexpr (IT > 0) {
#pragma unroll
        for (int i = 0; i < IT; i++) put(i * 64 * WPR + t, held[i]);
    } else {
        for (int c = t; c * 16 < Kp; c += 64 * WPR) put(c, load(c));
    }
}

template <typename X>
static void quantize_types(const void* x, size_t m, size_t K, size_t Kp, int8_t* q, float* scale, bool whole, hipStream_t s) {
    auto go = [&](auto wpr, auto rows, auto it) {
        constexpr int W = decltype(wpr)::value, R = decltype(rows)::value;
        const size_t n = whole ? round_up(m, 16) : m;
        TH_LAUNCH((quantize_rows_kernel<X, W, R, decltype(it)::value>), dim3((unsigned)ceil_div(n, (size_t)R)), dim3(64 * W * R), 0, s, (const X*)x,
                  (int)m, (int)K, (int)Kp, q, scale, (int)whole);
    };
    using std::integral_constant;
    const integral_constant<int, 1> one;
    const integral_constant<int, 2> two;
    const integral_constant<int, 4> four;
    if (m >= 1024 && Kp <= 4096) go(two, four, two);
    else if (m >= 1024 && Kp <= 16384) go(four, four, four);
    else if (Kp <= 4096) go(four, one, one);
    else if (Kp <= 16384) go(four, one, four);
    else go(four, one, integral_constant<int, 0>{});
    TH_LAUNCH_CHECK();
}

void launch_quantize_rows(const void* x, th_dtype xdt, size_t m, size_t K, int8_t* q, float* scale, bool whole, hipStream_t s) {
    constexpr size_t ROWS = (size_t)1 << 22;  // a launch has below 2^32 threads
    const size_t Kp = round_up(K, 64);
    for (size_t m0 = 0; m0 < m; m0 += ROWS) {
        const void* xo = (const char*)x + m0 * K * dtype_size(xdt);
        const size_t n = std::min(ROWS, m - m0);
        int8_t* qo = q + m0 * Kp;
        if (xdt == TH_F32) quantize_types<float>(xo, n, K, Kp, qo, scale + m0, whole, s);
        else if (xdt == TH_F16) quantize_types<_Float16>(xo, n, K, Kp, qo, scale + m0, whole, s);
        else quantize_types<__bf16>(xo, n, K, Kp, qo, scale + m0, whole, s);
    }
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
    TH_LAUNCH(k, dim3((unsigned)ceil_div(w->Np / 16, (size_t)RT)), dim3(64 * NW), smem, s, (const uint4*)w->data, xq, out, (int)m, (int)w->Kp);
    TH_LAUNCH_CHECK();
}

template <int TM, int TN, int KW, int ST, int WPE>
static void i8_tile_launch(const th_qweight* w, const int8_t* xq, const I8Out& out, size_t m, hipStream_t s) {
    constexpr int smem = I8TileLds<TM, TN, KW>::BYTES;
    auto k = i8_tile_kernel<TM, TN, KW, ST, WPE>;
    (void)hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, smem);
    const dim3 grid((unsigned)ceil_div(w->rows, (size_t)(64 * TN)), (unsigned)ceil_div(m, (size_t)(64 * TM)));
    TH_LAUNCH(k, grid, dim3(256 * KW), smem, s, (const uint4*)w->data, xq, out, (int)m, (int)w->Kp);
    TH_LAUNCH_CHECK();
}

static void i8_launch(I8Form form, const th_qweight* w, const int8_t* xq, const I8Out& out, size_t m, hipStream_t s) {
    switch (form) {
        case I8Form::ROWS_1X1: return i8_rows_launch<1, 1, 8>(w, xq, out, m, s);
        case I8Form::ROWS_1X2: return i8_rows_launch<1, 2, 4>(w, xq, out, m, s);
        case I8Form::ROWS_2X2: return i8_rows_launch<2, 2, 4>(w, xq, out, m, s);
        case I8Form::ROWS_1X4: return i8_rows_launch<1, 4, 2>(w, xq, out, m, s);
        case I8Form::ROWS_2X4: return i8_rows_launch<2, 4, 2>(w, xq, out, m, s);
        case I8Form::ROWS_3X4: return i8_rows_launch<3, 4, 2>(w, xq, out, m, s);
        case I8Form::TILE_64X64: return i8_tile_launch<1, 1, 1, 4, 4>(w, xq, out, m, s);
        case I8Form::TILE_64X128_TWO: return i8_tile_launch<1, 2, 2, 2, 2>(w, xq, out, m, s);
        case I8Form::TILE_64X128: return i8_tile_launch<1, 2, 1, 4, 3>(w, xq, out, m, s);
        case I8Form::TILE_128X128: return i8_tile_launch<2, 2, 1, 2, 2>(w, xq, out, m, s);
        case I8Form::TILE_128X256: return i8_tile_launch<2, 4, 1, 2, 2>(w, xq, out, m, s);
        case I8Form::TILE_256X256: return i8_tile_launch<4, 4, 1, 2, 1>(w, xq, out, m, s);
    }
}

void launch_i8_linear(th_device* dev, const th_qweight* w, const int8_t* xq, const I8Out& out, size_t m) {
    const size_t rows = i8_rows_at_once(w->rows);
    for (size_t m0 = 0; m0 < m; m0 += rows) {
        I8Out o = out;
        o.y = (char*)out.y + m0 * w->rows * dtype_size(out.dt);
        o.xs = out.xs + m0;
        const size_t n = std::min(rows, m - m0);
        i8_launch(i8_form(n, w->rows, w->cols, (size_t)dev->num_cus), w, xq + m0 * w->Kp, o, n, dev->stream);
    }
}

}  // namespace th
