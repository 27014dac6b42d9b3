// Norms of query and key heads in the same pass as their rotation, into rows
// or into the pages of a cache.
//
// A head h of hd dims becomes h / sqrt(mean(h^2) + eps) * w, then its pairs turn
// as in kvpages.hip.  All in f32, rounded once to the output's type.
#include <algorithm>

#include "kvcache.hpp"
#include "kvrows.hpp"
#include "ops.hpp"

namespace th {

// Sums of squares outside of this range (f32's squares may have left its range,
// above or below) are formed again in f64.
constexpr float NORM_LOW = 1e-30f, NORM_HIGH = 1e38f;

template <int G>
__device__ __forceinline__ double group_sum64(double v) {
#pragma unroll
    for (int o = 1; o < G; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// v[i] over the root mean square of the head's values, which G lanes hold.
template <int G, int N>
__device__ __forceinline__ void norm_head(float (&v)[N], int hd, float eps) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) ss = __builtin_fmaf(v[i], v[i], ss);
    ss = group_sum<G>(ss);
    if (ss > NORM_LOW && ss < NORM_HIGH) {
        const float inv = 1.0f / sqrtf(ss / (float)hd + eps);
#pragma unroll
        for (int i = 0; i < N; i++) v[i] *= inv;
    } else {
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < N; i++) s += (double)v[i] * (double)v[i];
        const double inv = 1.0 / sqrt(group_sum64<G>(s) / (double)hd + (double)eps);
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = (float)((double)v[i] * inv);
    }
}

__device__ __forceinline__ kv_f8 load_w8(const void* w, int bf16, int d) {
    kv_f8 r;
    if (!w) {
#pragma unroll
        for (int i = 0; i < 8; i++) r.v[i] = 1.0f;
        return r;
    }
    return bf16 ? kv_load8((const __bf16*)w + d) : kv_load8((const float*)w + d);
}

// Where head hh of row `row` is read, where it goes, and what is done to it.
struct HeadAt {
    size_t src, at;
    const void* in;
    void* out;
    th_dtype dt;
    int kind;  // 0: query, 1: key, 2: value (as it is)
};
template <bool APPEND>
__device__ __forceinline__ HeadAt head_at(const KvRopeArgs& a, const KvPages& p, th_dtype cache, const KvRow& r, size_t row, int hh) {
    HeadAt t;
    if (hh < a.n_heads) {
        t.kind = 0;
        t.in = a.q;
        t.src = row * a.q_row + (size_t)hh * a.hd;
        t.out = a.q_out;
        t.dt = a.qdt;
        t.at = row * a.qo_row + (size_t)hh * a.hd;
        return t;
    }
    const int n_kv = APPEND ? p.n_kv_heads : a.n_kv;
    int h = hh - a.n_heads;
    t.kind = 1;
    if (APPEND && h >= n_kv) {
        t.kind = 2;
        h -= n_kv;
    }
    t.in = t.kind == 1 ? a.k : a.v;
    t.src = row * (t.kind == 1 ? a.k_row : a.v_row) + (size_t)h * a.hd;
    if (APPEND) {
        const int page = p.table[(size_t)r.seq * p.pages_per_seq + (r.pos >> p.shift)];
        t.out = const_cast<void*>(t.kind == 1 ? p.k : p.v);
        t.dt = cache;
        t.at = ((((size_t)page * p.n_kv_heads + h) << p.shift) + (r.pos & ((1 << p.shift) - 1))) * a.hd;
    } else {
        t.out = a.k_out;
        t.dt = a.kdt;
        t.at = row * a.ko_row + (size_t)h * a.hd;
    }
    return t;
}

// A head is held by G lanes, sixteen of its dims in each: two chunks of eight
// that hold the lane's eight pairs whole in either layout (so one table row's
// eight cosines and sines serve both).  G: the next power of two (80 and 96 dims
// leave lanes of eight idle).  Bound by memory: q and k are read once and written
// once; 16000 packed bf16 rows of 32 + 8 heads of 128 80 us, 4.1 TB/s; 16000 f32 rows of 32 + 8 + 8
// heads into an f16 cache 138 us, 5.3 TB/s.  One token: a launch.
template <typename X, int G, bool APPEND>
__global__ __launch_bounds__(256) void norm_heads_kernel(KvRopeArgs a, KvPages p, th_dtype cache, const int* __restrict__ n_rows_dev,
                                                         const KvRow* __restrict__ rows, size_t n_rows, int heads, int slots) {
    if (APPEND) n_rows = (size_t)*n_rows_dev;
    const int c = threadIdx.x % G, turned = a.rot / 16, hr = a.rot / 2;
    const bool pairs = c < turned;
    const int d0 = a.half && pairs ? 8 * c : 16 * c, d1 = a.half && pairs ? 8 * c + hr : 16 * c + 8;
    const bool has0 = d0 < a.hd, has1 = d1 < a.hd;
    const size_t total = n_rows * slots, step = (size_t)gridDim.x * (256 / G);
    for (size_t g = blockIdx.x * (size_t)(256 / G) + threadIdx.x / G; g < total; g += step) {
        const size_t row = total >> 32 ? g / slots : (uint32_t)g / (uint32_t)slots;
        const int slot = (int)(g - row * slots);
        KvRow r = {};
        if (APPEND) r = rows[row];
        const size_t pos = a.positions ? (size_t)a.positions[row] : APPEND ? (size_t)r.pos : a.start + row;
        const bool known = pos < a.table_rows;
        kv_f8 cs, sn;
        if (pairs) {
            cs = kv_load8(a.cos_t + (known ? pos : 0) * hr + 8 * c);
            sn = kv_load8(a.sin_t + (known ? pos : 0) * hr + 8 * c);
        }
        typedef X x8_t __attribute__((ext_vector_type(8)));
        x8_t nx = {}, ny = {};  // the next head's dims, on their way while one is worked on
        auto fetch = [&](int hh) {
            const HeadAt t = head_at<APPEND>(a, p, cache, r, row, hh);
            const X* src = (const X*)t.in + t.src;
            if (has0) nx = *(const x8_t*)(src + d0);
            if (has1) ny = *(const x8_t*)(src + d1);
        };
        fetch(slot);
        for (int hh = slot; hh < heads; hh += slots) {
            const HeadAt t = head_at<APPEND>(a, p, cache, r, row, hh);
            float v[16];
            kv_f8 x, y;
#pragma unroll
            for (int i = 0; i < 8; i++) x.v[i] = (float)nx[i], y.v[i] = (float)ny[i];
            if (hh + slots < heads) fetch(hh + slots);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = x.v[i], v[8 + i] = y.v[i];
            if (t.kind != 2) {
                norm_head<G>(v, a.hd, a.eps);
                const void* w = t.kind == 0 ? a.qw : a.kw;
                const int bf16 = t.kind == 0 ? a.qw_bf16 : a.kw_bf16;
                if (w) {
                    kv_f8 w0 = {}, w1 = {};
                    if (has0) w0 = load_w8(w, bf16, d0);
                    if (has1) w1 = load_w8(w, bf16, d1);
#pragma unroll
                    for (int i = 0; i < 8; i++) v[i] *= w0.v[i], v[8 + i] *= w1.v[i];
                }
                if (pairs) {
                    float u[16];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int e = a.half ? 0 : 1;
                        const float s = e ? v[2 * i] : v[i], o = e ? v[2 * i + 1] : v[8 + i];
                        const float first = known ? s * cs.v[i] - o * sn.v[i] : __builtin_nanf("");
                        const float second = known ? s * sn.v[i] + o * cs.v[i] : __builtin_nanf("");
                        u[i] = first;
                        u[8 + i] = second;
                    }
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        // (both forms by constant indexes: the arrays stay in registers)
                        const float a0 = u[i], a1 = u[8 + i], b0 = (i & 1) ? u[8 + i / 2] : u[i / 2],
                                    b1 = (i & 1) ? u[8 + 4 + i / 2] : u[4 + i / 2];
                        v[i] = a.half ? a0 : b0;
                        v[8 + i] = a.half ? a1 : b1;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 8; i++) x.v[i] = v[i], y.v[i] = v[8 + i];
            if (has0) kv_store8(t.out, t.dt, t.at + d0, x);
            if (has1) kv_store8(t.out, t.dt, t.at + d1, y);
        }
    }
}

// Any head size, pair count, stride: a wave takes a head, and its lanes the
// elements one by one (its second look at them comes from the caches).  Bound by its loads and stores of
// one element: 16000 packed bf16 rows of 32 + 8 heads of 128, 20 dims turned, 453 us, 0.72 TB/s, where widths that are a
// multiple of 16 take 74 to 77; 61 rows 4.7 against 4.0.
template <typename X, bool APPEND>
__global__ __launch_bounds__(256) void norm_any_kernel(KvRopeArgs a, KvPages p, th_dtype cache, const int* __restrict__ n_rows_dev,
                                                       const KvRow* __restrict__ rows, size_t n_rows, int heads) {
    if (APPEND) n_rows = (size_t)*n_rows_dev;
    const int lane = threadIdx.x & 63, hr = a.rot / 2;
    const size_t total = n_rows * heads, step = (size_t)gridDim.x * 4;
    for (size_t g = blockIdx.x * (size_t)4 + (threadIdx.x >> 6); g < total; g += step) {
        const size_t row = g / heads;
        KvRow r = {};
        if (APPEND) r = rows[row];
        const HeadAt t = head_at<APPEND>(a, p, cache, r, row, (int)(g - row * heads));
        const X* src = (const X*)t.in + t.src;
        if (t.kind == 2) {
            for (int d = lane; d < a.hd; d += 64) kv_store1(t.out, t.dt, t.at + d, (float)src[d]);
            continue;
        }
        const size_t pos = a.positions ? (size_t)a.positions[row] : APPEND ? (size_t)r.pos : a.start + row;
        const bool known = pos < a.table_rows;
        const float *ct = a.cos_t + (known ? pos : 0) * hr, *st = a.sin_t + (known ? pos : 0) * hr;
        float ss = 0.0f;
        for (int d = lane; d < a.hd; d += 64) {
            const float v = (float)src[d];
            ss = __builtin_fmaf(v, v, ss);
        }
        ss = group_sum<64>(ss);
        const bool plain = ss > NORM_LOW && ss < NORM_HIGH;
        float inv = 1.0f / sqrtf(ss / (float)a.hd + a.eps);
        double inv64 = 0.0;
        if (!plain) {
            double s = 0.0;
            for (int d = lane; d < a.hd; d += 64) s += (double)(float)src[d] * (double)(float)src[d];
            inv64 = 1.0 / sqrt(group_sum64<64>(s) / (double)a.hd + (double)a.eps);
        }
        const void* w = t.kind == 0 ? a.qw : a.kw;
        const int bf16 = t.kind == 0 ? a.qw_bf16 : a.kw_bf16;
        auto value = [&](int d) {
            const float x = (float)src[d], v = plain ? x * inv : (float)((double)x * inv64);
            return w ? v * load_w(w, bf16, d) : v;
        };
        for (int i = lane; i < a.hd - hr; i += 64) {
            if (i >= hr) {
                kv_store1(t.out, t.dt, t.at + i + hr, value(i + hr));
                continue;
            }
            const int e0 = a.half ? i : 2 * i, e1 = a.half ? i + hr : 2 * i + 1;
            const float x = value(e0), y = value(e1), cs = ct[i], sn = st[i];
            kv_store1(t.out, t.dt, t.at + e0, known ? x * cs - y * sn : __builtin_nanf(""));
            kv_store1(t.out, t.dt, t.at + e1, known ? x * sn + y * cs : __builtin_nanf(""));
        }
    }
}

// Chunks of eight need rows and heads that start on 16 bytes, and whole chunks of pairs.
static bool norm_vec(const KvRopeArgs& a, bool append) {
    const size_t ins = dtype_size(a.xdt), qs = dtype_size(a.qdt), ks = dtype_size(a.kdt);
    bool ok = a.hd % 8 == 0 && a.rot % 16 == 0 && a.hd <= 1024 && a.k_row * ins % 16 == 0;
    if (a.n_heads) ok = ok && a.q_row * ins % 16 == 0 && a.qo_row * qs % 16 == 0;
    return ok && (append ? a.v_row * ins % 16 == 0 : a.ko_row * ks % 16 == 0);
}

template <bool APPEND>
static void norm_launch(const KvRopeArgs& a, const KvPages& p, th_dtype cache, const int* n_rows_dev, const KvRow* rows, size_t n_rows,
                        int heads, hipStream_t s) {
    if (n_rows == 0 || heads == 0) return;
    const bool vec = norm_vec(a, APPEND);
    auto blocks = [&](size_t per_block, size_t units) { return dim3((unsigned)std::min<size_t>(ceil_div(units, per_block), 16384)); };
    auto types = [&](auto x) {
        using X = decltype(x);
        if (!vec) {
            TH_LAUNCH((norm_any_kernel<X, APPEND>), blocks(4, n_rows * heads), dim3(256), 0, s, a, p, cache, n_rows_dev, rows, n_rows, heads);
            return;
        }
        auto lanes = [&](auto g) {
            constexpr int G = decltype(g)::value;
            // Beyond two rounds of the chip's waves each group of lanes takes four heads of its row, for one reading of the tables
            // (16000 rows of 40 heads in bf16: 105 against 80 us; 61 rows of 32 heads, four layers: 28.6 against 18.1).  n_rows is what
            // the launch is for: a captured append's max_rows (61 rows of 16 + 8 + 8 heads of 64, four layers a replay: 20.7 us
            // captured for 64 rows, 20.5 for 4096, 32.9 for 16000).
            const int slots = n_rows * heads * G >= (size_t)1 << 20 ? (heads + 3) / 4 : heads;
            TH_LAUNCH((norm_heads_kernel<X, G, APPEND>), blocks(256 / G, n_rows * slots), dim3(256), 0, s, a, p, cache, n_rows_dev, rows,
                      n_rows, heads, slots);
        };
        if (a.hd <= 64) lanes(std::integral_constant<int, 4>{});
        else if (a.hd <= 128) lanes(std::integral_constant<int, 8>{});
        else if (a.hd <= 256) lanes(std::integral_constant<int, 16>{});
        else lanes(std::integral_constant<int, 64>{});
    };
    if (a.xdt == TH_F32) types(float{});
    else if (a.xdt == TH_F16) types((_Float16)0);
    else types((__bf16)0.0f);
    TH_LAUNCH_CHECK();
}

void launch_norm_append(const KvRopeArgs& a, const KvPages& p, th_dtype cache, const int* n_rows_dev, const KvRow* rows, size_t n_rows,
                        hipStream_t s) {
    norm_launch<true>(a, p, cache, n_rows_dev, rows, n_rows, a.n_heads + 2 * p.n_kv_heads, s);
}

void launch_norm_rows(const KvRopeArgs& a, size_t n_rows, hipStream_t s) {
    norm_launch<false>(a, KvPages{}, TH_F32, nullptr, nullptr, n_rows, a.n_heads + a.n_kv, s);
}

}  // namespace th
