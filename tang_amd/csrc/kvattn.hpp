// Device code that the two attention kernels over a paged cache share.
#pragma once

#include "kvcache.hpp"
#include "ops.hpp"
#include "qlinear.hpp"

namespace th {

typedef float kv_f32x4_t __attribute__((ext_vector_type(4)));
typedef float kv_f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t kv_u4_t __attribute__((ext_vector_type(4)));
typedef short kv_s4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) kv_s4_t kv_lds_s4_t;

template <typename E> struct KvVec;
template <> struct KvVec<_Float16> {
    typedef _Float16 x8 __attribute__((ext_vector_type(8)));
    typedef _Float16 x2 __attribute__((ext_vector_type(2)));
};
template <> struct KvVec<__bf16> {
    typedef __bf16 x8 __attribute__((ext_vector_type(8)));
    typedef __bf16 x2 __attribute__((ext_vector_type(2)));
};

__device__ __forceinline__ kv_f32x4_t kv_mfma16(KvVec<_Float16>::x8 a, KvVec<_Float16>::x8 b, kv_f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ kv_f32x4_t kv_mfma16(KvVec<__bf16>::x8 a, KvVec<__bf16>::x8 b, kv_f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ kv_f32x16_t kv_mfma32(KvVec<_Float16>::x8 a, KvVec<_Float16>::x8 b, kv_f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ kv_f32x16_t kv_mfma32(KvVec<__bf16>::x8 a, KvVec<__bf16>::x8 b, kv_f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// Operands that are wider than the cache's type (f32 queries, the
// probabilities of f32 results) go in as a sum of NP values of that type: each
// takes the bits that the ones before left, rounded to nearest.  Two f16 are off by
// 2^-24 of the value at most (2^-12 is left behind the first, and 2^-12 of that), three
// bf16 by 2^-27: an f32's own rounding or less.  NP = 1 is for queries and
// results of the cache's type.  Their weights are two values in rows items, which leaves 2^-18 (bf16) or less and is hidden behind the
// reads of K and V (48 ragged sequences 120 us with one and with two), and one in tiles, where a second takes half as many MFMAs again (a prompt of 8192
// in bf16: 605 us, with two 807).  Its rounding, half a step, comes on top of the result's own half step, for each weight in a direction of its own.
template <typename E> constexpr int kv_wide_parts() { return sizeof(E) == 2 && std::is_same<E, __bf16>::value ? 3 : 2; }

template <typename E, int NP>
__device__ __forceinline__ void kv_split(float x, E (&part)[NP]) {
#pragma unroll
    for (int i = 0; i < NP; i++) {
        part[i] = (E)x;
        x -= (float)part[i];
    }
}
// The parts of x * up and y * up, up a power of two, as pairs.  Each rest is one operation on x itself, and the first
// pair a new value to the compiler, which would else make half of it twice.
template <typename E, int NP>
__device__ __forceinline__ void kv_split_pair(float x, float y, float up, typename KvVec<E>::x2 (&part)[NP]) {
    typedef typename KvVec<E>::x2 x2;
    part[0] = x2{(E)(x * up), (E)(y * up)};
    if constexpr (NP > 1) {
        uint32_t pair = __builtin_bit_cast(uint32_t, part[0]);
        asm("" : "+v"(pair));
        part[0] = __builtin_bit_cast(x2, pair);
        float r = __builtin_fmaf(x, up, -(float)part[0][0]), s = __builtin_fmaf(y, up, -(float)part[0][1]);
#pragma unroll
        for (int i = 1; i < NP; i++) {
            part[i] = x2{(E)r, (E)s};
            r -= (float)part[i][0];
            s -= (float)part[i][1];
        }
    }
}
// f16 parts keep their bits if the largest is near the type's end: queries are brought to
// [2^14, 2^15) by a power of two for each row, probabilities (at most 1) by 2^14.
constexpr int KV_Q_TOP = 15;
constexpr float KV_P_UP = 16384.0f;
// Weights of queries and results of the cache's type are taken against a reference that lies KV_*_LOW below the running
// maximum, so that f16's largest come near 2^15 (in tiles the reference may lag by 2^KV_LAG): a weight of 2^-14 of the largest would
// else lose bits below f16's normal range, and one of 2^-25 all of them, and together such weights can be most of a row.  bf16 has f32's range.
constexpr float KV_LAG = 6.0f;
template <typename E> constexpr float kv_rows_low() { return std::is_same<E, _Float16>::value ? 15.0f : 0.0f; }
template <typename E> constexpr float kv_tiles_low() { return std::is_same<E, _Float16>::value ? 15.0f - KV_LAG : 0.0f; }

// sum + a pair's two values, in f32.  The divisor sums the weights as they went into the product, rounded: the quotient is then a mean
// with weights that add up to one, whatever way they were all rounded (equal values give that value).  One instruction, where
// adding the unrounded weights takes two.
__device__ __forceinline__ float kv_add_pair(KvVec<_Float16>::x2 a, float sum) {
    return __builtin_amdgcn_fdot2(a, KvVec<_Float16>::x2{(_Float16)1.0f, (_Float16)1.0f}, sum, false);
}
__device__ __forceinline__ float kv_add_pair(KvVec<__bf16>::x2 a, float sum) {
    return __builtin_amdgcn_fdot2_f32_bf16(a, KvVec<__bf16>::x2{(__bf16)1.0f, (__bf16)1.0f}, sum, false);
}

__device__ __forceinline__ float kv_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// A value that the compiler takes for a new one: what is computed from it stays where it is written. (Addresses that
// a few instructions make again for each block would else fill registers for the whole loop.)
__device__ __forceinline__ int kv_fresh(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// Chain of MFMAs before a branch: what follows may read their results.
__device__ __forceinline__ void kv_mfma_wait() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 15\n\ts_nop 3");
    __builtin_amdgcn_sched_barrier(0);
}

__device__ __forceinline__ float kv_load_q(const void* q, th_dtype dt, size_t at) {
    if (dt == TH_F32) return ((const float*)q)[at];
    if (dt == TH_F16) return (float)((const _Float16*)q)[at];
    return (float)((const __bf16*)q)[at];
}

// N pieces of eight values of a row as f32, all on their way before the first is used;
// piece i starts at `at` + 8 * chunk(i).
template <int N, typename F>
__device__ __forceinline__ void kv_load_row(const void* q, th_dtype dt, size_t at, F&& chunk, float (&x)[N][8]) {
    if (dt == TH_F32) {
        kv_f32x4_t v[N][2];
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int y = 0; y < 2; y++) v[i][y] = *(const kv_f32x4_t*)((const float*)q + at + 8 * chunk(i) + 4 * y);
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) x[i][e] = v[i][e >> 2][e & 3];
    } else {
        kv_u4_t v[N];
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = *(const kv_u4_t*)((const uint16_t*)q + at + 8 * chunk(i));
        auto widen = [&](auto f) {
#pragma unroll
            for (int i = 0; i < N; i++)
#pragma unroll
                for (int e = 0; e < 8; e++) x[i][e] = f((uint16_t)(v[i][e >> 1] >> (16 * (e & 1))));
        };
        if (dt == TH_F16) widen([](uint16_t u) { return (float)__builtin_bit_cast(_Float16, u); });
        else widen([](uint16_t u) { return __uint_as_float((uint32_t)u << 16); });
    }
}

__device__ __forceinline__ void kv_store_out(void* out, th_dtype dt, size_t at, float v) {
    if (dt == TH_F32) ((float*)out)[at] = v;
    else if (dt == TH_F16) ((_Float16*)out)[at] = (_Float16)v;
    else ((__bf16*)out)[at] = (__bf16)v;
}

__device__ __forceinline__ void kv_store_out4(void* out, th_dtype dt, size_t at, kv_f32x4_t v) {
    if (dt == TH_F32) {
        *(kv_f32x4_t*)((float*)out + at) = v;
    } else if (dt == TH_F16) {
        typedef _Float16 h4 __attribute__((ext_vector_type(4)));
        *(h4*)((_Float16*)out + at) = h4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
    } else {
        typedef __bf16 b4 __attribute__((ext_vector_type(4)));
        *(b4*)((__bf16*)out + at) = b4{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
    }
}

// An item, in scalar registers (the workgroup's waves all have the same).
__device__ __forceinline__ KvItem kv_item(const KvItem* items, int n) {
    const kv_u4_t a = ((const kv_u4_t*)(items + n))[0], b = ((const kv_u4_t*)(items + n))[1];
    auto one = [](uint32_t x) { return (int)__builtin_amdgcn_readfirstlane(x); };
    return KvItem{one(a[0]), one(a[1]), one(a[2]), one(a[3]), one(b[0]), one(b[1]), one(b[2]), one(b[3])};
}

// Key j of an item's numbers.
__device__ __forceinline__ int kv_key(const KvItem& it, int j) { return j + (j >= it.sink_end ? it.gap : 0); }
__device__ __forceinline__ uint32_t kv_row(const KvPages& p, int page, int h, int key) {
    return (((uint32_t)page * p.n_kv_heads + h) << p.shift) + (key & ((1 << p.shift) - 1));
}

// Where an item's keys lie.  Sixteen numbers from a multiple of 16 on are sixteen
// neighbouring rows of one page (pages, hidden runs and pieces begin at multiples of 16), so
// addresses are a scalar for sixteen rows and constants of the lane.  One load finds the pages of
// the next 64 such groups, one a lane, a window ahead of their use.
struct KvGroups {
    const int* table;
    int pages, next, base, last;  // this lane's pages; first group of the window; last group of the item
    __device__ __forceinline__ int find(const KvPages& p, const KvItem& it, int b) const {
        return table[kv_key(it, 16 * min(b + (int)(threadIdx.x & 63), last)) >> p.shift];
    }
    __device__ __forceinline__ KvGroups(const KvPages& p, const KvItem& it) {
        table = p.table + (size_t)it.seq * p.pages_per_seq;
        base = it.j0 >> 4;
        last = max(it.j1 - 1, it.j0) >> 4;
        pages = find(p, it, base);
        next = pages;
        if (base + 64 <= last) next = find(p, it, base + 64);
    }
    // before the rows of a block that begins at group b: blocks lie in one window each
    __device__ __forceinline__ void reach(const KvPages& p, const KvItem& it, int b) {
        if (b < base + 64 || b > last) return;  // (behind the end: the last group again)
        base += 64;
        pages = next;
        if (base + 64 <= last) next = find(p, it, base + 64);
    }
    // element offset of group b's first row
    __device__ __forceinline__ size_t at(const KvPages& p, const KvItem& it, int h, int hd, int b) const {
        b = min(b, last);
        const int page = __builtin_amdgcn_readlane(pages, min(b - base, 63));
        return (size_t)kv_row(p, page, h, kv_key(it, 16 * b)) * hd;
    }
};
// 16 bytes at a scalar place plus a lane's byte offset.
template <typename E>
__device__ __forceinline__ kv_u4_t kv_load16(const void* base, size_t at, uint32_t off) {
    return *(const kv_u4_t*)((const char*)((const E*)base + at) + off);
}

// Largest of three (two fmaxf take up to four more instructions: each first quiets its operands).
__device__ __forceinline__ float kv_max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// Whether the row at position pos sees the key.
__device__ __forceinline__ bool kv_sees(int key, int pos, int window, int sinks) {
    return (key <= pos) & ((window == 0) | (key > pos - window) | (key < sinks));
}
// The same in an item's numbers: the row sees number j if j <= hi and not from <= j <= to.
struct KvSeen {
    int hi, from, to;
    __device__ __forceinline__ KvSeen(const KvItem& it, int pos, int window, int sinks) {
        // the last number whose key is at most x
        auto upto = [&](int x) { return x < it.sink_end ? x : max(it.sink_end - 1, x - it.gap); };
        hi = min(upto(pos), it.j1 - 1);
        from = upto(sinks - 1) + 1;
        to = window ? upto(pos - window) : -1;
    }
};

// Split work: a piece of a token's keys leaves, for each query head, its sums and {maximum,
// sum of weights} in a record; a kernel of its own joins them in the records' order.  (Joined by the piece that arrives last,
// with stores and loads past the XCDs' L2s: 28.8 us against 16.2 + 6.2 for one row of 8192 keys, 32 heads of 128 on 8.)
__device__ __forceinline__ size_t kv_record(const KvItem& it, const KvTok& t, int n_heads, int head) {
    const int s = (it.rec & KV_REC_OWN) ? (it.rec & ~KV_REC_OWN) + (t.own_n & 0xFFFF) : it.rec;
    return ((size_t)t.rec + s) * n_heads + head;
}

// Whether a row's sums of weights stand.  A weight's exponent is fma(q.k, scale, -m) with m rounded, so all weights
// share a factor of up to 2^(|m| 2^-24): no more than 2^(1/16) up to the bound, and past any type's range for the largest m.
__device__ __forceinline__ bool kv_fine(float m, float l) {
    return (l == l) & ((fabsf(m) <= 1048576.0f) | (m == -INFINITY));
}
// q.k * scale rounded, as m is: never one operation with the subtraction that follows.
__device__ __forceinline__ float kv_score(float d, float scale) {
#pragma clang fp contract(off)
    return d * scale;
}

// One row over some of an item's keys by one wave in plain f32, for rows
// whose MFMA sums are not finite or whose scores are huge: an infinity times a part that is zero is NaN
// there, and hidden keys carry weight zero rather than being left out.  (A key a wave at a time: hundreds of times slower
// than the MFMAs, for rows that no sound model makes.)  Blocks of `block` numbers every `step`
// from `from` on.  Lane l ends with dims l, l + 64, ...; m and l are every lane's.
template <typename E, int DE>
__device__ __forceinline__ void kv_row_plain(const KvAttnArgs& a, const KvItem& it, const int* table, int h, size_t q_at, int pos,
                                          int from, int block, int step, float& m, float& l, float (&acc)[DE]) {
    const int lane = threadIdx.x & 63, hd = a.pages.hd;
    float qv[DE];
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int e = 0; e < DE; e++) {
        acc[e] = 0.0f;
        qv[e] = lane + 64 * e < hd ? kv_load_q(a.q, a.qdt, q_at + lane + 64 * e) : 0.0f;
    }
    for (int base = from; base < it.j1; base += step) {
        for (int j = base; j < min(it.j1, base + block); j++) {
            const int key = kv_key(it, j);
            if (!kv_sees(key, pos, a.window, a.sinks)) continue;
            const size_t row = (size_t)kv_row(a.pages, table[key >> a.pages.shift], h, key) * hd;
            float d = 0.0f;
#pragma unroll
            for (int e = 0; e < DE; e++)
                if (lane + 64 * e < hd) d += qv[e] * (float)((const E*)a.pages.k)[row + lane + 64 * e];
            const float s = kv_score(wave_sum(d), a.scale), mn = fmaxf(m, s), ref = mn == -INFINITY ? 0.0f : mn;
            const float p = kv_exp2(s - ref), f = kv_exp2(m - ref);
            l = l * f + p;
#pragma unroll
            for (int e = 0; e < DE; e++)
                acc[e] = acc[e] * f + p * (lane + 64 * e < hd ? (float)((const E*)a.pages.v)[row + lane + 64 * e] : 0.0f);
            m = mn;
            if (l != l) return;  // a NaN among the weights: the row's sums are NaN for good
        }
    }
}

}  // namespace th
