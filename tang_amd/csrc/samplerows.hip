// The choice of a token for each row of logits (th_sample_rows).
//
// With M the largest logit, w_i = 2^((l_i - M) log2(e) / T).  Kept are: top-k, the
// logits from the k-th largest on; top-p, the shortest run of those in
// descending order (equal ones: the lower index first) whose weights reach p of
// theirs all; min-p, weights from min_p on.  The token is the first, by index,
// at which the running sum of kept weights exceeds u times their whole sum.
//
// A token hangs on which side of a border u falls, so the borders have to be
// right far beyond f32: weights are formed in f64 and held as integers, w 2^S to
// the nearest (S = 62 - log2(vocab), at most 51; weights below 2^-(S+1) are none), which moves a
// border by vocab 2^-(S+1) of the largest weight at most (2^-33 at 32000, 2^-23 at 2^20).  Their
// sums have no rounding, so histograms with atomics, sums by wave and by row
// agree to the bit in any order, and replays repeat.
#include <algorithm>

#include "ops.hpp"
#include "samplerows.hpp"

namespace th {

constexpr int SNT = 1024, SBINS = 2048, SLIST = 64, SCAP = 4096, SBITS = 5, STABLE = 1 << SBITS;
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef unsigned long long u64_t;

struct SampleLds {
    u64_t sum[SBINS];
    uint32_t count[SBINS];
    double table[STABLE];  // 2^(S + i / STABLE), its high word less i << 10
    u64_t list_w[SLIST];
    uint32_t list_key[SLIST];
    u64_t wave[SNT / 64], wave2[SNT / 64], part[SNT / 64];
    u64_t above, eq, end;
    uint32_t bin, key, n, lo, hi, found;
    u64_t list[SCAP];  // order_entry's of candidates
};

// One workgroup's; the kernel and the path for many candidates share it.
static __shared__ SampleLds s;

__device__ __forceinline__ u64_t shfl_up64(u64_t v, int d) {
    const uint32_t lo = (uint32_t)__shfl_up((int)(uint32_t)v, d, 64), hi = (uint32_t)__shfl_up((int)(v >> 32), d, 64);
    return (u64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
__device__ __forceinline__ float uniform(float v) { return __uint_as_float(uniform(__float_as_uint(v))); }
__device__ __forceinline__ u64_t shfl_64(u64_t v, int from) {
    const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)v, from, 64), hi = (uint32_t)__shfl((int)(v >> 32), from, 64);
    return (u64_t)hi << 32 | lo;
}
__device__ __forceinline__ u64_t wave_scan(u64_t v, int lane) {  // inclusive
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const u64_t t = shfl_up64(v, o);
        if (lane >= o) v += t;
    }
    return v;
}
__device__ __forceinline__ u64_t wave_total(u64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        v += (u64_t)(uint32_t)__shfl_xor((int)(v >> 32), o, 64) << 32 | (uint32_t)__shfl_xor((int)(uint32_t)v, o, 64);
    return v;
}

// Order of f32 values as unsigned integers.
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);  // (-0 as +0)
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// A row's logits.  A wave has a sixteenth of them, as they lie, and of its block j
// a lane has eight, so that sums by wave are sums of runs of indexes.  A pass
// streams them, two blocks ahead (later passes from the caches).  Rows held in
// registers were slower by half: every pass is unrolled then, and 32 logits a thread no longer fit the instruction cache.
template <typename X>
struct SampleRow {
    typedef X x8_t __attribute__((ext_vector_type(8), aligned(sizeof(X))));
    typedef X r8_t __attribute__((ext_vector_type(8)));
    const X* x;
    int V, blocks, start;  // start: of the wave
    bool infinite;  // the largest is +inf: such logits count as 0 and all others as -inf

    __device__ __forceinline__ SampleRow(const X* at, int n, bool inf)
        : x(at), V(n), blocks((n + SNT * 8 - 1) / (SNT * 8)), start((int)uniform(threadIdx.x >> 6) * blocks * 512), infinite(inf) {}
    // Eight a lane from index `at` of the wave on, -inf from `end` on (at most V).  All branches are the whole wave's:
    // where lanes took ways of their own at the end of a row and registers were short, the compiler copied
    // some before all lanes were back, and the others lost what was in them.
    __device__ __forceinline__ r8_t read_at(int at, int end) const {
        const int i = at + ((int)threadIdx.x & 63) * 8;
        r8_t r;
        if (at + 512 <= end) {
            r = *(const x8_t*)(x + i);
        } else if (at < end) {
#pragma unroll
            for (int e = 0; e < 8; e++) r[e] = x[min(i + e, V - 1)];
#pragma unroll
            for (int e = 0; e < 8; e++) r[e] = i + e < end ? r[e] : (X)-INFINITY;
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) r[e] = (X)-INFINITY;
        }
        return r;
    }
    __device__ __forceinline__ float value(float l) const { return !infinite ? l : l == INFINITY ? 0.0f : -INFINITY; }
    __device__ __forceinline__ void values(const r8_t& r, float (&v)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = (float)r[e];
        if (infinite) {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = value(v[e]);
        }
    }
    // f(index of the first, the eight values); what lies behind the row holds -inf
    template <typename F>
    __device__ __forceinline__ void blocks_of(F&& f) const {
        auto read = [&](int j) { return read_at(start + j * 512, j < blocks ? V : 0); };
        r8_t a = read(0), b = read(1);
#pragma unroll 1
        for (int j = 0; j < blocks; j++) {
            const r8_t now = a;
            a = b;
            b = read(j + 2);
            float v[8];
            values(now, v);
            f(start + j * 512 + ((int)threadIdx.x & 63) * 8, v);
        }
    }
    __device__ __forceinline__ int passed() const { return blocks * 8; }  // logits of a lane in a pass, with those behind the end
    template <typename F>
    __device__ __forceinline__ void each(F&& f) const {
        blocks_of([&](int i, const float (&v)[8]) {
#pragma unroll
            for (int e = 0; e < 8; e++) f(i + e, v[e]);
        });
    }
};

// Weights of a row.
struct SampleWeights {
    float M, cb, bins;  // cb: bins a unit of a logit; how many there are
    double Md, c, least;  // c: log2(e) / T in steps of the table
    int S;
    const double* table;

    // Bins that a logit is below the largest, in f32: monotone in l.  Bins have equal widths in the logarithm
    // of the weight; behind the last (NaN, too) a weight is below 2^-(S+1).
    __device__ __forceinline__ float below(float l) const { return (M - l) * cb; }
    __device__ __forceinline__ bool alive(float l) const { return below(l) < bins; }
    __device__ __forceinline__ int bin_of(float l) const { return (int)min(below(l), (float)(SBINS - 1)); }
    // w 2^S to the nearest, as the bits of 2^52 + w 2^S.  With x = n + i/32 + r the table has 2^(i/32), and
    // 2^r is its series to the fifth power (r up to 2^-6: off by 2^-48).  All rows' elements pass through here,
    // and as instructions are what the passes are bound by, there is no branch: a logit that has no weight, NaN
    // too, is lifted to 2^-(S+2), which rounds to none (256 rows of 131072 without a filter: 44 us,
    // 61 with such branches and 64 entries; 1024 entries and two terms less: 52, as lanes then meet in the banks).
    __device__ __forceinline__ u64_t bits(float l) const {
        const double big = 0x1.8p52, x = fmax(((double)l - Md) * c, least), y = x + big;
        const uint32_t k = (uint32_t)(u64_t)__double_as_longlong(y);
        const double r = x - (y - big);
        constexpr double h = 1.0 / STABLE;
        double p = __builtin_fma(r, 1.3333558146428443e-3 * h * h * h * h * h, 9.618129107628477e-3 * h * h * h * h);  // ln(2)^n / n!
        p = __builtin_fma(p, r, 5.550410866482158e-2 * h * h * h);
        p = __builtin_fma(p, r, 2.402265069591007e-1 * h * h);
        p = __builtin_fma(p, r, 6.931471805599453e-1 * h);
        p = __builtin_fma(p, r, 1.0);
        u32x2_t m = __builtin_bit_cast(u32x2_t, table[k & (STABLE - 1)]);
        m.y += k << (20 - SBITS);  // (the table's index is in both: it cancels)
        return __builtin_bit_cast(u64_t, __builtin_fma(__builtin_bit_cast(double, m), p, 0x1p52));
    }
    static constexpr u64_t NONE = (u64_t)0x43300000 << 32;  // the bits of 2^52
    __device__ __forceinline__ u64_t weight(float l) const { return bits(l) - NONE; }
};

// The first of SBINS bins at which the running sum reaches target (1 to the sum of all): in s.bin, what lies
// before it in s.above.  Returns the sum of all.  Call with the whole block, after a barrier; ends with one.
template <typename T>
__device__ __forceinline__ u64_t total_of(const T* hist, u64_t& mine, u64_t& before) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    mine = (u64_t)hist[2 * tid] + hist[2 * tid + 1];
    const u64_t incl = wave_scan(mine, lane);
    if (lane == 63) s.wave[wave] = incl;
    __syncthreads();
    u64_t all = 0, prev = 0;
#pragma unroll
    for (int w = 0; w < SNT / 64; w++) {
        if (w == wave) prev = all;
        all += s.wave[w];
    }
    before = prev + incl - mine;
    return all;
}
template <typename T>
__device__ __forceinline__ void find_bin(const T* hist, u64_t mine, u64_t before, u64_t target) {
    if (before < target && target <= before + mine) {
        const u64_t a = hist[2 * threadIdx.x];
        const bool second = before + a < target;
        s.bin = 2 * threadIdx.x + second;
        s.above = before + (second ? a : 0);
    }
    __syncthreads();
}

__device__ __forceinline__ void clear_bins(bool sums, bool counts) {
    const int tid = threadIdx.x;
    if (sums) s.sum[2 * tid] = s.sum[2 * tid + 1] = 0;
    if (counts) s.count[2 * tid] = s.count[2 * tid + 1] = 0;
}

// Among the elements for which in(l, key) holds, the key at which the running
// sum of their counts (or weights) in descending order reaches target: in s.key, with what
// lies above it in s.above and the sum of the elements that have it in s.eq (0: not known).  Up
// to 64 of them are ranked by one wave; more are sorted into bins by key, until
// one bin has no more, or one key alone.
template <bool WEIGHTS, typename Row, typename In>
__device__ __forceinline__ void select_key(const Row& row, const SampleWeights& sw, u64_t target, In&& in) {
    const int tid = threadIdx.x;
    uint32_t lo = 0, hi = 0xFFFFFFFFu;
    u64_t above = 0;
    for (;;) {
        if (tid == 0) {
            s.n = 0;
            s.lo = 0xFFFFFFFFu;
            s.hi = 0;
        }
        __syncthreads();
        uint32_t least = 0xFFFFFFFFu, most = 0;
        row.each([&](int, float l) {
            const uint32_t key = order_key(l);
            if (key < lo || key > hi || !in(l, key)) return;
            least = min(least, key);
            most = max(most, key);
            const uint32_t at = atomicAdd(&s.n, 1u);
            if (at < SLIST) {
                s.list_key[at] = key;
                s.list_w[at] = WEIGHTS ? sw.weight(l) : 1;
            }
        });
        if (least <= most) {
            atomicMin(&s.lo, least);
            atomicMax(&s.hi, most);
        }
        __syncthreads();
        const uint32_t n = s.n;
        lo = s.lo;
        hi = s.hi;
        if (lo >= hi) {  // one key
            if (tid == 0) {
                s.key = lo;
                s.above = above;
                s.eq = 0;
            }
            break;
        }
        if (n <= SLIST) {
            if (tid < (int)n) {
                const uint32_t key = s.list_key[tid];
                u64_t over = above, eq = 0;
                for (uint32_t i = 0; i < n; i++) {
                    const uint32_t k = s.list_key[i];
                    const u64_t w = s.list_w[i];
                    over += k > key ? w : 0;
                    eq += k == key ? w : 0;
                }
                if (over < target && target <= over + eq) {
                    s.key = key;
                    s.above = over;
                    s.eq = eq;
                }
            }
            break;
        }
        clear_bins(WEIGHTS, !WEIGHTS);
        const int shift = max(0, 21 - __builtin_clz(hi - lo));  // (hi - lo) >> shift is below 2048
        __syncthreads();
        row.each([&](int, float l) {
            const uint32_t key = order_key(l);
            if (key < lo || key > hi || !in(l, key)) return;
            if (WEIGHTS) atomicAdd(&s.sum[(hi - key) >> shift], sw.weight(l));
            else atomicAdd(&s.count[(hi - key) >> shift], 1u);
        });
        __syncthreads();
        u64_t mine, before;
        if (WEIGHTS) {
            (void)total_of(s.sum, mine, before);
            find_bin(s.sum, mine, before, target - above);
        } else {
            (void)total_of(s.count, mine, before);
            find_bin(s.count, mine, before, target - above);
        }
        const uint32_t bin = s.bin, first = bin << shift;
        above += s.above;
        lo = hi - lo - first < (1u << shift) ? lo : hi - first - ((1u << shift) - 1);
        hi -= first;
        __syncthreads();
    }
    __syncthreads();
}

// Sums of what the waves have in v: the sum of all, and what lies before each wave's.
__device__ __forceinline__ u64_t over_waves(u64_t v, u64_t* room, u64_t& before) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane == 0) room[wave] = v;
    __syncthreads();
    u64_t all = 0;
#pragma unroll
    for (int w = 0; w < SNT / 64; w++) {
        if (w == wave) before = all;
        all += room[w];
    }
    return all;
}

// The index at which the running sum, by index, of f(logits from an index on) reaches target, where s.part has the waves' sums: in s.found.
template <typename Row, typename F>
__device__ __forceinline__ void pick(const Row& row, u64_t target, F&& f) {
    const int tid = threadIdx.x, lane = tid & 63;
    int w = 0;
    u64_t before = 0;
    while (w < SNT / 64 - 1 && before + s.part[w] < target) before += s.part[w++];
    u64_t rest = target - before;
    // the wave's logits, by the whole block
    const int first = (int)uniform((uint32_t)w) * row.blocks * 512, end = min(row.V, first + row.blocks * 512), wave = (int)uniform((uint32_t)tid >> 6);
    for (int at = first; at < end; at += SNT * 8) {
        const int i = at + tid * 8;
        float v[8];
        row.values(row.read_at(at + wave * 512, end), v);
        u64_t mine = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) mine += f(i + e, v[e]);
        const u64_t incl = wave_scan(mine, lane);
        u64_t upto;
        __syncthreads();  // (the last round has read s.wave)
        const u64_t all = over_waves(shfl_64(incl, 63), s.wave, upto);
        upto += incl - mine;
        if (upto < rest && rest <= upto + mine) {
            bool done = false;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                upto += f(i + e, v[e]);
                if (!done && upto >= rest) {
                    s.found = (uint32_t)(i + e);
                    done = true;
                }
            }
        }
        if (rest <= all) break;
        rest -= all;
    }
    __syncthreads();
}

// The index at which the running sum, by index, of f(index, logit) reaches target(sum of all): in s.found, or not at all
// if the sum is 0.  Returns the sum.  f's sums are over a wave's logits, `extra` for each that passes (see NONE).
template <typename Row, typename F, typename T>
__device__ __forceinline__ u64_t find_index(const Row& row, u64_t extra, F&& f, T&& target_of) {
    u64_t t = 0, before;
    row.each([&](int i, float l) { t += f(i, l); });
    t -= extra * (u64_t)row.passed();
    __syncthreads();
    const u64_t all = over_waves(wave_total(t), s.part, before);
    if (all == 0) {
        __syncthreads();
        return 0;
    }
    pick(row, target_of(all), [&](int i, float l) { return f(i, l) - extra; });
    return all;
}

// Descending logits and, among equal ones, ascending indexes, as ascending integers.
__device__ __forceinline__ u64_t order_entry(uint32_t key, uint32_t index) { return (u64_t)~key << 32 | index; }
__device__ __forceinline__ float key_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key); }

// Of eight logits from index i on, those that are `in`, to the list.  (Asked for eight at a time: few blocks have any.)
__device__ __forceinline__ void list_some(int i, const float (&v)[8], const bool (&in)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e++)
        if (in[e]) {
            const uint32_t at = atomicAdd(&s.n, 1u);
            if (at < SCAP) s.list[at] = order_entry(order_key(v[e]), (uint32_t)(i + e));
        }
}

__device__ __forceinline__ u64_t shfl_xor64(u64_t v, int d) {
    return (u64_t)(uint32_t)__shfl_xor((int)(v >> 32), d, 64) << 32 | (uint32_t)__shfl_xor((int)(uint32_t)v, d, 64);
}

// s.list[0, n), n a power of two from 2 on, in ascending order (all different, but for ones behind the end).  Up to 128
// by counting: the lanes of an entry count those below it.  More pass a bitonic network, up to 1024 with an
// entry a thread, where only what passes between waves goes through shared memory (1024 entries: 9 us, 13 us with every step there).
__device__ __forceinline__ void sort_list(int n) {
    const int tid = threadIdx.x;
    if (n > SNT) {
        for (int size = 2; size <= n; size *= 2)
            for (int d = size / 2; d > 0; d /= 2) {
                __syncthreads();
                for (int i = tid; i < n / 2; i += SNT) {
                    const int lo = 2 * i - (i & (d - 1)), hi = lo + d;
                    const u64_t a = s.list[lo], b = s.list[hi];
                    if ((a > b) == ((lo & size) == 0)) {
                        s.list[lo] = b;
                        s.list[hi] = a;
                    }
                }
            }
        __syncthreads();
        return;
    }
    if (n > 128) {
        __syncthreads();
        u64_t v = tid < n ? s.list[tid] : ~(u64_t)0;
        int at = SNT;  // two places in turn
        for (int size = 2; size <= n; size *= 2)
            for (int d = size / 2; d > 0; d /= 2) {
                u64_t o;
                if (d >= 64) {
                    s.list[at + tid] = v;
                    __syncthreads();
                    o = s.list[at + (tid ^ d)];
                    at = 3 * SNT - at;
                } else {
                    o = shfl_xor64(v, d);
                }
                const bool least = ((tid & d) == 0) == ((tid & size) == 0);
                v = (o < v) == least ? o : v;
            }
        s.list[tid] = v;
        __syncthreads();
        return;
    }
    __syncthreads();
    const int g = min(64, SNT / n), e = tid / g, part = tid % g, len = (n + g - 1) / g;  // (2 entries: 128 threads are enough)
    const bool mine = e < n;
    const u64_t v = mine ? s.list[e] : 0;
    int below = 0;
    if (mine)
        for (int i = 0; i < len; i++) {
            const int at = part * len + i;
            if (at < n) below += s.list[at] < v || (s.list[at] == v && at < e);
        }
    for (int o = 1; o < g; o *= 2) below += __shfl_xor(below, o, 64);
    __syncthreads();
    if (mine && part == 0) s.list[below] = v;
    __syncthreads();
}

// Sums of what is in front of each thread's four entries of a list, and of all (f(entry's place)).
template <typename F>
__device__ __forceinline__ u64_t scan_list(int n, u64_t (&w)[4], u64_t& before, F&& f) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    u64_t mine = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        w[e] = 4 * tid + e < n ? f(4 * tid + e) : 0;
        mine += w[e];
    }
    const u64_t incl = wave_scan(mine, lane);
    if (lane == 63) s.wave[wave] = incl;
    __syncthreads();
    u64_t all = 0, prev = 0;
#pragma unroll
    for (int v = 0; v < SNT / 64; v++) {
        if (v == wave) prev = all;
        all += s.wave[v];
    }
    __syncthreads();
    before = prev + incl - mine;
    return all;
}

// The running sum that the token's is the first to reach.
__device__ __forceinline__ u64_t drawn(float u, u64_t sum) {
    const double t = (double)u * (double)sum;
    return t >= (double)sum ? sum : t >= 0.0 ? min((u64_t)t, sum - 1) + 1 : (u64_t)1;
}
__device__ __forceinline__ u64_t run_of(float p, u64_t all) {  // that top-p's run reaches
    return p > 0.0f ? max((u64_t)1, min(all, (u64_t)ceil((double)p * (double)all))) : 1;
}

// A row with more candidates than a list holds: thresholds by refined histograms, then the sum over the row.  The
// token goes to s.found, the sum to s.above.  Up to some ten passes, each bound by one CU's vector instructions (48 rows of 50001 normal
// logits: top-k 8000 74 us, and top-p 0.9 of those 122; all logits in one bin 184 and 293, top-p alone 227, where lists take 40).
template <typename X>
__device__ __noinline__ void sample_many(const X* x, int V, bool infinite, SampleWeights sw, uint32_t k, bool by_k, float p, bool by_p, u64_t least_w, float u) {
    const int tid = threadIdx.x, lane = tid & 63;
    // scalars come to a function in vector registers
    const u64_t at = (u64_t)x;
    const SampleRow<X> row((const X*)((u64_t)uniform((uint32_t)(at >> 32)) << 32 | uniform((uint32_t)at)), (int)uniform((uint32_t)V), uniform((uint32_t)infinite));
    uint32_t key = 0, last = 0xFFFFFFFFu;  // kept: keys above `key`, and that one up to index `last`
    if (by_k || by_p) {
        clear_bins(by_p, by_k);
        __syncthreads();
        row.each([&](int, float l) {
            if (!sw.alive(l)) return;
            const int b = sw.bin_of(l);
            if (by_k) atomicAdd(&s.count[b], 1u);
            if (by_p) atomicAdd(&s.sum[b], sw.weight(l));
        });
        __syncthreads();
        u64_t mine, before, kept = 0;
        uint32_t kbin = SBINS;
        if (by_k) {
            const u64_t n = total_of(s.count, mine, before);
            if (n > k) {  // (otherwise all that have a weight are kept)
                find_bin(s.count, mine, before, k);
                kbin = s.bin;
                const u64_t rest = k - s.above;
                __syncthreads();
                // the sums are needed again: they move to registers while keys are sorted
                const u64_t s0 = s.sum[2 * tid], s1 = s.sum[2 * tid + 1];
                select_key<false>(row, sw, rest, [&](float l, uint32_t) { return sw.alive(l) && sw.bin_of(l) == (int)kbin; });
                key = s.key;
                if (by_p) {
                    s.sum[2 * tid] = s0;
                    s.sum[2 * tid + 1] = s1;
                    u64_t part = 0;
                    row.each([&](int, float l) {
                        if (sw.alive(l) && sw.bin_of(l) == (int)kbin && order_key(l) >= key) part += sw.weight(l);
                    });
                    part = wave_total(part);
                    __syncthreads();
                    if (tid == 0) s.sum[kbin] = 0;
                    __syncthreads();
                    if (lane == 0 && part) atomicAdd(&s.sum[kbin], part);
                    if ((uint32_t)(2 * tid) > kbin) s.sum[2 * tid] = 0;
                    if ((uint32_t)(2 * tid + 1) > kbin) s.sum[2 * tid + 1] = 0;
                }
                __syncthreads();
            } else {
                __syncthreads();
            }
        }
        if (by_p) {
            kept = total_of(s.sum, mine, before);
            const u64_t want = run_of(p, kept);
            find_bin(s.sum, mine, before, want);
            const int pbin = (int)s.bin;
            const u64_t rest = want - s.above;
            __syncthreads();
            const uint32_t least = key;
            select_key<true>(row, sw, rest, [&](float l, uint32_t kk) { return sw.alive(l) && sw.bin_of(l) == pbin && kk >= least; });
            key = s.key;
            const u64_t w = sw.weight(key_value(key)), ties = (rest - s.above + w - 1) / w;  // so many of the equal ones are kept
            const bool some = s.eq != ties * w;
            __syncthreads();
            if (some) {
                find_index(row, 0, [&](int, float l) { return (u64_t)(order_key(l) == key); }, [&](u64_t) { return ties; });
                last = s.found;
                __syncthreads();
            }
        }
    }
    const u64_t all = find_index(
        row, 0,
        [&](int i, float l) -> u64_t {
            const uint32_t kk = order_key(l);
            if (kk < key || (kk == key && (uint32_t)i > last) || !sw.alive(l)) return 0;
            const u64_t w = sw.weight(l);
            return w >= least_w ? w : 0;
        },
        [&](u64_t sum) { return drawn(u, sum); });
    if (tid == 0) s.above = all;
    __syncthreads();
}

// Top-p without top-k.  The token goes to s.found, the sum to s.above; false: too many to list.  (Inlined: as a
// function it saves 48 registers a lane, and 256 rows of 32000 take 46 us, not 34.)
template <typename X>
__device__ __forceinline__ bool sample_run(const SampleRow<X>& row, const SampleWeights& sw, float p, u64_t least, float u) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // Runs of any length: f32 sums of the weights find the bin where the run
    // ends, and one pass with the weights themselves sums up what lies
    // before it (for the whole row, and for the draw by wave) and lists that bin.
    clear_bins(true, false);
    __syncthreads();
    const int per_bit = SBINS / (sw.S + 1);
    const float a_bin = 1.0f / (float)per_bit;
    row.each([&](int, float l) {  // each bin in units of its own, 2^-31 of the power of two above its weights
        const float b = sw.below(l);
        if (b < sw.bins) atomicAdd(&s.sum[(int)b], (u64_t)(uint32_t)__builtin_amdgcn_exp2f(31.0f - __builtin_amdgcn_fractf(b * a_bin)));
    });
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; i++) s.sum[2 * tid + i] = s.sum[2 * tid + i] << 11 >> (2 * tid + i) / per_bit;  // in 2^-42 of the largest weight
    __syncthreads();
    u64_t mine, before;
    // Up to a bin, these sums are off by 2^-18 of the sum of all (roundings of b shift the weights by up to 2^-22 of the bits that they
    // are below the largest, which is less than log2(vocab) on average, and most of that is the same for all), and by less than 1 a
    // bin that is cut off.  Were it more, the exact sums below would tell, and the row go to sample_many.
    const u64_t about = total_of(s.sum, mine, before), want_about = run_of(p, about), off = (about >> 18) + 2 * SBINS;
    find_bin(s.sum, mine, before, want_about > off ? want_about - off : 1);
    const float first = (float)uniform(s.bin);
    __syncthreads();
    find_bin(s.sum, mine, before, min(want_about + off, about));
    const float past = (float)(uniform(s.bin) + 1);
    __syncthreads();
    if (tid == 0) s.n = 0;
    __syncthreads();
    u64_t all = 0, sure = 0, part = 0;
    auto pass = [&](auto by_least) {
        row.blocks_of([&](int i, const float (&v)[8]) {
            bool in[8], any = false;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const u64_t w = sw.bits(v[e]);
                const float b = sw.below(v[e]);
                all += w;
                const u64_t before_it = b < first ? w : SampleWeights::NONE;
                sure += before_it;
                if (by_least) part += before_it >= least + SampleWeights::NONE ? before_it : SampleWeights::NONE;
                in[e] = b >= first && b < past;
                any |= in[e];
            }
            if (any) list_some(i, v, in);
        });
    };
    if (uniform((uint32_t)(least > 1))) pass(std::true_type{});
    else pass(std::false_type{});
    const u64_t none = SampleWeights::NONE * (u64_t)row.passed();
    all -= none;
    sure -= none;
    part = least > 1 ? part - none : sure;
    part = wave_total(part);
    if (lane == 0) s.part[wave] = part;
    all = over_waves(wave_total(all), s.wave, before);
    sure = over_waves(wave_total(sure), s.wave2, before);
    const int n = (int)uniform(s.n);
    const u64_t want = run_of(p, all);
    __syncthreads();
    if (n <= SCAP && sure < want) {
        int room = 2;
        while (room < n) room *= 2;
        for (int i = n + tid; i < room; i += SNT) s.list[i] = ~(u64_t)0;
        sort_list(room);
        u64_t w[4];
        const u64_t listed = scan_list(n, w, before, [&](int i) { return sw.weight(key_value(~(uint32_t)(s.list[i] >> 32))); });
        if (want <= sure + listed) {
            u64_t run = sure + before;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (w[e] && run < want) {
                    const u64_t v = s.list[4 * tid + e];
                    if (w[e] >= least) atomicAdd(&s.part[((uint32_t)v >> 9) / (uint32_t)row.blocks], w[e]);
                    if (run + w[e] >= want) s.end = v;
                }
                run += w[e];
            }
            __syncthreads();
            const u64_t end = s.end;
            u64_t sum = 0;
#pragma unroll
            for (int v = 0; v < SNT / 64; v++) sum += s.part[v];
            pick(row, drawn(u, sum), [&](int i, float l) -> u64_t {
                const float b = sw.below(l);
                if (!(b < past) || (b >= first && order_entry(order_key(l), (uint32_t)i) > end)) return 0;
                const u64_t w = sw.weight(l);
                return w >= least ? w : 0;
            });
            if (tid == 0) s.above = sum;
            __syncthreads();
            return true;
        }
    }
    return false;
}

template <typename X>
__global__ __launch_bounds__(SNT) void sample_rows_kernel(SampleArgs a, int S) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = blockIdx.x;
    const X* const x = (const X*)a.x + (size_t)r * a.vocab;
    const float T = uniform(a.temp ? a.temp[r] : 1.0f);
    // the largest (NaN is none); greedy: and where it is first
    float M = -INFINITY;
    uint32_t first_of = 0;
    const bool greedy = !(T > 0.0f);
    if (!greedy && tid >= SNT - STABLE) {  // (the last wave has the least of a row)
        const int i = tid - (SNT - STABLE);
        s.table[i] = __longlong_as_double(__double_as_longlong(exp2(i / (double)STABLE)) + ((long long)S << 52) - ((long long)i << (52 - SBITS)));
    }
    {
        const SampleRow<X> raw(x, a.vocab, false);
        if (greedy) raw.each([&](int i, float l) {
            first_of = l > M ? (uint32_t)i : first_of;
            M = l > M ? l : M;
        });
        else raw.each([&](int, float l) { M = fmaxf(M, l); });
    }
    const float mine_M = M;
    M = wave_max(M);
    if (lane == 0) s.wave[wave] = __float_as_uint(M);
    if (tid == 0) {
        s.found = greedy ? 0xFFFFFFFFu : 0;  // (otherwise always places in the row and in the bins)
        s.bin = 0;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SNT / 64; w++) M = fmaxf(M, __uint_as_float((uint32_t)s.wave[w]));
    M = uniform(M);
    if (greedy || M == -INFINITY) {  // (no logit at all: token 0)
        if (M != -INFINITY && mine_M == M) atomicMin(&s.found, first_of);
        __syncthreads();
        if (tid == 0) {
            a.token[r] = M == -INFINITY ? 0 : s.found;
            if (a.prob) a.prob[r] = M == -INFINITY ? 0.0f : 1.0f;
        }
        return;
    }
    __syncthreads();
    const bool infinite = M == INFINITY;
    const SampleRow<X> row(x, a.vocab, infinite);
    SampleWeights sw;
    const double c = 1.44269504088896340736 / (double)T;
    sw.M = infinite ? 0.0f : M;
    sw.Md = sw.M;
    sw.c = c * STABLE;
    sw.least = -(double)(S + 2) * STABLE;
    const float per_bit = (float)(SBINS / (S + 1));  // (whole: a bin's weights are between two powers of two)
    sw.bins = per_bit * (float)(S + 1);
    sw.cb = (float)min(c * per_bit, 0x1p127);  // (finite: 0 times it has to be 0)
    sw.S = S;
    sw.table = s.table;
    const uint32_t k = uniform(a.top_k ? a.top_k[r] : 0u);
    const float p = uniform(a.top_p ? a.top_p[r] : 1.0f), low = uniform(a.min_p ? a.min_p[r] : 0.0f);
    const bool by_k = k > 0 && k < (uint32_t)a.vocab, by_p = p < 1.0f;
    const float u = a.u[r];
    const u64_t least = low > 0.0f ? (u64_t)ceil((double)min(low, 1.0f) * (double)((u64_t)1 << S)) : 1;
    auto answer = [&](uint32_t index, float l, u64_t all) {
        a.token[r] = index;
        if (a.prob) a.prob[r] = (float)(exp2(l == sw.M ? 0.0 : ((double)l - sw.Md) * c) * (double)((u64_t)1 << S) / (double)all);
    };
    bool many = true;
    if (by_p && !by_k) {
        many = !sample_run(row, sw, p, least, u);
    } else if (by_k || low > 0.0f) {
        // Few candidates are the usual case: they are listed and sorted.
        float edge = sw.bins;  // behind the last bin that can hold a kept one
        u64_t want = 0;
        bool cut = false;  // by k
        if (by_k) {
            clear_bins(false, true);
            __syncthreads();
            row.each([&](int, float l) {
                const float b = sw.below(l);
                if (b < sw.bins) atomicAdd(&s.count[(int)b], 1u);
            });
            __syncthreads();
            u64_t mine, before;
            cut = total_of(s.count, mine, before) > k;  // (otherwise all that have a weight are kept)
            if (cut) {
                find_bin(s.count, mine, before, k);
                edge = (float)(uniform(s.bin) + 1);
            }
        }
        if (low > 0.0f && !by_p) edge = min(edge, per_bit * (0.01f - log2f(min(low, 1.0f))) + 1.0f);
        if (tid == 0) s.n = 0;
        __syncthreads();
        row.blocks_of([&](int i, const float (&v)[8]) {
            bool in[8], any = false;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                in[e] = sw.below(v[e]) < edge;
                any |= in[e];
            }
            if (any) list_some(i, v, in);
        });
        __syncthreads();
        const int n = (int)uniform(s.n);
        if (n <= SCAP) {
            int room = 2;
            while (room < n) room *= 2;
            for (int i = n + tid; i < room; i += SNT) s.list[i] = ~(u64_t)0;
            sort_list(room);
            // (where min-p's edge came first, all that are listed are among the k)
            const uint32_t kth = cut && k <= (uint32_t)n ? (uint32_t)(s.list[k - 1] >> 32) : 0xFFFFFFFFu;
            u64_t w[4], before;
            u64_t all = scan_list(n, w, before, [&](int i) -> u64_t {
                const uint32_t inverse = (uint32_t)(s.list[i] >> 32);
                return inverse <= kth ? sw.weight(key_value(~inverse)) : 0;
            });
            if (by_p) want = run_of(p, all);
            // kept: up to where the sum reaches `want`, and weights from `least` on
            all = 0;
            u64_t kept_w[4], kept_before;
            u64_t run = before;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                kept_w[e] = w[e] >= least && (!by_p || run < want) ? w[e] : 0;
                run += w[e];
            }
            // in the order of indexes: what is not kept goes behind
            u64_t mine4[4];
#pragma unroll
            for (int e = 0; e < 4; e++) mine4[e] = 4 * tid + e < n ? s.list[4 * tid + e] : 0;
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (4 * tid + e < n)
                    s.list[4 * tid + e] = kept_w[e] ? (mine4[e] & 0xFFFFFFFFu) << 32 | (uint32_t)(mine4[e] >> 32) : ~(u64_t)0;
            sort_list(room);
            all = scan_list(n, w, kept_before, [&](int i) -> u64_t {
                const u64_t v = s.list[i];
                return v == ~(u64_t)0 ? 0 : sw.weight(key_value(~(uint32_t)v));
            });
            const u64_t target = drawn(u, all);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (kept_before < target && target <= kept_before + w[e]) {
                    const u64_t v = s.list[4 * tid + e];
                    answer((uint32_t)(v >> 32), key_value(~(uint32_t)v), all);
                }
                kept_before += w[e];
            }
            return;
        }
    }
    if ((by_p && !by_k) ? many : (by_k || low > 0.0f)) {
        sample_many<X>(x, a.vocab, infinite, sw, k, by_k, p, by_p, least, u);
    } else if (!(by_p && !by_k)) {
        const u64_t all = find_index(row, SampleWeights::NONE, [&](int, float l) { return sw.bits(l); }, [&](u64_t sum) { return drawn(u, sum); });
        if (tid == 0) s.above = all;
        __syncthreads();
    }
    if (tid == 0) answer(s.found, row.value((float)x[s.found]), s.above);
}

void launch_sample_rows(const SampleArgs& all, hipStream_t s) {
    constexpr int ROWS = 1 << 21;  // a launch has below 2^32 threads
    if (all.rows == 0) return;
    SampleArgs a = all;
    if (all.rows > ROWS) {
        a.rows = ROWS;
        launch_sample_rows(a, s);
        a.rows = all.rows - ROWS;
        a.x = (const char*)all.x + (size_t)ROWS * all.vocab * dtype_size(all.xdt);
        for (const float** v : {&a.u, &a.temp, &a.top_p, &a.min_p})
            if (*v) *v += ROWS;
        if (a.top_k) a.top_k += ROWS;
        a.token += ROWS;
        if (a.prob) a.prob += ROWS;
        return launch_sample_rows(a, s);
    }
    int bits = 0;
    while (((size_t)1 << bits) < (size_t)a.vocab) bits++;
    const int S = std::min(51, 62 - bits);
    auto types = [&](auto x) {
        TH_LAUNCH((sample_rows_kernel<decltype(x)>), dim3((unsigned)a.rows), dim3(SNT), 0, s, a, S);
    };
    if (a.xdt == TH_F32) types(float{});
    else if (a.xdt == TH_F16) types((_Float16)0);
    else types((__bf16)0.0f);
    TH_LAUNCH_CHECK();
}

}  // namespace th
