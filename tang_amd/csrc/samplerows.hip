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
// the nearest (S = 62 - log2(vocab), at most 51; weights below 2^-(S+1) are none).  Their
// sums have no rounding, so histograms with atomics, sums by wave and by row
// agree to the bit in any order, and replays repeat.
#include <algorithm>

#include "ops.hpp"
#include "samplerows.hpp"

namespace th {

constexpr int SNT = 1024, SBINS = 2048, SLIST = 64, SCAP = 4096;
typedef unsigned long long u64_t;

struct SampleLds {
    u64_t sum[SBINS];
    uint32_t count[SBINS];
    double table[64];  // 2^(i / 64)
    u64_t list_w[SLIST];
    uint32_t list_key[SLIST];
    u64_t wave[SNT / 64], wave2[SNT / 64];
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

// Order of f32 values as unsigned integers (a -0 is made +0 before).
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// A row's logits: thread t has elements (j 1024 + t) 8 + e of block j.  A pass
// streams them, two blocks at a time and two ahead (later passes from the
// caches).  Rows held in registers were slower: every pass is unrolled then, and 32 logits
// a thread no longer fit the instruction cache (32000 logits, no filter: 28 against 18.5 us).
template <typename X>
struct SampleRow {
    typedef X x8_t __attribute__((ext_vector_type(8), aligned(sizeof(X))));
    typedef X r8_t __attribute__((ext_vector_type(8)));
    const X* x;
    int V, blocks;

    __device__ __forceinline__ r8_t read(int j) const {
        const int i = (j * SNT + (int)threadIdx.x) * 8;
        if (i + 8 <= V) return *(const x8_t*)(x + i);
        r8_t r;
#pragma unroll
        for (int e = 0; e < 8; e++) r[e] = i + e < V ? x[i + e] : (X)-INFINITY;
        return r;
    }
    __device__ __forceinline__ SampleRow(const X* at, int n) : x(at), V(n), blocks((n + SNT * 8 - 1) / (SNT * 8)) {}
    // NaN as -inf, -0 as +0
    static __device__ __forceinline__ void values(const r8_t& r, float (&v)[8]) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            v[e] = (float)r[e] + 0.0f;
            v[e] = v[e] == v[e] ? v[e] : -INFINITY;
        }
    }
    // f(block, the eight values); blocks behind the last hold -inf
    template <typename F>
    __device__ __forceinline__ void blocks_of(F&& f) const {
        auto one = [&](int j, const r8_t& r) {
            float v[8];
            values(r, v);
            f(j, v);
        };
        r8_t a = read(0), b = read(1);
#pragma unroll 1
        for (int j = 0; j < blocks; j += 2) {
            const r8_t a0 = a, b0 = b;
            a = read(j + 2);
            b = read(j + 3);
            one(j, a0);
            one(j + 1, b0);
        }
    }
    template <typename F>
    __device__ __forceinline__ void each(F&& f) const {
        blocks_of([&](int j, const float (&v)[8]) {
#pragma unroll
            for (int e = 0; e < 8; e++) f((j * SNT + (int)threadIdx.x) * 8 + e, v[e]);
        });
    }
};

// Weights of a row.
struct SampleWeights {
    float M, cf, limit;
    double c, Mc;  // log2(e) / T; times M
    int S;
    const double* table;

    // Bits that a logit is below the largest, in f32: monotone in l, and what decides whether it has a weight at all.
    __device__ __forceinline__ float below(float l) const { return l == M ? 0.0f : (M - l) * cf; }
    __device__ __forceinline__ bool alive(float l) const { return below(l) < limit; }
    // of a logit that is alive: 2^x = 2^n 2^(i/64) 2^r, the last by its series in r ln 2 to the fifth power (r up to 1/128: off by 2^-54)
    __device__ __forceinline__ u64_t weight(float l) const {
        if (l == M) return (u64_t)1 << S;
        const double x = __builtin_fma((double)l, c, -Mc);
        const double big = 0x1.8p52, y = __builtin_fma(x, 64.0, big);
        const int k = (int)(uint32_t)(u64_t)__double_as_longlong(y);
        const double r = __builtin_fma(y - big, -1.0 / 64, x);
        double p = __builtin_fma(r, 1.3333558146428443e-3, 9.618129107628477e-3);  // ln(2)^n / n!
        p = __builtin_fma(p, r, 5.550410866482158e-2);
        p = __builtin_fma(p, r, 2.402265069591007e-1);
        p = __builtin_fma(p, r, 6.931471805599453e-1);
        p = __builtin_fma(p, r, 1.0);
        const double m = table[k & 63] * p;  // from 0.99 to 2
        const double w = __longlong_as_double(__double_as_longlong(m) + ((long long)((k >> 6) + S) << 52));
        return (u64_t)__double_as_longlong(w + 0x1p52) & (((u64_t)1 << 52) - 1);
    }
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

// Of the part s.bin of a row (a wave's share of a block), the index at which the running sum of f(index, logit) reaches rest: in s.found.
template <typename Row, typename F>
__device__ __forceinline__ void pick_in(const Row& row, u64_t rest, F&& f) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, bin = (int)s.bin;
    if ((bin & (SNT / 64 - 1)) != wave) return;
    const int j = bin / (SNT / 64);
    float v[8];
    row.values(row.read(j), v);
    u64_t mine = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) mine += f((j * SNT + tid) * 8 + e, v[e]);
    u64_t upto = wave_scan(mine, lane) - mine;
    if (!(upto < rest && rest <= upto + mine)) return;
    bool done = false;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        upto += f((j * SNT + tid) * 8 + e, v[e]);
        if (!done && upto >= rest) {
            s.found = (uint32_t)((j * SNT + tid) * 8 + e);
            done = true;
        }
    }
}

// The index at which the running sum, by index, of f(index, logit) reaches target(sum of all): in s.found, or not at all
// if the sum is 0.  Returns the sum.
template <typename Row, typename F, typename T>
__device__ __forceinline__ u64_t find_index(const Row& row, F&& f, T&& target_of) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    clear_bins(true, false);
    __syncthreads();
    auto of_block = [&](int j, const float (&v)[8]) {
        u64_t t = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) t += f((j * SNT + tid) * 8 + e, v[e]);
        return t;
    };
    row.blocks_of([&](int j, const float (&v)[8]) {
        const u64_t t = wave_total(of_block(j, v));
        if (lane == 0 && t) s.sum[j * (SNT / 64) + wave] = t;
    });
    __syncthreads();
    u64_t mine, before;
    const u64_t all = total_of(s.sum, mine, before);
    if (all == 0) {
        __syncthreads();
        return 0;
    }
    const u64_t target = target_of(all);
    find_bin(s.sum, mine, before, target);
    const u64_t rest = target - s.above;
    pick_in(row, rest, f);
    __syncthreads();
    return all;
}

// Descending logits and, among equal ones, ascending indexes, as ascending integers.
__device__ __forceinline__ u64_t order_entry(uint32_t key, uint32_t index) { return (u64_t)~key << 32 | index; }
__device__ __forceinline__ float key_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key); }

// s.list[0, n), n a power of two from 2 on, in ascending order (all different, but for ones behind the end).  Short lists
// by counting: the lanes of an entry count those below it.
__device__ __forceinline__ void sort_list(int n) {
    const int tid = threadIdx.x;
    if (n <= 256) {
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
        return;
    }
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
// token goes to s.found, the sum to s.above.
template <typename X>
__device__ __noinline__ void sample_many(const X* x, int V, SampleWeights sw, uint32_t k, bool by_k, float p, bool by_p, u64_t least_w, float u) {
    const int tid = threadIdx.x, lane = tid & 63;
    const float per_bit = (float)SBINS / sw.limit;
    auto bin_of = [&](float l) { return (int)min(sw.below(l) * per_bit, (float)(SBINS - 1)); };
    const SampleRow<X> row(x, V);
    uint32_t key = 0, last = 0xFFFFFFFFu;  // kept: keys above `key`, and that one up to index `last`
    if (by_k || by_p) {
        clear_bins(by_p, by_k);
        __syncthreads();
        row.each([&](int, float l) {
            if (!sw.alive(l)) return;
            const int b = bin_of(l);
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
                select_key<false>(row, sw, rest, [&](float l, uint32_t) { return sw.alive(l) && bin_of(l) == (int)kbin; });
                key = s.key;
                if (by_p) {
                    s.sum[2 * tid] = s0;
                    s.sum[2 * tid + 1] = s1;
                    u64_t part = 0;
                    row.each([&](int, float l) {
                        if (sw.alive(l) && bin_of(l) == (int)kbin && order_key(l) >= key) part += sw.weight(l);
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
            select_key<true>(row, sw, rest, [&](float l, uint32_t kk) { return sw.alive(l) && bin_of(l) == pbin && kk >= least; });
            key = s.key;
            const u64_t w = sw.weight(key_value(key)), ties = (rest - s.above + w - 1) / w;  // so many of the equal ones are kept
            const bool some = s.eq != ties * w;
            __syncthreads();
            if (some) {
                find_index(row, [&](int, float l) { return (u64_t)(order_key(l) == key); }, [&](u64_t) { return ties; });
                last = s.found;
                __syncthreads();
            }
        }
    }
    const u64_t all = find_index(
        row,
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

template <typename X>
__global__ __launch_bounds__(SNT) void sample_rows_kernel(SampleArgs a, int S) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (tid < 64) s.table[tid] = exp2(tid / 64.0);
    const int r = blockIdx.x;
    const SampleRow<X> row((const X*)a.x + (size_t)r * a.vocab, a.vocab);
    // the largest
    float M = -INFINITY;
    row.each([&](int, float l) { M = fmaxf(M, l); });
    M = wave_max(M);
    if (lane == 0) s.wave[wave] = __float_as_uint(M);
    if (tid == 0) s.found = s.bin = 0;  // (always places in the row and in the bins)
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SNT / 64; w++) M = fmaxf(M, __uint_as_float((uint32_t)s.wave[w]));
    __syncthreads();
    const float T = a.temp ? a.temp[r] : 1.0f;
    if (!(T > 0.0f) || M == -INFINITY) {  // greedy, or no logit at all: token 0
        if (tid == 0) s.found = 0xFFFFFFFFu;
        __syncthreads();
        uint32_t first = 0xFFFFFFFFu;
        row.each([&](int i, float l) { first = l == M ? min(first, (uint32_t)i) : first; });
        if (first != 0xFFFFFFFFu) atomicMin(&s.found, first);
        __syncthreads();
        if (tid == 0) {
            a.token[r] = M == -INFINITY ? 0 : s.found;
            if (a.prob) a.prob[r] = M == -INFINITY ? 0.0f : 1.0f;
        }
        return;
    }
    SampleWeights sw;
    sw.M = M;
    sw.c = 1.44269504088896340736 / (double)T;
    sw.Mc = (double)M * sw.c;
    sw.cf = (float)sw.c;
    sw.S = S;
    sw.limit = (float)(S + 1);
    sw.table = s.table;
    const uint32_t k = a.top_k ? a.top_k[r] : 0;
    const float p = a.top_p ? a.top_p[r] : 1.0f, low = a.min_p ? a.min_p[r] : 0.0f;
    const bool by_k = k > 0 && k < (uint32_t)a.vocab, by_p = p < 1.0f;
    const float u = a.u[r];
    const u64_t least = low > 0.0f ? (u64_t)ceil((double)min(low, 1.0f) * (double)((u64_t)1 << S)) : 1;
    auto answer = [&](uint32_t index, float l, u64_t all) {
        a.token[r] = index;
        if (a.prob)
            a.prob[r] = (float)((l == M ? 1.0 : exp2(((double)l - (double)M) * sw.c)) * (double)((u64_t)1 << S) / (double)all);
    };
    // bins of equal width in the logarithm of the weight, from the largest down
    const float per_bit = (float)SBINS / sw.limit;
    auto bin_of = [&](float l) { return (int)min(sw.below(l) * per_bit, (float)(SBINS - 1)); };
    bool many = true;
    if (by_p && !by_k) {
        // Runs of any length: f32 sums of the weights find the bin where the run
        // ends, and one pass with the weights themselves sums up what lies
        // before it (for the whole row, and for the draw in parts of a wave's
        // share of a block) and lists that bin and its neighbours.
        clear_bins(true, false);
        __syncthreads();
        row.each([&](int, float l) {
            if (sw.alive(l)) atomicAdd(&s.sum[bin_of(l)], (u64_t)(uint32_t)(__builtin_amdgcn_exp2f(-sw.below(l)) * 0x1p31f));
        });
        __syncthreads();
        u64_t mine, before;
        const u64_t about = total_of(s.sum, mine, before);
        find_bin(s.sum, mine, before, run_of(p, about));
        const int first = max((int)s.bin - 1, 0), final = (int)s.bin + 1;
        __syncthreads();
        clear_bins(true, false);
        if (tid == 0) s.n = 0;
        __syncthreads();
        u64_t all = 0, sure = 0;
        row.blocks_of([&](int j, const float (&v)[8]) {
            u64_t part = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float l = v[e];
                if (!sw.alive(l)) continue;
                const u64_t w = sw.weight(l);
                const int b = bin_of(l);
                all += w;
                if (b < first) {
                    sure += w;
                    part += w >= least ? w : 0;
                } else if (b <= final) {
                    const uint32_t at = atomicAdd(&s.n, 1u);
                    if (at < SCAP) s.list[at] = order_entry(order_key(l), (uint32_t)((j * SNT + tid) * 8 + e));
                }
            }
            part = wave_total(part);
            if (lane == 0 && part) s.sum[j * (SNT / 64) + wave] = part;
        });
        all = wave_total(all);
        sure = wave_total(sure);
        if (lane == 0) {
            s.wave[wave] = all;
            s.wave2[wave] = sure;
        }
        __syncthreads();
        all = sure = 0;
#pragma unroll
        for (int w = 0; w < SNT / 64; w++) {
            all += s.wave[w];
            sure += s.wave2[w];
        }
        const int n = (int)s.n;
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
                many = false;
                u64_t run = sure + before;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (w[e] && run < want) {
                        const u64_t v = s.list[4 * tid + e];
                        if (w[e] >= least) atomicAdd(&s.sum[(uint32_t)v >> 9], w[e]);  // (an index's part: 512 lie in one)
                        if (run + w[e] >= want) s.end = v;
                    }
                    run += w[e];
                }
                __syncthreads();
                const u64_t end = s.end, sum = total_of(s.sum, mine, before);
                const u64_t target = drawn(u, sum);
                find_bin(s.sum, mine, before, target);
                const u64_t rest = target - s.above;
                pick_in(row, rest, [&](int i, float l) -> u64_t {
                    if (!sw.alive(l)) return 0;
                    const int b = bin_of(l);
                    if (b > final || (b >= first && order_entry(order_key(l), (uint32_t)i) > end)) return 0;
                    const u64_t w = sw.weight(l);
                    return w >= least ? w : 0;
                });
                __syncthreads();  // (the others have read s.above)
                if (tid == 0) s.above = sum;
                __syncthreads();
            }
        }
    } else if (by_k || low > 0.0f) {
        // Few candidates are the usual case: they are listed and sorted.
        int edge = SBINS - 1;  // the last bin that can hold a kept one
        u64_t want = 0;
        bool cut = false;  // by k
        if (by_k) {
            clear_bins(false, true);
            __syncthreads();
            row.each([&](int, float l) {
                if (sw.alive(l)) atomicAdd(&s.count[bin_of(l)], 1u);
            });
            __syncthreads();
            u64_t mine, before;
            cut = total_of(s.count, mine, before) > k;  // (otherwise all that have a weight are kept)
            if (cut) {
                find_bin(s.count, mine, before, k);
                edge = (int)s.bin;
            }
        }
        if (low > 0.0f && !by_p) edge = min(edge, (int)min(per_bit * (0.01f - log2f(min(low, 1.0f))), (float)(SBINS - 1)));
        if (tid == 0) s.n = 0;
        __syncthreads();
        row.each([&](int i, float l) {
            if (!sw.alive(l) || bin_of(l) > edge) return;
            const uint32_t at = atomicAdd(&s.n, 1u);
            if (at < SCAP) s.list[at] = order_entry(order_key(l), (uint32_t)i);
        });
        __syncthreads();
        const int n = (int)s.n;
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
        sample_many<X>((const X*)a.x + (size_t)r * a.vocab, a.vocab, sw, k, by_k, p, by_p, least, u);
    } else if (!(by_p && !by_k)) {
        const u64_t all = find_index(row, [&](int, float l) -> u64_t { return sw.alive(l) ? sw.weight(l) : 0; }, [&](u64_t sum) { return drawn(u, sum); });
        if (tid == 0) s.above = all;
        __syncthreads();
    }
    if (tid == 0) answer(s.found, (float)((const X*)a.x)[(size_t)r * a.vocab + s.found], s.above);
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
