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

constexpr int SNT = 1024, SBINS = 2048, SLIST = 64;
typedef unsigned long long u64_t;

struct SampleLds {
    u64_t sum[SBINS];
    uint32_t count[SBINS];
    double table[64];  // 2^(i / 64)
    u64_t list_w[SLIST];
    uint32_t list_key[SLIST];
    u64_t wave[SNT / 64];
    u64_t above, eq;
    uint32_t bin, key, n, lo, hi, found;
};

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

// A row's logits: thread t has elements (j 1024 + t) 8 + e of block j.  Every pass
// streams them, a block ahead (later passes from the caches).
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
    // NaN as -inf, -0 as +0
    static __device__ __forceinline__ void values(const r8_t& r, float (&v)[8]) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            v[e] = (float)r[e] + 0.0f;
            v[e] = v[e] == v[e] ? v[e] : -INFINITY;
        }
    }
    // f(block, the eight values)
    template <typename F>
    __device__ __forceinline__ void blocks_of(F&& f) const {
        r8_t next = read(0);
#pragma unroll 1
        for (int j = 0; j < blocks; j++) {
            const r8_t now = next;
            if (j + 1 < blocks) next = read(j + 1);
            float v[8];
            values(now, v);
            f(j, v);
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
    double c;
    int S;
    const double* table;

    // Bits that a logit is below the largest, in f32: monotone in l, and what decides whether it has a weight at all.
    __device__ __forceinline__ float below(float l) const { return l == M ? 0.0f : (M - l) * cf; }
    __device__ __forceinline__ bool alive(float l) const { return below(l) < limit; }
    // of a logit that is alive: 2^x = 2^n 2^(i/64) 2^r, the last by its series to r^5 (r below 1/128: 2^-53)
    __device__ __forceinline__ u64_t weight(float l) const {
        if (l == M) return (u64_t)1 << S;
        const double x = ((double)l - (double)M) * c;
        const double big = 0x1.8p52, y = __builtin_fma(x, 64.0, big);
        const int k = (int)(uint32_t)(u64_t)__double_as_longlong(y);
        const double z = __builtin_fma(y - big, -1.0 / 64, x) * 0.69314718055994530942;
        double p = __builtin_fma(z, 1.0 / 120, 1.0 / 24);
        p = __builtin_fma(p, z, 1.0 / 6);
        p = __builtin_fma(p, z, 0.5);
        p = __builtin_fma(p, z, 1.0);
        p = __builtin_fma(p, z, 1.0);
        const double m = table[k & 63] * p;  // from 0.99 to 2
        const double w = __longlong_as_double(__double_as_longlong(m) + ((long long)((k >> 6) + S) << 52));
        return (u64_t)__double_as_longlong(w + 0x1p52) & (((u64_t)1 << 52) - 1);
    }
};

// The first of SBINS bins at which the running sum reaches target (1 to the sum of all): in s.bin, what lies
// before it in s.above.  Returns the sum of all.  Call with the whole block, after a barrier; ends with one.
template <typename T>
__device__ __forceinline__ u64_t total_of(const T* hist, SampleLds& s, u64_t& mine, u64_t& before) {
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
__device__ __forceinline__ void find_bin(const T* hist, SampleLds& s, u64_t mine, u64_t before, u64_t target) {
    if (before < target && target <= before + mine) {
        const u64_t a = hist[2 * threadIdx.x];
        const bool second = before + a < target;
        s.bin = 2 * threadIdx.x + second;
        s.above = before + (second ? a : 0);
    }
    __syncthreads();
}

__device__ __forceinline__ void clear_bins(SampleLds& s, bool sums, bool counts) {
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
__device__ __forceinline__ void select_key(const Row& row, const SampleWeights& sw, SampleLds& s, u64_t target, In&& in) {
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
        clear_bins(s, WEIGHTS, !WEIGHTS);
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
            (void)total_of(s.sum, s, mine, before);
            find_bin(s.sum, s, mine, before, target - above);
        } else {
            (void)total_of(s.count, s, mine, before);
            find_bin(s.count, s, mine, before, target - above);
        }
        const uint32_t bin = s.bin, first = bin << shift;
        above += s.above;
        lo = hi - lo - first < (1u << shift) ? lo : hi - first - ((1u << shift) - 1);
        hi -= first;
        __syncthreads();
    }
    __syncthreads();
}

// The index at which the running sum, by index, of f(index, logit) reaches target(sum of all): in s.found, or not at all
// if the sum is 0.  Returns the sum.
template <typename Row, typename F, typename T>
__device__ __forceinline__ u64_t find_index(const Row& row, SampleLds& s, F&& f, T&& target_of) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    clear_bins(s, true, false);
    __syncthreads();
    auto of_block = [&](int j, const float (&v)[8]) {
        u64_t t = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) t += f((j * SNT + tid) * 8 + e, v[e]);
        return t;
    };
    row.blocks_of([&](int j, const float (&v)[8]) {
        const u64_t t = wave_total(of_block(j, v));
        if (lane == 0) s.sum[j * (SNT / 64) + wave] = t;
    });
    __syncthreads();
    u64_t mine, before;
    const u64_t all = total_of(s.sum, s, mine, before);
    if (all == 0) {
        __syncthreads();
        return 0;
    }
    const u64_t target = target_of(all);
    find_bin(s.sum, s, mine, before, target);
    const int bin = (int)s.bin;
    const u64_t rest = target - s.above;
    if ((bin & (SNT / 64 - 1)) == wave) {
        const int j = bin / (SNT / 64);
        float v[8];
        row.values(row.read(j), v);
        const u64_t mine_here = of_block(j, v);
        u64_t upto = wave_scan(mine_here, lane) - mine_here;
        if (upto < rest && rest <= upto + mine_here) {
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
    }
    __syncthreads();
    return all;
}

template <typename X>
__global__ __launch_bounds__(SNT) void sample_rows_kernel(SampleArgs a, int S) {
    __shared__ SampleLds s;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (tid < 64) s.table[tid] = exp2(tid / 64.0);
    for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
        SampleRow<X> row;
        row.x = (const X*)a.x + (size_t)r * a.vocab;
        row.V = a.vocab;
        row.blocks = (a.vocab + SNT * 8 - 1) / (SNT * 8);
        // the largest
        float M = -INFINITY;
        row.each([&](int, float l) { M = fmaxf(M, l); });
        M = wave_max(M);
        if (lane == 0) s.wave[wave] = __float_as_uint(M);
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
            __syncthreads();
            continue;
        }
        SampleWeights sw;
        sw.M = M;
        sw.c = 1.44269504088896340736 / (double)T;
        sw.cf = (float)sw.c;
        sw.S = S;
        sw.limit = (float)(S + 1);
        sw.table = s.table;
        const uint32_t k = a.top_k ? a.top_k[r] : 0;
        const float p = a.top_p ? a.top_p[r] : 1.0f, low = a.min_p ? a.min_p[r] : 0.0f;
        const bool by_k = k > 0 && k < (uint32_t)a.vocab, by_p = p < 1.0f;
        uint32_t key = 0, last = 0xFFFFFFFFu;  // kept: keys above `key`, and that one up to index `last`
        if (by_k || by_p) {
            // bins of equal width in the logarithm of the weight, from the largest down
            clear_bins(s, by_p, by_k);
            __syncthreads();
            const float per_bit = (float)SBINS / sw.limit;
            auto bin_of = [&](float l) { return (int)min(sw.below(l) * per_bit, (float)(SBINS - 1)); };
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
                const u64_t n = total_of(s.count, s, mine, before);
                if (n > k) {  // (otherwise all that have a weight are kept)
                    find_bin(s.count, s, mine, before, k);
                    kbin = s.bin;
                    const u64_t rest = k - s.above;
                    __syncthreads();
                    // the sums are needed again: they move to registers while keys are sorted
                    const u64_t s0 = s.sum[2 * tid], s1 = s.sum[2 * tid + 1];
                    select_key<false>(row, sw, s, rest, [&](float l, uint32_t) { return sw.alive(l) && bin_of(l) == (int)kbin; });
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
                kept = total_of(s.sum, s, mine, before);
                const u64_t want = p > 0.0f ? max((u64_t)1, min(kept, (u64_t)ceil((double)p * (double)kept))) : 1;
                find_bin(s.sum, s, mine, before, want);
                const int pbin = (int)s.bin;
                const u64_t rest = want - s.above;
                __syncthreads();
                const uint32_t least = key;
                select_key<true>(row, sw, s, rest, [&](float l, uint32_t kk) { return sw.alive(l) && bin_of(l) == pbin && kk >= least; });
                key = s.key;
                const float at = __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
                const u64_t w = sw.weight(at), ties = (rest - s.above + w - 1) / w;  // so many of the equal ones are kept
                const bool some = s.eq != ties * w;
                __syncthreads();
                if (some) {
                    find_index(row, s, [&](int, float l) { return (u64_t)(order_key(l) == key); }, [&](u64_t) { return ties; });
                    last = s.found;
                    __syncthreads();
                }
            }
        }
        const u64_t least = low > 0.0f ? (u64_t)ceil((double)min(low, 1.0f) * (double)((u64_t)1 << S)) : 1;
        const float u = a.u[r];
        auto kept = [&](int i, float l) -> u64_t {
            const uint32_t kk = order_key(l);
            if (kk < key || (kk == key && (uint32_t)i > last) || !sw.alive(l)) return 0;
            const u64_t w = sw.weight(l);
            return w >= least ? w : 0;
        };
        const u64_t all = find_index(row, s, kept, [&](u64_t sum) {
            const double t = (double)u * (double)sum;
            return t >= (double)sum ? sum : t >= 0.0 ? min((u64_t)t, sum - 1) + 1 : (u64_t)1;
        });
        if (tid == 0) {
            a.token[r] = s.found;
            if (a.prob) {
                const float l = (float)row.x[s.found];
                a.prob[r] = (float)((l == M ? 1.0 : exp2(((double)l - (double)M) * sw.c)) * (double)((u64_t)1 << S) / (double)all);
            }
        }
        __syncthreads();
    }
}

void launch_sample_rows(const SampleArgs& a, hipStream_t s) {
    if (a.rows == 0) return;
    int bits = 0;
    while (((size_t)1 << bits) < (size_t)a.vocab) bits++;
    const int S = std::min(51, 62 - bits);
    const dim3 grid((unsigned)std::min(a.rows, 1 << 16));
    auto types = [&](auto x) { TH_LAUNCH((sample_rows_kernel<decltype(x)>), grid, dim3(SNT), 0, s, a, S); };
    if (a.xdt == TH_F32) types(float{});
    else if (a.xdt == TH_F16) types((_Float16)0);
    else types((__bf16)0.0f);
    TH_LAUNCH_CHECK();
}

}  // namespace th
