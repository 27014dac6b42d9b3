// Kernels that move a paged cache's rows: uploads of tables and plans, copies
// of pages, gathers of rows, and the rotary step that fills the pages.
#include <algorithm>

#include "kvcache.hpp"
#include "kvrows.hpp"
#include "ops.hpp"

namespace th {

typedef uint32_t kv_u32x4_t __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------
// Uploads
// ---------------------------------------------------------------------------

// A step's tables and plans are some hundred words: as launch arguments they
// need no copy, no staging memory and no event.  More comes from pinned host
// memory, which the kernel reads across the bus by itself.
__device__ __forceinline__ void kv_upload_words(int block, int blocks, const uint32_t* src, const KvTableWork& work,
                                                const KvRuns& runs, uint32_t* dst) {
    const int i0 = block * 256 + threadIdx.x, step = blocks * 256;
    for (int r = block; r < work.n_rows; r += blocks) {
        const int *from = work.table + src[3 * r], n = (int)src[3 * r + 2];
        int* to = work.table + src[3 * r + 1];
        for (int i = threadIdx.x; i < n; i += 256) to[i] = from[i];
    }
    src += 3 * work.n_rows;
    for (int i = i0; i < work.n_pairs; i += step) work.table[src[2 * i]] = (int)src[2 * i + 1];
    src += 2 * work.n_pairs;
    const int n_words = runs.words();
    for (int i = i0; i < n_words; i += step) {
        int to = i, end = 0;
#pragma unroll
        for (int r = 0; r < KvRuns::MAX; r++) {
            if (i >= end) to = runs.at[r] + i - end;
            end += runs.n[r];
        }
        dst[to] = src[i];
    }
}

__global__ __launch_bounds__(256) void kv_upload_kernel(KvWords w, KvTableWork work, KvRuns runs, uint32_t* dst) {
    kv_upload_words(blockIdx.x, gridDim.x, work.src ? work.src : w.w, work, runs, dst);
}

void launch_kv_upload(const KvWords& w, const KvTableWork& work, const KvRuns& runs, uint32_t* dst, hipStream_t s) {
    const size_t n = std::max(ceil_div((size_t)work.n_pairs + runs.words(), 256), (size_t)work.n_rows);
    if (n == 0) return;
    TH_LAUNCH(kv_upload_kernel, dim3((unsigned)std::min<size_t>(n, 64)), dim3(256), 0, s, w, work, runs, dst);
    TH_LAUNCH_CHECK();
}

// ---------------------------------------------------------------------------
// Pages and rows
// ---------------------------------------------------------------------------

// A page is one contiguous piece of each of the 2 * layers planes; 16 KiB of it
// to a workgroup, four 16-byte loads of every thread in flight.  Bound by
// memory: each byte is read once and written once, at 5.5 TB/s both ways for 700 pages of eight layers.
constexpr int KV_COPY_BYTES = 16384;

__device__ __forceinline__ void kv_copy_piece(char* pool, size_t page_bytes, size_t n_pages, uint32_t from, uint32_t to) {
    const size_t plane = (size_t)blockIdx.z * n_pages * page_bytes;
    const size_t at = (size_t)blockIdx.y * KV_COPY_BYTES + threadIdx.x * 16;
    const char* src = pool + plane + from * page_bytes + at;
    char* dst = pool + plane + to * page_bytes + at;
    kv_u32x4_t v[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (at + i * 4096 < page_bytes) v[i] = *(const kv_u32x4_t*)(src + i * 4096);
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (at + i * 4096 < page_bytes) *(kv_u32x4_t*)(dst + i * 4096) = v[i];
}

__global__ __launch_bounds__(256) void kv_copy_pages_kernel(char* __restrict__ pool, size_t page_bytes, size_t n_pages,
                                                            const uint32_t* __restrict__ pairs) {
    kv_copy_piece(pool, page_bytes, n_pages, pairs[2 * blockIdx.x], pairs[2 * blockIdx.x + 1]);
}

// A step whose sequences get copies of shared pages: the copies and the upload touch different memory, so they share a
// launch (2.4 us of host time); the upload is the work of one more plane.
__global__ __launch_bounds__(256) void kv_copy_upload_kernel(char* __restrict__ pool, size_t page_bytes, size_t n_pages, KvWords w,
                                                             KvTableWork work, KvRuns runs, uint32_t* dst) {
    if (blockIdx.z + 1 < gridDim.z)
        kv_copy_piece(pool, page_bytes, n_pages, w.w[2 * blockIdx.x], w.w[2 * blockIdx.x + 1]);
    else
        kv_upload_words(blockIdx.y * gridDim.x + blockIdx.x, gridDim.x * gridDim.y, work.src ? work.src : w.w + 2 * gridDim.x, work, runs,
                        dst);
}

void launch_kv_copy_pages(void* pool, size_t page_bytes, size_t n_pages, int n_planes, const uint32_t* pairs, size_t n,
                          hipStream_t s) {
    // (a launch has below 2^32 threads: more pages go in slices)
    for (size_t at = 0; at < n; at += KV_MAX_BLOCKS) {
        const dim3 grid((unsigned)std::min(n - at, KV_MAX_BLOCKS), (unsigned)ceil_div(page_bytes, (size_t)KV_COPY_BYTES), (unsigned)n_planes);
        TH_LAUNCH(kv_copy_pages_kernel, grid, dim3(256), 0, s, (char*)pool, page_bytes, n_pages, pairs + 2 * at);
        TH_LAUNCH_CHECK();
    }
}

void launch_kv_copy_upload(void* pool, size_t page_bytes, size_t n_pages, int n_planes, const KvWords& w, size_t n,
                           const KvTableWork& work, const KvRuns& runs, uint32_t* dst, hipStream_t s) {
    TH_LAUNCH(kv_copy_upload_kernel,
              dim3((unsigned)n, (unsigned)ceil_div(page_bytes, (size_t)KV_COPY_BYTES), (unsigned)n_planes + 1), dim3(256), 0, s,
              (char*)pool, page_bytes, n_pages, w, work, runs, dst);
    TH_LAUNCH_CHECK();
}

// Workgroup = (page to fill, kv head, plane): its rows lie together, so writes
// are whole lines; reads are a row (hd * 2 bytes) at a time.
__global__ __launch_bounds__(256) void kv_gather_rows_kernel(char* __restrict__ pool, size_t n_pages, int n_kv_heads, int shift,
                                                             int cpr, const uint32_t* __restrict__ from,
                                                             const uint32_t* __restrict__ to, int n) {
    const size_t row_bytes = (size_t)cpr * 16;
    char* plane = pool + (size_t)blockIdx.z * n_pages * (((size_t)n_kv_heads * row_bytes) << shift);
    const int first = blockIdx.x << shift, rows = min(1 << shift, n - first), h = blockIdx.y;
    char* dst = plane + ((((size_t)to[blockIdx.x] * n_kv_heads + h) << shift) * row_bytes);
    const uint32_t mask = (1u << shift) - 1;
    for (int i0 = threadIdx.x; i0 < rows * cpr; i0 += 1024) {
        kv_u32x4_t v[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int i = i0 + 256 * u;
            if (i >= rows * cpr) continue;
            const uint32_t at = from[first + i / cpr];
            const size_t row = (((size_t)(at >> shift) * n_kv_heads + h) << shift) + (at & mask);
            v[u] = *(const kv_u32x4_t*)(plane + row * row_bytes + (size_t)(i % cpr) * 16);
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (i0 + 256 * u < rows * cpr) *(kv_u32x4_t*)(dst + (size_t)(i0 + 256 * u) * 16) = v[u];
    }
}

void launch_kv_gather_rows(void* pool, size_t n_pages, int n_planes, int n_kv_heads, int shift, size_t row_bytes,
                           const uint32_t* from, const uint32_t* to, size_t n, hipStream_t s) {
    const size_t pages = ceil_div(n, (size_t)1 << shift);
    for (size_t at = 0; at < pages; at += KV_MAX_BLOCKS) {
        const dim3 grid((unsigned)std::min(pages - at, KV_MAX_BLOCKS), (unsigned)n_kv_heads, (unsigned)n_planes);
        TH_LAUNCH(kv_gather_rows_kernel, grid, dim3(256), 0, s, (char*)pool, n_pages, n_kv_heads, shift, (int)(row_bytes / 16),
                  from + (at << shift), to + at, (int)(n - (at << shift)));
        TH_LAUNCH_CHECK();
    }
}

__global__ __launch_bounds__(256) void kv_read_kernel(KvPages p, int seq, size_t from, size_t total, int cpr,
                                                      kv_u32x4_t* __restrict__ k, kv_u32x4_t* __restrict__ v) {
    const int* table = p.table + (size_t)seq * p.pages_per_seq;
    const uint32_t mask = (1u << p.shift) - 1;
    for (size_t i = blockIdx.x * (size_t)256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
        const size_t rh = i / cpr, pos = from + rh / p.n_kv_heads;
        const int c = (int)(i % cpr), h = (int)(rh % p.n_kv_heads);
        const size_t row = (((size_t)table[pos >> p.shift] * p.n_kv_heads + h) << p.shift) + (pos & mask);
        k[i] = ((const kv_u32x4_t*)p.k)[row * cpr + c];
        v[i] = ((const kv_u32x4_t*)p.v)[row * cpr + c];
    }
}

void launch_kv_read(const KvPages& p, int seq, size_t from, size_t n, size_t row_bytes, void* k, void* v, hipStream_t s) {
    const size_t cpr = row_bytes / 16, total = n * p.n_kv_heads * cpr;
    if (total == 0) return;
    TH_LAUNCH(kv_read_kernel, dim3((unsigned)std::min<size_t>(ceil_div(total, 256), 8192)), dim3(256), 0, s, p, seq, from, total,
              (int)cpr, (kv_u32x4_t*)k, (kv_u32x4_t*)v);
    TH_LAUNCH_CHECK();
}

// ---------------------------------------------------------------------------
// Rotary positions
// ---------------------------------------------------------------------------

// A pair (x, y) at position p turns by p * freq: (x c - y s, x s + y c), in f32,
// rounded once to the output's type; dims from `rot` on pass through.  One
// thread holds eight dims (and, in the half layout, the eight that they are paired
// with): 16-byte loads and stores of 16-bit types, two of f32.  Bound by
// memory: q, k and v are read once and written once, in one launch; the tables'
// rows are shared by a token's heads and stay in the caches.  16000 f32 tokens of 32 + 8 + 8 heads of 128
// into an f16 cache: 167 us, 4.4 TB/s.  One token: a launch.
// One head of one row: thread c of `lanes` takes its chunks.  VEC: rot is a
// multiple of 16, so that chunks of eight never straddle halves or the rest.
template <typename X, bool VEC>
__device__ __forceinline__ void kv_turn_head(const KvRopeArgs& a, const X* src, void* dst, th_dtype ddt, size_t at, size_t pos,
                                             int c, bool turn) {
    const int rot = turn ? a.rot : 0, hr = rot >> 1;
    const bool known = pos < a.table_rows;
    const float *ct = a.cos_t + (known ? pos : 0) * hr, *st = a.sin_t + (known ? pos : 0) * hr;
    if constexpr (VEC) {
        const int d = c * 8;
        if (d >= rot) {  // passes through
            kv_store8(dst, ddt, at + d, kv_load8(src + d));
        } else if (a.half) {
            if (d >= hr) return;  // its partner's thread writes it
            const kv_f8 x = kv_load8(src + d), y = kv_load8(src + d + hr), cs = kv_load8(ct + d), sn = kv_load8(st + d);
            kv_f8 u, w;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                u.v[i] = known ? x.v[i] * cs.v[i] - y.v[i] * sn.v[i] : __builtin_nanf("");
                w.v[i] = known ? y.v[i] * cs.v[i] + x.v[i] * sn.v[i] : __builtin_nanf("");
            }
            kv_store8(dst, ddt, at + d, u);
            kv_store8(dst, ddt, at + d + hr, w);
        } else {
            const kv_f8 x = kv_load8(src + d);
            const float4 cs = *(const float4*)(ct + d / 2), sn = *(const float4*)(st + d / 2);
            const float cc[4] = {cs.x, cs.y, cs.z, cs.w}, ss[4] = {sn.x, sn.y, sn.z, sn.w};
            kv_f8 u;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                u.v[2 * i] = known ? x.v[2 * i] * cc[i] - x.v[2 * i + 1] * ss[i] : __builtin_nanf("");
                u.v[2 * i + 1] = known ? x.v[2 * i] * ss[i] + x.v[2 * i + 1] * cc[i] : __builtin_nanf("");
            }
            kv_store8(dst, ddt, at + d, u);
        }
    } else {  // any even rot: thread c takes pairs and rests one by one
        for (int i = c; i < a.hd - hr; i += (a.hd + 7) / 8) {
            if (i >= hr) {
                const int d = i + hr;
                kv_store1(dst, ddt, at + d, (float)src[d]);
                continue;
            }
            const int d0 = a.half ? i : 2 * i, d1 = a.half ? i + hr : 2 * i + 1;
            const float x = (float)src[d0], y = (float)src[d1], cs = ct[i], sn = st[i];
            kv_store1(dst, ddt, at + d0, known ? x * cs - y * sn : __builtin_nanf(""));
            kv_store1(dst, ddt, at + d1, known ? x * sn + y * cs : __builtin_nanf(""));
        }
    }
}

// Thread = (row, head of q | k | v, chunk of eight dims).
template <typename X, bool VEC>
__global__ __launch_bounds__(256) void kv_append_kernel(KvRopeArgs a, KvPages p, th_dtype cache, const int* __restrict__ n_rows,
                                                        const KvRow* __restrict__ rows) {
    const int cpr = a.hd / 8, heads = a.n_heads + 2 * p.n_kv_heads, per_row = heads * cpr;
    const size_t total = (size_t)*n_rows * per_row;
    for (size_t idx = blockIdx.x * (size_t)256 + threadIdx.x; idx < total; idx += (size_t)gridDim.x * 256) {
        const uint32_t row = (uint32_t)(idx / per_row);
        const int i = (int)(idx - (size_t)row * per_row), hh = i / cpr, c = i - hh * cpr;
        const KvRow r = rows[row];
        const size_t pos = a.positions ? (size_t)a.positions[row] : (size_t)r.pos;
        if (hh < a.n_heads) {
            const size_t at = ((size_t)row * a.n_heads + hh) * a.hd;
            kv_turn_head<X, VEC>(a, (const X*)a.q + at, a.q_out, a.qdt, at, pos, c, true);
            continue;
        }
        const bool is_k = hh < a.n_heads + p.n_kv_heads;
        const int h = hh - a.n_heads - (is_k ? 0 : p.n_kv_heads);
        const int page = p.table[(size_t)r.seq * p.pages_per_seq + (r.pos >> p.shift)];
        const size_t at = ((((size_t)page * p.n_kv_heads + h) << p.shift) + (r.pos & ((1 << p.shift) - 1))) * a.hd;
        const X* src = (const X*)(is_k ? a.k : a.v) + ((size_t)row * p.n_kv_heads + h) * a.hd;
        kv_turn_head<X, VEC>(a, src, const_cast<void*>(is_k ? p.k : p.v), cache, at, pos, c, is_k);
    }
}

template <typename X, bool VEC>
__global__ __launch_bounds__(256) void rope_rows_kernel(KvRopeArgs a, size_t n_rows) {
    const int cpr = (a.hd + 7) / 8, per_row = a.n_heads * cpr;
    const size_t total = n_rows * per_row;
    for (size_t idx = blockIdx.x * (size_t)256 + threadIdx.x; idx < total; idx += (size_t)gridDim.x * 256) {
        const size_t row = idx / per_row;
        const int i = (int)(idx - row * per_row), h = i / cpr, c = i - h * cpr;
        const size_t at = (row * a.n_heads + h) * a.hd;
        kv_turn_head<X, VEC>(a, (const X*)a.q + at, a.q_out, a.qdt, at, a.positions ? (size_t)a.positions[row] : a.start + row, c, true);
    }
}

// Chunks of eight need every row to start on 16 bytes (hd a multiple of 8).
static bool rope_vec(const KvRopeArgs& a) { return a.hd % 8 == 0 && a.rot % 16 == 0; }

static unsigned rope_grid(size_t threads) { return (unsigned)std::max<size_t>(1, std::min<size_t>(ceil_div(threads, 256), 16384)); }

template <typename F>
static void rope_types(const KvRopeArgs& a, F&& f) {
    const bool vec = rope_vec(a);
    auto with = [&](auto x) {
        if (vec) f(x, std::true_type{});
        else f(x, std::false_type{});
    };
    if (a.xdt == TH_F32) with(float{});
    else if (a.xdt == TH_F16) with((_Float16)0);
    else with((__bf16)0.0f);
}

void launch_kv_append(const KvRopeArgs& a, const KvPages& p, th_dtype cache, const int* n_rows_dev, const KvRow* rows,
                      size_t n_rows, hipStream_t s) {
    if (n_rows == 0) return;
    if (a.norm) return launch_norm_append(a, p, cache, n_rows_dev, rows, n_rows, s);
    const unsigned grid = rope_grid(n_rows * (a.n_heads + 2 * p.n_kv_heads) * (a.hd / 8));
    rope_types(a, [&](auto x, auto vec) {
        TH_LAUNCH((kv_append_kernel<decltype(x), decltype(vec)::value>), dim3(grid), dim3(256), 0, s, a, p, cache, n_rows_dev, rows);
    });
    TH_LAUNCH_CHECK();
}

void launch_rope_rows(const KvRopeArgs& a, size_t n_rows, hipStream_t s) {
    if (a.norm) return launch_norm_rows(a, n_rows, s);
    const size_t threads = n_rows * a.n_heads * ((a.hd + 7) / 8);
    if (threads == 0) return;
    rope_types(a, [&](auto x, auto vec) {
        TH_LAUNCH((rope_rows_kernel<decltype(x), decltype(vec)::value>), dim3(rope_grid(threads)), dim3(256), 0, s, a, n_rows);
    });
    TH_LAUNCH_CHECK();
}

}  // namespace th
