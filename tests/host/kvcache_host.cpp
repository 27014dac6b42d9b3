// The host side of the paged cache (kvcache.cpp, included whole) over a runtime and launchers that work in host memory: what the kernels
// would be handed is checked and done by plain loops, allocations can be made to fail, and attention plans can be read.
#include <cstdio>
#include <cstdlib>

#include "../../tang_amd/csrc/kvcache.cpp"

// ---------------------------------------------------------------------------
// Runtime
// ---------------------------------------------------------------------------

static long g_fail = -1, g_allocs = 0;  // the allocation that fails (counted from now on), and how many there were
static size_t g_bytes = 0;              // asked for since the last reset
static long g_launches = 0;

static bool refused(size_t bytes) {
    g_allocs++;
    g_bytes += bytes;
    if (g_fail < 0) return false;
    return g_fail-- == 0;
}

#define CHECK(x)                                                          \
    do {                                                                  \
        if (!(x)) {                                                       \
            fprintf(stderr, "%s:%d: %s\n", __FILE__, __LINE__, #x);       \
            abort();                                                      \
        }                                                                 \
    } while (0)

extern "C" {
hipError_t hipMalloc(void** p, size_t n) {
    if (refused(n)) return hipErrorOutOfMemory;
    *p = malloc(n ? n : 1);
    return *p ? hipSuccess : hipErrorOutOfMemory;
}
hipError_t hipHostMalloc(void** p, size_t n, unsigned) { return hipMalloc(p, n); }
hipError_t hipFree(void* p) { free(p); return hipSuccess; }
hipError_t hipHostFree(void* p) { free(p); return hipSuccess; }
hipError_t hipMemset(void* p, int v, size_t n) { memset(p, v, n); return hipSuccess; }
hipError_t hipDeviceSynchronize(void) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* s) { *s = hipStreamCaptureStatusNone; return hipSuccess; }
hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) {
    if (refused(0)) return hipErrorOutOfMemory;
    *e = (hipEvent_t)1;
    return hipSuccess;
}
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetLastError(void) { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "error"; }
hipError_t hipLaunchKernel(const void*, dim3, dim3, void**, size_t, hipStream_t) { abort(); }
}

namespace th {

static thread_local std::string g_error;
void set_last_error(const std::string& m) { g_error = m; }
AqlSeq* aql_recording() { return nullptr; }
void aql_record_launch(AqlSeq*, const void*, dim3, dim3, size_t, const void*, size_t) { abort(); }
void aql_wait(th_device*) {}

void* device_scratch(th_device* d, size_t bytes) {
    if (bytes <= d->scratch_bytes) return d->scratch;
    if (d->scratch) (void)hipFree(d->scratch);
    d->scratch = nullptr;
    d->scratch_bytes = 0;
    TH_HIP(hipMalloc(&d->scratch, bytes));
    d->scratch_bytes = bytes;
    return d->scratch;
}
void require_len_any(const th_buffer* b, size_t n, const char* what) {
    if (!b || b->n < n) throw Error(TH_ERR_INVALID, std::string("buffer ") + what + " null or too small");
}
void require_len(const th_buffer* b, th_dtype dt, size_t n, const char* what) {
    require_len_any(b, n, what);
    if (b->dtype != dt) throw Error(TH_ERR_INVALID, std::string("buffer ") + what + " has the wrong dtype");
}

// ---------------------------------------------------------------------------
// Launchers
// ---------------------------------------------------------------------------

void launch_kv_upload(const KvWords& w, const KvTableWork& work, const KvRuns& runs, uint32_t* dst, hipStream_t) {
    g_launches++;
    CHECK(work.src || 3 * work.n_rows + 2 * work.n_pairs + runs.words() <= KV_ARG_WORDS);
    const uint32_t *rows = work.src ? work.src : w.w, *pairs = rows + 3 * work.n_rows, *words = pairs + 2 * work.n_pairs;
    // the parts run at the same time: nothing that one writes may be another's
    std::vector<uint32_t> wrote;
    for (int i = 0; i < work.n_pairs; i++) wrote.push_back(pairs[2 * i]);
    std::sort(wrote.begin(), wrote.end());
    CHECK(std::adjacent_find(wrote.begin(), wrote.end()) == wrote.end());
    auto none = [&](uint32_t at, uint32_t n) {
        const auto x = std::lower_bound(wrote.begin(), wrote.end(), at);
        return x == wrote.end() || *x >= at + n;
    };
    for (int i = 0; i < work.n_rows; i++) {
        CHECK(none(rows[3 * i], rows[3 * i + 2]) && none(rows[3 * i + 1], rows[3 * i + 2]));
        for (int j = 0; j < work.n_rows; j++)
            CHECK(rows[3 * i] >= rows[3 * j + 1] + rows[3 * j + 2] || rows[3 * j + 1] >= rows[3 * i] + rows[3 * i + 2]);
    }
    for (int i = 0; i < work.n_pairs; i++) work.table[pairs[2 * i]] = (int)pairs[2 * i + 1];
    for (int i = 0; i < work.n_rows; i++)
        for (uint32_t j = 0; j < rows[3 * i + 2]; j++) work.table[rows[3 * i + 1] + j] = work.table[rows[3 * i] + j];
    for (int r = 0; r < KvRuns::MAX; r++) {
        std::copy(words, words + runs.n[r], dst + runs.at[r]);
        words += runs.n[r];
    }
}

void launch_kv_copy_pages(void* pool, size_t page_bytes, size_t n_pages, int n_planes, const uint32_t* pairs, size_t n, hipStream_t) {
    g_launches++;
    std::vector<char> wrote(n_pages, 0);
    for (size_t i = 0; i < n; i++) {
        CHECK(pairs[2 * i] < n_pages && pairs[2 * i + 1] < n_pages && !wrote[pairs[2 * i + 1]]);
        wrote[pairs[2 * i + 1]] = 1;
    }
    for (size_t i = 0; i < n; i++) CHECK(!wrote[pairs[2 * i]]);  // no page is both read and written
    for (int p = 0; p < n_planes; p++)
        for (size_t i = 0; i < n; i++)
            memcpy((char*)pool + (p * n_pages + pairs[2 * i + 1]) * page_bytes, (char*)pool + (p * n_pages + pairs[2 * i]) * page_bytes, page_bytes);
}

void launch_kv_copy_upload(void* pool, size_t page_bytes, size_t n_pages, int n_planes, const KvWords& w, size_t n, const KvTableWork& work,
                           const KvRuns& runs, uint32_t* dst, hipStream_t s) {
    CHECK(n > 0 && 2 * n <= KV_ARG_WORDS);
    CHECK(work.src || 2 * n + 3 * work.n_rows + 2 * work.n_pairs + runs.words() <= KV_ARG_WORDS);
    launch_kv_copy_pages(pool, page_bytes, n_pages, n_planes, w.w, n, s);
    KvTableWork at = work;
    if (!at.src) at.src = w.w + 2 * n;
    launch_kv_upload(w, at, runs, dst, s);
}

void launch_kv_gather_rows(void* pool, size_t n_pages, int n_planes, int n_kv_heads, int shift, size_t row_bytes, const uint32_t* from,
                           const uint32_t* to, size_t n, hipStream_t) {
    g_launches++;
    const size_t ps = (size_t)1 << shift, plane = n_pages * n_kv_heads * ps * row_bytes;
    const std::vector<char> was((char*)pool, (char*)pool + n_planes * plane);
    auto row = [&](size_t place, size_t h) { return (((place >> shift) * n_kv_heads + h) * ps + place % ps) * row_bytes; };
    for (int p = 0; p < n_planes; p++)
        for (size_t i = 0; i < n; i++) {
            const size_t a = from[i], b = ((size_t)to[i >> shift] << shift) + i % ps;
            CHECK(a < n_pages * ps && b < n_pages * ps);
            for (int h = 0; h < n_kv_heads; h++) memcpy((char*)pool + p * plane + row(b, h), was.data() + p * plane + row(a, h), row_bytes);
        }
}

static size_t row_of(const KvPages& p, int seq, size_t pos, int h) {
    return (((size_t)p.table[(size_t)seq * p.pages_per_seq + (pos >> p.shift)] * p.n_kv_heads + h) << p.shift) + pos % ((size_t)1 << p.shift);
}
void launch_kv_read(const KvPages& p, int seq, size_t from, size_t n, size_t row_bytes, void* k, void* v, hipStream_t) {
    for (size_t i = 0; i < n; i++)
        for (int h = 0; h < p.n_kv_heads; h++) {
            const size_t at = row_of(p, seq, from + i, h) * row_bytes, to = (i * p.n_kv_heads + h) * row_bytes;
            memcpy((char*)k + to, (const char*)p.k + at, row_bytes);
            memcpy((char*)v + to, (const char*)p.v + at, row_bytes);
        }
}
// 16-bit rows as they are
void launch_kv_append(const KvRopeArgs& a, const KvPages& p, th_dtype cache, const int* n_rows, const KvRow* rows, size_t, hipStream_t) {
    CHECK(a.xdt == cache && a.rot == 0 && !a.q);
    const size_t row_bytes = (size_t)p.hd * 2;
    for (int r = 0; r < *n_rows; r++)
        for (int h = 0; h < p.n_kv_heads; h++) {
            const size_t at = row_of(p, rows[r].seq, (size_t)rows[r].pos, h) * row_bytes, from = ((size_t)r * p.n_kv_heads + h) * row_bytes;
            memcpy((char*)p.k + at, (const char*)a.k + from, row_bytes);
            memcpy((char*)p.v + at, (const char*)a.v + from, row_bytes);
        }
}
void launch_rope_rows(const KvRopeArgs&, size_t, hipStream_t) {}

// A plan is kept for the tests to read.
static KvAttnArgs g_plan;
static const KvTok* g_joins;
static void keep(const KvAttnArgs& a) { g_plan = a; }
void launch_kv_attn_rows(const KvAttnArgs& a, th_dtype, size_t, hipStream_t) { keep(a); }
void launch_kv_attn_tiles(const KvAttnArgs& a, th_dtype, size_t, int, hipStream_t) { keep(a); }
void launch_kv_attn_both(const KvAttnArgs& a, th_dtype, size_t, int, hipStream_t) { keep(a); }
bool kv_join_many(size_t, size_t, size_t) { return false; }
void launch_kv_attn_join(const KvAttnArgs&, const KvTok* list, size_t, size_t, int, hipStream_t) { g_joins = list; }

}  // namespace th

// ---------------------------------------------------------------------------
// Entry points
// ---------------------------------------------------------------------------

extern "C" {
const char* th_last_error(void) { return g_error.c_str(); }
int th_device_create(int, th_device** out) {
    *out = new th_device();
    (*out)->num_cus = 256;
    return TH_OK;
}
int th_device_destroy(th_device* d) {
    free(d->scratch);
    for (void* p : d->retired) free(p);
    d->closed = true;
    if (d->live == 0) delete d;
    return TH_OK;
}
int th_capture_begin(th_device* d) {
    d->capturing = true;
    d->graphs++;
    d->graph_ids.push_back(++d->captures);
    return TH_OK;
}
int th_capture_end(th_device* d, th_graph** out) {
    d->capturing = false;
    device_retain(d);
    *out = new th_graph();
    (*out)->dev = d;
    (*out)->id = d->captures;
    return TH_OK;
}
int th_graph_destroy(th_graph* g) {
    th_device* d = g->dev;
    d->graph_ids.erase(std::find(d->graph_ids.begin(), d->graph_ids.end(), g->id));
    delete g;
    d->graphs--;
    device_release(d);
    return TH_OK;
}
int th_buffer_alloc(th_device* d, th_dtype t, size_t n, th_buffer** out) {
    th_buffer* b = new th_buffer();
    b->dev = d;
    b->dtype = t;
    b->n = n;
    b->ptr = calloc(n + 1, dtype_size(t));
    device_retain(d);
    *out = b;
    return TH_OK;
}
int th_buffer_free(th_buffer* b) {
    th_device* d = b->dev;
    free(b->ptr);
    delete b;
    device_release(d);
    return TH_OK;
}
int th_buffer_upload(th_buffer* b, const void* h, size_t n) { memcpy(b->ptr, h, n * dtype_size(b->dtype)); return TH_OK; }
int th_buffer_download(th_buffer* b, void* h, size_t n) { memcpy(h, b->ptr, n * dtype_size(b->dtype)); return TH_OK; }

void host_fail(long which) { g_fail = which; }
long host_allocs(void) { return g_allocs; }
size_t host_bytes(void) { return g_bytes; }
long host_launches(void) { return g_launches; }
// The last attention call's plan: how many rows items, tile items and joined tokens it has, and copies of its parts.
void host_plan_sizes(int* n) {
    n[0] = g_plan.head->n_rows_items;
    n[1] = g_plan.head->n_tile_items;
    n[2] = g_plan.head->n_joins;
}
void host_plan(int n_toks, int* toks, int* rows_items, int* tile_items, int* joins) {
    memcpy(toks, g_plan.toks, n_toks * sizeof(KvTok));
    memcpy(rows_items, g_plan.rows_items, g_plan.head->n_rows_items * sizeof(KvItem));
    memcpy(tile_items, g_plan.tile_items, g_plan.head->n_tile_items * sizeof(KvItem));
    memcpy(joins, g_joins, g_plan.head->n_joins * sizeof(KvTok));
}
}
