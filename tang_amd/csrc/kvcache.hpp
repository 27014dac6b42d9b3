// The paged key/value cache, its batches, and the launchers of its kernels.
#pragma once

#include <map>
#include <vector>

#include "capi_util.hpp"

namespace th {

// ---------------------------------------------------------------------------
// What kernels read
// ---------------------------------------------------------------------------

// One layer's pages: [page][kv head][place][dim] of the cache's type, so the
// rows of one head of one page lie together.  A row number is
// (page * kv_heads + head) * page_size + place; it fits 32 bits (checked when a
// cache is made), its address needs 64.
struct KvPages {
    const void *k, *v;
    const int* table;  // [sequence][pages_per_seq]
    int pages_per_seq, shift, n_kv_heads, hd;
};

// A row of a batch: its sequence and its position in it.
struct KvRow { int seq, pos; };

// A token of an attention plan: its row in the batch, its position, its first
// record (-1: none), and where its own keys' records start (low half) and how many records it has
// (high half).
struct KvTok { int row, pos, rec, own_n; };

// A piece of attention work: tokens [tok0, tok0 + ntok) against the keys of a
// range of sequence `seq`.  The range is in numbers that leave hidden keys out:
// number j is key j below `sink_end`, key j + gap from there on.  rec: the
// piece's number among the records of its tokens (bit 30: counted from their own
// keys' first), or -1 where the piece has all their keys and writes the result.
struct KvItem { int tok0, ntok, seq, j0, j1, sink_end, gap, rec; };
constexpr int KV_REC_OWN = 1 << 30;

// An attention plan in device memory: counts, tokens, the two kernels'
// items and the tokens whose records are joined, each part at a place of its own that does not change with the step.
struct KvPlanHead { int n_rows_items, n_tile_items, n_joins, flags; };
// flags: an item of tiles has more than KV_LONG_ITEM keys; the join is that of many rows.  What they choose adds up in another order, so a captured
// call, which runs on whatever plan there is, goes by them as an eager one does.
constexpr int KV_PLAN_FAR = 1, KV_PLAN_MANY = 2;
constexpr int KV_HEAD_WORDS = sizeof(KvPlanHead) / 4;

struct KvAttnArgs {
    KvPages pages;
    const KvPlanHead* head;
    const KvTok* toks;
    const KvItem *rows_items, *tile_items;
    const void* q;
    void* out;
    th_dtype qdt, odt;
    int n_heads, window, sinks;
    float scale;        // of the scores, times log2(e)
    float* rec_o;       // [record][query head][dim]
    float2* rec_ml;     // [record][query head] {maximum, sum}
};

// ---------------------------------------------------------------------------
// Launchers (kvpages.hip, kvattn_*.hip)
// ---------------------------------------------------------------------------

// Words that go into a kernel's argument block.
constexpr int KV_ARG_WORDS = 224, KV_ARG_COPIES = KV_ARG_WORDS / 2;
constexpr unsigned KV_STAGES = 8;
struct KvWords { uint32_t w[KV_ARG_WORDS]; };

// Runs of words that follow one another in an upload's source: their lengths and where each goes.
struct KvRuns {
    static constexpr int MAX = 5;
    int n[MAX] = {}, at[MAX] = {};
    __host__ __device__ int words() const { return n[0] + n[1] + n[2] + n[3] + n[4]; }
};
// Changes of a table: n_rows times {from, to, n} (n entries copied from one place to another; none of a place that changes),
// n_pairs times {index, value}, then an upload's words; all from src (device-visible host memory) or, where that is null,
// from a launch's arguments.
struct KvTableWork {
    const uint32_t* src;
    int n_rows, n_pairs;
    int* table;
};
void launch_kv_upload(const KvWords& w, const KvTableWork& work, const KvRuns& runs, uint32_t* dst, hipStream_t s);
// Whole pages, every layer's K and V.  pairs (device): {from, to}.
void launch_kv_copy_pages(void* pool, size_t page_bytes, size_t n_pages, int n_planes, const uint32_t* pairs, size_t n,
                          hipStream_t s);
// n copies whose pairs are the first of w, and an upload whose words follow them there or are in src.
void launch_kv_copy_upload(void* pool, size_t page_bytes, size_t n_pages, int n_planes, const KvWords& w, size_t n,
                           const KvTableWork& work, const KvRuns& runs, uint32_t* dst, hipStream_t s);
// Rows: place i of the pages to[] takes the row that is at place from[i] of the
// line of all places, every layer's K and V.
void launch_kv_gather_rows(void* pool, size_t n_pages, int n_planes, int n_kv_heads, int shift, size_t row_bytes,
                           const uint32_t* from, const uint32_t* to, size_t n, hipStream_t s);
// Rows of one sequence in one layer to [n][kv heads][dim].
void launch_kv_read(const KvPages& p, int seq, size_t from, size_t n, size_t row_bytes, void* k, void* v, hipStream_t s);

struct KvRopeArgs {
    const void *q, *k, *v;
    void* q_out;
    th_dtype xdt, qdt;           // of q, k and v; of q_out
    const float *cos_t, *sin_t;  // [table_rows][rot/2]; null: nothing is turned
    const uint32_t* positions;   // of each row, or null: the row's place in its sequence (or start + row)
    size_t table_rows, start;
    int n_heads, hd, rot, half;  // half: pairs (i, i + rot/2), else (2i, 2i+1)
};
// q_out = turned q.  n_rows_dev (device) bounds the rows of a batch, n_rows the grid.
void launch_kv_append(const KvRopeArgs& a, const KvPages& p, th_dtype cache, const int* n_rows_dev, const KvRow* rows,
                      size_t n_rows, hipStream_t s);
void launch_rope_rows(const KvRopeArgs& a, size_t n_rows, hipStream_t s);

// grid: how many items the launch covers at a time (the kernels walk the rest; a launch has below 2^32 threads).
// flags: of the plan, or KV_BY_PLAN for a call that is captured.
constexpr size_t KV_LONG_ITEM = 16384;
constexpr size_t KV_MAX_BLOCKS = (size_t)1 << 23;
constexpr int KV_BY_PLAN = -1;
void launch_kv_attn_rows(const KvAttnArgs& a, th_dtype cache, size_t grid, hipStream_t s);
void launch_kv_attn_tiles(const KvAttnArgs& a, th_dtype cache, size_t grid, int flags, hipStream_t s);
void launch_kv_attn_both(const KvAttnArgs& a, th_dtype cache, size_t grid, int flags, hipStream_t s);
// n: tokens to join (captured: how many the launch covers at a time), room: entries that the list has memory for.
bool kv_join_many(size_t n, size_t n_recs, size_t n_heads);
void launch_kv_attn_join(const KvAttnArgs& a, const KvTok* list, size_t n, size_t room, int flags, hipStream_t s);

// Rows (tokens x query heads of a kv head) that one item has at most.
constexpr int KV_ROWS = 16, KV_TILE = 128;

// Makes the device current for a call and puts the caller's back.
struct DeviceScope {
    int was = -1;
    explicit DeviceScope(const th_device* d) {
        int cur = -1;
        TH_HIP(hipGetDevice(&cur));
        if (cur != d->ordinal) {
            TH_HIP(hipSetDevice(d->ordinal));
            was = cur;
        }
    }
    ~DeviceScope() {
        if (was >= 0) (void)hipSetDevice(was);
    }
    DeviceScope(const DeviceScope&) = delete;
};

}  // namespace th

// ---------------------------------------------------------------------------
// The objects behind the handles
// ---------------------------------------------------------------------------

// Pinned memory that uploads pass through, one behind the other; once it is left (busy), `done` says when it is free again.
struct th_kv_stage {
    void* host = nullptr;
    size_t bytes = 0, at = 0;
    hipEvent_t done = nullptr;
    bool busy = false;
};

struct th_kv_cache {
    th_device* dev = nullptr;
    th_dtype dtype = TH_F16;
    size_t n_layers = 0, n_kv_heads = 0, hd = 0, page_size = 0, n_pages = 0, max_seqs = 0, max_len = 0;
    int shift = 0;
    size_t pages_per_seq = 0, page_bytes = 0;  // page_bytes: one page of one layer's K (or V)
    char* pool = nullptr;                      // [layer][K, V][page]
    int* table = nullptr;                      // device [max_seqs][pages_per_seq]
    std::vector<int> mirror;                   // the same on the host
    struct Seq {
        bool used = false;
        size_t len = 0, n_pages = 0;
        // to upload: entries [dirty_from, dirty_to), if any (dirty_to > 0), and the first row_n, which are those of row_of's
        // row on the device
        size_t dirty_from = 0, dirty_to = 0, row_n = 0;
        int32_t row_of = 0;
        bool listed = false;  // in `dirty`
        uint64_t version = 0;  // changes whenever a batch begun on the sequence no longer fits it
    };
    std::vector<Seq> seqs;
    std::vector<int> refs;         // sequences that have the page
    std::vector<uint64_t> vacant;  // a bit for each page without any
    size_t n_vacant = 0, hint = 0;
    std::vector<int32_t> dirty;    // sequences with table entries to upload (room for all is there)
    uint64_t versions = 0;
    th_kv_stage stages[th::KV_STAGES];
    unsigned stage_at = 0;
    int live = 1;  // the handle, and the batches
    bool closed = false;
};

struct th_kv_batch {
    th_kv_cache* cache = nullptr;
    size_t max_seqs = 0, max_rows = 0, n_heads = 0;
    struct Step {
        std::vector<int> seqs;
        std::vector<size_t> start, n;
        std::vector<uint64_t> versions;
        size_t rows = 0, top = 0;  // new rows, and one past the highest position
    } step;
    bool begun = false;
    int* block = nullptr;      // device: the number of rows (16 bytes), then KvRow[max_rows]
    struct Plan {
        int* block = nullptr;  // device
        size_t n_rows_items = 0, n_tile_items = 0, n_joins = 0;
        int flags = 0;         // KvPlanHead::flags
        bool built = false;    // for the batch as it is begun
        std::vector<uint64_t> graphs;  // th_graph::id of those that may read it (and of some that are gone)
    };
    typedef std::pair<size_t, size_t> Key;  // window, sinks
    std::map<Key, Plan> plans;
    float* rec_o = nullptr;    // records of split work
    float2* rec_ml = nullptr;
    size_t max_recs = 0, max_items = 0;
};
