// The paged key/value cache: sequences and their pages, batches of new
// positions, and the plans of the attention over them.
//
// All of a cache's pages lie in one allocation; a sequence is a list of page
// numbers.  What is where is decided here, on the host, and handed to the
// kernels as tables: they never see a page number that was not checked.  Pages are
// shared by reference count (a fork copies nothing) and copied when a sequence
// that shares one writes to it.  The lowest vacant page goes first.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <memory>
#include <unordered_map>

#include "kvcache.hpp"

namespace th {

// ---------------------------------------------------------------------------
// Memory that kernels of a captured graph may name
// ---------------------------------------------------------------------------

static void free_drained(th_device* d, void* p) {
    if (!p) return;
    if (!d->closed && d->graphs > 0) d->retired.push_back(p);
    else (void)hipFree(p);
}

static void cache_release(th_kv_cache* c) {
    if (--c->live > 0) return;
    th_device* d = c->dev;
    device_drain(d);
    free_drained(d, c->pool);
    free_drained(d, c->table);
    for (th_kv_stage& s : c->stages) {
        if (s.host) (void)hipHostFree(s.host);
        if (s.done) (void)hipEventDestroy(s.done);
    }
    delete c;
    device_release(d);
}

static void require_open(const th_kv_cache* c, const char* what) {
    if (!c) throw Error(TH_ERR_INVALID, std::string(what) + ": null cache");
    if (c->closed) throw Error(TH_ERR_INVALID, std::string(what) + ": the cache was destroyed");
    if (c->dev->closed) throw Error(TH_ERR_INVALID, std::string(what) + ": the device was destroyed");
}

// Calls that change tables are made between replays, not recorded.
static void require_eager(const th_kv_cache* c, const char* what) {
    if (c->dev->capturing)
        throw Error(TH_ERR_INVALID, std::string(what) + ": changes the cache's tables and cannot be captured");
}

static th_kv_cache::Seq& the_seq(th_kv_cache* c, int32_t s, const char* what) {
    if (s < 0 || (size_t)s >= c->seqs.size() || !c->seqs[s].used)
        throw Error(TH_ERR_INVALID, std::string(what) + ": no sequence " + std::to_string(s));
    return c->seqs[s];
}

// ---------------------------------------------------------------------------
// Uploads
// ---------------------------------------------------------------------------

static void stage_alloc(th_kv_stage& st, size_t bytes) {
    void* host = nullptr;
    if (hipHostMalloc(&host, bytes, hipHostMallocDefault) != hipSuccess) {
        (void)hipGetLastError();
        throw Error(TH_ERR_OOM, "no pinned memory for uploads");
    }
    if (st.host) (void)hipHostFree(st.host);
    st.host = host;
    st.bytes = bytes;
}

// Room for a call's uploads: behind the last one's, or in the next stage when this one is full.  A stage's event is recorded
// once, when it is left (an event for each upload cost 1.5 us of a step's host time).
static char* stage(th_kv_cache* c, size_t bytes) {
    if (bytes == 0) return nullptr;
    th_kv_stage* st = &c->stages[c->stage_at];
    if (st->at + bytes > st->bytes) {
        if (st->at) {
            if (!st->done) TH_HIP(hipEventCreateWithFlags(&st->done, hipEventDisableTiming));
            TH_HIP(hipEventRecord(st->done, c->dev->stream));
            st->busy = true;
            c->stage_at = (c->stage_at + 1) % KV_STAGES;
            st = &c->stages[c->stage_at];
        }
        if (st->busy) TH_HIP(hipEventSynchronize(st->done));
        st->busy = false;
        st->at = 0;
        if (st->bytes < bytes) stage_alloc(*st, bytes + bytes / 2);
    }
    char* to = (char*)st->host + st->at;
    st->at += bytes;
    return to;
}

// Table entries of a sequence to upload: first and count.  (What it no longer has is read by nobody.)
static std::pair<size_t, size_t> changed(const th_kv_cache::Seq& q) {
    const size_t end = std::min(q.dirty_to, q.n_pages);
    return {q.dirty_from, end > q.dirty_from ? end - q.dirty_from : 0};
}

// How many of a fork's first entries the device copies from the row it was forked from.  That row holds them as long as
// nothing is uploaded; one that changes in this very upload is not read, and the entries go up like any others.
static size_t copied_row(const th_kv_cache* c, const th_kv_cache::Seq& q) {
    const size_t n = std::min(q.row_n, q.n_pages);
    if (n == 0) return 0;
    const th_kv_cache::Seq& o = c->seqs[q.row_of];
    return o.row_n > 0 || (o.dirty_to > 0 && o.dirty_from < n) ? 0 : n;
}

// What an upload of the table holds: copies of rows, and entries.
struct TableSize {
    size_t rows = 0, pairs = 0;
    size_t words() const { return 3 * rows + 2 * pairs; }
};
static TableSize table_size(const th_kv_cache* c) {
    TableSize t;
    for (const int32_t s : c->dirty) {
        const th_kv_cache::Seq& q = c->seqs[s];
        const size_t n = copied_row(c, q);
        t.rows += n > 0;
        t.pairs += changed(q).second + (n ? 0 : std::min(q.row_n, q.n_pages));
    }
    return t;
}

// Staging memory of an upload of so many words next to copies of pages: none where all fit a launch's arguments.
static size_t staged(size_t words, size_t n_copies = 0) { return 2 * n_copies + words > KV_ARG_WORDS ? round_up(words * 4, 16) : 0; }

// The table entries that changed, and `words` to the runs' places in dst, in stream order; and copies of pages
// ({from, to}, at most KV_ARG_COPIES) in the same launch.  room: staged() bytes, taken before (stage), and moved behind them.
static void upload(th_kv_cache* c, const uint32_t* words, const KvRuns& runs, void* dst, char*& room,
                   const std::vector<uint32_t>* copies = nullptr) {
    const size_t n_words = (size_t)runs.words(), n_copies = copies ? copies->size() / 2 : 0;
    const TableSize table = table_size(c);
    const size_t rows = table.rows, pairs = table.pairs, total = table.words() + n_words;
    if (total + n_copies == 0) return;
    KvWords w;
    if (n_copies) std::copy(copies->begin(), copies->end(), w.w);
    const size_t far = staged(total, n_copies);
    uint32_t *const from = far ? (uint32_t*)room : w.w + 2 * n_copies, *row = from, *to = from + 3 * rows;
    room += far;
    auto entries = [&](size_t at, size_t n) {
        for (size_t i = at; i < at + n; i++) {
            *to++ = (uint32_t)i;
            *to++ = (uint32_t)c->mirror[i];
        }
    };
    for (const int32_t s : c->dirty) {
        const th_kv_cache::Seq& q = c->seqs[s];
        const size_t at = (size_t)s * c->pages_per_seq;
        if (const size_t n = copied_row(c, q)) {
            *row++ = (uint32_t)(q.row_of * c->pages_per_seq);
            *row++ = (uint32_t)at;
            *row++ = (uint32_t)n;
        } else {
            entries(at, std::min(q.row_n, q.n_pages));
        }
        const auto d = changed(q);
        entries(at + d.first, d.second);
    }
    if (n_words) std::memcpy(to, words, n_words * 4);
    const KvTableWork work{far ? from : nullptr, (int)rows, (int)pairs, c->table};
    if (n_copies)
        launch_kv_copy_upload(c->pool, c->page_bytes, c->n_pages, (int)(2 * c->n_layers), w, n_copies, work, runs, (uint32_t*)dst,
                              c->dev->stream);
    else
        launch_kv_upload(w, work, runs, (uint32_t*)dst, c->dev->stream);
    for (const int32_t s : c->dirty) {
        th_kv_cache::Seq& q = c->seqs[s];
        q.dirty_from = q.dirty_to = q.row_n = 0;
        q.listed = false;
    }
    c->dirty.clear();
}

static KvRuns one_run(size_t n) {
    KvRuns r;
    r.n[0] = (int)n;
    return r;
}

// What a call sends: copies of pages ({from, to}), then the table and `words` as in upload.  The memory for it is taken first (here, as the
// tables stand), so that a call that finds none has sent nothing and can put back what it changed.
struct Sending {
    char* room = nullptr;
    uint32_t* pairs = nullptr;  // device: copies beyond those that a launch's arguments hold
};
// more: staging bytes of uploads behind these
static Sending prepare(th_kv_cache* c, const std::vector<uint32_t>& pairs, size_t n_words, size_t more = 0) {
    const size_t n = pairs.size() / 2, table = table_size(c).words();
    Sending to;
    if (n > KV_ARG_COPIES) to.pairs = (uint32_t*)device_scratch(c->dev, 8 * n);
    to.room = stage(c, (n > KV_ARG_COPIES ? staged(table + 2 * n) + staged(n_words) : staged(table + n_words, n)) + more);
    return to;
}
static void send(th_kv_cache* c, Sending& to, const std::vector<uint32_t>& pairs, const uint32_t* words, const KvRuns& runs, void* dst) {
    const size_t n = pairs.size() / 2;
    if (n <= KV_ARG_COPIES) {
        upload(c, words, runs, dst, to.room, &pairs);
        return;
    }
    upload(c, pairs.data(), one_run(2 * n), to.pairs, to.room);
    launch_kv_copy_pages(c->pool, c->page_bytes, c->n_pages, (int)(2 * c->n_layers), to.pairs, n, c->dev->stream);
    upload(c, words, runs, dst, to.room);
}

// ---------------------------------------------------------------------------
// Pages
// ---------------------------------------------------------------------------

static int take_page(th_kv_cache* c) {  // n_vacant > 0
    size_t w = c->hint;
    while (!c->vacant[w]) w++;
    c->hint = w;
    const int p = (int)(64 * w + __builtin_ctzll(c->vacant[w]));
    c->vacant[w] &= c->vacant[w] - 1;
    c->n_vacant--;
    c->refs[p] = 1;
    return p;
}

static void drop_page(th_kv_cache* c, int p) {
    if (--c->refs[p] > 0) return;
    c->vacant[p / 64] |= 1ull << (p % 64);
    c->n_vacant++;
    c->hint = std::min(c->hint, (size_t)p / 64);
}

static int* seq_table(th_kv_cache* c, int32_t s) { return c->mirror.data() + (size_t)s * c->pages_per_seq; }

static void list(th_kv_cache* c, int32_t s) {
    if (!c->seqs[s].listed) c->dirty.push_back(s);
    c->seqs[s].listed = true;
}

static void touch(th_kv_cache* c, int32_t s, size_t first, size_t n) {
    if (n == 0) return;
    th_kv_cache::Seq& q = c->seqs[s];
    list(c, s);
    size_t end = first + n;
    if (first < q.row_n) {  // the rest of a copied row goes up with the entries from here on
        end = std::max(end, q.row_n);
        q.row_n = first;
    }
    q.dirty_from = q.dirty_to ? std::min(q.dirty_from, first) : first;
    q.dirty_to = std::max(q.dirty_to, end);
}

// What growing a sequence to `len` takes: pages, and whether its last one has to be
// copied first (it is shared and will be written).
static bool must_copy(const th_kv_cache* c, int32_t s, size_t len) {
    const th_kv_cache::Seq& q = c->seqs[s];
    if (len <= q.len || q.len % c->page_size == 0) return false;
    return c->refs[c->mirror[(size_t)s * c->pages_per_seq + q.n_pages - 1]] > 1;
}

// Grows a sequence; the pages are there (counted before), and room in `copies`: nothing here fails.
static void grow(th_kv_cache* c, int32_t s, size_t len, std::vector<uint32_t>& copies) {
    th_kv_cache::Seq& q = c->seqs[s];
    int* t = seq_table(c, s);
    if (must_copy(c, s, len)) {
        const int old = t[q.n_pages - 1], fresh = take_page(c);
        copies.push_back((uint32_t)old);
        copies.push_back((uint32_t)fresh);
        drop_page(c, old);
        t[q.n_pages - 1] = fresh;
        touch(c, s, q.n_pages - 1, 1);
    }
    const size_t need = ceil_div(len, c->page_size), had = q.n_pages;
    while (q.n_pages < need) t[q.n_pages++] = take_page(c);
    touch(c, s, had, q.n_pages - had);
    q.len = len;
}

// A sequence as it was before it grew, and back to that, where the rest of the call found no memory.
struct SeqWas {
    size_t len, n_pages;
    uint64_t version;
    int last;  // page (-1: none)
};
static SeqWas seq_was(th_kv_cache* c, int32_t s) {
    const th_kv_cache::Seq& q = c->seqs[s];
    return {q.len, q.n_pages, q.version, q.n_pages ? seq_table(c, s)[q.n_pages - 1] : -1};
}
static void ungrow(th_kv_cache* c, int32_t s, const SeqWas& was) {
    th_kv_cache::Seq& q = c->seqs[s];
    int* t = seq_table(c, s);
    while (q.n_pages > was.n_pages) drop_page(c, t[--q.n_pages]);
    if (was.n_pages && t[was.n_pages - 1] != was.last) {
        drop_page(c, t[was.n_pages - 1]);
        t[was.n_pages - 1] = was.last;
        c->refs[was.last]++;
    }
    q.len = was.len;
    q.version = was.version;
}

static void shrink(th_kv_cache* c, int32_t s, size_t len) {
    th_kv_cache::Seq& q = c->seqs[s];
    int* t = seq_table(c, s);
    const size_t need = ceil_div(len, c->page_size);
    while (q.n_pages > need) drop_page(c, t[--q.n_pages]);
    q.len = len;
    q.version = ++c->versions;
}

static void no_pages(const char* what, size_t need, size_t have) {
    throw Error(TH_ERR_OOM, std::string(what) + ": " + std::to_string(need) + " pages needed, " + std::to_string(have) + " vacant");
}

static KvPages layer_pages(const th_kv_cache* c, size_t layer) {
    const size_t plane = c->n_pages * c->page_bytes;
    KvPages p;
    p.k = c->pool + 2 * layer * plane;
    p.v = c->pool + (2 * layer + 1) * plane;
    p.table = c->table;
    p.pages_per_seq = (int)c->pages_per_seq;
    p.shift = c->shift;
    p.n_kv_heads = (int)c->n_kv_heads;
    p.hd = (int)c->hd;
    return p;
}

// ---------------------------------------------------------------------------
// Attention plans
// ---------------------------------------------------------------------------

// A tile: tokens against a range of their sequence's numbers (KvItem), before splitting.
struct PlanTile { KvItem it; bool small, own; };

// Shared prefixes shorter than this are read by each sequence.
constexpr size_t KV_MIN_PREFIX = 128;
constexpr size_t KV_MAX_PLANS = 16;
// Least keys of a piece.  Rows items: two blocks for each of the four waves; one of them makes the join longer than the
// pieces get shorter (one row of 8192 keys, 32 heads of 128 on 8, four layers: 62 us, with 128 71, with 512 67,
// with 1024 83; 24 rows with a window of 1000: 22 us, with 512 25.5, unsplit 23.7).  Tiles: eight samples of a prompt
// of 992 take 32 us, with 512 40.
constexpr size_t KV_MIN_ROWS_KEYS = 256, KV_MIN_TILE_KEYS = 256;
constexpr size_t KV_ROWS_SHARE = 8;  // pieces of rows items a CU (PlanMaker::split)
constexpr size_t KV_LONG_PIECE = KV_LONG_ITEM * 4 / 5 / 64 * 64;

class PlanMaker {
   public:
    PlanMaker(const th_kv_batch* b, size_t window, size_t sinks)
        : b_(b), c_(b->cache), G_(b->n_heads / b->cache->n_kv_heads), window_(window), sinks_(sinks) {}

    void make() {
        order();
        // Pieces of one kind get longer, those that take more of what does not suffice.  Unsplit work fits: order() has seen to it.
        for (size_t scale[2] = {1, 1};;) {
            const int longer = split(scale);
            if (longer < 0) return;
            TH_REQUIRE(scale[longer] <= c_->max_len, "an unsplit plan exceeds its block");
            scale[longer] *= 2;
        }
    }

    std::vector<uint32_t> words;  // head, tokens, rows items, tile items, joined tokens
    int flags = 0;                // KvPlanHead::flags
    size_t n_toks = 0, n_items[2] = {0, 0}, n_joins = 0;  // items: [0] tiles, [1] rows

   private:
    const int* table(int s) const { return c_->mirror.data() + (size_t)s * c_->pages_per_seq; }

    // Sequences whose first KV_MIN_PREFIX positions are in the same pages, next to each other; the tokens in that order.  A group reads as
    // tiles what all its sequences have in common.  Tokens that share a prefix take two
    // records at least; they get three quarters of all, so that long sequences can be split whatever else is in the batch, and
    // sequences beyond that read the prefix by themselves.
    void order() {
        const size_t B = b_->step.seqs.size(), ps = c_->page_size;
        std::vector<size_t> row(B + 1, 0);
        for (size_t i = 0; i < B; i++) row[i + 1] = row[i] + b_->step.n[i];
        std::vector<std::vector<size_t>> groups;
        std::unordered_map<int, size_t> by_page;
        size_t left = b_->max_recs * 3 / 8;
        for (size_t i = 0; i < B; i++) {
            const size_t n = b_->step.n[i];
            if (n == 0) continue;
            // (the page that holds the last position of the shortest prefix: forks that have it in common have all before it, and
            // those that only share less belong to other groups)
            const bool can = b_->step.start[i] >= KV_MIN_PREFIX;
            const int first = can ? table(b_->step.seqs[i])[(KV_MIN_PREFIX - 1) / ps] : -1;
            if (can && c_->refs[first] > 1) {
                auto [at, fresh] = by_page.try_emplace(first, groups.size());
                if (!fresh) {
                    std::vector<size_t>& g = groups[at->second];
                    const size_t other = g.size() == 1 ? b_->step.n[g[0]] : 0;
                    if (n + other <= left) {
                        left -= n + other;
                        g.push_back(i);
                        continue;
                    }
                    if (n < other) at->second = groups.size();  // shorter ones may share with this one
                }
            }
            groups.push_back({i});
        }
        for (const auto& g : groups) {
            size_t common = 0;
            if (g.size() > 1) {
                common = b_->step.start[g[0]] / ps;
                const int* t0 = table(b_->step.seqs[g[0]]);
                for (size_t k = 1; k < g.size() && common; k++) {
                    const int* t = table(b_->step.seqs[g[k]]);
                    const size_t most = std::min(common, b_->step.start[g[k]] / ps);
                    common = (size_t)(std::mismatch(t, t + most, t0).first - t);
                }
                if (common * ps < KV_MIN_PREFIX) common = 0;
            }
            const size_t tok0 = toks_.size();
            for (size_t i : g)
                for (size_t j = 0; j < b_->step.n[i]; j++)
                    toks_.push_back(KvTok{(int)(row[i] + j), (int)(b_->step.start[i] + j), 0, 0});
            if (common) tile(tok0, toks_.size() - tok0, b_->step.seqs[g[0]], 0, common * ps, false);
            size_t at = tok0;
            for (size_t i : g) {
                tile(at, b_->step.n[i], b_->step.seqs[i], common * ps, b_->step.start[i] + b_->step.n[i], true);
                at += b_->step.n[i];
            }
        }
        keys_[0] = keys_[1] = 0;
        for (const PlanTile& t : tiles_) keys_[t.small] += (size_t)(t.it.j1 - t.it.j0);
    }

    // Tokens [tok0, tok0 + n) against keys [from, to) of a sequence.
    void tile(size_t tok0, size_t n, int seq, size_t from, size_t to, bool own) {
        const bool small = n * G_ <= KV_ROWS;
        const size_t per = small ? n : KV_TILE / G_;
        for (size_t k = 0; k < n; k += per) {
            const size_t m = std::min(per, n - k);
            int lo = toks_[tok0 + k].pos, hi = lo;
            for (size_t x = 1; x < m; x++) {
                lo = std::min(lo, toks_[tok0 + k + x].pos);
                hi = std::max(hi, toks_[tok0 + k + x].pos);
            }
            const size_t end = std::min(to, (size_t)hi + 1);
            size_t sink_end = end, main = end;  // hidden: [sink_end, main)
            if (window_ && (size_t)lo + 1 > window_) {
                // (the run begins and ends at multiples of 16: rows mask what is left of it)
                main = std::max(from, ((size_t)lo + 1 - window_) / 16 * 16);
                sink_end = std::max(from, round_up(std::min(sinks_, end), 16));
                if (sink_end >= std::min(main, end)) sink_end = main = end;
                main = std::min(main, end);
            }
            const size_t keys = sink_end - from + (end - main);
            if (end <= from || keys == 0) continue;
            KvItem it;
            it.tok0 = (int)(tok0 + k);
            it.ntok = (int)m;
            it.seq = seq;
            it.j0 = (int)from;
            it.j1 = (int)(from + keys);
            it.sink_end = (int)sink_end;
            it.gap = (int)(main - sink_end);
            it.rec = 0;
            tiles_.push_back(PlanTile{it, small, own});
        }
    }

    // Cuts the tiles into pieces.  -1: done; else the kind of items (0 tiles, 1 rows) whose pieces have to be longer.
    int split(const size_t (&scale)[2]) {
        const size_t kvh = c_->n_kv_heads, cus = (size_t)c_->dev->num_cus;
        // Keys of a piece.  The chip holds 2 * CUs workgroups at a time.  Rows items are a quarter of an even share, so
        // that uneven lengths level out.  Tiles are longer, since each of their pieces leaves 128 rows of
        // records: 1.5 pieces a CU (six ragged prompt chunks behind a window 49 us, 64 rows on a prefix
        // of 8192 99 us, 512 tokens beside 32 decode steps 146 us, 128 rows on a prefix of 16000 115 us; with 4 a CU 59 and
        // 112, with 2 54 and 109, with 1 59, 95, 138 and 126; the last two workloads on pages of zeros: 166 and 125 us on random values).
        size_t per[2];
        per[1] = round_up(std::max<size_t>(KV_MIN_ROWS_KEYS, ceil_div(keys_[1] * kvh, KV_ROWS_SHARE * cus)), 64) * scale[1];
        per[0] = round_up(std::max<size_t>(KV_MIN_TILE_KEYS, ceil_div(keys_[0] * kvh, cus * 3 / 2)), 64) * scale[0];
        // Where there are records for it, no tile's piece is so long that it needs additions of its own (a quarter
        // more than `per` is one piece).  A multiple of 64 like any other: pieces begin at blocks, and the last of many shall have keys left.
        if (scale[0] == 1) per[0] = std::min(per[0], KV_LONG_PIECE);
        std::vector<int> shared(toks_.size(), 0), own(toks_.size(), 0), pieces(tiles_.size());
        size_t extra[2] = {0, 0}, more[2] = {0, 0};  // items and records that splitting takes
        for (size_t i = 0; i < tiles_.size(); i++) {
            const PlanTile& t = tiles_[i];
            const size_t keys = (size_t)(t.it.j1 - t.it.j0), p = per[t.small];
            pieces[i] = (int)(keys <= p + p / 4 ? 1 : ceil_div(keys, p));
            extra[t.small] += (size_t)pieces[i] - 1;
            more[t.small] += ((size_t)pieces[i] - 1) * t.it.ntok;
            for (int k = 0; k < t.it.ntok; k++) (t.own ? own : shared)[t.it.tok0 + k] = pieces[i];
        }
        // The tokens of one tile have one count of records each kind, whatever tiles hold their other keys.
        size_t recs = 0;
        for (size_t i = 0; i < toks_.size(); i++) {
            if (shared[i] + own[i] <= 1) continue;
            recs += (size_t)(shared[i] + own[i]);
        }
        // tiles with a token that has records write records for all of theirs
        std::vector<char> recorded(toks_.size(), 0);
        for (const PlanTile& t : tiles_) {
            bool any = false;
            for (int k = 0; k < t.it.ntok; k++) any |= shared[t.it.tok0 + k] + own[t.it.tok0 + k] > 1;
            if (any)
                for (int k = 0; k < t.it.ntok; k++) {
                    const int x = t.it.tok0 + k;
                    if (!recorded[x] && shared[x] + own[x] == 1) recs++;
                    recorded[x] = 1;
                }
        }
        // (a token recorded through one tile has records in its other one: settled in a second look)
        for (bool again = true; again;) {
            again = false;
            for (const PlanTile& t : tiles_) {
                int any = 0;
                for (int k = 0; k < t.it.ntok; k++) any += recorded[t.it.tok0 + k];
                if (any == 0 || any == t.it.ntok) continue;
                for (int k = 0; k < t.it.ntok; k++) {
                    const int x = t.it.tok0 + k;
                    if (!recorded[x]) recs += (size_t)(shared[x] + own[x]);
                    recorded[x] = 1;
                }
                again = true;
            }
        }
        if (recs > b_->max_recs) return more[1] > more[0];
        if (tiles_.size() + extra[0] + extra[1] > b_->max_items) return extra[1] > extra[0];
        size_t rec = 0;
        std::vector<KvTok> joins;
        for (size_t i = 0; i < toks_.size(); i++) {
            KvTok& t = toks_[i];
            t.rec = (int)rec;
            t.own_n = shared[i] | (shared[i] + own[i]) << 16;
            if (!recorded[i]) continue;
            rec += (size_t)(shared[i] + own[i]);
            joins.push_back(t);
        }
        std::vector<KvItem> items[2];
        for (size_t i = 0; i < tiles_.size(); i++) {
            const PlanTile& t = tiles_[i];
            const bool direct = !recorded[t.it.tok0];
            const size_t keys = (size_t)(t.it.j1 - t.it.j0), block = t.small ? 32 : 64;
            const size_t chunk = round_up(ceil_div(keys, (size_t)pieces[i]), block);
            for (int s = 0; s < pieces[i]; s++) {
                KvItem it = t.it;
                it.j0 = (int)std::min((size_t)t.it.j1, t.it.j0 + s * chunk);
                it.j1 = (int)std::min((size_t)t.it.j1, t.it.j0 + (s + 1) * chunk);
                it.rec = direct ? -1 : s | (t.own ? KV_REC_OWN : 0);
                items[t.small].push_back(it);
            }
        }
        // the longest first: the last workgroups to start are short
        for (auto& v : items)
            std::stable_sort(v.begin(), v.end(), [](const KvItem& x, const KvItem& y) { return x.j1 - x.j0 > y.j1 - y.j0; });
        if (!items[0].empty() && (size_t)(items[0][0].j1 - items[0][0].j0) > KV_LONG_ITEM) flags |= KV_PLAN_FAR;
        if (kv_join_many(joins.size(), rec, b_->n_heads)) flags |= KV_PLAN_MANY;
        n_toks = toks_.size();
        n_items[0] = items[0].size();
        n_items[1] = items[1].size();
        n_joins = joins.size();
        KvPlanHead head = {};
        head.flags = flags;
        head.n_joins = (int)n_joins;
        head.n_rows_items = (int)n_items[1];
        head.n_tile_items = (int)n_items[0];
        words.resize(KV_HEAD_WORDS + n_toks * sizeof(KvTok) / 4 + (n_items[0] + n_items[1]) * sizeof(KvItem) / 4 + n_joins * sizeof(KvTok) / 4);
        uint32_t* to = words.data();
        auto put = [&](const void* p, size_t bytes) {
            if (bytes) std::memcpy(to, p, bytes);
            to += bytes / 4;
        };
        put(&head, sizeof(head));
        put(toks_.data(), n_toks * sizeof(KvTok));
        put(items[1].data(), n_items[1] * sizeof(KvItem));
        put(items[0].data(), n_items[0] * sizeof(KvItem));
        put(joins.data(), n_joins * sizeof(KvTok));
        return -1;
    }

    const th_kv_batch* b_;
    const th_kv_cache* c_;
    size_t G_, window_, sinks_;
    std::vector<KvTok> toks_;
    std::vector<PlanTile> tiles_;
    size_t keys_[2] = {0, 0};
};

// Where a plan's parts are, in words.
static size_t plan_toks(const th_kv_batch*) { return KV_HEAD_WORDS; }
static size_t plan_rows(const th_kv_batch* b) { return plan_toks(b) + b->max_rows * sizeof(KvTok) / 4; }
static size_t plan_tiles(const th_kv_batch* b) { return plan_rows(b) + b->max_items * sizeof(KvItem) / 4; }
static size_t plan_joins(const th_kv_batch* b) { return plan_tiles(b) + b->max_items * sizeof(KvItem) / 4; }
static size_t plan_words(const th_kv_batch* b) { return plan_joins(b) + b->max_rows * sizeof(KvTok) / 4; }

static KvRuns plan_runs(const th_kv_batch* b, const PlanMaker& m) {
    KvRuns runs;
    runs.n[0] = KV_HEAD_WORDS;
    runs.n[1] = (int)(m.n_toks * sizeof(KvTok) / 4);
    runs.at[1] = (int)plan_toks(b);
    runs.n[2] = (int)(m.n_items[1] * sizeof(KvItem) / 4);
    runs.at[2] = (int)plan_rows(b);
    runs.n[3] = (int)(m.n_items[0] * sizeof(KvItem) / 4);
    runs.at[3] = (int)plan_tiles(b);
    runs.n[4] = (int)(m.n_joins * sizeof(KvTok) / 4);
    runs.at[4] = (int)plan_joins(b);
    TH_REQUIRE(m.n_items[0] <= b->max_items && m.n_items[1] <= b->max_items, "attention plan exceeds its block");
    return runs;
}

static void send_plan(th_kv_batch* b, const PlanMaker& m, const KvRuns& runs, th_kv_batch::Plan& p, char*& room) {
    upload(b->cache, m.words.data(), runs, p.block, room);
    p.n_tile_items = m.n_items[0];
    p.n_rows_items = m.n_items[1];
    p.n_joins = m.n_joins;
    p.flags = m.flags;
    p.built = true;
}

static void build_plan(th_kv_batch* b, const th_kv_batch::Key& key, th_kv_batch::Plan& p) {
    PlanMaker m(b, key.first, key.second);
    m.make();
    const KvRuns runs = plan_runs(b, m);
    char* room = stage(b->cache, staged(table_size(b->cache).words() + m.words.size()));
    send_plan(b, m, runs, p, room);
}

// Whether a graph that is still there may read the plan.
static bool captured(const th_device* d, th_kv_batch::Plan& p) {
    auto gone = [&](uint64_t id) { return std::find(d->graph_ids.begin(), d->graph_ids.end(), id) == d->graph_ids.end(); };
    p.graphs.erase(std::remove_if(p.graphs.begin(), p.graphs.end(), gone), p.graphs.end());
    return !p.graphs.empty();
}

// Room for another plan: of its own, or, where there are KV_MAX_PLANS that no graph reads, that of one of them (uploads
// are in stream order, behind the calls that read the old plan).
static std::map<th_kv_batch::Key, th_kv_batch::Plan>::iterator add_plan(th_kv_batch* b, const th_kv_batch::Key& key) {
    th_device* d = b->cache->dev;
    th_kv_batch::Plan p;
    size_t spare = 0;
    for (auto& x : b->plans) spare += !captured(d, x.second);
    for (auto at = b->plans.begin(); at != b->plans.end() && spare >= KV_MAX_PLANS;) {
        if (!at->second.graphs.empty()) {
            ++at;
            continue;
        }
        if (p.block) {  // left by graphs that are gone
            device_drain(d);
            free_drained(d, p.block);
        }
        p.block = at->second.block;
        at = b->plans.erase(at);
        spare--;
    }
    if (!p.block) {
        const hipError_t e = hipMalloc((void**)&p.block, plan_words(b) * 4);
        if (e != hipSuccess) {
            (void)hipGetLastError();
            throw Error(e == hipErrorOutOfMemory ? TH_ERR_OOM : TH_ERR_HIP, "no memory for an attention plan");
        }
    }
    return b->plans.emplace(key, p).first;
}

// The batch as it was begun, and still so.
static void require_begun(const th_kv_batch* b, size_t layer, const char* what) {
    if (!b) throw Error(TH_ERR_INVALID, std::string(what) + ": null batch");
    require_open(b->cache, what);
    const th_kv_cache* c = b->cache;
    if (!b->begun) throw Error(TH_ERR_INVALID, std::string(what) + ": the batch has not begun");
    if (layer >= c->n_layers) throw Error(TH_ERR_INVALID, std::string(what) + ": no layer " + std::to_string(layer));
    for (size_t i = 0; i < b->step.seqs.size(); i++)
        if (!c->seqs[b->step.seqs[i]].used || c->seqs[b->step.seqs[i]].version != b->step.versions[i])
            throw Error(TH_ERR_INVALID, std::string(what) + ": sequence " + std::to_string(b->step.seqs[i]) +
                                            " has changed since the batch began");
}

static void require_x(const th_kv_cache* c, const th_buffer* b, size_t n, const char* what) {
    require_len_any(b, n, what);
    if (b->dtype != TH_F32 && b->dtype != TH_F16 && b->dtype != TH_BF16)
        throw Error(TH_ERR_INVALID, std::string("buffer ") + what + " must be f32, f16 or bf16");
    if (b->dev != c->dev) throw Error(TH_ERR_INVALID, std::string("buffer ") + what + " is on another device handle");
}

// Tables, pairs and positions of a rotary call, checked.  out: what it writes, which other threads' tables must not be.
static void rope_args(KvRopeArgs& a, const th_device* dev, const th_buffer* cos_t, const th_buffer* sin_t, const th_buffer* positions,
                      size_t rows, size_t hd, size_t rot, int layout, size_t top, const th_buffer* out) {
    TH_REQUIRE(!out || (out != cos_t && out != sin_t), "the result must not be a table");
    TH_REQUIRE(rot % 2 == 0 && rot <= hd, "rot_dim must be even and at most head_dim");
    TH_REQUIRE(layout == TH_ROPE_INTERLEAVED || layout == TH_ROPE_HALF, "unknown pair layout");
    a.rot = (int)rot;
    a.half = layout == TH_ROPE_HALF;
    a.cos_t = a.sin_t = nullptr;
    a.positions = nullptr;
    a.table_rows = 0;
    if (positions) {
        require_len(positions, TH_U32, rows, "positions");
        TH_REQUIRE(positions->dev == dev, "buffer positions is on another device handle");
        a.positions = (const uint32_t*)positions->ptr;
    }
    if (rot == 0) return;
    TH_REQUIRE(cos_t && sin_t, "null table");
    require_len(cos_t, TH_F32, 0, "cos table");
    require_len(sin_t, TH_F32, 0, "sin table");
    TH_REQUIRE(cos_t->dev == dev && sin_t->dev == dev, "a table is on another device handle");
    a.table_rows = std::min(cos_t->n, sin_t->n) / (rot / 2);
    TH_REQUIRE(positions || top <= a.table_rows, "the tables end before the last position");
    a.cos_t = (const float*)cos_t->ptr;
    a.sin_t = (const float*)sin_t->ptr;
    TH_REQUIRE(a.table_rows > 0 || rows == 0, "empty tables");
}

// Weights of the heads' norms, checked (null: ones).  hd: dims of a head.
static void norm_args(KvRopeArgs& a, const th_device* dev, const th_buffer* qw, const th_buffer* kw, float eps, size_t hd) {
    TH_REQUIRE(std::isfinite(eps) && eps >= 0.0f, "eps must be finite and not negative");
    for (const th_buffer* w : {qw, kw}) {
        if (!w) continue;
        require_len_any(w, hd, "weight");
        TH_REQUIRE(w->dtype == TH_F32 || w->dtype == TH_BF16, "weights must be f32 or bf16");
        TH_REQUIRE(w->dev == dev, "a weight is on another device handle");
    }
    a.norm = true;
    a.eps = eps;
    a.qw = qw ? qw->ptr : nullptr;
    a.kw = kw ? kw->ptr : nullptr;
    a.qw_bf16 = qw && qw->dtype == TH_BF16;
    a.kw_bf16 = kw && kw->dtype == TH_BF16;
}
// What a launch writes must not be what its other threads read.
static void require_apart(const th_buffer* out, std::initializer_list<const th_buffer*> in, const char* what) {
    for (const th_buffer* b : in)
        if (b && b == out) throw Error(TH_ERR_INVALID, std::string("buffer ") + what + " is also an input that others read");
}

}  // namespace th

using namespace th;

extern "C" {

int th_kv_cache_create(th_device* dev, const th_kv_cache_config* cfg, th_kv_cache** out) {
    TH_API_BEGIN
    TH_REQUIRE(dev && cfg && out, "null argument");
    TH_REQUIRE(!dev->closed, "the device was destroyed");
    TH_REQUIRE(!dev->capturing, "a cache cannot be made while work is captured");
    TH_REQUIRE(cfg->n_layers > 0 && cfg->n_kv_heads > 0 && cfg->head_dim > 0 && cfg->n_pages > 0 && cfg->max_seqs > 0 && cfg->max_len > 0,
               "every size must be positive");
    TH_REQUIRE(cfg->page_size >= 16 && cfg->page_size <= 1024 && (cfg->page_size & (cfg->page_size - 1)) == 0,
               "page_size must be a power of two from 16 to 1024");
    if (cfg->dtype != TH_F16 && cfg->dtype != TH_BF16)
        throw Error(TH_ERR_UNSUPPORTED, "th_kv_cache_create: the cache holds f16 or bf16");
    if (cfg->head_dim % 8 != 0 || cfg->head_dim > 256)
        throw Error(TH_ERR_UNSUPPORTED, "th_kv_cache_create: head_dim must be a multiple of 8, at most 256");
    TH_REQUIRE(cfg->n_layers <= 16384 && cfg->n_kv_heads <= 1024 && cfg->max_seqs <= 65536, "too many layers, heads or sequences");
    TH_REQUIRE(cfg->max_len <= (size_t)1 << 28, "max_len above 2^28");
    TH_REQUIRE(cfg->n_pages <= (size_t)1 << 30 && cfg->n_pages * cfg->n_kv_heads * cfg->page_size < (size_t)1 << 32,
               "rows of a layer exceed 2^32");
    DeviceScope scope(dev);
    std::unique_ptr<th_kv_cache> c(new th_kv_cache());
    c->dev = dev;
    c->dtype = cfg->dtype;
    c->n_layers = cfg->n_layers;
    c->n_kv_heads = cfg->n_kv_heads;
    c->hd = cfg->head_dim;
    c->page_size = cfg->page_size;
    c->shift = __builtin_ctzll(cfg->page_size);
    c->n_pages = cfg->n_pages;
    c->max_seqs = cfg->max_seqs;
    c->max_len = cfg->max_len;
    c->pages_per_seq = std::min(ceil_div(cfg->max_len, cfg->page_size), cfg->n_pages);
    TH_REQUIRE(c->max_seqs * c->pages_per_seq < (size_t)1 << 29, "page tables exceed 2^29 entries");
    c->page_bytes = c->n_kv_heads * c->page_size * c->hd * 2;
    c->mirror.assign(c->max_seqs * c->pages_per_seq, 0);
    c->seqs.resize(c->max_seqs);
    c->dirty.reserve(c->max_seqs);
    c->refs.assign(c->n_pages, 0);
    c->vacant.assign(ceil_div(c->n_pages, 64), ~0ull);
    if (c->n_pages % 64) c->vacant.back() = (1ull << (c->n_pages % 64)) - 1;
    c->n_vacant = c->n_pages;
    const size_t bytes = 2 * c->n_layers * c->n_pages * c->page_bytes;
    try {
        TH_HIP(hipMalloc((void**)&c->pool, bytes));
        TH_HIP(hipMalloc((void**)&c->table, c->mirror.size() * 4));
        TH_HIP(hipMemset(c->table, 0, c->mirror.size() * 4));
        TH_HIP(hipMemset(c->pool, 0, bytes));
        TH_HIP(hipDeviceSynchronize());
        for (th_kv_stage& st : c->stages) stage_alloc(st, (size_t)64 << 10);
    } catch (...) {
        for (th_kv_stage& st : c->stages)
            if (st.host) (void)hipHostFree(st.host);
        if (c->pool) (void)hipFree(c->pool);
        if (c->table) (void)hipFree(c->table);
        (void)hipGetLastError();  // the next launch's check must not find it
        throw;
    }
    device_retain(dev);
    *out = c.release();
    TH_API_END
}

int th_kv_cache_destroy(th_kv_cache* c) {
    TH_API_BEGIN
    if (!c) return TH_OK;
    TH_REQUIRE(!c->closed, "the cache was destroyed already");
    c->closed = true;
    cache_release(c);
    TH_API_END
}

int th_kv_cache_info(const th_kv_cache* c, size_t* pages_vacant, size_t* seqs_vacant) {
    TH_API_BEGIN
    require_open(c, __func__);
    if (pages_vacant) *pages_vacant = c->n_vacant;
    if (seqs_vacant) *seqs_vacant = (size_t)std::count_if(c->seqs.begin(), c->seqs.end(), [](const th_kv_cache::Seq& q) { return !q.used; });
    TH_API_END
}

int th_kv_cache_pages(th_kv_cache* c, size_t layer, void** k, void** v) {
    TH_API_BEGIN
    require_open(c, __func__);
    TH_REQUIRE(layer < c->n_layers, "no such layer");
    const KvPages p = layer_pages(c, layer);
    if (k) *k = const_cast<void*>(p.k);
    if (v) *v = const_cast<void*>(p.v);
    TH_API_END
}

int th_kv_cache_compact(th_kv_cache* c, size_t* n_moved) {
    TH_API_BEGIN
    require_open(c, __func__);
    require_eager(c, __func__);
    DeviceScope scope(c->dev);
    // Pages above the live ones' count move into the holes below it: no page is both
    // read and written, so one launch moves all.
    const size_t live = c->n_pages - c->n_vacant;
    std::vector<int> moved(c->n_pages, -1);
    std::vector<uint32_t> pairs;
    size_t hole = 0;
    for (size_t p = live; p < c->n_pages; p++) {
        if (c->refs[p] == 0) continue;
        while (c->refs[hole] > 0) hole++;
        pairs.push_back((uint32_t)p);
        pairs.push_back((uint32_t)hole++);
    }
    if (!pairs.empty()) {
        std::vector<uint64_t> versions(c->seqs.size());
        for (size_t s = 0; s < c->seqs.size(); s++) versions[s] = c->seqs[s].version;
        // moves pages in the books: those of `pairs` from their item `from` to the other
        auto move = [&](int from) {
            for (size_t i = 0; i < pairs.size(); i += 2) {
                const int a = (int)pairs[i + from], z = (int)pairs[i + 1 - from];
                c->refs[z] = c->refs[a];
                c->refs[a] = 0;
                c->vacant[a / 64] |= 1ull << (a % 64);
                c->vacant[z / 64] &= ~(1ull << (z % 64));
                moved[a] = z;
            }
            c->hint = 0;
            for (size_t s = 0; s < c->seqs.size(); s++) {
                if (!c->seqs[s].used) continue;
                int* t = seq_table(c, (int32_t)s);
                bool any = false;
                for (size_t i = 0; i < c->seqs[s].n_pages; i++) {
                    if (moved[t[i]] < 0) continue;
                    t[i] = moved[t[i]];
                    touch(c, (int32_t)s, i, 1);
                    any = true;
                }
                if (any) c->seqs[s].version = from ? versions[s] : ++c->versions;
            }
            for (size_t i = 0; i < pairs.size(); i += 2) moved[pairs[i + from]] = -1;
        };
        move(0);
        Sending to;
        try {
            to = prepare(c, pairs, 0);
        } catch (...) {
            move(1);
            throw;
        }
        send(c, to, pairs, nullptr, KvRuns(), nullptr);
    }
    if (n_moved) *n_moved = pairs.size() / 2;
    TH_API_END
}

int th_kv_seq_create(th_kv_cache* c, size_t n, int32_t* seqs) {
    TH_API_BEGIN
    require_open(c, __func__);
    TH_REQUIRE(seqs || n == 0, "null argument");
    std::vector<int32_t> got;
    for (size_t s = 0; s < c->seqs.size() && got.size() < n; s++)
        if (!c->seqs[s].used) got.push_back((int32_t)s);
    if (got.size() < n) throw Error(TH_ERR_OOM, "th_kv_seq_create: no sequence is vacant");
    for (size_t i = 0; i < n; i++) {
        th_kv_cache::Seq& q = c->seqs[got[i]];
        q.used = true;
        q.len = q.n_pages = 0;
        q.dirty_from = q.dirty_to = q.row_n = 0;
        q.version = ++c->versions;
        seqs[i] = got[i];
    }
    TH_API_END
}

int th_kv_seq_free(th_kv_cache* c, const int32_t* seqs, size_t n) {
    TH_API_BEGIN
    require_open(c, __func__);
    TH_REQUIRE(seqs || n == 0, "null argument");
    std::vector<char> seen(c->seqs.size(), 0);
    for (size_t i = 0; i < n; i++) {
        the_seq(c, seqs[i], __func__);
        TH_REQUIRE(!seen[seqs[i]], "a sequence twice");
        seen[seqs[i]] = 1;
    }
    for (size_t i = 0; i < n; i++) {
        shrink(c, seqs[i], 0);
        c->seqs[seqs[i]].used = false;
    }
    TH_API_END
}

int th_kv_seq_len(const th_kv_cache* c, int32_t seq, size_t* len) {
    TH_API_BEGIN
    require_open(c, __func__);
    TH_REQUIRE(len, "null argument");
    *len = the_seq(const_cast<th_kv_cache*>(c), seq, __func__).len;
    TH_API_END
}

int th_kv_seq_resize(th_kv_cache* c, int32_t seq, size_t len) {
    TH_API_BEGIN
    require_open(c, __func__);
    const th_kv_cache::Seq& q = the_seq(c, seq, __func__);
    TH_REQUIRE(len <= c->max_len, "longer than max_len");
    if (len <= q.len) {
        if (len < q.len) shrink(c, seq, len);
        return TH_OK;
    }
    require_eager(c, __func__);
    DeviceScope scope(c->dev);
    const size_t need = ceil_div(len, c->page_size) - q.n_pages + (must_copy(c, seq, len) ? 1 : 0);
    if (need > c->n_vacant) no_pages(__func__, need, c->n_vacant);
    std::vector<uint32_t> copies;
    copies.reserve(2);
    const SeqWas was = seq_was(c, seq);
    grow(c, seq, len, copies);
    c->seqs[seq].version = ++c->versions;
    if (!copies.empty()) {
        Sending to;
        try {
            to = prepare(c, copies, 0);
        } catch (...) {
            ungrow(c, seq, was);
            throw;
        }
        send(c, to, copies, nullptr, KvRuns(), nullptr);
    }
    TH_API_END
}

int th_kv_seq_fork(th_kv_cache* c, int32_t seq, size_t len, size_t n, int32_t* children) {
    TH_API_BEGIN
    require_open(c, __func__);
    TH_REQUIRE(children || n == 0, "null argument");
    const size_t had = the_seq(c, seq, __func__).len;
    TH_REQUIRE(len <= had, "longer than the sequence");
    check_status(th_kv_seq_create(c, n, children));
    const size_t pages = ceil_div(len, c->page_size);
    const int* from = seq_table(c, seq);
    const bool row = c->seqs[seq].row_n == 0 && c->seqs[seq].dirty_to == 0;  // the device has the parent's row
    for (size_t i = 0; i < n; i++) {
        th_kv_cache::Seq& q = c->seqs[children[i]];
        std::copy(from, from + pages, seq_table(c, children[i]));
        q.len = len;
        q.n_pages = pages;
        if (row && pages) {
            q.row_of = seq;
            q.row_n = pages;
            list(c, children[i]);
        } else {
            touch(c, children[i], 0, pages);
        }
    }
    for (size_t p = 0; p < pages; p++) c->refs[from[p]] += (int)n;
    TH_API_END
}

int th_kv_seq_select(th_kv_cache* c, int32_t seq, const uint32_t* positions, size_t n) {
    TH_API_BEGIN
    require_open(c, __func__);
    require_eager(c, __func__);
    const size_t had = the_seq(c, seq, __func__).len;
    TH_REQUIRE(positions || n == 0, "null argument");
    TH_REQUIRE(n <= c->max_len, "longer than max_len");
    for (size_t i = 0; i < n; i++) TH_REQUIRE(positions[i] < had, "position behind the sequence's end");
    const size_t pages = ceil_div(n, c->page_size);
    if (pages > c->n_vacant) no_pages(__func__, pages, c->n_vacant);
    DeviceScope scope(c->dev);
    int* t = seq_table(c, seq);
    std::vector<uint32_t> w(n + pages);
    for (size_t i = 0; i < n; i++)
        w[i] = (uint32_t)(((size_t)t[positions[i] >> c->shift] << c->shift) + (positions[i] & (c->page_size - 1)));
    // the rows go to pages of their own: the old ones may be shared, and order is free
    th_kv_cache::Seq& q = c->seqs[seq];
    const SeqWas was = seq_was(c, seq);
    const std::vector<int> old(t, t + q.n_pages);
    auto put = [&](size_t len, size_t n_pages, uint64_t version) {
        q.len = len;
        q.n_pages = n_pages;
        q.version = version;
        touch(c, seq, 0, n_pages);
    };
    for (size_t p = 0; p < pages; p++) w[n + p] = (uint32_t)(t[p] = take_page(c));
    put(n, pages, ++c->versions);
    uint32_t* dev = nullptr;
    char* room = nullptr;
    try {
        if (n) {
            dev = (uint32_t*)device_scratch(c->dev, w.size() * 4);
            room = stage(c, staged(table_size(c).words() + w.size()));
        }
    } catch (...) {
        for (size_t p = 0; p < pages; p++) drop_page(c, t[p]);
        std::copy(old.begin(), old.end(), t);
        put(was.len, was.n_pages, was.version);
        throw;
    }
    for (const int p : old) drop_page(c, p);
    if (n) {
        upload(c, w.data(), one_run(w.size()), dev, room);
        launch_kv_gather_rows(c->pool, c->n_pages, (int)(2 * c->n_layers), (int)c->n_kv_heads, c->shift, c->hd * 2, dev, dev + n, n,
                              c->dev->stream);
    }
    TH_API_END
}

int th_kv_seq_read(th_kv_cache* c, int32_t seq, size_t layer, size_t from, size_t n, th_buffer* k, th_buffer* v) {
    TH_API_BEGIN
    require_open(c, __func__);
    const size_t len = the_seq(c, seq, __func__).len;
    TH_REQUIRE(k && v, "null argument");
    TH_REQUIRE(layer < c->n_layers, "no such layer");
    TH_REQUIRE(from <= len && n <= len - from, "positions behind the sequence's end");
    require_len(k, c->dtype, n * c->n_kv_heads * c->hd, "k");
    require_len(v, c->dtype, n * c->n_kv_heads * c->hd, "v");
    TH_REQUIRE(k->dev == c->dev && v->dev == c->dev, "a buffer is on another device handle");
    TH_REQUIRE(k != v, "k and v must be two buffers");
    DeviceScope scope(c->dev);
    if (!c->dirty.empty()) {
        require_eager(c, __func__);
        char* room = stage(c, staged(table_size(c).words()));
        upload(c, nullptr, KvRuns(), nullptr, room);
    }
    launch_kv_read(layer_pages(c, layer), seq, from, n, c->hd * 2, k->ptr, v->ptr, c->dev->stream);
    TH_API_END
}

int th_kv_batch_create(th_kv_cache* c, size_t max_seqs, size_t max_rows, size_t n_heads, th_kv_batch** out) {
    TH_API_BEGIN
    require_open(c, __func__);
    TH_REQUIRE(out, "null argument");
    TH_REQUIRE(!c->dev->capturing, "a batch cannot be made while work is captured");
    TH_REQUIRE(max_seqs > 0 && max_seqs <= c->max_seqs, "max_seqs must be from 1 to the cache's");
    TH_REQUIRE(max_rows > 0 && max_rows <= (size_t)1 << 24, "max_rows must be from 1 to 2^24");
    TH_REQUIRE(n_heads > 0 && n_heads % c->n_kv_heads == 0, "n_heads must be a multiple of the cache's kv heads");
    TH_REQUIRE(n_heads / c->n_kv_heads <= KV_TILE, "more than 128 query heads to a kv head");
    DeviceScope scope(c->dev);
    std::unique_ptr<th_kv_batch> b(new th_kv_batch());
    b->cache = c;
    b->max_seqs = max_seqs;
    b->max_rows = max_rows;
    b->n_heads = n_heads;
    // Pieces of attention work that a plan may have, and the records of tokens whose work
    // is split (a plan that would need more splits less), 1 GiB of them at most.
    const size_t G = n_heads / c->n_kv_heads;
    b->max_recs = std::max<size_t>(64, std::min<size_t>(8192, ((size_t)1 << 30) / (n_heads * c->hd * 4)));
    // ... and no more than max_rows tokens can have: a piece of each of a token's two ranges of keys at most by length, and by the chip's share
    const size_t by_len = c->max_len / std::min(KV_MIN_ROWS_KEYS, KV_MIN_TILE_KEYS) + 2;
    const size_t by_share = 2 * (KV_ROWS_SHARE * (size_t)c->dev->num_cus / c->n_kv_heads + 2) + c->max_len / KV_LONG_PIECE + 2;
    b->max_recs = std::min(b->max_recs, std::max<size_t>(4, std::min(by_len, by_share)) * max_rows);
    b->max_items = 2 * (max_seqs + ceil_div(max_rows, std::max<size_t>(1, KV_TILE / G))) + 4096;
    try {
        TH_HIP(hipMalloc((void**)&b->block, 16 + max_rows * sizeof(KvRow)));
        TH_HIP(hipMalloc((void**)&b->rec_o, b->max_recs * n_heads * c->hd * 4));
        TH_HIP(hipMalloc((void**)&b->rec_ml, b->max_recs * n_heads * 8));
    } catch (...) {
        for (void* p : {(void*)b->block, (void*)b->rec_o, (void*)b->rec_ml})
            if (p) (void)hipFree(p);
        (void)hipGetLastError();
        throw;
    }
    c->live++;
    *out = b.release();
    TH_API_END
}

int th_kv_batch_destroy(th_kv_batch* b) {
    TH_API_BEGIN
    if (!b) return TH_OK;
    th_device* d = b->cache->dev;
    device_drain(d);
    free_drained(d, b->block);
    free_drained(d, b->rec_o);
    free_drained(d, b->rec_ml);
    for (auto& p : b->plans) free_drained(d, p.second.block);
    th_kv_cache* c = b->cache;
    delete b;
    cache_release(c);
    TH_API_END
}

int th_kv_batch_begin(th_kv_batch* b, const int32_t* seqs, const uint32_t* n_new, size_t n) {
    TH_API_BEGIN
    TH_REQUIRE(b, "null batch");
    th_kv_cache* c = b->cache;
    require_open(c, __func__);
    require_eager(c, __func__);
    TH_REQUIRE((seqs && n_new) || n == 0, "null argument");
    TH_REQUIRE(n <= b->max_seqs, "more sequences than max_seqs");
    size_t rows = 0, need = 0;
    std::unordered_map<int, int> copied;  // a shared last page goes to its last holder without a copy
    std::vector<char> seen(c->seqs.size(), 0);
    for (size_t i = 0; i < n; i++) {
        const th_kv_cache::Seq& q = the_seq(c, seqs[i], __func__);
        TH_REQUIRE(!seen[seqs[i]], "a sequence twice");
        seen[seqs[i]] = 1;
        TH_REQUIRE(n_new[i] <= c->max_len && q.len + n_new[i] <= c->max_len, "a sequence longer than max_len");
        rows += n_new[i];
        need += ceil_div(q.len + n_new[i], c->page_size) - q.n_pages;
        if (must_copy(c, seqs[i], q.len + n_new[i])) {
            const int page = seq_table(c, seqs[i])[q.n_pages - 1];
            if (++copied[page] < c->refs[page]) need++;
        }
    }
    TH_REQUIRE(rows <= b->max_rows, "more new positions than max_rows");
    if (need > c->n_vacant) no_pages(__func__, need, c->n_vacant);
    DeviceScope scope(c->dev);
    std::vector<uint32_t> copies, words(4 + rows * sizeof(KvRow) / 4);
    copies.reserve(2 * n);
    words[0] = (uint32_t)rows;
    th_kv_batch::Step step;
    step.seqs.assign(seqs, seqs + n);
    step.n.assign(n_new, n_new + n);
    step.start.resize(n);
    step.versions.resize(n);
    step.rows = rows;
    std::vector<SeqWas> was(n);
    size_t at = 4;
    for (size_t i = 0; i < n; i++) {
        th_kv_cache::Seq& q = c->seqs[seqs[i]];
        was[i] = seq_was(c, seqs[i]);
        step.start[i] = q.len;
        if (n_new[i]) {
            grow(c, seqs[i], q.len + n_new[i], copies);
            q.version = ++c->versions;
            step.top = std::max(step.top, q.len);
        }
        step.versions[i] = q.version;
        for (size_t j = 0; j < n_new[i]; j++) {
            words[at++] = (uint32_t)seqs[i];
            words[at++] = (uint32_t)(step.start[i] + j);
        }
    }
    std::swap(b->step, step);
    // graphs read their plans at replay; the others are built by the step's first call that needs them
    struct Made { th_kv_batch::Plan* plan; PlanMaker maker; KvRuns runs; };
    std::vector<Made> made;
    Sending to;
    try {
        size_t more = 0;
        for (auto& p : b->plans) {
            if (!captured(c->dev, p.second)) continue;
            made.push_back({&p.second, PlanMaker(b, p.first.first, p.first.second), {}});
            Made& m = made.back();
            m.maker.make();
            m.runs = plan_runs(b, m.maker);
            more += staged(m.maker.words.size());
        }
        to = prepare(c, copies, words.size(), more);
    } catch (...) {
        std::swap(b->step, step);
        for (size_t i = n; i-- > 0;) ungrow(c, seqs[i], was[i]);
        throw;
    }
    b->begun = false;
    for (auto& p : b->plans) p.second.built = false;
    send(c, to, copies, words.data(), one_run(words.size()), b->block);
    for (Made& m : made) send_plan(b, m.maker, m.runs, *m.plan, to.room);
    b->begun = true;
    TH_API_END
}

int th_kv_batch_trim(th_kv_batch* b, const uint32_t* n_keep, size_t n) {
    TH_API_BEGIN
    require_begun(b, 0, __func__);
    TH_REQUIRE(n_keep || n == 0, "null argument");
    TH_REQUIRE(n == b->step.seqs.size(), "one count for each sequence of the batch");
    for (size_t i = 0; i < n; i++) TH_REQUIRE(n_keep[i] <= b->step.n[i], "more kept than were new");
    for (size_t i = 0; i < n; i++)
        if (n_keep[i] < b->step.n[i]) shrink(b->cache, b->step.seqs[i], b->step.start[i] + n_keep[i]);
    b->begun = false;
    TH_API_END
}

int th_kv_append(th_kv_batch* b, size_t layer, const th_buffer* q, const th_buffer* k, const th_buffer* v, const th_buffer* cos_t,
                 const th_buffer* sin_t, const th_buffer* positions, size_t rot_dim, int layout, th_buffer* q_out) {
    TH_API_BEGIN
    require_begun(b, layer, __func__);
    th_kv_cache* c = b->cache;
    TH_REQUIRE(k && v, "null argument");
    TH_REQUIRE((q == nullptr) == (q_out == nullptr), "q and q_out go together");
    DeviceScope scope(c->dev);
    // a captured call runs on whatever the batch begins with later
    const size_t rows = c->dev->capturing ? b->max_rows : b->step.rows;
    const size_t kv = rows * c->n_kv_heads * c->hd, qn = rows * b->n_heads * c->hd;
    require_x(c, k, kv, "k");
    require_x(c, v, kv, "v");
    TH_REQUIRE(k->dtype == v->dtype && (!q || q->dtype == k->dtype), "q, k and v must be of one type");
    KvRopeArgs a = {};
    if (q) {
        require_x(c, q, qn, "q");
        require_x(c, q_out, qn, "q_out");
        TH_REQUIRE(q_out != k && q_out != v, "q_out must not be k or v");
    }
    rope_args(a, c->dev, cos_t, sin_t, positions, rows, c->hd, rot_dim, layout, b->step.top, q_out);
    a.q = q ? q->ptr : nullptr;
    a.k = k->ptr;
    a.v = v->ptr;
    a.q_out = q_out ? q_out->ptr : nullptr;
    a.xdt = k->dtype;
    a.qdt = q_out ? q_out->dtype : TH_F32;
    a.n_heads = q ? (int)b->n_heads : 0;
    a.hd = (int)c->hd;
    launch_kv_append(a, layer_pages(c, layer), c->dtype, b->block, (const KvRow*)(b->block + 4), rows, c->dev->stream);
    TH_API_END
}

int th_kv_append_norm(th_kv_batch* b, size_t layer, const th_buffer* q, const th_buffer* k, const th_buffer* v,
                      const th_buffer* q_weight, const th_buffer* k_weight, float eps, const th_buffer* cos_t,
                      const th_buffer* sin_t, const th_buffer* positions, size_t rot_dim, int layout, th_buffer* q_out) {
    TH_API_BEGIN
    require_begun(b, layer, __func__);
    th_kv_cache* c = b->cache;
    TH_REQUIRE((k == nullptr) == (v == nullptr), "k and v go together");
    TH_REQUIRE((q == nullptr) == (q_out == nullptr), "q and q_out go together");
    TH_REQUIRE(q || k, "null argument");
    DeviceScope scope(c->dev);
    // a captured call runs on whatever the batch begins with later
    const size_t rows = c->dev->capturing ? b->max_rows : b->step.rows;
    const size_t kv = c->n_kv_heads * c->hd, qn = b->n_heads * c->hd;
    KvRopeArgs a = {};
    if (k) {
        require_x(c, k, rows * kv, "k");
        require_x(c, v, rows * kv, "v");
        TH_REQUIRE(k->dtype == v->dtype && (!q || q->dtype == k->dtype), "q, k and v must be of one type");
        a.q = q ? q->ptr : nullptr;
        a.k = k->ptr;
        a.v = v->ptr;
        a.q_row = qn;
        a.k_row = a.v_row = kv;
        a.xdt = k->dtype;
    } else {  // one row holds all three
        a.q = q->ptr;
        a.k = (const char*)q->ptr + qn * dtype_size(q->dtype);
        a.v = (const char*)a.k + kv * dtype_size(q->dtype);
        a.q_row = a.k_row = a.v_row = qn + 2 * kv;
        a.xdt = q->dtype;
    }
    if (q) {
        require_x(c, q, rows * a.q_row, "q");
        require_x(c, q_out, rows * qn, "q_out");
        TH_REQUIRE(k || q_out != q, "q_out must not be the packed rows");
        require_apart(q_out, {k, v, q_weight, k_weight, positions}, "q_out");
    }
    rope_args(a, c->dev, cos_t, sin_t, positions, rows, c->hd, rot_dim, layout, b->step.top, q_out);
    norm_args(a, c->dev, q_weight, k_weight, eps, c->hd);
    a.q_out = q_out ? q_out->ptr : nullptr;
    a.qdt = q_out ? q_out->dtype : TH_F32;
    a.qo_row = qn;
    a.n_heads = q ? (int)b->n_heads : 0;
    a.hd = (int)c->hd;
    launch_kv_append(a, layer_pages(c, layer), c->dtype, b->block, (const KvRow*)(b->block + 4), rows, c->dev->stream);
    TH_API_END
}

int th_kv_batch_attention(th_kv_batch* b, size_t layer, const th_buffer* q, size_t window, size_t n_sinks, float scale, th_buffer* out) {
    TH_API_BEGIN
    require_begun(b, layer, __func__);
    th_kv_cache* c = b->cache;
    TH_REQUIRE(q && out, "null argument");
    TH_REQUIRE(q != out, "out must not be q");
    // (finite times log2(e) too, which the kernels take)
    TH_REQUIRE(std::isfinite(scale * 1.44269504f) && scale >= 0.0f, "scale must be finite and not negative");
    DeviceScope scope(c->dev);
    const bool capturing = c->dev->capturing;
    const size_t n = (capturing ? b->max_rows : b->step.rows) * b->n_heads * c->hd;
    require_x(c, q, n, "q");
    require_x(c, out, n, "out");
    // a window as long as any sequence hides nothing, and without one there are no sinks
    if (window >= c->max_len) window = 0;
    n_sinks = window ? std::min(n_sinks, c->max_len) : 0;
    const th_kv_batch::Key key(window, n_sinks);
    auto at = b->plans.find(key);
    if (at == b->plans.end() || !at->second.built) {
        TH_REQUIRE(!capturing, "make the call once before it is captured");
        if (at == b->plans.end()) at = add_plan(b, key);
        build_plan(b, key, at->second);
    }
    if (capturing && (at->second.graphs.empty() || at->second.graphs.back() != c->dev->captures)) at->second.graphs.push_back(c->dev->captures);
    const th_kv_batch::Plan& p = at->second;
    KvAttnArgs a;
    a.pages = layer_pages(c, layer);
    a.toks = (const KvTok*)(p.block + plan_toks(b));
    a.q = q->ptr;
    a.out = out->ptr;
    a.qdt = q->dtype;
    a.odt = out->dtype;
    a.n_heads = (int)b->n_heads;
    a.window = (int)window;
    a.sinks = (int)n_sinks;
    a.scale = (scale > 0.0f ? scale : 1.0f / std::sqrt((float)c->hd)) * 1.44269504f;
    a.rec_o = b->rec_o;
    a.rec_ml = b->rec_ml;
    a.head = (const KvPlanHead*)p.block;
    a.rows_items = (const KvItem*)(p.block + plan_rows(b));
    a.tile_items = (const KvItem*)(p.block + plan_tiles(b));
    const KvTok* joins = (const KvTok*)(p.block + plan_joins(b));
    const size_t items = p.n_tile_items + p.n_rows_items;
    if (capturing) {
        // whatever plan the batch has at replay: every kernel, on grids that walk their lists
        launch_kv_attn_both(a, c->dtype, std::max(items, ceil_div(4 * (size_t)c->dev->num_cus, c->n_kv_heads)),
                            c->max_len > KV_LONG_ITEM ? KV_BY_PLAN : 0, c->dev->stream);
        launch_kv_attn_join(a, joins, std::min<size_t>(b->max_rows, 1024), b->max_rows, KV_BY_PLAN, c->dev->stream);
    } else {
        if (p.n_tile_items && p.n_rows_items) launch_kv_attn_both(a, c->dtype, items, p.flags, c->dev->stream);
        else if (p.n_tile_items) launch_kv_attn_tiles(a, c->dtype, items, p.flags, c->dev->stream);
        else launch_kv_attn_rows(a, c->dtype, items, c->dev->stream);
        launch_kv_attn_join(a, joins, p.n_joins, b->max_rows, p.flags, c->dev->stream);
    }
    TH_API_END
}

// ---------------------------------------------------------------------------
// Rotary tables and rows
// ---------------------------------------------------------------------------

int th_rope_tables_scaled(size_t rot_dim, size_t max_seq, double base, const th_rope_scaling* s, float* cos_t, float* sin_t) {
    TH_API_BEGIN
    TH_REQUIRE(cos_t && sin_t, "null table");
    TH_REQUIRE(rot_dim > 0 && rot_dim % 2 == 0, "rot_dim must be even and positive");
    TH_REQUIRE(base > 1.0 && std::isfinite(base), "base must be above 1");
    const size_t half = rot_dim / 2;
    const double two_pi = 2.0 * std::acos(-1.0);
    double factor = 1.0, warm = 1.0;
    const int kind = s ? s->kind : TH_ROPE_PLAIN;
    TH_REQUIRE(kind >= TH_ROPE_PLAIN && kind <= TH_ROPE_RAMP, "unknown scaling");
    if (kind != TH_ROPE_PLAIN) {
        TH_REQUIRE(std::isfinite(s->factor) && s->factor >= 1.0, "factor must be at least 1");
        factor = s->factor;
    }
    if (kind == TH_ROPE_BANDS || kind == TH_ROPE_RAMP) {
        TH_REQUIRE(s->original_len > 0, "original_len must be positive");
        TH_REQUIRE(s->low > 0.0 && s->high > s->low && std::isfinite(s->high), "0 < low < high is needed");
    }
    if (kind == TH_ROPE_BASE) {
        TH_REQUIRE(rot_dim > 2, "rot_dim must be above 2 to scale the base");
        base *= std::pow(factor, (double)rot_dim / ((double)rot_dim - 2.0));
    }
    std::vector<double> freq(half);
    double ramp_lo = 0.0, ramp_hi = 0.0;
    if (kind == TH_ROPE_RAMP) {
        // the (fractional) pair whose wave turns `turns` times over the original length
        auto pair_of = [&](double turns) {
            return (double)rot_dim * std::log((double)s->original_len / (turns * two_pi)) / (2.0 * std::log(base));
        };
        ramp_lo = std::max(std::floor(pair_of(s->high)), 0.0);
        ramp_hi = std::min(std::ceil(pair_of(s->low)), (double)rot_dim - 1.0);
        warm = s->warmth > 0.0 ? s->warmth : 0.1 * std::log(factor) + 1.0;
        TH_REQUIRE(std::isfinite(warm), "warmth must be finite");
    }
    for (size_t i = 0; i < half; i++) {
        const double f = std::pow(base, -(double)i / (double)half);
        if (kind == TH_ROPE_LINEAR) {
            freq[i] = f / factor;
        } else if (kind == TH_ROPE_BANDS) {
            const double turns = (double)s->original_len * f / two_pi;
            const double keep = std::min(1.0, std::max(0.0, (turns - s->low) / (s->high - s->low)));
            freq[i] = keep * f + (1.0 - keep) * f / factor;
        } else if (kind == TH_ROPE_RAMP) {
            const double ramp = std::min(1.0, std::max(0.0, ((double)i - ramp_lo) / std::max(ramp_hi - ramp_lo, 0.001)));
            freq[i] = (1.0 - ramp) * f + ramp * f / factor;
        } else {
            freq[i] = f;
        }
    }
#pragma omp parallel for schedule(static)
    for (long pos = 0; pos < (long)max_seq; pos++)
        for (size_t i = 0; i < half; i++) {
            const double angle = (double)pos * freq[i];
            cos_t[(size_t)pos * half + i] = (float)(std::cos(angle) * warm);
            sin_t[(size_t)pos * half + i] = (float)(std::sin(angle) * warm);
        }
    TH_API_END
}

int th_rope_rows(th_device* dev, const th_buffer* in, const th_buffer* cos_t, const th_buffer* sin_t, const th_buffer* positions,
                 size_t start_pos, size_t n_rows, size_t n_heads, size_t head_dim, size_t rot_dim, int layout, th_buffer* out) {
    TH_API_BEGIN
    TH_REQUIRE(dev && in && out, "null argument");
    TH_REQUIRE(!dev->closed, "the device was destroyed");
    auto ok = [&](const th_buffer* b) { return (b->dtype == TH_F32 || b->dtype == TH_F16 || b->dtype == TH_BF16) && b->dev == dev; };
    TH_REQUIRE(ok(in) && ok(out), "buffers must be f32, f16 or bf16, of this device handle");
    TH_REQUIRE(n_heads <= (size_t)1 << 20 && head_dim <= (size_t)1 << 16 && n_rows < (size_t)1 << 31, "sizes out of range");
    TH_REQUIRE(n_heads * ceil_div(head_dim, 8) < (size_t)1 << 31, "sizes out of range: a row of 2^34 elements");
    TH_REQUIRE(n_rows == 0 || start_pos <= SIZE_MAX - n_rows, "sizes out of range");
    require_len_any(in, n_rows * n_heads * head_dim, "input");
    require_len_any(out, n_rows * n_heads * head_dim, "out");
    TH_REQUIRE(in != out || in->dtype == out->dtype, "out in place of the input needs its type");
    KvRopeArgs a = {};
    rope_args(a, dev, cos_t, sin_t, positions, n_rows, head_dim, rot_dim, layout, start_pos + n_rows, out);
    a.q = in->ptr;
    a.q_out = out->ptr;
    a.xdt = in->dtype;
    a.qdt = out->dtype;
    a.start = start_pos;
    a.n_heads = (int)n_heads;
    a.hd = (int)head_dim;
    DeviceScope scope(dev);
    launch_rope_rows(a, n_rows, dev->stream);
    TH_API_END
}

int th_qk_norm_rope(th_device* dev, const th_buffer* q, size_t q_stride, const th_buffer* k, size_t k_stride, const th_buffer* q_weight,
                    const th_buffer* k_weight, float eps, const th_buffer* cos_t, const th_buffer* sin_t, const th_buffer* positions,
                    size_t start_pos, size_t n_rows, size_t n_heads, size_t n_kv_heads, size_t head_dim, size_t rot_dim, int layout,
                    th_buffer* q_out, th_buffer* k_out) {
    TH_API_BEGIN
    TH_REQUIRE(dev && q && q_out, "null argument");
    TH_REQUIRE(!dev->closed, "the device was destroyed");
    auto ok = [&](const th_buffer* b) { return !b || ((b->dtype == TH_F32 || b->dtype == TH_F16 || b->dtype == TH_BF16) && b->dev == dev); };
    TH_REQUIRE(ok(q) && ok(k) && ok(q_out) && ok(k_out), "buffers must be f32, f16 or bf16, of this device handle");
    TH_REQUIRE(!k || k->dtype == q->dtype, "q and k must be of one type");
    TH_REQUIRE(n_kv_heads > 0 || (!k && !k_out), "keys without key heads");
    TH_REQUIRE(n_heads > 0 && head_dim > 0, "no queries");
    constexpr size_t HEADS = (size_t)1 << 16, WIDE = (size_t)1 << 32;
    TH_REQUIRE(n_heads <= HEADS && n_kv_heads <= HEADS && head_dim <= HEADS && n_rows < (size_t)1 << 31, "sizes out of range");
    TH_REQUIRE(q_stride < WIDE && k_stride < WIDE, "strides out of range");
    TH_REQUIRE(n_rows == 0 || start_pos <= SIZE_MAX - n_rows, "sizes out of range");
    const size_t qn = n_heads * head_dim, kn = n_kv_heads * head_dim;
    const size_t q_in = k ? qn : qn + kn, q_to = k_out ? qn : qn + kn;  // keys behind the queries in a row
    // the last row ends with its heads
    auto reach = [&](size_t row, size_t width) { return n_rows ? (n_rows - 1) * row + width : 0; };
    KvRopeArgs a = {};
    a.q_row = q_stride ? q_stride : q_in;
    a.k_row = k ? (k_stride ? k_stride : kn) : a.q_row;
    TH_REQUIRE(a.q_row >= q_in && a.k_row >= kn, "a stride shorter than its row");
    TH_REQUIRE(k || k_stride == 0, "a stride of no keys");
    a.qo_row = q_out == q ? a.q_row : q_to;
    a.ko_row = !k_out ? a.qo_row : k_out == k ? a.k_row : kn;
    TH_REQUIRE(a.qo_row >= q_to, "no room for the keys behind the queries");
    require_len_any(q, reach(a.q_row, q_in), "q");
    require_len_any(q_out, reach(a.qo_row, q_to), "q_out");
    if (k) require_len_any(k, reach(a.k_row, kn), "k");
    if (k_out) require_len_any(k_out, reach(a.ko_row, kn), "k_out");
    TH_REQUIRE(k != q && q_out != k_out, "queries and keys must be buffers of their own");
    require_apart(q_out, {k, q_weight, k_weight, positions}, "q_out");
    if (k_out) require_apart(k_out, {q, q_weight, k_weight, positions}, "k_out");
    rope_args(a, dev, cos_t, sin_t, positions, n_rows, head_dim, rot_dim, layout, start_pos + n_rows, q_out);
    TH_REQUIRE(!k_out || (k_out != cos_t && k_out != sin_t), "the result must not be a table");
    norm_args(a, dev, q_weight, k_weight, eps, head_dim);
    a.q = q->ptr;
    a.k = k ? k->ptr : (const char*)q->ptr + qn * dtype_size(q->dtype);
    a.q_out = q_out->ptr;
    a.k_out = k_out ? k_out->ptr : (char*)q_out->ptr + qn * dtype_size(q_out->dtype);
    a.xdt = q->dtype;
    a.qdt = q_out->dtype;
    a.kdt = k_out ? k_out->dtype : q_out->dtype;
    a.start = start_pos;
    a.n_heads = (int)n_heads;
    a.n_kv = (int)n_kv_heads;
    a.hd = (int)head_dim;
    DeviceScope scope(dev);
    launch_rope_rows(a, n_rows, dev->stream);
    TH_API_END
}

}  // extern "C"
