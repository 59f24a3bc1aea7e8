// gq8_paged_cache.cpp -- the C ABI of the paged cache (include/gemma_q8.h):
// the checks of its operators' arguments, and the page pool, which keeps on
// the host which sequence holds which pages.
//
// The pool.  A page counts its holders; a fork adds a holder to each of its
// parent's pages.  A page is written by one holder only: extending a sequence
// whose last page is partly full and shared gives it a page of its own and
// records a copy.  Recorded copies are run by the caller in one launch, all at
// once, so the list must not depend on an order: a page that a recorded copy
// reads is not given out again before the list is taken, a copy whose target
// is dropped is dropped, and a copy from the target of another reads that
// one's source.
#include "gemma_q8.h"
#include "gq8_checkpoint.hpp"
#include "gq8_paged.hpp"

#include <algorithm>
#include <climits>
#include <cmath>
#include <mutex>
#include <new>
#include <string>
#include <vector>

using gq8::report;

namespace {

bool aligned(const void *p)
{
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}

bool type16(int type)
{
    return type == GQ8_DTYPE_F16 || type == GQ8_DTYPE_BF16;
}

bool row_type(int type)
{
    return type == GQ8_DTYPE_F32 || type16(type);
}

// rows of a type lie on 16 bytes
bool row_stride(int stride, int64_t width, int type)
{
    return stride >= width && stride % (type == GQ8_DTYPE_F32 ? 4 : 8) == 0;
}

int launched(hipError_t status, const char *what)
{
    if (status == hipErrorInvalidValue)
        return report(GQ8_ERR_ARGUMENT, std::string(what) + ": arguments refused");
    if (status != hipSuccess)
        return report(GQ8_ERR_DEVICE, std::string(what) + ": " + hipGetErrorString(status));
    return GQ8_OK;
}

int check_heads(const char *what, int heads, int kv_heads, int head_dim)
{
    if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || heads / kv_heads > 32
        || head_dim <= 0 || head_dim % 8 != 0 || head_dim > gq8::kPagedMaxHeadDim
        || (int64_t) heads * head_dim > INT_MAX / 4)
        return report(GQ8_ERR_SHAPE, std::string(what)
                                         + ": heads a multiple of kv heads, at most 32 of them each, "
                                           "head width a multiple of 8 up to 256");
    return GQ8_OK;
}

int check_cache(const char *what, const gq8_page_cache *c)
{
    if (!c)
        return report(GQ8_ERR_ARGUMENT, std::string(what) + ": null cache");
    if (int s = check_heads(what, c->kv_heads, c->kv_heads, c->head_dim))
        return s;
    if (!type16(c->type))
        return report(GQ8_ERR_SHAPE, std::string(what) + ": a cache holds F16 or BF16");
    if (c->layers <= 0 || c->pages < 0 || c->page_rows <= 0 || (c->page_rows & (c->page_rows - 1)) != 0
        || (int64_t) c->pages * c->page_rows > INT_MAX)
        return report(GQ8_ERR_SHAPE, std::string(what)
                                         + ": layers >= 1, page rows a power of two, rows below 2^31");
    if (c->pages > 0 && (!c->keys || !c->values || !aligned(c->keys) || !aligned(c->values)))
        return report(GQ8_ERR_ARGUMENT, std::string(what) + ": null or unaligned pool");
    return GQ8_OK;
}

int shift_of(int page_rows)
{
    int shift = 0;
    while ((1 << shift) < page_rows)
        ++shift;
    return shift;
}

gq8::PagedLayer layer_of(const gq8_page_cache &c, int layer)
{
    const int width = c.kv_heads * c.head_dim;
    const int64_t at = (int64_t) layer * c.pages * c.page_rows * width;
    auto pool = [&](void *p) { return p && c.pages > 0 ? static_cast<uint16_t *>(p) + at : nullptr; };
    return {pool(c.keys), pool(c.values), c.pages, shift_of(c.page_rows), width};
}

int check_sequences(const char *what, const gq8_page_cache &c, int layer, const gq8_sequences *q)
{
    if (layer < 0 || layer >= c.layers)
        return report(GQ8_ERR_ARGUMENT, std::string(what) + ": no such layer");
    if (!q || q->sequences < 0 || q->rows < 0 || (q->sequences > 0 && !q->starts) || q->table_width < 0)
        return report(GQ8_ERR_ARGUMENT, std::string(what) + ": bad sequences");
    if ((int64_t) q->table_width * c.page_rows > gq8::kPagedMaxRows || q->rows > gq8::kPagedMaxRows)
        return report(GQ8_ERR_SHAPE, std::string(what) + ": at most 2^30 rows, cached and new ones each");
    if (q->cached && q->sequences > 0 && (!q->page_table || q->table_width == 0))
        return report(GQ8_ERR_ARGUMENT, std::string(what) + ": cached rows without a page table");
    return GQ8_OK;
}

gq8::PackedSequences sequences_of(const gq8_sequences &q)
{
    return {q.sequences, q.rows, q.starts, q.cached, q.page_table, q.table_width};
}

int attention(const char *what, const gq8_page_cache *cache, int layer, const gq8_sequences *seq,
              const void *q, int q_type, int q_stride, int heads, const void *k, const void *v,
              int kv_stride, bool causal, const uint64_t *masks, int mask_words, float scale, void *out,
              int out_stride, void *workspace, size_t workspace_bytes, void *stream)
{
    if (int s = check_cache(what, cache))
        return s;
    if (int s = check_heads(what, heads, cache->kv_heads, cache->head_dim))
        return s;
    if (int s = check_sequences(what, *cache, layer, seq))
        return s;
    if (q_type != cache->type && !(q_type == GQ8_DTYPE_F32 && cache->type == GQ8_DTYPE_F16))
        return report(GQ8_ERR_SHAPE, std::string(what)
                                         + ": queries of the cache's type, or F32 over an F16 cache");
    if (seq->rows == 0 || seq->sequences == 0)
        return GQ8_OK;
    const int64_t width = (int64_t) cache->kv_heads * cache->head_dim;
    if (width > gq8::kPagedMaxApart || ((k || v) && kv_stride > gq8::kPagedMaxApart))
        return report(GQ8_ERR_SHAPE, std::string(what) + ": rows of keys at most 2^26 values apart");
    if (!q || !out || !workspace || !aligned(q) || !aligned(out) || !aligned(workspace)
        || !row_stride(q_stride, (int64_t) heads * cache->head_dim, q_type)
        || !row_stride(out_stride, (int64_t) heads * cache->head_dim, q_type) || !std::isfinite(scale))
        return report(GQ8_ERR_ARGUMENT, std::string(what) + ": bad arguments");
    if (k || v || causal) {
        if (!k || !v || !aligned(k) || !aligned(v) || !row_stride(kv_stride, width, cache->type))
            return report(GQ8_ERR_ARGUMENT, std::string(what) + ": bad keys or values");
        if (!causal && (!masks || mask_words < 1 || mask_words > 1024))
            return report(GQ8_ERR_ARGUMENT, std::string(what) + ": 1 to 1024 mask words a row");
    }
    if (workspace_bytes < gq8::packed_attention_workspace_bytes(heads, cache->kv_heads, cache->head_dim))
        return report(GQ8_ERR_ARGUMENT, std::string(what) + ": workspace too small");
    gq8::PackedAttentionArgs a{};
    a.layer = layer_of(*cache, layer);
    a.seq = sequences_of(*seq);
    a.q = q;
    a.q_stride = q_stride;
    a.heads = heads;
    a.kv_heads = cache->kv_heads;
    a.head_dim = cache->head_dim;
    a.k = static_cast<const uint16_t *>(k);
    a.v = static_cast<const uint16_t *>(v);
    a.kv_stride = kv_stride;
    a.causal = causal;
    a.masks = masks;
    a.mask_words = mask_words;
    a.scale = scale;
    a.out = out;
    a.out_stride = out_stride;
    a.workspace = static_cast<float *>(workspace);
    return launched(gq8::launch_packed_attention(a, q_type, static_cast<hipStream_t>(stream)), what);
}

} // namespace

extern "C" int gq8_head_norm_rope(const void *x, int x_type, int x_stride, int rows, int heads,
                                  int kv_heads, int head_dim, const float *q_weight,
                                  const float *k_weight, float epsilon, const int32_t *positions,
                                  const float *cosines, const float *sines, int max_positions, void *q,
                                  int q_type, int q_stride, void *k, void *v, int kv_type,
                                  int kv_stride, void *stream)
{
    if (int s = check_heads("head_norm_rope", heads, kv_heads, head_dim))
        return s;
    if (!row_type(x_type) || !row_type(q_type) || ((k || v) && !type16(kv_type)))
        return report(GQ8_ERR_SHAPE, "head_norm_rope: rows of F32, F16 or BF16, keys of F16 or BF16");
    if (rows == 0)
        return GQ8_OK;
    const int64_t width = (int64_t) kv_heads * head_dim;
    if (rows < 0 || !x || !positions || !cosines || !sines || !q || max_positions <= 0
        || !std::isfinite(epsilon) || epsilon < 0.f || !aligned(x) || !aligned(q) || !aligned(k)
        || !aligned(v) || !aligned(cosines) || !aligned(sines) || !aligned(q_weight)
        || !aligned(k_weight) || !row_stride(x_stride, (int64_t) heads * head_dim + 2 * width, x_type)
        || !row_stride(q_stride, (int64_t) heads * head_dim, q_type)
        || ((k || v) && !row_stride(kv_stride, width, kv_type)))
        return report(GQ8_ERR_ARGUMENT, "head_norm_rope: bad arguments");
    gq8::NormRopeArgs a{x, x_stride, rows, heads, kv_heads, head_dim, q_weight, k_weight, epsilon,
                        positions, cosines, sines, max_positions, q, k, v, q_stride, kv_stride};
    return launched(gq8::launch_head_norm_rope(a, x_type, q_type, kv_type,
                                               static_cast<hipStream_t>(stream)),
                    "head_norm_rope");
}

extern "C" int gq8_page_append(const gq8_page_cache *cache, int layer, const gq8_sequences *seq,
                               const void *k, const void *v, int kv_stride, const int32_t *places,
                               void *stream)
{
    if (int s = check_cache("page_append", cache))
        return s;
    if (int s = check_sequences("page_append", *cache, layer, seq))
        return s;
    if (seq->rows == 0 || seq->sequences == 0)
        return GQ8_OK;
    if (!k || !v || !aligned(k) || !aligned(v) || cache->pages == 0 || !seq->page_table
        || !row_stride(kv_stride, (int64_t) cache->kv_heads * cache->head_dim, cache->type))
        return report(GQ8_ERR_ARGUMENT, "page_append: bad arguments");
    return launched(gq8::launch_page_append(layer_of(*cache, layer), sequences_of(*seq),
                                            static_cast<const uint16_t *>(k),
                                            static_cast<const uint16_t *>(v), kv_stride, places,
                                            static_cast<hipStream_t>(stream)),
                    "page_append");
}

extern "C" int gq8_page_copy(const gq8_page_cache *cache, const int32_t *pairs, int count, void *stream)
{
    if (int s = check_cache("page_copy", cache))
        return s;
    if (count == 0)
        return GQ8_OK;
    if (!pairs || count < 0 || cache->pages == 0)
        return report(GQ8_ERR_ARGUMENT, "page_copy: bad arguments");
    const int64_t bytes = (int64_t) cache->page_rows * cache->kv_heads * cache->head_dim * 2;
    return launched(gq8::launch_page_copy(cache->keys, cache->values, cache->layers, cache->pages, bytes,
                                          pairs, count, static_cast<hipStream_t>(stream)),
                    "page_copy");
}

extern "C" size_t gq8_packed_attention_workspace_bytes(int heads, int kv_heads, int head_dim)
{
    if (check_heads("packed_attention", heads, kv_heads, head_dim))
        return 0;
    return gq8::packed_attention_workspace_bytes(heads, kv_heads, head_dim);
}

extern "C" int gq8_packed_attention(const gq8_page_cache *cache, int layer, const gq8_sequences *seq,
                                    const void *q, int q_type, int q_stride, int heads, const void *k,
                                    const void *v, int kv_stride, float scale, void *out, int out_stride,
                                    void *workspace, size_t workspace_bytes, void *stream)
{
    return attention("packed_attention", cache, layer, seq, q, q_type, q_stride, heads, k, v, kv_stride,
                     true, nullptr, 0, scale, out, out_stride, workspace, workspace_bytes, stream);
}

extern "C" int gq8_tree_attention(const gq8_page_cache *cache, int layer, const gq8_sequences *seq,
                                  const void *q, int q_type, int q_stride, int heads, const void *k,
                                  const void *v, int kv_stride, const uint64_t *ancestors,
                                  int mask_words, float scale, void *out, int out_stride,
                                  void *workspace, size_t workspace_bytes, void *stream)
{
    return attention("tree_attention", cache, layer, seq, q, q_type, q_stride, heads, k, v, kv_stride,
                     false, ancestors, mask_words, scale, out, out_stride, workspace, workspace_bytes,
                     stream);
}

// ---- the page pool ----------------------------------------------------------------
namespace {

// The free pages: a bit a page, and over each 64 words a word of which have one,
// up to a single word.  The lowest is found in as many steps as there are levels
// (two up to 4096 pages, four up to 16 million), and nothing is allocated after the start.
class FreePages {
public:
    explicit FreePages(int pages) : free(pages)
    {
        size_t bits = (size_t) pages;
        do {
            const size_t words = (bits + 63) / 64;
            std::vector<uint64_t> level(words, ~0ull);
            if (bits % 64 != 0)
                level.back() = (1ull << bits % 64) - 1;
            levels.push_back(std::move(level));
            bits = words;
        } while (bits > 1);
    }

    int count() const { return free; }

    int lowest() const // there is one
    {
        size_t at = 0;
        for (size_t l = levels.size(); l-- > 0;)
            at = at * 64 + (size_t) __builtin_ctzll(levels[l][at]);
        return (int) at;
    }

    void insert(int page)
    {
        size_t at = (size_t) page;
        ++free;
        for (auto &level : levels) {
            level[at / 64] |= 1ull << at % 64;
            at /= 64;
        }
    }

    void erase(int page)
    {
        size_t at = (size_t) page;
        --free;
        for (auto &level : levels) {
            if (level[at / 64] &= ~(1ull << at % 64))
                break;
            at /= 64;
        }
    }

private:
    std::vector<std::vector<uint64_t>> levels;
    int free;
};

} // namespace

struct gq8_page_pool {
    struct Sequence {
        bool open = false;
        int64_t rows = 0;
        std::vector<int> pages;
    };
    // The recorded copy into a page: from where (-1: none is), and the targets of
    // the ones recorded before and after it.
    struct Copy {
        int from = -1, before = -1, after = -1;
    };

    int pages, page_rows, table_width;
    std::vector<int> holders; // of each page
    std::vector<int> reads;   // recorded copies that read it
    std::vector<Copy> copies; // by the page they write
    int first = -1, last = -1, recorded = 0; // targets of the list's ends, and its length
    FreePages unused;         // no holder, not read: the lowest is given out first
    std::vector<Sequence> sequences;
    std::mutex mutex;

    gq8_page_pool(int pages_, int page_rows_, int sequences_, int width)
        : pages(pages_), page_rows(page_rows_), table_width(width), holders(pages_, 0), reads(pages_, 0),
          copies(pages_), unused(pages_), sequences(sequences_)
    {
    }

    bool known(int s) const
    {
        return s >= 0 && s < (int) sequences.size() && sequences[s].open;
    }

    int take()
    {
        const int page = unused.lowest();
        unused.erase(page);
        holders[page] = 1;
        return page;
    }

    void settle(int page)
    {
        if (holders[page] == 0 && reads[page] == 0)
            unused.insert(page);
    }

    // where the rows of `page` are before the recorded copies run
    int source(int page) const
    {
        return copies[page].from >= 0 ? copies[page].from : page;
    }

    void record(int from, int to)
    {
        copies[to] = {from, last, -1};
        (last >= 0 ? copies[last].after : first) = to;
        last = to;
        ++recorded;
        ++reads[from];
    }

    // Takes the recorded copy into `page` out of the list, if there is one.
    void forget(int page)
    {
        const Copy copy = copies[page];
        if (copy.from < 0)
            return;
        (copy.before >= 0 ? copies[copy.before].after : first) = copy.after;
        (copy.after >= 0 ? copies[copy.after].before : last) = copy.before;
        copies[page] = Copy{};
        --recorded;
        --reads[copy.from];
        settle(copy.from);
    }

    void release(int page)
    {
        if (--holders[page] > 0)
            return;
        forget(page);
        settle(page);
    }
};

namespace {

template <typename F>
int guarded(const char *what, gq8_page_pool *pool, F body)
{
    if (!pool)
        return report(GQ8_ERR_ARGUMENT, std::string(what) + ": null pool");
    try {
        std::lock_guard<std::mutex> lock(pool->mutex);
        return body();
    } catch (const std::bad_alloc &) {
        return report(GQ8_ERR_MEMORY, std::string(what) + ": host allocation failed");
    } catch (const std::exception &e) {
        return report(GQ8_ERR_ARGUMENT, std::string(what) + ": " + e.what());
    }
}

int no_sequence(const char *what)
{
    return report(GQ8_ERR_ARGUMENT, std::string(what) + ": no such open sequence");
}

} // namespace

extern "C" int gq8_page_pool_create(int pages, int page_rows, int sequences, int table_width,
                                    gq8_page_pool **out)
{
    if (!out)
        return report(GQ8_ERR_ARGUMENT, "page_pool_create: null out");
    *out = nullptr;
    if (pages <= 0 || page_rows <= 0 || (page_rows & (page_rows - 1)) != 0 || sequences <= 0
        || table_width <= 0 || (int64_t) pages * page_rows > INT_MAX
        || (int64_t) table_width * page_rows > gq8::kPagedMaxRows)
        return report(GQ8_ERR_SHAPE, "page_pool_create: sizes positive, page rows a power of two, rows "
                                     "below 2^31, a sequence's at most 2^30");
    try {
        *out = new gq8_page_pool(pages, page_rows, sequences, table_width);
    } catch (const std::bad_alloc &) {
        return report(GQ8_ERR_MEMORY, "page_pool_create: host allocation failed");
    }
    return GQ8_OK;
}

extern "C" void gq8_page_pool_destroy(gq8_page_pool *pool)
{
    delete pool;
}

extern "C" int gq8_page_pool_open(gq8_page_pool *pool)
{
    return guarded("page_pool_open", pool, [&] {
        for (size_t s = 0; s < pool->sequences.size(); ++s)
            if (!pool->sequences[s].open) {
                pool->sequences[s].open = true;
                return (int) s;
            }
        return report(GQ8_ERR_CAPACITY, "page_pool_open: every sequence is open");
    });
}

extern "C" int gq8_page_pool_fork(gq8_page_pool *pool, int sequence)
{
    return guarded("page_pool_fork", pool, [&] {
        if (!pool->known(sequence))
            return no_sequence("page_pool_fork");
        for (size_t s = 0; s < pool->sequences.size(); ++s)
            if (!pool->sequences[s].open) {
                gq8_page_pool::Sequence copy = pool->sequences[sequence];
                for (int page : copy.pages)
                    ++pool->holders[page];
                pool->sequences[s] = std::move(copy);
                return (int) s;
            }
        return report(GQ8_ERR_CAPACITY, "page_pool_fork: every sequence is open");
    });
}

extern "C" int gq8_page_pool_extend(gq8_page_pool *pool, int sequence, int rows)
{
    return guarded("page_pool_extend", pool, [&] {
        if (!pool->known(sequence))
            return no_sequence("page_pool_extend");
        if (rows < 0)
            return report(GQ8_ERR_ARGUMENT, "page_pool_extend: negative rows");
        auto &s = pool->sequences[sequence];
        const int64_t after = s.rows + rows;
        if (after > (int64_t) pool->table_width * pool->page_rows)
            return report(GQ8_ERR_WINDOW, "page_pool_extend: past the table's width");
        const size_t wanted = (size_t) ((after + pool->page_rows - 1) / pool->page_rows);
        // rows go into the last page, which then has to be this sequence's alone
        const bool partly = rows > 0 && s.rows % pool->page_rows != 0;
        const bool copies = partly && pool->holders[s.pages.back()] > 1;
        const size_t fresh = wanted > s.pages.size() ? wanted - s.pages.size() : 0;
        if (fresh + (copies ? 1 : 0) > (size_t) pool->unused.count())
            return report(GQ8_ERR_CAPACITY, "page_pool_extend: no free pages");
        if (s.pages.capacity() < wanted) // the last that can fail
            s.pages.reserve(std::max(wanted, 2 * s.pages.capacity()));
        if (copies) {
            const int shared = s.pages.back(), own = pool->take();
            pool->record(pool->source(shared), own);
            s.pages.back() = own;
            pool->release(shared);
        }
        for (size_t i = 0; i < fresh; ++i)
            s.pages.push_back(pool->take());
        s.rows = after;
        return (int) GQ8_OK;
    });
}

extern "C" int gq8_page_pool_truncate(gq8_page_pool *pool, int sequence, int rows)
{
    return guarded("page_pool_truncate", pool, [&] {
        if (!pool->known(sequence))
            return no_sequence("page_pool_truncate");
        auto &s = pool->sequences[sequence];
        if (rows < 0 || rows > s.rows)
            return report(GQ8_ERR_ARGUMENT, "page_pool_truncate: more rows than there are");
        const size_t kept = (size_t) (((int64_t) rows + pool->page_rows - 1) / pool->page_rows);
        while (s.pages.size() > kept) {
            pool->release(s.pages.back());
            s.pages.pop_back();
        }
        s.rows = rows;
        return (int) GQ8_OK;
    });
}

extern "C" int gq8_page_pool_close(gq8_page_pool *pool, int sequence)
{
    return guarded("page_pool_close", pool, [&] {
        if (!pool->known(sequence))
            return no_sequence("page_pool_close");
        auto &s = pool->sequences[sequence];
        for (int page : s.pages)
            pool->release(page);
        s = gq8_page_pool::Sequence{};
        return (int) GQ8_OK;
    });
}

extern "C" int gq8_page_pool_compact(gq8_page_pool *pool)
{
    return guarded("page_pool_compact", pool, [&] {
        int used = 0, moved = 0;
        for (int count : pool->holders)
            used += count > 0;
        std::vector<int> now(pool->pages);
        for (int page = 0; page < pool->pages; ++page)
            now[page] = page;
        for (int page = pool->pages - 1; page >= used; --page) {
            if (pool->holders[page] == 0)
                continue;
            if (pool->unused.count() == 0 || pool->unused.lowest() >= used)
                break; // the rest of the low pages wait for recorded copies
            const int count = pool->holders[page], to = pool->take();
            pool->holders[to] = count;
            pool->record(pool->source(page), to); // read by the new copy before the old one goes
            pool->holders[page] = 0;
            pool->forget(page);
            pool->settle(page);
            now[page] = to;
            ++moved;
        }
        for (auto &s : pool->sequences)
            for (int &page : s.pages)
                page = now[page];
        return moved;
    });
}

extern "C" int gq8_page_pool_copy_count(gq8_page_pool *pool)
{
    return guarded("page_pool_copy_count", pool, [&] { return pool->recorded; });
}

extern "C" int gq8_page_pool_take_copies(gq8_page_pool *pool, int32_t *pairs, int capacity)
{
    return guarded("page_pool_take_copies", pool, [&] {
        const int count = pool->recorded;
        if (count == 0)
            return 0;
        if (!pairs || capacity < count)
            return report(GQ8_ERR_CAPACITY, "page_pool_take_copies: " + std::to_string(count)
                                                + " copies are recorded");
        for (int i = 0; i < count; ++i) {
            const int to = pool->first;
            pairs[2 * i] = pool->copies[to].from;
            pairs[2 * i + 1] = to;
            pool->forget(to);
        }
        return count;
    });
}

extern "C" int gq8_page_pool_rows(gq8_page_pool *pool, int sequence)
{
    return guarded("page_pool_rows", pool, [&] {
        return pool->known(sequence) ? (int) pool->sequences[sequence].rows
                                     : no_sequence("page_pool_rows");
    });
}

extern "C" int gq8_page_pool_free_pages(gq8_page_pool *pool)
{
    return guarded("page_pool_free_pages", pool, [&] { return pool->unused.count(); });
}

extern "C" int gq8_page_pool_tables(gq8_page_pool *pool, const int32_t *sequences, int count,
                                    int32_t *table, int32_t *rows)
{
    return guarded("page_pool_tables", pool, [&] {
        if (count < 0 || (count > 0 && (!sequences || !table || !rows)))
            return report(GQ8_ERR_ARGUMENT, "page_pool_tables: bad arguments");
        for (int i = 0; i < count; ++i)
            if (!pool->known(sequences[i]))
                return no_sequence("page_pool_tables");
        for (int i = 0; i < count; ++i) {
            const auto &s = pool->sequences[sequences[i]];
            int32_t *to = table + (int64_t) i * pool->table_width;
            for (int j = 0; j < pool->table_width; ++j)
                to[j] = j < (int) s.pages.size() ? s.pages[j] : -1;
            rows[i] = (int32_t) s.rows;
        }
        return (int) GQ8_OK;
    });
}
