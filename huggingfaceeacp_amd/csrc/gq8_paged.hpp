// gq8_paged.hpp -- the operators of a paged key/value cache that many
// sequences share: launch functions of the kernels in gq8_paged.hip (norms and
// rotation of a step's rows, appends, page copies) and
// gq8_paged_attention.hip (attention of packed sequences).
//
// Every length, page and mask is read on the device, so a captured launch
// replays with new ones; the host checks sizes, strides and alignment.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace gq8 {

constexpr int kPagedMaxHeadDim = 256;
constexpr int kPagedMaxRows = 1 << 30;  // of a step, and of a sequence's pages
constexpr int kPagedMaxApart = 1 << 26; // values from a row of keys to the next: 16 rows' bytes fit 32 bits

// One layer of the cache.
struct PagedLayer {
    uint16_t *keys, *values; // [pages, page_rows, width]
    int pages, page_shift;   // page_rows = 1 << page_shift
    int width;               // kv_heads * head_dim
};

// Sequence s owns the packed rows starts[s] .. starts[s + 1] - 1, behind
// cached[s] rows in the pages of its row of the table.
struct PackedSequences {
    int sequences, rows;
    const int *starts, *cached, *table; // cached may be null: none
    int table_width;
};

struct NormRopeArgs {
    const void *x;
    int x_stride, rows, heads, kv_heads, head_dim;
    const float *q_weight, *k_weight; // null: no norm
    float epsilon;
    const int *positions;
    const float *cosines, *sines;
    int max_positions;
    void *q, *k, *v; // k and v may be null
    int q_stride, kv_stride;
};
// types: GQ8_DTYPE_F32, _F16 or _BF16 (q as x or any of them; kv 16 bits)
hipError_t launch_head_norm_rope(const NormRopeArgs &a, int x_type, int q_type, int kv_type,
                                 hipStream_t stream);

// the same with keys and values into their pages; positions may be null
hipError_t launch_append_rope(const NormRopeArgs &a, int x_type, int q_type, int kv_type,
                              const PagedLayer &layer, const PackedSequences &seq, const int *places,
                              hipStream_t stream);

hipError_t launch_page_append(const PagedLayer &layer, const PackedSequences &seq,
                              const uint16_t *k, const uint16_t *v, int kv_stride,
                              const int *places, hipStream_t stream);

hipError_t launch_page_copy(void *keys, void *values, int layers, int pages, int64_t page_bytes,
                            const int *pairs, int count, hipStream_t stream);

struct PackedAttentionArgs {
    PagedLayer layer;
    PackedSequences seq;
    const void *q;
    int q_stride, heads, kv_heads, head_dim;
    const uint16_t *k, *v; // the packed rows' own; null: the cache alone is attended
    int kv_stride;
    bool causal;           // row i over new rows 0 .. i; else by masks
    const uint64_t *masks; // [rows, mask_words]
    int mask_words;
    float scale;
    void *out;
    int out_stride;
    float *workspace;
};
size_t packed_attention_workspace_bytes(int heads, int kv_heads, int head_dim);
hipError_t launch_packed_attention(const PackedAttentionArgs &a, int q_type, hipStream_t stream);

// Bounds of the keys in the pages that rows went into: lows and highs [pages, width],
// of the cache's type.
hipError_t launch_page_bounds(const PagedLayer &layer, const PackedSequences &seq, const int *taken,
                              uint16_t *lows, uint16_t *highs, int type, hipStream_t stream);

struct PageSelectArgs {
    PagedLayer layer;
    PackedSequences seq;
    const uint16_t *lows, *highs;
    const void *q;
    int q_stride, heads, kv_heads, head_dim;
    int first, last, top;
    uint32_t *ranks; // [rows, kv_heads, table_width]
    int *pages;      // [rows, kv_heads, top]
};
hipError_t launch_page_select(const PageSelectArgs &a, int cache_type, int q_type, hipStream_t stream);

// Few rows over long caches (gq8_paged_streams.hip): rows over the pages listed for
// them, list [rows, kv_heads, top] (a.k, a.v, a.causal and the masks are not used),
// and sequences first[i] .. first[i + 1] - 1 that share their first shared[i] rows.
size_t sparse_attention_workspace_bytes(int64_t rows, int heads, int kv_heads, int head_dim);
hipError_t launch_sparse_attention(const PackedAttentionArgs &a, const int *list, int top, int q_type,
                                   hipStream_t stream);
size_t prefix_attention_workspace_bytes(int64_t rows, int heads, int kv_heads, int head_dim);
hipError_t launch_prefix_attention(const PackedAttentionArgs &a, int groups, const int *first, const int *shared,
                                   int q_type, hipStream_t stream);

} // namespace gq8
