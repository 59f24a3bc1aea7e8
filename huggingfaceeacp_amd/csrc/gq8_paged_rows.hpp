// gq8_paged_rows.hpp -- where a packed row belongs and where its sequence's keys
// lie in the pool.
#pragma once

#include "gq8_paged.hpp"

#include <hip/hip_runtime.h>

namespace gq8 {
namespace {

// The sequence that holds packed row t, counted by a wave 64 starts at a time;
// -1 before the first and behind the last.
__device__ inline int sequence_of_row(const PackedSequences &seq, int t)
{
    const int lane = threadIdx.x & 63;
    int s = 0;
    for (int base = 0; base < seq.sequences; base += 64) {
        const bool before = base + lane < seq.sequences && seq.starts[base + lane + 1] <= t;
        s += __popcll(__ballot(before));
    }
    return s >= seq.sequences || seq.starts[s] > t ? -1 : s;
}

// The row of the pool that holds a sequence's key, -1 for one that is nowhere.
__device__ inline int64_t pool_row(const PagedLayer &layer, const PackedSequences &seq, int s, int64_t key)
{
    const int64_t slot = key >> layer.page_shift;
    if (key < 0 || slot >= seq.table_width)
        return -1;
    const int page = seq.table[(int64_t) s * seq.table_width + slot];
    if (page < 0 || page >= layer.pages)
        return -1;
    return ((int64_t) page << layer.page_shift) + (key & ((1 << layer.page_shift) - 1));
}

} // namespace
} // namespace gq8
