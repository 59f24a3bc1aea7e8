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

// The sum of the lanes up to each, by moves inside rows of 16 and from a row's last lane
// to the next rows: no round trips through the LDS crossbar.  All 64 lanes are active.
__device__ inline int sum_upto(int v)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true); // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true); // row_shr:2
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true); // row_shr:4
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true); // row_shr:8
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, true); // row_bcast:15, to rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, true); // row_bcast:31, to rows 2 and 3
    return v;
}

// Finds part number `wanted` of a list whose entry i of `count` has parts_of(i) of them,
// by a wave, 64 entries at a time.
template <typename F>
__device__ inline bool find_part(int wanted, int count, F parts_of, int &which, int &within)
{
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < count; base += 64) {
        const int mine = base + lane < count ? parts_of(base + lane) : 0;
        const int upto = sum_upto(mine);
        const uint64_t past = __ballot(base + lane < count && before + upto > wanted);
        if (past) {
            const int found = __ffsll((unsigned long long) past) - 1;
            which = base + found;
            within = wanted - before - (__builtin_amdgcn_readlane(upto, found) - __builtin_amdgcn_readlane(mine, found));
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, min(count - base, 64) - 1);
    }
    return false;
}

} // namespace
} // namespace gq8
