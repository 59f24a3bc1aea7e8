// gq8_paged_streams.hip -- attention of few rows over long paged caches: sequences
// that share a prefix, whose keys are read once for all of them, and rows that each
// attend a list of pages.
//
// Mathematics.  As in gq8_paged_attention.hip: o = sum_j p_j v_j / sum_j p_j,
// p_j = 2^(c q.k_j - m), in one pass over the keys with a running reference m; sums
// about different references are joined by bringing both to the larger.
//
// Work.  A tile is up to 32 (row, head) pairs of one KV head: rows of a prefix's
// sequences, of one sequence, or one row with its list.  A workgroup takes a tile and a
// run of its keys, cut into units of 32, which its four waves take in turn.  Every wave
// streams its own keys and values through a part of LDS that is its alone, so no wave
// waits for another before the end.  There the waves' sums are joined through LDS, and
// what several workgroups hold of a row is left as parts, which merge_parts joins.
// (Tiles of 128 pairs, 32 a wave, read keys once for four of these, but leave four
// times the sums: 16 tokens of 8 heads behind 4096 rows took 43 us so.)
//
// Where there are many pairs and queries are of 16 bits, a prefix's tiles are of 64, whose
// keys two waves share.
//
// What bounds it (both launches, a call).
// - 16 tokens, 8 heads of 256, fp32, behind 4096 shared rows: 16.9 us, 13 + 4.  A workgroup
//   of one turn takes 11 of them: code that runs once and dependent reads.
// - 4 groups of drafted trees, 8 heads of 256, bf16, behind 1000 to 4000 rows: 33.6 us, 9 of
//   them the same, the others a chain of loads, two products and what is between them, of
//   one wave a SIMD.  (Long prefixes cut into more parts than short ones: no gain.)
// - 64 tokens, 32 heads of 128 over 8 KV heads, fp16, behind 8192 shared rows: 51.4 us; the
//   150 MB of their own rows alone take 34, which is memory.
// - Listed pages: a row's 64 of 16 rows, fp32, 11.7 us, 8.5 + 3.4; 16 rows' 64 of 32, fp16,
//   134 MB, 31.7 us (4.2 TB/s); 512 rows' 16 of 64, bf16, 537 MB 50.6 us (10.6 TB/s, half
//   of it from L2, half from the last-level cache).
//
// Lengths are read on the device; the host knows the rows, so it cuts keys into as
// many parts as fill the chip and a workgroup whose part is empty says so and ends.
#include "gemma_q8.h"
#include "gq8_lanes.hpp"
#include "gq8_paged.hpp"
#include "gq8_paged_rows.hpp"
#include "gq8_paged_tiles.hpp"

#include <algorithm>
#include <cmath>

namespace gq8 {
namespace {

constexpr int64_t kMostBlocks = (1 << 24) - 1; // of 256 threads a launch
constexpr int kUnit = 32;  // keys a unit
constexpr int kPairs = 32; // of a tile
constexpr int kWaves = 4;

// workgroups that are resident at once (32 keys and values a wave: 128 KB of LDS at 256 channels)
template <int HD>
constexpr int kResident = HD == 256 ? 256 : 512;

struct StreamArgs {
    PagedLayer layer;
    PackedSequences seq;
    const void *q;
    int q_stride, heads, kv_heads, head_dim, group;
    const uint16_t *k, *v; // the rows' own; null: the cache alone
    int kv_stride;
    const uint64_t *masks; // null: causal
    int mask_words;
    float scale;
    void *out;
    int out_stride;
    // sequences first[i] .. first[i + 1] - 1 share their first shared[i] cached rows
    int groups;
    const int *first, *shared;
    const int *list; // [rows, kv_heads, top] pages of a sequence
    int top;
    // parts of a row: prefix_parts of its prefix, then own_parts
    int tile_rows;                             // of own rows
    bool wide;                                 // the prefixes' tiles are of 64 pairs
    int prefix_rows, prefix_tiles, prefix_parts; // their rows, tiles at most, parts
    int prefix_eights;                         // their blocks, in eights; the others follow
    int list_jobs, list_eights;                // of lists, in eights where a row is one job
    int own_first, own_parts, parts;           // the first of this launch's others
    float *sums;   // [rows, heads, parts][HD]
    float4 *stats; // [rows, heads, parts]: reference, what its rounding left out, total
};

__device__ const word4 kZeroRow[64] = {}; // 1 KB: a row of any type

// A workgroup's tile and its place among the tile's parts.
struct Tile {
    int row, rows;   // packed rows
    int s;           // whose row of the table
    int skip, c;     // cached keys skip .. c - 1
    int i, start, n; // first row in its sequence, the sequence's first packed row and rows
    int g, part, parts, slot;
    bool prefix, shares; // a prefix's tile; an own tile whose sequence has a prefix
};

__device__ inline int start_of(const StreamArgs &p, int s)
{
    return min(max(p.seq.starts[s], 0), p.seq.rows);
}

__device__ inline int cached_of(const StreamArgs &p, int rows)
{
    return min(max(rows, 0), p.seq.table_width << p.layer.page_shift);
}

__device__ inline int tiles_of_rows(int n, int each)
{
    return n > 0 ? (int) ((uint32_t) (n + each - 1) / (uint32_t) each) : 0;
}

// first packed row and rows of prefix i's sequences
__device__ inline void rows_of_prefix(const StreamArgs &p, int i, int &a, int &start, int &n)
{
    a = min(max(p.first[i], 0), p.seq.sequences);
    const int b = min(max(p.first[i + 1], a), p.seq.sequences);
    start = start_of(p, a);
    n = max(start_of(p, b) - start, 0);
}

// `at`: this block's place among the prefixes'
__device__ inline bool prefix_tile(const StreamArgs &p, int at, Tile &tile)
{
    // every eighth block runs on one XCD: it takes jobs in a row, tiles that read the same keys
    const int job = (at & 7) * p.prefix_eights + (at >> 3);
    const int unit = job / p.prefix_tiles;
    if (unit >= p.prefix_parts * p.kv_heads)
        return false;
    int which, within;
    if (!find_part(job - unit * p.prefix_tiles, p.groups, [&](int i) {
            int a, start, n;
            rows_of_prefix(p, i, a, start, n);
            return cached_of(p, p.shared[i]) > 0 ? tiles_of_rows(n, p.prefix_rows) : 0;
        }, which, within))
        return false;
    int n;
    rows_of_prefix(p, which, tile.s, tile.row, n);
    tile.row += within * p.prefix_rows;
    tile.rows = min(p.prefix_rows, n - within * p.prefix_rows);
    tile.skip = 0;
    tile.c = cached_of(p, p.shared[which]);
    tile.i = tile.start = tile.n = 0;
    tile.g = unit / p.prefix_parts;
    tile.part = tile.slot = unit % p.prefix_parts;
    tile.parts = p.prefix_parts;
    tile.prefix = true;
    return true;
}

// Lane i's value of an array of `count`, the last one past it.
__device__ inline int lane_value(const int *values, int base, int count)
{
    return values[min(base + (int) (threadIdx.x & 63), count - 1)];
}

// An own tile: everything that is looked up by lanes is requested at once.
template <bool kList>
__device__ inline bool own_tile(const StreamArgs &p, int at, Tile &tile)
{
    const int lane = threadIdx.x & 63;
    if (kList && p.list_eights > 0) { // one KV head's rows after each other
        tile.part = 0;
        tile.g = (int) ((uint32_t) at / (uint32_t) p.seq.rows);
        at -= tile.g * p.seq.rows;
    } else {
        tile.part = at % p.own_parts;
        at /= p.own_parts;
        tile.g = at % p.kv_heads;
        at /= p.kv_heads; // the number of the row, or of the tile of rows
    }
    tile.parts = p.own_parts;
    tile.slot = p.prefix_parts + tile.part;
    tile.prefix = tile.shares = false;
    tile.skip = 0;
    int first = 0, next = 0, shared = 0;
    if (!kList && p.groups > 0) {
        first = lane_value(p.first, 0, p.groups);
        next = lane_value(p.first + 1, 0, p.groups);
        shared = lane_value(p.shared, 0, p.groups);
    }
    int tiles_before = 0;
    for (int base = 0;; base += 64) {
        if (base >= p.seq.sequences)
            return false;
        const bool mine = base + lane < p.seq.sequences;
        const int raw = lane_value(p.seq.starts, base, p.seq.sequences);
        const int start = min(max(raw, 0), p.seq.rows);
        const int end = min(max(lane_value(p.seq.starts + 1, base, p.seq.sequences), 0), p.seq.rows);
        const int cached = p.seq.cached ? lane_value(p.seq.cached, base, p.seq.sequences) : 0;
        uint64_t past;
        int upto = 0, tiles = 0;
        if constexpr (kList) { // the first sequence that ends behind the row
            past = __ballot(mine && end > at);
        } else {
            tiles = mine ? tiles_of_rows(end - start, p.tile_rows) : 0;
            upto = sum_upto(tiles);
            past = __ballot(mine && tiles_before + upto > at);
        }
        if (!past) {
            tiles_before += __builtin_amdgcn_readlane(upto, 63);
            continue;
        }
        const int found = __ffsll((unsigned long long) past) - 1;
        tile.s = base + found;
        tile.start = __builtin_amdgcn_readlane(start, found);
        tile.n = __builtin_amdgcn_readlane(end, found) - tile.start;
        tile.c = cached_of(p, __builtin_amdgcn_readlane(cached, found));
        if constexpr (kList) {
            if (__builtin_amdgcn_readlane(raw, found) > at)
                return false; // before the first sequence
            tile.row = at;
            tile.rows = 1;
            tile.i = at - tile.start;
        } else {
            const int within = at - tiles_before
                               - (__builtin_amdgcn_readlane(upto, found) - __builtin_amdgcn_readlane(tiles, found));
            tile.i = within * p.tile_rows;
            tile.row = tile.start + tile.i;
            tile.rows = min(p.tile_rows, tile.n - tile.i);
        }
        break;
    }
    if constexpr (!kList) // the rows of the prefix that it shares, if it is in one
        for (int base = 0; base < p.groups; base += 64) {
            if (base > 0) {
                first = lane_value(p.first, base, p.groups);
                next = lane_value(p.first + 1, base, p.groups);
                shared = lane_value(p.shared, base, p.groups);
            }
            const uint64_t in = __ballot(base + lane < p.groups && first <= tile.s && tile.s < next);
            if (in) {
                tile.skip = cached_of(p, __builtin_amdgcn_readlane(shared, __ffsll((unsigned long long) in) - 1));
                tile.shares = tile.skip > 0;
                break;
            }
        }
    return true;
}

__device__ inline word4 global_word4(const void *p)
{
    return *(const __attribute__((address_space(1))) word4 *) (uintptr_t) p;
}

// pair / group for pairs below 256 and groups up to 32: by = ceil(2^16 / group)
__device__ inline int divided(int pair, int by)
{
    return (int) ((uint32_t) (pair * by) >> 16);
}

// The queries of the tile's pairs into LDS, in the pieces that the products take; all
// waves of the workgroup, each some rows.
// Rows are read 16 bytes a lane: a lane a pair would touch 32 rows an instruction,
// which takes four times as long.  Few rows a round keep the code short, which counts
// where it runs once.
struct Staged {
    uint32_t pieces; // LDS address of the first
    int apart;       // and bytes to the second
};

template <int HD>
__device__ inline uint32_t query_chunk(Staged to, int piece, int row, int c)
{
    constexpr int kMask = HD / 8 < 16 ? HD / 8 - 1 : 15;
    return to.pieces + piece * to.apart + row * HD * 2 + ((c ^ (row & kMask)) << 4);
}

template <typename Q, int HD, typename F>
__device__ inline void stage_queries(const StreamArgs &p, const Tile &tile, int pairs, int by, Staged to,
                                     float *factors, F meanwhile)
{
    constexpr int LANES = HD * sizeof(Q) / 16, ROWS = 64 / LANES, EACH = 2; // of a row, an instruction, a round
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int channel = lane % LANES * (16 / (int) sizeof(Q));
    const float scale = p.scale * kLog2e;
    // every wave once at least, for what is done meanwhile
    const int begin = wave * EACH * ROWS;
#pragma unroll 1
    for (int base = begin; base == begin || base < pairs; base += kWaves * EACH * ROWS) {
        word4 x[EACH];
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            const int pair = min(base + j * ROWS + lane / LANES, pairs - 1), row = divided(pair, by);
            const Q *at = (const Q *) p.q + (int64_t) (tile.row + row) * p.q_stride
                          + (int64_t) (tile.g * p.group + pair - row * p.group) * p.head_dim + channel;
            x[j] = global_word4(channel < p.head_dim ? (const void *) at : (const void *) kZeroRow);
        }
        if (base == begin)
            meanwhile();
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            const int pair = min(base + j * ROWS + lane / LANES, pairs - 1);
            if constexpr (sizeof(Q) == 2) {
                lds_word4(query_chunk<HD>(to, 0, pair, lane % LANES), x[j] ^ (scale < 0.f ? 0x80008000u : 0u));
            } else {
                float largest = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    largest = fmaxf(largest, fabsf(__uint_as_float(x[j][i])));
                largest = max_lanes<LANES / 2>(largest);
                // 2^-e brings the largest to [2^13, 2^14), rows below 2^-87 near it
                const int e = max((int) ((__float_as_uint(largest) >> 23) & 0xFF) - 127 - 13, -100);
                const float down = ldexpf(scale < 0.f ? -1.f : 1.f, -e);
                factors[pair] = ldexpf(fabsf(scale), e);
                typedef uint32_t word2 __attribute__((ext_vector_type(2)));
                word2 pieces[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float two[2] = {__uint_as_float(x[j][2 * i]) * down, __uint_as_float(x[j][2 * i + 1]) * down};
                    uint32_t words[2];
                    Arithmetic<Q>::split(two, words);
                    pieces[0][i] = words[0];
                    pieces[1][i] = words[1];
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    *(__attribute__((address_space(3))) word2 *) (uintptr_t) (
                        query_chunk<HD>(to, i, pair, lane % LANES / 2) + lane % 2 * 8) = pieces[i];
            }
        }
    }
}

// A wave's operands from there: a lane holds pair first + lane % 32 (the last one where
// there are fewer), of every 16 channels 8 (lane / 32) .. + 7.
template <typename Q, int HD>
__device__ inline void take_queries(const StreamArgs &p, int first, int pairs, Staged from, const float *factors,
                                    State<Q, HD> &w)
{
    const int lane = threadIdx.x & 63, half = lane >> 5, pair = min(first + (lane & 31), pairs - 1);
    // never zero, so that a masked score (minus infinity) keeps its weight of zero
    w.c = fmaxf(sizeof(Q) == 4 ? factors[pair] : fabsf(p.scale * kLog2e), kLeast);
#pragma unroll
    for (int s = 0; s < HD / 16; ++s)
#pragma unroll
        for (int i = 0; i < State<Q, HD>::A::kPieces; ++i)
            w.q[s][i] = __builtin_bit_cast(typename State<Q, HD>::A::Operand,
                                           lds_word4(query_chunk<HD>(from, i, pair, 2 * s + half)));
    // 256 channels: to accumulation registers, where matrix instructions read them
    // as well; the others have to hold the sums
    if constexpr (HD == 256) {
#pragma unroll
        for (int s = 0; s < HD / 16; ++s)
#pragma unroll
            for (int i = 0; i < State<Q, HD>::A::kPieces; ++i)
                asm volatile("" : "+a"(w.q[s][i]));
    }
}

// Where a unit's 32 rows lie in a pool, keys and values alike: 16 rows that follow each
// other, of one page, take one address.
struct UnitRows {
    int row;          // the lane's (lanes 32 on repeat the first's), -1 for zeros
    bool cache;       // of the pool, not of the packed rows
    int stride;       // values
    uint64_t at[2];   // bytes to the first of 16 rows
    bool follow[2];
};

template <int HD>
__device__ inline UnitRows unit_rows(const StreamArgs &p, int row, bool cache, int channel)
{
    const int lane = threadIdx.x & 63;
    UnitRows rows{row, cache, cache ? p.layer.width : p.kv_stride, {}, {}};
    const uint64_t after = __ballot(row == __shfl(row, lane & 16) + (lane & 15));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int first = __builtin_amdgcn_readlane(row, 16 * i);
        rows.at[i] = (uint64_t) (((int64_t) first * rows.stride + channel) * 2);
        rows.follow[i] = p.head_dim == HD && first >= 0 && (after >> (16 * i) & 0xFFFF) == 0xFFFF;
    }
    return rows;
}

// Its rows 16 i .. 16 i + 15 of `pool`, HD / 32 loads.
template <int HD>
__device__ inline void load_half(const StreamArgs &p, const uint16_t *pool, const UnitRows &rows, int i, int channel,
                                 uint32_t to, Offsets<HD> &offsets)
{
    constexpr int kChunks = HD / 8, kRows = 64 / kChunks;
    const int lane = threadIdx.x & 63;
    const uint32_t area = to + i * 16 * HD * 2;
    if (i ? rows.follow[1] : rows.follow[0]) {
        if (rows.stride * 2 != offsets.stride)
            set_offsets(offsets, rows.stride * 2);
        load_follow<HD, 0, HD / 32>(uniform64((uint64_t) pool + (i ? rows.at[1] : rows.at[0])), offsets, area);
        return;
    }
#pragma unroll 1
    for (int j = 0; j < HD / 32; ++j) {
        const int r = j * kRows + lane / kChunks, c = (lane % kChunks ^ swizzle<HD>(r)) * 8;
        const int at = __shfl(rows.row, 16 * i + r);
        load_to_lds(at >= 0 && c < p.head_dim ? (const void *) (pool + (int64_t) at * rows.stride + channel + c)
                                              : (const void *) kZeroRow, area + j * 1024);
    }
}

template <int HD>
__device__ inline void load_unit(const StreamArgs &p, const uint16_t *pool, const UnitRows &rows, int channel,
                                 uint32_t to, Offsets<HD> &offsets)
{
#pragma unroll
    for (int i = 0; i < 2; ++i)
        load_half<HD>(p, pool, rows, i, channel, to, offsets);
}

// 0 x infinity is not 0: values that are not finite are taken out of a wave's unit
// where some of its pairs attend it in part, and each channel remembers the keys that
// had them: plus infinities and NaNs, minus infinities and NaNs.
template <typename Q, int HD>
__device__ inline bool take_out_unit(uint32_t values, uint64_t (*taken)[2])
{
    using A = Arithmetic<Q>;
    constexpr int kPieces = HD / 16; // KB of the unit
    const int lane = threadIdx.x & 63;
    uint32_t odd = 0;
#pragma unroll 4
    for (int j = 0; j < kPieces; ++j) {
        const word4 x = lds_word4(values + j * 1024 + lane * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) // an exponent of all ones and one carries into the sign
            odd |= (x[i] & A::kExponent) + A::kStep;
    }
    if (!__ballot((odd & 0x80008000u) != 0))
        return false;
    for (int c = lane; c < HD; c += 64)
        taken[c][0] = taken[c][1] = 0;
    __builtin_amdgcn_wave_barrier();
    for (int j = 0; j < kPieces * 8; ++j) {
        const int at = j * 64 + lane; // of the unit's values
        const int row = at / HD, chunk = (at % HD) / 8 ^ swizzle<HD>(row);
        auto *value = (__attribute__((address_space(3))) uint16_t *) (uintptr_t) (values + at * 2);
        const uint32_t x = *value, exponent = A::kExponent & 0xFFFFu;
        if ((x & exponent) == exponent) {
            const bool nan = (x & 0x7FFFu) != exponent;
            auto *words = (unsigned long long *) taken[chunk * 8 + at % 8];
            if (nan || !(x & 0x8000u))
                atomicOr(words, 1ull << row);
            if (nan || (x & 0x8000u))
                atomicOr(words + 1, 1ull << row);
            *value = 0;
        }
    }
    __builtin_amdgcn_wave_barrier();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    return true;
}

// A wave's loads of a unit are under way while it works on the one before: keys go to
// their half of the wave's area once the scores have read it, values to theirs once the
// second product has.  Loads end in the order of their requests, so of the last 2 n
// instructions (n of the keys, n of the values) "n are not done" means that the earlier
// n are.
template <int N>
__device__ inline void wait_loads()
{
    asm volatile("s_waitcnt vmcnt(%0)" :: "i"(N) : "memory");
}

// All waves have written (and read) what they would of LDS.  By hand, since the
// compiler's barrier waits for all loads too.
__device__ inline void lds_barrier()
{
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// A prefix's tile of 64 pairs: waves 0 and 1 take the units of even number, 2 and 3 the
// odd ones, each wave 32 of the pairs.  A unit is loaded by both of its waves, half
// of the rows each, into the one of their two areas that the unit before is not in, so
// there is a barrier a unit, after the waits for its loads and before the next one's are
// asked for.  Half the bytes of two tiles of 32: 4 groups of drafted trees, 8 heads of 256,
// bf16, 33.6 us for 35.5 (35.5 too with a unit's 16 loads in a row, which takes its four waves
// 1,100 cycles, at 64 bytes a clock: they go between the steps of the scores), 64 tokens of 32
// heads behind 8192 rows 51.4 for 53.2.  A turn takes some 4,600 cycles; of those, stamped (which
// adds to it), 800 to 1,600 wait for loads, 1,200 to 1,700 are places and barrier, 1,000 to 2,100
// products and the next loads, 1,400 to 1,700 what is between the products.
template <typename Q, int HD>
__device__ inline void wide_tile(const StreamArgs &p, const Tile &tile, uint32_t areas,
                                 float4 (&exchange)[kWaves][kPairs], float4 (&join_factors)[kWaves][kPairs])
{
    static_assert(Arithmetic<Q>::kPieces == 1, "no factors of the queries");
    constexpr int kArea = 2 * kUnit * HD * 2, kQuads = HD / 4;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), half = lane >> 5, key_lane = lane & 31;
    const int side = wave & 1, stream = wave >> 1; // of the pairs, of the units
    const int pairs = tile.rows * p.group, by = (65536 + p.group - 1) / p.group;
    const int units = (tile.c + kUnit - 1) / kUnit;
    int each = (int) ((uint32_t) (units + tile.parts - 1) / (uint32_t) tile.parts);
    each = (each + 1) & -2;
    const int begin = min(tile.part * each, units), end = min(units, begin + each);
    auto stat_of = [&](int pair) {
        const int row = divided(pair, by);
        return ((int64_t) (tile.row + row) * p.heads + tile.g * p.group + pair - row * p.group) * p.parts + tile.slot;
    };
    if (begin >= end) {
        for (int j = threadIdx.x; j < pairs; j += 256)
            p.stats[stat_of(j)] = float4{kLow, 0.f, 0.f, 0.f};
        return;
    }
    const int page_shift = p.layer.page_shift, page_mask = (1 << page_shift) - 1;
    int window = INT32_MAX, page_here = -1; // lane i's page is that of place window + i
    auto row_of = [&](int u) {
        const int key = u * kUnit;
        if (key >> page_shift < window || (key + kUnit - 1) >> page_shift > window + 63) {
            window = key >> page_shift;
            const int slot = window + lane;
            page_here = slot <= (tile.c - 1) >> page_shift ? p.seq.table[(int64_t) tile.s * p.seq.table_width + slot] : -1;
            asm volatile("" : "+v"(page_here)); // the wait for it (and all loads) is here alone
        }
        const int at = key + key_lane, page = __shfl(page_here, (at >> page_shift) - window);
        return (uint32_t) page < (uint32_t) p.layer.pages && at < tile.c ? (page << page_shift) + (at & page_mask) : -1;
    };
    const int channel = tile.g * p.head_dim;
    const uint32_t mine = areas + stream * 2 * kArea;
    Offsets<HD> offsets;
    set_offsets(offsets, p.layer.width * 2);
    auto load = [&](const UnitRows &rows, uint32_t to) {
        load_half<HD>(p, p.layer.keys, rows, side, channel, to, offsets);
        load_half<HD>(p, p.layer.values, rows, side, channel, to + kArea / 2, offsets);
    };
    int u = begin + stream;
    UnitRows rows{};
    // the first units go to areas 0 and 2, the queries to 1
    const Staged staged{areas + kArea, 0};
    stage_queries<Q, HD>(p, tile, pairs, by, staged, nullptr, [&] {
        if (u < end)
            rows = unit_rows<HD>(p, row_of(u), true, channel);
    });
    State<Q, HD> w;
    clear(w);
    if (u < end)
        load(rows, mine);
    lds_barrier();
    take_queries<Q, HD>(p, side * kPairs, pairs, staged, nullptr, w);
    uint32_t here = mine;
    for (int first = begin; first < end; first += 2, u += 2) { // all waves
        wait_loads<0>();
        lds_barrier();
        const uint64_t allowed = __ballot(rows.row >= 0) & 0xFFFFFFFFull;
        const uint32_t keys = here, values = here + kArea / 2;
        here = mine + (here == mine ? kArea : 0);
        bool between = false; // the next unit's loads go between the steps of the scores
        if (u + 2 < end) {
            rows = unit_rows<HD>(p, row_of(u + 2), true, channel);
            between = side ? rows.follow[1] : rows.follow[0];
            if (!between)
                load(rows, here);
        }
        if (u >= end)
            continue;
        float16v s[1];
        const uint64_t at = side ? rows.at[1] : rows.at[0];
        const uint64_t key_rows = uniform64((uint64_t) p.layer.keys + at), value_rows = uniform64((uint64_t) p.layer.values + at);
        const uint32_t to_keys = here + side * 16 * HD * 2, to_values = to_keys + kArea / 2;
        scores<Q, HD, 1>(w, keys, 0, s, [&](int i) {
            if (between)
                unrolled<HD / 32>([&](auto j) { // as many steps as loads
                    if (i == j)
                        load_to_lds<j * 1024>(key_rows, offsets.of[j], to_keys);
                    if (i == j + HD / 32)
                        load_to_lds<j * 1024>(value_rows, offsets.of[j], to_values);
                });
        });
        const bool masked = allowed != 0xFFFFFFFFull;
        float largest = masked ? largest_of(s, lane_bits(allowed, 0)) : largest_of(s);
        const bool far = refer(w, largest);
        const bool own = fabsf(w.reference) > kFar;
        const float minus = Arithmetic<Q>::kShift - (own ? 0.f : w.reference);
        if (masked || far) {
            const uint64_t bits = lane_bits(allowed, 0);
            const float raw = own ? w.raw : 0.f;
#pragma unroll
            for (int j = 0; j < 16; ++j)
                s[0][j] = (bits >> score_bit(j)) & 1 ? s[0][j] - raw : -INFINITY;
        }
        Weights<Q, 1> weights;
        exponentiate(w, s, weights, minus);
        weigh<Q, HD, 1, false>(w, values, 0, weights, s, largest);
    }

    float total = w.before + (w.total[0] + w.total[1]);
    total += xor_lane<32>(total);
    if (half == 0)
        exchange[wave][lane] = float4{w.reference, beside(w.reference, w.raw, w.c), total, 0.f};
    lds_barrier(); // all have read their units
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) {
        const float16v &x = w.sums[j / 4];
        const int i = j % 4 * 4;
        const float four[4] = {x[i], x[i + 1], x[i + 2], x[i + 3]};
        lds_word4(areas + wave * kArea + (lane & 31) * HD * 4 + (((2 * j + half) ^ (lane & 15)) << 4),
                  __builtin_bit_cast(word4, four));
    }
    __syncthreads();
    // pair i: waves i / 32 and i / 32 + 2
    {
        const float4 a = exchange[lane >> 5][lane & 31], b = exchange[(lane >> 5) + 2][lane & 31];
        const bool past = b.x - a.x + (b.y - a.y) > 0.f;
        const float m = past ? b.x : a.x, rest = past ? b.y : a.y;
        const float2 by_two = {__builtin_amdgcn_exp2f(a.x - m + (a.y - rest)), __builtin_amdgcn_exp2f(b.x - m + (b.y - rest))};
        ((float2 *) join_factors)[wave * 64 + lane] = by_two;
        if (wave == 0 && lane < pairs)
            p.stats[stat_of(lane)] = float4{m, rest, a.z * by_two.x + b.z * by_two.y, 0.f};
    }
    __builtin_amdgcn_wave_barrier();
    const int quad = threadIdx.x % kQuads;
    if (quad * 4 >= p.head_dim)
        return;
#pragma unroll 2
    for (int of = threadIdx.x / kQuads; of < pairs; of += 256 / kQuads) {
        const float2 factor = ((const float2 *) join_factors)[wave * 64 + of];
        const uint32_t at = areas + (of >> 5) * kArea + (of & 31) * HD * 4 + ((quad ^ (of & 15)) << 4);
        const float4v a = __builtin_bit_cast(float4v, lds_word4(at)), b = __builtin_bit_cast(float4v, lds_word4(at + 2 * kArea));
        *(float4v *) (p.sums + stat_of(of) * HD + quad * 4) = a * factor.x + b * factor.y;
    }
}

template <typename Q, int HD, bool kList>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(HD == 256 ? 1 : 2)))
void stream_kernel(StreamArgs p)
{
    constexpr int kTile = kUnit * HD * 2, kArea = 2 * kTile; // a wave's: keys and values, or 32 pairs of HD floats
    constexpr int kLoads = HD / 16, kQuads = HD / 4;
    __shared__ __align__(1024) uint8_t lds[kWaves * kArea];
    __shared__ float4 exchange[kWaves][kPairs];
    __shared__ float query_factors[kPairs];
    __shared__ float4 join_factors[kWaves][kPairs];
    __shared__ float join_over[kWaves][kPairs];
    __shared__ uint64_t taken[kList ? 1 : kWaves][kList ? 1 : HD][2];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), half = lane >> 5, key_lane = lane & 31;
    Tile tile;
    const bool is_prefix = !kList && (int) blockIdx.x < p.prefix_eights * 8;
    int at = (int) blockIdx.x - (is_prefix ? 0 : p.prefix_eights * 8 - p.own_first);
    if constexpr (kList)
        // Every eighth block runs on one XCD: it takes jobs in a row, which are one KV head's
        // rows after each other, since rows next to each other list much the same pages.  (512
        // rows of 8 heads of 256 that change 2 of their 16 pages from row to row, of 60000
        // rows: 40.5 us, 51.4 with rows over all XCDs; pages at random 70.8 and 71.6.  Rows of
        // all KV heads in a row: 1037 for 622, 1000 rows of 8 KV heads.)
        if (p.list_eights > 0) {
            const int job = (int) (blockIdx.x & 7) * p.list_eights + (int) (blockIdx.x >> 3);
            if (job >= p.list_jobs)
                return;
            at = p.own_first + job;
        }
    if (!(is_prefix ? prefix_tile(p, at, tile) : own_tile<kList>(p, at, tile)))
        return;
    if constexpr (!kList && sizeof(Q) == 2)
        if (is_prefix && p.wide) {
            wide_tile<Q, HD>(p, tile, uniform(lds_address(lds)), exchange, join_factors);
            return;
        }
    const int pairs = tile.rows * p.group, by = (65536 + p.group - 1) / p.group;

    // the tile's units, and the run of them that is this workgroup's
    int cached_units, units, own_keys = 0;
    if constexpr (kList) {
        cached_units = units = (int) (((int64_t) p.top << p.layer.page_shift) + kUnit - 1) / kUnit;
    } else {
        cached_units = (max(tile.c - tile.skip, 0) + kUnit - 1) / kUnit;
        if (!is_prefix && p.k)
            own_keys = p.masks ? min(tile.n, p.mask_words * 64) : min(tile.n, tile.i + tile.rows);
        units = cached_units + (own_keys + kUnit - 1) / kUnit;
    }
    int each = (int) ((uint32_t) (units + tile.parts - 1) / (uint32_t) tile.parts);
    each = (each + kWaves - 1) & -kWaves;
    const int begin = min(tile.part * each, units), end = min(units, begin + each);
    auto stat_of = [&](int pair, int slot) {
        const int row = divided(pair, by);
        return ((int64_t) (tile.row + row) * p.heads + tile.g * p.group + pair - row * p.group) * p.parts + slot;
    };
    if (!kList && !is_prefix && tile.part == 0 && !tile.shares) // nobody else fills these
        for (int j = threadIdx.x; j < pairs * p.prefix_parts; j += 256)
            p.stats[stat_of(j / p.prefix_parts, j % p.prefix_parts)] = float4{kLow, 0.f, 0.f, 0.f};
    if (begin >= end && p.parts > 1) {
        for (int j = threadIdx.x; j < pairs; j += 256)
            p.stats[stat_of(j, tile.slot)] = float4{kLow, 0.f, 0.f, 0.f};
        return;
    }

    // ---- where the lane's key of a unit is.  Lane i holds entry `window` + i: its page
    // of the pool, and of a list which page of the sequence it is.
    const int page_shift = p.layer.page_shift, page_mask = (1 << page_shift) - 1;
    const int position = tile.c + tile.i; // of a list's row; the host keeps it in 32 bits
    const int first_key = kList ? 0 : tile.skip;
    int window = INT32_MAX, page_here = -1, slot_here = -1;
    auto look_up = [&](int entry) { // pages of the entries from `entry` on
        window = entry;
        const int at = entry + lane;
        if constexpr (kList)
            slot_here = at < p.top ? p.list[((int64_t) tile.row * p.kv_heads + tile.g) * p.top + at] : -1;
        else
            slot_here = at;
        const bool there = slot_here >= 0 && slot_here < p.seq.table_width
                           && (kList || slot_here <= (tile.c - 1) >> page_shift);
        page_here = there ? p.seq.table[(int64_t) tile.s * p.seq.table_width + slot_here] : -1;
        slot_here = there ? slot_here : -1;
        asm volatile("" : "+v"(page_here)); // the wait for it (and all loads) is here alone
    };
    auto row_of = [&](int u) { // -1: none
        if (u >= cached_units) {
            const int j = (u - cached_units) * kUnit + key_lane;
            return j < own_keys ? tile.start + j : -1;
        }
        const int key = first_key + u * kUnit;
        if (key >> page_shift < window || (key + kUnit - 1) >> page_shift > window + 63)
            look_up(key >> page_shift);
        const int at = key + key_lane, entry = (at >> page_shift) - window;
        const int page = __shfl(page_here, entry);
        bool there = (uint32_t) page < (uint32_t) p.layer.pages;
        if constexpr (kList) {
            const int slot = __shfl(slot_here, entry);
            there = there && slot >= 0 && (slot << page_shift) + (at & page_mask) <= position;
        } else {
            there = there && at < tile.c;
        }
        return there ? (page << page_shift) + (at & page_mask) : -1;
    };
    const int channel = tile.g * p.head_dim;
    const uint32_t areas = uniform(lds_address(lds)), keys = areas + wave * kArea, values = keys + kTile;
    Offsets<HD> offsets;
    set_offsets(offsets, p.layer.width * 2);
    auto load_keys = [&](const UnitRows &rows) {
        load_unit<HD>(p, rows.cache ? p.layer.keys : p.k, rows, channel, keys, offsets);
    };
    auto load_values = [&](const UnitRows &rows) {
        load_unit<HD>(p, rows.cache ? p.layer.values : p.v, rows, channel, values, offsets);
    };

    // The queries pass through LDS while the pages are looked up and the first keys come.
    const bool live = (lane & 31) < pairs;
    const int pair_row = divided(min(lane & 31, pairs - 1), by); // of the tile
    int u = begin + wave;
    UnitRows rows{};
    const Staged staged{areas + kTile, kArea}; // where the values of waves 0 and 1 will be
    stage_queries<Q, HD>(p, tile, pairs, by, staged, query_factors, [&] {
        if (u < end)
            rows = unit_rows<HD>(p, row_of(u), u < cached_units, channel);
    });
    State<Q, HD> w;
    clear(w);
    if (u < end)
        load_keys(rows);
    lds_barrier();
    take_queries<Q, HD>(p, 0, pairs, staged, query_factors, w);
    lds_barrier();
    if (u < end) {
        load_values(rows);
        for (;;) {
            const int next = u + kWaves;
            const bool more = next < end;
            wait_loads<kLoads>(); // the keys
            float16v s[1];
            scores<Q, HD, 1>(w, keys, 0, s, [](int) {});
            uint64_t allowed = __ballot(rows.row >= 0) & 0xFFFFFFFFull;
            if (more) {
                rows = unit_rows<HD>(p, row_of(next), next < cached_units, channel);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // the keys are read
                load_keys(rows);
            }
            bool masked = allowed != 0xFFFFFFFFull, took = false;
            if constexpr (!kList) {
                if (u >= cached_units) {
                    const int key = (u - cached_units) * kUnit; // of the sequence's own rows
                    masked = true;
                    if (p.masks) {
                        allowed &= p.masks[(int64_t) (tile.row + pair_row) * p.mask_words + key / 64] >> (key & 32);
                    } else {
                        const int last = tile.i + pair_row - key;
                        allowed &= last >= 31 ? ~0ull : last < 0 ? 0 : (2ull << last) - 1;
                    }
                }
            }
            if (more) // the values
                wait_loads<kLoads>();
            else
                wait_loads<0>();
            if constexpr (!kList)
                if (u >= cached_units)
                    took = take_out_unit<Q, HD>(values, taken[wave]);
            float largest = masked ? largest_of(s, lane_bits(allowed, 0)) : largest_of(s);
            const bool far = refer(w, largest);
            const bool own = fabsf(w.reference) > kFar;
            const float minus = Arithmetic<Q>::kShift - (own ? 0.f : w.reference);
            if (masked || far) {
                const uint64_t bits = lane_bits(allowed, 0);
                const float raw = own ? w.raw : 0.f;
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    s[0][j] = (bits >> score_bit(j)) & 1 ? s[0][j] - raw : -INFINITY;
            }
            if constexpr (!kList)
                if (took)
                    put_back(w, taken[wave], allowed);
            Weights<Q, 1> weights;
            exponentiate(w, s, weights, minus);
            weigh<Q, HD, 1, false>(w, values, 0, weights, s, largest);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // the values are read
            if (!more)
                break;
            u = next;
            load_values(rows);
        }
    }

    // ---- the waves' sums of each pair through their areas
    float total = w.before + (w.total[0] + w.total[1]);
    total += xor_lane<32>(total);
    if (half == 0)
        exchange[wave][lane] = float4{w.reference, beside(w.reference, w.raw, w.c), total, 0.f};
    if (live)
#pragma unroll
        for (int j = 0; j < HD / 8; ++j) {
            const float16v &x = w.sums[j / 4];
            const int i = j % 4 * 4;
            const float four[4] = {x[i], x[i + 1], x[i + 2], x[i + 3]};
            lds_word4(keys + (lane & 31) * HD * 4 + (((2 * j + half) ^ (lane & 15)) << 4), __builtin_bit_cast(word4, four));
        }
    __syncthreads();
    // Lane i (and i + 32): how the waves' sums of pair i are joined, each wave for itself.
    {
        const int pair = min(lane & 31, pairs - 1);
        float4 stat[kWaves];
#pragma unroll
        for (int k = 0; k < kWaves; ++k)
            stat[k] = exchange[k][pair];
        float m = stat[0].x, rest = stat[0].y, sum = 0.f, factor[kWaves];
#pragma unroll
        for (int k = 1; k < kWaves; ++k) { // the largest reference
            const bool past = stat[k].x - m + (stat[k].y - rest) > 0.f;
            m = past ? stat[k].x : m;
            rest = past ? stat[k].y : rest;
        }
#pragma unroll
        for (int k = 0; k < kWaves; ++k) {
            factor[k] = __builtin_amdgcn_exp2f(stat[k].x - m + (stat[k].y - rest));
            sum += stat[k].z * factor[k];
        }
        if (half == 0) {
            join_factors[wave][lane] = float4{factor[0], factor[1], factor[2], factor[3]};
            join_over[wave][lane] = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
        }
        if (p.parts > 1 && wave == 0 && lane < pairs)
            p.stats[stat_of(lane, tile.slot)] = float4{m, rest, sum, 0.f};
    }
    __builtin_amdgcn_wave_barrier();
    // a thread takes four channels of every 256 / kQuads-th pair
    const int quad = threadIdx.x % kQuads;
    if (quad * 4 >= p.head_dim)
        return;
#pragma unroll 2
    for (int of = threadIdx.x / kQuads; of < pairs; of += 256 / kQuads) {
        const float4 factor = join_factors[wave][of];
        const float over = join_over[wave][of];
        float4v sums[kWaves], x;
#pragma unroll
        for (int k = 0; k < kWaves; ++k)
            sums[k] = __builtin_bit_cast(float4v, lds_word4(areas + k * kArea + of * HD * 4 + ((quad ^ (of & 15)) << 4)));
#pragma unroll
        for (int i = 0; i < 4; ++i)
            x[i] = ((sums[0][i] * factor.x + sums[1][i] * factor.y) + sums[2][i] * factor.z) + sums[3][i] * factor.w;
        if (p.parts == 1) {
            const int row = divided(of, by);
            Q *out = (Q *) p.out + (int64_t) (tile.row + row) * p.out_stride
                     + (int64_t) (tile.g * p.group + of - row * p.group) * p.head_dim + quad * 4;
            typedef Q Q4 __attribute__((ext_vector_type(4)));
            *(Q4 *) out = Q4{(Q) (x[0] * over), (Q) (x[1] * over), (Q) (x[2] * over), (Q) (x[3] * over)};
        } else {
            *(float4v *) (p.sums + stat_of(of, tile.slot) * HD + quad * 4) = x;
        }
    }
}

// Joins the parts of each row and head.  A wave takes a pair (of many parts a quarter
// of them): lane i the statistics of part i, so the common reference and every part's
// factor are there at once, then all lanes the channels of the parts that hold any.
constexpr int kFewParts = 16;

template <typename Q, int HD>
__global__ __launch_bounds__(256) void merge_parts_kernel(StreamArgs p, int first)
{
    constexpr int EACH = HD / 64;
    typedef float Some __attribute__((ext_vector_type(EACH)));
    __shared__ float others[3][HD + 3];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const bool split = p.parts > kFewParts;
    const unsigned of = split ? blockIdx.x : blockIdx.x * 4 + wave; // rows and heads from row `first` on
    const int row = first + (int) (of / (unsigned) p.heads), head = (int) (of % (unsigned) p.heads);
    const int64_t pair = (int64_t) row * p.heads + head;
    if (row >= p.seq.rows || row < start_of(p, 0) || row >= start_of(p, p.seq.sequences))
        return; // of all the block's waves where they share a pair
    const int each = split ? (p.parts + 3) / 4 : p.parts;
    const int begin = split ? wave * each : 0, end = min(p.parts, begin + each);
    float m = kLow, rest = 0.f, total = 0.f;
    Some sums = {};
    for (int base = begin; base < end; base += 64) {
        const bool there = base + lane < end;
        const float4 stat = there ? p.stats[pair * p.parts + base + lane] : float4{kLow, 0.f, 0.f, 0.f};
        const uint64_t held = __ballot(stat.z != 0.f);
        // the largest reference, and of those at it the one with the most left out
        const float most = max_lanes<32>(stat.x);
        const float most_rest = max_lanes<32>(stat.x == most ? stat.y : -INFINITY);
        const Factors by = factors(m, rest, most, most_rest);
        const float factor = __builtin_amdgcn_exp2f(stat.x - most + (stat.y - most_rest));
        const float sum = sum_lanes<32>(stat.z != 0.f ? stat.z * factor : 0.f);
        total = total * by.a + sum * by.b;
        Some more = {};
        for (uint64_t left = held; left;) {
            Some x[4];
            float f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int part = left ? __ffsll((unsigned long long) left) - 1 : 0;
                f[i] = left ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(factor), part)) : 0.f;
                x[i] = left ? *(const Some *) (p.sums + (pair * p.parts + base + part) * HD + lane * EACH) : Some{};
                left &= left - 1;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                more += x[i] * f[i];
        }
        sums = sums * by.a + more * by.b;
        m = by.m;
        rest = by.rest;
    }
    if (split) {
        if (wave > 0) {
#pragma unroll
            for (int i = 0; i < EACH; ++i)
                others[wave - 1][lane * EACH + i] = sums[i];
            if (lane == 0) {
                others[wave - 1][HD] = m;
                others[wave - 1][HD + 1] = rest;
                others[wave - 1][HD + 2] = total;
            }
        }
        __syncthreads();
        if (wave > 0)
            return;
        for (int v = 0; v < 3; ++v) {
            const Factors by = factors(m, rest, others[v][HD], others[v][HD + 1]);
            total = total * by.a + others[v][HD + 2] * by.b;
#pragma unroll
            for (int i = 0; i < EACH; ++i)
                sums[i] = sums[i] * by.a + others[v][lane * EACH + i] * by.b;
            m = by.m;
            rest = by.rest;
        }
    }
    const float by = total > 0.f || total != total ? 1.f / total : 0.f;
    if (lane * EACH >= p.head_dim)
        return;
    typedef Q Out __attribute__((ext_vector_type(EACH)));
    Out x;
#pragma unroll
    for (int i = 0; i < EACH; ++i)
        x[i] = (Q) (sums[i] * by);
    *(Out *) ((Q *) p.out + (int64_t) row * p.out_stride + (int64_t) head * p.head_dim + lane * EACH) = x;
}

int padded_head_dim(int head_dim)
{
    return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
}

// ---- how keys are cut ------------------------------------------------------------------
constexpr int kMostPrefixParts = 128, kMostOwnParts = 32;

int rows_of_tile(int group, bool wide = false)
{
    return (wide ? 2 * kPairs : kPairs) / group;
}

// Tiles of 32 pairs (of all KV heads) from which on prefixes take tiles of 64 where queries
// are of 16 bits: half as many, each in twice the parts.  us of single tokens behind 16000
// rows, 32 and 64 pairs a tile, with 16, 32, 64 and 128 tiles of 32:
//   8 heads of 256, bf16:                 40 41, 68 65, 121 113, 227 210
//   32 heads of 128 over 8 KV heads, fp16: 22 22, 33 30, 54 48, 95 84
// and behind 4000: 20 22, 27 29, 40 40, 68 65 and 16 18, 17 18, 22 23, 37 36.  fp32 queries, whose
// products are twice as many, gain nothing (24 28, 33 36, 49 51, 85 84).
constexpr int kWideFrom = 64;

bool takes_wide(int64_t tiles, int kv_heads, bool queries16)
{
    return queries16 && tiles * kv_heads >= kWideFrom;
}

int resident(int head_dim)
{
    return padded_head_dim(head_dim) == 256 ? kResident<256> : kResident<128>;
}

// Parts that bring `tiles` tiles of each KV head to `workgroups`, or just past it.
int parts_for(int64_t tiles, int kv_heads, int workgroups, int most)
{
    return (int) std::clamp<int64_t>((workgroups + tiles * kv_heads - 1) / (tiles * kv_heads), 1, most);
}

// Parts of a prefix for half of what is resident.
int prefix_parts_of(int64_t tiles, int kv_heads, int head_dim, bool wide)
{
    return std::min((wide ? 2 : 1) * parts_for(tiles, kv_heads, resident(head_dim) / 2, kMostPrefixParts), kMostPrefixParts);
}

// Tiles of n rows that belong to `owners`, at most: a part of one's last tile is empty.
int64_t tiles_of(int64_t n, int64_t owners, int tile_rows)
{
    return (n + std::min(owners, n) * (tile_rows - 1)) / tile_rows;
}

template <typename Q, int HD, bool kList>
hipError_t launch(StreamArgs p, int64_t own_tiles, hipStream_t stream)
{
    const int64_t prefix_eights = ((int64_t) p.prefix_tiles * p.prefix_parts * p.kv_heads + 7) / 8;
    const int64_t own_blocks = own_tiles * p.kv_heads * p.own_parts;
    if (prefix_eights * 8 >= kMostBlocks / 8 * 8 || own_blocks > INT32_MAX)
        return hipErrorInvalidValue;
    p.prefix_eights = (int) prefix_eights;
    for (int64_t at = 0; at < own_blocks;) { // the prefixes' with the first of them
        const int64_t some = std::min(own_blocks - at, kMostBlocks / 8 * 8 - p.prefix_eights * 8);
        p.own_first = (int) at;
        p.list_jobs = (int) some;
        p.list_eights = kList && p.own_parts == 1 ? (int) ((some + 7) / 8) : 0;
        const int64_t blocks = p.list_eights > 0 ? p.list_eights * 8 : p.prefix_eights * 8 + some;
        hipLaunchKernelGGL((stream_kernel<Q, HD, kList>), dim3((unsigned) blocks), dim3(256), 0, stream, p);
        if (hipError_t s = hipGetLastError())
            return s;
        p.prefix_eights = 0;
        at += some;
    }
    if (p.parts > 1) {
        const int64_t each = p.parts > kFewParts ? 1 : 4; // pairs a block
        const int64_t most_rows = kMostBlocks / p.heads * each;
        if (most_rows < 1)
            return hipErrorInvalidValue;
        for (int64_t first = 0; first < p.seq.rows; first += most_rows) {
            const int64_t pairs = std::min(p.seq.rows - first, most_rows) * p.heads;
            hipLaunchKernelGGL((merge_parts_kernel<Q, HD>), dim3((unsigned) ((pairs + each - 1) / each)), dim3(256), 0,
                               stream, p, (int) first);
            if (hipError_t s = hipGetLastError())
                return s;
        }
    }
    return hipSuccess;
}

template <bool kList>
hipError_t launch_type(StreamArgs p, int64_t own_tiles, int q_type, float *workspace, hipStream_t stream)
{
    const int hd = padded_head_dim(p.head_dim);
    p.sums = workspace;
    p.stats = (float4 *) (workspace + (int64_t) p.seq.rows * p.heads * p.parts * hd);
    auto width = [&](auto q) {
        typedef decltype(q) Q;
        switch (hd) {
        case 64: return launch<Q, 64, kList>(p, own_tiles, stream);
        case 128: return launch<Q, 128, kList>(p, own_tiles, stream);
        default: return launch<Q, 256, kList>(p, own_tiles, stream);
        }
    };
    switch (q_type) {
    case GQ8_DTYPE_F32: return width(0.f);
    case GQ8_DTYPE_F16: return width((_Float16) 0.f);
    case GQ8_DTYPE_BF16: return width((__bf16) 0.f);
    default: return hipErrorInvalidValue;
    }
}

// Sequences whose rows fill tiles of 128 pairs by themselves gain nothing from sharing
// but a part of what they read: their own attention is faster then, over the same rows
// in their own pages, and sooner where nothing is shared.  us, here and there:
//   16 sequences behind 8000 rows, 8 heads of 256, bf16: 64 pairs each 40, 43; 80 41, 44;
//   96 49, 45; 128 67, 49.  fp32: 80 50, 53; 96 60, 55.  40 of them behind 4000, bf16: 80 50,
//   49; 96 56, 49.  32 heads of 128 over 8 KV heads, fp16: 64 95, 100; 80 110, 100.
//   8 sequences of 4000 rows that share nothing, those heads: 48 54, 39.  Single tokens and
//   4 of 8 heads of 256 (16 sequences of 1024 rows, fp32): 16 and 19 here, 28 and 29 there.
// Few rows in all leave its tiles to too few workgroups: 4 sequences behind 4000, 256 pairs
// each, 28 and 37, 512 pairs 41 and 36.
bool fills_tiles(int64_t rows, int heads, int group, int sequences, bool shares)
{
    return rows * heads >= 2048 && rows * group >= (int64_t) (shares ? 96 : 48) * sequences;
}

// Sums and statistics of `row_parts` parts (rows times parts of a row), all heads; past 64
// bits more than any workspace holds.
size_t bytes_of(int64_t row_parts, int heads, int head_dim)
{
    int64_t bytes;
    if (__builtin_mul_overflow(row_parts, (int64_t) heads * (padded_head_dim(head_dim) + 4) * 4, &bytes)
        || __builtin_add_overflow(bytes, (int64_t) 256, &bytes))
        return SIZE_MAX;
    return (size_t) bytes;
}

// Rows times parts_for(their tiles) at most, for any number of rows up to `rows`: fewer rows
// are cut into more parts, and a workspace for many has to hold them too.  Of r rows in
// t >= r / tile_rows tiles, ceil(w / (t k)) <= (w - 1) / (t k) + 1 parts, times r, are at most
// r + tile_rows (w - 1) / k.
int64_t most_row_parts(int64_t rows, int tile_rows, int kv_heads, int workgroups, int most)
{
    return std::min(rows * most, rows + (int64_t) tile_rows * (workgroups - 1) / kv_heads);
}

bool good(const StreamArgs &p)
{
    return p.seq.sequences > 0 && p.seq.rows > 0 && p.kv_heads > 0 && p.group > 0 && p.group <= kPairs
           && p.heads == p.group * p.kv_heads && p.head_dim > 0 && p.head_dim <= kPagedMaxHeadDim
           && p.head_dim % 8 == 0;
}

} // namespace

size_t prefix_attention_workspace_bytes(int64_t rows, int heads, int kv_heads, int head_dim)
{
    const int tile_rows = rows_of_tile(heads / kv_heads), all = resident(head_dim);
    // twice the parts from where on prefixes may take tiles of 64 pairs
    const bool wide = takes_wide(tiles_of(rows, rows, tile_rows), kv_heads, true);
    const int64_t prefixes = std::min((wide ? 2 : 1) * most_row_parts(rows, tile_rows, kv_heads, all / 2, kMostPrefixParts),
                                      rows * kMostPrefixParts);
    const size_t own = bytes_of(prefixes + most_row_parts(rows, tile_rows, kv_heads, all, kMostOwnParts), heads, head_dim);
    return fills_tiles(rows, heads, heads / kv_heads, 1, false)
               ? std::max(own, packed_attention_workspace_bytes(heads, kv_heads, head_dim)) : own;
}

size_t sparse_attention_workspace_bytes(int64_t rows, int heads, int kv_heads, int head_dim)
{
    // rows that fill the chip by themselves have one part, which needs no workspace
    const int all = resident(head_dim);
    return bytes_of(most_row_parts(std::min<int64_t>(rows, (all - 1) / kv_heads), 1, kv_heads, all, kMostOwnParts), heads,
                    head_dim);
}

hipError_t launch_prefix_attention(const PackedAttentionArgs &a, int groups, const int *first, const int *shared,
                                   int q_type, hipStream_t stream)
{
    StreamArgs p{};
    p.layer = a.layer;
    p.seq = a.seq;
    p.q = a.q;
    p.q_stride = a.q_stride;
    p.heads = a.heads;
    p.kv_heads = a.kv_heads;
    p.head_dim = a.head_dim;
    p.group = a.kv_heads > 0 ? a.heads / a.kv_heads : 0;
    p.k = a.k;
    p.v = a.v;
    p.kv_stride = a.kv_stride;
    p.masks = a.causal ? nullptr : a.masks;
    p.mask_words = a.mask_words;
    p.scale = a.scale;
    p.out = a.out;
    p.out_stride = a.out_stride;
    if (!good(p) || groups < 0 || !a.workspace)
        return hipErrorInvalidValue;
    const int64_t rows = a.seq.rows;
    if (fills_tiles(rows, a.heads, p.group, a.seq.sequences, groups > 0)) {
        PackedAttentionArgs packed = a;
        packed.causal = a.causal && a.k;
        return launch_packed_attention(packed, q_type, stream);
    }
    p.groups = groups;
    p.first = first;
    p.shared = shared;
    p.tile_rows = rows_of_tile(p.group);
    const int64_t own_tiles = tiles_of(rows, a.seq.sequences, p.tile_rows);
    const int64_t keys = a.seq.cached ? (int64_t) a.seq.table_width << a.layer.page_shift : 0;
    // Prefixes have half of what is resident and come first; the own rows, bound by memory,
    // run beside them.  (All of it for the prefixes: 64 tokens behind 8192 rows 58.6 us, 53.6
    // with half; blocks of both kinds in turn 65 where it was 60, the drafted trees 61 for 38.)
    if (groups > 0) {
        const int64_t tiles = tiles_of(rows, groups, p.tile_rows);
        p.wide = takes_wide(tiles, p.kv_heads, q_type != GQ8_DTYPE_F32);
        p.prefix_rows = rows_of_tile(p.group, p.wide);
        p.prefix_tiles = (int) tiles_of(rows, groups, p.prefix_rows);
        p.prefix_parts = (int) std::min<int64_t>(
            prefix_parts_of(tiles, p.kv_heads, p.head_dim, p.wide),
            std::max<int64_t>(1, (keys + kUnit * kWaves - 1) / (kUnit * kWaves)));
    }
    p.own_parts = parts_for(own_tiles, p.kv_heads, resident(p.head_dim) / (groups > 0 ? 4 : 1), kMostOwnParts);
    p.parts = p.prefix_parts + p.own_parts;
    return launch_type<false>(p, own_tiles, q_type, a.workspace, stream);
}

hipError_t launch_sparse_attention(const PackedAttentionArgs &a, const int *list, int top, int q_type,
                                   hipStream_t stream)
{
    StreamArgs p{};
    p.layer = a.layer;
    p.seq = a.seq;
    p.q = a.q;
    p.q_stride = a.q_stride;
    p.heads = a.heads;
    p.kv_heads = a.kv_heads;
    p.head_dim = a.head_dim;
    p.group = a.kv_heads > 0 ? a.heads / a.kv_heads : 0;
    p.scale = a.scale;
    p.out = a.out;
    p.out_stride = a.out_stride;
    p.list = list;
    p.top = top;
    if (!good(p) || top <= 0 || !a.workspace)
        return hipErrorInvalidValue;
    const int64_t units = (((int64_t) top << a.layer.page_shift) + kUnit - 1) / kUnit;
    p.tile_rows = 1;
    p.own_parts = (int) std::min<int64_t>(parts_for(a.seq.rows, p.kv_heads, resident(p.head_dim), kMostOwnParts),
                                          (units + kWaves - 1) / kWaves);
    p.parts = p.own_parts;
    return launch_type<true>(p, a.seq.rows, q_type, a.workspace, stream);
}

} // namespace gq8
