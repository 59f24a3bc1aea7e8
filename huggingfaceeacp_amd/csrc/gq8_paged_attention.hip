// gq8_paged_attention.hip -- attention of packed sequences over a paged cache
// and their own rows: causal (prompts), or by a word of mask bits a row (trees
// of drafted tokens, single tokens).
//
// Mathematics.  Row i of a sequence, query head h, KV head h / group:
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c q.k_j - m),  c = scale log2(e),
// over every cached row and the new rows that the mask leaves; m is a running
// reference of the row's scores.  One pass over the keys with p, m and the sums
// in registers (32 bits); m moves, and the sums are rescaled, only where a
// tile's maximum passes it by more than kMargin.  A row that attends nothing
// is zeros.
//
// Work.  A tile of query rows is up to M (row, head) pairs of one KV head, so
// a group's heads share the keys they read.  A unit is 64 keys for one tile;
// the units of all sequences, KV heads and tiles in a row are cut into equal
// runs, one a workgroup, whatever the lengths are (they are read on the
// device).  A workgroup writes the tiles that it holds whole; of a tile that
// others share it leaves its sums, and merge_kernel joins those in the order
// of the keys, so results do not depend on which workgroup ends first.
//
// Matrix instructions.  S^T = K Q^T with v_mfma_f32_32x32x16: lane l holds the
// scores of pair l % 32 against keys 8 (i / 4) + 4 (l / 32) + i % 4, i = 0..15.
// O^T = V^T P^T contracts over keys in whatever order both operands agree on,
// so a lane's own 8 scores of a 16-key step are its B operand as they stand:
// P never moves between lanes, and a row's statistics are its lane's registers
// and one exchange with lane ^ 32.  V^T comes from the row-major tile by
// transposing LDS reads (ds_read_b64_tr_b16: of the 16 lanes' 4 x 16 values,
// lane i receives column i).
//
// fp32 queries: q and p are split in two fp16 pieces each (q scaled by a power of
// two to below 2^14 a row, p by 2^kOffset; what both leave is at most 2^-23 of the
// row's largest), and each product is two MFMAs on the same key or value operand.
// fp16 and bf16 queries: p is rounded once to the operands' type (half a step of
// it, as the output's own rounding; weights are normalized by the sum of the
// unrounded p).  fp16 weights are held times 2^kOffset too: their steps are relative
// down to 2^-24 of the reference's weight and 2^-34 of it below, so a long tail
// under one dominant key keeps its mass.  The second product adds 16 keys at a time
// to fp32 sums: what these come to below 2^-24 of a sum is lost to it.
//
// What bounds it.  Prompts: a wave's 64 matrix instructions a unit of 256
// channels are about 2050 cycles (twice that for fp32 queries, whose products are
// two), and a wave alone on its SIMD issues an instruction about every four
// cycles.  Exponentials and LDS reads fit between the matrix steps (1850 and 1500
// cycles for the two products in bf16); a unit's addresses, masks and reference
// come to 1000 more.  8192 rows of 8 heads of 256 in bf16: 328 us (840 TFLOP/s);
// 2048 rows with fp32 queries: 60 us (290, and twice that in the instructions); 16
// ragged prompts of 32 heads of 128 in fp16: 258 us (570).  Single tokens and
// trees: memory where the caches are long (8 x 20,000 rows of 8 KV heads of 128:
// 133 us, 4.9 TB/s), else what a workgroup does once beside its one or two units:
// at fp32 queries of 256 channels 28,000 to 36,000 cycles, of which a unit's products
// are 4,500, its place and the wait for pages, keys and queries 10,000, the queries'
// split 5,200, the join of the two waves and the sums' way out 7,500 (16 x 1024 rows:
// 28 us, one sequence of 512: 20 us).
#include "gemma_q8.h"
#include "gq8_lanes.hpp"
#include "gq8_paged.hpp"

#include <algorithm>
#include <cmath>

namespace gq8 {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));
typedef uint32_t word4 __attribute__((ext_vector_type(4)));

constexpr int kKeys = 64;          // keys a unit
constexpr float kLow = -3.0e38f;   // a row's reference before its first key
constexpr float kMargin = 4.f;     // how far (in powers of two) a score may pass it
constexpr float kFar = 65536.f;    // 2^-24 of it stays below a hundredth of a power
constexpr float kLeast = 1.0e-30f; // of the factor on a score
constexpr float kOffset = 10.f;    // fp16 weights are held times 2^10 (2^14 at most)
constexpr float kLog2e = 1.44269504088896340736f;

// workgroups of a launch: as many as are resident (128 KB of LDS at 256
// channels, 64 KB at 128), so that every run of units starts at once
template <int HD>
constexpr int kWorkers = HD == 256 ? 256 : 512;

// The tile that a worker begins and others end: how many of them share it
// (0: there is none), its first packed row and head, and its pairs.
struct Shared {
    int workers, row, head, pairs;
};

struct AttentionArgs {
    PackedAttentionArgs a;
    int group, row_shift; // rows a tile = 1 << row_shift, each with its `group` heads
    int pairs;            // M
    int fixed;            // what a tile costs beside its units, in units
    int workers;
    float *sums, *stats;  // [workers, 2][M][HD], [workers, 2][M][4]
    Shared *shared;       // [workers], and 64 times 16 bytes that are never read
};

__device__ const word4 kZeroChunk = {0, 0, 0, 0};

// ---- where a unit lies -----------------------------------------------------------
// Workers take equal runs of slots: a tile is `fixed` slots for its queries and
// its outputs, then one for each of its units.
struct Cursor {
    int s, g, r;         // sequence, KV head, tile of rows
    int chunk, chunks;   // the unit in its tile, the tile's units
    int start, n, c, tiles; // the sequence: first packed row, rows, cached rows, tiles
};

__device__ inline int uniform(int v)
{
    return __builtin_amdgcn_readfirstlane(v);
}

__device__ inline uint64_t uniform64(uint64_t v)
{
    return ((uint64_t) (uint32_t) uniform((int) (v >> 32)) << 32) | (uint32_t) uniform((int) v);
}

__device__ inline int units_of(int keys)
{
    return (int) ((uint32_t) (keys + kKeys - 1) / kKeys);
}

__device__ inline void sequence_of(const AttentionArgs &p, int s, int &start, int &n, int &c)
{
    const PackedSequences &q = p.a.seq;
    start = min(max(q.starts[s], 0), q.rows);
    n = min(max(q.starts[s + 1], start), q.rows) - start;
    c = q.cached ? min(max(q.cached[s], 0), q.table_width << p.a.layer.page_shift) : 0;
}

__device__ inline int tiles_of(const AttentionArgs &p, int n)
{
    return (n + (1 << p.row_shift) - 1) >> p.row_shift;
}

// units of new rows of tile r of a sequence of n rows
__device__ inline int own_chunks(const AttentionArgs &p, int r, int n)
{
    if (!p.a.k)
        return 0;
    return units_of(p.a.causal ? min((r + 1) << p.row_shift, n) : min(n, p.a.mask_words * kKeys));
}

__device__ inline int tile_chunks(const AttentionArgs &p, int r, int n, int c)
{
    return max(1, units_of(c) + own_chunks(p, r, n));
}

// slots of the first t of a KV head's tiles, in closed form: the rows of a tile
// and a unit's keys are powers of two (the host keeps them below 2^31)
__device__ inline int slots_before(const AttentionArgs &p, int t, int tiles, int n, int c)
{
    if (!p.a.causal)
        return t * (p.fixed + max(1, units_of(c) + own_chunks(p, 0, n)));
    int own;
    if (p.row_shift < 6) { // the sum of ceil((r + 1) / q), q tiles a unit of keys
        const int shift = 6 - p.row_shift;
        const int whole = t >> shift, rest = t & ((1 << shift) - 1);
        own = (whole + 1) * ((whole << shift >> 1) + rest);
    } else {
        const int per = 1 << (p.row_shift - 6);
        const int full = t < tiles ? t : t - 1;
        own = full * (full + 1) / 2 * per + (t == tiles && t > 0 ? units_of(n) : 0);
    }
    return t * (p.fixed + units_of(c)) + own;
}

// the tile that holds a KV head's slot `offset`: by the root of the sum, which
// floating point may miss by some
__device__ inline int tile_at(const AttentionArgs &p, int offset, int tiles, int n, int c)
{
    float guess;
    if (!p.a.causal) {
        guess = (float) offset * __builtin_amdgcn_rcpf((float) (p.fixed + max(1, units_of(c) + own_chunks(p, 0, n))));
    } else { // t (a + t / (2 q)) slots, about
        const float a = (float) (p.fixed + units_of(c)) + 0.5f;
        const float q = 64.f / (float) (1 << p.row_shift), twice = (float) (1 << p.row_shift) / 32.f;
        guess = q * (__builtin_amdgcn_sqrtf(a * a + twice * (float) offset) - a);
    }
    int t = min(max((int) guess, 0), tiles - 1);
    while (t > 0 && slots_before(p, t, tiles, n, c) > offset)
        --t;
    while (t + 1 < tiles && slots_before(p, t + 1, tiles, n, c) <= offset)
        ++t;
    return t;
}

__device__ inline int64_t broadcast(int64_t v, int lane)
{
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t) v, lane);
    const uint32_t hi = __builtin_amdgcn_readlane((uint32_t) (v >> 32), lane);
    return (int64_t) (((uint64_t) hi << 32) | lo);
}

// 64 sequences, one a lane, with their slots and all slots up to theirs.
struct Slots {
    int base;
    int start, n, c;
    int64_t mine, upto;
};

__device__ inline Slots slots_from(const AttentionArgs &p, int base, int64_t before)
{
    const int lane = threadIdx.x & 63, count = p.a.seq.sequences - base;
    Slots slots{base, 0, 0, 0, 0, 0};
    sequence_of(p, base + min(lane, count - 1), slots.start, slots.n, slots.c);
    const int tiles = tiles_of(p, slots.n);
    if (lane < count && tiles > 0)
        slots.mine = (int64_t) p.a.kv_heads * slots_before(p, tiles, tiles, slots.n, slots.c);
    slots.upto = slots.mine + (lane == 0 ? before : 0);
    for (int d = 1; d < min(count, 64); d <<= 1) {
        const int64_t other = __shfl_up(slots.upto, d);
        slots.upto += lane >= d ? other : 0;
    }
    if (lane >= count)
        slots.upto = INT64_MAX; // past all sequences
    return slots;
}

// the slots of the whole batch; `slots` is left at the last sequences
__device__ inline int64_t all_slots(const AttentionArgs &p, Slots &slots)
{
    int64_t total = 0;
    int base = 0;
    do {
        slots = slots_from(p, base, total);
        total = broadcast(slots.upto, min(p.a.seq.sequences - base, 64) - 1);
        base += 64;
    } while (base < p.a.seq.sequences);
    return total;
}

// The places of two slots, and how far into their tiles they are (in slots);
// even lanes work on the one and odd lanes on the other.
__device__ inline void locate(const AttentionArgs &p, Slots &slots, const int64_t (&slot)[2],
                              Cursor (&at)[2], int (&into)[2])
{
    const int lane = threadIdx.x & 63;
    int64_t offset[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        int64_t before = 0;
        if (p.a.seq.sequences > 64)
            slots = slots_from(p, 0, 0);
        uint64_t past = __ballot(slots.upto > slot[k]);
        while (!past) {
            before = broadcast(slots.upto, 63);
            slots = slots_from(p, slots.base + 64, before);
            past = __ballot(slots.upto > slot[k]);
        }
        const int found = __ffsll((unsigned long long) past) - 1;
        at[k].s = slots.base + found;
        at[k].start = __builtin_amdgcn_readlane(slots.start, found);
        at[k].n = __builtin_amdgcn_readlane(slots.n, found);
        at[k].c = __builtin_amdgcn_readlane(slots.c, found);
        at[k].tiles = tiles_of(p, at[k].n);
        offset[k] = slot[k] - (broadcast(slots.upto, found) - broadcast(slots.mine, found));
    }
    const bool odd = lane & 1;
    const int n = odd ? at[1].n : at[0].n, c = odd ? at[1].c : at[0].c;
    const int tiles = odd ? at[1].tiles : at[0].tiles;
    int64_t rest = odd ? offset[1] : offset[0];
    int g = 0;
    if (p.a.kv_heads > 1) {
        const int64_t per = slots_before(p, tiles, tiles, n, c);
        g = min(max((int) ((float) rest * __builtin_amdgcn_rcpf((float) per)), 0), p.a.kv_heads - 1);
        while (g > 0 && g * per > rest)
            --g;
        while (g + 1 < p.a.kv_heads && (g + 1) * per <= rest)
            ++g;
        rest -= g * per;
    }
    const int r = tile_at(p, (int) rest, tiles, n, c);
    const int within = (int) rest - slots_before(p, r, tiles, n, c);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        at[k].g = __builtin_amdgcn_readlane(g, k);
        at[k].r = __builtin_amdgcn_readlane(r, k);
        into[k] = __builtin_amdgcn_readlane(within, k);
        at[k].chunk = max(0, into[k] - p.fixed);
        at[k].chunks = tile_chunks(p, at[k].r, at[k].n, at[k].c);
    }
}

// To the next tile; false past the last.
__device__ inline bool advance(const AttentionArgs &p, Cursor &at)
{
    at.chunk = 0;
    if (++at.r >= at.tiles) {
        at.r = 0;
        if (++at.g >= p.a.kv_heads) {
            at.g = 0;
            at.n = 0;
            while (at.n == 0) {
                if (++at.s >= p.a.seq.sequences)
                    return false;
                sequence_of(p, at.s, at.start, at.n, at.c);
                at.start = uniform(at.start); at.n = uniform(at.n); at.c = uniform(at.c);
            }
            at.tiles = tiles_of(p, at.n);
        }
    }
    at.chunks = tile_chunks(p, at.r, at.n, at.c);
    return true;
}

// the XCD-major number of a workgroup: the 8 XCDs take blocks in turn, and
// neighbouring runs of units share their keys in one XCD's L2
__device__ inline int worker_of(int block, int workers)
{
    const int xcd = block & 7, each = workers >> 3, rest = workers & 7;
    return xcd * each + min(xcd, rest) + (block >> 3);
}

// ---- keys and values of a unit into LDS ------------------------------------------
// Row j of a tile's 64 rows of HD values, in 16-byte chunks; chunk c of row r
// lies at c ^ swizzle(r), so that over all 64 banks (256 bytes) 16 rows' same
// chunk meet no two in a bank, nor do 4 rows' same four chunks.
template <int HD>
__device__ inline int swizzle(int row)
{
    return HD >= 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : ((row & 2) << 1) | ((row >> 2) & 3);
}

// Where a unit's keys and values are: the row of the pool or of the packed
// tensors that holds the unit's key `lane`, -1 where it holds none (past the
// cached rows or the new ones, or in a page outside the pool).
struct Source {
    int row, slot; // until it is resolved: the page and the key's place in it
    bool cache;
    int channel; // of the KV head
};

// Looks the unit's pages up.  A wait for the entry is a wait for every load
// before it, the unit's keys and values among them: resolve() comes a turn later.
__device__ inline Source request(const AttentionArgs &p, const Cursor &at)
{
    const int lane = threadIdx.x & 63;
    const int cached = units_of(at.c);
    Source from{-1, 0, at.chunk < cached, at.g * p.a.head_dim};
    if (from.cache) {
        const int key = at.chunk * kKeys + lane, shift = p.a.layer.page_shift;
        from.slot = key & ((1 << shift) - 1);
        if (key < at.c)
            from.row = p.a.seq.table[(int64_t) at.s * p.a.seq.table_width + (key >> shift)];
    } else {
        const int j = (at.chunk - cached) * kKeys + lane;
        if (p.a.k && j < at.n)
            from.row = at.start + j;
    }
    return from;
}

__device__ inline void resolve(const AttentionArgs &p, Source &from)
{
    asm volatile("" : "+v"(from.row)); // not before here
    if (from.cache) // -1 is past all pages
        from.row = (uint32_t) from.row < (uint32_t) p.a.layer.pages
                       ? (from.row << p.a.layer.page_shift) + from.slot : -1;
}

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm" // m0 is named as written
// 16 bytes a lane from its own address to LDS at base + 16 lane.  By hand,
// since the compiler would wait for all of them at the next LDS read; the loop
// waits once an iteration.
__device__ inline void load_to_lds(const void *from, uint32_t base)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
                 :: "v"(from), "s"(base) : "memory", "m0");
}

// the same from a wave's address and a lane's offset, to base + AT.  The address
// passes through a scalar copy: a vector instruction that wrote it (a saved
// register read back) would have to lie five instructions before the load.
template <int AT>
__device__ inline void load_to_lds(uint64_t from, uint32_t offset, uint32_t base)
{
    uint64_t copy;
    asm volatile("s_add_u32 m0, %3, %4\n\ts_mov_b64 %0, %2\n\tglobal_load_lds_dwordx4 %1, %0"
                 : "=&s"(copy) : "v"(offset), "s"(from), "s"(base), "i"(AT) : "memory", "m0", "scc");
}
#pragma clang diagnostic pop

__device__ inline uint32_t lds_address(const void *p)
{
    return (uint32_t) (uintptr_t) (__attribute__((address_space(3))) const void *) p;
}

// 16 rows of a unit that one wave loads, 512 / HD an instruction: where they
// follow each other (all of one page, or the packed rows) one address does for
// the wave, and the lanes' offsets from it are those of every such unit.
struct Rows {
    uint64_t keys, values; // the first row's
    int stride;            // bytes
    bool follow;
};

template <int HD>
__device__ inline Rows rows_of(const AttentionArgs &p, const Source &from, int base)
{
    const int lane = threadIdx.x & 63;
    const int first = __builtin_amdgcn_readlane(from.row, base);
    const uint64_t follows = __ballot(from.row == first + lane - base) >> base;
    Rows rows;
    rows.stride = (from.cache ? p.a.layer.width : p.a.kv_stride) * 2;
    const uint64_t offset = (uint64_t) ((int64_t) first * rows.stride + from.channel * 2);
    rows.keys = uniform64((uint64_t) (from.cache ? p.a.layer.keys : p.a.k) + offset);
    rows.values = uniform64((uint64_t) (from.cache ? p.a.layer.values : p.a.v) + offset);
    rows.follow = first >= 0 && (follows & 0xFFFF) == 0xFFFF && p.a.head_dim == HD;
    return rows;
}

template <int HD>
struct Offsets {
    uint32_t of[HD / 32]; // of the instructions
    int stride;           // the rows' that they are for
};

template <int HD>
__device__ inline void set_offsets(Offsets<HD> &offsets, int stride)
{
    constexpr int kChunks = HD / 8, kRows = 64 / kChunks;
    const int lane = threadIdx.x & 63;
    offsets.stride = stride;
#pragma unroll
    for (int j = 0; j < HD / 32; ++j) {
        const int row = j * kRows + lane / kChunks; // below 16: kPagedMaxApart keeps this in 32 bits
        offsets.of[j] = row * (uint32_t) stride + ((lane % kChunks ^ swizzle<HD>(row)) << 4);
    }
}

// instructions J .. J + N - 1 of such rows
template <int HD, int J, int N>
__device__ inline void load_follow(uint64_t first, const Offsets<HD> &offsets, uint32_t to)
{
    load_to_lds<J * 1024>(first, offsets.of[J], to);
    if constexpr (N > 1)
        load_follow<HD, J + 1, N - 1>(first, offsets, to);
}

// A unit's 64 rows of keys or of values, WAVES waves.  Rows that do not follow
// each other take an address a lane; rows and channels that there are not are
// read as zeros.
template <int HD, int WAVES, bool kKeysNotValues>
__device__ inline void load_rows(const AttentionArgs &p, const Source &from, uint32_t to,
                                 Offsets<HD> &offsets)
{
    constexpr int kChunks = HD / 8, kRows = 64 / kChunks;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
#pragma unroll
    for (int part = 0; part < 4 / WAVES; ++part) {
        const int base = (wave * (4 / WAVES) + part) * 16;
        const uint32_t area = to + base * HD * 2;
        const Rows rows = rows_of<HD>(p, from, base);
        if (rows.follow) {
            if (rows.stride != offsets.stride)
                set_offsets(offsets, rows.stride);
            load_follow<HD, 0, HD / 32>(kKeysNotValues ? rows.keys : rows.values, offsets, area);
            continue;
        }
        const uint16_t *pool = kKeysNotValues ? (from.cache ? p.a.layer.keys : p.a.k)
                                              : (from.cache ? p.a.layer.values : p.a.v);
        const int stride = from.cache ? p.a.layer.width : p.a.kv_stride;
#pragma unroll 1
        for (int j = 0; j < 16 / kRows; ++j) {
            const int r = base + j * kRows + lane / kChunks;
            const int c = (lane % kChunks ^ swizzle<HD>(r)) * 8, at = __shfl(from.row, r);
            const void *zero = &kZeroChunk;
            load_to_lds(at >= 0 && c < p.a.head_dim
                            ? (const void *) (pool + (int64_t) at * stride + from.channel + c) : zero,
                        area + j * kRows * HD * 2);
        }
    }
}

// ---- the arithmetic of a type ------------------------------------------------------
template <typename Q>
struct Arithmetic; // Q: float, _Float16 or __bf16 queries

template <>
struct Arithmetic<_Float16> {
    typedef half8 Operand;
    static constexpr int kPieces = 1;
    static constexpr uint32_t kExponent = 0x7C007C00u, kStep = 0x04000400u;
    static constexpr float kShift = kOffset;
    __device__ static float16v mfma(half8 a, half8 b, float16v c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    __device__ static void split(const float (&x)[2], uint32_t (&out)[1])
    {
        typedef _Float16 half2 __attribute__((ext_vector_type(2)));
        out[0] = __builtin_bit_cast(uint32_t, half2{(_Float16) x[0], (_Float16) x[1]});
    }
};

template <>
struct Arithmetic<__bf16> {
    typedef bf8 Operand;
    static constexpr int kPieces = 1;
    static constexpr uint32_t kExponent = 0x7F807F80u, kStep = 0x00800080u;
    static constexpr float kShift = 0.f;
    __device__ static float16v mfma(bf8 a, bf8 b, float16v c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    __device__ static void split(const float (&x)[2], uint32_t (&out)[1])
    {
        typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
        out[0] = __builtin_bit_cast(uint32_t, bf2{(__bf16) x[0], (__bf16) x[1]});
    }
};

template <>
struct Arithmetic<float> : Arithmetic<_Float16> {
    static constexpr int kPieces = 2;
    __device__ static void split(const float (&x)[2], uint32_t (&out)[2])
    {
        typedef _Float16 half2 __attribute__((ext_vector_type(2)));
        const half2 high = {(_Float16) x[0], (_Float16) x[1]};
        const half2 low = {(_Float16) (x[0] - (float) high[0]), (_Float16) (x[1] - (float) high[1])};
        out[0] = __builtin_bit_cast(uint32_t, high);
        out[1] = __builtin_bit_cast(uint32_t, low);
    }
};

// ---- a wave's state -----------------------------------------------------------------
template <typename Q, int HD>
struct State {
    using A = Arithmetic<Q>;
    typename A::Operand q[HD / 16][A::kPieces];
    float16v sums[HD / 32];
    // This lane's part of sum p: the unit's, and that of the units before it.  A unit is
    // summed by itself, since next to a dominant key's weight a small one alone would
    // round to nothing (65,536 keys 2^24.4 below it: 7e-4 of the total went; 1.6e-5 do).
    float total[2], before;
    float reference, raw, c; // m, and the score it stands for (m = c raw); scale log2(e)
};

template <typename Q, int HD>
__device__ inline void clear(State<Q, HD> &w)
{
#pragma unroll
    for (int i = 0; i < HD / 32; ++i)
        w.sums[i] = float16v{};
    w.total[0] = w.total[1] = w.before = 0.f;
    w.reference = w.raw = kLow;
}

__device__ inline word4 lds_word4(uint32_t address)
{
    return *(__attribute__((address_space(3))) const word4 *) (uintptr_t) address;
}

__device__ inline void lds_word4(uint32_t address, word4 x)
{
    *(__attribute__((address_space(3))) word4 *) (uintptr_t) address = x;
}

__device__ inline short4v lds_transposed(uint32_t address)
{
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) short4v *) (uintptr_t) address);
}

// A wave's 32 rows of queries, sums or outputs lie a row a lane pair in its
// registers, and rows in memory: loads and stores of 16 bytes a lane would touch
// 32 rows each (a tile's queries took 25 us so).  They pass through LDS in rounds
// of HD bytes a row, 16-byte chunk c of row r at c ^ r.
template <int HD>
__device__ inline uint32_t staged(uint32_t area, int row, int chunk)
{
    constexpr int kChunks = HD / 16;
    return area + row * HD + ((chunk ^ (row & (kChunks - 1))) << 4);
}

// the row of a round's instruction j that this lane moves a chunk of
template <int HD>
__device__ inline int staged_row(int j)
{
    return j * (1024 / HD) + (threadIdx.x & 63) / (HD / 16);
}

// The wave's queries on their way, 16 bytes a lane.
template <typename Q, int HD>
struct Fetched {
    word4 x[sizeof(Q)][HD / 32];
};

// `at` is the pair's row in memory, null if it has none (zeros)
template <typename Q, int HD>
__device__ inline void fetch_query(const AttentionArgs &p, const Q *at, Fetched<Q, HD> &f)
{
    constexpr int ROUNDS = sizeof(Q), EACH = HD / 32, kChannels = HD / ROUNDS;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        const Q *from = (const Q *) __shfl((unsigned long long) at, staged_row<HD>(j));
        const int channel = lane % (HD / 16) * (16 / ROUNDS);
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const int c = r * kChannels + channel;
            // every lane loads: around a branch the compiler has saved registers for
            // the lanes inside it alone (the loads of these queries then went astray)
            const bool there = from && c < p.a.head_dim;
            const uintptr_t address = there ? (uintptr_t) (from + c) : (uintptr_t) &kZeroChunk;
            f.x[r][j] = *(const __attribute__((address_space(1))) word4 *) address;
        }
    }
}

// area: 32 HD bytes of LDS that this wave alone reads and writes
template <typename Q, int HD>
__device__ inline void load_query(const AttentionArgs &p, const Fetched<Q, HD> &f, uint32_t area,
                                  State<Q, HD> &w)
{
    constexpr int ROUNDS = sizeof(Q), EACH = HD / 32, kChannels = HD / ROUNDS;
    const int lane = threadIdx.x & 63, row = lane & 31, half = lane >> 5;
    const float scale = p.a.scale * kLog2e;
    // never zero, so that a masked score (minus infinity) keeps its weight of zero
    w.c = fmaxf(fabsf(scale), kLeast);
    float y[ROUNDS == 4 ? HD / 16 : 1][8];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
#pragma unroll
        for (int j = 0; j < EACH; ++j)
            lds_word4(staged<HD>(area, staged_row<HD>(j), lane % (HD / 16)), f.x[r][j]);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int s = 0; s < kChannels / 16; ++s) {
            const int step = r * (kChannels / 16) + s; // channels 16 s + 8 half of the round
            if constexpr (ROUNDS == 4) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const word4 v = lds_word4(staged<HD>(area, row, 4 * s + 2 * half + i));
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        y[step][4 * i + k] = __uint_as_float(v[k]);
                }
            } else {
                word4 v = lds_word4(staged<HD>(area, row, 2 * s + half));
                v ^= scale < 0.f ? 0x80008000u : 0u;
                w.q[step][0] = __builtin_bit_cast(typename State<Q, HD>::A::Operand, v);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
    if constexpr (ROUNDS == 4) {
        float largest = 0.f;
#pragma unroll
        for (int s = 0; s < HD / 16; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                largest = fmaxf(largest, fabsf(y[s][i]));
        largest = fmaxf(largest, xor_lane<32>(largest));
        // 2^-e brings the largest to [2^13, 2^14), rows below 2^-87 near it
        const int e = max((int) ((__float_as_uint(largest) >> 23) & 0xFF) - 127 - 13, -100);
        const float down = ldexpf(scale < 0.f ? -1.f : 1.f, -e);
        w.c = fmaxf(ldexpf(fabsf(scale), e), kLeast);
        word4 pieces[HD / 16][2];
#pragma unroll
        for (int s = 0; s < HD / 16; ++s) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float pair[2] = {y[s][2 * i] * down, y[s][2 * i + 1] * down};
                uint32_t words[2];
                State<Q, HD>::A::split(pair, words);
                pieces[s][0][i] = words[0];
                pieces[s][1][i] = words[1];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
                w.q[s][i] = __builtin_bit_cast(typename State<Q, HD>::A::Operand, pieces[s][i]);
        }
    }
    // 256 channels: to accumulation registers, where matrix instructions read them
    // as well; the others have to hold the sums and the scores of two units
    if constexpr (HD == 256) {
#pragma unroll
        for (int s = 0; s < HD / 16; ++s)
#pragma unroll
            for (int i = 0; i < State<Q, HD>::A::kPieces; ++i)
                asm volatile("" : "+a"(w.q[s][i]));
    }
}

// The wave's sums times `by` to its pairs' rows: `to` is the pair's, null if it
// has none; channels below `limit`.  What goes nowhere goes to `nowhere` (16
// bytes a lane): the stores follow each other without branches.
template <typename T, typename Q, int HD>
__device__ inline void store_rows(const State<Q, HD> &w, float by, T *to, int limit, uint32_t area,
                                  word4 *nowhere)
{
    constexpr int ROUNDS = sizeof(T), EACH = HD / 32, kChannels = HD / ROUNDS;
    const int lane = threadIdx.x & 63, row = lane & 31, half = lane >> 5;
    uint64_t rows[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j)
        rows[j] = __shfl((unsigned long long) to, staged_row<HD>(j));
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
#pragma unroll
        for (int s = 0; s < kChannels / 8; ++s) {
            const int j = r * (kChannels / 8) + s; // channels 8 j + 4 half
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                x[i] = w.sums[j / 4][4 * (j % 4) + i] * by;
            if constexpr (ROUNDS == 4) {
                lds_word4(staged<HD>(area, row, 2 * s + half), __builtin_bit_cast(word4, x));
            } else {
                typedef T T4 __attribute__((ext_vector_type(4)));
                typedef uint32_t word2 __attribute__((ext_vector_type(2)));
                const T4 y = {(T) x[0], (T) x[1], (T) x[2], (T) x[3]};
                *(__attribute__((address_space(3))) word2 *) (uintptr_t) (staged<HD>(area, row, s) + 8 * half) =
                    __builtin_bit_cast(word2, y);
            }
        }
        __builtin_amdgcn_wave_barrier();
        word4 x[EACH];
#pragma unroll
        for (int j = 0; j < EACH; ++j)
            x[j] = lds_word4(staged<HD>(area, staged_row<HD>(j), lane % (HD / 16)));
        const int c = r * kChannels + lane % (HD / 16) * (16 / ROUNDS);
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            const uint64_t at = rows[j] && c < limit ? rows[j] + c * sizeof(T) : (uint64_t) (nowhere + lane);
            *(__attribute__((address_space(1))) word4 *) at = x[j];
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// What makes x stays in this step: the compiler would move it to where its value
// is used.
template <typename T>
__device__ inline void pin(T &x)
{
    asm volatile("" : "+v"(x));
}

// The weights of the unit's 16-key steps as the second product's operand, two a
// word.
template <typename Q, int BLOCKS>
struct Weights {
    word4 b[2 * BLOCKS][Arithmetic<Q>::kPieces];
};

// Score number i of a lane becomes a weight in three stages, which depend on each
// other: the exponent, the exponential, the sum and the operand.  Between matrix
// steps each runs a step after the one before, since a wave waits for what an
// instruction needs.
template <typename Q, int HD, int BLOCKS>
__device__ inline void exponentiate(State<Q, HD> &w, float16v (&s)[BLOCKS], Weights<Q, BLOCKS> &p,
                                    float minus, int stage, int i)
{
    if (i < 0 || i >= 16 * BLOCKS)
        return;
    float x = s[i / 16][i % 16];
    if (stage == 0) {
        x = fmaf(x, w.c, minus);
        pin(x);
        s[i / 16][i % 16] = x;
    } else if (stage == 1) {
        x = __builtin_amdgcn_exp2f(x);
        pin(x);
        s[i / 16][i % 16] = x;
    } else {
        w.total[i % 2] += x;
        pin(w.total[i % 2]);
        if (i % 2 == 1) {
            const float y[2] = {s[i / 16][i % 16 - 1], x};
            uint32_t words[Arithmetic<Q>::kPieces];
            Arithmetic<Q>::split(y, words);
#pragma unroll
            for (int j = 0; j < Arithmetic<Q>::kPieces; ++j) {
                pin(words[j]);
                p.b[i / 8][j][i % 8 / 2] = words[j];
            }
        }
    }
}

template <typename Q, int HD, int BLOCKS>
__device__ inline void exponentiate(State<Q, HD> &w, float16v (&s)[BLOCKS], Weights<Q, BLOCKS> &p,
                                    float minus)
{
#pragma unroll
    for (int stage = 0; stage < 3; ++stage)
#pragma unroll
        for (int i = 0; i < 16 * BLOCKS; ++i)
            exponentiate<Q, HD, BLOCKS>(w, s, p, minus, stage, i);
}

// Matrix steps read one operand each from LDS.  The compiler would read each
// right before its step and wait for it; here kAhead operands are under way,
// and the order of the steps is held, kGroup at once.  8192 rows of 256 channels: 326
// us, with two 345.  At narrower heads the second wave on the SIMD covers the wait and
// registers are short: two do (16 ragged prompts of heads of 128: 256 us, as with four).
template <int HD>
constexpr int kAheadOf = HD == 256 ? 4 : 2;
constexpr int kGroup = 2;

// `next` = scores of key blocks [first, first + BLOCKS) of 32 keys; between(i)
// is what else step i does.
template <typename Q, int HD, int BLOCKS, typename F>
__device__ inline void scores(const State<Q, HD> &w, uint32_t keys, int first, float16v (&next)[BLOCKS],
                              F between)
{
    using A = Arithmetic<Q>;
    constexpr int STEPS = HD / 16 * BLOCKS, kAhead = kAheadOf<HD>;
    const int lane = threadIdx.x & 63, row = lane & 31, half = lane >> 5;
    const uint32_t base = keys + (first * 32 + row) * HD * 2 + ((half ^ swizzle<HD>(row)) << 4);
    auto address = [&](int i) { return base ^ (i / BLOCKS * 32); };
    auto operand = [&](uint32_t at, int i) { return lds_word4(at + i % BLOCKS * 32 * HD * 2); };
    word4 a[kAhead];
    uint32_t at[kGroup]; // the addresses of the next step's reads, made a step before
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
        a[i] = operand(address(i), i);
#pragma unroll
    for (int g = 0; g < kGroup; ++g)
        at[g] = address(kAhead + g);
    // Two steps at once, on two sums: a step on the sum of the one before waits for it.
    float16v sums[2] = {};
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < STEPS; i += kGroup) {
#pragma unroll
        for (int j = 0; j < A::kPieces; ++j)
#pragma unroll
            for (int g = 0; g < kGroup; ++g) {
                const auto key = __builtin_bit_cast(typename A::Operand, a[(i + g) % kAhead]);
                sums[(i + g) % 2] = A::mfma(key, w.q[(i + g) / BLOCKS][j], sums[(i + g) % 2]);
            }
#pragma unroll
        for (int g = 0; g < kGroup; ++g) {
            if (i + g + kAhead < STEPS) {
                a[(i + g + kAhead) % kAhead] = operand(at[g], i + g + kAhead);
                at[g] = address(i + g + kAhead + kGroup);
            }
        }
#pragma unroll
        for (int g = 0; g < kGroup; ++g)
            between(i + g);
        __builtin_amdgcn_sched_barrier(0);
    }
    next[0] = sums[0];
    if constexpr (BLOCKS == 2)
        next[1] = sums[1];
    else
        next[0] += sums[1];
}

// the largest of a pair's scores in these blocks
template <int BLOCKS>
__device__ inline float largest_of(const float16v (&s)[BLOCKS])
{
    float largest = s[0][0];
#pragma unroll
    for (int i = 1; i < 16 * BLOCKS; ++i)
        largest = fmaxf(largest, s[i / 16][i % 16]);
    return fmaxf(largest, xor_lane<32>(largest));
}

// 0 x infinity is not 0: in a unit that some pairs attend in part, values
// that are not finite are taken out of the tile, and each channel remembers the
// keys that had them: plus infinities and NaNs, minus infinities and NaNs.
// Returns whether there were any.  All waves of the workgroup call it.
template <typename Q, int HD, int WAVES>
__device__ inline bool take_out(uint32_t values, uint32_t *found, uint64_t (*taken)[2])
{
    using A = Arithmetic<Q>;
    constexpr int kEach = HD / 8 / WAVES; // KB of the tile a wave
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    uint32_t odd = 0;
#pragma unroll 4
    for (int j = 0; j < kEach; ++j) {
        const word4 x = lds_word4(values + (wave * kEach + j) * 1024 + lane * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) // an exponent of all ones and one carries into the sign
            odd |= (x[i] & A::kExponent) + A::kStep;
    }
    const bool mine = __ballot((odd & 0x80008000u) != 0) != 0;
    if (lane == 0)
        found[wave] = mine;
    __syncthreads();
    uint32_t any = 0;
#pragma unroll
    for (int v = 0; v < WAVES; ++v)
        any |= found[v];
    if (!any)
        return false;
    for (int c = threadIdx.x; c < HD; c += 64 * WAVES)
        taken[c][0] = taken[c][1] = 0;
    __syncthreads();
    if (mine)
        for (int j = 0; j < kEach * 8; ++j) {
            const int at = (wave * kEach * 8 + j) * 64 + lane; // of the tile's values
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
    __syncthreads();
    return true;
}

// What take_out took, for the keys that the lane's pair attends (a NaN counts
// as both infinities, whose sum is one).
template <typename Q, int HD>
__device__ inline void put_back(State<Q, HD> &w, const uint64_t (*taken)[2], uint64_t attends)
{
    const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int cb = 0; cb < HD / 32; ++cb) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint64_t *t = taken[32 * cb + 8 * (i / 4) + 4 * half + i % 4];
            w.sums[cb][i] += (t[0] & attends ? INFINITY : 0.f) - (t[1] & attends ? INFINITY : 0.f);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

// sums += P V over the wave's keys; between the steps (kMax) the largest of the
// next unit's scores is found.
template <typename Q, int HD, int BLOCKS, bool kMax>
__device__ inline void weigh(State<Q, HD> &w, uint32_t values, int first, const Weights<Q, BLOCKS> &p,
                             const float16v (&next)[BLOCKS], float &largest)
{
    using A = Arithmetic<Q>;
    constexpr int STEPS = HD / 32 * 2 * BLOCKS, kEach = 16 / (HD / 16), kAhead = kAheadOf<HD>;
    const int lane = threadIdx.x & 63, half = lane >> 5, i16 = lane & 15;
    const int row = first * 32 + 4 * half + (i16 >> 2); // of a step's first four keys
    const int chunk = 2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1);
    const uint32_t base = values + row * HD * 2 + ((chunk ^ swizzle<HD>(row)) << 4) + (i16 & 1) * 8;
    typedef short short8v __attribute__((ext_vector_type(8)));
    struct Address {
        uint32_t low, high; // the step's first four keys, and 8 rows on
    };
    auto address = [&](int i) { // channel block i % (HD / 32)
        return Address{base ^ (i % (HD / 32) * 64), base ^ (i % (HD / 32) * 64) ^ 32};
    };
    auto operand = [&](const Address &at, int i) { // 16-key step i / (HD / 32)
        const int step = i / (HD / 32) * 16 * HD * 2;
        const short4v low = lds_transposed(at.low + step);
        const short4v high = lds_transposed(at.high + step + 8 * HD * 2);
        return (short8v) __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    short8v a[kAhead];
    Address at[kGroup]; // of the next step's reads, made a step before
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
        a[i] = operand(address(i), i);
#pragma unroll
    for (int g = 0; g < kGroup; ++g)
        at[g] = address(kAhead + g);
    float most = -INFINITY;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < STEPS; i += kGroup) {
#pragma unroll
        for (int j = 0; j < A::kPieces; ++j)
#pragma unroll
            for (int g = 0; g < kGroup; ++g) {
                const int t = (i + g) / (HD / 32), cb = (i + g) % (HD / 32);
                const auto value = __builtin_bit_cast(typename A::Operand, a[(i + g) % kAhead]);
                w.sums[cb] = A::mfma(value, __builtin_bit_cast(typename A::Operand, p.b[t][j]), w.sums[cb]);
            }
#pragma unroll
        for (int g = 0; g < kGroup; ++g) {
            if (i + g + kAhead < STEPS) {
                a[(i + g + kAhead) % kAhead] = operand(at[g], i + g + kAhead);
                at[g] = address(i + g + kAhead + kGroup);
            }
        }
#pragma unroll
        for (int g = 0; g < kGroup; ++g) {
            if constexpr (kMax) {
#pragma unroll
                for (int j = (i + g) * kEach; j < (i + g + 1) * kEach; ++j)
                    most = fmaxf(most, next[j / 16][j % 16]);
                pin(most);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (kMax)
        largest = fmaxf(most, xor_lane<32>(most));
}

// The lane's bits of `allowed`, which has one for each of the unit's keys; score
// number i's is bit score_bit(i).
__device__ inline uint64_t lane_bits(uint64_t allowed, int first)
{
    return allowed >> (32 * first + 4 * ((threadIdx.x & 63) >> 5));
}

constexpr int score_bit(int i)
{
    return 32 * (i / 16) + 8 * ((i % 16) / 4) + i % 4;
}

// the largest of the scores that the pair attends
template <int BLOCKS>
__device__ inline float largest_of(const float16v (&s)[BLOCKS], uint64_t bits)
{
    float largest = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16 * BLOCKS; ++i)
        largest = fmaxf(largest, (bits >> score_bit(i)) & 1 ? s[i / 16][i % 16] : -INFINITY);
    return fmaxf(largest, xor_lane<32>(largest));
}

// A reference far from zero is rounded, by up to 2^-24 |m| powers.  The weights of a
// far row are taken from c raw itself (its scores from the reference's own first,
// which leaves the largest an exact zero), those of a near row from m as it is
// held; this is what c raw has beside a far m, for the factors between references.
// Without it exact scores that lie a few apart brought errors of 1e-4 of the largest
// value at scores of 2e5, and of 1.5e-3 at 1e8.
__device__ inline float beside(float reference, float raw, float c)
{
    const float size = fabsf(reference); // from 1e30 on there is no reference, or no difference left
    return size > kFar && size < 1.0e30f ? fmaf(raw, c, -reference) : 0.f;
}

// Moves the reference where the unit's largest score passes it by more than the
// margin.  Returns whether it is far for some row of the wave.  The sum of the unit
// before joins the total here.
template <typename Q, int HD>
__device__ inline bool refer(State<Q, HD> &w, float largest)
{
    w.before += w.total[0] + w.total[1];
    w.total[0] = w.total[1] = 0.f;
    if (__ballot((largest - w.raw) * w.c > kMargin)) {
        const float next = fmaxf(largest * w.c, w.reference), last = beside(w.reference, w.raw, w.c);
        w.raw = fmaxf(largest, w.raw);
        const float factor = __builtin_amdgcn_exp2f(w.reference - next + (last - beside(next, w.raw, w.c)));
        w.reference = next;
        pin(w.reference); // else the loop is there twice, for far rows and others
        w.before *= factor;
#pragma unroll
        for (int cb = 0; cb < HD / 32; ++cb)
            w.sums[cb] *= factor;
    }
    return __ballot(fabsf(w.reference) > kFar) != 0;
}

// Of sums about m + rest and about another reference: the larger, and the factors
// that bring both to it.
struct Factors {
    float m, rest, a, b;
};

__device__ inline Factors factors(float m, float rest, float other, float other_rest)
{
    const float past = other - m + (other_rest - rest), less = __builtin_amdgcn_exp2f(-fabsf(past));
    Factors by;
    by.m = past > 0.f ? other : m;
    by.rest = past > 0.f ? other_rest : rest;
    by.a = past > 0.f ? less : 1.f;
    by.b = past > 0.f ? 1.f : less;
    return by;
}

// A workgroup's run of units.  ROWS waves take 32 pairs each, of all 64 keys of
// a unit (ROWS > 1), or KEYS waves take 32 keys each, of the same 32 pairs.
//
// kPipelined: one unit's exponentials run between the matrix steps of the next
// one's scores, so keys are loaded two units ahead and values one: unit u's turn
// waits for the keys of u + 1 and the values of u, all requested a turn before.
// Not for tiles of 32 pairs, which wait for memory.
template <typename Q, int HD, int ROWS, int KEYS>
__global__ __launch_bounds__(64 * ROWS * KEYS)
__attribute__((amdgpu_waves_per_eu(HD == 256 || KEYS == 2 ? 1 : 2))) void attention_kernel(AttentionArgs p)
{
    static_assert(KEYS == 1 || (KEYS == 2 && ROWS == 1), "a unit is two blocks of 32 keys");
    // a wave's own part of a buffer: the rows it loads, and where it stages its pairs
    constexpr int kPart = kKeys * HD * 2 / (ROWS * KEYS);
    static_assert(kPart >= 32 * HD, "32 pairs of HD bytes");
    constexpr int WAVES = ROWS * KEYS, BLOCKS = 2 / KEYS, kTile = kKeys * HD * 2;
    constexpr bool kPipelined = KEYS == 1;
    __shared__ __align__(1024) uint8_t lds[4 * kTile]; // keys twice, values twice
    __shared__ float exchange[KEYS == 2 ? 192 : 1];
    __shared__ uint64_t taken[HD][2];
    __shared__ uint32_t found[WAVES];
    const uint32_t keys = uniform(lds_address(lds)), values = keys + 2 * kTile;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), half = lane >> 5;
    const int pair = (KEYS == 2 ? 0 : wave * 32) + (lane & 31); // of the tile
    const int first = KEYS == 2 ? wave : 0;                     // key block

    Slots slots;
    const int64_t all = all_slots(p, slots);
    const int64_t share = (all + p.workers - 1) / p.workers;
    const int worker = worker_of(blockIdx.x, p.workers);
    const int64_t from = worker * share, to = min(all, from + share);
    Shared shared{};
    // the run ends before this unit; past the last sequence at the end
    Cursor ends_of[2] = {};
    int into[2] = {};
    if (from < to)
        locate(p, slots, {from, min(to, all - 1)}, ends_of, into);
    Cursor at = ends_of[0], stop = ends_of[1];
    if (to == all)
        stop.s = p.a.seq.sequences;
    const int stop_into = into[1];
    auto here = [&](const Cursor &x) { return x.s == stop.s && x.g == stop.g && x.r == stop.r; };
    auto last_unit = [&](const Cursor &x) { return here(x) ? stop.chunk : x.chunks; }; // of its tile, and one
    if (from >= to || at.chunk == last_unit(at)) {
        if (threadIdx.x == 0)
            p.shared[worker] = shared;
        return;
    }

    Cursor ahead = at;
    int left = last_unit(ahead) - ahead.chunk; // units of its tile, itself among them
    auto to_next = [&] {                       // false past the run
        if (--left > 0) {
            ++ahead.chunk;
            return true;
        }
        if (here(ahead) || !advance(p, ahead))
            return false;
        left = last_unit(ahead);
        return left > 0;
    };
    Source second{}, third{}; // of units u + 1 and u + 2, and whether there are they and u + 3
    bool more1 = false, more2 = false, more3 = false;
    uint64_t present;         // the keys of unit u
    Offsets<HD> offsets;
    set_offsets(offsets, (at.chunk * kKeys < at.c ? p.a.layer.width : p.a.kv_stride) * 2);
    {
        Source unit = request(p, ahead);
        more1 = to_next();
        if (more1) {
            second = request(p, ahead);
            more2 = to_next();
        }
        if (more2) {
            third = request(p, ahead);
            more3 = to_next();
        }
        resolve(p, unit);
        resolve(p, second);
        present = __ballot(unit.row >= 0);
        load_rows<HD, WAVES, true>(p, unit, keys, offsets);
        load_rows<HD, WAVES, false>(p, unit, values, offsets);
        if (kPipelined && more1)
            load_rows<HD, WAVES, true>(p, second, keys + kTile, offsets);
    }
    Rows next_rows{}; // of unit u + 1
    if constexpr (kPipelined)
        next_rows = rows_of<HD>(p, second, wave * 16);

    const int pair_row = pair / p.group, pair_head = pair - pair_row * p.group;
    for (int u = 0;;) {
        // the tile's units in this run; row i of the sequence is this lane's pair's
        const int first_chunk = at.chunk, end = u + last_unit(at) - at.chunk;
        const int i = (at.r << p.row_shift) + pair_row;
        const bool live = pair_row < (1 << p.row_shift) && i < at.n;
        const int head = at.g * p.group + pair_head;
        const bool busy = __ballot(live) != 0;
        const int cached = units_of(at.c);
        State<Q, HD> w;
        Weights<Q, BLOCKS> weights;
        float16v s[BLOCKS];
        float largest = 0.f, minus = 0.f;
        bool ends = false; // the run
        Fetched<Q, HD> fetched;
        fetch_query(p, live ? (const Q *) p.a.q + (int64_t) (at.start + i) * p.a.q_stride
                                  + (int64_t) head * p.a.head_dim : nullptr, fetched);
        // every wave has done with the last tile's values, and this unit's rows are there
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        load_query(p, fetched, values + (1 - (u & 1)) * kTile + wave * kPart, w);
        clear(w);
        if constexpr (kPipelined) { // the other units' scores are made a turn ahead
            if (busy) {
                scores<Q, HD, BLOCKS>(w, keys + (u & 1) * kTile, first, s, [](int) {});
                largest = largest_of(s);
            }
            __syncthreads(); // every wave has done with this unit's keys
        }
        for (;; ++u) {
            const uint32_t this_keys = keys + (u & 1) * kTile, next_keys = keys + (1 - (u & 1)) * kTile;
            const uint32_t value_tile = values + (u & 1) * kTile;
            const uint32_t next_values = values + (1 - (u & 1)) * kTile;
            resolve(p, third);
            Rows ahead_rows{};
            if constexpr (kPipelined) {
                ahead_rows = rows_of<HD>(p, third, wave * 16);
                if (next_rows.stride != offsets.stride)
                    set_offsets(offsets, next_rows.stride);
            }
            uint64_t allowed = present;
            present = __ballot(second.row >= 0);
            bool masked = allowed != ~0ull;
            const int key = (at.chunk - cached) * kKeys; // the first new row of the unit
            if (key >= 0) {
                if (!p.a.causal) {
                    uint64_t word = 0;
                    if (live && p.a.k)
                        word = p.a.masks[(int64_t) (at.start + i) * p.a.mask_words + key / kKeys];
                    asm volatile("" : "+v"(word)); // the wait for it (and all loads) is this branch's alone
                    masked = true;
                    allowed &= word;
                } else if (key + kKeys - 1 > at.r << p.row_shift) {
                    const int last = i - key;
                    masked = true;
                    allowed &= last >= 63 ? ~0ull : last < 0 ? 0 : (2ull << last) - 1;
                }
            }
            // most units: nothing masked, all rows follow each other; the loads are
            // requested between the matrix steps then
            const bool plain = kPipelined && busy && !masked && u + 1 < end && more2
                               && next_rows.follow && ahead_rows.follow
                               && ahead_rows.stride == offsets.stride;
            if (!plain) {
                if (kPipelined && more2)
                    load_rows<HD, WAVES, true>(p, third, this_keys, offsets);
                if (!kPipelined && more1)
                    load_rows<HD, WAVES, true>(p, second, next_keys, offsets);
                if (more1)
                    load_rows<HD, WAVES, false>(p, second, next_values, offsets);
            }
            const uint64_t value_rows = next_rows.values;
            next_rows = ahead_rows;
            second = third;
            const bool last = !more1;
            more1 = more2;
            more2 = more3;
            if (more3) {
                third = request(p, ahead);
                more3 = to_next();
            }
            const bool took = masked && take_out<Q, HD, WAVES>(value_tile, found, taken);
            if (busy) {
                if constexpr (!kPipelined) {
                    scores<Q, HD, BLOCKS>(w, this_keys, first, s, [](int) {});
                    largest = largest_of(s);
                }
                if (masked)
                    largest = largest_of(s, lane_bits(allowed, first));
                const bool far = refer(w, largest);
                const bool own = fabsf(w.reference) > kFar;
                minus = Arithmetic<Q>::kShift - (own ? 0.f : w.reference);
                if (masked || far) { // in one place: around each the scores change registers
                    uint64_t bits = lane_bits(allowed, first);
                    pin(bits); // made here: held from before they cost eight registers
                    const float raw = own ? w.raw : 0.f;
#pragma unroll
                    for (int j = 0; j < 16 * BLOCKS; ++j)
                        s[j / 16][j % 16] = (bits >> score_bit(j)) & 1 ? s[j / 16][j % 16] - raw : -INFINITY;
                }
                if (took)
                    put_back(w, taken, KEYS == 2 ? allowed & 0xFFFFFFFFull << (32 * first) : allowed);
            }
            if (u + 1 == end) {
                ends = last;
                break;
            }
            if (busy) {
                if constexpr (kPipelined) {
                    constexpr int LOADS = HD / 32, STEPS = HD / 16 * BLOCKS, EACH = 16 / (HD / 16);
                    const uint32_t to_keys = this_keys + wave * kPart, to_values = next_values + wave * kPart;
                    float16v next[BLOCKS];
                    scores<Q, HD, BLOCKS>(w, next_keys, first, next, [&](int i) {
                        // at four steps, half of the keys or of the values each
                        constexpr int HALF = LOADS / 2 > 0 ? LOADS / 2 : 1;
                        if (i == 0 && plain)
                            load_follow<HD, 0, HALF>(next_rows.keys, offsets, to_keys);
                        if (i == STEPS / 8 && plain)
                            load_follow<HD, LOADS - HALF, HALF>(next_rows.keys, offsets, to_keys);
                        if (i == STEPS / 4 && plain)
                            load_follow<HD, 0, HALF>(value_rows, offsets, to_values);
                        if (i == STEPS * 3 / 8 && plain)
                            load_follow<HD, LOADS - HALF, HALF>(value_rows, offsets, to_values);
#pragma unroll
                        for (int stage = 2; stage >= 0; --stage)
#pragma unroll
                            for (int j = 0; j < EACH; ++j)
                                exponentiate<Q, HD, BLOCKS>(w, s, weights, minus, stage, (i - stage) * EACH + j);
                    });
#pragma unroll
                    for (int i = 16 * BLOCKS - 2 * EACH; i < 16 * BLOCKS; ++i) {
                        if (i >= 16 * BLOCKS - EACH)
                            exponentiate<Q, HD, BLOCKS>(w, s, weights, minus, 1, i);
                        exponentiate<Q, HD, BLOCKS>(w, s, weights, minus, 2, i);
                    }
                    weigh<Q, HD, BLOCKS, true>(w, value_tile, first, weights, next, largest);
#pragma unroll
                    for (int b = 0; b < BLOCKS; ++b)
                        s[b] = next[b];
                } else {
                    exponentiate(w, s, weights, minus);
                    weigh<Q, HD, BLOCKS, false>(w, value_tile, first, weights, s, largest);
                }
            }
            ++at.chunk;
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
        }
        if (busy) {
            exponentiate(w, s, weights, minus);
            weigh<Q, HD, BLOCKS, false>(w, values + (u & 1) * kTile, first, weights, s, largest);
        }

        {
            const bool last_of_tile = at.chunk + 1 == at.chunks;
            float total = w.before + (w.total[0] + w.total[1]);
            total += xor_lane<32>(total);
            float rest = beside(w.reference, w.raw, w.c);
            bool writes = live;
            if constexpr (KEYS == 2) { // the second wave's sums through the unit's values
                float4v *area = (float4v *) (lds + 2 * kTile + (u & 1) * kTile);
                auto four = [&](int j) {
                    const float16v &x = w.sums[j / 4];
                    const int i = j % 4 * 4;
                    return float4v{x[i], x[i + 1], x[i + 2], x[i + 3]};
                };
                __syncthreads();
                if (wave == 1) {
#pragma unroll
                    for (int j = 0; j < HD / 8; ++j)
                        area[j * 64 + lane] = four(j);
                    exchange[lane] = total;
                    exchange[64 + lane] = w.reference;
                    exchange[128 + lane] = rest;
                }
                __syncthreads();
                writes = writes && wave == 0;
                if (wave == 0) {
                    const Factors by = factors(w.reference, rest, exchange[64 + lane], exchange[128 + lane]);
                    const float a = by.a, b = by.b;
                    total = total * a + exchange[lane] * b;
                    w.reference = by.m;
                    rest = by.rest;
#pragma unroll
                    for (int j = 0; j < HD / 8; ++j) {
                        const float4v x = area[j * 64 + lane];
#pragma unroll
                        for (int i = 4 * j; i < 4 * j + 4; ++i)
                            w.sums[i / 16][i % 16] = w.sums[i / 16][i % 16] * a + x[i % 4] * b;
                    }
                }
            }
            word4 *nowhere = (word4 *) (p.shared + kWorkers<HD>);
            // the unit's values have been read by all
            const uint32_t area = values + (u & 1) * kTile + wave * kPart;
            __syncthreads();
            if (first_chunk == 0 && last_of_tile) {
                const float by = total > 0.f || total != total ? 1.f / total : 0.f;
                store_rows<Q>(w, by, writes ? (Q *) p.a.out + (int64_t) (at.start + i) * p.a.out_stride
                                                  + (int64_t) head * p.a.head_dim : nullptr,
                              p.a.head_dim, area, nowhere);
            } else {
                // slot 0: the tile began with an earlier worker; 1: it begins here
                const int64_t slot = ((int64_t) worker * 2 + (first_chunk == 0)) * p.pairs + pair;
                store_rows<float>(w, 1.f, writes ? p.sums + slot * HD : nullptr, HD, area, nowhere);
                if (writes && half == 0)
                    *(float4 *) (p.stats + slot * 4) = float4{w.reference, rest, total, 0.f};
                if (first_chunk == 0) {
                    // the tile's first slot is `to` less stop_into, its last fixed + chunks on
                    shared.workers = (int) ((to - stop_into + p.fixed + at.chunks - 1) / share) - worker + 1;
                    shared.row = at.start + (at.r << p.row_shift);
                    shared.pairs = min(1 << p.row_shift, at.n - (at.r << p.row_shift)) * p.group;
                    shared.head = at.g * p.group;
                }
            }
        }
        if (ends)
            break;
        advance(p, at);
        ++u;
    }
    if (threadIdx.x == 0)
        p.shared[worker] = shared;
}

// Joins the tiles that several workers share.  Blocks (worker, y): the tile that
// this worker began and did not end.  A row of sums takes HD / 4 lanes, 16 bytes a
// lane (33 MB of them in 10 us: memory).  Of many workers' sums four waves take a
// pair's in turn, of few each wave takes pairs of its own: one sequence of 60,000
// rows, whose tile all 256 workers share, takes 39 us with the attention, 59 without
// the turns; at 8 or 9 workers a tile both ways are within 2 us (46 with turns, 44).
constexpr int kMergeWays = 16; // up to as many workers: pairs of its own a wave

struct Joined {
    float m, rest, total;
    float4v sums;
};

// sums and weights about m + rest and another reference, about the larger
__device__ inline void join(Joined &x, float m, float rest, float total, float4v sums)
{
    const Factors by = factors(x.m, x.rest, m, rest);
    x.m = by.m;
    x.rest = by.rest;
    x.total = x.total * by.a + total * by.b;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        x.sums[i] = x.sums[i] * by.a + sums[i] * by.b;
}

template <typename Q, int HD>
__global__ __launch_bounds__(256) void merge_kernel(AttentionArgs p)
{
    constexpr int LANES = HD / 4, PAIRS = 64 / LANES; // pairs a wave
    __shared__ Joined others[3][64];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const Shared tile = p.shared[blockIdx.x];
    if (tile.workers < 2)
        return;
    const bool split = tile.workers > kMergeWays;
    const int step = split ? 4 : 1, begin = split ? wave : 0;
    const int each = split ? PAIRS : 4 * PAIRS; // pairs a block
    const int channel = lane % LANES * 4;
    for (int base = blockIdx.y * each; base < tile.pairs; base += gridDim.y * each) {
        const int pair = base + (split ? 0 : wave * PAIRS) + lane / LANES;
        const int read = min(pair, tile.pairs - 1);
        Joined x{kLow, 0.f, 0.f, {}};
#pragma unroll 4
        for (int v = begin; v < tile.workers; v += step) {
            const int64_t slot = ((int64_t) (blockIdx.x + v) * 2 + (v == 0)) * p.pairs + read;
            const float4 stat = *(const float4 *) (p.stats + slot * 4);
            join(x, stat.x, stat.y, stat.z, *(const float4v *) (p.sums + slot * HD + channel));
        }
        if (split) {
            __syncthreads(); // the last pairs' have been read
            if (wave > 0)
                others[wave - 1][lane] = x;
            __syncthreads();
            if (wave != 0)
                continue;
#pragma unroll
            for (int v = 0; v < 3; ++v)
                join(x, others[v][lane].m, others[v][lane].rest, others[v][lane].total, others[v][lane].sums);
        }
        if (pair >= tile.pairs || channel >= p.a.head_dim)
            continue;
        const float by = x.total > 0.f || x.total != x.total ? 1.f / x.total : 0.f;
        Q *out = (Q *) p.a.out + (int64_t) (tile.row + pair / p.group) * p.a.out_stride
                 + (int64_t) (tile.head + pair % p.group) * p.a.head_dim + channel;
        typedef Q Q4 __attribute__((ext_vector_type(4)));
        *(Q4 *) out = Q4{(Q) (x.sums[0] * by), (Q) (x.sums[1] * by), (Q) (x.sums[2] * by), (Q) (x.sums[3] * by)};
    }
}

int padded_head_dim(int head_dim)
{
    return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
}

constexpr int kWidePairs = 128, kNarrowPairs = 32;

// A tile's queries and outputs take about as long as three units where tiles are
// wide (at one unit 8192 rows of bf16 take 411 us and 2048 rows of fp32 67, at three
// 326 and 60, at five 326 and 61), and one where they are narrow (a worker there has a
// unit or two; at three, 16 x 7000 rows take 47 us instead of 45).
constexpr int kFixedWide = 3, kFixedNarrow = 1;

template <typename Q, int HD>
hipError_t launch(const PackedAttentionArgs &a, hipStream_t stream)
{
    AttentionArgs p{};
    p.a = a;
    p.group = a.heads / a.kv_heads;
    // A sequence's pairs on average: one tile of 32 pairs, whose two waves
    // share the keys, where they fit into it; else tiles of 128 pairs.  One token
    // of 8 x 4000 rows of 32 / 8 heads of 128: 38 us narrow, 39 wide (fp32 queries
    // 41 and 51); 8 tokens (32 pairs) 41 and 43; 12 tokens 54 and 44.  The average of a
    // batch of prompts and single tokens chooses one of them for both.
    const int64_t average = ((int64_t) a.seq.rows + a.seq.sequences - 1) / a.seq.sequences * p.group;
    const bool narrow = average <= kNarrowPairs;
    p.pairs = narrow ? kNarrowPairs : kWidePairs;
    int shift = 0;
    while ((2 << shift) * p.group <= p.pairs && (1 << shift) < a.seq.rows)
        ++shift;
    p.row_shift = shift;
    // no more workers than there can be units
    const int64_t tiles = ((int64_t) a.seq.rows >> shift) + a.seq.sequences;
    const int64_t keys = ((int64_t) (a.seq.cached ? a.seq.table_width : 0) << a.layer.page_shift);
    const int64_t most = tiles * a.kv_heads
                         * std::max<int64_t>(1, (keys + kKeys - 1) / kKeys
                                                    + (a.k ? (a.seq.rows + kKeys - 1) / kKeys : 0));
    // a KV head's slots of one sequence are counted in 32 bits
    const int64_t own = !a.k ? 0 : a.causal ? a.seq.rows : std::min(a.seq.rows, a.mask_words * kKeys);
    if ((((int64_t) a.seq.rows >> shift) + 2) * ((keys + own) / kKeys + 8) > INT32_MAX)
        return hipErrorInvalidValue;
    p.workers = (int) std::min<int64_t>(kWorkers<HD>, most);
    p.fixed = narrow ? kFixedNarrow : kFixedWide;
    p.sums = a.workspace;
    p.stats = p.sums + (int64_t) kWorkers<HD> * 2 * kWidePairs * HD;
    p.shared = (Shared *) (p.stats + (int64_t) kWorkers<HD> * 2 * kWidePairs * 4);
    if (narrow)
        hipLaunchKernelGGL((attention_kernel<Q, HD, 1, 2>), dim3(p.workers), dim3(128), 0, stream, p);
    else
        hipLaunchKernelGGL((attention_kernel<Q, HD, 4, 1>), dim3(p.workers), dim3(256), 0, stream, p);
    if (p.workers > 1) {
        const int blocks = std::min(((1 << shift) * p.group * HD + 255) / 256, 32);
        hipLaunchKernelGGL((merge_kernel<Q, HD>), dim3(p.workers - 1, blocks), dim3(256), 0, stream, p);
    }
    return hipGetLastError();
}

template <typename Q>
hipError_t launch_width(const PackedAttentionArgs &a, hipStream_t stream)
{
    switch (padded_head_dim(a.head_dim)) {
    case 64: return launch<Q, 64>(a, stream);
    case 128: return launch<Q, 128>(a, stream);
    default: return launch<Q, 256>(a, stream);
    }
}

} // namespace

size_t packed_attention_workspace_bytes(int heads, int kv_heads, int head_dim)
{
    (void) heads;
    (void) kv_heads;
    const int hd = padded_head_dim(head_dim);
    const int64_t workers = hd == 256 ? kWorkers<256> : kWorkers<128>;
    return (size_t) (workers * (2 * kWidePairs * (hd + 4) * 4 + (int64_t) sizeof(Shared)) + 64 * 16);
}

hipError_t launch_packed_attention(const PackedAttentionArgs &a, int q_type, hipStream_t stream)
{
    const int group = a.kv_heads > 0 ? a.heads / a.kv_heads : 0;
    if (a.seq.sequences <= 0 || a.seq.rows <= 0 || group <= 0 || group > kNarrowPairs
        || a.heads != group * a.kv_heads || a.head_dim <= 0 || a.head_dim > kPagedMaxHeadDim
        || a.head_dim % 8 != 0 || !a.workspace)
        return hipErrorInvalidValue;
    switch (q_type) {
    case GQ8_DTYPE_F32: return launch_width<float>(a, stream);
    case GQ8_DTYPE_F16: return launch_width<_Float16>(a, stream);
    case GQ8_DTYPE_BF16: return launch_width<__bf16>(a, stream);
    default: return hipErrorInvalidValue;
    }
}

} // namespace gq8
