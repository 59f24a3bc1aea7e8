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
// fp32 queries: q and p are split in two fp16 pieces each (q scaled by a power
// of two to below 2^14 a row, p by 2^kOffset; 22 bits, the rest below 2^-25 of
// the row's largest), and each product is two MFMAs on the same key or value
// operand.  fp16 and bf16 queries: p is rounded once to the operands' type
// (half a step of it, as the output's own rounding; weights are normalized by
// the sum of the unrounded p).
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
typedef float float16v __attribute__((ext_vector_type(16)));
typedef uint32_t word4 __attribute__((ext_vector_type(4)));

constexpr int kKeys = 64;          // keys a unit
constexpr float kLow = -3.0e38f;   // a row's reference before its first key
constexpr float kMargin = 4.f;     // how far (in powers of two) a score may pass it
constexpr float kFar = 65536.f;    // 2^-24 of it stays below a hundredth of a power
constexpr float kLeast = 1.0e-30f; // of the factor on a score
constexpr float kOffset = 10.f;    // fp32 queries: p is held times 2^10 (2^14 at most)
constexpr float kLog2e = 1.44269504088896340736f;

// workgroups of a launch: as many as are resident (128 KB of LDS at 256
// channels, 64 KB at 128), so that every run of units starts at once
template <int HD>
constexpr int kWorkers = HD == 256 ? 256 : 512;

struct AttentionArgs {
    PackedAttentionArgs a;
    int group, row_shift; // rows a tile = 1 << row_shift, each with its `group` heads
    int pairs;            // M
    int workers;
    float *sums, *stats;  // [workers, 2][M][HD], [workers, 2][M][2]
};

__device__ const word4 kZeroChunk = {0, 0, 0, 0};

// ---- where a unit lies -----------------------------------------------------------
struct Cursor {
    int s, g, r;         // sequence, KV head, tile of rows
    int chunk, chunks;   // the unit in its tile, the tile's units
    int start, n, c, tiles; // the sequence: first packed row, rows, cached rows, tiles
};

__device__ inline int uniform(int v)
{
    return __builtin_amdgcn_readfirstlane(v);
}

__device__ inline void sequence_of(const AttentionArgs &p, int s, int &start, int &n, int &c)
{
    const PackedSequences &q = p.a.seq;
    start = min(max(q.starts[s], 0), q.rows);
    n = min(max(q.starts[s + 1], start), q.rows) - start;
    c = q.cached ? min(max(q.cached[s], 0), q.table_width << p.a.layer.page_shift) : 0;
}

// new-row units of tile r (of `tiles`) of a sequence of n rows
__device__ inline int own_chunks(const AttentionArgs &p, int r, int n)
{
    if (!p.a.k)
        return 0;
    const int last = p.a.causal ? min((r + 1) << p.row_shift, n) : min(n, p.a.mask_words * kKeys);
    return (last + kKeys - 1) / kKeys;
}

__device__ inline int tile_chunks(const AttentionArgs &p, int r, int n, int c)
{
    return max(1, (c + kKeys - 1) / kKeys + own_chunks(p, r, n));
}

// units of the first t tiles of a KV head, in closed form: the rows of a tile
// and a unit's keys are powers of two
__device__ inline int64_t units_before(const AttentionArgs &p, int t, int tiles, int n, int c)
{
    const int cached = (c + kKeys - 1) / kKeys;
    if (!p.a.causal || !p.a.k)
        return (int64_t) t * max(1, cached + own_chunks(p, 0, n));
    int64_t own;
    if (p.row_shift < 6) { // sum of ceil((r + 1) / q), q tiles a unit of keys
        const int shift = 6 - p.row_shift;
        const int64_t whole = t >> shift, rest = t & ((1 << shift) - 1);
        own = (whole * (whole + 1) / 2 << shift) + rest * (whole + 1);
    } else {
        const int per = 1 << (p.row_shift - 6);
        const int64_t full = t < tiles ? t : t - 1;
        own = full * (full + 1) / 2 * per + (t == tiles && t > 0 ? (n + kKeys - 1) / kKeys : 0);
    }
    return (int64_t) t * cached + own;
}

__device__ inline int tiles_of(const AttentionArgs &p, int n)
{
    return (n + (1 << p.row_shift) - 1) >> p.row_shift;
}

__device__ inline int64_t sequence_units(const AttentionArgs &p, int s)
{
    int start, n, c;
    sequence_of(p, s, start, n, c);
    const int tiles = tiles_of(p, n);
    return tiles > 0 ? p.a.kv_heads * units_before(p, tiles, tiles, n, c) : 0;
}

__device__ inline int64_t broadcast(int64_t v, int lane)
{
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t) v, lane);
    const uint32_t hi = __builtin_amdgcn_readlane((uint32_t) (v >> 32), lane);
    return (int64_t) (((uint64_t) hi << 32) | lo);
}

// the sum over the lanes up to this one
__device__ inline int64_t scan(int64_t v, int lane)
{
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t other = __shfl_up(v, d);
        v += lane >= d ? other : 0;
    }
    return v;
}

// units of the whole batch (the same in every lane of every wave)
__device__ inline int64_t all_units(const AttentionArgs &p)
{
    const int lane = threadIdx.x & 63;
    int64_t total = 0;
    for (int s = lane; s < p.a.seq.sequences; s += 64)
        total += sequence_units(p, s);
    return broadcast(scan(total, lane), 63);
}

// the place of `unit` (below all_units)
__device__ inline Cursor locate(const AttentionArgs &p, int64_t unit)
{
    const int lane = threadIdx.x & 63;
    Cursor at{};
    int64_t before = 0;
    for (int base = 0; base < p.a.seq.sequences; base += 64) {
        const int64_t mine = base + lane < p.a.seq.sequences ? sequence_units(p, base + lane) : 0;
        const int64_t upto = scan(mine, lane) + before;
        const uint64_t past = __ballot(upto > unit);
        if (past) {
            const int found = __ffsll((unsigned long long) past) - 1;
            at.s = base + found;
            before = broadcast(upto - mine, found);
            break;
        }
        before = broadcast(upto, 63);
    }
    sequence_of(p, at.s, at.start, at.n, at.c);
    at.tiles = tiles_of(p, at.n);
    int64_t offset = unit - before;
    const int64_t per = max((int64_t) 1, units_before(p, at.tiles, at.tiles, at.n, at.c));
    at.g = (int) (offset / per);
    offset -= at.g * per;
    int low = 0, high = at.tiles - 1; // the last tile that starts at or before it
    while (low < high) {
        const int middle = (low + high + 1) >> 1;
        if (units_before(p, middle, at.tiles, at.n, at.c) <= offset)
            low = middle;
        else
            high = middle - 1;
    }
    at.r = low;
    at.chunk = (int) (offset - units_before(p, low, at.tiles, at.n, at.c));
    at.chunks = tile_chunks(p, at.r, at.n, at.c);
    at.s = uniform(at.s); at.g = uniform(at.g); at.r = uniform(at.r);
    at.chunk = uniform(at.chunk); at.chunks = uniform(at.chunks);
    at.start = uniform(at.start); at.n = uniform(at.n); at.c = uniform(at.c);
    at.tiles = uniform(at.tiles);
    return at;
}

__device__ inline void advance(const AttentionArgs &p, Cursor &at)
{
    if (++at.chunk < at.chunks)
        return;
    at.chunk = 0;
    if (++at.r >= at.tiles) {
        at.r = 0;
        if (++at.g >= p.a.kv_heads) {
            at.g = 0;
            at.n = 0;
            while (at.n == 0 && at.s + 1 < p.a.seq.sequences) {
                ++at.s;
                sequence_of(p, at.s, at.start, at.n, at.c);
                at.start = uniform(at.start); at.n = uniform(at.n); at.c = uniform(at.c);
            }
            at.tiles = tiles_of(p, at.n);
        }
    }
    at.chunks = tile_chunks(p, at.r, at.n, at.c);
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
// lies at c ^ swizzle(r), so that 8 rows' same chunk fill all banks and so do
// 4 rows' same pair of chunks.
template <int HD>
__device__ inline int swizzle(int row)
{
    return ((row & 3) << 1) | ((row >> 2) & 1) | (HD >= 128 ? row & 8 : 0);
}

// The row of the packed tensors or of the pool that holds the unit's key
// `lane`, -1 where it holds none (past the cached rows or the new ones, or in a
// page outside the pool).
__device__ inline int key_row(const AttentionArgs &p, const Cursor &at, int lane)
{
    const int cached = (at.c + kKeys - 1) / kKeys;
    if (at.chunk < cached) {
        const int key = at.chunk * kKeys + lane;
        if (key >= at.c)
            return -1;
        const int shift = p.a.layer.page_shift;
        const int page = p.a.seq.table[(int64_t) at.s * p.a.seq.table_width + (key >> shift)];
        if (page < 0 || page >= p.a.layer.pages)
            return -1;
        return (page << shift) + (key & ((1 << shift) - 1));
    }
    const int j = (at.chunk - cached) * kKeys + lane;
    return p.a.k && j < at.n ? at.start + j : -1;
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
#pragma clang diagnostic pop

__device__ inline uint32_t lds_address(const void *p)
{
    return (uint32_t) (uintptr_t) (__attribute__((address_space(3))) const void *) p;
}

// One unit's keys and values: 64 rows, WAVES waves, a wave 512 / HD rows an
// instruction.  Rows and channels that there are not are read as zeros.
template <int HD, int WAVES>
__device__ inline void load_unit(const AttentionArgs &p, const Cursor &at, int row, uint32_t keys,
                                 uint32_t values)
{
    constexpr int kChunks = HD / 8, kRows = 64 / kChunks;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const bool cache = at.chunk < (at.c + kKeys - 1) / kKeys;
    const uint16_t *k = cache ? p.a.layer.keys : p.a.k, *v = cache ? p.a.layer.values : p.a.v;
    const int stride = cache ? p.a.layer.width : p.a.kv_stride;
    const int channel = at.g * p.a.head_dim;
#pragma unroll
    for (int j = 0; j < 64 / WAVES / kRows; ++j) {
        const int r = wave * (64 / WAVES) + j * kRows + lane / kChunks;
        const int chunk = (lane % kChunks) ^ swizzle<HD>(r);
        const int from = __shfl(row, r);
        const bool there = from >= 0 && chunk * 8 < p.a.head_dim;
        const int64_t offset = (int64_t) from * stride + channel + chunk * 8;
        const void *zero = &kZeroChunk;
        const uint32_t to = (wave * (64 / WAVES) + j * kRows) * HD * 2;
        load_to_lds(there ? (const void *) (k + offset) : zero, keys + to);
        load_to_lds(there ? (const void *) (v + offset) : zero, values + to);
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
    static constexpr float kShift = 0.f;
    __device__ static float16v mfma(half8 a, half8 b, float16v c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    __device__ static void split(const float (&x)[8], Operand (&out)[1])
    {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            out[0][i] = (_Float16) x[i];
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
    __device__ static void split(const float (&x)[8], Operand (&out)[1])
    {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            out[0][i] = (__bf16) x[i];
    }
};

template <>
struct Arithmetic<float> : Arithmetic<_Float16> {
    static constexpr int kPieces = 2;
    static constexpr float kShift = kOffset;
    __device__ static void split(const float (&x)[8], Operand (&out)[2])
    {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const _Float16 high = (_Float16) x[i];
            out[0][i] = high;
            out[1][i] = (_Float16) (x[i] - (float) high);
        }
    }
};

// ---- a wave's state -----------------------------------------------------------------
template <typename Q, int HD>
struct State {
    using A = Arithmetic<Q>;
    typename A::Operand q[HD / 16][A::kPieces];
    float16v sums[HD / 32];
    // this lane's part of sum p; m, and the score it stands for (m = c raw); scale log2(e)
    float total, reference, raw, c;
};

template <typename Q, int HD>
__device__ inline void clear(State<Q, HD> &w)
{
#pragma unroll
    for (int i = 0; i < HD / 32; ++i)
        w.sums[i] = float16v{};
    w.total = 0.f;
    w.reference = w.raw = kLow;
}

// the pair's query (row `row` of the packed tensor, head `head`), zeros if not live
template <typename Q, int HD>
__device__ inline void load_query(const AttentionArgs &p, int64_t row, int head, bool live,
                                  State<Q, HD> &w)
{
    const int half = (threadIdx.x & 63) >> 5;
    const float scale = p.a.scale * kLog2e;
    const Q *from = (const Q *) p.a.q + (live ? row * p.a.q_stride + (int64_t) head * p.a.head_dim : 0);
    // never zero, so that a masked score (minus infinity) keeps its weight of zero
    w.c = fmaxf(fabsf(scale), kLeast);
    if constexpr (State<Q, HD>::A::kPieces == 2) {
        float x[HD / 16][8], largest = 0.f;
#pragma unroll
        for (int s = 0; s < HD / 16; ++s) {
            const int channel = 16 * s + 8 * half;
            const bool there = live && channel < p.a.head_dim;
            const float4 *at = (const float4 *) (from + (there ? channel : 0));
            const float4 a = at[0], b = at[1];
            const float y[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[s][i] = there ? y[i] : 0.f;
                largest = fmaxf(largest, fabsf(x[s][i]));
            }
        }
        largest = fmaxf(largest, xor_lane<32>(largest));
        // 2^-e brings the largest to [2^13, 2^14), rows below 2^-87 near it
        const int e = max((int) ((__float_as_uint(largest) >> 23) & 0xFF) - 127 - 13, -100);
        const float down = ldexpf(scale < 0.f ? -1.f : 1.f, -e);
        w.c = fmaxf(ldexpf(fabsf(scale), e), kLeast);
#pragma unroll
        for (int s = 0; s < HD / 16; ++s) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                x[s][i] *= down;
            State<Q, HD>::A::split(x[s], w.q[s]);
        }
    } else {
        const uint32_t sign = scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
        for (int s = 0; s < HD / 16; ++s) {
            const int channel = 16 * s + 8 * half;
            const bool there = live && channel < p.a.head_dim;
            word4 y = *(const word4 *) (from + (there ? channel : 0));
#pragma unroll
            for (int i = 0; i < 4; ++i)
                y[i] = there ? y[i] ^ sign : 0u;
            w.q[s][0] = __builtin_bit_cast(typename State<Q, HD>::A::Operand, y);
        }
    }
}

__device__ inline word4 lds_word4(uint32_t address)
{
    return *(__attribute__((address_space(3))) const word4 *) (uintptr_t) address;
}

__device__ inline short4v lds_transposed(uint32_t address)
{
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) short4v *) (uintptr_t) address);
}

// scores of key blocks [first, first + BLOCKS) of 32 keys
template <typename Q, int HD, int BLOCKS>
__device__ inline void scores(const State<Q, HD> &w, uint32_t keys, int first,
                              float16v (&s)[BLOCKS])
{
    using A = Arithmetic<Q>;
    const int lane = threadIdx.x & 63, row = lane & 31, half = lane >> 5;
    const uint32_t base = keys + (first * 32 + row) * HD * 2 + ((half ^ swizzle<HD>(row)) << 4);
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
        s[b] = float16v{};
#pragma unroll
    for (int k = 0; k < HD / 16; ++k) {
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
            const auto a = __builtin_bit_cast(typename A::Operand,
                                              lds_word4((base ^ (k * 32)) + b * 32 * HD * 2));
#pragma unroll
            for (int i = 0; i < A::kPieces; ++i)
                s[b] = A::mfma(a, w.q[k][i], s[b]);
        }
    }
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

// sums += P V over the wave's keys
template <typename Q, int HD, int BLOCKS>
__device__ inline void weigh(State<Q, HD> &w, uint32_t values, int first, const float16v (&p)[BLOCKS])
{
    using A = Arithmetic<Q>;
    const int lane = threadIdx.x & 63, half = lane >> 5, i16 = lane & 15;
    const int row = first * 32 + 4 * half + (i16 >> 2); // of a step's first four keys
    const int chunk = 2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1);
    const uint32_t base = values + row * HD * 2 + ((chunk ^ swizzle<HD>(row)) << 4) + (i16 & 1) * 8;
#pragma unroll
    for (int t = 0; t < 2 * BLOCKS; ++t) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x[i] = p[t / 2][8 * (t & 1) + i];
        typename A::Operand b[A::kPieces];
        A::split(x, b);
#pragma unroll
        for (int cb = 0; cb < HD / 32; ++cb) {
            const uint32_t at = (base ^ (cb * 64)) + t * 16 * HD * 2;
            const short4v low = lds_transposed(at);
            const short4v high = lds_transposed((HD >= 128 ? at ^ 128 : at) + 8 * HD * 2);
            typedef short short8v __attribute__((ext_vector_type(8)));
            const short8v both = __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
            const auto a = __builtin_bit_cast(typename A::Operand, both);
#pragma unroll
            for (int i = 0; i < A::kPieces; ++i)
                w.sums[cb] = A::mfma(a, b[i], w.sums[cb]);
        }
    }
}

// One unit for this wave's pairs: keys of blocks [first, first + BLOCKS).
// `masked`: some keys are not for all pairs; `allowed` has a bit for each of
// the unit's keys that this lane's pair attends.
template <typename Q, int HD, int BLOCKS>
__device__ inline void attend(State<Q, HD> &w, uint32_t keys, uint32_t values, int first,
                              bool masked, uint64_t allowed)
{
    using A = Arithmetic<Q>;
    const int half = (threadIdx.x & 63) >> 5;
    float16v s[BLOCKS];
    scores<Q, HD, BLOCKS>(w, keys, first, s);
    if (masked) {
        const uint64_t mine = allowed >> (32 * first + 4 * half);
#pragma unroll
        for (int i = 0; i < 16 * BLOCKS; ++i)
            if (!((mine >> (32 * (i / 16) + 8 * ((i % 16) / 4) + i % 4)) & 1))
                s[i / 16][i % 16] = -INFINITY;
    }
    float largest = s[0][0];
#pragma unroll
    for (int i = 1; i < 16 * BLOCKS; ++i)
        largest = fmaxf(largest, s[i / 16][i % 16]);
    largest = fmaxf(largest, xor_lane<32>(largest));
    if (__ballot(largest * w.c > w.reference + kMargin)) {
        w.raw = fmaxf(largest, w.raw);
        const float next = fmaxf(largest * w.c, w.reference);
        const float factor = __builtin_amdgcn_exp2f(w.reference - next);
        w.reference = next;
        w.total *= factor;
#pragma unroll
        for (int cb = 0; cb < HD / 32; ++cb)
            w.sums[cb] *= factor;
    }
    float minus = A::kShift - w.reference;
    // m is rounded: by up to 2^-24 |m|, which is the same power for all of a
    // row's weights, unless it leaves their range.  Far scores are taken from
    // theirs first, which leaves the largest an exact zero.
    if (__ballot(fabsf(w.reference) > kFar)) {
#pragma unroll
        for (int i = 0; i < 16 * BLOCKS; ++i)
            s[i / 16][i % 16] -= w.raw;
        minus = A::kShift;
    }
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < 16 * BLOCKS; ++i) {
        const float e = __builtin_amdgcn_exp2f(fmaf(s[i / 16][i % 16], w.c, minus));
        s[i / 16][i % 16] = e;
        total += e;
    }
    w.total += total;
    weigh<Q, HD, BLOCKS>(w, values, first, s);
}

template <typename Q>
__device__ inline void store4(Q *to, const float (&x)[4])
{
    if constexpr (sizeof(Q) == 4) {
        *(float4 *) to = float4{x[0], x[1], x[2], x[3]};
    } else {
        typedef Q Q4 __attribute__((ext_vector_type(4)));
        *(Q4 *) to = Q4{(Q) x[0], (Q) x[1], (Q) x[2], (Q) x[3]};
    }
}

// A workgroup's run of units.  ROWS waves take 32 pairs each, of all 64 keys of
// a unit (ROWS > 1), or KEYS waves take 32 keys each, of the same 32 pairs.
template <typename Q, int HD, int ROWS, int KEYS>
__global__ __launch_bounds__(64 * ROWS * KEYS) void attention_kernel(AttentionArgs p)
{
    static_assert(KEYS == 1 || (KEYS == 2 && ROWS == 1), "a unit is two blocks of 32 keys");
    constexpr int WAVES = ROWS * KEYS, BLOCKS = 2 / KEYS, kTile = kKeys * HD * 2;
    __shared__ __align__(1024) uint8_t lds[4 * kTile]; // keys, values, twice
    __shared__ float exchange[KEYS == 2 ? 128 : 1];
    __shared__ uint64_t taken[HD][2];
    __shared__ uint32_t found[WAVES];
    const uint32_t tiles = uniform(lds_address(lds));
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), half = lane >> 5;
    const int pair = (KEYS == 2 ? 0 : wave * 32) + (lane & 31); // of the tile
    const int first = KEYS == 2 ? wave : 0;                     // key block

    const int64_t units = all_units(p);
    const int64_t share = (units + p.workers - 1) / p.workers;
    const int worker = worker_of(blockIdx.x, p.workers);
    const int64_t from = worker * share, to = min(units, from + share);
    if (from >= to)
        return;
    const int count = (int) (to - from);

    Cursor at = locate(p, from), ahead = at;
    int row = key_row(p, ahead, lane);
    uint64_t present = __ballot(row >= 0), next_present = 0;
    load_unit<HD, WAVES>(p, ahead, row, tiles, tiles + kTile);
    advance(p, ahead);
    int next_row = count > 1 ? key_row(p, ahead, lane) : -1;

    const int pair_row = pair / p.group, pair_head = pair - pair_row * p.group;
    State<Q, HD> w;
    bool fresh = true;
    int first_chunk = 0;
    for (int u = 0; u < count; ++u) {
        const uint32_t keys = tiles + (u & 1) * 2 * kTile, values = keys + kTile;
        // row i of the sequence that this lane's pair belongs to
        const int i = (at.r << p.row_shift) + pair_row;
        const bool live = pair_row < (1 << p.row_shift) && i < at.n;
        const int head = at.g * p.group + pair_head;
        if (fresh) {
            clear(w);
            load_query(p, (int64_t) at.start + i, head, live, w);
            first_chunk = at.chunk;
            fresh = false;
        }
        // this unit's rows are there, and every wave has done with the other buffer
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (u + 1 < count) {
            const uint32_t other = tiles + (1 - (u & 1)) * 2 * kTile;
            next_present = __ballot(next_row >= 0);
            load_unit<HD, WAVES>(p, ahead, next_row, other, other + kTile);
            advance(p, ahead);
            next_row = u + 2 < count ? key_row(p, ahead, lane) : -1;
        }
        const int cached = (at.c + kKeys - 1) / kKeys;
        uint64_t allowed = present;
        bool masked = present != ~0ull;
        if (at.chunk >= cached) {
            const int key = (at.chunk - cached) * kKeys; // the first new row of the unit
            if (p.a.causal) {
                masked |= key + kKeys - 1 > at.r << p.row_shift;
                const int last = i - key;
                allowed &= last >= 63 ? ~0ull : last < 0 ? 0 : (2ull << last) - 1;
            } else {
                masked = true;
                allowed &= live && p.a.k ? p.a.masks[(int64_t) (at.start + i) * p.a.mask_words + key / kKeys] : 0;
            }
        }
        const bool took = masked && take_out<Q, HD, WAVES>(values, found, taken);
        if (__ballot(live)) {
            attend<Q, HD, BLOCKS>(w, keys, values, first, masked, allowed);
            if (took)
                put_back(w, taken, KEYS == 2 ? allowed & 0xFFFFFFFFull << (32 * first) : allowed);
        }

        const bool last_of_tile = at.chunk + 1 == at.chunks;
        if (last_of_tile || u + 1 == count) {
            float total = w.total + xor_lane<32>(w.total);
            bool writes = live;
            if constexpr (KEYS == 2) { // the second wave's sums through the unit's buffer
                float *area = (float *) (lds + (u & 1) * 2 * kTile);
                __syncthreads();
                if (wave == 1) {
#pragma unroll
                    for (int j = 0; j < HD / 2; ++j)
                        area[j * 64 + lane] = w.sums[j / 16][j % 16];
                    exchange[lane] = total;
                    exchange[64 + lane] = w.reference;
                }
                __syncthreads();
                writes = writes && wave == 0;
                if (wave == 0) {
                    const float theirs = exchange[64 + lane];
                    const float next = fmaxf(w.reference, theirs);
                    const float a = __builtin_amdgcn_exp2f(w.reference - next);
                    const float b = __builtin_amdgcn_exp2f(theirs - next);
                    total = total * a + exchange[lane] * b;
                    w.reference = next;
#pragma unroll
                    for (int j = 0; j < HD / 2; ++j)
                        w.sums[j / 16][j % 16] = w.sums[j / 16][j % 16] * a + area[j * 64 + lane] * b;
                }
            }
            if (first_chunk == 0 && last_of_tile) {
                const float by = total > 0.f || total != total ? 1.f / total : 0.f;
                Q *out = (Q *) p.a.out + (writes ? (int64_t) (at.start + i) * p.a.out_stride
                                                       + (int64_t) head * p.a.head_dim : 0);
#pragma unroll
                for (int j = 0; j < HD / 8; ++j) {
                    const int channel = 8 * j + 4 * half;
                    const float x[4] = {w.sums[j / 4][4 * (j % 4)] * by, w.sums[j / 4][4 * (j % 4) + 1] * by,
                                        w.sums[j / 4][4 * (j % 4) + 2] * by, w.sums[j / 4][4 * (j % 4) + 3] * by};
                    if (writes && channel < p.a.head_dim)
                        store4(out + channel, x);
                }
            } else if (writes) {
                // slot 0: the tile began with an earlier worker; 1: it begins here
                const int64_t slot = ((int64_t) worker * 2 + (first_chunk == 0)) * p.pairs + pair;
                float *sums = p.sums + slot * HD;
#pragma unroll
                for (int j = 0; j < HD / 8; ++j)
                    *(float4 *) (sums + 8 * j + 4 * half) =
                        float4{w.sums[j / 4][4 * (j % 4)], w.sums[j / 4][4 * (j % 4) + 1],
                               w.sums[j / 4][4 * (j % 4) + 2], w.sums[j / 4][4 * (j % 4) + 3]};
                if (half == 0)
                    *(float2 *) (p.stats + slot * 2) = float2{w.reference, total};
            }
            fresh = true;
        }
        advance(p, at);
        present = next_present;
    }
}

// Joins the tiles that several workers share.  Block (b, y): the tile across
// the end of worker b's run, if b is the first of its workers; four waves take
// its workers in turn, for the pairs y, y + gridDim.y, ...
template <typename Q, int HD>
__global__ __launch_bounds__(256) void merge_kernel(AttentionArgs p)
{
    constexpr int N = HD / 64; // channels a lane
    __shared__ float sSums[4][HD], sStats[4][2];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int64_t units = all_units(p);
    const int64_t share = (units + p.workers - 1) / p.workers;
    const int worker = blockIdx.x;
    const int64_t end = (worker + 1) * share; // the first unit past it
    if (end >= units)
        return;
    const Cursor at = locate(p, end - 1);
    if (at.chunk + 1 == at.chunks)
        return; // the tile ends with the run
    const int64_t begin = end - 1 - at.chunk;
    if (begin < worker * share)
        return; // an earlier worker's
    const int last = (int) ((begin + at.chunks - 1) / share); // its last worker
    const int group = p.group;
    const int pairs = min(1 << p.row_shift, at.n - (at.r << p.row_shift)) * group;
    for (int pair = blockIdx.y; pair < pairs; pair += gridDim.y) {
        float m = kLow, total = 0.f, sums[N] = {};
        for (int v = worker + wave; v <= last; v += 4) {
            const int64_t slot = ((int64_t) v * 2 + (v == worker)) * p.pairs + pair;
            const float2 stat = *(const float2 *) (p.stats + slot * 2);
            float x[N];
#pragma unroll
            for (int i = 0; i < N; ++i)
                x[i] = p.sums[slot * HD + lane * N + i];
            const float next = fmaxf(m, stat.x);
            const float a = __builtin_amdgcn_exp2f(m - next), b = __builtin_amdgcn_exp2f(stat.x - next);
            m = next;
            total = total * a + stat.y * b;
#pragma unroll
            for (int i = 0; i < N; ++i)
                sums[i] = sums[i] * a + x[i] * b;
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
            sSums[wave][lane * N + i] = sums[i];
        if (lane == 0) {
            sStats[wave][0] = m;
            sStats[wave][1] = total;
        }
        __syncthreads();
        const int channel = threadIdx.x;
        if (channel < p.a.head_dim) {
            float most = sStats[0][0];
#pragma unroll
            for (int v = 1; v < 4; ++v)
                most = fmaxf(most, sStats[v][0]);
            float sum = 0.f, all = 0.f;
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const float f = __builtin_amdgcn_exp2f(sStats[v][0] - most);
                sum += sSums[v][channel] * f;
                all += sStats[v][1] * f;
            }
            const int i = (at.r << p.row_shift) + pair / group;
            const int head = at.g * group + pair % group;
            const float by = all > 0.f || all != all ? 1.f / all : 0.f;
            ((Q *) p.a.out)[(int64_t) (at.start + i) * p.a.out_stride + (int64_t) head * p.a.head_dim
                            + channel] = (Q) (sum * by);
        }
        __syncthreads();
    }
}

int padded_head_dim(int head_dim)
{
    return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
}

constexpr int kWidePairs = 128, kNarrowPairs = 32;

template <typename Q, int HD>
hipError_t launch(const PackedAttentionArgs &a, hipStream_t stream)
{
    AttentionArgs p{};
    p.a = a;
    p.group = a.heads / a.kv_heads;
    // A sequence's pairs on average: one tile of 32 pairs, whose two waves
    // share the keys, where they fit into it; else tiles of 128 pairs.
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
    p.workers = (int) std::min<int64_t>(kWorkers<HD>, most);
    p.sums = a.workspace;
    p.stats = p.sums + (int64_t) kWorkers<HD> * 2 * kWidePairs * HD;
    if (narrow)
        hipLaunchKernelGGL((attention_kernel<Q, HD, 1, 2>), dim3(p.workers), dim3(128), 0, stream, p);
    else
        hipLaunchKernelGGL((attention_kernel<Q, HD, 4, 1>), dim3(p.workers), dim3(256), 0, stream, p);
    if (p.workers > 1) {
        const int pairs = std::min((1 << shift) * p.group, p.pairs);
        hipLaunchKernelGGL((merge_kernel<Q, HD>), dim3(p.workers - 1, std::min(pairs, 32)), dim3(256), 0,
                           stream, p);
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
    return (size_t) (workers * 2 * kWidePairs * (hd + 2) * 4);
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
