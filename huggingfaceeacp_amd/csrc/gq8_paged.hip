// gq8_paged.hip -- rows of a paged cache: the norms and rotation of a step's
// queries and keys, the append of packed rows (after those or with them), and the
// copy of whole pages.
// At a few rows all three are bound by the launch (3 to 5 us of kernel, 7 to 8 a
// call back to back).
#include "gemma_q8.h"
#include "gq8_lanes.hpp"
#include "gq8_paged.hpp"
#include "gq8_paged_rows.hpp"

#include <algorithm>
#include <cmath>

namespace gq8 {
namespace {

typedef uint32_t word4 __attribute__((ext_vector_type(4)));

// ---- norms and rotation ----------------------------------------------------------
// y = x / sqrt(mean(x^2) + eps) (1 + w), then the halves (a, b) of the head
// become (a cos - b sin, a sin + b cos).  P lanes take a head, each four
// channels of either half, so a lane holds both values of its four rotations;
// the sum of squares is added across the P lanes.  Sums, the root and the
// rotation are double, as in the decoder's own norm; the result is rounded
// once, to its type.
//
// 2048 rows of 32 + 2 x 8 heads of 128 in bf16 (50 MB of rows read and written)
// take 15.5 us, 3.2 TB/s, where a copy of as much takes 11: the double operations
// bound it (19.0 us with a division and a root of their own a head, and the row
// found by dividing in every lane).
template <typename X>
__device__ inline void load4(const X *p, float (&x)[4])
{
    if constexpr (sizeof(X) == 4) {
        const float4 v = *(const float4 *) p;
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
        typedef X X4 __attribute__((ext_vector_type(4)));
        const X4 v = *(const X4 *) p;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            x[i] = (float) v[i];
    }
}

// To fp32 with the last bit set where that is not exact: what is rounded from there on
// is rounded once.
__device__ inline float to_odd(double x)
{
    const float near = (float) x;
    uint32_t bits = __float_as_uint(near);
    if (((double) near < x || (double) near > x) && !(bits & 1))
        bits += fabs((double) near) < fabs(x) ? 1 : -1;
    return __uint_as_float(bits);
}

// To fp32 first: at most 2^-24 of the value on top of the type's half step.  Of 16 bits the
// first of four alone, the others are rounded once: which of them are is written down here
// (and each multiply-add below by itself), since a compiler that chooses gives a row other
// bits in another kernel.
template <typename Y>
__device__ inline void store_as(void *to, int64_t at, const double (&x)[4])
{
    typedef Y Y4 __attribute__((ext_vector_type(4)));
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[i] = sizeof(Y) == 2 && i > 0 ? to_odd(x[i]) : (float) x[i];
        asm("" : "+v"(f[i]));
    }
    *(Y4 *) ((Y *) to + at) = Y4{(Y) f[0], (Y) f[1], (Y) f[2], (Y) f[3]};
}

__device__ inline void store4(void *to, int type, int64_t at, const double (&x)[4])
{
    if (type == GQ8_DTYPE_F32)
        store_as<float>(to, at, x);
    else if (type == GQ8_DTYPE_F16)
        store_as<_Float16>(to, at, x);
    else
        store_as<__bf16>(to, at, x);
}

template <int D>
__device__ inline double sum_group(double v, int lanes)
{
    if constexpr (D > 0) {
        if (lanes > D)
            v += xor_lane<D>(v);
        return sum_group<D / 2>(v, lanes);
    }
    return v;
}

// A lane's place in its head, and its channels' rotation at a position.
struct Turn {
    int lanes, half, channel;
    bool there; // the position is in the tables, the channels in the head
    double cosine[4], sine[4];
};

__device__ inline Turn turn_at(const NormRopeArgs &a, int shift, int position)
{
    Turn turn;
    turn.lanes = 1 << shift;
    turn.half = a.head_dim / 2;
    turn.channel = (threadIdx.x & (turn.lanes - 1)) * 4;
    turn.there = turn.channel < turn.half && position >= 0 && position < a.max_positions;
    float cosine[4] = {}, sine[4] = {};
    if (turn.there) {
        load4(a.cosines + (int64_t) position * turn.half + turn.channel, cosine);
        load4(a.sines + (int64_t) position * turn.half + turn.channel, sine);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        turn.cosine[i] = cosine[i];
        turn.sine[i] = sine[i];
    }
    return turn;
}

// What P lanes do with head `slot` of row `row`: the query to its row of q, a key or a
// value to its row, k_row or v_row (null: nowhere).
template <typename X>
__device__ inline void norm_rope_head(const NormRopeArgs &a, int q_type, int kv_type, const Turn &turn,
                                      double one_of_head, int row, int slot, bool with_k, bool with_v,
                                      uint16_t *k_row, uint16_t *v_row)
{
    const int slots = a.heads + (with_k ? a.kv_heads : 0) + (with_v ? a.kv_heads : 0);
    const int half = turn.half, channel = turn.channel;
    const bool there = turn.there && slot < slots;
    const bool is_q = slot < a.heads;
    const int kv = slot - a.heads; // its k heads, then its v heads
    const bool is_k = !is_q && with_k && kv < a.kv_heads;
    // the fused row's columns: q heads, k heads, v heads
    const int column = is_q || with_k ? slot : slot + a.kv_heads;
    const X *x = (const X *) a.x + (int64_t) row * a.x_stride + (int64_t) column * a.head_dim + channel;
    float first[4] = {}, second[4] = {};
    if (there) {
        load4(x, first);
        load4(x + half, second);
    }
    double u[4], w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        u[i] = first[i];
        w[i] = second[i];
    }
    const float *weight = is_q ? a.q_weight : is_k ? a.k_weight : nullptr;
    double squares = 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        squares += fma(u[i], u[i], w[i] * w[i]);
    squares = sum_group<32>(squares, turn.lanes);
    if (!there)
        return;
    if (weight) {
        const double by = rsqrt(fma(squares, one_of_head, (double) a.epsilon));
        float g0[4], g1[4];
        load4(weight + channel, g0);
        load4(weight + half + channel, g1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u[i] *= fma(by, (double) g0[i], by);
            w[i] *= fma(by, (double) g1[i], by);
        }
    }
    if (is_q || is_k) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double x0 = u[i], x1 = w[i];
            u[i] = fma(x0, turn.cosine[i], -(x1 * turn.sine[i]));
            w[i] = fma(x0, turn.sine[i], x1 * turn.cosine[i]);
        }
    }
    const int head = is_q ? slot : with_k && !is_k ? kv - a.kv_heads : kv;
    void *to = is_q ? a.q : is_k ? k_row : v_row;
    if (!to)
        return;
    const int type = is_q ? q_type : kv_type;
    const int64_t at = (is_q ? (int64_t) row * a.q_stride : 0) + (int64_t) head * a.head_dim + channel;
    store4(to, type, at, u);
    store4(to, type, at + half, w);
}

template <typename X>
__global__ __launch_bounds__(256) void norm_rope_kernel(NormRopeArgs a, int q_type, int kv_type,
                                                        int shift, int blocks, double one_of_head)
{
    // a block's heads are of one row: its place is found in scalar registers
    const int row = (int) ((unsigned) blockIdx.x / (unsigned) blocks);
    const int slot = (((int) blockIdx.x - row * blocks) << (8 - shift)) + (int) (threadIdx.x >> shift);
    auto row_of = [&](void *to) { return to ? (uint16_t *) to + (int64_t) row * a.kv_stride : nullptr; };
    norm_rope_head<X>(a, q_type, kv_type, turn_at(a, shift, a.positions[row]), one_of_head, row, slot,
                      a.k != nullptr, a.v != nullptr, row_of(a.k), row_of(a.v));
}

// The same with keys and values straight into their pages: the rows of k and v are
// neither written nor read again, and a launch goes.  A row's position is its place
// in its sequence where none are given, and a row left out of the cache has none then.  Block (row, y) takes every gridDim.y-th turn of the
// row's heads: it finds the row's page once, and the position's rotation.  113 MB of bf16
// prompts (4493 rows) take 31.5 us, 3.6 TB/s, bound by its double operations; one row 3.5 us
// traced, 7.9 a call.
template <typename X>
__global__ __launch_bounds__(256) void append_rope_kernel(NormRopeArgs a, int q_type, int kv_type,
                                                          int shift, int turns, double one_of_head,
                                                          PagedLayer layer, PackedSequences seq,
                                                          const int *places, int first)
{
    const int row = first + (int) blockIdx.x;
    const int s = sequence_of_row(seq, row);
    if (s < 0)
        return;
    const int64_t place = places ? places[row] : row - (int64_t) max(seq.starts[s], 0);
    const int64_t key = (seq.cached ? max(seq.cached[s], 0) : 0) + place;
    const int position = a.positions ? a.positions[row] : place < 0 || key > INT32_MAX ? -1 : (int) key;
    const int64_t at = place < 0 ? -1 : pool_row(layer, seq, s, key);
    const Turn turn = turn_at(a, shift, position);
    auto row_of = [&](uint16_t *pool) { return at < 0 ? nullptr : pool + at * layer.width; };
    uint16_t *k_row = row_of(layer.keys), *v_row = row_of(layer.values);
#pragma unroll 1
    for (int t = blockIdx.y; t < turns; t += gridDim.y)
        norm_rope_head<X>(a, q_type, kv_type, turn, one_of_head, row, (t << (8 - shift)) + (int) (threadIdx.x >> shift),
                          true, true, k_row, v_row);
}

// ---- rows into pages ----------------------------------------------------------------
// A wave takes a packed row: it finds the row's sequence (the starts at or
// before it, counted 64 at a time), looks up the page and moves the row's keys
// and values in 16-byte pieces.  Bound by that chain of three reads: 7464 rows of
// 256 in 16 prompts take 4.6 us (15 MB read and written, 3.3 TB/s).
__global__ __launch_bounds__(256) void page_append_kernel(PagedLayer layer, PackedSequences seq,
                                                          const uint16_t *k, const uint16_t *v,
                                                          int kv_stride, const int *places, int first)
{
    const int lane = threadIdx.x & 63;
    const int t = first + blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (t >= seq.rows)
        return;
    const int s = sequence_of_row(seq, t);
    if (s < 0)
        return;
    const int64_t place = places ? places[t] : t - (int64_t) max(seq.starts[s], 0);
    const int64_t row = place < 0 ? -1 : pool_row(layer, seq, s, (seq.cached ? max(seq.cached[s], 0) : 0) + place);
    if (row < 0)
        return;
    const int chunks = layer.width / 8;
    for (int i = lane; i < 2 * chunks; i += 64) {
        const bool value = i >= chunks;
        const int at = (value ? i - chunks : i) * 8;
        const word4 x = *(const word4 *) ((value ? v : k) + (int64_t) t * kv_stride + at);
        *(word4 *) ((value ? layer.values : layer.keys) + row * layer.width + at) = x;
    }
}

// ---- whole pages -----------------------------------------------------------------------
constexpr int kCopyChunks = 4; // 16-byte chunks a thread
constexpr int kCopyBytes = 256 * 16 * kCopyChunks;

// Block (pair and piece of the page, layer and pool): 16 KB, read before it is
// written.  Bound by memory: 500 pages of 16 rows of 256 in 18 layers (295 MB read
// and written) take 46 us, 6.4 TB/s, more than a copy of 4 GB reaches (4.8),
// since a part of it stays in the last-level cache.
__global__ __launch_bounds__(256) void page_copy_kernel(uint8_t *keys, uint8_t *values, int pages,
                                                        int64_t page_bytes, const int *pairs,
                                                        int pieces)
{
    const int pair = blockIdx.x / pieces, piece = blockIdx.x % pieces;
    const int from = pairs[2 * pair], to = pairs[2 * pair + 1];
    if (from < 0 || from >= pages || to < 0 || to >= pages)
        return;
    uint8_t *pool = (blockIdx.y & 1 ? values : keys) + (int64_t) (blockIdx.y >> 1) * pages * page_bytes;
    const uint8_t *source = pool + from * page_bytes;
    uint8_t *target = pool + to * page_bytes;
    word4 x[kCopyChunks];
    const int64_t at = (int64_t) piece * kCopyBytes + threadIdx.x * 16;
#pragma unroll
    for (int i = 0; i < kCopyChunks; ++i)
        if (at + i * 4096 < page_bytes)
            x[i] = *(const word4 *) (source + at + i * 4096);
#pragma unroll
    for (int i = 0; i < kCopyChunks; ++i)
        if (at + i * 4096 < page_bytes)
            *(word4 *) (target + at + i * 4096) = x[i];
}

// A grid's threads are counted in 32 bits: blocks of 256 a launch at most.  What
// takes more is launched in parts.
constexpr int64_t kMostBlocks = (1 << 24) - 1;

int64_t bytes_of(int type)
{
    return type == GQ8_DTYPE_F32 ? 4 : 2;
}

} // namespace

hipError_t launch_head_norm_rope(const NormRopeArgs &a, int x_type, int q_type, int kv_type,
                                 hipStream_t stream)
{
    int shift = 0;
    while ((8 << shift) < a.head_dim)
        ++shift;
    const int64_t slots = (int64_t) a.heads + (a.k ? a.kv_heads : 0) + (a.v ? a.kv_heads : 0);
    const int64_t each = ((slots << shift) + 255) / 256; // blocks a row
    if (a.rows <= 0 || a.head_dim > kPagedMaxHeadDim || a.head_dim % 8 != 0 || slots <= 0
        || each > kMostBlocks)
        return hipErrorInvalidValue;
    const double one_of_head = 1.0 / a.head_dim;
    for (int64_t row = 0; row < a.rows;) {
        NormRopeArgs part = a;
        part.rows = (int) std::min(a.rows - row, kMostBlocks / each);
        part.x = (const uint8_t *) a.x + row * a.x_stride * bytes_of(x_type);
        part.positions = a.positions + row;
        part.q = (uint8_t *) a.q + row * a.q_stride * bytes_of(q_type);
        part.k = a.k ? (uint8_t *) a.k + row * a.kv_stride * 2 : nullptr;
        part.v = a.v ? (uint8_t *) a.v + row * a.kv_stride * 2 : nullptr;
        const dim3 grid((unsigned) (part.rows * each)), block(256);
        switch (x_type) {
        case GQ8_DTYPE_F32:
            hipLaunchKernelGGL(norm_rope_kernel<float>, grid, block, 0, stream, part, q_type, kv_type, shift,
                               (int) each, one_of_head);
            break;
        case GQ8_DTYPE_F16:
            hipLaunchKernelGGL(norm_rope_kernel<_Float16>, grid, block, 0, stream, part, q_type, kv_type, shift,
                               (int) each, one_of_head);
            break;
        case GQ8_DTYPE_BF16:
            hipLaunchKernelGGL(norm_rope_kernel<__bf16>, grid, block, 0, stream, part, q_type, kv_type, shift,
                               (int) each, one_of_head);
            break;
        default:
            return hipErrorInvalidValue;
        }
        if (hipError_t s = hipGetLastError())
            return s;
        row += part.rows;
    }
    return hipSuccess;
}

hipError_t launch_append_rope(const NormRopeArgs &a, int x_type, int q_type, int kv_type,
                              const PagedLayer &layer, const PackedSequences &seq, const int *places,
                              hipStream_t stream)
{
    int shift = 0;
    while ((8 << shift) < a.head_dim)
        ++shift;
    const int64_t slots = (int64_t) a.heads + 2 * a.kv_heads;
    const int64_t turns = ((slots << shift) + 255) / 256; // of a block for a row's heads
    if (a.rows <= 0 || seq.sequences <= 0 || a.head_dim > kPagedMaxHeadDim || a.head_dim % 8 != 0
        || layer.width != a.kv_heads * a.head_dim || turns > INT32_MAX)
        return hipErrorInvalidValue;
    const double one_of_head = 1.0 / a.head_dim;
    // Few rows: a block a turn, so that their heads run at once.  Many: one block a row,
    // which finds its page and rotation once (4493 rows of 48 heads: 32.1 us, a block a
    // turn 40.5).
    const int64_t parts = std::clamp<int64_t>(2048 / a.rows, 1, std::min<int64_t>(turns, 65535));
    for (int64_t row = 0; row < a.rows;) {
        const int64_t rows = std::min(a.rows - row, kMostBlocks / parts);
        auto launch = [&](auto *kernel) {
            hipLaunchKernelGGL(kernel, dim3((unsigned) rows, (unsigned) parts), dim3(256), 0, stream, a, q_type, kv_type,
                               shift, (int) turns, one_of_head, layer, seq, places, (int) row);
        };
        switch (x_type) {
        case GQ8_DTYPE_F32: launch(append_rope_kernel<float>); break;
        case GQ8_DTYPE_F16: launch(append_rope_kernel<_Float16>); break;
        case GQ8_DTYPE_BF16: launch(append_rope_kernel<__bf16>); break;
        default: return hipErrorInvalidValue;
        }
        if (hipError_t s = hipGetLastError())
            return s;
        row += rows;
    }
    return hipSuccess;
}

hipError_t launch_page_append(const PagedLayer &layer, const PackedSequences &seq,
                              const uint16_t *k, const uint16_t *v, int kv_stride,
                              const int *places, hipStream_t stream)
{
    if (seq.rows <= 0 || seq.sequences <= 0 || layer.width % 8 != 0)
        return hipErrorInvalidValue;
    for (int64_t row = 0; row < seq.rows; row += kMostBlocks * 4) {
        const int64_t blocks = std::min((seq.rows - row + 3) / 4, kMostBlocks);
        hipLaunchKernelGGL(page_append_kernel, dim3((unsigned) blocks), dim3(256), 0, stream, layer, seq, k, v,
                           kv_stride, places, (int) row);
        if (hipError_t s = hipGetLastError())
            return s;
    }
    return hipSuccess;
}

hipError_t launch_page_copy(void *keys, void *values, int layers, int pages, int64_t page_bytes,
                            const int *pairs, int count, hipStream_t stream)
{
    const int64_t pieces = (page_bytes + kCopyBytes - 1) / kCopyBytes;
    if (count <= 0 || layers <= 0 || layers > 32767 || page_bytes % 16 != 0 || pieces > kMostBlocks)
        return hipErrorInvalidValue;
    for (int64_t pair = 0; pair < count;) {
        const int64_t some = std::min(count - pair, kMostBlocks / pieces);
        hipLaunchKernelGGL(page_copy_kernel, dim3((unsigned) (some * pieces), 2 * layers), dim3(256), 0, stream,
                           (uint8_t *) keys, (uint8_t *) values, pages, page_bytes, pairs + 2 * pair,
                           (int) pieces);
        if (hipError_t s = hipGetLastError())
            return s;
        pair += some;
    }
    return hipSuccess;
}

} // namespace gq8
