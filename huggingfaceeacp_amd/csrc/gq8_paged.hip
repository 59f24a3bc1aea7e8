// gq8_paged.hip -- rows of a paged cache: the norms and rotation of a step's
// queries and keys, the append of packed rows, and the copy of whole pages.
// At a few rows all three are bound by the launch (3 to 5 us of kernel, 7 to 8 a
// call back to back).
#include "gemma_q8.h"
#include "gq8_lanes.hpp"
#include "gq8_paged.hpp"

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

template <typename Y>
__device__ inline void store_as(void *to, int64_t at, const double (&x)[4])
{
    typedef Y Y4 __attribute__((ext_vector_type(4)));
    // to fp32 first: at most 2^-24 of the value on top of the type's half step
    *(Y4 *) ((Y *) to + at) = Y4{(Y) (float) x[0], (Y) (float) x[1], (Y) (float) x[2], (Y) (float) x[3]};
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

template <typename X>
__global__ __launch_bounds__(256) void norm_rope_kernel(NormRopeArgs a, int q_type, int kv_type,
                                                        int shift, int blocks, double one_of_head)
{
    const int slots = a.heads + (a.k ? a.kv_heads : 0) + (a.v ? a.kv_heads : 0);
    const int lanes = 1 << shift, lane = threadIdx.x & (lanes - 1);
    // a block's heads are of one row: its place is found in scalar registers
    const int row = (int) ((unsigned) blockIdx.x / (unsigned) blocks);
    const int slot = (((int) blockIdx.x - row * blocks) << (8 - shift)) + (int) (threadIdx.x >> shift);
    const int position = a.positions[row];
    const int half = a.head_dim / 2;
    const int channel = lane * 4;
    const bool there = channel < half && slot < slots && position >= 0
                       && position < a.max_positions;
    const bool is_q = slot < a.heads;
    const int kv = slot - a.heads; // its k heads, then its v heads
    const bool is_k = !is_q && a.k && kv < a.kv_heads;
    // the fused row's columns: q heads, k heads, v heads
    const int column = is_q || a.k ? slot : slot + a.kv_heads;
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
        squares += u[i] * u[i] + w[i] * w[i];
    squares = sum_group<32>(squares, lanes);
    if (!there)
        return;
    if (weight) {
        const double by = rsqrt(squares * one_of_head + (double) a.epsilon);
        float g0[4], g1[4];
        load4(weight + channel, g0);
        load4(weight + half + channel, g1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u[i] *= by + by * (double) g0[i];
            w[i] *= by + by * (double) g1[i];
        }
    }
    if (is_q || is_k) {
        float cosine[4], sine[4];
        load4(a.cosines + (int64_t) position * half + channel, cosine);
        load4(a.sines + (int64_t) position * half + channel, sine);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double x0 = u[i], x1 = w[i];
            u[i] = x0 * cosine[i] - x1 * sine[i];
            w[i] = x0 * sine[i] + x1 * cosine[i];
        }
    }
    const int head = is_q ? slot : a.k && !is_k ? kv - a.kv_heads : kv;
    void *to = is_q ? a.q : is_k ? a.k : a.v;
    const int type = is_q ? q_type : kv_type;
    const int64_t at = (int64_t) row * (is_q ? a.q_stride : a.kv_stride) + (int64_t) head * a.head_dim
                       + channel;
    store4(to, type, at, u);
    store4(to, type, at + half, w);
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
    int s = 0;
    for (int base = 0; base < seq.sequences; base += 64) {
        const bool before = base + lane < seq.sequences && seq.starts[base + lane + 1] <= t;
        s += __popcll(__ballot(before));
    }
    if (s >= seq.sequences || seq.starts[s] > t)
        return; // behind the last sequence
    const int64_t place = places ? places[t] : t - (int64_t) max(seq.starts[s], 0);
    const int64_t key = (seq.cached ? max(seq.cached[s], 0) : 0) + place;
    const int64_t slot = key >> layer.page_shift;
    if (place < 0 || slot >= seq.table_width)
        return;
    const int page = seq.table[(int64_t) s * seq.table_width + slot];
    if (page < 0 || page >= layer.pages)
        return;
    const int64_t row = ((int64_t) page << layer.page_shift) + (key & ((1 << layer.page_shift) - 1));
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
