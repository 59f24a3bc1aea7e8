// gq8_paged_select.hip -- which pages of a long sequence a row attends: bounds of
// the keys in each page, a score from them that no key of the page passes, and the
// pages with the largest scores.
//
// Mathematics.  A page holds low_d <= k_d <= high_d for each channel of a KV head,
// so for a query q of its group
//   q.k <= sum_d max(q_d low_d, q_d high_d) = 1/2 sum_d (q_d (high_d + low_d) + |q_d| (high_d - low_d)),
// two products a channel, of which one takes the absolute value for nothing.  The
// page's score is the largest over the group's heads.  Scores are ranked, and what
// is chosen by them has to be the same whichever order the channels are added in:
// sums are double, rounded once to fp32 for the ranking (two orders differ by some
// 1e-16 of a score, so a choice differs once in 1e8 near ties); equal scores go to
// the lower page.
#include "gemma_q8.h"
#include "gq8_lanes.hpp"
#include "gq8_paged.hpp"
#include "gq8_paged_rows.hpp"

#include <algorithm>

namespace gq8 {
namespace {

typedef uint32_t word4 __attribute__((ext_vector_type(4)));

constexpr int64_t kMostBlocks = (1 << 24) - 1; // blocks of 256 threads a launch

template <typename T>
__device__ inline float value_of(uint32_t bits16)
{
    if constexpr (__is_same(T, __bf16))
        return __uint_as_float(bits16 << 16);
    else
        return (float) __builtin_bit_cast(_Float16, (uint16_t) bits16);
}

// ---- bounds ------------------------------------------------------------------------
// Less (or greater) than the bound, or a NaN, which stays.
__device__ inline float lower(float bound, float x)
{
    return x < bound || x != x ? x : bound;
}

__device__ inline float higher(float bound, float x)
{
    return x > bound || x != x ? x : bound;
}

constexpr int kSlice = 32; // 16-byte chunks of a row that a block takes (256 channels)

// Block (packed rows, slice): each page that one of its rows is the first appended
// row of is read whole, as far as the sequence's rows go, 8 rows at once.
template <typename T>
__global__ __launch_bounds__(256) void page_bounds_kernel(PagedLayer layer, PackedSequences seq,
                                                          const int *taken, uint16_t *lows, uint16_t *highs,
                                                          int each)
{
    constexpr int ROWS = 256 / kSlice;
    __shared__ float least[ROWS - 1][kSlice][8], most[ROWS - 1][kSlice][8];
    const int chunk = blockIdx.y * kSlice + threadIdx.x % kSlice, group = threadIdx.x / kSlice;
    const bool there = chunk * 8 < layer.width;
    const int64_t first = (int64_t) blockIdx.x * each;
    for (int t = (int) first; t < min(first + each, (int64_t) seq.rows); ++t) {
        const int s = sequence_of_row(seq, t);
        if (s < 0)
            continue;
        const int start = max(seq.starts[s], 0);
        int count = min(seq.starts[s + 1], seq.rows) - start;
        if (taken)
            count = min(count, taken[s]);
        const int64_t cached = seq.cached ? max(seq.cached[s], 0) : 0;
        const int64_t key = cached + (t - start);
        const int mask = (1 << layer.page_shift) - 1;
        if (t - start >= count || (t != start && (key & mask) != 0))
            continue;
        const int64_t row = pool_row(layer, seq, s, key);
        if (row < 0)
            continue;
        const int64_t page = row >> layer.page_shift;
        const int held = (int) min((int64_t) mask + 1, cached + count - (key & ~(int64_t) mask));
        float low[8], high[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            low[i] = INFINITY;
            high[i] = -INFINITY;
        }
        if (there) {
            const uint16_t *from = layer.keys + (page << layer.page_shift) * layer.width + chunk * 8;
#pragma unroll 4
            for (int r = group; r < held; r += ROWS) {
                const word4 x = *(const word4 *) (from + (int64_t) r * layer.width);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float v = value_of<T>(x[i / 2] >> (16 * (i % 2)) & 0xFFFFu);
                    low[i] = lower(low[i], v);
                    high[i] = higher(high[i], v);
                }
            }
        }
        __syncthreads(); // the last page's have been read
        if (group > 0)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                least[group - 1][threadIdx.x % kSlice][i] = low[i];
                most[group - 1][threadIdx.x % kSlice][i] = high[i];
            }
        __syncthreads();
        if (group > 0 || !there)
            continue;
        for (int r = 0; r < ROWS - 1; ++r)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                low[i] = lower(low[i], least[r][threadIdx.x][i]);
                high[i] = higher(high[i], most[r][threadIdx.x][i]);
            }
        typedef T T8 __attribute__((ext_vector_type(8)));
        T8 l, h;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            l[i] = (T) low[i];
            h[i] = (T) high[i];
        }
        *(T8 *) (lows + page * layer.width + chunk * 8) = l;
        *(T8 *) (highs + page * layer.width + chunk * 8) = h;
    }
}

// ---- scores --------------------------------------------------------------------------
// What is ranked: an order of 32-bit words.  A page that is not there is below all
// scores; one whose score is not finite or past fp32 is above them, and the pages
// that are always taken are above that.
constexpr uint32_t kAbsent = 0, kUnbounded = 0xFFFFFFFEu, kAlways = 0xFFFFFFFFu;

__device__ inline uint32_t rank_of(double twice)
{
    const float score = (float) (0.5 * twice) + 0.f; // minus zero is zero
    if (!(score < INFINITY))
        return kUnbounded;
    const uint32_t bits = __float_as_uint(score);
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

struct SelectArgs {
    PagedLayer layer;
    PackedSequences seq;
    const uint16_t *lows, *highs;
    const void *q;
    int q_stride, kv_heads, head_dim, group, first, last, top;
    uint32_t *ranks; // [rows, kv_heads, table_width]
    int *pages;      // [rows, kv_heads, top]
};

// The row's pages: all up to its own.  Few of them are all taken.
__device__ inline int pages_of_row(const SelectArgs &p, int t, int s)
{
    const int64_t cached = p.seq.cached ? max(p.seq.cached[s], 0) : 0;
    const int64_t own = (cached + (t - max(p.seq.starts[s], 0))) >> p.layer.page_shift;
    return (int) min(own + 1, (int64_t) p.seq.table_width);
}

template <typename Q>
__device__ inline double query_value(const Q *q, int i)
{
    return (double) (float) q[i];
}

// Block (row, KV head, 64 pages): a lane takes a page, a wave a quarter of the
// channels, so that a line of a page's bounds is read by one wave, at once; queries
// are the same for all lanes and come through scalar registers.
template <typename T, typename Q, int HEADS>
__global__ __launch_bounds__(256) void page_score_kernel(SelectArgs p, int chunks, int64_t first)
{
    __shared__ double parts[3][HEADS][64];
    const int64_t block = first + blockIdx.x / (unsigned) chunks;
    const int base = (int) (blockIdx.x % (unsigned) chunks) * 64;
    const int t = (int) (block / p.kv_heads), g = (int) (block % p.kv_heads);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int s = sequence_of_row(p.seq, t);
    if (s < 0)
        return;
    const int pages = pages_of_row(p, t, s);
    if (pages <= p.top || base >= pages)
        return;
    const int slot = base + lane;
    int page = slot < pages ? p.seq.table[(int64_t) s * p.seq.table_width + slot] : -1;
    const bool there = page >= 0 && page < p.layer.pages;
    const int64_t at = (int64_t) (there ? page : 0) * p.layer.width + g * p.head_dim;
    const int all = p.head_dim / 8, quarter = (all + 3) / 4;
    const int begin = wave * quarter, end = min(all, begin + quarter);
    uint32_t best = 0;
    for (int block_of_heads = 0; block_of_heads < p.group; block_of_heads += HEADS) {
        double sum[HEADS];
#pragma unroll
        for (int h = 0; h < HEADS; ++h)
            sum[h] = 0.0;
#pragma unroll 2
        for (int c = begin; c < end; ++c) {
            const word4 l = *(const word4 *) (p.lows + at + c * 8), h4 = *(const word4 *) (p.highs + at + c * 8);
            double both[8], apart[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const double low = value_of<T>(l[i / 2] >> (16 * (i % 2)) & 0xFFFFu);
                const double high = value_of<T>(h4[i / 2] >> (16 * (i % 2)) & 0xFFFFu);
                both[i] = high + low;
                apart[i] = high - low;
            }
#pragma unroll
            for (int h = 0; h < HEADS; ++h) {
                const int head = g * p.group + min(block_of_heads + h, p.group - 1);
                const Q *q = (const Q *) p.q + (int64_t) t * p.q_stride + (int64_t) head * p.head_dim + c * 8;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const double x = query_value(q, i);
                    sum[h] = fma(x, both[i], sum[h]);
                    sum[h] = fma(fabs(x), apart[i], sum[h]);
                }
            }
        }
        __syncthreads(); // the last heads' have been read
        if (wave > 0)
#pragma unroll
            for (int h = 0; h < HEADS; ++h)
                parts[wave - 1][h][lane] = sum[h];
        __syncthreads();
        if (wave == 0)
#pragma unroll
            for (int h = 0; h < HEADS; ++h)
                best = max(best, rank_of(sum[h] + parts[0][h][lane] + parts[1][h][lane] + parts[2][h][lane]));
    }
    if (wave != 0 || slot >= pages)
        return;
    const int64_t own = ((p.seq.cached ? max(p.seq.cached[s], 0) : 0) + (int64_t) (t - max(p.seq.starts[s], 0)))
                        >> p.layer.page_shift;
    const bool always = slot < p.first || slot > own - p.last;
    p.ranks[block * p.seq.table_width + slot] = always ? kAlways : there ? best : kAbsent;
}

// ---- the largest ----------------------------------------------------------------------
// Block (row, KV head): the rank of the top-th page is found a byte at a time from
// a count of the bytes, then the pages above it and the lowest of those at it are
// written in their order.
__global__ __launch_bounds__(256) void page_choose_kernel(SelectArgs p, int64_t first)
{
    __shared__ int counts[256], wave_counts[4][2], found[2];
    const int64_t block = first + blockIdx.x;
    const int t = (int) (block / p.kv_heads);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int s = sequence_of_row(p.seq, t);
    if (s < 0)
        return;
    const int pages = pages_of_row(p, t, s);
    int *out = p.pages + block * p.top;
    if (pages <= p.top) {
        for (int i = threadIdx.x; i < p.top; i += 256)
            out[i] = i < pages ? i : -1;
        return;
    }
    const uint32_t *ranks = p.ranks + block * p.seq.table_width;
    uint32_t rank = 0, known = 0; // of the top-th: the bytes known so far
    int wanted = p.top;           // the how manieth of those that begin with them
#pragma unroll 1
    for (int shift = 24; shift >= 0; shift -= 8) {
        counts[threadIdx.x] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < pages; i += 256)
            if ((ranks[i] & known) == rank)
                atomicAdd(&counts[ranks[i] >> shift & 255], 1);
        __syncthreads();
        if (wave == 0) { // lane l: bytes 255 - 4 l and the three below it
            int mine[4], sum = 0;
            for (int i = 0; i < 4; ++i)
                sum += mine[i] = counts[255 - 4 * lane - i];
            int upto = sum;
            for (int d = 1; d < 64; d <<= 1) {
                const int other = __shfl_up(upto, d);
                upto += lane >= d ? other : 0;
            }
            int before = upto - sum;
            if (before < wanted && upto >= wanted)
                for (int i = 0; i < 4; ++i) {
                    if (before + mine[i] >= wanted) {
                        found[0] = 255 - 4 * lane - i;
                        found[1] = wanted - before;
                        break;
                    }
                    before += mine[i];
                }
        }
        __syncthreads();
        rank |= (uint32_t) found[0] << shift;
        known |= 255u << shift;
        wanted = found[1];
    }
    int above = 0, at = 0; // written, and pages at the rank seen
    for (int base = 0; base < pages; base += 256) {
        const int i = base + threadIdx.x;
        const uint32_t x = i < pages ? ranks[i] : 0;
        const bool more = i < pages && x > rank, equal = i < pages && x == rank;
        const uint64_t mores = __ballot(more), equals = __ballot(equal), below = (1ull << lane) - 1;
        __syncthreads();
        if (lane == 0) {
            wave_counts[wave][0] = __popcll(mores);
            wave_counts[wave][1] = __popcll(equals);
        }
        __syncthreads();
        int before_more = above, before_equal = at;
        for (int w = 0; w < 4; ++w) {
            before_more += w < wave ? wave_counts[w][0] : 0;
            before_equal += w < wave ? wave_counts[w][1] : 0;
            above += wave_counts[w][0];
            at += wave_counts[w][1];
        }
        before_more += __popcll(mores & below);
        before_equal += __popcll(equals & below);
        if (more || (equal && before_equal < wanted))
            out[before_more + min(before_equal, wanted)] = i;
    }
}

template <typename T, typename Q>
void launch_scores(const SelectArgs &p, int chunks, int64_t first, unsigned blocks, hipStream_t stream)
{
    auto launch = [&](auto *kernel) {
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, stream, p, chunks, first);
    };
    // the heads of a group whose sums a lane holds at once
    if (p.group == 1)
        launch(page_score_kernel<T, Q, 1>);
    else if (p.group == 2)
        launch(page_score_kernel<T, Q, 2>);
    else if (p.group <= 4)
        launch(page_score_kernel<T, Q, 4>);
    else
        launch(page_score_kernel<T, Q, 8>);
}

} // namespace

hipError_t launch_page_bounds(const PagedLayer &layer, const PackedSequences &seq, const int *taken,
                              uint16_t *lows, uint16_t *highs, int type, hipStream_t stream)
{
    const int64_t slices = (layer.width / 8 + kSlice - 1) / kSlice;
    if (seq.rows <= 0 || seq.sequences <= 0 || layer.width % 8 != 0 || slices > 65535)
        return hipErrorInvalidValue;
    // most rows begin no page: up to a page of them a block, in 2048 blocks or more
    const int64_t each = std::min<int64_t>(1 << layer.page_shift, (seq.rows + 2047) / 2048);
    const int64_t blocks = (seq.rows + each - 1) / each;
    if (blocks * slices > kMostBlocks)
        return hipErrorInvalidValue;
    const dim3 grid((unsigned) blocks, (unsigned) slices);
    if (type == GQ8_DTYPE_F16)
        hipLaunchKernelGGL(page_bounds_kernel<_Float16>, grid, dim3(256), 0, stream, layer, seq, taken, lows,
                           highs, (int) each);
    else
        hipLaunchKernelGGL(page_bounds_kernel<__bf16>, grid, dim3(256), 0, stream, layer, seq, taken, lows,
                           highs, (int) each);
    return hipGetLastError();
}

hipError_t launch_page_select(const PageSelectArgs &a, int cache_type, int q_type, hipStream_t stream)
{
    const int group = a.kv_heads > 0 ? a.heads / a.kv_heads : 0;
    if (a.seq.sequences <= 0 || a.seq.rows <= 0 || group <= 0 || a.heads != group * a.kv_heads
        || a.head_dim <= 0 || a.head_dim > kPagedMaxHeadDim || a.head_dim % 8 != 0
        || a.layer.width != a.kv_heads * a.head_dim || a.seq.table_width <= 0)
        return hipErrorInvalidValue;
    SelectArgs p{a.layer, a.seq, a.lows, a.highs, a.q, a.q_stride, a.kv_heads, a.head_dim, group,
                 a.first, a.last, a.top, a.ranks, a.pages};
    const int64_t all = (int64_t) a.seq.rows * a.kv_heads;
    const int64_t chunks = (a.seq.table_width + 63) / 64;
    if (chunks > kMostBlocks)
        return hipErrorInvalidValue;
    if (a.seq.table_width > a.top) // else every row takes all of its pages
        for (int64_t first = 0; first < all;) {
            const int64_t some = std::min(all - first, kMostBlocks / chunks);
            const unsigned blocks = (unsigned) (some * chunks);
            const bool bf16 = cache_type == GQ8_DTYPE_BF16;
            if (q_type == GQ8_DTYPE_F32 && bf16)
                launch_scores<__bf16, float>(p, (int) chunks, first, blocks, stream);
            else if (q_type == GQ8_DTYPE_F32)
                launch_scores<_Float16, float>(p, (int) chunks, first, blocks, stream);
            else if (bf16)
                launch_scores<__bf16, __bf16>(p, (int) chunks, first, blocks, stream);
            else
                launch_scores<_Float16, _Float16>(p, (int) chunks, first, blocks, stream);
            if (hipError_t s = hipGetLastError())
                return s;
            first += some;
        }
    for (int64_t first = 0; first < all; first += kMostBlocks) {
        hipLaunchKernelGGL(page_choose_kernel, dim3((unsigned) std::min(all - first, kMostBlocks)), dim3(256), 0,
                           stream, p, first);
        if (hipError_t s = hipGetLastError())
            return s;
    }
    return hipSuccess;
}

} // namespace gq8
