// gq8_paged_select.hip -- which pages of a long sequence a row attends: bounds of
// the keys in each page, a score from them that no key of the page passes, and the
// pages with the largest scores.
//
// Mathematics.  A page holds low_d <= k_d <= high_d for each channel of a KV head,
// so for a query q of its group
//   q.k <= sum_d max(q_d low_d, q_d high_d) = sum_d q_d (q_d < 0 ? low_d : high_d),
// a choice and a product a channel.  (Two products with sums and differences of the bounds
// are no bound: where one channel's bounds are 2^53 times the other terms, what is left of
// those cancels.)  The page's score is the largest over the group's heads.  Scores are ranked, and what
// is chosen by them has to be the same whichever order the channels are added in:
// sums are double, rounded once to fp32 for the ranking (two orders differ by some
// 1e-16 of a score, so a choice differs once in 1e8 near ties); equal scores go to
// the lower page.
#include "gemma_q8.h"
#include "gq8_lanes.hpp"
#include "gq8_numerics.hpp"
#include "gq8_paged.hpp"
#include "gq8_paged_list.hpp"
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
// 16-bit numbers in the order of 16-bit integers, two a word: of negative ones the bits
// below the sign are turned over (and back).  Minus zero lies below zero, NaNs lie past
// the infinities of their sign.
typedef short short2v __attribute__((ext_vector_type(2)));

__device__ inline word4 ordered(word4 x)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const short2v v = __builtin_bit_cast(short2v, (uint32_t) x[i]);
        x[i] ^= __builtin_bit_cast(uint32_t, v >> 15) & 0x7FFF7FFFu;
    }
    return x;
}

__device__ inline word4 lower(word4 a, word4 b)
{
#pragma unroll
    for (int i = 0; i < 4; ++i)
        a[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(short2v, (uint32_t) a[i]),
                                                                      __builtin_bit_cast(short2v, (uint32_t) b[i])));
    return a;
}

__device__ inline word4 higher(word4 a, word4 b)
{
#pragma unroll
    for (int i = 0; i < 4; ++i)
        a[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(short2v, (uint32_t) a[i]),
                                                                      __builtin_bit_cast(short2v, (uint32_t) b[i])));
    return a;
}

// The lower or the higher of a lane's and those of the lanes at distances D, 2 D .. 32.
template <int D, typename F>
__device__ inline word4 across(word4 x, F better)
{
    if constexpr (D < 64) {
        word4 other;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            other[i] = xor_lane_u32<D>(x[i]);
        return across<2 * D>(better(x, other), better);
    }
    return x;
}

// 16-byte chunks of a row that a block takes: 20 MB of ragged prompts 8.0 us a call; 32 of
// them, fewer blocks, 8.8, 8 of them, half lines, 9.5.
constexpr int kSlice = 16;

// Block (page, slice): the page is one of those that a sequence's appended rows lie in,
// found among all sequences' as tiles are; a thread reads 8 of its rows at once.  Bound by
// the chain of reads to the page (one page a sequence: 4.3 us traced, 7.2 a call) and then
// by memory: 20 MB take 8.0 us a call, 4.3 at the rate of a copy.
template <typename T>
__global__ __launch_bounds__(256) void page_bounds_kernel(PagedLayer layer, PackedSequences seq,
                                                          const int *taken, uint16_t *lows, uint16_t *highs,
                                                          int first)
{
    constexpr int ROWS = 256 / kSlice;
    __shared__ word4 least[3][kSlice], most[3][kSlice];
    const int chunk = blockIdx.y * kSlice + threadIdx.x % kSlice, group = threadIdx.x / kSlice;
    const bool there = chunk * 8 < layer.width;
    const int64_t capacity = (int64_t) seq.table_width << layer.page_shift;
    auto rows_of = [&](int s, int64_t &from) { // appended to sequence s, behind its row `from`
        const int start = min(max(seq.starts[s], 0), seq.rows);
        int count = min(max(seq.starts[s + 1], start), seq.rows) - start;
        if (taken)
            count = min(count, taken[s]);
        from = seq.cached ? max(seq.cached[s], 0) : 0;
        return (int) max(min((int64_t) count, capacity - from), (int64_t) 0);
    };
    int s, within;
    if (!find_part(first + (int) blockIdx.x, seq.sequences, [&](int i) {
            int64_t from;
            const int count = rows_of(i, from);
            return count > 0 ? (int) ((from + count - 1) >> layer.page_shift) - (int) (from >> layer.page_shift) + 1 : 0;
        }, s, within))
        return;
    int64_t from;
    const int count = rows_of(s, from);
    const int slot = (int) (from >> layer.page_shift) + within;
    const int page = seq.table[(int64_t) s * seq.table_width + slot];
    if (page < 0 || page >= layer.pages)
        return;
    const int held = (int) min((int64_t) 1 << layer.page_shift, from + count - ((int64_t) slot << layer.page_shift));
    word4 low = {0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu}, high = ~low;
    if (there) {
        const uint16_t *at = layer.keys + ((int64_t) page << layer.page_shift) * layer.width + chunk * 8;
#pragma unroll 8
        for (int r = group; r < held; r += ROWS) {
            const word4 x = ordered(*(const word4 *) (at + (int64_t) r * layer.width));
            low = lower(low, x);
            high = higher(high, x);
        }
    }
    // of the wave's rows, then of the four waves'
    low = across<kSlice>(low, [](word4 x, word4 y) { return lower(x, y); });
    high = across<kSlice>(high, [](word4 x, word4 y) { return higher(x, y); });
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (wave > 0 && lane < kSlice) {
        least[wave - 1][lane] = low;
        most[wave - 1][lane] = high;
    }
    __syncthreads();
    if (threadIdx.x >= kSlice || !there)
        return;
#pragma unroll
    for (int w = 0; w < 3; ++w) {
        low = lower(low, least[w][lane]);
        high = higher(high, most[w][lane]);
    }
    // a NaN of either sign is both bounds
    constexpr short kInfinity = __is_same(T, __bf16) ? 0x7F80 : 0x7C00;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        short2v l = __builtin_bit_cast(short2v, (uint32_t) low[i]), h = __builtin_bit_cast(short2v, (uint32_t) high[i]);
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (h[j] > kInfinity || l[j] < (short) ~kInfinity)
                l[j] = h[j] = 0x7FFF;
        low[i] = __builtin_bit_cast(uint32_t, l);
        high[i] = __builtin_bit_cast(uint32_t, h);
    }
    *(word4 *) (lows + (int64_t) page * layer.width + chunk * 8) = ordered(low);
    *(word4 *) (highs + (int64_t) page * layer.width + chunk * 8) = ordered(high);
}

// ---- scores --------------------------------------------------------------------------
// What is ranked: an order of 32-bit words.  A page that is not there is below all
// scores; one whose score is not finite or past fp32 is above them, and the pages
// that are always taken are above that.
constexpr uint32_t kAbsent = 0, kUnbounded = 0xFFFFFFFEu, kAlways = 0xFFFFFFFFu;

__device__ inline uint32_t rank_of(double sum)
{
    const float score = (float) sum + 0.f; // minus zero is zero
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

__device__ inline int64_t own_page(const SelectArgs &p, int t, int s)
{
    const int64_t cached = p.seq.cached ? max(p.seq.cached[s], 0) : 0;
    return (cached + (t - max(p.seq.starts[s], 0))) >> p.layer.page_shift;
}

// The row's pages: all up to its own.  Few of them are all taken.
__device__ inline int pages_of_row(const SelectArgs &p, int t, int s)
{
    return (int) min(own_page(p, t, s) + 1, (int64_t) p.seq.table_width);
}

// What a lane's 8 channels are as numbers: a chunk of 16-bit bounds, or of a query.
template <typename T>
__device__ inline float value_at(const word4 &x, int i)
{
    return value_of<T>(x[i / 2] >> (16 * (i % 2)) & 0xFFFFu);
}

// N sums over the lanes of a group of 2 D: at each distance a lane keeps half of them
// and hands the other half over, until it has one, whose remaining lanes are added.
template <int N, int D>
__device__ inline void sum_halving(double (&v)[N])
{
    if constexpr (D > 0 && N > 1) {
        const bool upper = threadIdx.x & D;
        double half[N / 2];
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const double keep = upper ? v[N / 2 + i] : v[i], give = upper ? v[i] : v[N / 2 + i];
            half[i] = keep + xor_lane<D>(give);
        }
        sum_halving<N / 2, D / 2>(half);
        v[0] = half[0];
    } else if constexpr (D > 0) {
        v[0] += xor_lane<D>(v[0]);
        sum_halving<N, D / 2>(v);
    }
}

template <int D>
__device__ inline uint32_t largest_rank(uint32_t v)
{
    if constexpr (D > 0) {
        v = max(v, xor_lane_u32<D>(v));
        return largest_rank<D / 2>(v);
    }
    return v;
}

// Block (row, KV head, pages): LANES lanes take a page, 8 channels each, a wave
// 64 / LANES pages a turn; the queries' channels stay in registers, HEADS heads at once.
// A page's bounds are read a line at a time and the next ones while these are summed.
// Lanes past a narrower head's channels take its first ones times zero: what is not finite
// among those is so for the page.
// Bound by the instructions that it issues: of a turn's 186 for four heads 32 double
// multiply-adds, 32 choices of their bounds, 32 conversions and 16 for bounds that are not
// finite.  16 rows' 24000 (41 MB of bounds) take 20.3 us a call, both kernels (21.2 with two
// multiply-adds in place of a choice and one); 32 heads of one KV head, where a turn does not
// make up for finding the choices, 25.0 (23.9).  (A lane a page, queries through scalar
// registers: 10.9 us for one row's 512 pages, which take 4.  Two turns at once, for one
// exchange of their sums: 1.4 us more, as are 5 waves a SIMD instead of 4 at 3 us, whose
// registers do not hold the queries.)
template <typename T, typename Q, int HEADS, int LANES>
__global__ __launch_bounds__(256) void page_score_kernel(SelectArgs p, int chunks, int turns, int first)
{
    constexpr int PAGES = 64 / LANES;
    const unsigned of = blockIdx.x / (unsigned) chunks; // rows and KV heads from row `first` on
    const int t = first + (int) (of / (unsigned) p.kv_heads), g = (int) (of % (unsigned) p.kv_heads);
    const int64_t block = (int64_t) t * p.kv_heads + g;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int base = ((int) (blockIdx.x % (unsigned) chunks) * 4 + wave) * PAGES * turns; // at most 64 pages a wave
    const int s = sequence_of_row(p.seq, t);
    if (s < 0)
        return;
    const int pages = pages_of_row(p, t, s);
    if (pages <= p.top || base >= pages)
        return;
    const int64_t own = own_page(p, t, s);
    int found = base + lane < pages ? p.seq.table[(int64_t) s * p.seq.table_width + base + lane] : -1;
    found = found < p.layer.pages ? found : -1;
    const int channel = lane % LANES * 8;
    const bool live = channel < p.head_dim;
    const uint32_t kept = live ? ~0u : 0u; // bits of a query
    const int64_t offset = g * p.head_dim + (live ? channel : 0);
    for (int heads = 0; heads < p.group; heads += HEADS) {
        double x[HEADS][8];
#pragma unroll
        for (int h = 0; h < HEADS; ++h) {
            const int head = g * p.group + min(heads + h, p.group - 1);
            const Q *q = (const Q *) p.q + (int64_t) t * p.q_stride + (int64_t) head * p.head_dim + (live ? channel : 0);
            if constexpr (sizeof(Q) == 4) {
                const word4 a = *(const word4 *) q & kept, b = *(const word4 *) (q + 4) & kept;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    x[h][i] = __uint_as_float(i < 4 ? a[i] : b[i - 4]);
            } else {
                const word4 a = *(const word4 *) q & kept;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    x[h][i] = value_at<Q>(a, i);
            }
        }
        // A negative query takes a channel's lower bound.  Which are is found once: a pair of
        // scalar registers each, past 28 of them, which is what there is, a vector register.
        constexpr int kScalar = 28 / HEADS < 8 ? 28 / HEADS : 8;
        int negative[HEADS][8 - kScalar + 1];
#pragma unroll
        for (int h = 0; h < HEADS; ++h)
#pragma unroll
            for (int i = kScalar; i < 8; ++i) {
                negative[h][i - kScalar] = __double2hiint(x[h][i]) >> 31;
                asm("" : "+v"(negative[h][i - kScalar]));
            }
        int page = __shfl(found, lane / LANES);
        int64_t at = (int64_t) max(page, 0) * p.layer.width + offset;
        word4 low = *(const word4 *) (p.lows + at), high = *(const word4 *) (p.highs + at);
#pragma unroll 1
        for (int turn = 0; turn < turns && base + turn * PAGES < pages; ++turn) {
            const bool there = page >= 0;
            const word4 this_low = low, this_high = high;
            if (turn + 1 < turns) {
                page = __shfl(found, (turn + 1) * PAGES + lane / LANES);
                at = (int64_t) max(page, 0) * p.layer.width + offset;
                low = *(const word4 *) (p.lows + at);
                high = *(const word4 *) (p.highs + at);
            }
            float odd = 0.f; // a NaN where a bound is not finite, whatever the queries are
            double sum[HEADS];
#pragma unroll
            for (int h = 0; h < HEADS; ++h)
                sum[h] = 0.0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float l = value_at<T>(this_low, i), r = value_at<T>(this_high, i);
                odd = fmaf(r, 0.f, fmaf(l, 0.f, odd));
                // as doubles their lower words are zero
                const int low_word = __double2hiint(l), high_word = __double2hiint(r);
#pragma unroll
                for (int h = 0; h < HEADS; ++h) {
                    int word = x[h][i] < 0.0 ? low_word : high_word;
                    if (i >= kScalar)
                        word = high_word ^ ((low_word ^ high_word) & negative[h][i - kScalar]);
                    sum[h] = fma(x[h][i], __hiloint2double(word, 0), sum[h]);
                }
            }
#pragma unroll
            for (int h = 0; h < HEADS; ++h)
                sum[h] += odd;
            sum_halving<HEADS, LANES / 2>(sum);
            uint32_t best = largest_rank<LANES / 2>(rank_of(sum[0]));
            const int slot = base + turn * PAGES + lane / LANES;
            if (lane % LANES == 0 && slot < pages) {
                uint32_t *rank = p.ranks + block * p.seq.table_width + slot;
                best = heads > 0 ? max(best, *rank) : best;
                const bool always = slot < p.first || slot > own - p.last;
                *rank = always ? kAlways : there ? best : kAbsent;
            }
        }
    }
}

// ---- the largest ----------------------------------------------------------------------
// Block (row, KV head).  The pages that are always taken are counted first, and the
// range of the others' ranks; then the rank of the last page to take is found a byte at
// a time from a count of the bytes, beginning where the ranks differ and ending where
// all with the bytes known so far are taken.  The pages above it and the lowest of
// those at it are written in their order.  Bound by the chain of these steps: 4.8 us for
// 512 pages, 6 for 1500.
constexpr int kHeld = 16; // ranks that a thread keeps: of 4096 pages

template <bool kKept>
__global__ __launch_bounds__(256) void page_choose_kernel(SelectArgs p, int first)
{
    __shared__ int counts[256], found[3];
    __shared__ uint32_t range[4][3];
    __shared__ int4 wave_counts[kKept ? kHeld : 1]; // of the four waves: pages above | at the rank << 16
    const int t = first + (int) (blockIdx.x / (unsigned) p.kv_heads);
    const int64_t block = (int64_t) t * p.kv_heads + blockIdx.x % (unsigned) p.kv_heads;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t *ranks = p.ranks + block * p.seq.table_width;
    uint32_t held[kKept ? kHeld : 1];
    if constexpr (kKept) // before it is known how many there are
#pragma unroll
        for (int j = 0; j < kHeld; ++j)
            if (256 * j < p.seq.table_width) {
                const int i = threadIdx.x + 256 * j;
                held[j] = ranks[min(i, p.seq.table_width - 1)];
            }
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
    auto each = [&](auto f) { // of the thread's pages
        if constexpr (kKept) {
#pragma unroll
            for (int j = 0; j < kHeld; ++j)
                if ((int) threadIdx.x + 256 * j < pages)
                    f(held[j]);
        } else {
            for (int i = threadIdx.x; i < pages; i += 256)
                f(ranks[i]);
        }
    };
    uint32_t least = kAlways, most = 0, always = 0;
    each([&](uint32_t x) {
        always += x == kAlways;
        least = min(least, x);
        most = max(most, x == kAlways ? 0 : x);
    });
    least = ~largest_rank<32>(~least);
    most = largest_rank<32>(most);
    always = (uint32_t) sum_lanes<32>((int) always);
    if (lane == 0) {
        range[wave][0] = least;
        range[wave][1] = most;
        range[wave][2] = always;
    }
    __syncthreads();
    always = 0;
    for (int w = 0; w < 4; ++w) {
        least = min(least, range[w][0]);
        most = max(most, range[w][1]);
        always += range[w][2];
    }
    // Ranks at or above `rank` in their bits `known` are taken, of those that equal it there
    // the `wanted` lowest pages.  There is a page that is not always taken.
    int wanted = p.top - (int) always, shift = 32 - __clz(most ^ least);
    uint32_t known = shift < 32 ? ~0u << shift : 0, rank = most & known;
    if (wanted == 0) {
        known = ~0u;
        rank = kAlways;
        wanted = (int) always;
        shift = 0;
    }
#pragma unroll 1
    while (shift > 0) {
        const int from = max(shift - 8, 0);
        counts[threadIdx.x] = 0;
        __syncthreads();
        each([&](uint32_t x) {
            if ((x & known) == rank && x != kAlways)
                atomicAdd(&counts[x >> from & ((1u << (shift - from)) - 1)], 1);
        });
        __syncthreads();
        if (wave == 0) { // lane l: bytes 255 - 4 l and the three below it
            int mine[4], sum = 0;
            for (int i = 0; i < 4; ++i)
                sum += mine[i] = counts[255 - 4 * lane - i];
            const int upto = sum_upto(sum);
            int before = upto - sum;
            if (before < wanted && upto >= wanted)
                for (int i = 0; i < 4; ++i) {
                    if (before + mine[i] >= wanted) {
                        found[0] = 255 - 4 * lane - i;
                        found[1] = wanted - before;
                        found[2] = mine[i];
                        break;
                    }
                    before += mine[i];
                }
        }
        __syncthreads();
        rank |= (uint32_t) found[0] << from;
        known = ~0u << from;
        wanted = found[1];
        shift = found[1] == found[2] ? 0 : from;
    }
    // Where a page goes: behind those above the rank and the wanted ones at it before it.
    const uint64_t below = (1ull << lane) - 1;
    auto group_of = [&](int i, uint32_t x, bool &more, bool &equal) { // -> the wave's counts before the lane
        const bool taken = x == kAlways && rank != kAlways;
        x &= known;
        more = i < pages && (taken || x > rank);
        equal = i < pages && !more && x == rank;
        const uint64_t mores = __ballot(more), equals = __ballot(equal);
        if (lane == 0)
            ((int *) &wave_counts[kKept ? i / 256 : 0])[wave] = __popcll(mores) | __popcll(equals) << 16;
        return __popcll(mores & below) | __popcll(equals & below) << 16;
    };
    int above = 0, at = 0; // before these 256 pages
    auto write = [&](int i, int inside, bool more, bool equal) {
        const int4 c = wave_counts[kKept ? i / 256 : 0];
        inside += (wave > 0 ? c.x : 0) + (wave > 1 ? c.y : 0) + (wave > 2 ? c.z : 0);
        const int to = place_in_list(more, equal, above + (inside & 0xFFFF), at + (inside >> 16), wanted, p.top);
        if (to >= 0)
            out[to] = i;
        const int sum = c.x + c.y + c.z + c.w;
        above += sum & 0xFFFF;
        at += sum >> 16;
    };
    if constexpr (kKept) {
        int inside[kHeld];
        uint32_t mores = 0, equals = 0;
#pragma unroll
        for (int j = 0; j < kHeld; ++j)
            if (256 * j < pages) {
                bool more, equal;
                inside[j] = group_of(256 * j + threadIdx.x, held[j], more, equal);
                mores |= (uint32_t) more << j;
                equals |= (uint32_t) equal << j;
            }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kHeld; ++j)
            if (256 * j < pages)
                write(256 * j + threadIdx.x, inside[j], mores >> j & 1, equals >> j & 1);
    } else {
        for (int base = 0; base < pages; base += 256) {
            const int i = base + threadIdx.x;
            bool more, equal;
            const uint32_t x = i < pages ? ranks[i] : 0;
            __syncthreads();
            const int inside = group_of(i, x, more, equal);
            __syncthreads();
            write(i, inside, more, equal);
        }
    }
}

// Pages a block takes in `turns` turns of its waves.
int lanes_of(int head_dim)
{
    return head_dim <= 64 ? 8 : head_dim <= 128 ? 16 : 32;
}

template <typename T, typename Q, int HEADS>
void launch_scores(const SelectArgs &p, int chunks, int turns, int first, unsigned blocks, hipStream_t stream)
{
    auto launch = [&](auto *kernel) {
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, stream, p, chunks, turns, first);
    };
    switch (lanes_of(p.head_dim)) {
    case 8: launch(page_score_kernel<T, Q, HEADS, 8>); break;
    case 16: launch(page_score_kernel<T, Q, HEADS, 16>); break;
    default: launch(page_score_kernel<T, Q, HEADS, 32>); break;
    }
}

template <typename T, typename Q>
void launch_scores(const SelectArgs &p, int chunks, int turns, int first, unsigned blocks, hipStream_t stream)
{
    // the heads of a group whose sums a lane holds at once
    if (p.group == 1)
        launch_scores<T, Q, 1>(p, chunks, turns, first, blocks, stream);
    else if (p.group == 2)
        launch_scores<T, Q, 2>(p, chunks, turns, first, blocks, stream);
    else if (p.group <= 4)
        launch_scores<T, Q, 4>(p, chunks, turns, first, blocks, stream);
    else
        launch_scores<T, Q, 8>(p, chunks, turns, first, blocks, stream);
}

} // namespace

hipError_t launch_page_bounds(const PagedLayer &layer, const PackedSequences &seq, const int *taken,
                              uint16_t *lows, uint16_t *highs, int type, hipStream_t stream)
{
    const int64_t slices = (layer.width / 8 + kSlice - 1) / kSlice;
    if (seq.rows <= 0 || seq.sequences <= 0 || layer.width % 8 != 0 || slices > 65535)
        return hipErrorInvalidValue;
    // a sequence's rows lie in as many pages as they fill and up to two more (one row: in one)
    const int64_t page_rows = 1 << layer.page_shift, owners = std::min(seq.sequences, seq.rows);
    const int64_t blocks = (seq.rows + owners * (2 * page_rows - 2)) / page_rows;
    if (blocks > INT32_MAX)
        return hipErrorInvalidValue;
    for (int64_t first = 0; first < blocks;) {
        const int64_t some = std::min(blocks - first, kMostBlocks / slices);
        const dim3 grid((unsigned) some, (unsigned) slices);
        if (type == GQ8_DTYPE_F16)
            hipLaunchKernelGGL(page_bounds_kernel<_Float16>, grid, dim3(256), 0, stream, layer, seq, taken, lows,
                               highs, (int) first);
        else
            hipLaunchKernelGGL(page_bounds_kernel<__bf16>, grid, dim3(256), 0, stream, layer, seq, taken, lows,
                               highs, (int) first);
        if (hipError_t s = hipGetLastError())
            return s;
        first += some;
    }
    return hipSuccess;
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
    // Turns of a block's waves: as many as leave 2048 blocks, since a block finds its row
    // and turns its queries into doubles once; at most 64 pages a wave.  (16 rows behind
    // 24000, both kernels: 512 blocks 28.3 us, 1024 21.7, 2048 21.9, 4096 29.8; fewer rows
    // want the blocks.)
    const int64_t a_turn = 4 * 64 / lanes_of(a.head_dim);
    const int64_t all_turns = all * ((a.seq.table_width + a_turn - 1) / a_turn);
    const int turns = (int) std::clamp<int64_t>(all_turns / 2048, 1, lanes_of(a.head_dim));
    const int64_t chunks = (a.seq.table_width + a_turn * turns - 1) / (a_turn * turns);
    const int64_t most_rows = kMostBlocks / (chunks * a.kv_heads); // a launch
    if (most_rows < 1)
        return hipErrorInvalidValue;
    if (a.seq.table_width > a.top) // else every row takes all of its pages
        for (int64_t first = 0; first < a.seq.rows; first += most_rows) {
            const unsigned blocks = (unsigned) (std::min(a.seq.rows - first, most_rows) * a.kv_heads * chunks);
            const bool bf16 = cache_type == GQ8_DTYPE_BF16;
            if (q_type == GQ8_DTYPE_F32 && bf16)
                launch_scores<__bf16, float>(p, (int) chunks, turns, (int) first, blocks, stream);
            else if (q_type == GQ8_DTYPE_F32)
                launch_scores<_Float16, float>(p, (int) chunks, turns, (int) first, blocks, stream);
            else if (bf16)
                launch_scores<__bf16, __bf16>(p, (int) chunks, turns, (int) first, blocks, stream);
            else
                launch_scores<_Float16, _Float16>(p, (int) chunks, turns, (int) first, blocks, stream);
            if (hipError_t s = hipGetLastError())
                return s;
        }
    const int64_t each = kMostBlocks / a.kv_heads;
    for (int64_t first = 0; first < a.seq.rows; first += each) {
        const dim3 grid((unsigned) (std::min(a.seq.rows - first, each) * a.kv_heads));
        if (a.seq.table_width <= 256 * kHeld)
            hipLaunchKernelGGL(page_choose_kernel<true>, grid, dim3(256), 0, stream, p, (int) first);
        else
            hipLaunchKernelGGL(page_choose_kernel<false>, grid, dim3(256), 0, stream, p, (int) first);
        if (hipError_t s = hipGetLastError())
            return s;
    }
    return hipSuccess;
}

} // namespace gq8
