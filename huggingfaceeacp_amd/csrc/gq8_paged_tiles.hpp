// gq8_paged_tiles.hpp -- what the attentions of a paged cache do alike: the matrix
// products of a tile of 32 (row, head) pairs with keys and values, the running
// reference of a row's scores, and the joining of sums about different references.
// gq8_paged_attention.hip says what the arithmetic is and why.
#pragma once

#include "gq8_lanes.hpp"

#include <hip/hip_runtime.h>

#include <cstdint>

namespace gq8 {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));
typedef uint32_t word4 __attribute__((ext_vector_type(4)));

constexpr float kLow = -3.0e38f;   // a row's reference before its first key
constexpr float kMargin = 4.f;     // how far (in powers of two) a score may pass it
constexpr float kFar = 65536.f;    // 2^-24 of it stays below a hundredth of a power
constexpr float kLeast = 1.0e-30f; // of the factor on a score
constexpr float kOffset = 10.f;    // fp16 weights are held times 2^10 (2^14 at most)
constexpr float kLog2e = 1.44269504088896340736f;

__device__ const word4 kZeroChunk = {0, 0, 0, 0};

__device__ inline int uniform(int v)
{
    return __builtin_amdgcn_readfirstlane(v);
}

__device__ inline uint64_t uniform64(uint64_t v)
{
    return ((uint64_t) (uint32_t) uniform((int) (v >> 32)) << 32) | (uint32_t) uniform((int) v);
}

// ---- keys and values in LDS -------------------------------------------------------
// Row j of a tile's 64 rows of HD values, in 16-byte chunks; chunk c of row r
// lies at c ^ swizzle(r), so that over all 64 banks (256 bytes) 16 rows' same
// chunk meet no two in a bank, nor do 4 rows' same four chunks.
template <int HD>
__device__ inline int swizzle(int row)
{
    return HD >= 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : ((row & 2) << 1) | ((row >> 2) & 3);
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

// Rows that follow each other, 16 of one wave: one address does for the wave, and the
// lanes' offsets from it, 512 / HD rows an instruction.
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

} // namespace
} // namespace gq8
