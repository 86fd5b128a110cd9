// A row of logits counted by value, as hyp_sample_batch and hyp_verify_batch do it (sample_batch.hip has the why).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "hyperion_hip.h"
#include "wave.h"

namespace hyperion::hip::sampling {

#define HYP_INLINE __attribute__((always_inline))

constexpr uint32_t kThreads = 1024;
constexpr uint32_t kWaves = kThreads / 64u;
constexpr uint32_t kPer = 9;                          // bins of a thread (odd: no bank conflicts)
constexpr uint32_t kLow = (127u - 25u) << 7;          // bits of 2^-25
constexpr uint32_t kFine = 32u << 7;                  // values a sign has in [2^-25, 2^7)
constexpr uint32_t kAbove = 0u;                       // the bin of larger values
constexpr uint32_t kCentre = kFine + 1u;
constexpr uint32_t kBelow = 2u * kFine + 2u;
constexpr uint32_t kBins = kBelow + 1u;
// Where a bin's count stands: first the fine values by their bits less those of 2^-25, positive ones, then
// negative ones (so that the place follows from the bits in few steps), then the other three.
constexpr uint32_t kCentreAt = 2u * kFine;
constexpr uint32_t kAboveAt = kCentreAt + 1u;
constexpr uint32_t kBelowAt = kCentreAt + 2u;
static_assert(kBelowAt == kBelow, "the places behind the last bin are their own");
__device__ __forceinline__ uint32_t count_at(uint32_t bin) {
    const uint32_t at = bin <= kFine ? kFine - bin : (bin < kBelow ? bin - 2u : bin);
    return bin == kAbove ? kAboveAt : (bin == kCentre ? kCentreAt : at);
}
constexpr uint32_t kWindow = 8192;                    // values of one window of the long way
constexpr uint32_t kWindows = 65536u / kWindow;
constexpr uint32_t kMaxVocab = 1u << 23;
static_assert(kBins <= kThreads * kPer, "a thread's bins");

struct RowParams {
    double by_t;     // 1 / the weights' temperature (1 for a greedy row)
    double top_p, min_p, u;
    uint32_t top_k;  // 0: off
    bool greedy;
};

__device__ __forceinline__ RowParams row_params(const HypSamplingConfig& config, float u) {
    const HypSamplingConfig c = config;   // (one load)
    RowParams r;
    r.greedy = !(c.temperature > 0.0f);
    r.by_t = r.greedy ? 1.0 : 1.0 / static_cast<double>(c.temperature);
    r.top_p = c.top_p > 0.0f && c.top_p < 1.0f ? static_cast<double>(c.top_p) : 0.0;
    r.min_p = c.min_p > 0.0f ? static_cast<double>(c.min_p) : 0.0;
    r.top_k = c.top_k > 0 ? static_cast<uint32_t>(c.top_k) : 0u;
    r.u = u > 0.0f ? static_cast<double>(fminf(u, 0x1.fffffep-1f)) : 0.0;
    return r;
}

// A value's bits with -0 as +0, and its place in the descending order of all 65536.
__device__ __forceinline__ uint32_t plain_bits(uint32_t b) { return b == 0x8000u ? 0u : b; }
__device__ __forceinline__ uint32_t place_of(uint32_t b) { return 0xFFFFu - ((b & 0x8000u) != 0u ? (~b & 0xFFFFu) : (b | 0x8000u)); }
__device__ __forceinline__ uint32_t bits_at(uint32_t place) {
    const uint32_t up = 0xFFFFu - place;
    return (up & 0x8000u) != 0u ? (up & 0x7FFFu) : (~up & 0xFFFFu);
}
__device__ __forceinline__ bool finite_bits(uint32_t b) { return (b & 0x7F80u) != 0x7F80u; }
__device__ __forceinline__ double value_of(uint32_t b) { return static_cast<double>(__uint_as_float(b << 16)); }

struct alignas(2) Eight {
    uint16_t v[8];
};

// f(index, bits) of the tokens [begin, end) of a row, in 16-byte loads (a row's alignment is its
// values').
template <typename F>
__device__ __forceinline__ void for_tokens(const uint16_t* row, uint32_t begin, uint32_t end, uint32_t lane, uint32_t lanes,
                                           F&& f) {
    uint32_t i = begin + 8u * lane;
#pragma unroll 4
    for (; i + 8u <= end; i += 8u * lanes) {
        Eight e;
        __builtin_memcpy(&e, row + i, 16);
#pragma unroll
        for (uint32_t k = 0; k < 8u; ++k) f(i + k, static_cast<uint32_t>(e.v[k]));
    }
    for (uint32_t k = i; k < end && k < i + 8u; ++k) f(k, static_cast<uint32_t>(row[k]));
}

struct Block {
    double d[kWaves];
    uint32_t u[kWaves];
};

// e^x of an x <= 0: 2^n e^r with r = x - n ln 2 in [-ln 2 / 2, ln 2 / 2], the series to r^13 (the rest is below 2^-57).
// Without the library's branches nine of them run side by side.
__device__ __forceinline__ double exp_below(double x) {
    x = fmin(fmax(x, -1100.0), 0.0);
    const double n = __builtin_rint(x * 0x1.71547652b82fep+0);
    const double r = __builtin_fma(n, -0x1.abc9e3b39803fp-56, __builtin_fma(n, -0x1.62e42fefa39efp-1, x));
    double y = 1.0 / 6227020800.0;
    constexpr double kSeries[] = {1.0 / 479001600.0, 1.0 / 39916800.0, 1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0,
                                  1.0 / 5040.0,      1.0 / 720.0,      1.0 / 120.0,     1.0 / 24.0,     1.0 / 6.0,
                                  0.5,               1.0,              1.0};
#pragma unroll
    for (const double c : kSeries) y = __builtin_fma(y, r, c);
    return __builtin_amdgcn_ldexp(y, static_cast<int>(n));
}

struct alignas(16) RowLds {
    uint32_t count[kThreads * kPer];
    Block block;
    uint32_t infinite;             // +inf tokens
    uint32_t centre_lo, centre_hi; // least and largest place of the values next to 0
    uint32_t below;                // bits of the largest value below the fine ones (their least)
    uint32_t drawn, number;        // the drawn value's bits, the token's number among those
    uint32_t bin;                  // and its bin, kBins where that is none of the first way
    double kept;                   // the kept tokens' mass
    uint32_t keep, rank;           // how many tokens the filters keep, the drawn one's rank
    uint32_t lead[kWaves];         // a wave's first bin with a token
};

// s.count, s.infinite, s.centre_lo, s.centre_hi and s.below of the tokens [begin, end) of a row. (A call has a barrier at its
// end.) kAhead > 0: the 16-byte loads of a thread, at most so many for all of [begin, end), are all on their way before the
// counts are cleared.
template <uint32_t kAhead>
__device__ __forceinline__ void count_values(const uint16_t* row, uint32_t begin, uint32_t end, RowLds& s) {
    const uint32_t tid = threadIdx.x;
    uint32_t i = begin + 8u * tid;
    uint32_t ahead[kAhead != 0u ? kAhead : 1u][4];
    if constexpr (kAhead != 0u) {
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k)
            if (i + k * 8u * kThreads + 8u <= end) __builtin_memcpy(ahead[k], row + i + k * 8u * kThreads, 16);
        __builtin_amdgcn_sched_barrier(0);
    }
    for (uint32_t i = tid; i < kThreads * kPer; i += kThreads) s.count[i] = 0u;
    if (tid == 0u) {
        s.infinite = 0u;
        s.centre_lo = 0xFFFFFFFFu;
        s.centre_hi = 0u;
        s.below = 0xFFFFFFFFu;
    }
    __syncthreads();
    // What is no fine value, most of a row maybe (masked tokens, zeros), is counted in registers: of 576 rows of 262144 60 % at
    // the type's lowest value, at 0 or at +inf took a verification 367, 1900 and 390 us through LDS, and take 123, 198 and 195.
    uint32_t below = 0u, below_bits = 0xFFFFFFFFu;
    uint32_t centre = 0u, centre_lo = 0xFFFFFFFFu, centre_hi = 0u, above = 0u, infinite = 0u;
    // The bits less kLow, in 16 bits: a fine value has 0 in bits 12 to 14, its sign in bit 15.
    const auto usual = [&](uint32_t b) HYP_INLINE {   // a fine value, one of -2^7 to the lowest, -inf; false: another
        const uint32_t t = b - kLow;
        const bool fine = (t & 0x7000u) == 0u;
        if (fine) atomicAdd(&s.count[(t & 0xFFFu) | ((t >> 3) & 0x1000u)], 1u);
        const bool low = b - 0xC300u < 0xFF80u - 0xC300u;
        below += low ? 1u : 0u;
        below_bits = min(below_bits, low ? b : 0xFFFFFFFFu);
        return fine || b - 0xC300u <= 0xFF80u - 0xC300u;
    };
    const auto other = [&](uint32_t b) HYP_INLINE {
        b = plain_bits(b);
        const bool small = (b & 0x7FFFu) < kLow;
        centre += small ? 1u : 0u;
        centre_lo = min(centre_lo, small ? place_of(b) : 0xFFFFFFFFu);
        centre_hi = max(centre_hi, small ? place_of(b) : 0u);
        above += b - 0x4300u < 0x7F80u - 0x4300u ? 1u : 0u;   // 2^7 to the largest
        infinite += b == 0x7F80u ? 1u : 0u;
    };
    // Eight tokens at once, two in a register, unless one of them is no fine value (the counting of 64 rows of
    // 262144 took 12.2 us one by one and takes 9.5).
    typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
    const auto eight = [&](const uint32_t (&w)[4]) HYP_INLINE {
        uint32_t at[4], odd = 0u;
#pragma unroll
        for (uint32_t k = 0; k < 4u; ++k) {
            const uint32_t t = __builtin_bit_cast(uint32_t, __builtin_bit_cast(u16x2_t, w[k]) - u16x2_t{kLow, kLow});
            odd |= t;
            at[k] = ((t & 0x0FFF0FFFu) | ((t >> 3) & 0x10001000u)) << 2;   // in bytes
        }
        if ((odd & 0x70007000u) == 0u) {
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) {
                atomicAdd(&s.count[(at[k] & 0xFFFFu) / 4u], 1u);
                atomicAdd(&s.count[at[k] >> 18], 1u);
            }
        } else {
            uint32_t others = 0u;
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) {
                others |= usual(w[k] & 0xFFFFu) ? 0u : 1u << (2u * k);
                others |= usual(w[k] >> 16) ? 0u : 2u << (2u * k);
            }
            if (others != 0u) {
#pragma unroll
                for (uint32_t k = 0; k < 4u; ++k) {
                    if (((others >> (2u * k)) & 1u) != 0u) other(w[k] & 0xFFFFu);
                    if (((others >> (2u * k)) & 2u) != 0u) other(w[k] >> 16);
                }
            }
        }
    };
    if constexpr (kAhead != 0u) {
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k)
            if (i + 8u <= end) {
                eight(ahead[k]);
                i += 8u * kThreads;
            }
    } else {
#pragma unroll 4
        for (; i + 8u <= end; i += 8u * kThreads) {
            uint32_t w[4];
            __builtin_memcpy(w, row + i, 16);
            eight(w);
        }
    }
    for (uint32_t k = i; k < end && k < i + 8u; ++k)
        if (!usual(row[k])) other(row[k]);
    const auto least = [](uint32_t v) HYP_INLINE {
        return from_lane(wave_scan(v, 0xFFFFFFFFu, [](uint32_t a, uint32_t b) { return min(a, b); }), 63u);
    };
    if (__ballot(below != 0u) != 0u) {
        below = wave_sum(below);
        below_bits = least(below_bits);
        if ((tid & 63u) == 0u) {
            atomicAdd(&s.count[kBelowAt], below);
            atomicMin(&s.below, below_bits);
        }
    }
    if (__ballot((centre | above | infinite) != 0u) != 0u) {
        centre = wave_sum(centre);
        centre_lo = least(centre_lo);
        centre_hi = wave_max(centre_hi);
        above = wave_sum(above);
        infinite = wave_sum(infinite);
        if ((tid & 63u) == 0u) {
            atomicAdd(&s.count[kCentreAt], centre);
            atomicMin(&s.centre_lo, centre_lo);
            atomicMax(&s.centre_hi, centre_hi);
            atomicAdd(&s.count[kAboveAt], above);
            atomicAdd(&s.infinite, infinite);
        }
    }
    __syncthreads();
}

// A chunk's counts between two launches (a chunk has fewer than 65536 tokens: 16 bits do).
constexpr uint32_t kStoredBins = (kBins + 7u) & ~7u;
constexpr uint32_t kMaxChunk = 32768;
struct alignas(16) ChunkCounts {
    uint16_t count[kStoredBins];
    uint32_t infinite, centre_lo, centre_hi, below;
};
static_assert(kStoredBins <= kThreads * kPer && kMaxChunk < 65536u, "a chunk's counts");

struct Chunks {
    uint32_t n, tokens;   // chunks of a row, tokens of a chunk (the last one's may be fewer)
};

__device__ __forceinline__ void store_counts(const RowLds& s, ChunkCounts& c) {
    uint2* const out = reinterpret_cast<uint2*>(c.count);
    for (uint32_t i = threadIdx.x; i < kStoredBins / 4u; i += kThreads) {
        const uint4 n = *reinterpret_cast<const uint4*>(&s.count[4u * i]);
        out[i] = make_uint2(n.x | n.y << 16, n.z | n.w << 16);
    }
    if (threadIdx.x == 0u) {
        c.infinite = s.infinite;
        c.centre_lo = s.centre_lo;
        c.centre_hi = s.centre_hi;
        c.below = s.below;
    }
}

// The chunk that holds the number-th of the tokens that the chunks count at place `at`, by every wave for itself; number is then
// that among the chunk's own.
__device__ __forceinline__ uint32_t find_chunk(const ChunkCounts* counts, uint32_t n, uint32_t at, uint32_t& number) {
    const uint32_t lane = threadIdx.x & 63u;
    for (uint32_t base = 0; base < n; base += 64u) {
        const uint32_t here = base + lane < n ? counts[base + lane].count[at] : 0u;
        const uint32_t incl = wave_incl(here);
        const uint64_t past = __ballot(incl > number);
        if (past != 0u) {
            const uint32_t holder = static_cast<uint32_t>(__builtin_ctzll(past));
            number -= from_lane(incl - here, holder);
            return base + holder;
        }
        number -= from_lane(incl, 63u);
    }
    return 0u;
}

#undef HYP_INLINE

}  // namespace hyperion::hip::sampling
