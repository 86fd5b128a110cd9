// One row of logits and its filters, as hyp_sample_batch and hyp_verify_batch take it (sample_batch.hip has the
// steps): counts by value, the weights' sums, how many tokens the filters keep, and the token at a rank. A workgroup
// of kThreads to a row.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

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

__device__ __forceinline__ RowParams row_params(const HypSamplingConfig& c, float u) {
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

__device__ __forceinline__ uint32_t block_min(uint32_t v, Block& s) {
    v = from_lane(wave_scan(v, 0xFFFFFFFFu, [](uint32_t a, uint32_t b) { return min(a, b); }), 63u);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0u) s.u[threadIdx.x >> 6] = v;
    __syncthreads();
    uint32_t r = 0xFFFFFFFFu;
    for (uint32_t w = 0; w < kWaves; ++w) r = min(r, s.u[w]);
    return r;
}

// Mass and count before this thread's bins, and the totals: added in the same order for every thread.
struct Before {
    double mass, mass_all;
    uint32_t count, count_all;
};

// (Every wave has left the block's words.)
__device__ __forceinline__ Before block_scan(double mass, uint32_t count, Block& s) {
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = threadIdx.x >> 6;
    const double m = wave_incl64(mass);
    const uint32_t c = wave_incl(count);
    if (lane == 63u) {
        s.d[wave] = m;
        s.u[wave] = c;
    }
    __syncthreads();
    Before b{0.0, 0.0, 0u, 0u};
    for (uint32_t w = 0; w < kWaves; ++w) {
        if (w == wave) {
            b.mass = b.mass_all;
            b.count = b.count_all;
        }
        b.mass_all += s.d[w];
        b.count_all += s.u[w];
    }
    const double mx = __shfl_up(m, 1u, 64);
    if (lane != 0u) b.mass += mx;
    b.count += c - count;
    return b;
}

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
    uint32_t drawn, number;        // the drawn value's bits, the token's number among those
    uint32_t bin;                  // and its bin, kBins where that is none of the first way
    double top, total, kept;       // the largest value, the tokens' mass, the kept tokens'
    uint32_t keep, rank;           // how many tokens the filters keep, the drawn one's rank
    uint32_t lead[kWaves];         // a wave's first bin with a token
    uint32_t whole;                // without a draw: every token of the last kept value is kept
    uint32_t redo;                 // and: by windows after all
};

// s.count, s.infinite, s.centre_lo and s.centre_hi of the tokens [begin, end) of a row. (A call has a barrier at its end.)
__device__ __forceinline__ void count_values(const uint16_t* row, uint32_t begin, uint32_t end, RowLds& s) {
    const uint32_t tid = threadIdx.x;
    for (uint32_t i = tid; i < kThreads * kPer; i += kThreads) s.count[i] = 0u;
    if (tid == 0u) {
        s.infinite = 0u;
        s.centre_lo = 0xFFFFFFFFu;
        s.centre_hi = 0u;
    }
    __syncthreads();
    // The bits less kLow, in 16 bits: a fine value has 0 in bits 12 to 14, its sign in bit 15.
    const auto one = [&](uint32_t b) HYP_INLINE {
        const uint32_t t = b - kLow;
        if ((t & 0x7000u) == 0u) {
            atomicAdd(&s.count[(t & 0xFFFu) | ((t >> 3) & 0x1000u)], 1u);
            return;
        }
        b = plain_bits(b);
        if (!finite_bits(b)) {
            if (b == 0x7F80u) atomicAdd(&s.infinite, 1u);
        } else if ((b & 0x7FFFu) < kLow) {
            atomicMin(&s.centre_lo, place_of(b));
            atomicMax(&s.centre_hi, place_of(b));
            atomicAdd(&s.count[kCentreAt], 1u);
        } else {
            atomicAdd(&s.count[(b & 0x8000u) != 0u ? kBelowAt : kAboveAt], 1u);
        }
    };
    // Eight tokens at once, two in a register, unless one of them is no fine value (the counting of 64 rows of
    // 262144 took 12.2 us one by one and takes 9.5).
    typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
    uint32_t i = begin + 8u * tid;
#pragma unroll 4
    for (; i + 8u <= end; i += 8u * kThreads) {
        uint32_t w[4], at[4], odd = 0u;
        __builtin_memcpy(w, row + i, 16);
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
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) {
                one(w[k] & 0xFFFFu);
                one(w[k] >> 16);
            }
        }
    }
    for (uint32_t k = i; k < end && k < i + 8u; ++k) one(row[k]);
    __syncthreads();
}

// A chunk's counts between the two launches (a chunk has at most kMaxChunk tokens: 16 bits do).
constexpr uint32_t kStoredBins = (kBins + 7u) & ~7u;
constexpr uint32_t kMaxChunk = 32768;
struct alignas(16) ChunkCounts {
    uint16_t count[kStoredBins];
    uint32_t infinite, centre_lo, centre_hi, unused;
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
    }
}

// s.count and the rest for a whole row, from its chunks: eight bins to a thread, the last ones to the first lanes, a chunk each.
__device__ __forceinline__ void sum_counts(const ChunkCounts* counts, uint32_t n, RowLds& s) {
    const uint32_t tid = threadIdx.x;
    static_assert(kStoredBins == 8u * kThreads + 8u && kBins <= 8u * kThreads + 4u, "a thread's bins");
    uint32_t sum[8] = {};
    const auto add = [&](uint4 v) HYP_INLINE {
        const uint32_t word[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (uint32_t k = 0; k < 4u; ++k) {
            sum[2u * k] += word[k] & 0xFFFFu;
            sum[2u * k + 1u] += word[k] >> 16;
        }
    };
    if (tid < 64u) {
        uint32_t infinite = 0u, lo = 0xFFFFFFFFu, hi = 0u, last[4] = {};
        for (uint32_t c = tid; c < n; c += 64u) {
            const uint2 v = *reinterpret_cast<const uint2*>(counts[c].count + 8u * kThreads);
            infinite += counts[c].infinite;
            lo = min(lo, counts[c].centre_lo);
            hi = max(hi, counts[c].centre_hi);
            last[0] += v.x & 0xFFFFu;
            last[1] += v.x >> 16;
            last[2] += v.y & 0xFFFFu;
            last[3] += v.y >> 16;
        }
        infinite = wave_sum(infinite);
        lo = from_lane(wave_scan(lo, 0xFFFFFFFFu, [](uint32_t a, uint32_t b) { return min(a, b); }), 63u);
        hi = wave_max(hi);
#pragma unroll
        for (uint32_t k = 0; k < 4u; ++k) last[k] = wave_sum(last[k]);
        if (tid == 0u) {
            s.infinite = infinite;
            s.centre_lo = lo;
            s.centre_hi = hi;
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) s.count[8u * kThreads + k] = last[k];
        }
    }
    uint32_t c = 0;
    for (; c + 8u <= n; c += 8u) {
        uint4 v[8];
#pragma unroll
        for (uint32_t k = 0; k < 8u; ++k) v[k] = reinterpret_cast<const uint4*>(counts[c + k].count)[tid];
#pragma unroll
        for (uint32_t k = 0; k < 8u; ++k) add(v[k]);
    }
#pragma unroll 4
    for (; c < n; ++c) add(reinterpret_cast<const uint4*>(counts[c].count)[tid]);
    *reinterpret_cast<uint4*>(&s.count[8u * tid]) = make_uint4(sum[0], sum[1], sum[2], sum[3]);
    *reinterpret_cast<uint4*>(&s.count[8u * tid + 4u]) = make_uint4(sum[4], sum[5], sum[6], sum[7]);
    for (uint32_t i = 8u * kThreads + 4u + tid; i < kThreads * kPer; i += kThreads) s.count[i] = 0u;
    __syncthreads();
}

// From the row's counts in s (after a barrier): the drawn value (kDraw) or the last one that the filters keep, as s.drawn,
// and the token's number among those of that value, s.number; s.top (+inf: only such tokens weigh, 1 each), s.total and
// s.kept. s.bin is its bin if the counts of chunks tell in which chunk it is. False for a row with nothing above -inf. (A
// call has a barrier at its end.)
template <bool kDraw>
__device__ __forceinline__ bool find_row(const uint16_t* row, uint32_t vocab, const RowParams& prm, RowLds& s) {
    const uint32_t tid = threadIdx.x;
    const uint32_t lane = tid & 63u;
    const uint32_t wave = tid >> 6;
    const uint32_t first = kPer * tid;
    const uint32_t infinite = s.infinite;
    uint32_t num[kPer];   // this thread's bins: tokens,
    double weight[kPer];  // weights
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) num[i] = s.count[count_at(first + i)];
    {
        uint32_t lead = 0xFFFFFFFFu;
#pragma unroll
        for (uint32_t i = kPer; i-- > 0u;) lead = num[i] != 0u ? first + i : lead;
        const uint64_t has = __ballot(lead != 0xFFFFFFFFu);
        lead = from_lane(lead, has != 0u ? static_cast<uint32_t>(__builtin_ctzll(has)) : 0u);
        if (lane == 0u) s.lead[wave] = lead;
    }
    if (tid == 0u) {
        s.bin = kBins;
        s.keep = s.rank = 0xFFFFFFFFu;
    }
    __syncthreads();
    if (infinite != 0u) {
        // Weight 1 for each, 0 for everything else.
        uint32_t kept = infinite;
        if (prm.top_k != 0u) kept = min(kept, prm.top_k);
        if (prm.top_p != 0.0) kept = min(kept, static_cast<uint32_t>(ceil(prm.top_p * infinite)));
        if (prm.greedy || prm.min_p > 1.0) kept = 1u;
        if (tid == 0u) {
            s.drawn = 0x7F80u;
            s.number = kDraw ? static_cast<uint32_t>(fmin(prm.u * kept, static_cast<double>(kept - 1u))) : kept - 1u;
            s.whole = kept == infinite;
            s.top = __builtin_huge_val();
            s.total = infinite;
            s.kept = kept;
        }
        __syncthreads();
        return true;
    }
    {
        uint32_t lead = 0xFFFFFFFFu;
        for (uint32_t w = 0; w < kWaves; ++w) lead = min(lead, s.lead[w]);
        if (lead == 0xFFFFFFFFu) return false;   // nothing above -inf
        const auto fine_bits = [&](uint32_t bin) HYP_INLINE {
            return bin <= kFine ? kLow + (kFine - bin) : (bin == kCentre ? bits_at(s.centre_lo) : 0x8000u | (kLow + (bin - kCentre - 1u)));
        };
        // The long way's windows that hold values, and its largest value.
        const bool centres = s.count[kCentreAt] != 0u && s.centre_lo != s.centre_hi;
        bool windowed = lead == kAbove || lead == kBelow || (centres && (kDraw || lead == kCentre));
        if (!windowed && s.count[kBelowAt] != 0u)   // (2^23 times e^-80)
            windowed = !((value_of(fine_bits(lead)) + 128.0) * prm.by_t > 80.0);
        double top = 0.0;
        uint32_t windows = 1u;
        const auto look_for_windows = [&]() HYP_INLINE {
            uint32_t best = 0xFFFFFFFFu;
            uint32_t held = 0u;
            for_tokens(row, 0u, vocab, tid, kThreads, [&](uint32_t, uint32_t b) {
                b = plain_bits(b);
                if (!finite_bits(b)) return;
                best = min(best, place_of(b));
                held |= 1u << (place_of(b) / kWindow);
            });
            best = block_min(best, s.block);
            windows = 0u;
            for (uint32_t w = 0; w < kWindows; ++w)
                if (block_min((held >> w) & 1u ? 0u : 1u, s.block) == 0u) windows |= 1u << w;
            top = value_of(bits_at(best));
        };
        // (Written out for either way. For one row of 262144: 19.3 us so, 19.8 with one copy and a test at each step, 22.9
        // with one loop over the steps.)
        // False where one bin cannot tell: the cut is among the values below -2^7 (e^-80 is above 2^-116) or next to 0, or
        // several values next to 0, less than 2^-24 apart, weigh enough for that to matter to an fp64 sum.
        const auto find = [&](auto by_windows) HYP_INLINE {
            constexpr bool slow = decltype(by_windows)::value;
            uint32_t window = 0u;   // the first place of the window in hand
            const auto bits_of = [&](uint32_t bin) HYP_INLINE { return slow ? bits_at(window + bin) : fine_bits(bin); };
            Before at{};
            uint32_t here = 0u;     // this thread's tokens
            const auto weigh = [&]() HYP_INLINE {
                here = 0u;
#pragma unroll
                for (uint32_t i = 0; i < kPer; ++i) {
                    here += num[i];
                    weight[i] = 0.0;
                }
                double mass = 0.0;
                if (here != 0u) {
#pragma unroll
                    for (uint32_t i = 0; i < kPer; ++i) {
                        const uint32_t bin = first + i;
                        const double w = exp_below((value_of(bits_of(bin)) - top) * prm.by_t);
                        if (num[i] != 0u && (slow || bin != kBelow)) weight[i] = w;
                        mass += num[i] * weight[i];
                    }
                }
                at = block_scan(mass, here, s.block);
            };
            if (!slow) weigh();
            // f() with each window's counts and weights in hand, and what lies before this thread's bins.
            const auto over_windows = [&](auto&& f) HYP_INLINE {
                if (!slow) {
                    f(at.mass, at.count);
                    return;
                }
                double mass = 0.0;
                uint32_t count = 0u;
                for (uint32_t w = 0; w < kWindows; ++w) {
                    if (((windows >> w) & 1u) == 0u) continue;
                    __syncthreads();
                    for (uint32_t i = tid; i < kThreads * kPer; i += kThreads) s.count[i] = 0u;
                    __syncthreads();
                    window = w * kWindow;
                    for_tokens(row, 0u, vocab, tid, kThreads, [&](uint32_t, uint32_t b) {
                        b = plain_bits(b);
                        const uint32_t d = place_of(b) - window;
                        if (finite_bits(b) && d < kWindow) atomicAdd(&s.count[d], 1u);
                    });
                    __syncthreads();
#pragma unroll
                    for (uint32_t i = 0; i < kPer; ++i) num[i] = s.count[first + i];
                    weigh();
                    f(mass + at.mass, count + at.count);
                    mass += at.mass_all;
                    count += at.count_all;
                }
            };
            // The mass up to and with this thread's bins.
            const auto mass_with = [&](double mass) HYP_INLINE {
#pragma unroll
                for (uint32_t i = 0; i < kPer; ++i) mass += num[i] * weight[i];
                return mass;
            };
            double total = 0.0;
            uint32_t all = 0u;
            if (slow) {
                over_windows([&](double, uint32_t) HYP_INLINE {
                    total += at.mass_all;
                    all += at.count_all;
                });
            } else {
                total = at.mass_all;
                all = at.count_all;
            }
            uint32_t kept = all;
            if (prm.top_k != 0u) kept = min(kept, prm.top_k);
            if (prm.top_p != 0.0 || prm.min_p != 0.0) {
                // A wave's first lane whose bins a filter does not keep whole goes through them.
                const double enough = prm.top_p * total;
                over_windows([&](double mass, uint32_t count) HYP_INLINE {
                    uint32_t keep = 0xFFFFFFFFu;
                    if (prm.top_p != 0.0) {
                        const uint64_t past = __ballot(mass_with(mass) > enough);
                        if (past != 0u && lane == static_cast<uint32_t>(__builtin_ctzll(past))) {
                            keep = count;
                            double m = mass;
#pragma unroll
                            for (uint32_t i = 0; i < kPer; ++i) {
                                const double room = enough - m;
                                const double some = num[i] * weight[i];
                                if (num[i] != 0u && room > 0.0)
                                    keep += room >= some ? num[i] : min(num[i], static_cast<uint32_t>(ceil(room / weight[i])));
                                m += some;
                            }
                        }
                    }
                    uint32_t light = 0u;   // before the first token that min-p drops
                    bool dropped = false;
#pragma unroll
                    for (uint32_t i = 0; i < kPer; ++i) {
                        dropped = dropped || (num[i] != 0u && weight[i] < prm.min_p);
                        light += dropped ? 0u : num[i];
                    }
                    const uint64_t drops = __ballot(dropped);
                    if (drops != 0u && lane == static_cast<uint32_t>(__builtin_ctzll(drops))) keep = min(keep, count + light);
                    if (keep != 0xFFFFFFFFu) atomicMin(&s.keep, keep);
                });
                __syncthreads();
                kept = min(kept, s.keep);
            }
            kept = prm.greedy ? 1u : max(kept, 1u);
            if constexpr (!kDraw && !slow) {
                const uint32_t below = s.count[kBelowAt];
                if (below != 0u && ((kept > all - below && kept != all) || (prm.min_p != 0.0 && prm.min_p < 0x1p-110)))
                    return false;
                if (centres) {
                    uint32_t count = at.count;
#pragma unroll
                    for (uint32_t i = 0; i < kPer; ++i) {
                        if (first + i == kCentre)
                            s.redo = kept - 1u - count < num[i] || num[i] * weight[i] * prm.by_t > 0x1p-30 * total;
                        count += num[i];
                    }
                    __syncthreads();
                    if (s.redo != 0u) return false;
                }
            }
            // The kept tokens' mass, the rank of the draw, its value.
            over_windows([&](double mass, uint32_t count) HYP_INLINE {
                if (kept - 1u - count >= here) return;
#pragma unroll
                for (uint32_t i = 0; i < kPer; ++i) {
                    if (kept - 1u - count < num[i]) s.kept = mass + (kept - count) * weight[i];
                    mass += num[i] * weight[i];
                    count += num[i];
                }
            });
            __syncthreads();
            if (tid == 0u) {
                s.top = top;
                s.total = total;
            }
            uint32_t rank = kept - 1u;
            if constexpr (kDraw) {
                const double goal = prm.u * s.kept;
                over_windows([&](double mass, uint32_t count) HYP_INLINE {
                    const uint64_t past = __ballot(mass_with(mass) > goal);
                    if (past == 0u || lane != static_cast<uint32_t>(__builtin_ctzll(past))) return;
                    uint32_t rank = 0xFFFFFFFFu;
#pragma unroll
                    for (uint32_t i = 0; i < kPer; ++i) {
                        if (rank == 0xFFFFFFFFu && num[i] != 0u && mass + num[i] * weight[i] > goal) {
                            const double j = (goal - mass) / weight[i];
                            rank = count + (j > 0.0 ? min(static_cast<uint32_t>(fmin(j, 4.0e9)), num[i] - 1u) : 0u);
                        }
                        mass += num[i] * weight[i];
                        count += num[i];
                    }
                    atomicMin(&s.rank, rank);
                });
                __syncthreads();
                rank = min(s.rank, kept - 1u);
            }
            over_windows([&](double, uint32_t count) HYP_INLINE {
                if (rank - count >= here) return;
#pragma unroll
                for (uint32_t i = 0; i < kPer; ++i) {
                    if (rank - count < num[i]) {
                        s.drawn = bits_of(first + i);
                        s.number = rank - count;
                        if (!slow) s.bin = first + i;
                        if (!kDraw) s.whole = num[i] == rank - count + 1u;
                        if (!kDraw && !slow && first + i == kBelow) s.drawn = 0xFF7Fu;   // (all are kept)
                    }
                    count += num[i];
                }
            });
            __syncthreads();
            return true;
        };
        if constexpr (kDraw) {
            if (windowed) look_for_windows(); else top = value_of(fine_bits(lead));
            if (windowed) find(std::true_type{}); else find(std::false_type{});
        } else {
            if (!windowed) {
                top = value_of(fine_bits(lead));
                windowed = !find(std::false_type{});
                if (windowed && tid == 0u) s.keep = 0xFFFFFFFFu;
            }
            if (windowed) {
                look_for_windows();
                find(std::true_type{});
            }
        }
        return true;
    }
}

// f(index) by the lane that holds it, of the s.number-th token of value s.drawn in the row; kSplit: `counts` are its
// chunks' counts. Each wave marks the value's places in its stretch, 512 tokens a step.
template <bool kSplit, typename F>
__device__ __forceinline__ void find_token(const uint16_t* row, uint32_t vocab, Chunks chunks, const ChunkCounts* counts,
                                           RowLds& s, F&& f) {
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = threadIdx.x >> 6;
    const uint32_t drawn = s.drawn;
    uint32_t number = s.number;
    uint32_t from_token = 0u, to_token = vocab;
    if (kSplit && s.bin != kBins) {
        const uint32_t at = count_at(s.bin);
        uint32_t chunk = 0u;
        for (uint32_t base = 0; base < chunks.n; base += 64u) {   // (every wave for itself)
            const uint32_t n = base + lane < chunks.n ? counts[base + lane].count[at] : 0u;
            const uint32_t incl = wave_incl(n);
            const uint64_t past = __ballot(incl > number);
            if (past != 0u) {
                const uint32_t holder = static_cast<uint32_t>(__builtin_ctzll(past));
                chunk = base + holder;
                number -= from_lane(incl - n, holder);
                break;
            }
            number -= from_lane(incl, 63u);
        }
        from_token = min(vocab, chunk * chunks.tokens);
        to_token = min(vocab, from_token + chunks.tokens);
    }
    constexpr uint32_t kStep = 512u, kSteps = 8u;
    for (uint32_t base = from_token; base < to_token; base += kWaves * kSteps * kStep) {
        const uint32_t end = min(to_token, base + kWaves * kSteps * kStep);
        const uint32_t steps = (end - base + kWaves * kStep - 1u) / (kWaves * kStep);
        const uint32_t begin = base + wave * steps * kStep + 8u * lane;   // the lane's, of the first step
        Eight e[kSteps];
#pragma unroll
        for (uint32_t k = 0; k < kSteps; ++k)
            if (k < steps && begin + k * kStep + 8u <= end) __builtin_memcpy(&e[k], row + begin + k * kStep, 16);
        uint64_t hits = 0u;   // a byte a step
#pragma unroll
        for (uint32_t k = 0; k < kSteps; ++k) {
            const uint32_t from = begin + k * kStep;
            if (k >= steps || from >= end) continue;
            uint32_t bits = 0u;
            if (from + 8u <= end) {
#pragma unroll
                for (uint32_t i = 0; i < 8u; ++i) bits |= plain_bits(e[k].v[i]) == drawn ? 1u << i : 0u;
            } else {
                for (uint32_t i = 0; from + i < end; ++i) bits |= plain_bits(row[from + i]) == drawn ? 1u << i : 0u;
            }
            hits |= static_cast<uint64_t>(bits) << (8u * k);
        }
        const uint32_t mine = wave_sum(static_cast<uint32_t>(__popcll(hits)));
        __syncthreads();
        if (lane == 0u) s.block.u[wave] = mine;
        __syncthreads();
        uint32_t before = 0u, all = 0u;
        for (uint32_t w = 0; w < kWaves; ++w) {
            if (w == wave) before = all;
            all += s.block.u[w];
        }
        if (number >= all) {
            number -= all;
            continue;
        }
        uint32_t left = number - before;   // (wraps past the holder)
        if (left >= mine) return;
        for (uint32_t k = 0; k < steps; ++k) {
            uint32_t bits = static_cast<uint32_t>(hits >> (8u * k)) & 0xFFu;
            const uint32_t n = static_cast<uint32_t>(__popc(bits));
            const uint32_t incl = wave_incl(n);
            const uint32_t step = from_lane(incl, 63u);
            if (left < step) {
                if (left - (incl - n) < n) {
                    for (uint32_t i = left - (incl - n); i != 0u; --i) bits &= bits - 1u;
                    f(begin + k * kStep + static_cast<uint32_t>(__builtin_ctz(bits)));
                }
                return;
            }
            left -= step;
        }
        return;
    }
}

// A row's chunks: enough workgroups for the device (two are on a compute unit), but no more than the second launch
// reads in little time. Measured with 256 .. 1024 workgroups, chunks of 4096 .. 16384 and 16 .. 64 of them:
// 400 rows of 128000 took 83 us with 512 workgroups and more, 114 with 256; one row of 262144 took 27.5 us with 16
// chunks, 29 with 32 and 37 with 64; what else was tried differed by a tenth at most.
constexpr uint32_t kFill = 512;
constexpr uint32_t kMinChunk = 8192;
constexpr uint32_t kMostChunks = 16;
inline Chunks chunks_of(uint32_t rows, uint32_t vocab) {
    uint32_t n = rows == 0u ? 1u : std::min((kFill + rows - 1u) / rows, std::min(vocab / kMinChunk + 1u, kMostChunks));
    if (n <= 1u) return {1u, vocab};
    n = std::max(n, (vocab + kMaxChunk - 1u) / kMaxChunk);
    const uint32_t tokens = std::min(((vocab + n - 1u) / n + 511u) & ~511u, kMaxChunk);
    return {(vocab + tokens - 1u) / tokens, tokens};
}

#undef HYP_INLINE

}  // namespace hyperion::hip::sampling
