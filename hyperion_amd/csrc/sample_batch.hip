// Sampling of many rows from given uniforms (hyp_sample_batch): temperature, top-k, top-p and
// min-p of its own for every row.
//
// The order of a row's tokens is value descending, index ascending; w_j = exp((x_j - x_max) / T).
// Each filter keeps a prefix of that order (top-k: k tokens; top-p: those before which the running sum
// of w is below p times the total; min-p: w_j >= min_p), the kept tokens are the shortest prefix, and the
// draw is the first token whose running sum exceeds u times the kept total. The logits are bf16, so
// a row is described by how many tokens have each value: every running sum is
// sum over values of count * w(value), exact counts times a weight in fp64, in one fixed order. That
// leaves the result independent of how the counting went, and right next to a border up to fp64
// rounding.
//
// Steps, with one workgroup for 2 and 3 and, unless there are rows enough, several for 1:
//  1. counts by value in LDS, each workgroup's for its chunk of the row; a second launch adds a row's chunks. A bin for each bf16 value of magnitude 2^-25 .. 2^7 (8192), one for
//     what is nearer to 0, one for what is above and one for what is below;
//  2. every thread takes 9 neighbouring bins, their weights, and scans of count and mass over the
//     workgroup; then the kept count, the kept mass, the drawn rank, its bin and its number j there;
//  3. the j-th token of that value: the chunk that holds it by the chunks' counts, then by counting along it.
// Rows whose other three bins matter to the result (a value above 2^7; several values nearer to 0 than
// 2^-25; values below -2^7 that are not negligible at this temperature) take the same steps over
// windows of 8192 values of the whole order, counting the row again for each.
#include <algorithm>
#include <cstdint>

#include "common.h"
#include "kernels.h"
#include "sample_batch.h"

namespace hyperion::hip {
namespace {

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
constexpr uint32_t kWindow = 8192;                    // values of one window of the long way
constexpr uint32_t kWindows = 65536u / kWindow;
constexpr uint32_t kMaxVocab = 1u << 23;
static_assert(kBins <= kThreads * kPer, "a thread's bins");

struct RowParams {
    double t;        // the weights' temperature (1 for a greedy row)
    double top_p, min_p, u;
    uint32_t top_k;  // 0: off
    bool greedy;
};

__device__ __forceinline__ RowParams row_params(const HypSamplingConfig* configs, const float* uniforms, uint32_t row) {
    const HypSamplingConfig c = configs[row];
    RowParams r;
    r.greedy = !(c.temperature > 0.0f);
    r.t = r.greedy ? 1.0 : static_cast<double>(c.temperature);
    r.top_p = c.top_p > 0.0f && c.top_p < 1.0f ? static_cast<double>(c.top_p) : 0.0;
    r.min_p = c.min_p > 0.0f ? static_cast<double>(c.min_p) : 0.0;
    r.top_k = c.top_k > 0 ? static_cast<uint32_t>(c.top_k) : 0u;
    const float u = uniforms[row];
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

// Sums over the workgroup, each value in the same order for every thread.
struct Block {
    double d[kWaves];
    uint64_t u[kWaves];
};

__device__ __forceinline__ uint64_t block_sum(uint64_t v, Block& s) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m, 64);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0u) s.u[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t r = 0u;
    for (uint32_t w = 0; w < kWaves; ++w) r += s.u[w];
    return r;
}

__device__ __forceinline__ uint32_t block_min(uint32_t v, Block& s) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v = min(v, static_cast<uint32_t>(__shfl_xor(v, m, 64)));
    __syncthreads();
    if ((threadIdx.x & 63u) == 0u) s.u[threadIdx.x >> 6] = v;
    __syncthreads();
    uint32_t r = 0xFFFFFFFFu;
    for (uint32_t w = 0; w < kWaves; ++w) r = min(r, static_cast<uint32_t>(s.u[w]));
    return r;
}

// Mass and count before this thread's bins, and the totals.
struct Before {
    double mass, mass_all;
    uint32_t count, count_all;
};

__device__ __forceinline__ Before block_scan(double mass, uint32_t count, Block& s) {
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = threadIdx.x >> 6;
    double m = mass;
    uint32_t c = count;
#pragma unroll
    for (uint32_t d = 1; d < 64u; d <<= 1) {
        const double y = __shfl_up(m, d, 64);
        const uint32_t z = __shfl_up(c, d, 64);
        if (lane >= d) {
            m += y;
            c += z;
        }
    }
    __syncthreads();
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
        b.count_all += static_cast<uint32_t>(s.u[w]);
    }
    const double mx = __shfl_up(m, 1u, 64);
    const uint32_t cx = __shfl_up(c, 1u, 64);
    if (lane != 0u) {
        b.mass += mx;
        b.count += cx;
    }
    return b;
}

struct alignas(16) RowLds {
    uint32_t count[kThreads * kPer];
    Block block;
    uint32_t infinite;             // +inf tokens
    uint32_t centre_lo, centre_hi; // least and largest place of the values next to 0
    uint32_t drawn, number;        // the drawn value's bits, the token's number among those
    uint32_t bin;                  // and its bin, kBins where that is none of the first way
    double kept;
    uint32_t rank;
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
    for_tokens(row, begin, end, tid, kThreads, [&](uint32_t, uint32_t b) {
        const uint32_t f = (b & 0x7FFFu) - kLow;
        uint32_t bin = (b & 0x8000u) != 0u ? kCentre + 1u + f : kFine - f;
        if (f >= kFine) {
            b = plain_bits(b);
            if (!finite_bits(b)) {
                if (b == 0x7F80u) atomicAdd(&s.infinite, 1u);
                return;
            }
            bin = (b & 0x7FFFu) < kLow ? kCentre : ((b & 0x8000u) != 0u ? kBelow : kAbove);
            if (bin == kCentre) {
                atomicMin(&s.centre_lo, place_of(b));
                atomicMax(&s.centre_hi, place_of(b));
            }
        }
        atomicAdd(&s.count[bin], 1u);
    });
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

__global__ __launch_bounds__(kThreads) void sample_count_kernel(const uint16_t* __restrict__ logits, uint32_t vocab,
                                                                Chunks chunks, ChunkCounts* __restrict__ counts) {
    __shared__ RowLds s;
    const uint32_t row = blockIdx.x / chunks.n;
    const uint32_t begin = min(vocab, (blockIdx.x - row * chunks.n) * chunks.tokens);
    count_values(logits + static_cast<size_t>(row) * vocab, begin, min(vocab, begin + chunks.tokens), s);
    ChunkCounts& c = counts[blockIdx.x];
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

// The same for a whole row, from its chunks.
__device__ __forceinline__ void sum_counts(const ChunkCounts* counts, uint32_t n, RowLds& s) {
    const uint32_t tid = threadIdx.x;
    for (uint32_t i = kStoredBins + tid; i < kThreads * kPer; i += kThreads) s.count[i] = 0u;
    for (uint32_t i = tid; i < kStoredBins / 4u; i += kThreads) {
        uint4 sum = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 8
        for (uint32_t c = 0; c < n; ++c) {
            const uint2 v = reinterpret_cast<const uint2*>(counts[c].count)[i];
            sum.x += v.x & 0xFFFFu;
            sum.y += v.x >> 16;
            sum.z += v.y & 0xFFFFu;
            sum.w += v.y >> 16;
        }
        *reinterpret_cast<uint4*>(&s.count[4u * i]) = sum;
    }
    if (tid < 64u) {
        uint32_t infinite = 0u, lo = 0xFFFFFFFFu, hi = 0u;
        for (uint32_t c = tid; c < n; c += 64u) {
            infinite += counts[c].infinite;
            lo = min(lo, counts[c].centre_lo);
            hi = max(hi, counts[c].centre_hi);
        }
#pragma unroll
        for (int m = 32; m > 0; m >>= 1) {
            infinite += __shfl_xor(infinite, m, 64);
            lo = min(lo, static_cast<uint32_t>(__shfl_xor(lo, m, 64)));
            hi = max(hi, static_cast<uint32_t>(__shfl_xor(hi, m, 64)));
        }
        if (tid == 0u) {
            s.infinite = infinite;
            s.centre_lo = lo;
            s.centre_hi = hi;
        }
    }
    __syncthreads();
}

template <bool kSplit>
__global__ __launch_bounds__(kThreads) void sample_rows_kernel(const uint16_t* __restrict__ logits, uint32_t vocab,
                                                               const HypSamplingConfig* __restrict__ configs,
                                                               const float* __restrict__ uniforms, Chunks chunks,
                                                               const ChunkCounts* __restrict__ counts,
                                                               uint32_t* __restrict__ tokens, float* __restrict__ logprobs) {
    __shared__ RowLds s;
    const uint32_t tid = threadIdx.x;
    const uint32_t lane = tid & 63u;
    const uint32_t wave = tid >> 6;
    const uint32_t row_at = blockIdx.x;
    const uint16_t* row = logits + static_cast<size_t>(row_at) * vocab;
    const RowParams prm = row_params(configs, uniforms, row_at);

    // 1. Counts by value.
    if constexpr (kSplit) {
        counts += static_cast<size_t>(row_at) * chunks.n;
        sum_counts(counts, chunks.n, s);
    } else {
        count_values(row, 0u, vocab, s);
    }

    // 2. The drawn value and the token's number among those of that value.
    const uint32_t first = kPer * tid;
    uint32_t infinite = s.infinite;
    double logprob;
    if (tid == 0u) s.bin = kBins;
    if (infinite != 0u) {
        // Weight 1 for each, 0 for everything else.
        uint32_t kept = infinite;
        if (prm.top_k != 0u) kept = min(kept, prm.top_k);
        if (prm.top_p != 0.0) kept = min(kept, static_cast<uint32_t>(ceil(prm.top_p * infinite)));
        if (prm.greedy) kept = 1u;
        if (tid == 0u) {
            s.drawn = 0x7F80u;
            s.number = static_cast<uint32_t>(fmin(prm.u * kept, static_cast<double>(kept - 1u)));
        }
        logprob = -log(static_cast<double>(infinite));
        __syncthreads();
    } else {
        uint32_t lead = 0xFFFFFFFFu;
        for (uint32_t i = 0; i < kPer; ++i)
            if (lead == 0xFFFFFFFFu && s.count[first + i] != 0u) lead = first + i;
        lead = block_min(lead, s.block);
        if (lead == 0xFFFFFFFFu) {   // nothing above -inf
            if (tid == 0u) {
                tokens[row_at] = 0u;
                if (logprobs != nullptr) logprobs[row_at] = -__builtin_huge_valf();
            }
            return;
        }
        const auto fine_bits = [&](uint32_t bin) HYP_INLINE {
            return bin <= kFine ? kLow + (kFine - bin) : (bin == kCentre ? bits_at(s.centre_lo) : 0x8000u | (kLow + (bin - kCentre - 1u)));
        };
        // The long way's windows that hold values, and its largest value.
        const uint32_t below = s.count[kBelow];
        bool slow = lead == kAbove || lead == kBelow || (s.count[kCentre] != 0u && s.centre_lo != s.centre_hi);
        if (!slow && below != 0u) slow = !((value_of(fine_bits(lead)) + 128.0) / prm.t > 80.0);   // (2^23 times e^-80)
        double top = 0.0;
        uint32_t windows = 1u;
        if (slow) {
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
        } else {
            top = value_of(fine_bits(lead));
        }
        uint32_t window = 0u;   // the first place of the window in hand
        const auto bits_of = [&](uint32_t bin) HYP_INLINE { return slow ? bits_at(window + bin) : fine_bits(bin); };
        double weight[kPer];
        Before at{};
        const auto weigh = [&]() HYP_INLINE {
            double mass = 0.0;
            uint32_t count = 0u;
#pragma unroll
            for (uint32_t i = 0; i < kPer; ++i) {
                const uint32_t n = s.count[first + i];
                const uint32_t bin = first + i;
                weight[i] = 0.0;
                if (n != 0u && (slow || bin != kBelow)) weight[i] = exp((value_of(bits_of(bin)) - top) / prm.t);
                mass += n * weight[i];
                count += n;
            }
            at = block_scan(mass, count, s.block);
        };
        if (!slow) weigh();
        // f() with each window's counts and weights in hand, and what lies before the window.
        const auto over_windows = [&](auto&& f) HYP_INLINE {
            if (!slow) {
                f(0.0, 0u);
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
                weigh();
                f(mass, count);
                mass += at.mass_all;
                count += at.count_all;
            }
        };
        // Runs over this thread's bins: f(bin index, tokens, weight, mass before, tokens before).
        const auto over_bins = [&](double mass, uint32_t count, auto&& f) HYP_INLINE {
            mass += at.mass;
            count += at.count;
#pragma unroll
            for (uint32_t i = 0; i < kPer; ++i) {
                const uint32_t n = s.count[first + i];
                f(first + i, n, weight[i], mass, count);
                mass += n * weight[i];
                count += n;
            }
        };
        double total = 0.0;
        uint32_t all = 0u;
        over_windows([&](double mass, uint32_t count) HYP_INLINE {
            total = mass + at.mass_all;
            all = count + at.count_all;
        });
        uint32_t kept = all;
        if (prm.top_k != 0u) kept = min(kept, prm.top_k);
        if (prm.top_p != 0.0 || prm.min_p != 0.0) {
            uint64_t both = 0u;   // tokens that top-p keeps, and min-p
            over_windows([&](double m0, uint32_t c0) HYP_INLINE {
                over_bins(m0, c0, [&](uint32_t, uint32_t n, double w, double mass, uint32_t) HYP_INLINE {
                    if (n == 0u) return;
                    uint32_t c = n;
                    if (prm.top_p != 0.0) {
                        const double room = prm.top_p * total - mass;
                        c = room <= 0.0 ? 0u : (room >= n * w ? n : min(n, static_cast<uint32_t>(ceil(room / w))));
                    }
                    both += c;
                    if (w >= prm.min_p) both += static_cast<uint64_t>(n) << 32;
                });
            });
            both = block_sum(both, s.block);
            kept = min(kept, min(static_cast<uint32_t>(both), static_cast<uint32_t>(both >> 32)));
        }
        kept = prm.greedy ? 1u : max(kept, 1u);
        // The kept tokens' mass, the rank of the draw, its value.
        over_windows([&](double m0, uint32_t c0) HYP_INLINE {
            over_bins(m0, c0, [&](uint32_t, uint32_t n, double w, double mass, uint32_t count) HYP_INLINE {
                if (kept - 1u - count < n) s.kept = mass + (kept - count) * w;
            });
        });
        __syncthreads();
        const double goal = prm.u * s.kept;
        uint32_t rank = 0xFFFFFFFFu;
        over_windows([&](double m0, uint32_t c0) HYP_INLINE {
            over_bins(m0, c0, [&](uint32_t, uint32_t n, double w, double mass, uint32_t count) HYP_INLINE {
                if (rank != 0xFFFFFFFFu || n == 0u || !(mass + n * w > goal)) return;
                const double j = (goal - mass) / w;
                rank = count + (j > 0.0 ? min(static_cast<uint32_t>(fmin(j, 4.0e9)), n - 1u) : 0u);
            });
        });
        rank = min(block_min(rank, s.block), kept - 1u);
        over_windows([&](double m0, uint32_t c0) HYP_INLINE {
            over_bins(m0, c0, [&](uint32_t bin, uint32_t n, double, double, uint32_t count) HYP_INLINE {
                if (rank - count < n) {
                    s.drawn = bits_of(bin);
                    s.number = rank - count;
                    if (!slow) s.bin = bin;
                }
            });
        });
        __syncthreads();
        logprob = (value_of(s.drawn) - top) / prm.t - log(total);
    }

    // 3. The token: each wave counts a stretch of the row (or of the chunk that holds it), the one that
    // holds it looks again.
    const uint32_t drawn = s.drawn;
    uint32_t number = s.number;
    uint32_t from_token = 0u, to_token = vocab;
    if (kSplit && s.bin != kBins) {
        const uint32_t bin = s.bin;
        uint32_t chunk = 0u;
        for (uint32_t base = 0; base < chunks.n; base += 64u) {   // (every wave for itself)
            const uint32_t n = base + lane < chunks.n ? counts[base + lane].count[bin] : 0u;
            uint32_t incl = n;
#pragma unroll
            for (uint32_t d = 1; d < 64u; d <<= 1) {
                const uint32_t y = __shfl_up(incl, d, 64);
                if (lane >= d) incl += y;
            }
            const uint64_t past = __ballot(incl > number);
            if (past != 0u) {
                const int at = __builtin_ctzll(past);
                chunk = base + static_cast<uint32_t>(at);
                number -= __shfl(incl - n, at, 64);
                break;
            }
            number -= __shfl(incl, 63, 64);
        }
        from_token = min(vocab, chunk * chunks.tokens);
        to_token = min(vocab, from_token + chunks.tokens);
    }
    const uint32_t stretch = ((to_token - from_token + kWaves - 1u) / kWaves + 511u) & ~511u;
    const uint32_t begin = min(to_token, from_token + wave * stretch);
    const uint32_t end = min(to_token, begin + stretch);
    uint32_t mine = 0u;
    for_tokens(row, begin, end, lane, 64u, [&](uint32_t, uint32_t b) { mine += plain_bits(b) == drawn ? 1u : 0u; });
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) mine += __shfl_xor(mine, m, 64);
    __syncthreads();
    if (lane == 0u) s.block.u[wave] = mine;
    __syncthreads();
    for (uint32_t w = 0; w < wave; ++w) number -= static_cast<uint32_t>(s.block.u[w]);   // (wraps past the holder)
    if (number >= mine) return;
    for (uint32_t at = begin; at < end; at += 512u) {
        uint32_t n = 0u;
        const uint32_t from = at + 8u * lane;
        for (uint32_t k = from; k < min(end, from + 8u); ++k) n += plain_bits(row[k]) == drawn ? 1u : 0u;
        uint32_t incl = n;
#pragma unroll
        for (uint32_t d = 1; d < 64u; d <<= 1) {
            const uint32_t y = __shfl_up(incl, d, 64);
            if (lane >= d) incl += y;
        }
        const uint32_t before = incl - n;
        if (number - before < n) {
            uint32_t left = number - before;
            for (uint32_t k = from; k < min(end, from + 8u); ++k) {
                if (plain_bits(row[k]) != drawn) continue;
                if (left == 0u) {
                    tokens[row_at] = k;
                    if (logprobs != nullptr) logprobs[row_at] = static_cast<float>(logprob);
                }
                --left;
            }
        }
        const uint32_t here = __shfl(incl, 63, 64);
        if (number < here) return;
        number -= here;
    }
}

// A row's chunks: enough workgroups for the device (two are on a compute unit), but no more than the second launch
// reads in little time. Measured with 256 .. 1024 workgroups, chunks of 4096 .. 16384 and 16 .. 64 of them:
// 400 rows of 128000 took 83 us with 512 workgroups and more, 114 with 256; one row of 262144 took 27.5 us with 16
// chunks, 29 with 32 and 37 with 64; what else was tried differed by a tenth at most.
constexpr uint32_t kFill = 512;
constexpr uint32_t kMinChunk = 8192;
constexpr uint32_t kMostChunks = 16;
Chunks chunks_of(uint32_t rows, uint32_t vocab) {
    uint32_t n = rows == 0u ? 1u : std::min((kFill + rows - 1u) / rows, std::min(vocab / kMinChunk + 1u, kMostChunks));
    if (n <= 1u) return {1u, vocab};
    n = std::max(n, (vocab + kMaxChunk - 1u) / kMaxChunk);
    const uint32_t tokens = std::min(((vocab + n - 1u) / n + 511u) & ~511u, kMaxChunk);
    return {(vocab + tokens - 1u) / tokens, tokens};
}

}  // namespace

uint32_t sample_batch_max_vocab() { return kMaxVocab; }

size_t sample_batch_workspace_bytes(uint32_t rows, uint32_t vocab) {
    const Chunks c = chunks_of(rows, vocab);
    return c.n > 1u ? static_cast<size_t>(rows) * c.n * sizeof(ChunkCounts) : 0u;
}

void launch_sample_batch(const uint16_t* logits, uint32_t rows, uint32_t vocab, const HypSamplingConfig* configs,
                         const float* uniforms, uint32_t* tokens, float* logprobs, void* workspace,
                         size_t, hipStream_t stream) {
    const Chunks c = chunks_of(rows, vocab);
    if (c.n > 1u) {
        ChunkCounts* const counts = static_cast<ChunkCounts*>(workspace);
        hipLaunchKernelGGL(sample_count_kernel, dim3(rows * c.n), dim3(kThreads), 0, stream, logits, vocab, c, counts);
        HYP_HIP_CHECK(hipGetLastError());
        hipLaunchKernelGGL(sample_rows_kernel<true>, dim3(rows), dim3(kThreads), 0, stream, logits, vocab, configs, uniforms,
                           c, counts, tokens, logprobs);
    } else {
        hipLaunchKernelGGL(sample_rows_kernel<false>, dim3(rows), dim3(kThreads), 0, stream, logits, vocab, configs,
                           uniforms, c, nullptr, tokens, logprobs);
    }
    HYP_HIP_CHECK(hipGetLastError());
}

}  // namespace hyperion::hip
