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
//  1. counts by value in LDS, each workgroup's for its chunk of the row; a second launch adds a row's chunks.
//     A bin for each bf16 value of magnitude 2^-25 .. 2^7 (8192), one for what is nearer to 0, one for what
//     is above and one for what is below;
//  2. every thread takes 9 neighbouring bins, their weights, and scans of count and mass over the
//     workgroup; then the kept count, the kept mass, the drawn rank, its bin and its number j there;
//  3. the j-th token of that value: the chunk that holds it by the chunks' counts, then by counting along it.
// Rows whose other three bins matter to the result (a value above 2^7; several values nearer to 0 than
// 2^-25; values below -2^7 that would not be negligible at this temperature were they -2^7) take the same steps over
// windows of 8192 values of the whole order, counting the row again for each: one row of 262144 with half of it at
// bf16's lowest value 20 us at temperature 0.8, 1125 in windows at 2; with values past 2^7 566.
//
// What bounds it: the steps' latency (the second launch takes 13 to 16 us whatever the rows: 3 for the counts, 3.5 for the
// weights, 3 for the filters and the draw, 3 for the token) and the LDS additions (64 rows of 262144: 9.5 us of
// counting). One row of 262144 takes 18.4 us, 64 rows 24.0, 200 rows of 50001 21.8.
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "common.h"
#include "kernels.h"
#include "sample_batch.h"
#include "sample_row.h"
#include "wave.h"

namespace hyperion::hip {
namespace {

#define HYP_INLINE __attribute__((always_inline))

using namespace sampling;

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

__global__ __launch_bounds__(kThreads) void sample_count_kernel(const uint16_t* __restrict__ logits, uint32_t vocab,
                                                                Chunks chunks, ChunkCounts* __restrict__ counts) {
    __shared__ RowLds s;
    const uint32_t row = blockIdx.x / chunks.n;
    const uint32_t begin = min(vocab, (blockIdx.x - row * chunks.n) * chunks.tokens);
    count_values<0u>(logits + static_cast<size_t>(row) * vocab, begin, min(vocab, begin + chunks.tokens), s);
    store_counts(s, counts[blockIdx.x]);
}

// The same for a whole row, from its chunks: eight bins to a thread, the last ones to the first lanes, a chunk each.
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
    const RowParams prm = row_params(configs[row_at], uniforms[row_at]);

    // 1. Counts by value.
    if constexpr (kSplit) {
        counts += static_cast<size_t>(row_at) * chunks.n;
        sum_counts(counts, chunks.n, s);
    } else {
        count_values<0u>(row, 0u, vocab, s);
    }

    // 2. The drawn value and the token's number among those of that value.
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
    double logprob;
    if (infinite != 0u) {
        // Weight 1 for each, 0 for everything else.
        uint32_t kept = infinite;
        if (prm.top_k != 0u) kept = min(kept, prm.top_k);
        if (prm.top_p != 0.0) kept = min(kept, static_cast<uint32_t>(ceil(prm.top_p * infinite)));
        if (prm.greedy || prm.min_p > 1.0) kept = 1u;
        if (tid == 0u) {
            s.drawn = 0x7F80u;
            s.number = static_cast<uint32_t>(fmin(prm.u * kept, static_cast<double>(kept - 1u)));
        }
        logprob = -log(static_cast<double>(infinite));
        __syncthreads();
    } else {
        uint32_t lead = 0xFFFFFFFFu;
        for (uint32_t w = 0; w < kWaves; ++w) lead = min(lead, s.lead[w]);
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
        bool windowed = lead == kAbove || lead == kBelow || (s.count[kCentreAt] != 0u && s.centre_lo != s.centre_hi);
        if (!windowed && s.count[kBelowAt] != 0u)   // (2^23 times e^-80)
            windowed = !((value_of(fine_bits(lead)) + 128.0) * prm.by_t > 80.0);
        double top = 0.0;
        uint32_t windows = 1u;
        if (windowed) {
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
        // (Written out for either way. For one row of 262144: 19.3 us so, 19.8 with one copy and a test at each step, 22.9
        // with one loop over the steps.)
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
            const uint32_t rank = min(s.rank, kept - 1u);
            over_windows([&](double, uint32_t count) HYP_INLINE {
                if (rank - count >= here) return;
#pragma unroll
                for (uint32_t i = 0; i < kPer; ++i) {
                    if (rank - count < num[i]) {
                        s.drawn = bits_of(first + i);
                        s.number = rank - count;
                        if (!slow) s.bin = first + i;
                    }
                    count += num[i];
                }
            });
            __syncthreads();
            logprob = (value_of(s.drawn) - top) * prm.by_t - log(total);
        };
        if (windowed) find(std::true_type{}); else find(std::false_type{});
    }

    // 3. The token, in the row or in the chunk that holds it: each wave marks the value's places in its stretch, 512
    // tokens a step.
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
                    tokens[row_at] = begin + k * kStep + static_cast<uint32_t>(__builtin_ctz(bits));
                    if (logprobs != nullptr) logprobs[row_at] = static_cast<float>(logprob);
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
