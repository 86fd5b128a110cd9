// Verification of drafted tokens against the target's probabilities, from given uniforms (hyp_verify_batch).
//
// p and q are a row's distributions of the target and of the drafting model: weights w = exp((x - x_max) / T) of the
// tokens that the filters keep, over their sum. The draft x of a row is accepted iff u q(x) < p(x). The first row whose
// draft is not, or a request's last row, draws the next token from max(0, p - q) (from p behind the last draft): the
// first token along the index whose running sum exceeds u times the whole. So the accepted tokens and the drawn one are
// distributed as tokens drawn from p one by one.
//
// Steps, a launch each:
//  1. every row of both models counted by value, in chunks (sample_row.h): the one pass over all logits;
//  2. a workgroup a row: 32 neighbouring values to a thread, their weights, scans of mass and count, what the filters
//     keep. A row is then its largest logit, the kept and the whole mass, the last kept value and the last kept token of
//     that value: a token's p follows from its logit alone. And the probability of the row's draft;
//  3. each request's stop row, by those probabilities, and the sums of max(0, p - q) over tiles of that row;
//  4. a workgroup a request: the tile, then the token in it.
// All weights and sums are fp64; tokens that p does not keep have no weight, so their exponentials are not formed.
//
// A row takes windows of 8192 values instead of its counts (step 2 counts the row again for each, and again for those that a
// filter ends in) where the counts' bins of more than one value matter: a value above 2^7; values next to 0 that hold the
// cut, or weigh enough that their differences of less than 2^-24 do; values below -2^7 that are not negligible, or hold the
// cut. One request of 5 rows past 2^7 takes 180 to 540 us so. Masks go by their own size: 60 % of 576 rows of 262144 at the
// type's lowest value take 123 us, 3.0 ms at temperatures of 1.9 and more when all below -2^7 counted as -2^7.
//
// What bounds it: with many rows the one pass over the logits (64 requests of 1 to 8 rows of 262144, 268 MB: a call 108 us;
// its kernels 60, which is 4.5 TB/s, 23, 17 and 7.4), then the exponentials of the requests that keep most tokens. With few,
// latency: one request of 5 rows takes 22.6 us a call, its kernels 5.8, 8.9, 3.9 and 4.4, where its 4.7 MB are 1 us. (A call's
// time is that of one in a stream of calls, a kernel's that of a traced dispatch.) The instructions of steps 2 to 4 are
// mostly such that all waves of a workgroup issue alike (scans, parameters, borders): with 16 waves each is 16 cycles, so
// they have four (48 requests without a drafting model 72 us with 16, 52 with four). And as the code itself comes from
// memory in a short kernel, loops over a thread's values are kept rolled.
#include <algorithm>
#include <cstdint>

#include "batch.h"
#include "common.h"
#include "sample_row.h"
#include "verify_batch.h"
#include "verify_border.h"
#include "wave.h"

namespace hyperion::hip {
namespace {

#define HYP_INLINE __attribute__((always_inline))

using namespace sampling;

constexpr uint32_t kNone = 0xFFFFFFFFu;
constexpr uint32_t kFew = 256;              // threads of steps 2 to 4
constexpr uint32_t kFewWaves = kFew / 64u;
constexpr uint32_t kTile = 8u * kFew;       // eight consecutive tokens a thread
constexpr uint32_t kLongest = 65024;         // tokens of a chunk: its counts are 16 bits
static_assert((kMaxVocab + kLongest - 1u) / kLongest <= kFew, "a chunk to a thread");

// Nothing above -inf; by the counts; by windows; +inf among the logits.
enum RowKind : uint32_t { kEmpty = 0, kCounted = 1, kWindowed = 2, kInfinite = 3 };

// A row and its filters.
struct alignas(16) RowStat {
    double top, by_t, by_kept, total;   // largest logit, 1 / temperature, 1 / kept mass, mass of all tokens
    float cut;                          // the last value that is kept (NaN: none)
    uint32_t last;                      // the last kept token of that value
    uint32_t kind, unused;
};

struct VerifyParams {
    VerifyArgs a;
    Chunks chunks;
    uint32_t tiles, groups;   // tiles of a row, workgroups of a request in step 3
    // [rows], then those of the drafting model:
    RowStat* stats;
    double* chances;          // the draft's probability
    float* shares;            // ln of its share before the filters
    uint32_t* requests;       // whose row it is, kNone: of no use
    ChunkCounts* counts;      // [chunks.n] each
    double2* sums;            // [requests][tiles]: of max(0, p - q), of p
};

// The request whose rows hold row t < row_start[n]: the last r < n with row_start[r] <= t, by every wave for itself.
__device__ __forceinline__ uint32_t request_of(const uint32_t* row_start, uint32_t n, uint32_t t) {
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t lo = 0u, size = n;
    while (size > 1u) {
        const uint32_t step = (size + 63u) / 64u;
        const uint32_t at = lane * step;
        const uint64_t at_or_before = __ballot(at < size && row_start[lo + at] <= t);
        const uint32_t k = at_or_before != 0u ? 63u - static_cast<uint32_t>(__builtin_clzll(at_or_before)) : 0u;
        lo += k * step;
        size = min(step, size - k * step);
    }
    return lo;
}

__device__ __forceinline__ const uint16_t* logits_of(const VerifyArgs& a, uint32_t index) {
    return index < a.rows ? a.logits + static_cast<size_t>(index) * a.vocab
                          : a.draft_logits + static_cast<size_t>(index - a.rows) * a.vocab;
}

// ---- 1. counts ----------------------------------------------------------------------------------

// Rows that come from memory are waited for: with all of a chunk's loads on their way at once the counts of 64 requests'
// 268 MB take 60 us, 68 otherwise. What a cache holds is counted faster while the next comes in. A whole call in turn over
// 1, 3 and 8 sets of inputs, without and with all loads first: 42 MB 38.3, 39.3, 43.6 and 38.6, 39.1, 42.9 us; 63 MB 46.3,
// 46.9, 55.0 and 47.5, 48.1, 53.4; 70 MB 47.7, 48.4, 56.0 and 49.3, 49.6, 54.8; 125 MB 49.2, 58.3, 61.4 and 51.3, 55.0, 57.8.
// A step's logits are just written, and the rest of the step lies between two calls.
constexpr uint64_t kCached = 1ull << 26;   // bytes
constexpr uint32_t kChunkLoads = 8;
static_assert(kLongest <= kChunkLoads * 8u * kThreads, "a chunk's loads");
template <uint32_t kAhead>
__global__ __launch_bounds__(kThreads) void verify_count_kernel(VerifyParams p) {
    __shared__ RowLds s;
    const VerifyArgs& a = p.a;
    const uint32_t index = blockIdx.x / p.chunks.n;
    const uint32_t chunk = blockIdx.x - index * p.chunks.n;
    // Rows of no request, and the drafting model's behind which nothing was drafted, are of no use.
    const bool draft = index >= a.rows;
    const uint32_t row = draft ? index - a.rows : index;
    uint32_t request = kNone;
    if (row < a.row_start[a.requests]) {
        request = request_of(a.row_start, a.requests, row);
        if (draft && row + 1u >= a.row_start[request + 1u]) request = kNone;
    }
    if (chunk == 0u && threadIdx.x == 0u) p.requests[index] = request;
    if (request == kNone) return;
    const uint32_t begin = min(a.vocab, chunk * p.chunks.tokens);
    count_values<kAhead>(logits_of(a, index), begin, min(a.vocab, begin + p.chunks.tokens), s);
    store_counts(s, p.counts[blockIdx.x]);
}

// ---- 2. filters ---------------------------------------------------------------------------------

// A value that all lanes have, in scalar registers.
__device__ __forceinline__ double scalar(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint64_t lo = from_lane(static_cast<uint32_t>(b), 0u), hi = from_lane(static_cast<uint32_t>(b >> 32), 0u);
    return __builtin_bit_cast(double, lo | hi << 32);
}

__device__ __forceinline__ float logit_of(uint32_t bits) { return __uint_as_float(bits << 16); }
// Whether the filters keep a token (a NaN is above nothing, -inf above no cut).
__device__ __forceinline__ bool keeps(const RowStat& r, float x, uint32_t token) {
    return x > r.cut || (x == r.cut && token <= r.last);
}
// The probability of a token from its logit.
__device__ __forceinline__ double probability(const RowStat& r, uint32_t bits, uint32_t token) {
    const float x = logit_of(bits);
    if (!keeps(r, x, token)) return 0.0;
    return r.kind == kInfinite ? r.by_kept : exp_below((static_cast<double>(x) - r.top) * r.by_t) * r.by_kept;
}

// ln of a token's share of the mass before the filters.
__device__ __forceinline__ float log_share(const RowStat& r, uint32_t bits) {
    if (r.kind == kEmpty) return -__builtin_huge_valf();
    const double gap = r.kind == kInfinite ? 0.0 : (value_of(bits) - r.top) * r.by_t;
    return static_cast<float>(gap - log(r.total));
}

// Inclusive sums in thread order and the whole. (Every wave has left `waves`; a call has a barrier at its end.)
template <typename T>
struct Scan {
    T incl, all;
};
template <typename T>
__device__ __forceinline__ Scan<T> few_scan(T v, T* waves) {
    const uint32_t wave = threadIdx.x >> 6;
    T incl;
    if constexpr (sizeof(T) == 8u) incl = wave_incl64(v); else incl = wave_incl(v);
    if ((threadIdx.x & 63u) == 63u) waves[wave] = incl;
    __syncthreads();
    T before = 0, all = 0;
#pragma unroll
    for (uint32_t w = 0; w < kFewWaves; ++w) {
        if (w == wave) before = all;
        all += waves[w];
    }
    __syncthreads();
    return {before + incl, all};
}
__device__ __forceinline__ uint32_t few_min(uint32_t v, uint32_t* waves) {
    v = from_lane(wave_scan(v, kNone, [](uint32_t a, uint32_t b) { return min(a, b); }), 63u);
    if ((threadIdx.x & 63u) == 0u) waves[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kFewWaves; ++w) v = min(v, waves[w]);
    __syncthreads();
    return v;
}

// The 32 bins of a thread, neighbours in one binade and so equally far apart, in an order that gives the threads' in
// descending order of values.
constexpr uint32_t kBinsEach = kWindow / kFew;
__device__ __forceinline__ uint32_t bin_of(uint32_t tid, uint32_t i) {
    return tid < kFew / 2u ? kFine - 1u - (kBinsEach * tid + i) : kBinsEach * tid + i;
}
__device__ __forceinline__ uint32_t bits_of_bin(uint32_t tid, uint32_t i) {
    const uint32_t at = bin_of(tid, i);
    return (at & 0xFFFu) + kLow + ((at & 0x1000u) << 3);
}
static_assert(2u * kFine == kWindow && kFine == 0x1000u && 128u % kBinsEach == 0u, "a thread's fine values");

// e^((x - top) by_t) of those: the first one's, and from one to the next a factor, so that each is right to a few fp64
// roundings. (An exponential for each took five times as long.) The largest value's is 1 exactly, as min-p may be; those
// above it mean nothing.
struct Weights {
    double w, step;
    uint32_t at_top;   // which of them is the largest value
    __device__ __forceinline__ Weights(uint32_t tid, double top, double by_t) : w(0.0), step(0.0) {
        const double x = value_of(bits_of_bin(tid, 0u));
        const double apart = x - value_of(bits_of_bin(tid, 1u));
        const double which = (x - top) / apart;
        at_top = which >= 0.0 && which < kBinsEach ? static_cast<uint32_t>(which) : kBinsEach;
#pragma unroll 1
        for (uint32_t k = 0; k < 2u; ++k) {   // (the code of one exponential)
            const double v = exp_below((k == 0u ? x - top : -apart) * by_t);
            if (k == 0u) w = v; else step = v;
        }
        if (at_top == 0u) w = 1.0;
    }
    __device__ __forceinline__ void next(uint32_t i) { w = i + 1u == at_top ? 1.0 : w * step; }   // from i to the one after
};

constexpr uint32_t kSlots = 1u + kBinsEach;   // values of a thread: those next to 0 (thread 128's), its bins
constexpr uint32_t kCentreThread = kFew / 2u;
constexpr uint32_t kRow = kFew + 1u;            // (four lanes that store slots of one thread do not meet in a bank)

// What a row has beside its fine values.
struct Others {
    uint32_t infinite, centre, above, below;   // tokens
    uint32_t centre_lo, centre_hi;             // least and largest place of the values next to 0
    uint32_t below_bits;                       // of the largest below
    uint32_t lead;                             // kBinsEach * thread + i of the first bin with a token, kNone: none
};

struct alignas(16) FilterLds {
    double mass[kFewWaves], kept;        // ..., mass of the kept tokens
    uint32_t word[kFewWaves];
    uint32_t count[kSlots * kRow];       // of slot i of thread t at i * kRow + t; by value, of a window
    alignas(16) uint32_t others[kFewWaves][8];   // a wave's
    uint32_t keep, redo;
    uint32_t cut, number, whole;         // bits of the last kept value, the last kept token's number there, are all kept
    uint32_t last;
    // Of a row by windows: each one's.
    double window_mass[kWindows];
    uint32_t window_count[kWindows];
    uint32_t window_light;   // a bit each: min-p drops some
};

// The filters of a row from its counts in s: leaves s.kept, s.cut, s.number, s.whole and the mass of all tokens. False: the
// row takes windows. (A call has a barrier at its end.)
__device__ __forceinline__ bool filter_counts(const RowParams& prm, double top, const Others& others, FilterLds& s,
                                              double& total) {
    const uint32_t tid = threadIdx.x;
    const uint32_t lane = tid & 63u;
    const uint32_t centre = s.count[tid];
    double centre_weight = 0.0, sum = 0.0;
    uint32_t here = centre;
    bool light = false;   // min-p may drop some
    if (centre != 0u) {
        centre_weight = exp_below((value_of(bits_at(others.centre_lo)) - top) * prm.by_t);
        sum = centre * centre_weight;
        light = may_be_light(centre_weight, prm.min_p);
    }
    {
        Weights e(tid, top, prm.by_t);
#pragma unroll 1
        for (uint32_t base = 0; base < kBinsEach; base += 8u) {
            uint32_t n[8];
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) n[i] = s.count[(base + i + 1u) * kRow + tid];
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) {
                sum += n[i] * e.w;
                here += n[i];
                light = light || (n[i] != 0u && may_be_light(e.w, prm.min_p));
                e.next(base + i);
            }
        }
    }
    const Scan<double> mass_at = few_scan(sum, s.mass);
    const Scan<uint32_t> count_at = few_scan(here, s.word);
    const double mass_before = mass_at.incl - sum;
    const uint32_t count_before = count_at.incl - here;
    total = scalar(mass_at.all);
    // Tokens below -2^7 weigh next to nothing; masked ones nothing at all, so that it is the same whether they are kept.
    const bool masked = others.below != 0u && (top - value_of(others.below_bits)) * prm.by_t > 750.0;   // (e^-750 is 0)
    const uint32_t below = masked ? 0u : others.below;
    const uint32_t all = count_at.all + below;
    uint32_t kept = all;
    if (prm.top_k != 0u) kept = min(kept, prm.top_k);
    // The values of the thread of lane `from`, a slot to a lane.
    const auto spread = [&](uint32_t from) HYP_INLINE {
        OneValue o{0u, 0u, 0u, 0.0, 0.0};
        const uint32_t thread = (tid & ~63u) + from;
        if (lane < kSlots) {
            o.n = s.count[lane * kRow + thread];
            o.bits = lane == 0u ? bits_at(others.centre_lo & 0xFFFFu) : bits_of_bin(thread, lane - 1u);
            if (o.n != 0u) o.w = exp_below((value_of(o.bits) - top) * prm.by_t);
        }
        const double m = o.n * o.w;
        const uint64_t before = __builtin_bit_cast(uint64_t, mass_before);
        const uint64_t lo = from_lane(static_cast<uint32_t>(before), from);
        const uint64_t hi = from_lane(static_cast<uint32_t>(before >> 32), from);
        o.mass = __builtin_bit_cast(double, lo | hi << 32) + (wave_incl64(m) - m);
        o.before = from_lane(count_before, from) + (wave_incl(o.n) - o.n);
        return o;
    };
    if (prm.top_p != 0.0 || prm.min_p != 0.0) {
        const double enough = prm.top_p * total;
        const bool by_mass = prm.top_p != 0.0;
        const uint64_t maybe = __ballot(here != 0u && (light || (by_mass && may_be_past(mass_at.incl, enough))));
        const uint32_t border = wave_border(maybe, by_mass, enough, prm.min_p, spread);
        if (lane == 0u && border != kNone) atomicMin(&s.keep, border);
        __syncthreads();
        kept = min(kept, s.keep);
    }
    if (below != 0u) {
        // Nothing there weighs enough for top-p; min-p drops it unless it is tiny: e^-80 is above 2^-116.
        if (prm.min_p != 0.0) kept = min(kept, count_at.all);
        if ((kept > count_at.all && kept != all) || (prm.min_p != 0.0 && prm.min_p < 0x1p-110)) return false;
    }
    kept = prm.greedy ? 1u : max(kept, 1u);
    if (centre != 0u && others.centre_lo != others.centre_hi)   // several values next to 0
        s.redo = kept - 1u - count_before < centre || centre * centre_weight * prm.by_t > 0x1p-30 * total;
    const uint64_t holds = __ballot(kept - 1u - count_before < here);
    if (holds != 0u) {
        const OneValue o = spread(static_cast<uint32_t>(__builtin_ctzll(holds)));
        if (kept - 1u - o.before < o.n) {
            s.kept = o.mass + (kept - o.before) * o.w;
            s.cut = o.bits;
            s.number = kept - 1u - o.before;
            s.whole = kept - o.before == o.n;
        }
    }
    if (kept == all && below != 0u && tid == 0u) {   // everything
        s.kept = total;
        s.cut = 0xFF7Fu;
        s.number = 0u;
        s.whole = 1u;
    }
    __syncthreads();
    return s.redo == 0u;
}

// The same for a row by windows. (A call has a barrier at its end.)
__device__ __forceinline__ void filter_windows(const uint16_t* row, uint32_t vocab, const RowParams& prm, RowStat& r,
                                               FilterLds& s) {
    const uint32_t tid = threadIdx.x;
    uint32_t best = kNone, held = 0u, windows = 0u;
    for_tokens(row, 0u, vocab, tid, kFew, [&](uint32_t, uint32_t b) HYP_INLINE {
        b = plain_bits(b);
        if (!finite_bits(b)) return;
        best = min(best, place_of(b));
        held |= 1u << (place_of(b) / kWindow);
    });
    best = few_min(best, s.word);
    for (uint32_t w = 0; w < kWindows; ++w)
        if (few_min((held >> w) & 1u ? 0u : 1u, s.word) == 0u) windows |= 1u << w;
    r.top = scalar(value_of(bits_at(best)));
    for (uint32_t k = best / kWindow + 1u; k < kWindows; ++k)   // (e^-750 is 0: the same whether they are kept)
        if ((value_of(bits_at(k * kWindow)) - r.top) * prm.by_t < -750.0) windows &= ~(1u << k);
    if (tid == 0u) s.window_light = 0u;
    uint32_t kept = kNone, counted = kNone;
    // Step 0: the mass and number of all tokens; 1: what top-p and min-p keep; 2: the last kept one.
#pragma unroll 1
    for (uint32_t step = 0; step < 3u; ++step) {
        double mass_all = 0.0;
        uint32_t count_all = 0u;
#pragma unroll 1
        for (uint32_t k = 0; k < kWindows; ++k) {
            if (((windows >> k) & 1u) == 0u) continue;
            const uint32_t window = k * kWindow;
            const double enough = prm.top_p * r.total;
            // Those that a filter ends in or that hold the last kept token are looked into, the others have their sums.
            const bool ends = (prm.top_p != 0.0 && mass_all + s.window_mass[k] > enough) || ((s.window_light >> k) & 1u) != 0u;
            if ((step == 1u && !ends) || (step == 2u && kept - 1u - count_all >= s.window_count[k])) {
                mass_all += s.window_mass[k];
                count_all += s.window_count[k];
                continue;
            }
            __syncthreads();
            if (counted != k) {
                for (uint32_t i = tid; i < kWindow; i += kFew) s.count[i] = 0u;
                __syncthreads();
                for_tokens(row, 0u, vocab, tid, kFew, [&](uint32_t, uint32_t b) HYP_INLINE {
                    b = plain_bits(b);
                    const uint32_t d = place_of(b) - window;
                    if (finite_bits(b) && d < kWindow) atomicAdd(&s.count[d], 1u);
                });
                __syncthreads();
                counted = k;
            }
            const auto weight = [&](uint32_t i) HYP_INLINE {
                return exp_below((value_of(bits_at(window + kBinsEach * tid + i)) - r.top) * r.by_t);
            };
            double sum = 0.0;
            uint32_t here = 0u;
            bool light = false;
#pragma unroll 1
            for (uint32_t i = 0; i < kBinsEach; ++i) {
                const uint32_t n = s.count[kBinsEach * tid + i];
                if (n == 0u) continue;
                const double w = weight(i);
                sum += n * w;
                light = light || w < prm.min_p;
                here += n;
            }
            const Scan<double> mass_at = few_scan(sum, s.mass);
            const Scan<uint32_t> count_at = few_scan(here, s.word);
            double mass = mass_all + (mass_at.incl - sum);
            uint32_t count = count_all + (count_at.incl - here);
            if (step == 0u) {
                if (light) atomicOr(&s.window_light, 1u << k);
                if (tid == 0u) {
                    s.window_mass[k] = mass_at.all;
                    s.window_count[k] = count_at.all;
                }
            }
            if (step == 1u && here != 0u) {
                bool open = true;
#pragma unroll 1
                for (uint32_t i = 0; i < kBinsEach && open; ++i) {
                    const uint32_t n = s.count[kBinsEach * tid + i];
                    if (n == 0u) continue;
                    const double w = weight(i);
                    const bool dropped = w < prm.min_p;
                    const bool full = prm.top_p != 0.0 && n * w > enough - mass;
                    open = !dropped && !full;
                    if (open) count += n;
                    else if (!dropped && enough > mass) count += min(n, static_cast<uint32_t>(ceil((enough - mass) / w)));
                    mass += n * w;
                }
                if (!open) atomicMin(&s.keep, count);
            }
            if (step == 2u && kept - 1u - count < here) {
#pragma unroll 1
                for (uint32_t i = 0; i < kBinsEach; ++i) {
                    const uint32_t n = s.count[kBinsEach * tid + i];
                    const double w = n != 0u ? weight(i) : 0.0;
                    if (kept - 1u - count < n) {
                        s.kept = mass + (kept - count) * w;
                        s.cut = bits_at(window + kBinsEach * tid + i);
                        s.number = kept - 1u - count;
                        s.whole = kept - count == n;
                    }
                    mass += n * w;
                    count += n;
                }
            }
            mass_all += mass_at.all;
            count_all += count_at.all;
            if (step == 2u) break;
            if (step == 1u) {
                __syncthreads();
                if (s.keep != kNone) break;
            }
        }
        __syncthreads();
        if (step == 0u) {
            r.total = scalar(mass_all);
            kept = count_all;
            if (prm.top_k != 0u) kept = min(kept, prm.top_k);
            if (tid == 0u) s.keep = kNone;
        } else if (step == 1u) {
            kept = min(kept, s.keep);
            kept = prm.greedy ? 1u : max(kept, 1u);
        }
        __syncthreads();
    }
}

// The index of the number-th token of value `bits` among the tokens [begin, end) of a row, in s.last. Each wave counts the
// value's places in its stretch, 512 tokens a step, two to an instruction. (A call has a barrier at its end.)
__device__ __forceinline__ void find_last(const uint16_t* row, uint32_t begin, uint32_t end, uint32_t bits, uint32_t number,
                                          FilterLds& s) {
    typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = threadIdx.x >> 6;
    constexpr uint32_t kStep = 512u, kSteps = 16u;
    const uint32_t pattern = bits | bits << 16;
    const uint32_t mask = bits == 0u ? 0x7FFF7FFFu : 0xFFFFFFFFu;   // (-0 is +0)
#pragma unroll 1
    for (uint32_t base = begin; base < end; base += kFewWaves * kSteps * kStep) {
        const uint32_t stop = min(end, base + kFewWaves * kSteps * kStep);
        const uint32_t steps = (stop - base + kFewWaves * kStep - 1u) / (kFewWaves * kStep);
        const uint32_t first = base + wave * steps * kStep + 8u * lane;   // the lane's, of the first step
        const uint32_t room = first < stop ? stop - first : 0u;
        const uint32_t whole = room < 8u ? 0u : min(steps, (room - 8u) / kStep + 1u);   // steps with all eight tokens
        uint64_t found = 0u;   // the lane's of each step, four bits to one
        uint32_t mine = 0u;
#pragma unroll 1
        for (uint32_t k = 0; k < steps; k += 4u) {
            uint32_t w[4][4];
#pragma unroll
            for (uint32_t j = 0; j < 4u; ++j) {
                if (k + j < whole) {
                    __builtin_memcpy(w[j], row + first + (k + j) * kStep, 16);
                } else {
#pragma unroll
                    for (uint32_t i = 0; i < 4u; ++i) w[j][i] = ~pattern;
                }
            }
            uint32_t four = 0u;
#pragma unroll
            for (uint32_t j = 0; j < 4u; ++j) {
                u16x2_t same = {0, 0};
#pragma unroll
                for (uint32_t i = 0; i < 4u; ++i)
                    same += __builtin_elementwise_sub_sat(u16x2_t{1, 1},
                                                          __builtin_bit_cast(u16x2_t, (w[j][i] ^ pattern) & mask));
                const uint32_t n = static_cast<uint32_t>(same.x) + same.y;
                four |= n << (4u * j);
                mine += n;
            }
            found |= static_cast<uint64_t>(four) << (4u * k);
        }
        if (whole < steps && whole * kStep < room) {   // the row's last tokens
            uint32_t n = 0u;
            for (uint32_t i = first + whole * kStep; i < stop; ++i) n += plain_bits(row[i]) == bits ? 1u : 0u;
            found |= static_cast<uint64_t>(n) << (4u * whole);
            mine += n;
        }
        const uint32_t wave_all = wave_sum(mine);
        if (lane == 0u) s.word[wave] = wave_all;
        __syncthreads();
        uint32_t before = 0u, all = 0u;
#pragma unroll
        for (uint32_t w = 0; w < kFewWaves; ++w) {
            if (w == wave) before = all;
            all += s.word[w];
        }
        __syncthreads();
        if (number >= all) {
            number -= all;
            continue;
        }
        uint32_t left = number - before;   // (wraps past the holder)
        if (left < wave_all) {
#pragma unroll 1
            for (uint32_t k = 0; k < steps; ++k) {
                const uint32_t n = static_cast<uint32_t>(found >> (4u * k)) & 15u;
                if (__ballot(n != 0u) == 0u) continue;
                const uint32_t incl = wave_incl(n);
                const uint32_t step = from_lane(incl, 63u);
                if (left < step) {
                    if (left - (incl - n) < n) {
                        const uint32_t from = first + k * kStep;
                        uint32_t b[8], places = 0u;
#pragma unroll
                        for (uint32_t i = 0; i < 8u; ++i) b[i] = row[min(from + i, stop - 1u)];   // (copies: behind it)
#pragma unroll
                        for (uint32_t i = 0; i < 8u; ++i) places |= plain_bits(b[i]) == bits ? 1u << i : 0u;
                        for (uint32_t skip = left - (incl - n); skip != 0u; --skip) places &= places - 1u;
                        s.last = from + static_cast<uint32_t>(__builtin_ctz(places));
                    }
                    break;
                }
                left -= step;
            }
        }
        break;
    }
    __syncthreads();
}

__global__ __launch_bounds__(kFew) void verify_filter_kernel(VerifyParams p) {
    __shared__ FilterLds s;
    const VerifyArgs& a = p.a;
    const uint32_t index = blockIdx.x;
    const uint32_t tid = threadIdx.x;
    const uint32_t lane = tid & 63u;
    const uint32_t row_at = index < a.rows ? index : index - a.rows;
    const uint16_t* const row = logits_of(a, index);
    const ChunkCounts* const counts = p.counts + static_cast<size_t>(index) * p.chunks.n;
    const uint32_t request = p.requests[index];
    const uint32_t x = row_at + 1u < a.rows ? a.ids[row_at + 1u] : kNone;   // the row's draft
    if (tid == 0u) {
        s.redo = 0u;
        s.keep = kNone;
    }
    __syncthreads();
    // The row's counts from its chunks', the other bins a chunk to a thread.
    {
        uint32_t sum[4] = {}, least[4] = {kNone, kNone, kNone, kNone};
        if (tid < p.chunks.n) {
            const ChunkCounts& c = counts[tid];
            sum[0] = c.infinite;
            sum[1] = c.count[kCentreAt];
            sum[2] = c.count[kAboveAt];
            sum[3] = c.count[kBelowAt];
            least[0] = c.centre_lo;
            least[1] = ~c.centre_hi;
            least[2] = c.below;
        }
        // Eight bins in each quarter of them to a thread, which then go to the threads that have them.
        uint32_t n[kBinsEach] = {};
#pragma unroll 1
        for (uint32_t c = 0; c < p.chunks.n; c += 4u) {
            uint4 v[4][kBinsEach / 8u];
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) {
                const uint4* const from = reinterpret_cast<const uint4*>(counts[c + k].count) + tid;
#pragma unroll
                for (uint32_t q = 0; q < kBinsEach / 8u; ++q) {
                    v[k][q] = make_uint4(0u, 0u, 0u, 0u);
                    if (c + k < p.chunks.n) v[k][q] = from[kFew * q];
                }
            }
            __builtin_amdgcn_sched_barrier(0);   // (all of them on their way before the first is waited for)
            if (c == 0u) {   // (and those above with them, not where they are used)
#pragma unroll
                for (uint32_t i = 0; i < 4u; ++i) asm volatile("" : "+v"(sum[i]), "+v"(least[i]));
            }
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) {
#pragma unroll
                for (uint32_t q = 0; q < kBinsEach / 8u; ++q) {
                    const uint32_t word[4] = {v[k][q].x, v[k][q].y, v[k][q].z, v[k][q].w};
#pragma unroll
                    for (uint32_t j = 0; j < 4u; ++j) {
                        n[8u * q + 2u * j] += word[j] & 0xFFFFu;
                        n[8u * q + 2u * j + 1u] += word[j] >> 16;
                    }
                }
            }
        }
#pragma unroll
        for (uint32_t q = 0; q < kBinsEach / 8u; ++q) {
            const uint32_t bin = 8u * (kFew * q + tid);
            // (its place in descending order: positive values are stored ascending)
            const uint32_t place = bin < kFine ? kFine - 1u - bin : bin;
            const uint32_t thread = place / kBinsEach, slot = 1u + place % kBinsEach;
            uint32_t* const to = &s.count[slot * kRow + thread];
            uint32_t lead = kNone;
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) {
                to[(q < kBinsEach / 16u ? -static_cast<int>(i) : static_cast<int>(i)) * static_cast<int>(kRow)] = n[8u * q + i];
                if (n[8u * q + i] != 0u && (lead == kNone || q < kBinsEach / 16u))
                    lead = q < kBinsEach / 16u ? place - i : place + i;
            }
            least[3] = min(least[3], lead);
        }
        // (By the wave: with additions to one word in LDS by several lanes this took 4000 cycles.)
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            sum[i] = wave_sum(sum[i]);
            least[i] = from_lane(wave_scan(least[i], kNone, [](uint32_t x_, uint32_t y_) { return min(x_, y_); }), 63u);
        }
        if (lane == 0u) {
            uint4* const to = reinterpret_cast<uint4*>(s.others[tid >> 6]);
            to[0] = make_uint4(sum[0], sum[1], sum[2], sum[3]);
            to[1] = make_uint4(least[0], least[1], least[2], least[3]);
        }
    }
    if (request == kNone) return;
    RowParams prm = row_params((index < a.rows ? a.configs : a.draft_configs)[request], 0.0f);
    prm.by_t = scalar(prm.by_t);
    prm.top_p = scalar(prm.top_p);
    prm.min_p = scalar(prm.min_p);
    __syncthreads();
    Others others;
    {
        uint32_t sum[4] = {}, least[4] = {kNone, kNone, kNone, kNone};
#pragma unroll
        for (uint32_t w = 0; w < kFewWaves; ++w)
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) {
                sum[i] += s.others[w][i];
                least[i] = min(least[i], s.others[w][4u + i]);
            }
        others = {from_lane(sum[0], 0u),   from_lane(sum[1], 0u),    from_lane(sum[2], 0u),   from_lane(sum[3], 0u),
                  from_lane(least[0], 0u), ~from_lane(least[1], 0u), from_lane(least[2], 0u), from_lane(least[3], 0u)};
    }
    s.count[tid] = tid == kCentreThread ? others.centre : 0u;   // (this thread's alone)
    RowStat r{};
    r.by_t = prm.by_t;
    r.cut = __builtin_nanf("");
    if (others.infinite != 0u) {
        // Weight 1 for each, 0 for everything else.
        const uint32_t infinite = others.infinite;
        uint32_t kept = infinite;
        if (prm.top_k != 0u) kept = min(kept, prm.top_k);
        if (prm.top_p != 0.0) kept = min(kept, static_cast<uint32_t>(ceil(prm.top_p * infinite)));
        if (prm.greedy || prm.min_p > 1.0) kept = 1u;
        if (tid == 0u) {
            s.kept = kept;
            s.cut = 0x7F80u;
            s.number = kept - 1u;
            s.whole = kept == infinite;
        }
        r.kind = kInfinite;
        r.total = infinite;
        __syncthreads();
    } else if (others.lead != kNone || others.centre != 0u || others.above != 0u || others.below != 0u) {
        const uint32_t lead = others.lead;
        const bool next_to_0 = others.centre != 0u && lead >= kFine;   // the largest
        bool counted = others.above == 0u && (next_to_0 ? others.centre_lo == others.centre_hi : lead != kNone);
        r.top = scalar(value_of(next_to_0 ? bits_at(others.centre_lo)
                                          : bits_of_bin((lead / kBinsEach) % kFew, lead % kBinsEach)));
        // (2^23 times e^-80 is below a rounding.)
        if (counted && others.below != 0u) counted = (r.top - value_of(others.below_bits)) * prm.by_t > 80.0;
        if (counted) counted = filter_counts(prm, r.top, others, s, r.total);
        r.kind = counted ? kCounted : kWindowed;
        if (!counted) filter_windows(row, a.vocab, prm, r, s);
    }
    if (r.kind != kEmpty) {
        r.by_kept = 1.0 / s.kept;
        r.cut = logit_of(s.cut);
        r.last = a.vocab;
        if (s.whole == 0u) {   // some of the last kept value's tokens are dropped
            uint32_t number = s.number, begin = 0u, end = a.vocab;
            if (r.kind == kCounted) {
                const uint32_t t = s.cut - kLow;   // (the place of its count, as count_values has it)
                const uint32_t at = (t & 0x7000u) == 0u ? (t & 0xFFFu) | ((t >> 3) & 0x1000u) : kCentreAt;
                begin = min(a.vocab, find_chunk(counts, p.chunks.n, at, number) * p.chunks.tokens);
                end = min(a.vocab, begin + p.chunks.tokens);
            }
            find_last(row, begin, end, s.cut, number, s);
            r.last = s.last;
        }
    }
    // The draft of a target's row follows every row but a request's last (whose next row is another request's).
    if (tid == 0u) {
        p.stats[index] = r;
        const bool there = x < a.vocab;
        const uint32_t bits = there ? row[x] : 0u;
        p.chances[index] = there ? probability(r, bits, x) : 0.0;
        if (index < a.rows) p.shares[index] = there ? log_share(r, bits) : 0.0f;
    }
}

// ---- 3, 4. the stop row and its draw ------------------------------------------------------------

__device__ __forceinline__ double uniform_of(float u) {   // as a draw takes it
    return u > 0.0f ? static_cast<double>(fminf(u, 0x1.fffffep-1f)) : 0.0;
}

// Where a request stops: the first row whose draft is not accepted, or the last.
struct Stop {
    uint32_t first, rows, accepted;
    [[nodiscard]] __device__ uint32_t row() const { return first + accepted; }
    [[nodiscard]] __device__ bool rejects() const { return accepted + 1u < rows; }
};

// By every wave for itself.
__device__ __forceinline__ Stop find_stop(const VerifyParams& p, uint32_t request) {
    const VerifyArgs& a = p.a;
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t first = min(a.row_start[request], a.rows);
    const uint32_t end = min(a.row_start[request + 1u], a.rows);
    const uint32_t rows = end > first ? end - first : 0u;
    uint32_t accepted = rows != 0u ? rows - 1u : 0u;
#pragma unroll 1
    for (uint32_t base = 0; base + 1u < rows; base += 64u) {
        const uint32_t i = base + lane;
        bool falls = false;
        if (i + 1u < rows) {
            const uint32_t row = first + i;
            const double q = a.draft_logits != nullptr ? p.chances[a.rows + row] : 1.0;
            falls = !(uniform_of(a.uniforms[row]) * q < p.chances[row]);   // (a draft outside the vocabulary: 0 < 0)
        }
        const uint64_t fallen = __ballot(falls);
        if (fallen != 0u) {
            accepted = base + static_cast<uint32_t>(__builtin_ctzll(fallen));
            break;
        }
    }
    return {first, rows, accepted};
}

// e^x of many x <= 0: 2^(n / 64) e^r with |r| <= ln 2 / 128, the first by a table, the series to r^5 (the rest is below
// 2^-54). (15 instructions where exp_below takes 25: a request's whole vocabulary goes through it, without filters.)
constexpr uint32_t kPowers = 64;
struct Powers {
    double p[kPowers];   // 2^(j / 64) / 2
    __device__ __forceinline__ void fill() {   // (before a barrier)
        const uint32_t j = threadIdx.x;
        if (j < kPowers) p[j] = exp_below(-0x1.62e42fefa39efp-7 * static_cast<double>(kPowers - j));
    }
    __device__ __forceinline__ double exp(double x) const {
        x = fmax(x, -1100.0);
        const double n = __builtin_rint(x * 0x1.71547652b82fep+6);
        const double r = __builtin_fma(n, -0x1.abc9e3b39803fp-62, __builtin_fma(n, -0x1.62e42fefa39efp-7, x));
        const int k = static_cast<int>(n);
        double y = __builtin_fma(r, 1.0 / 120.0, 1.0 / 24.0);
        y = __builtin_fma(y, r, 1.0 / 6.0);
        y = __builtin_fma(y, r, 0.5);
        y = __builtin_fma(y, r, 1.0);
        y = __builtin_fma(y, r, 1.0);
        return __builtin_amdgcn_ldexp(y * p[k & 63], (k >> 6) + 1);
    }
};

// max(0, p - q) and p of tokens of the stop row.
struct Rest {
    const uint16_t* logits;
    const uint16_t* draft_logits;   // null: q is 1 at `without` and 0 elsewhere
    RowStat p, q;
    uint32_t without, vocab;
    __device__ __forceinline__ Rest(const VerifyParams& v, const Stop& stop)
        : logits(v.a.logits + static_cast<size_t>(stop.row()) * v.a.vocab), draft_logits(nullptr), p(v.stats[stop.row()]), q{},
          without(kNone), vocab(v.a.vocab) {
        if (!stop.rejects()) return;
        if (v.a.draft_logits != nullptr) {
            draft_logits = v.a.draft_logits + static_cast<size_t>(stop.row()) * vocab;
            q = v.stats[v.a.rows + stop.row()];
        } else {
            without = v.a.ids[stop.row() + 1u];
        }
    }
    static __device__ __forceinline__ double chance(const RowStat& r, const Powers& powers, float x) {   // of a token that r keeps
        return r.kind == kInfinite ? r.by_kept : powers.exp((static_cast<double>(x) - r.top) * r.by_t) * r.by_kept;
    }
    // f(k, max(0, p - q), p) for the tokens begin + k, k < 8, that p keeps.
    template <typename F>
    __device__ __forceinline__ void each(const Powers& powers, uint32_t begin, F&& f) const {
        Eight x, y;
        if (begin + 8u <= vocab) {
            __builtin_memcpy(&x, logits + begin, 16);
            if (draft_logits != nullptr) __builtin_memcpy(&y, draft_logits + begin, 16);
        } else {
            for (uint32_t k = 0; k < 8u; ++k) {
                const bool there = begin + k < vocab;
                x.v[k] = there ? logits[begin + k] : 0x7FFFu;   // (no number)
                y.v[k] = there && draft_logits != nullptr ? draft_logits[begin + k] : 0x7FFFu;
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < 8u; ++k) {
            const float l = logit_of(x.v[k]);
            if (!keeps(p, l, begin + k)) continue;
            const double here = chance(p, powers, l);
            double rest = here;
            if (draft_logits != nullptr) {
                const float d = logit_of(y.v[k]);
                if (keeps(q, d, begin + k)) rest = fmax(0.0, here - chance(q, powers, d));
            }
            if (begin + k == without) rest = 0.0;
            f(k, rest, here);
        }
    }
};

// The sums of max(0, p - q) and of p over the tiles of each request's stop row: `groups` workgroups to each.
__global__ __launch_bounds__(kFew) void verify_sum_kernel(VerifyParams p) {
    __shared__ double waves[2][kFewWaves];
    __shared__ Powers powers;
    const uint32_t tid = threadIdx.x;
    const uint32_t request = blockIdx.x / p.groups;
    powers.fill();
    const Stop stop = find_stop(p, request);
    if (stop.rows == 0u) return;
    const Rest rest(p, stop);
    __syncthreads();
#pragma unroll 1
    for (uint32_t tile = blockIdx.x - request * p.groups; tile < p.tiles; tile += p.groups) {
        double r_sum = 0.0, p_sum = 0.0;
        rest.each(powers, tile * kTile + 8u * tid, [&](uint32_t, double r, double here) HYP_INLINE {
            r_sum += r;
            p_sum += here;
        });
        const bool some = __ballot(p_sum != 0.0) != 0u;
        if (some) {
            r_sum = wave_incl64(r_sum);
            p_sum = wave_incl64(p_sum);
        }
        __syncthreads();
        if ((tid & 63u) == 63u) {
            waves[0][tid >> 6] = r_sum;
            waves[1][tid >> 6] = p_sum;
        }
        __syncthreads();
        if (tid == 0u) {
            double2 sum = make_double2(0.0, 0.0);
#pragma unroll
            for (uint32_t w = 0; w < kFewWaves; ++w) {
                sum.x += waves[0][w];
                sum.y += waves[1][w];
            }
            p.sums[static_cast<size_t>(request) * p.tiles + tile] = sum;
        }
    }
}

struct DrawLds {
    Powers powers;
    double mass[kFewWaves];
    double base;
    uint32_t pick[2], tile;
};

// The first thread with v > 0 whose inclusive sum exceeds the goal, or the last with v > 0 (rounding can leave none
// above); kNone where no v is above 0. (A call has a barrier at its end.)
__device__ __forceinline__ uint32_t draw_thread(double v, double incl, double goal, DrawLds& s) {
    if (threadIdx.x == 0u) {
        s.pick[0] = kNone;
        s.pick[1] = 0u;
    }
    __syncthreads();
    const uint64_t some = __ballot(v > 0.0);
    const uint64_t past = __ballot(v > 0.0 && incl > goal);
    const uint32_t first = threadIdx.x & ~63u;
    if ((threadIdx.x & 63u) == 0u) {
        if (past != 0u) atomicMin(&s.pick[0], first + static_cast<uint32_t>(__builtin_ctzll(past)));
        if (some != 0u) atomicMax(&s.pick[1], first + 64u - static_cast<uint32_t>(__builtin_clzll(some)));
    }
    __syncthreads();
    const uint32_t got = s.pick[0] != kNone ? s.pick[0] : (s.pick[1] != 0u ? s.pick[1] - 1u : kNone);
    __syncthreads();
    return got;
}

// A workgroup a request: accepted, rejected, the logprobs, and the token.
__global__ __launch_bounds__(kFew) void verify_draw_kernel(VerifyParams p) {
    __shared__ DrawLds s;
    const VerifyArgs& a = p.a;
    const uint32_t tid = threadIdx.x;
    const uint32_t request = blockIdx.x;
    s.powers.fill();
    // The sums of the request's tiles: consecutive ones to a thread.
    const double2* const sums = p.sums + static_cast<size_t>(request) * p.tiles;
    const uint32_t per = (p.tiles + kFew - 1u) / kFew;
    const uint32_t begin = min(tid * per, p.tiles);
    const uint32_t end = min(begin + per, p.tiles);
    double r_sum = 0.0, p_sum = 0.0;
    for (uint32_t t = begin; t < end; ++t) {
        r_sum += sums[t].x;
        p_sum += sums[t].y;
    }
    const Stop stop = find_stop(p, request);
    if (tid == 0u) {
        a.accepted[request] = stop.accepted;
        a.rejected[request] = stop.rejects() ? stop.rows - 1u - stop.accepted : 0u;
    }
    if (stop.rows == 0u) return;
    if (a.logprobs != nullptr)
        for (uint32_t i = tid; i < stop.accepted; i += kFew) a.logprobs[stop.first + i] = p.shares[stop.first + i];
    const double u = uniform_of(a.uniforms[stop.first + stop.rows - 1u]);
    const Rest rest(p, stop);
    Scan<double> scan = few_scan(r_sum, s.mass);
    const bool by_rest = scan.all > 0.0;
    double mine = r_sum;
    if (!by_rest) {
        scan = few_scan(p_sum, s.mass);
        mine = p_sum;
    }
    const double goal = u * scan.all;
    const uint32_t holder = draw_thread(mine, scan.incl, goal, s);
    if (holder == kNone) {   // nothing above -inf
        if (tid == 0u) {
            a.tokens[request] = 0u;
            if (a.logprobs != nullptr) a.logprobs[stop.row()] = -__builtin_huge_valf();
        }
        return;
    }
    if (tid == holder) {
        double sum = scan.incl - mine;
        uint32_t at = begin;
        double before = sum;
        for (uint32_t t = begin; t < end; ++t) {
            const double v = by_rest ? sums[t].x : sums[t].y;
            if (v > 0.0) {
                at = t;
                before = sum;
                if (sum + v > goal) break;
            }
            sum += v;
        }
        s.tile = at;
        s.base = before;
    }
    __syncthreads();
    const uint32_t from = s.tile * kTile + 8u * tid;
    const double base = s.base;
    double v[8] = {}, sum = 0.0;
    rest.each(s.powers, from, [&](uint32_t k, double r, double here) HYP_INLINE {
        v[k] = by_rest ? r : here;
        sum += v[k];
    });
    const Scan<double> in_tile = few_scan(sum, s.mass);
    if (tid != draw_thread(sum, base + in_tile.incl, goal, s)) return;
    double running = base + (in_tile.incl - sum);
    uint32_t token = from;
    bool found = false;
#pragma unroll
    for (uint32_t k = 0; k < 8u; ++k) {
        running += v[k];
        if (!found && v[k] > 0.0) {
            token = from + k;
            found = running > goal;
        }
    }
    a.tokens[request] = token;
    if (a.logprobs != nullptr) a.logprobs[stop.row()] = log_share(rest.p, rest.logits[token]);
}

// A row's chunks: enough workgroups to fill the device, but no more of them than the filters read in little time. Counts and
// filters of 100 requests of 50001 tokens take 18.0 + 10.5 us with 512 workgroups, 19.0 + 12.0 with 1024, 22.2 + 13.0 with
// 2048; those of one request of 5 rows 5.7 + 8.8 with 8 chunks a row, 6.8 + 8.4 with 4, 5.2 + 11.7 with 16.
constexpr uint32_t kFill = 512;
constexpr uint32_t kMinChunk = 8192;
constexpr uint32_t kMostChunks = 8;
Chunks chunks_of(uint32_t rows, uint32_t vocab) {
    if (rows == 0u || vocab == 0u) return {1u, vocab};
    uint32_t n = std::min((kFill + rows - 1u) / rows, std::min(vocab / kMinChunk + 1u, kMostChunks));
    n = std::max(n, (vocab + kLongest - 1u) / kLongest);
    const uint32_t tokens = std::min(((vocab + n - 1u) / n + 511u) & ~511u, kLongest);
    return {(vocab + tokens - 1u) / tokens, tokens};
}

// Workgroups that the sums of all requests are given: twice what the device runs at once, so that requests without filters,
// whose exponentials take their time, do not end alone. (With half as many the sums of 64 mixed requests take 17.8 us, so 17.0,
// of 100 of 50001 tokens without filters 16.2 and 13.9; of 48 with filters and no drafting model 9.0 and 9.8.)
constexpr uint32_t kSumGroups = 4096;

struct Layout {
    Chunks chunks;
    uint32_t tiles;
    size_t stats, sums, counts, chances, shares, requests, bytes;   // offsets, the whole
};
Layout layout_of(uint32_t rows, uint32_t vocab, uint32_t requests, bool drafted) {
    const size_t all = static_cast<size_t>(rows) * (drafted ? 2u : 1u);
    Layout l{chunks_of(static_cast<uint32_t>(all), vocab), (vocab + kTile - 1u) / kTile, 0, 0, 0, 0, 0, 0, 0};
    const auto add = [&](size_t bytes) {
        const size_t at = l.bytes;
        l.bytes += (bytes + 15u) & ~size_t{15u};
        return at;
    };
    l.stats = add(all * sizeof(RowStat));
    l.sums = add(static_cast<size_t>(requests) * l.tiles * sizeof(double2));
    l.counts = add(all * l.chunks.n * sizeof(ChunkCounts));
    l.chances = add(all * sizeof(double));
    l.shares = add(all * sizeof(float));
    l.requests = add(all * sizeof(uint32_t));
    return l;
}

}  // namespace

size_t verify_batch_workspace_bytes(uint32_t rows, uint32_t vocab, uint32_t requests, bool drafted) {
    return layout_of(rows, vocab, requests, drafted).bytes;
}

void launch_verify_batch(const VerifyArgs& a, hipStream_t stream) {
    const bool drafted = a.draft_logits != nullptr;
    const uint32_t all = a.rows * (drafted ? 2u : 1u);
    const Layout l = layout_of(a.rows, a.vocab, a.requests, drafted);
    char* const w = static_cast<char*>(a.workspace);
    VerifyParams p{};
    p.a = a;
    p.chunks = l.chunks;
    p.tiles = l.tiles;
    const uint32_t most = std::max(1u, std::min(l.tiles, kSumGroups / a.requests));
    const uint32_t each = std::max(1u, (l.tiles + most - 1u) / most);   // tiles of a workgroup, as even as they get
    p.groups = std::max(1u, (l.tiles + each - 1u) / each);
    p.stats = reinterpret_cast<RowStat*>(w + l.stats);
    p.sums = reinterpret_cast<double2*>(w + l.sums);
    p.counts = reinterpret_cast<ChunkCounts*>(w + l.counts);
    p.chances = reinterpret_cast<double*>(w + l.chances);
    p.shares = reinterpret_cast<float*>(w + l.shares);
    p.requests = reinterpret_cast<uint32_t*>(w + l.requests);
    if (all != 0u) {
        const bool cached = uint64_t{2} * all * a.vocab <= kCached;
        hipLaunchKernelGGL(cached ? verify_count_kernel<0u> : verify_count_kernel<kChunkLoads>, dim3(all * l.chunks.n),
                           dim3(kThreads), 0, stream, p);
        HYP_HIP_CHECK(hipGetLastError());
        hipLaunchKernelGGL(verify_filter_kernel, dim3(all), dim3(kFew), 0, stream, p);
        HYP_HIP_CHECK(hipGetLastError());
        hipLaunchKernelGGL(verify_sum_kernel, dim3(a.requests * p.groups), dim3(kFew), 0, stream, p);
        HYP_HIP_CHECK(hipGetLastError());
    }
    hipLaunchKernelGGL(verify_draw_kernel, dim3(a.requests), dim3(kFew), 0, stream, p);
    HYP_HIP_CHECK(hipGetLastError());
}

}  // namespace hyperion::hip
