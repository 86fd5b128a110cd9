// Verification of drafted tokens against the target's probabilities, from given uniforms (hyp_verify_batch).
//
// p and q are a row's distributions of the target and of the drafting model: weights w = exp((x - x_max) / T) of the
// tokens that the filters keep, over their sum. The draft x of a row is accepted iff u q(x) < p(x). The first row whose
// draft is not, or a request's last row, draws the next token from max(0, p - q) (from p behind the last draft): the
// first token along the index whose running sum exceeds u times the whole. So the accepted tokens and the drawn one are
// distributed as tokens drawn from p one by one.
//
// Steps:
//  1, 2. of every row of both models, what hyp_sample_batch counts and filters (sample_row.h), up to the last token that
//     is kept: a row is then its largest logit, the kept and the whole mass, the last kept value and the last kept
//     token of that value. With that any token's p follows from its logit alone;
//  3. each request's stop row, by every workgroup for itself (a few loads), and the sums of max(0, p - q) over tiles of
//     the vocabulary;
//  4. a workgroup a request: the tile, then the token in it.
// All weights and sums are fp64; tokens that p does not keep have no weight, so their exponentials are not formed.
#include <algorithm>
#include <cstdint>

#include "batch.h"
#include "common.h"
#include "sample_row.h"
#include "verify_batch.h"

namespace hyperion::hip {
namespace {

using namespace sampling;

constexpr uint32_t kDrawThreads = 256;
constexpr uint32_t kDrawWaves = kDrawThreads / 64u;
constexpr uint32_t kTile = 8u * kDrawThreads;   // eight consecutive tokens a thread
constexpr uint32_t kNoToken = 0xFFFFFFFFu;

enum RowKind : uint32_t { kEmpty = 0, kFinite = 1, kInfinite = 2 };   // nothing above -inf; ...; +inf among the logits

// A row and its filters.
struct alignas(16) RowStat {
    double top, by_t, by_kept, total;   // largest logit, 1 / temperature, 1 / kept mass, mass of all tokens
    uint32_t cut, last;                 // place of the last value that is kept, the last kept token of that value
    uint32_t kind, unused;
};

struct VerifyParams {
    VerifyArgs a;
    Chunks chunks;
    RowStat* stats;        // [rows], then those of the drafting model
    double2* sums;         // [requests][tiles]: of max(0, p - q), of p
    ChunkCounts* counts;   // [rows, then the drafting model's][chunks.n]
    uint32_t tiles;
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

// The row that a workgroup of the first two launches has, if it has one: nothing follows a request's last row, whose
// drafting model's logits do not matter.
struct Source {
    const uint16_t* logits;
    uint32_t request;
    bool live, draft;
};
__device__ __forceinline__ Source source_of(const VerifyArgs& a, uint32_t index) {
    Source s{nullptr, 0u, false, index >= a.rows};
    const uint32_t row = s.draft ? index - a.rows : index;
    if (row >= a.row_start[a.requests]) return s;
    s.request = request_of(a.row_start, a.requests, row);
    s.live = !s.draft || row + 1u < a.row_start[s.request + 1u];
    s.logits = (s.draft ? a.draft_logits : a.logits) + static_cast<size_t>(row) * a.vocab;
    return s;
}

__global__ __launch_bounds__(kThreads) void verify_count_kernel(VerifyParams p) {
    __shared__ RowLds s;
    const uint32_t index = blockIdx.x / p.chunks.n;
    const Source src = source_of(p.a, index);
    if (!src.live) return;
    const uint32_t begin = min(p.a.vocab, (blockIdx.x - index * p.chunks.n) * p.chunks.tokens);
    count_values(src.logits, begin, min(p.a.vocab, begin + p.chunks.tokens), s);
    store_counts(s, p.counts[blockIdx.x]);
}

template <bool kSplit>
__global__ __launch_bounds__(kThreads) void verify_filter_kernel(VerifyParams p) {
    __shared__ RowLds s;
    const uint32_t index = blockIdx.x;
    const Source src = source_of(p.a, index);
    if (!src.live) return;
    const RowParams prm = row_params((src.draft ? p.a.draft_configs : p.a.configs)[src.request], 0.0f);
    const ChunkCounts* const counts = kSplit ? p.counts + static_cast<size_t>(index) * p.chunks.n : nullptr;
    if constexpr (kSplit) {
        sum_counts(counts, p.chunks.n, s);
    } else {
        count_values(src.logits, 0u, p.a.vocab, s);
    }
    const bool any = find_row<false>(src.logits, p.a.vocab, prm, s);
    RowStat* const out = p.stats + index;
    const auto leave = [&](uint32_t last) {
        RowStat r{};
        r.top = s.top;
        r.by_t = prm.by_t;
        r.by_kept = 1.0 / s.kept;
        r.total = s.total;
        r.cut = place_of(s.drawn);
        r.last = last;
        r.kind = s.infinite != 0u ? kInfinite : kFinite;
        *out = r;
    };
    if (!any) {
        if (threadIdx.x == 0u) *out = RowStat{};
    } else if (s.whole != 0u) {
        if (threadIdx.x == 0u) leave(p.a.vocab);
    } else {
        find_token<kSplit>(src.logits, p.a.vocab, p.chunks, counts, s, leave);
    }
}

// The probability of a token from its logit.
__device__ __forceinline__ double probability(const RowStat& r, uint32_t bits, uint32_t token) {
    bits = plain_bits(bits);
    if (r.kind != kFinite) return r.kind == kInfinite && bits == 0x7F80u && token <= r.last ? r.by_kept : 0.0;
    const uint32_t place = place_of(bits);
    if (!finite_bits(bits) || place > r.cut || (place == r.cut && token > r.last)) return 0.0;
    return exp_below((value_of(bits) - r.top) * r.by_t) * r.by_kept;
}

// ln of a token's share of the mass before the filters.
__device__ __forceinline__ float log_share(const RowStat& r, uint32_t bits) {
    if (r.kind == kEmpty) return -__builtin_huge_valf();
    const double gap = r.kind == kInfinite ? 0.0 : (value_of(bits) - r.top) * r.by_t;
    return static_cast<float>(gap - log(r.total));
}

__device__ __forceinline__ double uniform_of(float u) {   // as a draw takes it
    return u > 0.0f ? static_cast<double>(fminf(u, 0x1.fffffep-1f)) : 0.0;
}

// Where a request stops.
struct Stop {
    uint32_t first, rows, accepted;
    [[nodiscard]] __device__ uint32_t row() const { return first + accepted; }
    [[nodiscard]] __device__ bool rejects() const { return accepted + 1u < rows; }
};

// By a whole workgroup; `least` is a word of its LDS. (A call has a barrier at its end.)
__device__ __forceinline__ Stop find_stop(const VerifyParams& p, uint32_t request, uint32_t& least) {
    const VerifyArgs& a = p.a;
    const uint32_t first = min(a.row_start[request], a.rows);
    const uint32_t end = min(a.row_start[request + 1u], a.rows);
    const uint32_t rows = end > first ? end - first : 0u;
    if (threadIdx.x == 0u) least = rows != 0u ? rows - 1u : 0u;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i + 1u < rows; i += kDrawThreads) {
        const uint32_t row = first + i;
        const uint32_t x = a.ids[row + 1u];
        bool taken = false;
        if (x < a.vocab) {
            const size_t at = static_cast<size_t>(row) * a.vocab + x;
            const double q = a.draft_logits != nullptr ? probability(p.stats[a.rows + row], a.draft_logits[at], x) : 1.0;
            taken = uniform_of(a.uniforms[row]) * q < probability(p.stats[row], a.logits[at], x);
        }
        if (!taken) {
            atomicMin(&least, i);
            break;
        }
    }
    __syncthreads();
    return {first, rows, least};
}

// max(0, p - q) and p of a tile's eight tokens of this thread, at the stop row.
struct Rest {
    const uint16_t* logits;
    const uint16_t* draft_logits;   // null: q is 1 at `without` and 0 elsewhere
    RowStat p, q;
    uint32_t without, vocab;
    __device__ Rest(const VerifyParams& v, const Stop& stop)
        : logits(v.a.logits + static_cast<size_t>(stop.row()) * v.a.vocab), draft_logits(nullptr), p(v.stats[stop.row()]), q{},
          without(kNoToken), vocab(v.a.vocab) {
        if (!stop.rejects()) return;
        if (v.a.draft_logits != nullptr) {
            draft_logits = v.a.draft_logits + static_cast<size_t>(stop.row()) * vocab;
            q = v.stats[v.a.rows + stop.row()];
        } else {
            without = v.a.ids[stop.row() + 1u];
        }
    }
    // f(k, max(0, p - q), p) for the tokens begin + k, k < 8, that there are.
    template <typename F>
    __device__ __forceinline__ void each(uint32_t begin, F&& f) const {
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
            const double here = probability(p, x.v[k], begin + k);
            double rest = here;
            if (here > 0.0) {
                if (draft_logits != nullptr) rest = fmax(0.0, here - probability(q, y.v[k], begin + k));
                if (begin + k == without) rest = 0.0;
            }
            f(k, rest, here);
        }
    }
};

// Exclusive sums in thread order and the whole, by a workgroup of kDrawThreads. (Every wave has left `waves`.)
struct DrawScan {
    double incl, all;
};
__device__ __forceinline__ DrawScan draw_scan(double v, double* waves) {
    const uint32_t wave = threadIdx.x >> 6;
    double incl = wave_incl64(v);
    if ((threadIdx.x & 63u) == 63u) waves[wave] = incl;
    __syncthreads();
    double all = 0.0;
    for (uint32_t w = 0; w < kDrawWaves; ++w) {
        if (w == wave) incl += all;
        all += waves[w];
    }
    __syncthreads();
    return {incl, all};
}

__global__ __launch_bounds__(kDrawThreads) void verify_sum_kernel(VerifyParams p, uint32_t groups) {
    __shared__ uint32_t least;
    __shared__ double waves[kDrawWaves];
    const uint32_t request = blockIdx.x / groups;
    const Stop stop = find_stop(p, request, least);
    if (stop.rows == 0u) return;
    const Rest rest(p, stop);
    for (uint32_t tile = blockIdx.x - request * groups; tile < p.tiles; tile += groups) {
        double r_sum = 0.0, p_sum = 0.0;
        rest.each(tile * kTile + 8u * threadIdx.x, [&](uint32_t, double r, double here) {
            r_sum += r;
            p_sum += here;
        });
        const double r_all = draw_scan(r_sum, waves).all;
        const double p_all = draw_scan(p_sum, waves).all;
        if (threadIdx.x == 0u) p.sums[static_cast<size_t>(request) * p.tiles + tile] = make_double2(r_all, p_all);
    }
}

// The first thread with v > 0 whose inclusive sum exceeds the goal, or the last with v > 0 (rounding can leave none
// above); kDrawThreads where no v is above 0. pick[0] and pick[1] are words of LDS.
__device__ __forceinline__ uint32_t draw_thread(double v, double incl, double goal, uint32_t* pick) {
    const uint32_t tid = threadIdx.x;
    if (tid == 0u) {
        pick[0] = kDrawThreads;
        pick[1] = 0u;
    }
    __syncthreads();
    if (v > 0.0) {
        if (incl > goal) atomicMin(&pick[0], tid);
        atomicMax(&pick[1], tid + 1u);
    }
    __syncthreads();
    const uint32_t got = pick[0] != kDrawThreads ? pick[0] : (pick[1] != 0u ? pick[1] - 1u : kDrawThreads);
    __syncthreads();
    return got;
}

__global__ __launch_bounds__(kDrawThreads) void verify_draw_kernel(VerifyParams p) {
    __shared__ uint32_t least, pick[2], tile_at;
    __shared__ double waves[kDrawWaves], before_tile;
    const uint32_t tid = threadIdx.x;
    const uint32_t request = blockIdx.x;
    const VerifyArgs& a = p.a;
    const Stop stop = find_stop(p, request, least);
    if (tid == 0u) {
        a.accepted[request] = stop.accepted;
        a.rejected[request] = stop.rejects() ? stop.rows - 1u - stop.accepted : 0u;
    }
    if (stop.rows == 0u) return;
    if (a.logprobs != nullptr) {
        for (uint32_t i = tid; i < stop.accepted; i += kDrawThreads) {
            const uint32_t row = stop.first + i;
            a.logprobs[row] = log_share(p.stats[row], a.logits[static_cast<size_t>(row) * a.vocab + a.ids[row + 1u]]);
        }
    }
    // The tile: consecutive ones to a thread.
    const double2* const sums = p.sums + static_cast<size_t>(request) * p.tiles;
    const uint32_t per = (p.tiles + kDrawThreads - 1u) / kDrawThreads;
    const uint32_t begin = min(tid * per, p.tiles);
    const uint32_t end = min(begin + per, p.tiles);
    double r_sum = 0.0, p_sum = 0.0;
    for (uint32_t t = begin; t < end; ++t) {
        r_sum += sums[t].x;
        p_sum += sums[t].y;
    }
    const DrawScan r_scan = draw_scan(r_sum, waves);
    const DrawScan p_scan = draw_scan(p_sum, waves);
    const bool by_rest = r_scan.all > 0.0;
    const double mine = by_rest ? r_sum : p_sum;
    const DrawScan scan = by_rest ? r_scan : p_scan;
    const double goal = uniform_of(a.uniforms[stop.first + stop.rows - 1u]) * scan.all;
    const uint32_t holder = draw_thread(mine, scan.incl, goal, pick);
    if (holder == kDrawThreads) {   // nothing above -inf
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
        tile_at = at;
        before_tile = before;
    }
    __syncthreads();
    const Rest rest(p, stop);
    const uint32_t from = tile_at * kTile + 8u * tid;
    double v[8], sum = 0.0;
    rest.each(from, [&](uint32_t k, double r, double here) {
        v[k] = by_rest ? r : here;
        sum += v[k];
    });
    const DrawScan in_tile = draw_scan(sum, waves);
    if (tid != draw_thread(sum, before_tile + in_tile.incl, goal, pick)) return;
    double running = before_tile + (in_tile.incl - sum);
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

// Workgroups that the sums of all requests are given: eight are on a compute unit.
constexpr uint32_t kSumGroups = 2048;

uint32_t tiles_of(uint32_t vocab) { return (vocab + kTile - 1u) / kTile; }

struct Layout {
    Chunks chunks;
    size_t stats, sums, counts, bytes;   // offsets, the whole
};
Layout layout_of(uint32_t rows, uint32_t vocab, uint32_t requests, bool drafted) {
    const uint32_t all = rows * (drafted ? 2u : 1u);
    Layout l{chunks_of(all, vocab), 0u, 0u, 0u, 0u};
    l.sums = l.stats + static_cast<size_t>(all) * sizeof(RowStat);
    l.counts = l.sums + static_cast<size_t>(requests) * tiles_of(vocab) * sizeof(double2);
    l.bytes = l.counts + (l.chunks.n > 1u ? static_cast<size_t>(all) * l.chunks.n * sizeof(ChunkCounts) : 0u);
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
    const VerifyParams p{a, l.chunks, reinterpret_cast<RowStat*>(w + l.stats), reinterpret_cast<double2*>(w + l.sums),
                         reinterpret_cast<ChunkCounts*>(w + l.counts), tiles_of(a.vocab)};
    if (all == 0u) {
        // (no row of any request)
    } else if (l.chunks.n > 1u) {
        hipLaunchKernelGGL(verify_count_kernel, dim3(all * l.chunks.n), dim3(kThreads), 0, stream, p);
        HYP_HIP_CHECK(hipGetLastError());
        hipLaunchKernelGGL(verify_filter_kernel<true>, dim3(all), dim3(kThreads), 0, stream, p);
    } else {
        hipLaunchKernelGGL(verify_filter_kernel<false>, dim3(all), dim3(kThreads), 0, stream, p);
    }
    HYP_HIP_CHECK(hipGetLastError());
    const uint32_t groups = std::max(1u, std::min(p.tiles, kSumGroups / a.requests));
    hipLaunchKernelGGL(verify_sum_kernel, dim3(a.requests * groups), dim3(kDrawThreads), 0, stream, p, groups);
    HYP_HIP_CHECK(hipGetLastError());
    hipLaunchKernelGGL(verify_draw_kernel, dim3(a.requests), dim3(kDrawThreads), 0, stream, p);
    HYP_HIP_CHECK(hipGetLastError());
}

}  // namespace hyperion::hip
