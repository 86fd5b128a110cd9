// Operations on the blocks of a batch's requests: fork, rewind, compact, copy (hyp_batch_fork and so on).
//
// Requests may hold a block in common (forked ones do). How many hold one is nowhere stored: rewind and compact mark the
// blocks in use from the tables and lengths, so there is no count that could go wrong between calls.
//
// What bounds the first three: the latency of launches and of dependent trips to memory within them; their data are a few
// KB to 1 MB. A call in a stream of calls takes: 12 requests forked 4.1 to 4.7 us, 480 8.0; 64 requests' drafts given back
// 8.3, 500 requests of which 71 end 20 (12.4 of a traced call's 22 are one workgroup that goes through 10000 blocks that
// may go back); 16 requests compacted 5.7, 400 in a pool of 78000 blocks 14.3. Copies are bound by memory: 1.05 GB in
// 210 us, 5.0 TB/s, the rate of a large copy; 29 MB in 7.2.
#include <algorithm>
#include <cstdint>

#include "batch.h"
#include "batch_pages.h"
#include "common.h"
#include "wave.h"

namespace hyperion::hip {
namespace {

constexpr uint32_t kThreads = 1024;
constexpr uint32_t kWaves = kThreads / 64u;
constexpr uint32_t kPer = kMaxRequests / kThreads;   // consecutive requests of a thread
constexpr uint32_t kEntryThreads = 256;

__device__ __forceinline__ uint32_t blocks_of(const BatchView& b, uint32_t tokens) {   // as far as the table goes
    const uint64_t n = (static_cast<uint64_t>(tokens) + ((1u << b.shift) - 1u)) >> b.shift;
    return static_cast<uint32_t>(min(n, static_cast<uint64_t>(b.max_blocks)));
}
__device__ __forceinline__ uint32_t* table_of(const BatchView& b, uint32_t request) {
    return b.tables + static_cast<size_t>(request) * b.max_blocks;
}

// The last index i < n with sums[i] <= at (sums[0] = 0, not decreasing, at < sums[n]).
__device__ __forceinline__ uint32_t owner(const uint32_t* sums, uint32_t n, uint32_t at) {
    uint32_t lo = 0u, hi = n;
    while (hi - lo > 1u) {
        const uint32_t mid = (lo + hi) / 2u;
        if (sums[mid] <= at) lo = mid; else hi = mid;
    }
    return lo;
}

struct Sum {
    uint32_t before, all;   // the threads before this one, all
};
// By the whole workgroup. (A call has a barrier at its end.)
__device__ __forceinline__ Sum block_sum(uint32_t v, uint32_t* waves) {
    const uint32_t wave = threadIdx.x >> 6;
    const uint32_t incl = wave_incl(v);
    if ((threadIdx.x & 63u) == 63u) waves[wave] = incl;
    __syncthreads();
    Sum s{incl - v, 0u};
    for (uint32_t w = 0; w < kWaves; ++w) {
        if (w < wave) s.before += waves[w];
        s.all += waves[w];
    }
    __syncthreads();
    return s;
}

// Small tables are gone through by the one workgroup that has the rest to do, all entries of all rows in a line: a launch
// takes longer than 32 entries a thread. (A call on 64 requests of up to 250 blocks: rewind 8.4 us so, 11.4 with clearing and
// marking by the whole device; 16 compacted 5.7 and 11.3; 12 forked 4.7 and 6.5. The marks of 32768 blocks fill LDS.)
constexpr uint32_t kSmallTable = 32u * kThreads;   // entries
constexpr uint32_t kSmallRequests = kThreads;
constexpr uint32_t kSmallPool = 32u * kThreads;    // blocks
bool small_table(const BatchView& b) {
    return b.requests <= kSmallRequests && static_cast<uint64_t>(b.requests) * b.max_blocks <= kSmallTable;
}
// f(request, entry, where it is) of each, four to a thread on their way together (of load(...), then use(..., loaded)).
template <typename Load, typename Use>
__device__ __forceinline__ void for_entries(const BatchView& b, Load&& load, Use&& use) {
    const uint32_t all = b.requests * b.max_blocks;
    const float by_width = 1.0f / static_cast<float>(b.max_blocks);   // (exact below 2^21 entries)
#pragma unroll 1
    for (uint32_t base = threadIdx.x; base < all; base += 4u * kThreads) {
        uint32_t r[4], e[4], v[4];
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            const uint32_t at = base + i * kThreads;
            r[i] = at < all ? static_cast<uint32_t>((static_cast<float>(at) + 0.5f) * by_width) : 0u;
            e[i] = at - r[i] * b.max_blocks;
            v[i] = at < all ? load(r[i], e[i], at) : 0u;
        }
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i)
            if (base + i * kThreads < all) use(r[i], e[i], base + i * kThreads, v[i]);
    }
}

// ---- fork -------------------------------------------------------------------------------------

struct ForkParams {
    BatchView b;
    const uint32_t* lens;
    const uint32_t* parents;
    const uint32_t* free_blocks;
    const uint32_t* taken;
    uint32_t* taken_out;
    uint32_t* served;
    HypBlockCopy* copies;
    uint32_t* n_copies;
};

// The parent of a request that becomes its copy, or HYP_PARENT_NONE.
__device__ __forceinline__ uint32_t parent_of(const ForkParams& p, uint32_t request) {
    const uint32_t parent = p.parents[request];
    if (parent >= p.b.requests || p.parents[parent] != HYP_PARENT_NONE) return HYP_PARENT_NONE;
    return parent;
}

// Lengths, the blocks of their own that copies get, and how far the free ones go; the entries of whole blocks too where the
// table is small.
template <bool kSmall>
__global__ __launch_bounds__(kThreads) void fork_kernel(ForkParams p) {
    __shared__ uint32_t waves[kWaves];
    __shared__ uint32_t parent_at[kSmall ? kSmallRequests : 1u], whole_of[kSmall ? kSmallRequests : 1u];
    __shared__ uint32_t served_at;
    const BatchView& b = p.b;
    const uint32_t tid = threadIdx.x;
    const uint32_t n = b.requests;
    const uint32_t per = (n + kThreads - 1u) / kThreads;
    const uint32_t first = tid * per;
    const uint32_t mask = (1u << b.shift) - 1u;
    const uint32_t taken = min(*p.taken, b.num_blocks);
    const uint32_t free_left = b.num_blocks - taken;
    uint32_t parent[kPer], len[kPer];
    uint32_t need = 0u;
    const auto needs = [&](uint32_t i) {   // a partly filled last block
        return parent[i] != HYP_PARENT_NONE && (len[i] & mask) != 0u && (len[i] >> b.shift) < b.max_blocks;
    };
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
        const uint32_t r = first + i;
        const bool live = i < per && r < n;
        parent[i] = live ? parent_of(p, r) : HYP_PARENT_NONE;
        len[i] = !live ? 0u : p.lens[parent[i] != HYP_PARENT_NONE ? parent[i] : r];
        need += needs(i) ? 1u : 0u;
    }
    if (tid == 0u) served_at = n;
    const Sum sum = block_sum(need, waves);
    uint32_t rank = sum.before;
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
        if (!needs(i)) continue;
        if (rank == free_left) atomicMin(&served_at, first + i);
        ++rank;
    }
    __syncthreads();
    const uint32_t served = served_at;
    rank = sum.before;
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
        const uint32_t r = first + i;
        if (i >= per || r >= n) continue;
        const bool in = parent[i] != HYP_PARENT_NONE && r < served;
        if (in && needs(i)) {
            const uint32_t entry = len[i] >> b.shift;
            const uint32_t fresh = p.free_blocks[taken + rank];
            p.copies[rank] = {table_of(b, parent[i])[entry], fresh, len[i] & mask};
            table_of(b, r)[entry] = fresh;
        }
        if (needs(i)) ++rank;
        b.lens[r] = parent[i] == HYP_PARENT_NONE || in ? len[i] : p.lens[r];
        if constexpr (kSmall) {
            parent_at[r] = parent[i];
            whole_of[r] = in ? min(len[i] >> b.shift, b.max_blocks) : 0u;
        }
    }
    if (tid == 0u) {
        const uint32_t copied = min(sum.all, free_left);
        *p.n_copies = copied;
        *p.taken_out = taken + copied;
        *p.served = served;
    }
    if constexpr (kSmall) {
        __syncthreads();
        for_entries(
            b, [&](uint32_t r, uint32_t e, uint32_t) { return e < whole_of[r] ? table_of(b, parent_at[r])[e] : 0u; },
            [&](uint32_t r, uint32_t e, uint32_t at, uint32_t v) {
                if (e < whole_of[r]) b.tables[at] = v;
            });
    }
}

// The entries of whole blocks.
__global__ __launch_bounds__(kEntryThreads) void fork_rows_kernel(ForkParams p) {
    const BatchView& b = p.b;
    const uint32_t r = blockIdx.x;
    if (r >= *p.served) return;
    const uint32_t parent = parent_of(p, r);
    if (parent == HYP_PARENT_NONE) return;
    const uint32_t whole = min(b.lens[parent] >> b.shift, b.max_blocks);
    const uint32_t* const from = table_of(b, parent);
    uint32_t* const to = table_of(b, r);
    for (uint32_t e = blockIdx.y * kEntryThreads + threadIdx.x; e < whole; e += gridDim.y * kEntryThreads) to[e] = from[e];
}

// ---- rewind -----------------------------------------------------------------------------------

// Workspace: for each block a word, the largest of: kFirmly where a request still holds it; 1 << 31 | r + 1 where request r was
// shortened into it; 1 << 30 | 4095 - r where request r gives it up. So a block that nobody holds names the first request that
// gave it up, and one that all its holders were shortened into the last of those.
constexpr uint32_t kFirmly = 0xFFFFFFFFu;
constexpr uint32_t kNobody = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t cut_by(uint32_t request) { return 0x80000000u | (request + 1u); }
__device__ __forceinline__ uint32_t left_by(uint32_t request) { return 0x40000000u | (kMaxRequests - 1u - request); }

struct RewindParams {
    BatchView b;
    const uint32_t* lens;
    const uint32_t* drop;
    uint32_t* free_blocks;
    const uint32_t* taken;
    uint32_t* taken_out;
    HypBlockCopy* copies;
    uint32_t* n_copies;
    uint32_t* state;    // [num_blocks]
};

__global__ __launch_bounds__(kEntryThreads) void rewind_clear_kernel(RewindParams p) {
    const uint32_t i = blockIdx.x * kEntryThreads + threadIdx.x;
    if (i < p.b.num_blocks) p.state[i] = 0u;
}

struct Shortened {
    uint32_t len, keep;
    uint32_t had, has;   // blocks
    uint32_t part;       // the entry of the block that it was shortened into and fills partly, kNobody if none
};
__device__ __forceinline__ Shortened shortened(const RewindParams& p, uint32_t request) {
    const BatchView& b = p.b;
    Shortened s;
    s.len = p.lens[request];
    s.keep = s.len - min(s.len, p.drop[request]);
    s.had = blocks_of(b, s.len);
    s.has = blocks_of(b, s.keep);
    const bool part = s.keep < s.len && (s.keep & ((1u << b.shift) - 1u)) != 0u && (s.keep >> b.shift) < b.max_blocks;
    s.part = part ? s.keep >> b.shift : kNobody;
    return s;
}

__global__ __launch_bounds__(kEntryThreads) void rewind_mark_kernel(RewindParams p) {
    const BatchView& b = p.b;
    const uint32_t r = blockIdx.x;
    const Shortened s = shortened(p, r);
    const uint32_t* const table = table_of(b, r);
    for (uint32_t e = blockIdx.y * kEntryThreads + threadIdx.x; e < s.had; e += gridDim.y * kEntryThreads) {
        const uint32_t block = table[e];
        if (block < b.num_blocks) atomicMax(&p.state[block], e >= s.has ? left_by(r) : (e == s.part ? cut_by(r) : kFirmly));
    }
}

// The entries given up, from the last to the first: so a block that goes back has its place in the stack, from the top down,
// without their number. kEach consecutive ones to a thread, with their loads on the way together. How many went back.
// (One to a thread while that does: the kernel takes 8.1 us for 64 requests' drafts so, 9.8 with four; for 10000 blocks of 71
// requests that end 12.5 with four, 19.6 with one, 13.4 with eight.)
template <uint32_t kEach>
__device__ __forceinline__ uint32_t give_back(const RewindParams& p, const uint32_t* state, const uint32_t* gone_sum,
                                              const uint32_t* first_gone, uint32_t all, uint32_t taken, uint32_t* waves) {
    const BatchView& b = p.b;
    const uint32_t n = b.requests;
    uint32_t returned = 0u;
    for (uint32_t base = 0u; base < all && returned < taken; base += kThreads * kEach) {
        uint32_t block[kEach], by[kEach], goes = 0u;
        const uint32_t at = base + threadIdx.x * kEach;   // from the end
        uint32_t r = at < all ? owner(gone_sum, n, all - 1u - at) : 0u;
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            block[i] = kNobody;
            by[i] = 0u;
            if (at + i >= all) continue;
            const uint32_t g = all - 1u - (at + i);
            while (g < gone_sum[r]) --r;
            by[i] = r;
            block[i] = table_of(b, r)[first_gone[r] + (g - gone_sum[r])];
        }
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i)
            if (block[i] < b.num_blocks && state[block[i]] == left_by(by[i])) goes |= 1u << i;
        const Sum here = block_sum(static_cast<uint32_t>(__popc(goes)), waves);
        uint32_t rank = returned + here.before;
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i)
            if ((goes >> i) & 1u) {
                if (rank < taken) p.free_blocks[taken - 1u - rank] = block[i];
                ++rank;
            }
        returned += here.all;
    }
    return min(returned, taken);
}

// kSmall: the marks are this workgroup's own. kMarks: they are in LDS, read at once where others made them (500 requests of
// which 71 end, 20000 blocks: the kernel takes 12.5 us, 15.2 with each mark from memory).
constexpr uint32_t kMarkPool = 28u * kThreads;   // blocks whose marks fit LDS beside 4096 requests
template <bool kSmall, bool kMarks>
__global__ __launch_bounds__(kThreads) void rewind_kernel(RewindParams p) {
    static_assert(kMarks || !kSmall, "the workgroup's own marks");
    constexpr uint32_t kRequests = kSmall ? kSmallRequests : kMaxRequests;
    __shared__ uint32_t gone_sum[kRequests + 1];   // entries given up by the requests before
    __shared__ uint32_t first_gone[kRequests];     // a request's first of them
    __shared__ uint32_t had[kSmall ? kRequests : 1u], part[kSmall ? kRequests : 1u];
    alignas(16) __shared__ uint32_t marks[kSmall ? kSmallPool : (kMarks ? kMarkPool : 1u)];
    __shared__ uint32_t waves[kWaves];
    uint32_t* const state = kMarks ? marks : p.state;
    const BatchView& b = p.b;
    const uint32_t tid = threadIdx.x;
    const uint32_t n = b.requests;
    const uint32_t per = (n + kThreads - 1u) / kThreads;
    const uint32_t first = tid * per;
    const uint32_t taken = min(*p.taken, b.num_blocks);
    if constexpr (kSmall)
        for (uint32_t i = tid; i < b.num_blocks; i += kThreads) marks[i] = 0u;
    if constexpr (kMarks && !kSmall) {   // (a workspace has whole words of 16 bytes)
#pragma unroll
        for (uint32_t k = 0; k < kMarkPool / (4u * kThreads); ++k) {
            const uint32_t i = k * kThreads + tid;
            if (4u * i < b.num_blocks) reinterpret_cast<uint4*>(marks)[i] = reinterpret_cast<const uint4*>(p.state)[i];
        }
    }
    Shortened s[kPer];
    uint32_t gone = 0u;
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
        const uint32_t r = first + i;
        if (i >= per || r >= n) continue;
        s[i] = shortened(p, r);
        gone += s[i].had - s[i].has;
    }
    const Sum sum = block_sum(gone, waves);
    {
        uint32_t at = sum.before;
#pragma unroll
        for (uint32_t i = 0; i < kPer; ++i) {
            const uint32_t r = first + i;
            if (i >= per || r >= n) continue;
            gone_sum[r] = at;
            first_gone[r] = s[i].has;
            at += s[i].had - s[i].has;
            if constexpr (kSmall) {
                had[r] = s[i].had;
                part[r] = s[i].part;
            }
        }
        if (tid == 0u) gone_sum[n] = sum.all;
    }
    __syncthreads();
    if constexpr (kSmall) {
        for_entries(
            b, [&](uint32_t r, uint32_t e, uint32_t at) { return e < had[r] ? b.tables[at] : kNobody; },
            [&](uint32_t r, uint32_t e, uint32_t, uint32_t block) {
                if (block < b.num_blocks)
                    atomicMax(&marks[block], e >= first_gone[r] ? left_by(r) : (e == part[r] ? cut_by(r) : kFirmly));
            });
        __syncthreads();
    }
    const uint32_t returned = sum.all <= kThreads ? give_back<1>(p, state, gone_sum, first_gone, sum.all, taken, waves)
                                                  : give_back<4>(p, state, gone_sum, first_gone, sum.all, taken, waves);
    const uint32_t c = taken - returned;
    __syncthreads();
    // Blocks that were shared and are now filled partly.
    uint32_t need = 0u, held[kPer];
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
        const uint32_t r = first + i;
        held[i] = kNobody;
        if (i >= per || r >= n || s[i].part == kNobody) continue;
        const uint32_t at = table_of(b, r)[s[i].part];
        if (at >= b.num_blocks || state[at] == cut_by(r)) continue;
        held[i] = at;
        ++need;
    }
    const Sum needed = block_sum(need, waves);
    const uint32_t copied = min(needed.all, b.num_blocks - c);
    uint32_t rank = needed.before;
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
        const uint32_t r = first + i;
        if (i >= per || r >= n) continue;
        uint32_t keep = s[i].keep;
        if (held[i] != kNobody) {
            if (rank < copied) {
                const uint32_t fresh = p.free_blocks[c + rank];
                p.copies[rank] = {held[i], fresh, keep & ((1u << b.shift) - 1u)};
                table_of(b, r)[s[i].part] = fresh;
            } else {
                keep = s[i].part << b.shift;
            }
            ++rank;
        }
        b.lens[r] = keep;
    }
    if (tid == 0u) {
        *p.n_copies = copied;
        *p.taken_out = c + copied;
    }
}

// ---- compact ----------------------------------------------------------------------------------

// Workspace: for each block its number among those that move, then a byte each that says whether it is in use.
struct CompactParams {
    BatchView b;
    uint32_t* tables_out;
    uint32_t* prefix_out;
    uint32_t* free_blocks;
    uint32_t* taken_out;
    HypBlockCopy* copies;
    uint32_t* n_copies;
    uint32_t* move;    // [num_blocks]
    uint4* live;       // [num_blocks] bytes, 16 to one
    uint32_t prefix_blocks;
};

__global__ __launch_bounds__(kEntryThreads) void compact_clear_kernel(CompactParams p) {
    const uint32_t i = blockIdx.x * kEntryThreads + threadIdx.x;
    if (16u * i < p.b.num_blocks) p.live[i] = make_uint4(0u, 0u, 0u, 0u);
}

// A row of blocks: a request's, or behind those the prefix's.
__device__ __forceinline__ const uint32_t* row_of(const CompactParams& p, uint32_t row, uint32_t& held, uint32_t& width) {
    if (row == p.b.requests) {
        held = width = p.prefix_blocks;
        return p.b.prefix_table;
    }
    held = blocks_of(p.b, p.b.lens[row]);
    width = p.b.max_blocks;
    return table_of(p.b, row);
}

__global__ __launch_bounds__(kEntryThreads) void compact_mark_kernel(CompactParams p) {
    uint8_t* const live = reinterpret_cast<uint8_t*>(p.live);
    uint32_t held, width;
    const uint32_t* const row = row_of(p, blockIdx.x, held, width);
    for (uint32_t e = blockIdx.y * kEntryThreads + threadIdx.x; e < held; e += gridDim.y * kEntryThreads) {
        const uint32_t block = row[e];
        if (block < p.b.num_blocks) live[block] = 1u;
    }
}

// Which of 16 blocks are in use, as bits (bytes of 0 or 1).
__device__ __forceinline__ uint32_t bits_of(uint4 v) {
    const auto four = [](uint32_t w) { return (w * 0x01020408u) >> 24; };   // bit i from byte i, and nothing carried over
    return four(v.x) | four(v.y) << 4 | four(v.z) << 8 | four(v.w) << 12;
}

// The moves: with L blocks in use, the i-th of those from L upwards goes to the i-th free one below L. How many in use are
// before a block gives its number: before block j < L are j less that many free ones. Every workgroup forms L and what comes
// before its own words for itself, from all of them: a byte for each block, where one workgroup alone for all took 42 us at
// 78000 blocks.
constexpr uint32_t kMoveGroups = 64;
__global__ __launch_bounds__(kThreads) void compact_moves_kernel(CompactParams p) {
    __shared__ uint32_t waves[kWaves];
    const uint32_t tid = threadIdx.x;
    const uint32_t words = (p.b.num_blocks + 15u) / 16u;
    const uint32_t each = (words + gridDim.x - 1u) / gridDim.x;
    const uint32_t begin = min(blockIdx.x * each, words);
    const uint32_t end = min(begin + each, words);
    uint32_t mine = 0u, before = 0u;
#pragma unroll 4
    for (uint32_t i = tid; i < words; i += kThreads) {
        const uint32_t n = static_cast<uint32_t>(__popc(bits_of(p.live[i])));
        mine += n;
        before += i < begin ? n : 0u;
    }
    const uint32_t count = block_sum(mine, waves).all;
    before = block_sum(before, waves).all;
    mine = 0u;   // in use below L
#pragma unroll 4
    for (uint32_t i = tid; i <= count / 16u && i < words; i += kThreads) {
        const uint32_t used = bits_of(p.live[i]);
        mine += static_cast<uint32_t>(__popc(i < count / 16u ? used : used & ((1u << (count % 16u)) - 1u)));
    }
    const uint32_t low = block_sum(mine, waves).all;
    // A block to a thread.
    for (uint32_t base = 16u * begin; base < 16u * end; base += kThreads) {
        const uint32_t block = base + tid;
        const bool live = block < 16u * end && reinterpret_cast<const uint8_t*>(p.live)[block] != 0u;
        const Sum here = block_sum(live ? 1u : 0u, waves);
        const uint32_t number = before + here.before;   // in use before it
        if (live && block >= count) {
            p.copies[number - low].from = block;
            p.copies[number - low].tokens = 1u << p.b.shift;
            p.move[block] = number - low;
        } else if (!live && block < count && block < 16u * end) {
            p.copies[block - number].to = block;
        }
        before += here.all;
    }
    if (blockIdx.x == 0u && tid == 0u) {
        *p.n_copies = count - low;
        *p.taken_out = count;
    }
}

// All of it for a small table and pool, by one workgroup: 32 blocks to a thread, their marks a bit each.
__global__ __launch_bounds__(kThreads) void compact_small_kernel(CompactParams p) {
    static_assert(kSmallPool == 32u * kThreads, "a word to a thread");
    __shared__ uint32_t marks[kThreads], before[kThreads];   // blocks in use, how many before a word's
    __shared__ uint32_t held[kSmallRequests];
    __shared__ uint16_t holes[kSmallPool / 2u];
    __shared__ uint32_t waves[kWaves];
    __shared__ uint32_t below;   // blocks in use below L
    const BatchView& b = p.b;
    const uint32_t tid = threadIdx.x;
    const uint32_t num = b.num_blocks;
    marks[tid] = 0u;
    if (tid < b.requests) held[tid] = blocks_of(b, b.lens[tid]);
    __syncthreads();
    const auto mark = [&](uint32_t block) {
        if (block < num) atomicOr(&marks[block / 32u], 1u << (block % 32u));
    };
    for (uint32_t i = tid; i < p.prefix_blocks; i += kThreads) mark(b.prefix_table[i]);
    for_entries(
        b, [&](uint32_t r, uint32_t e, uint32_t at) { return e < held[r] ? b.tables[at] : HYP_PARENT_NONE; },
        [&](uint32_t, uint32_t, uint32_t, uint32_t block) { mark(block); });
    __syncthreads();
    const uint32_t used = marks[tid];
    const Sum in_use = block_sum(static_cast<uint32_t>(__popc(used)), waves);
    const uint32_t count = in_use.all;   // L
    before[tid] = in_use.before;
    if (tid == min(count / 32u, kThreads - 1u))   // (at kSmallPool, all)
        below = count == kSmallPool ? count
                                    : in_use.before + static_cast<uint32_t>(__popc(used & ((1u << (count % 32u)) - 1u)));
    __syncthreads();
    const uint32_t low = below;
    // Of this thread's blocks, those that move and the free ones below L.
    const auto up_to = [&](uint32_t first) {   // bits of the blocks below `first`
        return first <= 32u * tid ? 0u : (first >= 32u * tid + 32u ? 0xFFFFFFFFu : (1u << (first - 32u * tid)) - 1u);
    };
    for (uint32_t bits = used & ~up_to(count); bits != 0u; bits &= bits - 1u) {
        const uint32_t j = static_cast<uint32_t>(__builtin_ctz(bits));
        const uint32_t number = in_use.before + static_cast<uint32_t>(__popc(used & ((1u << j) - 1u))) - low;
        p.copies[number].from = 32u * tid + j;
        p.copies[number].tokens = 1u << b.shift;
    }
    for (uint32_t bits = ~used & up_to(count); bits != 0u; bits &= bits - 1u) {
        const uint32_t j = static_cast<uint32_t>(__builtin_ctz(bits));
        const uint32_t block = 32u * tid + j;
        const uint32_t number = block - (in_use.before + static_cast<uint32_t>(__popc(used & ((1u << j) - 1u))));
        p.copies[number].to = block;
        holes[number] = static_cast<uint16_t>(block);
    }
    __syncthreads();
    const auto moved = [&](uint32_t block) {
        if (block < count || block >= num) return block;
        const uint32_t word = marks[block / 32u];
        return static_cast<uint32_t>(
            holes[before[block / 32u] + static_cast<uint32_t>(__popc(word & ((1u << (block % 32u)) - 1u))) - low]);
    };
    for_entries(
        b, [&](uint32_t, uint32_t, uint32_t at) { return b.tables[at]; },
        [&](uint32_t r, uint32_t e, uint32_t at, uint32_t block) { p.tables_out[at] = e < held[r] ? moved(block) : block; });
    for (uint32_t i = tid; i < p.prefix_blocks; i += kThreads) p.prefix_out[i] = moved(b.prefix_table[i]);
    for (uint32_t i = count + tid; i < num; i += kThreads) p.free_blocks[i] = i;
    if (tid == 0u) {
        *p.n_copies = count - low;
        *p.taken_out = count;
    }
}

__global__ __launch_bounds__(kEntryThreads) void compact_tables_kernel(CompactParams p) {
    const uint32_t count = *p.taken_out;
    const uint32_t num = p.b.num_blocks;
    const uint32_t row_at = blockIdx.x;
    const uint32_t begin = blockIdx.y * kEntryThreads + threadIdx.x;
    const uint32_t stride = gridDim.y * kEntryThreads;
    if (row_at == p.b.requests + 1u) {   // the free blocks
        for (uint32_t i = begin; i < num; i += stride)
            if (i >= count) p.free_blocks[i] = i;
        return;
    }
    uint32_t held, width;
    const uint32_t* const row = row_of(p, row_at, held, width);
    uint32_t* const out = row_at == p.b.requests ? p.prefix_out : p.tables_out + static_cast<size_t>(row_at) * width;
    for (uint32_t e = begin; e < width; e += stride) {
        const uint32_t block = row[e];
        out[e] = e < held && block >= count && block < num ? p.copies[p.move[block]].to : block;
    }
}

// ---- copy -------------------------------------------------------------------------------------

struct CopyParams {
    BatchView b;
    const HypBlockCopy* copies;
    const uint32_t* n_copies;
    uint32_t max_copies, n_caches;
    uint32_t pieces;   // of a block, at most
    CopyCache caches[kCopyCaches];
};

// A workgroup to a piece of a block of one cache's K or V at a time, four 16-byte loads of a thread on their way together. (One
// block of 4096 tokens in 16 layers of 8 heads of 128, 537 MB moved: 99 us, 5.4 TB/s; 930 with whole blocks and a load at
// a time. A call on the 29 MB of a fork 7.2 and 8.3.)
constexpr uint32_t kCopyGroups = 16384;
constexpr uint32_t kPiece = 4u * 4u * kEntryThreads;   // words of 16 bytes
__global__ __launch_bounds__(kEntryThreads) void copy_kernel(CopyParams p) {
    typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
    const uint32_t count = min(*p.n_copies, p.max_copies);
    const uint32_t which = blockIdx.x / p.pieces;
    const CopyCache& cache = p.caches[which / 2u];
    uint8_t* const base = which % 2u != 0u ? cache.v : cache.k;
    const uint64_t token_words = cache.token_bytes / 16u;
    const uint64_t begin = static_cast<uint64_t>(blockIdx.x - which * p.pieces) * kPiece;
    const uint64_t step = static_cast<uint64_t>(p.pieces) * kPiece;
    for (uint32_t at = blockIdx.y; at < count; at += gridDim.y) {
        const HypBlockCopy c = p.copies[at];
        if (c.from >= p.b.num_blocks || c.to >= p.b.num_blocks || c.from == c.to) continue;
        const uint64_t words = min(c.tokens, 1u << p.b.shift) * token_words;
        const u32x4_t* const from = reinterpret_cast<const u32x4_t*>(base) + ((c.from * token_words) << p.b.shift);
        u32x4_t* const to = reinterpret_cast<u32x4_t*>(base) + ((c.to * token_words) << p.b.shift);
        for (uint64_t piece = begin; piece < words; piece += step) {
            const uint64_t end = min(words, piece + kPiece);
            uint64_t i = piece + threadIdx.x;
            for (; i + 3u * kEntryThreads < end; i += 4u * kEntryThreads) {
                u32x4_t v[4];
#pragma unroll
                for (uint32_t k = 0; k < 4u; ++k) v[k] = from[i + k * kEntryThreads];
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (uint32_t k = 0; k < 4u; ++k) to[i + k * kEntryThreads] = v[k];
            }
            for (; i < end; i += kEntryThreads) to[i] = from[i];
        }
    }
}

// Workgroups along a row of `entries`: a few entries a thread, and no more than a long row needs.
uint32_t pieces_of(uint32_t entries) { return std::min(16u, entries / (4u * kEntryThreads) + 1u); }

}  // namespace

void launch_batch_fork(const BatchView& b, const uint32_t* lens, const uint32_t* parents, const uint32_t* free_blocks,
                       const uint32_t* taken, uint32_t* taken_out, uint32_t* served, HypBlockCopy* copies,
                       uint32_t* n_copies, hipStream_t stream) {
    const ForkParams p{b, lens, parents, free_blocks, taken, taken_out, served, copies, n_copies};
    if (small_table(b)) {
        hipLaunchKernelGGL(fork_kernel<true>, dim3(1), dim3(kThreads), 0, stream, p);
        HYP_HIP_CHECK(hipGetLastError());
        return;
    }
    hipLaunchKernelGGL(fork_kernel<false>, dim3(1), dim3(kThreads), 0, stream, p);
    HYP_HIP_CHECK(hipGetLastError());
    hipLaunchKernelGGL(fork_rows_kernel, dim3(b.requests, pieces_of(b.max_blocks)), dim3(kEntryThreads), 0, stream, p);
    HYP_HIP_CHECK(hipGetLastError());
}

size_t batch_pages_workspace_bytes(const BatchView& b) {
    const size_t blocks = (static_cast<size_t>(b.num_blocks) + 15u) & ~size_t{15u};
    return 5u * blocks;   // a word and a byte each
}

void launch_batch_rewind(const BatchView& b, const uint32_t* lens, const uint32_t* drop, uint32_t* free_blocks,
                         const uint32_t* taken, uint32_t* taken_out, HypBlockCopy* copies, uint32_t* n_copies,
                         void* workspace, hipStream_t stream) {
    uint32_t* const w = static_cast<uint32_t*>(workspace);
    const RewindParams p{b, lens, drop, free_blocks, taken, taken_out, copies, n_copies, w};
    if (small_table(b) && b.num_blocks <= kSmallPool) {
        hipLaunchKernelGGL((rewind_kernel<true, true>), dim3(1), dim3(kThreads), 0, stream, p);
        HYP_HIP_CHECK(hipGetLastError());
        return;
    }
    if (b.requests != 0u && b.max_blocks != 0u) {
        hipLaunchKernelGGL(rewind_clear_kernel, dim3((b.num_blocks + kEntryThreads - 1u) / kEntryThreads),
                           dim3(kEntryThreads), 0, stream, p);
        HYP_HIP_CHECK(hipGetLastError());
        hipLaunchKernelGGL(rewind_mark_kernel, dim3(b.requests, pieces_of(b.max_blocks)), dim3(kEntryThreads), 0, stream, p);
        HYP_HIP_CHECK(hipGetLastError());
    }
    hipLaunchKernelGGL((b.num_blocks <= kMarkPool ? rewind_kernel<false, true> : rewind_kernel<false, false>), dim3(1),
                       dim3(kThreads), 0, stream, p);
    HYP_HIP_CHECK(hipGetLastError());
}

void launch_batch_compact(const BatchView& b, uint32_t* tables_out, uint32_t* prefix_out, uint32_t* free_blocks,
                          uint32_t* taken_out, HypBlockCopy* copies, uint32_t* n_copies, void* workspace,
                          hipStream_t stream) {
    uint32_t* const w = static_cast<uint32_t*>(workspace);
    const uint32_t prefix_blocks = static_cast<uint32_t>((static_cast<uint64_t>(b.prefix) + (1u << b.shift) - 1u) >> b.shift);
    uint4* const live = reinterpret_cast<uint4*>(w + ((b.num_blocks + 15u) & ~15u));
    const CompactParams p{b, tables_out, prefix_out, free_blocks, taken_out, copies, n_copies, w, live, prefix_blocks};
    if (small_table(b) && b.num_blocks <= kSmallPool && prefix_blocks <= kSmallTable) {
        hipLaunchKernelGGL(compact_small_kernel, dim3(1), dim3(kThreads), 0, stream, p);
        HYP_HIP_CHECK(hipGetLastError());
        return;
    }
    const uint32_t pieces = pieces_of(std::max(b.max_blocks, prefix_blocks));
    const uint32_t clear = (b.num_blocks + 16u * kEntryThreads - 1u) / (16u * kEntryThreads);
    hipLaunchKernelGGL(compact_clear_kernel, dim3(clear), dim3(kEntryThreads), 0, stream, p);
    HYP_HIP_CHECK(hipGetLastError());
    hipLaunchKernelGGL(compact_mark_kernel, dim3(b.requests + 1u, pieces), dim3(kEntryThreads), 0, stream, p);
    HYP_HIP_CHECK(hipGetLastError());
    const uint32_t groups = std::min(kMoveGroups, (b.num_blocks + kThreads - 1u) / kThreads);
    hipLaunchKernelGGL(compact_moves_kernel, dim3(groups), dim3(kThreads), 0, stream, p);
    HYP_HIP_CHECK(hipGetLastError());
    const uint32_t wide = std::max(pieces, pieces_of(b.num_blocks));
    hipLaunchKernelGGL(compact_tables_kernel, dim3(b.requests + 2u, wide), dim3(kEntryThreads), 0, stream, p);
    HYP_HIP_CHECK(hipGetLastError());
}

void launch_batch_copy(const BatchView& b, const CopyCache* caches, uint32_t n_caches, const HypBlockCopy* copies,
                       uint32_t max_copies, const uint32_t* n_copies, hipStream_t stream) {
    for (uint32_t at = 0u; at < n_caches; at += kCopyCaches) {
        CopyParams p{b, copies, n_copies, max_copies, std::min(kCopyCaches, n_caches - at), 1u, {}};
        std::copy(caches + at, caches + at + p.n_caches, p.caches);
        uint64_t longest = 0;
        for (uint32_t i = 0; i < p.n_caches; ++i) longest = std::max(longest, (p.caches[i].token_bytes / 16u) << b.shift);
        const uint32_t sides = 2u * p.n_caches;
        p.pieces = static_cast<uint32_t>(std::min<uint64_t>((longest + kPiece - 1u) / kPiece, std::max(1u, kCopyGroups / sides)));
        const uint32_t along = std::min(max_copies, std::max(1u, kCopyGroups / (sides * p.pieces)));
        hipLaunchKernelGGL(copy_kernel, dim3(sides * p.pieces, along), dim3(kEntryThreads), 0, stream, p);
        HYP_HIP_CHECK(hipGetLastError());
    }
}

}  // namespace hyperion::hip
