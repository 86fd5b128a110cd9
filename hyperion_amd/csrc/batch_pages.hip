// Operations on the blocks of a batch's requests: fork, rewind, compact, copy (hyp_batch_fork and so on).
//
// Requests may hold a block in common (forked ones do). How many hold one is nowhere stored: rewind and compact mark the
// blocks in use from the tables and lengths, so there is no count that could go wrong between calls.
//
// What bounds the first three: the latency of their steps, a few KB to MB of table entries. Copies are bound by memory.
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

// Lengths, the blocks of their own that copies get, and how far the free ones go.
__global__ __launch_bounds__(kThreads) void fork_kernel(ForkParams p) {
    __shared__ uint32_t waves[kWaves];
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
    }
    if (tid == 0u) {
        const uint32_t copied = min(sum.all, free_left);
        *p.n_copies = copied;
        *p.taken_out = taken + copied;
        *p.served = served;
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

// Workspace: for each block who still holds it (0: nobody; r + 1: request r, which was shortened into it, the
// largest such; kFirmly: a request that was not) and the first request that gives it up.
constexpr uint32_t kFirmly = 0xFFFFFFFFu;
constexpr uint32_t kNobody = 0xFFFFFFFFu;

struct RewindParams {
    BatchView b;
    const uint32_t* lens;
    const uint32_t* drop;
    uint32_t* free_blocks;
    const uint32_t* taken;
    uint32_t* taken_out;
    HypBlockCopy* copies;
    uint32_t* n_copies;
    uint32_t* holds;    // [num_blocks]
    uint32_t* leaves;   // [num_blocks]
};

__global__ __launch_bounds__(kEntryThreads) void rewind_clear_kernel(RewindParams p) {
    const uint32_t i = blockIdx.x * kEntryThreads + threadIdx.x;
    if (i >= p.b.num_blocks) return;
    p.holds[i] = 0u;
    p.leaves[i] = kNobody;
}

struct Shortened {
    uint32_t len, keep;
    uint32_t had, has;   // blocks
    uint32_t part;       // the block that it was shortened into and fills partly, kNobody if none
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
        if (block >= b.num_blocks) continue;
        if (e >= s.has) {
            atomicMin(&p.leaves[block], r);
        } else {
            atomicMax(&p.holds[block], e == s.part ? r + 1u : kFirmly);
        }
    }
}

__global__ __launch_bounds__(kThreads) void rewind_kernel(RewindParams p) {
    __shared__ uint32_t gone_sum[kMaxRequests + 1];   // entries given up by the requests before
    __shared__ uint32_t first_gone[kMaxRequests];     // a request's first of them
    __shared__ uint32_t waves[kWaves];
    const BatchView& b = p.b;
    const uint32_t tid = threadIdx.x;
    const uint32_t n = b.requests;
    const uint32_t per = (n + kThreads - 1u) / kThreads;
    const uint32_t first = tid * per;
    const uint32_t taken = min(*p.taken, b.num_blocks);
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
        }
        if (tid == 0u) gone_sum[n] = sum.all;
    }
    __syncthreads();
    // The blocks that go back, in order: how many, then where each goes.
    const auto back = [&](uint32_t g, uint32_t& block) {
        if (g >= sum.all) return false;
        const uint32_t r = owner(gone_sum, n, g);
        block = table_of(b, r)[first_gone[r] + (g - gone_sum[r])];
        return block < b.num_blocks && p.holds[block] == 0u && p.leaves[block] == r;
    };
    uint32_t mine = 0u, block = 0u;
    for (uint32_t g = tid; g < sum.all; g += kThreads) mine += back(g, block) ? 1u : 0u;
    const uint32_t returned = min(block_sum(mine, waves).all, taken);
    const uint32_t c = taken - returned;
    for (uint32_t base = 0u, before = 0u; base < sum.all && before < returned; base += kThreads) {
        const bool goes = back(base + tid, block);
        const Sum here = block_sum(goes ? 1u : 0u, waves);
        if (goes && before + here.before < returned) p.free_blocks[c + before + here.before] = block;
        before += here.all;
    }
    __syncthreads();
    // Blocks that were shared and are now filled partly.
    uint32_t need = 0u, held[kPer];
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
        const uint32_t r = first + i;
        held[i] = kNobody;
        if (i >= per || r >= n || s[i].part == kNobody) continue;
        const uint32_t at = table_of(b, r)[s[i].part];
        if (at >= b.num_blocks || p.holds[at] == r + 1u) continue;
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

struct CompactParams {
    BatchView b;
    uint32_t* tables_out;
    uint32_t* prefix_out;
    uint32_t* free_blocks;
    uint32_t* taken_out;
    HypBlockCopy* copies;
    uint32_t* n_copies;
    uint32_t* to;      // [num_blocks]: where a block goes, of those that move
    uint32_t* live;    // [num_blocks]: 1 for blocks in use
    uint32_t prefix_blocks;
};

__global__ __launch_bounds__(kEntryThreads) void compact_clear_kernel(CompactParams p) {
    const uint32_t i = blockIdx.x * kEntryThreads + threadIdx.x;
    if (i < p.b.num_blocks) p.live[i] = 0u;
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
    uint32_t held, width;
    const uint32_t* const row = row_of(p, blockIdx.x, held, width);
    for (uint32_t e = blockIdx.y * kEntryThreads + threadIdx.x; e < held; e += gridDim.y * kEntryThreads) {
        const uint32_t block = row[e];
        if (block < p.b.num_blocks) p.live[block] = 1u;
    }
}

// The moves: with L blocks in use, the i-th of those from L upwards goes to the i-th free one below L.
__global__ __launch_bounds__(kThreads) void compact_kernel(CompactParams p) {
    __shared__ uint32_t waves[kWaves];
    const uint32_t tid = threadIdx.x;
    const uint32_t num = p.b.num_blocks;
    uint32_t mine = 0u;
    for (uint32_t i = tid; i < num; i += kThreads) mine += p.live[i];
    const uint32_t count = block_sum(mine, waves).all;
    uint32_t movers = 0u, holes = 0u;
    for (uint32_t base = 0u; base < num; base += kThreads) {
        const uint32_t i = base + tid;
        const bool live = i < num && p.live[i] != 0u;
        const bool mover = live && i >= count;
        const bool hole = !live && i < count;
        const Sum m = block_sum(mover ? 1u : 0u, waves);
        const Sum h = block_sum(hole ? 1u : 0u, waves);
        if (mover) {
            p.copies[movers + m.before].from = i;
            p.copies[movers + m.before].tokens = 1u << p.b.shift;
        }
        if (hole) p.copies[holes + h.before].to = i;
        movers += m.all;
        holes += h.all;
    }
    __syncthreads();
    for (uint32_t i = tid; i < movers; i += kThreads) p.to[p.copies[i].from] = p.copies[i].to;
    if (tid == 0u) {
        *p.n_copies = movers;
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
        out[e] = e < held && block >= count && block < num ? p.to[block] : block;
    }
}

// ---- copy -------------------------------------------------------------------------------------

struct CopyParams {
    BatchView b;
    const HypBlockCopy* copies;
    const uint32_t* n_copies;
    uint32_t max_copies, n_caches;
    CopyCache caches[kCopyCaches];
};

// A workgroup to a block of one cache's K or V at a time.
__global__ __launch_bounds__(kEntryThreads) void copy_kernel(CopyParams p) {
    const uint32_t count = min(*p.n_copies, p.max_copies);
    const uint64_t units = static_cast<uint64_t>(count) * p.n_caches * 2u;
    for (uint64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const uint32_t which = static_cast<uint32_t>(u % (2u * p.n_caches));
        const HypBlockCopy c = p.copies[u / (2u * p.n_caches)];
        if (c.from >= p.b.num_blocks || c.to >= p.b.num_blocks || c.from == c.to) continue;
        const CopyCache& cache = p.caches[which / 2u];
        uint8_t* const base = which % 2u != 0u ? cache.v : cache.k;
        const size_t block_bytes = static_cast<size_t>(cache.token_bytes) << p.b.shift;
        const uint4* const from = reinterpret_cast<const uint4*>(base + c.from * block_bytes);
        uint4* const to = reinterpret_cast<uint4*>(base + c.to * block_bytes);
        const uint32_t words = min(c.tokens, 1u << p.b.shift) * (cache.token_bytes / 16u);
        for (uint32_t i = threadIdx.x; i < words; i += kEntryThreads) to[i] = from[i];
    }
}

// Workgroups along a row of `entries`: a few entries a thread, and no more than a long row needs.
uint32_t pieces_of(uint32_t entries) { return std::min(16u, entries / (4u * kEntryThreads) + 1u); }

}  // namespace

void launch_batch_fork(const BatchView& b, const uint32_t* lens, const uint32_t* parents, const uint32_t* free_blocks,
                       const uint32_t* taken, uint32_t* taken_out, uint32_t* served, HypBlockCopy* copies,
                       uint32_t* n_copies, hipStream_t stream) {
    const ForkParams p{b, lens, parents, free_blocks, taken, taken_out, served, copies, n_copies};
    hipLaunchKernelGGL(fork_kernel, dim3(1), dim3(kThreads), 0, stream, p);
    HYP_HIP_CHECK(hipGetLastError());
    if (b.requests == 0u || b.max_blocks == 0u) return;
    hipLaunchKernelGGL(fork_rows_kernel, dim3(b.requests, pieces_of(b.max_blocks)), dim3(kEntryThreads), 0, stream, p);
    HYP_HIP_CHECK(hipGetLastError());
}

size_t batch_pages_workspace_bytes(const BatchView& b) { return 2u * sizeof(uint32_t) * static_cast<size_t>(b.num_blocks); }

void launch_batch_rewind(const BatchView& b, const uint32_t* lens, const uint32_t* drop, uint32_t* free_blocks,
                         const uint32_t* taken, uint32_t* taken_out, HypBlockCopy* copies, uint32_t* n_copies,
                         void* workspace, hipStream_t stream) {
    uint32_t* const w = static_cast<uint32_t*>(workspace);
    const RewindParams p{b, lens, drop, free_blocks, taken, taken_out, copies, n_copies, w, w + b.num_blocks};
    if (b.requests != 0u && b.max_blocks != 0u) {
        hipLaunchKernelGGL(rewind_clear_kernel, dim3((b.num_blocks + kEntryThreads - 1u) / kEntryThreads),
                           dim3(kEntryThreads), 0, stream, p);
        HYP_HIP_CHECK(hipGetLastError());
        hipLaunchKernelGGL(rewind_mark_kernel, dim3(b.requests, pieces_of(b.max_blocks)), dim3(kEntryThreads), 0, stream, p);
        HYP_HIP_CHECK(hipGetLastError());
    }
    hipLaunchKernelGGL(rewind_kernel, dim3(1), dim3(kThreads), 0, stream, p);
    HYP_HIP_CHECK(hipGetLastError());
}

void launch_batch_compact(const BatchView& b, uint32_t* tables_out, uint32_t* prefix_out, uint32_t* free_blocks,
                          uint32_t* taken_out, HypBlockCopy* copies, uint32_t* n_copies, void* workspace,
                          hipStream_t stream) {
    uint32_t* const w = static_cast<uint32_t*>(workspace);
    const uint32_t prefix_blocks = static_cast<uint32_t>((static_cast<uint64_t>(b.prefix) + (1u << b.shift) - 1u) >> b.shift);
    const CompactParams p{b,      tables_out, prefix_out,         free_blocks, taken_out, copies,
                          n_copies, w,        w + b.num_blocks, prefix_blocks};
    const uint32_t pieces = pieces_of(std::max(b.max_blocks, prefix_blocks));
    hipLaunchKernelGGL(compact_clear_kernel, dim3((b.num_blocks + kEntryThreads - 1u) / kEntryThreads), dim3(kEntryThreads),
                       0, stream, p);
    HYP_HIP_CHECK(hipGetLastError());
    hipLaunchKernelGGL(compact_mark_kernel, dim3(b.requests + 1u, pieces), dim3(kEntryThreads), 0, stream, p);
    HYP_HIP_CHECK(hipGetLastError());
    hipLaunchKernelGGL(compact_kernel, dim3(1), dim3(kThreads), 0, stream, p);
    HYP_HIP_CHECK(hipGetLastError());
    const uint32_t wide = std::max(pieces, pieces_of(b.num_blocks));
    hipLaunchKernelGGL(compact_tables_kernel, dim3(b.requests + 2u, wide), dim3(kEntryThreads), 0, stream, p);
    HYP_HIP_CHECK(hipGetLastError());
}

void launch_batch_copy(const BatchView& b, const CopyCache* caches, uint32_t n_caches, const HypBlockCopy* copies,
                       uint32_t max_copies, const uint32_t* n_copies, hipStream_t stream) {
    for (uint32_t at = 0u; at < n_caches; at += kCopyCaches) {
        CopyParams p{b, copies, n_copies, max_copies, std::min(kCopyCaches, n_caches - at), {}};
        std::copy(caches + at, caches + at + p.n_caches, p.caches);
        const uint64_t units = static_cast<uint64_t>(max_copies) * p.n_caches * 2u;
        const uint32_t groups = static_cast<uint32_t>(std::min<uint64_t>(units, 4096u));
        hipLaunchKernelGGL(copy_kernel, dim3(groups), dim3(kEntryThreads), 0, stream, p);
        HYP_HIP_CHECK(hipGetLastError());
    }
}

}  // namespace hyperion::hip
