// A step's block tables, slot map and positions from the requests' lengths (hyp_batch_plan).
//
// Request b holds len_b tokens in ceil(len_b / bs) blocks and gets n_b more. Free blocks are a
// stack: free[taken .. num_blocks). With R the blocks of the requests that are done and
// c = taken - R, those go back to free[c .. taken) in (request, index) order, and the g-th new
// block of the step, counted over the requests in order, is free[c + g]. So everything follows
// from three running sums over the requests - rows, new blocks, returned blocks - and the
// requests are served up to the first whose rows, blocks or positions do not fit.
//
// What bounds it: the latency of its steps (lengths, sums, table entries, slots), a few KB of
// traffic. One workgroup keeps the sums in LDS and every thread finds its block's or row's
// request there by bisection. With more than kRowsHere rows the blocks and rows go to a second launch over
// all compute units: 509 prompts (352000 rows, 12000 blocks) take 14.3 us, of which the launch of the sums is about 6.
// 64 requests' decode step takes 7.1 us (7.9 with the waves' sums by LDS permutes), 6400 rows of 64 requests 10.3 in one
// launch; in two they took 1.6 us more.
#include "batch.h"
#include "common.h"
#include "wave.h"

namespace hyperion::hip {
namespace {

constexpr uint32_t kThreads = 1024;
constexpr uint32_t kWaves = kThreads / 64u;
constexpr uint32_t kPer = kMaxRequests / kThreads;   // consecutive requests of a thread
constexpr uint32_t kRowsHere = 8192;
constexpr uint32_t kRowThreads = 256;
constexpr uint32_t kRowsEach = 4;

struct PlanParams {
    BatchView b;
    const uint32_t* lens;
    const uint32_t* new_tokens;
    uint32_t* free_blocks;
    const uint32_t* taken;
    uint32_t* taken_out;
    uint32_t* served;
    uint32_t rows_here;   // the rows are written by this launch
};

// The last index i < n with sums[i] <= at (sums[0] = 0, not decreasing, at < sums[n]).
__device__ __forceinline__ uint32_t owner(const uint32_t* sums, uint32_t n, uint32_t at) {
    uint32_t lo = 0u, hi = n;
    while (hi - lo > 1u) {
        const uint32_t mid = (lo + hi) / 2u;
        if (sums[mid] <= at) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ uint32_t slot_of(const BatchView& b, uint32_t block, uint32_t token) {
    return block < b.num_blocks ? (block << b.shift) + (token & ((1u << b.shift) - 1u)) : HYP_SLOT_NONE;
}

__global__ __launch_bounds__(kThreads) void batch_plan_kernel(PlanParams p) {
    __shared__ uint32_t len_of[kMaxRequests];
    __shared__ uint32_t row_sum[kMaxRequests + 1];
    __shared__ uint32_t block_sum[kMaxRequests + 1];   // returned blocks, then new ones
    __shared__ uint64_t wave_total[3][kWaves];
    __shared__ uint32_t served_at;
    const BatchView& b = p.b;
    const uint32_t tid = threadIdx.x;
    const uint32_t lane = tid & 63u;
    const uint32_t wave = tid >> 6;
    const uint32_t n = b.requests;
    const uint32_t per = (n + kThreads - 1u) / kThreads;   // at most kPer
    const uint32_t first = tid * per;
    const uint32_t mask = (1u << b.shift) - 1u;
    const uint32_t taken = min(*p.taken, b.num_blocks);

    // This thread's requests: rows, new blocks and returned blocks, and their sums over all.
    uint32_t len[kPer], rows[kPer];
    uint64_t sum[3] = {0u, 0u, 0u};   // rows, new, returned
    const auto blocks_of = [&](uint64_t tokens) { return (tokens + mask) >> b.shift; };
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
        const uint32_t r = first + i;
        const bool live = i < per && r < n;
        len[i] = live ? p.lens[r] : 0u;
        rows[i] = live ? p.new_tokens[r] : 0u;
        if (!live) continue;
        len_of[r] = len[i];
        if (rows[i] == HYP_REQUEST_DONE) {
            sum[2] += min(blocks_of(len[i]), static_cast<uint64_t>(b.max_blocks));
        } else {
            sum[0] += rows[i];
            sum[1] += blocks_of(static_cast<uint64_t>(len[i]) + rows[i]) - blocks_of(len[i]);
        }
    }
    uint64_t before[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        const uint64_t incl = wave_incl64(sum[k]);
        before[k] = incl - sum[k];
        if (lane == 63u) wave_total[k][wave] = incl;
    }
    if (tid == 0u) served_at = n;
    __syncthreads();
    uint64_t returned_all = 0u;
    for (uint32_t w = 0; w < kWaves; ++w) {
#pragma unroll
        for (int k = 0; k < 3; ++k)
            if (w < wave) before[k] += wave_total[k][w];
        returned_all += wave_total[2][w];
    }
    const uint32_t returned = static_cast<uint32_t>(min(returned_all, static_cast<uint64_t>(taken)));
    const uint32_t c = taken - returned;
    const uint32_t avail = b.num_blocks - c;

    // The first request that does not fit; returned blocks' sums for the bisection.
    {
        uint64_t r_sum = before[0], n_sum = before[1], b_sum = before[2];
        uint32_t fails = n;
#pragma unroll
        for (uint32_t i = 0; i < kPer; ++i) {
            const uint32_t r = first + i;
            if (i >= per || r >= n) continue;
            block_sum[r] = static_cast<uint32_t>(min(b_sum, static_cast<uint64_t>(returned)));
            if (rows[i] == HYP_REQUEST_DONE) {
                b_sum += min(blocks_of(len[i]), static_cast<uint64_t>(b.max_blocks));
                continue;
            }
            const uint64_t total = static_cast<uint64_t>(len[i]) + rows[i];
            r_sum += rows[i];
            n_sum += blocks_of(total) - blocks_of(len[i]);
            if (r_sum > b.max_rows || n_sum > avail || blocks_of(total) > b.max_blocks ||
                b.prefix + total > kMaxPositions) {
                fails = min(fails, r);
            }
        }
        if (fails < n) atomicMin(&served_at, fails);
        if (tid == 0u) block_sum[n] = returned;
    }
    __syncthreads();
    const uint32_t served = served_at;

    // The blocks of the requests that are done go back first: new ones may be among them.
    for (uint32_t r = tid; r < returned; r += kThreads) {
        const uint32_t at = owner(block_sum, n, r);
        p.free_blocks[c + r] = b.tables[static_cast<size_t>(at) * b.max_blocks + (r - block_sum[at])];
    }
    __syncthreads();
    {
        uint64_t r_sum = before[0], n_sum = before[1];
#pragma unroll
        for (uint32_t i = 0; i < kPer; ++i) {
            const uint32_t r = first + i;
            if (i >= per || r >= n) continue;
            const bool done = rows[i] == HYP_REQUEST_DONE;
            const bool in = r < served && !done;
            if (r <= served) {   // (from `served` on the sums stay where they are)
                row_sum[r] = static_cast<uint32_t>(r_sum);
                block_sum[r] = static_cast<uint32_t>(n_sum);
            }
            if (in) {
                r_sum += rows[i];
                n_sum += blocks_of(static_cast<uint64_t>(len[i]) + rows[i]) - blocks_of(len[i]);
            }
            b.lens[r] = done ? 0u : (in ? len[i] + rows[i] : len[i]);
            if (r + 1u == n && served == n) {
                row_sum[n] = static_cast<uint32_t>(r_sum);
                block_sum[n] = static_cast<uint32_t>(n_sum);
            }
        }
        if (n == 0u && tid == 0u) row_sum[0] = block_sum[0] = 0u;
    }
    __syncthreads();
    const uint32_t total = row_sum[served];
    const uint32_t fresh = block_sum[served];
    for (uint32_t r = tid; r <= n; r += kThreads) b.row_start[r] = r < served ? row_sum[r] : total;
    if (tid == 0u) {
        *p.taken_out = c + fresh;
        *p.served = served;
    }
    if (p.rows_here == 0u) return;
    for (uint32_t g = tid; g < fresh; g += kThreads) {
        const uint32_t r = owner(block_sum, served, g);
        const uint32_t entry = static_cast<uint32_t>(blocks_of(len_of[r])) + (g - block_sum[r]);
        b.tables[static_cast<size_t>(r) * b.max_blocks + entry] = p.free_blocks[c + g];
    }
    for (uint32_t t = tid; t < b.max_rows; t += kThreads) {
        uint32_t slot = HYP_SLOT_NONE;
        uint32_t pos = 0u;
        if (t < total) {
            const uint32_t r = owner(row_sum, served, t);
            const uint32_t token = len_of[r] + (t - row_sum[r]);
            const uint32_t entry = token >> b.shift;
            const uint32_t have = static_cast<uint32_t>(blocks_of(len_of[r]));
            const uint32_t block = entry < have ? b.tables[static_cast<size_t>(r) * b.max_blocks + entry]
                                                : p.free_blocks[c + block_sum[r] + (entry - have)];
            slot = slot_of(b, block, token);
            pos = b.prefix + token;
        }
        b.slots[t] = slot;
        b.positions[t] = pos;
    }
}

// The new blocks and rows of a large step. lens holds the lengths with this step's rows, so row i of request b is
// token lens[b] - rows of b + i, and a request's new blocks follow from the two: every workgroup forms their sums
// for itself. A new block holds a new row, whose first one writes the table's entry.
__global__ __launch_bounds__(kRowThreads) void batch_rows_kernel(PlanParams p) {
    __shared__ uint32_t len_of[kMaxRequests];   // before the step
    __shared__ uint32_t row_sum[kMaxRequests + 1];
    __shared__ uint32_t block_sum[kMaxRequests];
    __shared__ uint32_t wave_total[kRowThreads / 64u];
    const BatchView& b = p.b;
    const uint32_t tid = threadIdx.x;
    const uint32_t n = b.requests;
    const uint32_t mask = (1u << b.shift) - 1u;
    const uint32_t taken = *p.taken_out;
    for (uint32_t r = tid; r <= n; r += kRowThreads) {
        row_sum[r] = b.row_start[r];
        if (r < n) len_of[r] = b.lens[r];
    }
    __syncthreads();
    const uint32_t total = row_sum[n];
    const uint32_t per = (n + kRowThreads - 1u) / kRowThreads;
    const uint32_t begin = min(tid * per, n);
    const uint32_t end = min(begin + per, n);
    uint32_t sum = 0u;
    for (uint32_t r = begin; r < end; ++r) {
        const uint32_t after = len_of[r];
        const uint32_t len = after - (row_sum[r + 1u] - row_sum[r]);
        len_of[r] = len;
        block_sum[r] = sum;
        sum += ((after + mask) >> b.shift) - ((len + mask) >> b.shift);
    }
    const uint32_t incl = wave_incl(sum);
    if ((tid & 63u) == 63u) wave_total[tid >> 6] = incl;
    __syncthreads();
    uint32_t before = incl - sum;
    uint32_t fresh = 0u;
    for (uint32_t w = 0; w < kRowThreads / 64u; ++w) {
        if (w < tid >> 6) before += wave_total[w];
        fresh += wave_total[w];
    }
    for (uint32_t r = begin; r < end; ++r) block_sum[r] += before;
    __syncthreads();
    const uint32_t c = taken - fresh;
#pragma unroll
    for (uint32_t i = 0; i < kRowsEach; ++i) {
        const uint32_t t = (blockIdx.x * kRowsEach + i) * kRowThreads + tid;
        if (t >= b.max_rows) continue;
        uint32_t slot = HYP_SLOT_NONE;
        uint32_t pos = 0u;
        if (t < total) {
            const uint32_t r = owner(row_sum, n, t);
            const uint32_t token = len_of[r] + (t - row_sum[r]);
            const uint32_t entry = token >> b.shift;
            const uint32_t have = (len_of[r] + mask) >> b.shift;
            uint32_t* const at = b.tables + static_cast<size_t>(r) * b.max_blocks + entry;
            const uint32_t block = entry < have ? *at : p.free_blocks[c + block_sum[r] + (entry - have)];
            if ((token & mask) == 0u) *at = block;
            slot = slot_of(b, block, token);
            pos = b.prefix + token;
        }
        b.slots[t] = slot;
        b.positions[t] = pos;
    }
}

}  // namespace

void launch_batch_plan(const BatchView& b, const uint32_t* lens, const uint32_t* new_tokens, uint32_t* free_blocks,
                       const uint32_t* taken, uint32_t* taken_out, uint32_t* served, hipStream_t stream) {
    HYP_REQUIRE(b.requests <= kMaxRequests, HYP_STATUS_INVALID_ARGUMENT, "batch plan: too many requests");
    const bool here = b.max_rows <= kRowsHere;
    const PlanParams p{b, lens, new_tokens, free_blocks, taken, taken_out, served, here ? 1u : 0u};
    hipLaunchKernelGGL(batch_plan_kernel, dim3(1), dim3(kThreads), 0, stream, p);
    HYP_HIP_CHECK(hipGetLastError());
    if (here) return;
    const uint32_t per = kRowThreads * kRowsEach;
    hipLaunchKernelGGL(batch_rows_kernel, dim3((b.max_rows + per - 1u) / per), dim3(kRowThreads), 0, stream, p);
    HYP_HIP_CHECK(hipGetLastError());
}

}  // namespace hyperion::hip
