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
// bf16's lowest value 25 us at temperature 0.8, 1125 in windows at 2; with values past 2^7 566.
//
// What bounds it: the steps' latency (the second launch takes 13 to 16 us whatever the rows: 3 for the counts, 3.5 for the
// weights, 3 for the filters and the draw, 3 for the token) and the LDS additions (64 rows of 262144: 9.5 us of
// counting). One row of 262144 takes 18.4 us, 64 rows 24.0, 200 rows of 50001 21.8.
#include <cstdint>

#include "common.h"
#include "kernels.h"
#include "sample_batch.h"
#include "sample_row.h"

namespace hyperion::hip {
namespace {

using namespace sampling;

__global__ __launch_bounds__(kThreads) void sample_count_kernel(const uint16_t* __restrict__ logits, uint32_t vocab,
                                                                Chunks chunks, ChunkCounts* __restrict__ counts) {
    __shared__ RowLds s;
    const uint32_t row = blockIdx.x / chunks.n;
    const uint32_t begin = min(vocab, (blockIdx.x - row * chunks.n) * chunks.tokens);
    count_values(logits + static_cast<size_t>(row) * vocab, begin, min(vocab, begin + chunks.tokens), s);
    store_counts(s, counts[blockIdx.x]);
}

template <bool kSplit>
__global__ __launch_bounds__(kThreads) void sample_rows_kernel(const uint16_t* __restrict__ logits, uint32_t vocab,
                                                               const HypSamplingConfig* __restrict__ configs,
                                                               const float* __restrict__ uniforms, Chunks chunks,
                                                               const ChunkCounts* __restrict__ counts,
                                                               uint32_t* __restrict__ tokens, float* __restrict__ logprobs) {
    __shared__ RowLds s;
    const uint32_t tid = threadIdx.x;
    const uint32_t row_at = blockIdx.x;
    const uint16_t* row = logits + static_cast<size_t>(row_at) * vocab;
    const RowParams prm = row_params(configs[row_at], uniforms[row_at]);

    // 1. Counts by value.
    if constexpr (kSplit) {
        counts += static_cast<size_t>(row_at) * chunks.n;
        sum_counts(counts, chunks.n, s);
    } else {
        count_values(row, 0u, vocab, s);
    }

    // 2. The drawn value and the token's number among those of that value.
    if (!find_row<true>(row, vocab, prm, s)) {
        if (tid == 0u) {
            tokens[row_at] = 0u;
            if (logprobs != nullptr) logprobs[row_at] = -__builtin_huge_valf();
        }
        return;
    }
    const double logprob = (s.infinite != 0u ? 0.0 : (value_of(s.drawn) - s.top) * prm.by_t) - log(s.total);

    // 3. The token, in the row or in the chunk that holds it.
    find_token<kSplit>(row, vocab, chunks, counts, s, [&](uint32_t token) {
        tokens[row_at] = token;
        if (logprobs != nullptr) logprobs[row_at] = static_cast<float>(logprob);
    });
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
