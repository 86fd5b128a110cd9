// A step of batched serving as the kernels see it (HypBatch, hyperion_hip.h): requests whose
// tokens lie in blocks of one paged cache per layer, behind a prefix that all of them share.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "hyperion_hip.h"

namespace hyperion::hip {

constexpr uint32_t kMaxRequests = 4096;            // their running sums fit one workgroup's LDS
constexpr uint32_t kMaxBatchRows = 1u << 20;
constexpr uint32_t kMaxPositions = 1u << 24;       // positions are exact in fp32 below

// Whether two arrays of so many bytes share any.
inline bool overlap(const void* a, uint64_t a_bytes, const void* b, uint64_t b_bytes) {
    const uint64_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + b_bytes && y < x + a_bytes;
}

struct BatchView {
    uint32_t requests, shift, num_blocks, max_blocks, max_rows, prefix;   // block size 1 << shift
    const uint32_t* prefix_table;
    uint32_t* tables;      // [requests][max_blocks]
    uint32_t* lens;        // [requests]
    uint32_t* row_start;   // [requests + 1]
    uint32_t* slots;       // [max_rows]
    uint32_t* positions;   // [max_rows]
};

void launch_batch_plan(const BatchView& b, const uint32_t* lens, const uint32_t* new_tokens, uint32_t* free_blocks,
                       const uint32_t* taken, uint32_t* taken_out, uint32_t* served, hipStream_t stream);

struct BatchPrepareArgs {
    const uint16_t* q;       // [max_rows][n_heads][head_dim]
    const uint16_t* k_raw;   // [max_rows][n_kv_heads][head_dim]
    const uint16_t* v_raw;   // the same, or null: V = norm(k_raw)
    const uint16_t* q_norm;
    const uint16_t* k_norm;
    uint16_t* q_out;
    uint16_t* cache_k;       // [capacity][n_kv_heads][head_dim]
    uint16_t* cache_v;
    uint32_t n_heads, n_kv_heads, head_dim, rotated, capacity;
    float base, eps;
};
void launch_batch_prepare(const BatchView& b, const BatchPrepareArgs& a, hipStream_t stream);

struct BatchAttentionArgs {
    const uint16_t* q;         // [max_rows][n_heads][head_dim]
    const uint16_t* cache_k;   // [capacity][n_kv_heads][head_dim]
    const uint16_t* cache_v;
    uint16_t* out;
    void* workspace;
    size_t workspace_bytes;
    uint32_t n_heads, n_kv_heads, head_dim, window;
    float scale;
};
size_t batch_attention_workspace_bytes(const BatchView& b, uint32_t n_heads, uint32_t head_dim);
void launch_batch_attention(const BatchView& b, const BatchAttentionArgs& a, hipStream_t stream);

}  // namespace hyperion::hip
