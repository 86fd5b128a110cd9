// Verification of drafted tokens; see verify_batch.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "hyperion_hip.h"

namespace hyperion::hip {

struct VerifyArgs {
    const uint16_t* logits;         // [rows][vocab]
    const uint16_t* draft_logits;   // the same, or null: drafts without a distribution
    uint32_t rows, vocab, requests;
    const uint32_t* row_start;      // [requests + 1]
    const uint32_t* ids;            // [rows]
    const HypSamplingConfig* configs;         // [requests]
    const HypSamplingConfig* draft_configs;
    const float* uniforms;          // [rows]
    uint32_t* accepted;             // [requests]
    uint32_t* rejected;
    uint32_t* tokens;
    float* logprobs;                // [rows], or null
    void* workspace;
};
size_t verify_batch_workspace_bytes(uint32_t rows, uint32_t vocab, uint32_t requests, bool drafted);
void launch_verify_batch(const VerifyArgs& a, hipStream_t stream);

}  // namespace hyperion::hip
