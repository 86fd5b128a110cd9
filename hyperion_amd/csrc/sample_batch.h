// Batch sampling from given uniforms; see sample_batch.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "hyperion_hip.h"

namespace hyperion::hip {

uint32_t sample_batch_max_vocab();
size_t sample_batch_workspace_bytes(uint32_t rows, uint32_t vocab);
// tokens[r] (and logprobs[r], unless null) of each of `rows` rows of vocab bf16 logits, drawn with
// configs[r] and uniforms[r]; all device memory.
void launch_sample_batch(const uint16_t* logits, uint32_t rows, uint32_t vocab, const HypSamplingConfig* configs,
                         const float* uniforms, uint32_t* tokens, float* logprobs, void* workspace,
                         size_t workspace_bytes, hipStream_t stream);

}  // namespace hyperion::hip
