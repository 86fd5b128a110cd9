// Operations on the blocks of a batch's requests; see batch_pages.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "batch.h"
#include "hyperion_hip.h"

namespace hyperion::hip {

void launch_batch_fork(const BatchView& b, const uint32_t* lens, const uint32_t* parents, const uint32_t* free_blocks,
                       const uint32_t* taken, uint32_t* taken_out, uint32_t* served, HypBlockCopy* copies,
                       uint32_t* n_copies, hipStream_t stream);

// What launch_batch_rewind and launch_batch_compact need.
size_t batch_pages_workspace_bytes(const BatchView& b);
void launch_batch_rewind(const BatchView& b, const uint32_t* lens, const uint32_t* drop, uint32_t* free_blocks,
                         const uint32_t* taken, uint32_t* taken_out, HypBlockCopy* copies, uint32_t* n_copies,
                         void* workspace, hipStream_t stream);
void launch_batch_compact(const BatchView& b, uint32_t* tables_out, uint32_t* prefix_out, uint32_t* free_blocks,
                          uint32_t* taken_out, HypBlockCopy* copies, uint32_t* n_copies, void* workspace,
                          hipStream_t stream);

// One cache's K and V as launch_batch_copy takes them: bytes of a token, a multiple of 16.
struct CopyCache {
    uint8_t* k;
    uint8_t* v;
    uint64_t token_bytes;
};
constexpr uint32_t kCopyCaches = 128;   // of one launch: they travel as its arguments
void launch_batch_copy(const BatchView& b, const CopyCache* caches, uint32_t n_caches, const HypBlockCopy* copies,
                       uint32_t max_copies, const uint32_t* n_copies, hipStream_t stream);

}  // namespace hyperion::hip
