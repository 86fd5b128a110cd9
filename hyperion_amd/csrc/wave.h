// Sums and scans over the 64 lanes of a wave, all of them active.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace hyperion::hip {

__device__ __forceinline__ uint32_t from_lane(uint32_t v, uint32_t lane) {
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}

// Inclusive scan over the wave by register moves between lanes: 1, 2, 4 and 8 lanes on within rows of
// 16, then the last lane of row 0 and 2 to the next row, of row 1 to the upper half. `none` is the operation's
// neutral value. (Through LDS permutes a reduction takes six times their latency, and a call forms ten.)
template <typename Op>
__device__ __forceinline__ uint32_t wave_scan(uint32_t v, uint32_t none, Op&& op) {
    const int n = static_cast<int>(none);
    v = op(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(n, static_cast<int>(v), 0x111, 0xF, 0xF, false)));
    v = op(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(n, static_cast<int>(v), 0x112, 0xF, 0xF, false)));
    v = op(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(n, static_cast<int>(v), 0x114, 0xF, 0xF, false)));
    v = op(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(n, static_cast<int>(v), 0x118, 0xF, 0xF, false)));
    v = op(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(n, static_cast<int>(v), 0x142, 0xA, 0xF, false)));
    return op(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(n, static_cast<int>(v), 0x143, 0xC, 0xF, false)));
}
__device__ __forceinline__ uint32_t wave_incl(uint32_t v) {
    return wave_scan(v, 0u, [](uint32_t a, uint32_t b) { return a + b; });
}
__device__ __forceinline__ uint32_t wave_sum(uint32_t v) { return from_lane(wave_incl(v), 63u); }
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    return from_lane(wave_scan(v, 0u, [](uint32_t a, uint32_t b) { return max(a, b); }), 63u);
}
__device__ __forceinline__ int32_t wave_min(int32_t v) {
    return static_cast<int32_t>(from_lane(wave_scan(static_cast<uint32_t>(v), 0x7FFFFFFFu, [](uint32_t a, uint32_t b) {
        return static_cast<uint32_t>(min(static_cast<int32_t>(a), static_cast<int32_t>(b)));
    }), 63u));
}
// Inclusive sums of 64-bit values, in the same steps.
template <typename T>
__device__ __forceinline__ T wave_incl64(T v) {
    static_assert(sizeof(T) == 8u, "two registers");
    const auto step = [](T v, auto moved) __attribute__((always_inline)) {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        const uint64_t lo = static_cast<uint32_t>(moved(static_cast<int>(static_cast<uint32_t>(b))));
        const uint64_t hi = static_cast<uint32_t>(moved(static_cast<int>(static_cast<uint32_t>(b >> 32))));
        return v + __builtin_bit_cast(T, lo | hi << 32);
    };
    v = step(v, [](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false); });
    v = step(v, [](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false); });
    v = step(v, [](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false); });
    v = step(v, [](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false); });
    v = step(v, [](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false); });
    return step(v, [](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false); });
}

}  // namespace hyperion::hip
