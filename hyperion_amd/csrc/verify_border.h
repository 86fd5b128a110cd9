// Where a row's filters end among the values of a wave's lanes, for verify_batch.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "wave.h"

namespace hyperion::hip {

// A lane's values are first weighed from one to the next by a factor, and summed as a whole: within 2^-44 of what each
// value's own weight says (32 factors of two roundings each, exponents of up to 104 rounded to 53 bits, some fifty
// additions). So that only names the lanes in whose values a filter may end, with 2^-40 to spare. Whether it does is
// decided by the values' own weights, and where it does not the next such lane is asked: a running sum or a weight that
// meets a border to a rounding would lose the filter otherwise, and the row would keep all its tokens.
constexpr double kSpare = 0x1p-40;
__device__ __forceinline__ bool may_be_past(double mass, double enough) { return mass > enough - enough * kSpare; }
__device__ __forceinline__ bool may_be_light(double weight, double min_p) { return weight < min_p + min_p * kSpare; }

// One value: its tokens, their weight, the tokens and the mass before it.
struct OneValue {
    uint32_t n, before, bits;
    double w, mass;
};

// How many tokens of the row the filters keep, if they end in the values of a lane in `maybe`, 0xFFFFFFFF otherwise:
// the tokens before which the running sum is below `enough` (by_mass), of weights not below min_p. spread(lane): that
// lane's values, one to a lane, in order. (By all lanes of a wave. Lanes without tokens are not in `maybe`: a wave behind
// the border would ask them all. Nearly always the first lane asked has the end; where all weights are within 2^-40 of
// min_p, at a temperature of 1e30 and a min_p of 1, every lane is: one request of 5 rows 41.6 us instead of 22.7.)
template <typename Spread>
__device__ __forceinline__ uint32_t wave_border(uint64_t maybe, bool by_mass, double enough, double min_p, Spread&& spread) {
#pragma unroll 1
    for (; maybe != 0u; maybe &= maybe - 1u) {
        const OneValue o = spread(static_cast<uint32_t>(__builtin_ctzll(maybe)));
        const bool dropped = o.n != 0u && o.w < min_p;
        const bool full = o.n != 0u && by_mass && o.n * o.w > enough - o.mass;
        uint32_t some = 0u;
        if (!dropped && full && enough > o.mass) some = min(o.n, static_cast<uint32_t>(ceil((enough - o.mass) / o.w)));
        const uint64_t ends = __ballot(dropped || full);
        if (ends != 0u) return from_lane(o.before + some, static_cast<uint32_t>(__builtin_ctzll(ends)));
    }
    return 0xFFFFFFFFu;
}

}  // namespace hyperion::hip
