// From the q/k/v projections of a batch's rows to the paged cache (hyp_batch_prepare): row t
// stands at positions[t] and its K and V go to slots[t],
//   y = x / sqrt(mean(x^2) + eps) * w,  then pairs (i, i + D/2) with i < rotated / 2 turned by
//   theta_i = fp32(position) * fp32(base^(-2i / D))
// for q and K; V takes the norm alone, without a weight. Everything from the bf16 input to the
// one rounding of the output is fp32 (the angle's cosine and sine come from fp64 arithmetic, as
// rope_kernel's do), so nothing is rounded between the norm and the rotation.
//
// D/8 lanes hold a head's row, 8 consecutive values each: the sum of squares meets in a butterfly
// over them and the two values of a pair lie half those lanes apart, so nothing but the angles
// goes through LDS. A workgroup computes its token's angles once for all of the token's heads
// (their fp64 cosines and sines would otherwise be the kernel's largest part), behind the first
// heads' loads.
//
// What bounds it: HBM for chunks (2 B read and written per value; 2047 rows of 16 heads and one kv head of 512: 16.0 us,
// 4.6 TB/s), latency for a decode step (48 rows of 16 heads and 8 of 256: 4.9 us).
#include <algorithm>
#include <cmath>

#include "batch.h"
#include "common.h"
#include "kernels.h"
#include "q4_rmsnorm.h"

namespace hyperion::hip {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kGridTarget = 2048;   // workgroups: a few for each compute unit

struct PrepareParams {
    BatchPrepareArgs a;
    const uint32_t* row_end;   // the step's rows
    const uint32_t* slots;
    const uint32_t* positions;
    double log2_base;
};

__device__ __forceinline__ void unpack8(const uint4& w, float (&f)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        f[2 * e] = __uint_as_float(u[e] << 16);
        f[2 * e + 1] = __uint_as_float(u[e] & 0xFFFF0000u);
    }
}

__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    return make_uint4(cvt_pk_bf16(f[0], f[1]), cvt_pk_bf16(f[2], f[3]), cvt_pk_bf16(f[4], f[5]), cvt_pk_bf16(f[6], f[7]));
}

// 1 / sqrt(mean + eps) of the row that LPR lanes hold.
template <uint32_t LPR>
__device__ __forceinline__ float row_inverse(const float (&f)[8], float eps, uint32_t lane) {
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss);
    ss += xor_lanes<1>(ss, lane);
    ss += xor_lanes<2>(ss, lane);
    ss += xor_lanes<4>(ss, lane);
    if constexpr (LPR >= 16u) ss += xor_lanes<8>(ss, lane);
    if constexpr (LPR >= 32u) ss = add_lane_xor16(ss);
    if constexpr (LPR >= 64u) ss = add_lane_xor32(ss);
    return 1.0f / sqrtf(ss / static_cast<float>(8u * LPR) + eps);
}

template <uint32_t D>
__global__ __launch_bounds__(kThreads) void batch_prepare_kernel(PrepareParams p) {
    constexpr uint32_t kLanes = D / 8u;
    constexpr uint32_t kHalf = D / 2u;
    constexpr uint32_t kRows = kThreads / kLanes;   // heads of one pass
    __shared__ __attribute__((aligned(16))) float2 angle[kHalf];
    const uint32_t t = blockIdx.x;
    if (t >= *p.row_end) return;   // uniform: rows behind the last request's stay as they are
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t c = threadIdx.x % kLanes;
    const uint32_t heads = p.a.n_heads + p.a.n_kv_heads;
    const uint32_t slot = p.slots[t];
    const bool stored = slot < p.a.capacity;
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);

    struct Row {
        uint4 x, w, v;
    };
    const auto load = [&](uint32_t hh) {
        Row r{zero, zero, zero};
        if (hh < p.a.n_heads) {
            r.x = reinterpret_cast<const uint4*>(p.a.q + (static_cast<size_t>(t) * p.a.n_heads + hh) * D)[c];
            r.w = reinterpret_cast<const uint4*>(p.a.q_norm)[c];
        } else if (hh < heads) {
            const size_t row = (static_cast<size_t>(t) * p.a.n_kv_heads + (hh - p.a.n_heads)) * D;
            r.x = reinterpret_cast<const uint4*>(p.a.k_raw + row)[c];
            r.w = reinterpret_cast<const uint4*>(p.a.k_norm)[c];
            if (p.a.v_raw != nullptr) r.v = reinterpret_cast<const uint4*>(p.a.v_raw + row)[c];
        }
        return r;
    };
    uint32_t hh = blockIdx.y * kRows + threadIdx.x / kLanes;
    Row r = load(hh);

    const float pos = static_cast<float>(p.positions[t]);
    for (uint32_t i = threadIdx.x; i < kHalf; i += kThreads) {
        float2 cs = make_float2(1.0f, 0.0f);
        if (2u * i < p.a.rotated) {
            const float inv = static_cast<float>(exp2(-2.0 * i / static_cast<double>(D) * p.log2_base));
            double s, co;
            sincos(static_cast<double>(pos * inv), &s, &co);
            cs = make_float2(static_cast<float>(co), static_cast<float>(s));
        }
        angle[i] = cs;
    }
    __syncthreads();
    float2 cs[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float4 v = reinterpret_cast<const float4*>(angle + (c % (kLanes / 2u)) * 8u)[e];
        cs[2 * e] = make_float2(v.x, v.y);
        cs[2 * e + 1] = make_float2(v.z, v.w);
    }
    const float side = c < kLanes / 2u ? -1.0f : 1.0f;
    const uint32_t passes = (heads + kRows - 1u) / kRows;
    for (uint32_t pass = blockIdx.y; pass < passes; pass += gridDim.y) {
        const Row next = load(hh + gridDim.y * kRows);   // (past the last head: nothing)
        float f[8], w[8], v[8];
        unpack8(r.x, f);
        unpack8(r.w, w);
        unpack8(p.a.v_raw != nullptr ? r.v : r.x, v);
        const float inv = row_inverse<kLanes>(f, p.a.eps, lane);
        const float inv_v = p.a.v_raw != nullptr ? row_inverse<kLanes>(v, p.a.eps, lane) : inv;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = f[e] * inv * w[e];
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float other = __shfl_xor(f[e], kLanes / 2u);
            y[e] = f[e] * cs[e].x + side * (other * cs[e].y);
        }
        if (hh < p.a.n_heads) {
            reinterpret_cast<uint4*>(p.a.q_out + (static_cast<size_t>(t) * p.a.n_heads + hh) * D)[c] = pack8(y);
        } else if (hh < heads && stored) {
            const size_t row = (static_cast<size_t>(slot) * p.a.n_kv_heads + (hh - p.a.n_heads)) * D;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= inv_v;
            reinterpret_cast<uint4*>(p.a.cache_k + row)[c] = pack8(y);
            reinterpret_cast<uint4*>(p.a.cache_v + row)[c] = pack8(v);
        }
        r = next;
        hh += gridDim.y * kRows;
    }
}

}  // namespace

void launch_batch_prepare(const BatchView& b, const BatchPrepareArgs& a, hipStream_t stream) {
    const PrepareParams p{a, b.row_start + b.requests, b.slots, b.positions, log2(static_cast<double>(a.base))};
    const uint32_t rows = kThreads / (a.head_dim / 8u);
    const uint32_t passes = (a.n_heads + a.n_kv_heads + rows - 1u) / rows;
    const uint32_t y = std::max(1u, std::min(passes, kGridTarget / b.max_rows));
    const dim3 grid(b.max_rows, y);
    switch (a.head_dim) {
        case 64: hipLaunchKernelGGL(batch_prepare_kernel<64>, grid, dim3(kThreads), 0, stream, p); break;
        case 128: hipLaunchKernelGGL(batch_prepare_kernel<128>, grid, dim3(kThreads), 0, stream, p); break;
        case 256: hipLaunchKernelGGL(batch_prepare_kernel<256>, grid, dim3(kThreads), 0, stream, p); break;
        case 512: hipLaunchKernelGGL(batch_prepare_kernel<512>, grid, dim3(kThreads), 0, stream, p); break;
        default: throw NativeError(HYP_STATUS_UNSUPPORTED, "batch prepare: head_dim must be 64, 128, 256 or 512");
    }
    HYP_HIP_CHECK(hipGetLastError());
}

}  // namespace hyperion::hip
