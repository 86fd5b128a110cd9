// Operand types and moves of the attention kernels that form their scores transposed
// (attention_chunk.hip, attention_batch.hip).
#pragma once

#include "attention.h"
#include "common.h"

namespace hyperion::hip {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint16_t u16x8_t __attribute__((ext_vector_type(8)));
typedef short short4_t __attribute__((ext_vector_type(4)));

#define HYP_LDS __attribute__((address_space(3)))
#define HYP_GLOBAL __attribute__((address_space(1)))

// The other half-wave's value (lane ^ 32) combined with this lane's.
__device__ __forceinline__ float half_max(float v) {
    float u = v, c = v;
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(u), "+v"(c));
    return fmaxf(u, c);
}

__device__ __forceinline__ float half_sum(float v) {
    float u = v, c = v;
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(u), "+v"(c));
    return u + c;
}

__device__ __forceinline__ bf16x8_t lds_read16(uint32_t at) {
    return *reinterpret_cast<const HYP_LDS bf16x8_t*>(at);
}

// A transposing read. The pointer is restrict so that the read carries alias information:
// without any, the compiler puts a wait for the loads to LDS in flight (the next block's)
// ahead of it. The block's own loads are waited for explicitly.
__device__ __forceinline__ short4_t lds_read_tr4(HYP_LDS short4_t* __restrict at) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(at);
}

// 8 keys of one dim per lane (two transposing reads of 4 keys, `hi` bytes apart).
__device__ __forceinline__ bf16x8_t lds_read_tr(uint32_t at, uint32_t hi) {
    const short4_t a = lds_read_tr4(reinterpret_cast<HYP_LDS short4_t*>(at));
    const short4_t b = lds_read_tr4(reinterpret_cast<HYP_LDS short4_t*>(at + hi));
    return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Eight probabilities rounded to bf16, a lane's operand of one product.
__device__ __forceinline__ bf16x8_t round_p(const float* p) {
    return __builtin_bit_cast(bf16x8_t, make_uint4(cvt_pk_bf16(p[0], p[1]), cvt_pk_bf16(p[2], p[3]),
                                                   cvt_pk_bf16(p[4], p[5]), cvt_pk_bf16(p[6], p[7])));
}

}  // namespace hyperion::hip
