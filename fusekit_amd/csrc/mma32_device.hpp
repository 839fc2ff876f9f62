// 32x32x16 bf16 matrix instructions whose sums stay in VGPRs, and what goes with them: the attention kernels over a group of rows share
// these (sdpa_prefill.hip, sdpa_paged.hip).
#pragma once
#include "dma_device.hpp"

namespace fk {

typedef __bf16 pf_bf16x8_t __attribute__((ext_vector_type(8)));
typedef float pf_f32x16_t __attribute__((ext_vector_type(16)));
typedef unsigned int pf_u32x2_t __attribute__((ext_vector_type(2)));
typedef unsigned int pf_u32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float other_half_max(float v) {
    const pf_u32x2_t r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float both_halves_sum(float v) {
    const pf_u32x2_t r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

typedef short pf_s16x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ void mfma32_acc(pf_f32x16_t& acc, const pf_u32x4_t& a, const pf_u32x4_t& b) {
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(acc) : "v"(a), "v"(b));
}

// scores stay in VGPRs, where the softmax takes them
template <bool FIRST>
__device__ __forceinline__ void mfma32_scores(pf_f32x16_t& s, const pf_u32x4_t& a, const pf_u32x4_t& b) {
    if constexpr (FIRST) asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(s) : "v"(a), "v"(b));
    else asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(s) : "v"(a), "v"(b));
}

}  // namespace fk
