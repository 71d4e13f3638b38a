// OCP MX codes to 16-bit operands of the matrix cores, by the hardware's conversions: v_cvt_scalef32_pk_{bf16,f16}_{fp4,fp8} turns two codes into
// a pair of values and multiplies by the power of two in the exponent field of its scale operand -- an E8M0 byte shifted into place, with
// E8M0's own meaning of 0 (2^-127) and 255 (NaN).
#pragma once
#include "common.hpp"

namespace mfq {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

template <int XF16>
__device__ __forceinline__ float4_t mx_mfma(u32x4_t a, u32x4_t b, float4_t c) {
    if constexpr (XF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
// eight E2M1 codes of a dword -> eight values of the activations' type, times 2^(exponent field of scale - 127)
template <int XF16>
__device__ __forceinline__ u32x4_t mx_cvt_fp4(uint32_t q, float scale) {
    u32x4_t b;
    if constexpr (XF16) {
        b.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, scale, 0));
        b.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, scale, 1));
        b.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, scale, 2));
        b.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, scale, 3));
    } else {
        b.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 0));
        b.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 1));
        b.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 2));
        b.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 3));
    }
    return b;
}
// eight E4M3FN codes of two dwords
template <int XF16>
__device__ __forceinline__ u32x4_t mx_cvt_fp8(uint32_t q0, uint32_t q1, float scale) {
    u32x4_t b;
    if constexpr (XF16) {
        b.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(q0, scale, false));
        b.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(q0, scale, true));
        b.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(q1, scale, false));
        b.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(q1, scale, true));
    } else {
        b.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q0, scale, false));
        b.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q0, scale, true));
        b.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q1, scale, false));
        b.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q1, scale, true));
    }
    return b;
}

}  // namespace mfq
