// Element types of the stand-alone operators (add_rmsnorm, route_logits, w4_matvec) and the
// conversions between them and fp32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/moe_b200.h"

namespace moe {
namespace op {

__host__ __device__ constexpr int size_of(int dtype) {
    return dtype == MOE_B200_DTYPE_F32 ? 4 : dtype == MOE_B200_DTYPE_E4M3 ? 1 : 2;
}

// 16 bits of type bf16 or f16 -> fp32.
__device__ __forceinline__ float half_to_float(uint32_t bits16, int dtype) {
    return dtype == MOE_B200_DTYPE_BF16 ? __uint_as_float(bits16 << 16)
                                        : __half2float(__ushort_as_half((unsigned short)bits16));
}

// fp32 -> 16 bits of type bf16 or f16, round to nearest even.
__device__ __forceinline__ uint32_t float_to_half(float f, int dtype) {
    return dtype == MOE_B200_DTYPE_BF16 ? (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(f))
                                        : (uint32_t)__half_as_ushort(__float2half_rn(f));
}

// Two fp32 -> packed bf16x2 / f16x2 (one conversion instruction), `lo` in the low half.
__device__ __forceinline__ uint32_t floats_to_half2(float lo, float hi, int dtype) {
    uint32_t r;
    if (dtype == MOE_B200_DTYPE_BF16)
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Two fp32 -> two e4m3 codes, `lo` in the low byte.  Values beyond 448 saturate, NaN stays NaN.
__device__ __forceinline__ uint32_t floats_to_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ float load_as_float(const void* p, long long i, int dtype) {
    return dtype == MOE_B200_DTYPE_F32 ? static_cast<const float*>(p)[i]
                                       : half_to_float(static_cast<const uint16_t*>(p)[i], dtype);
}

__device__ __forceinline__ void store_from_float(void* p, long long i, int dtype, float v) {
    if (dtype == MOE_B200_DTYPE_F32)
        static_cast<float*>(p)[i] = v;
    else
        static_cast<uint16_t*>(p)[i] = (uint16_t)float_to_half(v, dtype);
}

// 2^(byte - 127) of an e8m0 byte, byte 0 included (an fp32 subnormal).  Byte 255 is NaN.
__device__ __forceinline__ float e8m0_to_float(uint32_t byte) {
    return __uint_as_float(byte == 255 ? 0x7FC00000u : max(byte << 23, 0x00400000u));
}

}  // namespace op
}  // namespace moe
