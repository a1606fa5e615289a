// The 8-bit cache format: e4m3 values [num_slots, KVH, 128] and one fp32 scale for every kGrain slots and kv head
// [num_slots / kGrain, KVH]; an element stands for value * scale.
//
// The scale that the store chooses is a power of two, 2^k with the smallest k for which the largest finite magnitude of the
// block is at most 448 * 2^k.  e4m3 is a floating format, so a scale's fraction would buy no precision; a power of two makes
// a later change of the scale exact except where a value becomes subnormal, and value * scale a bf16 number (four
// significant bits), so attention over the 8-bit cache can be held bit for bit against attention over the same cache in bf16.
#pragma once

#include "common.cuh"

#include <cuda_fp16.h>

namespace nvllm {
namespace q8 {

constexpr int kGrain = 64;      // slots per scale: the decode kernel's tile
constexpr int kD = 128;         // head_dim
// k is kept within these: below, value * scale would leave the normal bf16 numbers (2^-9 * 2^-117 = 2^-126); above, exceed them.
constexpr int kMinExponent = -117, kMaxExponent = 119;

#ifdef __CUDACC__

// 2^k for a block whose largest finite magnitude is `amax`.  448 = 1.75 * 2^8.
__device__ __forceinline__ float scale_for(float amax) {
    const uint32_t bits = __float_as_uint(amax);
    int k = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    k = max(kMinExponent, min(kMaxExponent, k));
    return __uint_as_float((uint32_t)(k + 127) << 23);
}

// Two values -> e4m3, round to nearest even, saturating; NaN stays NaN.  `lo` goes to the lower byte.
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// e4m3 -> fp16 is exact.  The lower byte becomes the lower half.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t two_bytes) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two_bytes));
    return r;
}
__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t two_bytes) {
    const uint32_t h = e4m3x2_to_half2(two_bytes);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

#endif  // __CUDACC__

}  // namespace q8
}  // namespace nvllm
