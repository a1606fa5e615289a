// The 8-bit cache format: e4m3 values [num_slots, KVH, 128] and one fp32 scale for every kGrain slots and kv head
// [num_slots / kGrain, KVH]; an element stands for value * scale.
//
// The scale that the store chooses is a power of two, 2^k with the smallest k for which the largest finite magnitude of the
// block is at most 448 * 2^k.  e4m3 is a floating format, so a scale's fraction would buy no precision; a power of two makes
// a later change of the scale exact except where a value becomes subnormal, and value * scale a bf16 number (four
// significant bits): the same cache in bf16 holds the same keys and values.
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

// A bf16 row as the sum of two e4m3 rows.  `top`: its largest magnitude's bits.  The row is multiplied by `down`, a power of two
// that brings the largest magnitude to 224 < .. <= 448; `up` is its inverse.  A row of zeros stays as it is; one with a NaN or an
// infinity, whose softmax is NaN whatever the keys are, becomes NaN.
struct RowPower {
    float down, up;
    __device__ __forceinline__ explicit RowPower(uint32_t top) {
        const uint32_t shift = (top & 0x7fu) <= 0x60u ? 8 : 7, e = min(max(top == 0 ? 127u + shift : top >> 7, 9u), 254u);
        down = __uint_as_float(top < 0x7f80u ? (254u + shift - e) << 23 : 0x7fffffffu);
        up = __uint_as_float((e - shift) << 23);
    }
};
// Four elements (two words of bf16) -> upper and lower parts, a byte each: hi = e4m3(x), lo = e4m3(x - hi).  bf16 has eight
// significant bits and e4m3 four, so the sum is exact from 1/4 on, where what hi leaves is a multiple of e4m3's least step, 2^-9; below it
// is off by half of that step at most.
__device__ __forceinline__ void split_row(uint32_t w0, uint32_t w1, float down, uint32_t& hi, uint32_t& lo) {
    const float f[4] = {__uint_as_float(w0 << 16) * down, __uint_as_float(w0 & 0xffff0000u) * down, __uint_as_float(w1 << 16) * down,
                  __uint_as_float(w1 & 0xffff0000u) * down};
    const uint32_t h0 = to_e4m3x2(f[0], f[1]), h1 = to_e4m3x2(f[2], f[3]);
    const float2 g0 = e4m3x2_to_float2(h0), g1 = e4m3x2_to_float2(h1);
    hi = h0 | h1 << 16;
    lo = to_e4m3x2(f[0] - g0.x, f[1] - g0.y) | to_e4m3x2(f[2] - g1.x, f[3] - g1.y) << 16;
}

#endif  // __CUDACC__

}  // namespace q8
}  // namespace nvllm
