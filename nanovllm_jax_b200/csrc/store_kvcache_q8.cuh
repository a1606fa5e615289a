// store_kvcache_q8 device code, shared by the stand-alone store (store_kvcache_q8.cu) and the decode step's first kernel
// (paged_decode_q8.cu).
//
// A scale belongs to 64 slots, so the rows of one call that fall into the same block of slots have to be looked at together:
// one CTA of 128 threads takes a (block, kv head), finds the block's rows among the call's tokens, takes their largest
// magnitude, decides on the scale and writes the rows; where the scale of a block that holds rows already grows, it rounds
// those again.  No block is taken by two CTAs, so there are no atomics on the cache and results do not depend on any order.
#pragma once

#include "q8.cuh"

namespace nvllm {
namespace q8 {

constexpr int kStoreThreads = 128;
constexpr int kPasses = kGrain / (kStoreThreads / 8);  // eight threads a row, 16 dims each

struct Store {
    const void *k, *v;  // [T, KVH, 128] bf16 or fp32
    uint8_t *k_cache, *v_cache;
    float *k_scale, *v_scale;
    const int32_t* slots;
    int64_t T;
    int KVH;
    int64_t num_slots;
};

struct StoreShared {
    int owner[kGrain];  // the token whose row a slot of the block gets, or -1
    float amax[2][kStoreThreads / 32];
    int earlier;
};

// Block of slots a token's row goes to, or -1.
__device__ __forceinline__ int block_of(int slot, int64_t num_slots) {
    return slot >= 0 && slot < num_slots ? slot / kGrain : -1;
}

template <typename SrcT>
struct Row16;  // 16 consecutive elements of a row, as loaded
template <>
struct Row16<__nv_bfloat16> {
    uint4 a, b;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) {
        a = __ldg(reinterpret_cast<const uint4*>(p)), b = __ldg(reinterpret_cast<const uint4*>(p) + 1);
    }
    __device__ __forceinline__ void get(float (&x)[16]) const {
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
};
template <>
struct Row16<float> {
    float4 v[4];
    __device__ __forceinline__ void load(const float* p) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __ldg(reinterpret_cast<const float4*>(p) + i);
    }
    __device__ __forceinline__ void get(float (&x)[16]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[4 * i] = v[i].x, x[4 * i + 1] = v[i].y, x[4 * i + 2] = v[i].z, x[4 * i + 3] = v[i].w;
    }
};

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// One of the two caches: the rows in `sh.owner` of (block, kvh).  `which` picks the reduction's scratch.
template <typename SrcT>
__device__ __forceinline__ void store_rows(StoreShared& sh, int which, const SrcT* __restrict__ src, uint8_t* cache, float* scale,
                                           int block, int kvh, int KVH) {
    const int tid = threadIdx.x, r = tid >> 3, part = tid & 7;
    float* const my_scale = scale + (int64_t)block * KVH + kvh;
    const float before = *my_scale;
    Row16<SrcT> x[kPasses];
    int owner[kPasses];
    float amax = 0.f;
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        owner[p] = sh.owner[p * (kStoreThreads / 8) + r];
        if (owner[p] >= 0) x[p].load(src + ((int64_t)owner[p] * KVH + kvh) * kD + part * 16);
    }
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        if (owner[p] < 0) continue;
        float f[16];
        x[p].get(f);
#pragma unroll
        for (int i = 0; i < 16; ++i) amax = fmaxf(amax, finite(f[i]) ? fabsf(f[i]) : 0.f);
    }
    amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));  // not negative: bits order as values do
    if ((tid & 31) == 0) sh.amax[which][tid >> 5] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kStoreThreads / 32; ++w) amax = fmaxf(amax, sh.amax[which][w]);
    // A call that writes a block's first slot begins the block; another one may only let its scale grow.
    const float old = sh.owner[0] < 0 && before > 0.f ? before : 0.f;
    const float now = fmaxf(old, scale_for(amax));
    const float inv = 1.f / now;
    uint8_t* const base = cache + ((int64_t)block * kGrain * KVH + kvh) * kD + part * 16;
    const int64_t row_stride = (int64_t)KVH * kD;
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        if (owner[p] < 0) continue;
        float f[16];
        x[p].get(f);
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = finite(f[i]) ? f[i] * inv : __uint_as_float(0x7fffffffu);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = to_e4m3x2(f[4 * i], f[4 * i + 1]) | to_e4m3x2(f[4 * i + 2], f[4 * i + 3]) << 16;
        *reinterpret_cast<uint4*>(base + (p * (kStoreThreads / 8) + r) * row_stride) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (old > 0.f && now > old) {  // the rows that are there already are rounded again
        const float ratio = old / now;
        uint4 q[kPasses];
#pragma unroll
        for (int p = 0; p < kPasses; ++p)
            if (owner[p] < 0) q[p] = *reinterpret_cast<const uint4*>(base + (p * (kStoreThreads / 8) + r) * row_stride);
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
            if (owner[p] >= 0) continue;
            uint32_t w[4] = {q[p].x, q[p].y, q[p].z, q[p].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 a = e4m3x2_to_float2(w[i] & 0xffffu), b = e4m3x2_to_float2(w[i] >> 16);
                w[i] = to_e4m3x2(a.x * ratio, a.y * ratio) | to_e4m3x2(b.x * ratio, b.y * ratio) << 16;
            }
            *reinterpret_cast<uint4*>(base + (p * (kStoreThreads / 8) + r) * row_stride) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    if (tid == 0 && now != before) *my_scale = now;
}

template <typename SrcT>
__device__ __forceinline__ void store_block(StoreShared& sh, const Store& s, int block, int kvh) {
    store_rows(sh, 0, static_cast<const SrcT*>(s.k), s.k_cache, s.k_scale, block, kvh, s.KVH);
    store_rows(sh, 1, static_cast<const SrcT*>(s.v), s.v_cache, s.v_scale, block, kvh, s.KVH);
}

// Few tokens: CTA (t, kvh) reads all slots and takes the block of token t unless an earlier token has the same one.
template <typename SrcT>
__device__ __forceinline__ void store_token(StoreShared& sh, const Store& s, int t, int kvh) {
    const int block = block_of(__ldg(s.slots + t), s.num_slots);
    if (block < 0) return;
    const int tid = threadIdx.x;
    if (tid < kGrain) sh.owner[tid] = -1;
    if (tid == 0) sh.earlier = 0;
    __syncthreads();
    for (int j = tid; j < (int)s.T; j += kStoreThreads) {
        const int slot = __ldg(s.slots + j);
        if (block_of(slot, s.num_slots) == block) {
            atomicMax(&sh.owner[slot % kGrain], j);  // of two rows for one slot the later one stays
            if (j < t) sh.earlier = 1;
        }
    }
    __syncthreads();
    if (sh.earlier) return;
    store_block<SrcT>(sh, s, block, kvh);
}

// Up to so many tokens every CTA reads all slots; beyond, a kernel in front finds the runs.
constexpr int kScanTokens = 1024;

}  // namespace q8
}  // namespace nvllm
