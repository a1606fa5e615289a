// store_kvcache_q8 device code, shared by the stand-alone store (store_kvcache_q8.cu) and the decode step's first kernel
// (paged_decode_q8.cu).
//
// A scale belongs to 64 slots, so the rows of one call that fall into the same block of slots have to be looked at together:
// one CTA takes a (block, kv head), half of its threads K and half V: it finds the block's rows among the call's tokens, takes
// their largest magnitude, decides on the scale and writes the rows; where the scale of a block that holds rows already grows,
// it rounds those again.  No block is taken by two CTAs, so there are no atomics on the cache and results do not depend on any
// order.
#pragma once

#include "q8.cuh"

#include <type_traits>

namespace nvllm {
namespace q8 {

constexpr int kStoreThreads = 256;
constexpr int kHalf = kStoreThreads / 2;      // threads of K, and of V
constexpr int kRowsAtOnce = kHalf / 8;        // eight threads a row, 16 dims each
constexpr int kPasses = kGrain / kRowsAtOnce;

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
    uint32_t top[kStoreThreads / 32];
    int earlier;
};

// Block of slots a token's row goes to, or -1.
__device__ __forceinline__ int block_of(int slot, int64_t num_slots) {
    return slot >= 0 && slot < num_slots ? (int)((uint32_t)slot / kGrain) : -1;
}
__device__ __forceinline__ int place_of(int slot) { return (int)((uint32_t)slot % kGrain); }

constexpr uint32_t kInfinityBits = 0x7f800000u;
__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7fffffffu) < kInfinityBits; }

// 16 consecutive elements of a row, as loaded.  top(): the largest magnitude as the bits of a float (of a NaN or an infinity
// where there is one: their bits are larger than any finite number's).
template <typename SrcT>
struct Row16 {
    static constexpr int kChunks = 16 * sizeof(SrcT) / 16;
    uint4 c[kChunks];

    __device__ __forceinline__ void get(float (&x)[16]) const {
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const uint32_t w[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (sizeof(SrcT) == 2) {
                    x[8 * i + 2 * e] = __uint_as_float(w[e] << 16);
                    x[8 * i + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
                } else {
                    x[4 * i + e] = __uint_as_float(w[e]);
                }
            }
        }
    }
    __device__ __forceinline__ uint32_t top() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const uint32_t w[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) m = sizeof(SrcT) == 2 ? __vmaxu2(m, w[e] & 0x7fff7fffu) : max(m, w[e] & 0x7fffffffu);
        }
        return sizeof(SrcT) == 2 ? max(m << 16, m & 0xffff0000u) : m;
    }
};

// A thread's share of the rows in `sh.owner`, on their way.  (Into shared memory by cp.async, so that six CTAs fit an SM instead of
// four: 59 us instead of 42 for 16 prompts of 128..4096 tokens, 8 kv heads.)
template <typename SrcT>
struct Rows {
    using Row = Row16<SrcT>;
    Row x[kPasses];
    float before;  // the block's scale as it is

    __device__ __forceinline__ void load(const StoreShared& sh, const Store& s, int block, int kvh) {
        const int tid = threadIdx.x, r = (tid % kHalf) >> 3, part = tid & 7;
        const SrcT* src = static_cast<const SrcT*>(tid < kHalf ? s.k : s.v) + kvh * kD + part * 16;
        before = (tid < kHalf ? s.k_scale : s.v_scale)[(int64_t)block * s.KVH + kvh];
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
            const int owner = sh.owner[p * kRowsAtOnce + r];
            if (owner < 0) continue;
            const uint4* from = reinterpret_cast<const uint4*>(src + (int64_t)owner * (s.KVH * kD));
#pragma unroll
            for (int i = 0; i < Row::kChunks; ++i) x[p].c[i] = __ldg(from + i);
        }
    }
};

// Stores them.  Called by all threads.
template <typename SrcT>
__device__ __forceinline__ void store_rows(StoreShared& sh, const Store& s, const Rows<SrcT>& rows, int block, int kvh) {
    const int tid = threadIdx.x, r = (tid % kHalf) >> 3, part = tid & 7;
    uint32_t mine = 0;  // passes whose row is written
    uint32_t top = 0;
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        if (sh.owner[p * kRowsAtOnce + r] < 0) continue;
        mine |= 1u << p;
        top = max(top, rows.x[p].top());
    }
    uint32_t* const tops = sh.top + tid / kHalf * (kHalf / 32);
    const int bar = 1 + tid / kHalf;
    top = __reduce_max_sync(0xffffffffu, top);
    if ((tid & 31) == 0) tops[(tid % kHalf) >> 5] = top;
    named_barrier_sync(bar, kHalf);
#pragma unroll
    for (int w = 0; w < kHalf / 32; ++w) top = max(top, tops[w]);
    const bool odd = top >= kInfinityBits;  // a NaN or an infinity, which count for nothing: look again, without them
    if (odd) {
        top = 0;
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
            if (!(mine >> p & 1)) continue;
            float f[16];
            rows.x[p].get(f);
#pragma unroll
            for (int i = 0; i < 16; ++i) top = max(top, finite(f[i]) ? __float_as_uint(f[i]) & 0x7fffffffu : 0u);
        }
        named_barrier_sync(bar, kHalf);
        top = __reduce_max_sync(0xffffffffu, top);
        if ((tid & 31) == 0) tops[(tid % kHalf) >> 5] = top;
        named_barrier_sync(bar, kHalf);
#pragma unroll
        for (int w = 0; w < kHalf / 32; ++w) top = max(top, tops[w]);
    }
    // A call that writes a block's first slot begins the block; another one may only let its scale grow.
    const float old = sh.owner[0] < 0 && rows.before > 0.f ? rows.before : 0.f;
    const float now = fmaxf(old, scale_for(__uint_as_float(top)));
    const float inv = 1.f / now;
    uint8_t* const base = (tid < kHalf ? s.k_cache : s.v_cache) + (((int64_t)block * kGrain + r) * s.KVH + kvh) * kD + part * 16;
    const int64_t step = (int64_t)kRowsAtOnce * s.KVH * kD;
    auto write = [&](auto careful) {
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
            if (!(mine >> p & 1)) continue;
            float f[16];
            rows.x[p].get(f);
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 16; ++i) f[i] = decltype(careful)::value && !finite(f[i]) ? __uint_as_float(0x7fffffffu) : f[i] * inv;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = to_e4m3x2(f[4 * i], f[4 * i + 1]) | to_e4m3x2(f[4 * i + 2], f[4 * i + 3]) << 16;
            *reinterpret_cast<uint4*>(base + p * step) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    };
    if (odd)
        write(std::true_type{});
    else
        write(std::false_type{});
    if (old > 0.f && now > old) {  // the rows that are there already are rounded again
        const float ratio = old / now;
        uint4 q[kPasses];
#pragma unroll
        for (int p = 0; p < kPasses; ++p)
            if (!(mine >> p & 1)) q[p] = *reinterpret_cast<const uint4*>(base + p * step);
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
            if (mine >> p & 1) continue;
            uint32_t w[4] = {q[p].x, q[p].y, q[p].z, q[p].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 a = e4m3x2_to_float2(w[i] & 0xffffu), b = e4m3x2_to_float2(w[i] >> 16);
                w[i] = to_e4m3x2(a.x * ratio, a.y * ratio) | to_e4m3x2(b.x * ratio, b.y * ratio) << 16;
            }
            *reinterpret_cast<uint4*>(base + p * step) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    if (tid % kHalf == 0 && now != rows.before) (tid < kHalf ? s.k_scale : s.v_scale)[(int64_t)block * s.KVH + kvh] = now;
}

// A warp stores the only row that the call has for a block, of K (x = 0) or V: four dims a lane.
template <typename SrcT>
__device__ __forceinline__ void store_lone_row(const Store& s, int64_t t, int slot, int kvh, int x) {
    const int lane = threadIdx.x & 31, block = (int)((uint32_t)slot / kGrain), place = place_of(slot);
    float* const scale = (x ? s.v_scale : s.k_scale) + (int64_t)block * s.KVH + kvh;
    uint8_t* const cache = (x ? s.v_cache : s.k_cache) + ((int64_t)block * kGrain * s.KVH + kvh) * kD;
    const SrcT* from = static_cast<const SrcT*>(x ? s.v : s.k) + (t * s.KVH + kvh) * kD + lane * 4;
    const float before = *scale;
    float f[4];
    if constexpr (sizeof(SrcT) == 2) {
        const uint2 w = __ldg(reinterpret_cast<const uint2*>(from));
        f[0] = __uint_as_float(w.x << 16), f[1] = __uint_as_float(w.x & 0xffff0000u);
        f[2] = __uint_as_float(w.y << 16), f[3] = __uint_as_float(w.y & 0xffff0000u);
    } else {
        const float4 w = __ldg(reinterpret_cast<const float4*>(from));
        f[0] = w.x, f[1] = w.y, f[2] = w.z, f[3] = w.w;
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, finite(f[i]) ? __float_as_uint(f[i]) & 0x7fffffffu : 0u);
    top = __reduce_max_sync(0xffffffffu, top);
    const float old = place > 0 && before > 0.f ? before : 0.f;
    const float now = fmaxf(old, scale_for(__uint_as_float(top)));
    const float inv = 1.f / now;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = finite(f[i]) ? f[i] * inv : __uint_as_float(0x7fffffffu);
    *reinterpret_cast<uint32_t*>(cache + (int64_t)place * s.KVH * kD + lane * 4) = to_e4m3x2(f[0], f[1]) | to_e4m3x2(f[2], f[3]) << 16;
    if (old > 0.f && now > old) {  // the rows that are there already are rounded again: four at a time, eight lanes each
        const float ratio = old / now;
#pragma unroll 4
        for (int r = lane >> 3; r < kGrain; r += 4) {
            if (r == place) continue;
            uint4* const at = reinterpret_cast<uint4*>(cache + (int64_t)r * s.KVH * kD + (lane & 7) * 16);
            const uint4 q = *at;
            uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 a = e4m3x2_to_float2(w[i] & 0xffffu), b = e4m3x2_to_float2(w[i] >> 16);
                w[i] = to_e4m3x2(a.x * ratio, a.y * ratio) | to_e4m3x2(b.x * ratio, b.y * ratio) << 16;
            }
            *at = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    if (lane == 0 && now != before) *scale = now;
}

constexpr int kAllHeads = 1024;  // (token, head) pairs
// Few tokens: CTA (t, kvh) reads all slots and takes the block of token t unless an earlier token has the same one.  A token whose
// neighbours go to other blocks, as in a decode step, is taken by the CTA of kv head 0 for all heads, a warp a row.  (A CTA for each of
// its heads, each of which reads all slots: 256 appended rows, 8 kv heads, 7.7 us instead of 5.1, 1000 31.8 instead of 14.4.  Up to
// kAllHeads pairs the heads have CTAs of their own all the same: they fit the SMs at once.)
template <typename SrcT>
__device__ __forceinline__ void store_token(StoreShared& sh, const Store& s, int t, int kvh) {
    const int mine = __ldg(s.slots + t), left = t > 0 ? __ldg(s.slots + t - 1) : -1, right = t + 1 < (int)s.T ? __ldg(s.slots + t + 1) : -1;
    const int block = block_of(mine, s.num_slots);
    if (block < 0 || block_of(left, s.num_slots) == block) return;
    const bool lone = block_of(right, s.num_slots) != block;
    const bool all = lone && s.T * s.KVH > kAllHeads;
    if (all && kvh > 0) return;
    const int tid = threadIdx.x;
    if (tid < kGrain) sh.owner[tid] = -1;
    if (tid == 0) sh.earlier = 0;
    __syncthreads();
    bool others = false;
    for (int j = tid; j < (int)s.T; j += kStoreThreads) {
        const int slot = __ldg(s.slots + j);
        if (block_of(slot, s.num_slots) == block) {
            atomicMax(&sh.owner[place_of(slot)], j);  // of two rows for one slot the later one stays
            if (j < t) sh.earlier = 1;
            others |= j != t;
        }
    }
    others = __syncthreads_or(others);
    if (sh.earlier) return;
    if (!others) {
        const int rows = all ? 2 * s.KVH : 2;
        for (int i = tid >> 5; i < rows; i += kStoreThreads / 32) store_lone_row<SrcT>(s, t, mine, kvh + (i >> 1), i & 1);
        return;
    }
    for (int h = kvh; h < (all ? s.KVH : kvh + 1); ++h) {
        Rows<SrcT> rows;
        rows.load(sh, s, block, h);
        store_rows(sh, s, rows, block, h);
        __syncthreads();
    }
}

// Up to so many tokens every CTA reads all slots; beyond, another kernel looks for blocks that are reached twice: 1000 tokens of prompts, 2
// kv heads, fp32 7.1 us, with that kernel 7.9; 2000 10.9 and 8.0; 8 kv heads, bf16 11.7 and 7.5, 20 and 7.9.  Of a decode step, whose rows
// are alone in their blocks, up to kScanStep: 2000 rows, 8 kv heads 27 us, with that kernel 80; 4000 53 and 107.
constexpr int kScanTokens = 1024, kScanStep = 4096;

}  // namespace q8
}  // namespace nvllm
