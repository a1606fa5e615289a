// What the decode kernels have in common (paged_decode.cu, bf16 caches; paged_decode_q8.cu, 8-bit caches): the cut of the
// work into chunks, the walk of a chunk, the metadata of a tile, the partial results and how they are combined, and the host's
// argument checks.
#pragma once

#include "common.cuh"

#include <mutex>
#include <string.h>

namespace nvllm {
namespace decode {

constexpr int kTile = 64;                      // tokens per tile
constexpr int kD = 128;                        // head_dim
constexpr int kConsumerWarps = 4;
constexpr int kWarps = kConsumerWarps + 1;     // consumers, TMA producer
constexpr int kThreads = kWarps * 32;
constexpr int kMaxG = 8;                       // query heads per kv head packed in one CTA
constexpr int kOsStride = kD + 4;              // padded row of the cross-warp merge buffers (bank spread)
constexpr int kOsBytes = 2 * kMaxG * kOsStride * 4;  // two buffers [8][132] fp32
constexpr int kCtasPerSm = 2;
constexpr int kMergeBatch = 4;                 // partial results the combine has in flight
constexpr int kEarlySlots = 8;                 // slots per producer lane: batches up to 256 request tiles ahead of the wait
// Per-partial record in the workspace: O[G][128] fp32, then m[8], l[8].
__host__ __device__ inline size_t partial_floats(int G) { return (size_t)G * kD + 2 * kMaxG; }

struct Params {
    const __nv_bfloat16* q;
    const int32_t* block_tables;
    const int32_t* context_lens;
    const int32_t* slot_mapping;  // [B] slots that the kernel just before this one writes, or null: it writes none
    int q_in_flight;              // that kernel writes q too: tiles requested ahead of the wait for it (0: it does not)
    __nv_bfloat16* out;
    float* partials;        // [chunks][KVH][2][partial_floats]
    unsigned int* tickets;  // [B*KVH] partials delivered so far per (sequence, kv head); zero when the kernel starts
    int B, H, KVH, G, NB, block_size, MB;
    int num_groups;
    int item_cost;  // units a sequence boundary costs on the cost line (see units_of)
    float scale_log2;
};

__device__ __forceinline__ int clamp_ctx(int c, int max_ctx) { return c < 0 ? 0 : (c > max_ctx ? max_ctx : c); }
__device__ __forceinline__ int tiles_of(int ctx) { return (ctx + kTile - 1) / kTile; }

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// ------------------------------------------------------------------------------------------
// the cut of the work
// ------------------------------------------------------------------------------------------
// The cost line: sequence b with tb > 0 tiles occupies tb + item_cost units, the first item_cost of them standing
// for its boundary overhead, the rest for its tiles 0 .. tb-1; empty sequences occupy nothing.
__device__ __forceinline__ int units_of(int tb, int item_cost) { return tb > 0 ? tb + item_cost : 0; }

// The line of one kv head (`total` units) is cut into `groups` contiguous chunks, one per CTA: the first `rem` of
// `len + 1` units, the others of `len`.  The cut depends on the lengths alone: the results are bitwise reproducible.
// (Handing the last eighth of the line out dynamically in ever smaller chunks was measured: the CTAs then finish
// together, but at the same time as before -- the stream is bound by DRAM, not by its slowest CTA -- and the many small
// partial results of a long sequence cost up to 15 us to combine.)
struct Cut {
    int groups;
    long long len, rem;

    __device__ __forceinline__ long long bound(int chunk) const { return chunk * len + (chunk < rem ? chunk : rem); }
    // chunk that holds unit u
    __device__ __forceinline__ int chunk_of(long long u) const {
        const long long head = rem * (len + 1);
        return u < head ? (int)div(u, len + 1) : (int)(rem + div(u - head, len));
    }
    // 64-bit divisions are slow and only lines of more than 2^31 units need them
    static __device__ __forceinline__ long long div(long long a, long long b) {
        return ((a | b) >> 31) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
    }
};

// Less than kMinChunk units per CTA: chunks of kMinChunk units and fewer CTAs.  Five tiles take about as long as splitting
// them further would cost (partial, ticket, combine: 2.5 us).
constexpr int kMinChunk = 5;
__device__ __forceinline__ Cut make_cut(long long total, int num_groups, int min_chunk = kMinChunk) {
    Cut c;
    c.groups = num_groups;
    if (total < (long long)min_chunk * num_groups) c.groups = max(1, (int)total / min_chunk);
    c.len = Cut::div(total, c.groups);
    c.rem = total - c.len * c.groups;
    return c;
}

struct Walk {
    int b;             // next sequence to look at
    long long fv;      // unit at which sequence b starts
    long long x0, x1;  // the chunk's range of units
};
struct Item {
    int b, t0, n;      // sequence, first tile and number of tiles this chunk holds of it
    int ctx, tb;       // its context length and total tiles
    long long fv;      // unit at which the sequence starts (its tile 0 sits at fv + item_cost)
};

// Advance to the next sequence of which the chunk holds at least one tile; false when the chunk is exhausted.
// (hint_b, hint_ctx): a context length the caller has fetched ahead of time (hint_b < 0: none).
__device__ __forceinline__ bool next_item(Walk& w, const Params& p, int max_ctx, Item& it, int hint_b, int hint_ctx) {
    while (w.b < p.B && w.fv < w.x1) {
        const int ctx = clamp_ctx(w.b == hint_b ? hint_ctx : __ldg(p.context_lens + w.b), max_ctx);
        const int tb = tiles_of(ctx);
        const long long t_base = w.fv + p.item_cost;  // unit of tile 0
        it.b = w.b;
        it.fv = w.fv;
        ++w.b;
        w.fv += units_of(tb, p.item_cost);
        if (tb == 0) continue;
        const long long lo = w.x0 - t_base, hi = w.x1 - t_base;
        const int t0 = (int)(lo < 0 ? 0 : (lo > tb ? tb : lo));
        const int t1 = (int)(hi < 0 ? 0 : (hi > tb ? tb : hi));
        if (t0 >= t1) continue;  // only boundary units of this sequence fall into the chunk
        it.t0 = t0;
        it.n = t1 - t0;
        it.ctx = ctx;
        it.tb = tb;
        return true;
    }
    return false;
}

// What the producer tells the consumers about a tile, beside the tile in the ring.
struct TileMeta {
    int valid;   // live tokens from this tile's first token on
    int flags;   // kFirst | kLast | kWhole | kDone
    int b;       // sequence
    int part;    // record of the partial result (an item that is not a whole sequence)
    int gf, gl;  // first and last chunk that hold tiles of the sequence
    int pad[2];
};
constexpr int kFirst = 1, kLast = 2, kWhole = 4, kDone = 8;

// Combine the partials of sequence b (chunks gf .. gl) for kv head kvh and write its G output rows.  Called by the 128
// consumer threads: thread t owns row t / 16 and dims 8 (t % 16) .. 8 (t % 16) + 7.  Partials are taken in chunk order,
// kMergeBatch at a time (all loads of a batch are in flight together), so the result does not depend on which CTA runs this.
__device__ __forceinline__ void merge_sequence(const Params& p, int b, int kvh, int gf, int gl, int ctid) {
    const int r = ctid >> 4, c8 = (ctid & 15) * 8;
    if (r >= p.G) return;
    const size_t pf = partial_floats(p.G);
    float mt = -INFINITY, lt = 0.f;
    float acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    for (int g0 = gf; g0 <= gl; g0 += kMergeBatch) {
        float mv[kMergeBatch], lv[kMergeBatch];
        float4 oa[kMergeBatch], ob[kMergeBatch];
#pragma unroll
        for (int u = 0; u < kMergeBatch; ++u) {
            const int g = g0 + u;
            const bool live = g <= gl;
            const float* part = p.partials + ((size_t)(g * p.KVH + kvh) * 2 + (g == gf ? 1 : 0)) * pf;
            mv[u] = live ? __ldcg(part + p.G * kD + r) : -INFINITY;
            lv[u] = live ? __ldcg(part + p.G * kD + kMaxG + r) : 0.f;
            oa[u] = live ? __ldcg(reinterpret_cast<const float4*>(part + r * kD + c8)) : make_float4(0.f, 0.f, 0.f, 0.f);
            ob[u] = live ? __ldcg(reinterpret_cast<const float4*>(part + r * kD + c8) + 1) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        float mnew = mt;
#pragma unroll
        for (int u = 0; u < kMergeBatch; ++u) mnew = fmaxf(mnew, mv[u]);
        if (mnew == -INFINITY) continue;
        const float sc = (mt == -INFINITY) ? 0.f : fast_exp2(mt - mnew);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] *= sc;
        lt *= sc;
#pragma unroll
        for (int u = 0; u < kMergeBatch; ++u) {
            const float f = (mv[u] == -INFINITY) ? 0.f : fast_exp2(mv[u] - mnew);
            acc[0] += oa[u].x * f;
            acc[1] += oa[u].y * f;
            acc[2] += oa[u].z * f;
            acc[3] += oa[u].w * f;
            acc[4] += ob[u].x * f;
            acc[5] += ob[u].y * f;
            acc[6] += ob[u].z * f;
            acc[7] += ob[u].w * f;
            lt += lv[u] * f;
        }
        mt = mnew;
    }
    const float inv = 1.0f / (lt + 1e-9f);
    uint4 w;
    w.x = pack_bf16(acc[0] * inv, acc[1] * inv);
    w.y = pack_bf16(acc[2] * inv, acc[3] * inv);
    w.z = pack_bf16(acc[4] * inv, acc[5] * inv);
    w.w = pack_bf16(acc[6] * inv, acc[7] * inv);
    *reinterpret_cast<uint4*>(p.out + ((size_t)b * p.H + (size_t)kvh * p.G + r) * kD + c8) = w;
}

__device__ __forceinline__ unsigned int atomic_add_acq_rel(unsigned int* addr, unsigned int v) {
    unsigned int old;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], %2;" : "=r"(old) : "l"(addr), "r"(v) : "memory");
    return old;
}

__device__ __forceinline__ bool wait_or_abort(volatile int* abort, uint64_t* bar, uint32_t parity) {
    return mbar_try_wait(bar, parity) || (!*abort && mbar_wait(bar, parity));
}


// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
inline int main_grid() { return kCtasPerSm * sm_count(); }

inline size_t round256(size_t x) { return (x + 255) & ~size_t(255); }

inline size_t ticket_bytes(int B, int KVH) { return round256((size_t)B * KVH * 4); }
inline size_t partial_bytes(int ctas, int G) { return round256((size_t)ctas * 2 * partial_floats(G) * 4); }

// Tensor maps of the caches seen so far, keyed by what they encode (base address, slots, kv heads, type).  Encoding
// one costs the host a microsecond or two per call; a serving loop hands over the same few caches for ever.
// A map holds no reference to the memory: an entry stays valid for any later buffer with the same key.
inline int cached_cache_map(CUtensorMap* map, const void* base, int64_t num_slots, int KVH, bool bytes = false) {
    struct Entry {
        const void* base;
        int64_t num_slots;
        int kvh, dev;
        bool bytes;
        CUtensorMap map;
    };
    constexpr int kEntries = 256;  // two per layer of a 128-layer model
    static std::mutex mu;
    static Entry table[kEntries];
    static int used = 0, next = 0;
    int dev = 0;
    NVLLM_CUDA_OK(cudaGetDevice(&dev));
    {
        std::lock_guard<std::mutex> lock(mu);
        for (int i = 0; i < used; ++i) {
            const Entry& e = table[i];
            if (e.base == base && e.num_slots == num_slots && e.kvh == KVH && e.dev == dev && e.bytes == bytes) {
                memcpy(map, &e.map, sizeof(CUtensorMap));
                return NVLLM_B200_OK;
            }
        }
    }
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return fail(NVLLM_B200_EDRIVER, "cuTensorMapEncodeTiled entry point not available");
    // bf16: the head dimension is seen as two halves of 64 (the widest row a 128-byte swizzle takes) with the half as an outer
    // dimension: one load then brings the tile in as the two 64-dim panels.
    cuuint64_t dims[4] = {64, (cuuint64_t)num_slots, 2, (cuuint64_t)KVH};
    cuuint64_t strides[3] = {(cuuint64_t)KVH * kD * 2, 64 * 2, (cuuint64_t)kD * 2};
    cuuint32_t box[4] = {64, (cuuint32_t)kTile, 2, 1};
    // bytes: a row of 128 is as wide as the swizzle.
    cuuint64_t dims8[3] = {kD, (cuuint64_t)num_slots, (cuuint64_t)KVH};
    cuuint64_t strides8[2] = {(cuuint64_t)KVH * kD, kD};
    cuuint32_t box8[3] = {kD, (cuuint32_t)kTile, 1};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    CUresult r = enc(map, bytes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, bytes ? 3 : 4,
                     const_cast<void*>(base), bytes ? dims8 : dims, bytes ? strides8 : strides, bytes ? box8 : box, estr,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                     bytes ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(NVLLM_B200_EDRIVER, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
    std::lock_guard<std::mutex> lock(mu);
    Entry& e = table[used < kEntries ? used++ : (next = (next + 1) % kEntries)];
    e.base = base;
    e.num_slots = num_slots;
    e.kvh = KVH;
    e.dev = dev;
    e.bytes = bytes;
    memcpy(&e.map, map, sizeof(CUtensorMap));
    return NVLLM_B200_OK;
}

// What every decode entry point shares: the argument checks and the two launches.  `tickets` / `partials` point
// into whatever scratch the entry point owns; `step` (may be null) adds the scatter of the step's new K/V rows
// to the first launch.
struct DecodeArgs {
    const void *q, *k_cache, *v_cache;
    const int32_t *block_tables, *context_lens;
    void* out;
    int B, H, KVH, D, NB, block_size, MB;
    float scale;
    void* stream;
};
struct StepArgs {
    const void *k, *v;
    const int32_t* slot_mapping;
    int src_dtype;
};

inline int check_decode_args(const char* who, const DecodeArgs& a) {
    if (a.B < 0 || a.H <= 0 || a.KVH <= 0 || a.NB <= 0 || a.block_size <= 0 || a.MB <= 0)
        return fail(NVLLM_B200_EINVAL, "%s: non-positive size (B=%d H=%d KVH=%d NB=%d block=%d MB=%d)", who, a.B, a.H,
                    a.KVH, a.NB, a.block_size, a.MB);
    if (a.D != kD) return fail(NVLLM_B200_EUNSUPPORTED, "%s: head_dim %d (only 128)", who, a.D);
    if (a.block_size % kTile != 0)
        return fail(NVLLM_B200_EUNSUPPORTED, "%s: block_size %d must be a multiple of %d", who, a.block_size, kTile);
    if (a.H % a.KVH != 0 || a.H / a.KVH > kMaxG)
        return fail(NVLLM_B200_EUNSUPPORTED, "%s: H/KVH = %d/%d must be an integer <= %d", who, a.H, a.KVH, kMaxG);
    if ((long long)a.MB * a.block_size > 0x3fffffffLL || (long long)a.NB * a.block_size > 0x7fffffffLL)
        return fail(NVLLM_B200_EUNSUPPORTED, "%s: cache or context too large for 32-bit token indices", who);
    if ((long long)a.B * a.KVH > 0x3fffffffLL) return fail(NVLLM_B200_EUNSUPPORTED, "%s: batch too large", who);
    return NVLLM_B200_OK;
}

inline int check_decode_pointers(const char* who, const DecodeArgs& a) {
    if (!a.q || !a.k_cache || !a.v_cache || !a.block_tables || !a.context_lens || !a.out)
        return fail(NVLLM_B200_EINVAL, "%s: null pointer", who);
    if (((uintptr_t)a.q | (uintptr_t)a.k_cache | (uintptr_t)a.v_cache | (uintptr_t)a.out) & 15)
        return fail(NVLLM_B200_EINVAL, "%s: q/k_cache/v_cache/out must be 16-byte aligned", who);
    if (a.KVH > main_grid())
        return fail(NVLLM_B200_EUNSUPPORTED, "%s: KVH %d exceeds the CTA count %d", who, a.KVH, main_grid());
    return NVLLM_B200_OK;
}

}  // namespace decode
}  // namespace nvllm
