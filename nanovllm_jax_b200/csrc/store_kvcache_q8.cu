// store_kvcache_q8: the step's K/V rows into the 8-bit paged cache, with a scale for every 64 slots and kv head.
//
// The reference keeps its cache in bf16 (store_kv_to_cache, layers/attention.py:42-77); this is the same scatter into half the
// bytes.  Per token it reads KVH * 128 elements of K and of V and writes as many bytes to each cache.  What a block of slots
// gets is in store_kvcache_q8.cuh; here is how a call's blocks are found.
//
//  * Up to kScanTokens tokens, a CTA per (token, kv head) reads all slots and takes the token's block, if it is the first there.
//  * Beyond, a CTA per (kWindow tokens, kv head) takes the runs that begin among its tokens: tokens in a row whose slots lie in
//    one block.  A prompt makes one run per block, but a block could be reached again further on.  q8_runs_kernel, a cluster
//    of eight CTAs in front, chains the runs by a hash of their blocks.  The storing CTAs start beside it, load the rows and
//    wait only then; a run that is alone under its hash goes ahead, of others the first of a block takes the rows of all.
//    (CTAs that look through all slots themselves, while their rows are on their way, are no better in between: 48 prompts of
//    5..300 tokens, fp32, 2 kv heads: 11.1 us, with the kernel in front 9.6.)
//
// Measured: 16 prompts of 128..4096 tokens, 8 kv heads, bf16: 42.3 us, 4.9 TB/s, 0.76 of a plain copy's rate (the chain slots -> rows
// -> scale -> stores of four CTAs per SM: without the arithmetic it takes as long, without the stores 35 us; the window's rows asked for
// before its slots are known: 43.6; 128 tokens a CTA: 44.9; CTAs that stay and have the next window's slots at hand: 48.7, for
// they spill); 64 appended rows 4 to 5 us.  More than 1024 appended rows go one after the other, 64 a CTA: 2000, 8 kv heads, 80 us; a warp
// each in the same kernel 13, but the prompts then take 47 (a decode step has another way, see kScanStep).
#include "store_kvcache_q8.cuh"

#include <algorithm>
#include <cooperative_groups.h>

namespace nvllm {
namespace q8 {

constexpr int kRunCtas = 8;          // a cluster
constexpr int kRunThreads = 1024;
constexpr int kRunUnroll = 8;        // slots a thread has in flight
constexpr int kBuckets = 8192;
constexpr int kWindow = 64;
constexpr int kAhead = 128;          // slots behind the window that a storing CTA has at hand

// Workspace.  A run goes by its first token.
struct Runs {
    uint8_t* crowded;  // [kBuckets] more than one run has this hash
    int* first;        // [kBuckets] a run of the hash, or -1
    int* next;         // [T] the next run with the hash of the run that begins here, or -1 (where one begins)
};
static size_t run_bytes(int64_t T) { return ((size_t)T * 4 + kBuckets * 4 + kBuckets + 255) & ~size_t(255); }
static Runs runs_in(void* workspace) {
    uint8_t* p = static_cast<uint8_t*>(workspace);
    return Runs{p, reinterpret_cast<int*>(p + kBuckets), reinterpret_cast<int*>(p + 5 * kBuckets)};
}

__device__ __forceinline__ int bucket_of(int block) { return (int)((uint32_t)block * 2654435761u >> 19); }
static_assert(kBuckets == 1 << 13, "see bucket_of");

// The buckets are dealt to the CTAs by their lowest bits.  (One CTA with all of them took 16 us for 40 000 tokens, eight take 6.)
__global__ void __launch_bounds__(kRunThreads) __cluster_dims__(kRunCtas, 1, 1)
q8_runs_kernel(const int32_t* __restrict__ slots, int64_t T, int64_t num_slots, Runs runs) {
    __shared__ int first[kBuckets / kRunCtas];
    __shared__ int crowded[kBuckets / kRunCtas];
    const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, rank = (int)cluster.block_rank();
    for (int i = tid; i < kBuckets / kRunCtas; i += kRunThreads) first[i] = -1, crowded[i] = 0;
    griddep_wait();
    griddep_launch_dependents();
    cluster.sync();
    for (int64_t base = rank * kRunThreads; base < T; base += (int64_t)kRunCtas * kRunThreads * kRunUnroll) {
        int slot[kRunUnroll], before[kRunUnroll];
#pragma unroll
        for (int u = 0; u < kRunUnroll; ++u) {
            const int64_t t = base + u * (kRunCtas * kRunThreads) + tid;
            slot[u] = t < T ? __ldg(slots + t) : -1;
            before[u] = lane == 0 && t > 0 && t < T ? __ldg(slots + t - 1) : -1;
        }
#pragma unroll
        for (int u = 0; u < kRunUnroll; ++u) {
            const int block = block_of(slot[u], num_slots);
            const int left = __shfl_up_sync(0xffffffffu, block, 1);
            if (block >= 0 && block != (lane == 0 ? block_of(before[u], num_slots) : left)) {
                const int t = (int)(base + u * (kRunCtas * kRunThreads) + tid), h = bucket_of(block);
                const int other = atomicExch(cluster.map_shared_rank(first, h % kRunCtas) + h / kRunCtas, t);
                if (other >= 0) cluster.map_shared_rank(crowded, h % kRunCtas)[h / kRunCtas] = 1;
                runs.next[t] = other;
            }
        }
    }
    cluster.sync();
    for (int i = tid; i < kBuckets / kRunCtas; i += kRunThreads) {
        runs.first[i * kRunCtas + rank] = first[i];
        runs.crowded[i * kRunCtas + rank] = (uint8_t)crowded[i];
    }
}

// Tokens of the run that begins at `start`: into the owner table.  (Tokens behind its end that lie in the same block belong
// to runs of the same block: they are taken with this one anyway.)  Called by all threads; ends with a barrier.
__device__ __forceinline__ void take_run(StoreShared& sh, const Store& s, int64_t start, int block) {
    for (int64_t j = start + threadIdx.x;; j += kStoreThreads) {
        const int slot = j < s.T ? __ldg(s.slots + j) : -1;
        const bool in = block_of(slot, s.num_slots) == block;
        if (in) atomicMax(&sh.owner[place_of(slot)], (int)j);  // of two rows for one slot the later one stays
        if (!__syncthreads_and(in)) return;
    }
}

// Nothing but the chains depends on the kernel in front, which has let this one go once all before it was complete.
template <typename SrcT>
__global__ void __launch_bounds__(kStoreThreads, sizeof(SrcT) == 2 ? 4 : 2) store_runs_kernel(const Store s, const Runs runs) {
    __shared__ StoreShared sh;
    __shared__ int at[1 + kWindow + kAhead];  // slots of tokens t0 - 1 ..; -1: none
    __shared__ uint32_t begins[kWindow / 32];
    const int tid = threadIdx.x, kvh = blockIdx.x % s.KVH;
    const int64_t t0 = (int64_t)(blockIdx.x / s.KVH) * kWindow;
    if (tid < 1 + kWindow + kAhead) {
        const int64_t t = t0 - 1 + tid;
        const int slot = t >= 0 && t < s.T ? __ldg(s.slots + t) : -1;
        at[tid] = block_of(slot, s.num_slots) < 0 ? -1 : slot;
    }
    __syncthreads();
    if (tid < kWindow) {
        const int slot = at[1 + tid], before = at[tid];
        const uint32_t b = __ballot_sync(0xffffffffu, slot >= 0 && (before < 0 || (before ^ slot) >= kGrain));
        if ((tid & 31) == 0) begins[tid >> 5] = b;
    }
    __syncthreads();
    bool waited = false;
    for (int w = 0; w < kWindow / 32; ++w) {
        for (uint32_t left = begins[w]; left; left &= left - 1) {
            const int i = 32 * w + __ffs(left) - 1;
            const int64_t t = t0 + i;
            const int begin = at[1 + i], block = (int)((uint32_t)begin / kGrain);
            if (tid < kGrain) sh.owner[tid] = -1;
            __syncthreads();
            const int slot = tid < kWindow + kAhead ? at[1 + tid] : -1;
            const bool in = tid >= i && slot >= 0 && (slot ^ begin) < kGrain;
            if (in) atomicMax(&sh.owner[place_of(slot)], (int)(t0 + tid));  // of two rows for one slot the later one stays
            if (__syncthreads_and(in || tid < i || tid >= kWindow + kAhead)) take_run(sh, s, t0 + kWindow + kAhead, block);
            Rows<SrcT> rows;
            rows.load(sh, s, block, kvh);
            if (!waited) {
                griddep_wait();
                griddep_launch_dependents();
                waited = true;
            }
            const int h = bucket_of(block);
            if (runs.crowded[h]) {
                bool mine = true;  // the first run of the block takes all
                for (int o = runs.first[h]; o >= 0 && mine; o = runs.next[o])
                    mine = o >= t || block_of(__ldg(s.slots + o), s.num_slots) != block;
                if (!mine) {
                    __syncthreads();  // everyone has read the owners
                    continue;
                }
                for (int o = runs.first[h]; o >= 0; o = runs.next[o])
                    if (o != t && block_of(__ldg(s.slots + o), s.num_slots) == block) take_run(sh, s, o, block);
                rows.load(sh, s, block, kvh);
            }
            store_rows(sh, s, rows, block, kvh);
            __syncthreads();
        }
    }
    if (!waited) {  // this grid must not be complete before the kernel in front of it is
        griddep_wait();
        griddep_launch_dependents();
    }
}

template <typename SrcT>
__global__ void __launch_bounds__(kStoreThreads) store_tokens_kernel(const Store s) {
    __shared__ StoreShared sh;
    griddep_wait();
    griddep_launch_dependents();
    store_token<SrcT>(sh, s, blockIdx.x / s.KVH, blockIdx.x % s.KVH);
}

size_t store_workspace_bytes(int64_t T) { return T <= kScanTokens ? 256 : run_bytes(T); }

int check_store(const char* who, const Store& s, int64_t D, int src_dtype) {
    if (s.T < 0 || s.KVH <= 0 || s.num_slots < 0)
        return fail(NVLLM_B200_EINVAL, "%s: negative size (T=%lld KVH=%d num_slots=%lld)", who, (long long)s.T, s.KVH,
                    (long long)s.num_slots);
    if (D != kD) return fail(NVLLM_B200_EUNSUPPORTED, "%s: head_dim %lld (only 128)", who, (long long)D);
    if (s.num_slots % kGrain)
        return fail(NVLLM_B200_EUNSUPPORTED, "%s: num_slots %lld must be a multiple of %d", who, (long long)s.num_slots, kGrain);
    if (s.T > 0x7fffffffLL - 1024 || s.num_slots > 0x7fffffffLL || s.T * s.KVH > 0x7fffffffLL)
        return fail(NVLLM_B200_EUNSUPPORTED, "%s: more than 2^31-1 tokens, token heads or slots", who);
    if (src_dtype != NVLLM_B200_DTYPE_BF16 && src_dtype != NVLLM_B200_DTYPE_F32)
        return fail(NVLLM_B200_EUNSUPPORTED, "%s: src_dtype %d", who, src_dtype);
    if (s.T == 0 || s.num_slots == 0) return NVLLM_B200_OK;
    if (!s.k || !s.v || !s.k_cache || !s.v_cache || !s.k_scale || !s.v_scale || !s.slots)
        return fail(NVLLM_B200_EINVAL, "%s: null pointer", who);
    if (((uintptr_t)s.k | (uintptr_t)s.v | (uintptr_t)s.k_cache | (uintptr_t)s.v_cache) & 15)
        return fail(NVLLM_B200_EINVAL, "%s: k/v and caches must be 16-byte aligned", who);
    if (((uintptr_t)s.k_scale | (uintptr_t)s.v_scale | (uintptr_t)s.slots) & 3)
        return fail(NVLLM_B200_EINVAL, "%s: scales and slot_mapping must be 4-byte aligned", who);
    return NVLLM_B200_OK;
}

int launch_store(const char* who, const Store& s, int src_dtype, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
    if (s.T == 0 || s.num_slots == 0) return NVLLM_B200_OK;
    const size_t need = store_workspace_bytes(s.T);
    if (s.T > kScanTokens && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
        return fail(NVLLM_B200_EWORKSPACE, "%s: workspace of %zu bytes (16-byte aligned) required, got %zu", who, need,
                    workspace ? workspace_bytes : (size_t)0);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    const bool f32 = src_dtype == NVLLM_B200_DTYPE_F32;
    if (s.T <= kScanTokens) {
        cfg.gridDim = dim3((unsigned)(s.T * s.KVH));
        cfg.blockDim = dim3(kStoreThreads);
        NVLLM_CUDA_OK(cudaLaunchKernelEx(&cfg, f32 ? store_tokens_kernel<float> : store_tokens_kernel<__nv_bfloat16>, s));
        return NVLLM_B200_OK;
    }
    const Runs runs = runs_in(workspace);
    cfg.gridDim = dim3(kRunCtas);
    cfg.blockDim = dim3(kRunThreads);
    NVLLM_CUDA_OK(cudaLaunchKernelEx(&cfg, q8_runs_kernel, s.slots, s.T, s.num_slots, runs));
    cfg.gridDim = dim3((unsigned)((s.T + kWindow - 1) / kWindow * s.KVH));
    cfg.blockDim = dim3(kStoreThreads);
    NVLLM_CUDA_OK(cudaLaunchKernelEx(&cfg, f32 ? store_runs_kernel<float> : store_runs_kernel<__nv_bfloat16>, s, runs));
    return NVLLM_B200_OK;
}

}  // namespace q8
}  // namespace nvllm

extern "C" size_t nvllm_b200_store_kvcache_q8_workspace_bytes(int64_t T) {
    return nvllm::q8::store_workspace_bytes(T < 0 ? 0 : T);
}

extern "C" int nvllm_b200_store_kvcache_q8(const void* k, const void* v, void* k_cache, void* v_cache, float* k_scale,
                                           float* v_scale, const int32_t* slot_mapping, void* workspace, size_t workspace_bytes,
                                           int64_t T, int KVH, int D, int64_t num_slots, int src_dtype, void* stream) {
    using namespace nvllm::q8;
    const Store s = {k, v, (uint8_t*)k_cache, (uint8_t*)v_cache, k_scale, v_scale, slot_mapping, T, KVH, num_slots};
    const int rc = check_store("store_kvcache_q8", s, D, src_dtype);
    if (rc) return rc;
    return launch_store("store_kvcache_q8", s, src_dtype, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}
