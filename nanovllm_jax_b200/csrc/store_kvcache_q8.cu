// store_kvcache_q8: the step's K/V rows into the 8-bit paged cache, with a scale for every 64 slots and kv head.
//
// The reference keeps its cache in bf16 (store_kv_to_cache, layers/attention.py:42-77); this is the same scatter into half the
// bytes.  Per token it reads KVH * 128 elements of K and of V and writes as many bytes to each cache.  What a block of slots
// gets is in store_kvcache_q8.cuh; here is how a call's blocks are found.
//
//  * Up to kScanTokens tokens, a CTA per (token, kv head) reads all slots.
//  * Beyond, q8_runs_kernel lists the runs: tokens in a row whose slots lie in one block.  Runs of one block that lie apart
//    are linked through a hash table in shared memory, so that the first of them takes all (a prompt's tokens are one run per
//    block; slots in a random order give as many runs as tokens, and chains of a few).
#include "store_kvcache_q8.cuh"

#include <algorithm>

namespace nvllm {
namespace q8 {

constexpr int kRunThreads = 1024;
constexpr int kRunUnroll = 32;       // slots a thread has in flight
constexpr int kBuckets = 8192;

// Workspace: {number of runs, 0, 0, 0}, then per run {first token, block, next run of its bucket or -1, 1 if it is alone there},
// then the first run of every bucket.
struct RunList {
    int4* head;
    int4* runs;
    int* buckets;
};
static size_t run_bytes(int64_t T) { return ((size_t)(T + 1) * 16 + (size_t)kBuckets * 4 + 255) & ~size_t(255); }
static RunList run_list(void* workspace, int64_t T) {
    int4* p = static_cast<int4*>(workspace);
    return RunList{p, p + 1, reinterpret_cast<int*>(p + 1 + T)};
}

__device__ __forceinline__ int bucket_of(int block) { return (int)((uint32_t)block * 2654435761u >> 19); }

// One CTA: the runs of a call, in no particular order.
__global__ void __launch_bounds__(kRunThreads) q8_runs_kernel(const int32_t* __restrict__ slots, int64_t T, int64_t num_slots,
                                                              RunList list) {
    __shared__ int bucket[kBuckets];
    __shared__ int count;
    griddep_wait();
    griddep_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31;
    for (int i = tid; i < kBuckets; i += kRunThreads) bucket[i] = -1;
    if (tid == 0) count = 0;
    __syncthreads();
    for (int64_t base = 0; base < T; base += (int64_t)kRunThreads * kRunUnroll) {
        int block[kRunUnroll], before[kRunUnroll];
#pragma unroll
        for (int u = 0; u < kRunUnroll; ++u) {
            const int64_t t = base + u * kRunThreads + tid;
            block[u] = t < T ? __ldg(slots + t) : -1;
            before[u] = lane == 0 && t > 0 && t <= T ? __ldg(slots + t - 1) : -1;
        }
#pragma unroll
        for (int u = 0; u < kRunUnroll; ++u) {
            block[u] = block_of(block[u], num_slots);
            const int left = __shfl_up_sync(0xffffffffu, block[u], 1);
            const int prev = lane == 0 ? block_of(before[u], num_slots) : left;
            const bool first = block[u] >= 0 && block[u] != prev;
            const uint32_t firsts = __ballot_sync(0xffffffffu, first);
            int at = 0;
            if (lane == 0 && firsts) at = atomicAdd(&count, __popc(firsts));
            at = __shfl_sync(0xffffffffu, at, 0) + __popc(firsts & ((1u << lane) - 1));
            if (first) {
                const int next = atomicExch(&bucket[bucket_of(block[u])], at);
                list.runs[at] = make_int4((int)(base + u * kRunThreads + tid), block[u], next, 0);
            }
        }
    }
    __syncthreads();
    for (int i = tid; i < kBuckets; i += kRunThreads) {
        const int r = bucket[i];
        list.buckets[i] = r;
        if (r >= 0 && list.runs[r].z < 0) list.runs[r].w = 1;
    }
    if (tid == 0) list.head[0] = make_int4(count, 0, 0, 0);
}

// Tokens of the run that begins at `start`: their rows into the owner table.  (Tokens behind its end that lie in the same
// block belong to runs of the same block: they are taken with this one anyway.)
__device__ __forceinline__ void take_run(StoreShared& sh, const Store& s, int64_t start, int block) {
    for (int64_t j = start + threadIdx.x;; j += kStoreThreads) {
        const int slot = j < s.T ? __ldg(s.slots + j) : -1;
        const bool in = block_of(slot, s.num_slots) == block;
        if (in) atomicMax(&sh.owner[slot % kGrain], (int)j);
        if (!__syncthreads_and(in)) return;
    }
}

template <typename SrcT>
__global__ void __launch_bounds__(kStoreThreads) store_runs_kernel(const Store s, const RunList list) {
    __shared__ StoreShared sh;
    griddep_wait();
    griddep_launch_dependents();
    const int64_t units = (int64_t)list.head[0].x * s.KVH;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int r = (int)(u / s.KVH), kvh = (int)(u - (int64_t)r * s.KVH);
        const int4 run = list.runs[r];
        __syncthreads();  // the unit before this one has read the owners
        if (threadIdx.x < kGrain) sh.owner[threadIdx.x] = -1;
        __syncthreads();
        bool first = true;
        if (!run.w)
            for (int o = list.buckets[bucket_of(run.y)]; o >= 0 && first;) {
                const int4 other = list.runs[o];
                first = other.y != run.y || other.x >= run.x;
                o = other.z;
            }
        if (!first) continue;  // uniform
        take_run(sh, s, run.x, run.y);
        if (!run.w)
            for (int o = list.buckets[bucket_of(run.y)]; o >= 0;) {
                const int4 other = list.runs[o];
                if (other.y == run.y && o != r) take_run(sh, s, other.x, run.y);
                o = other.z;
            }
        store_block<SrcT>(sh, s, run.y, kvh);
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
    const RunList list = run_list(workspace, s.T);
    cfg.gridDim = dim3(1);
    cfg.blockDim = dim3(kRunThreads);
    NVLLM_CUDA_OK(cudaLaunchKernelEx(&cfg, q8_runs_kernel, s.slots, s.T, s.num_slots, list));
    cfg.gridDim = dim3((unsigned)std::min<int64_t>(s.T * s.KVH, (int64_t)sm_count() * 8));
    cfg.blockDim = dim3(kStoreThreads);
    NVLLM_CUDA_OK(cudaLaunchKernelEx(&cfg, f32 ? store_runs_kernel<float> : store_runs_kernel<__nv_bfloat16>, s, list));
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
