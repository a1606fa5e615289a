// copy_pages: pages of a paged cache copied to other pages, in many tensors at once, and block tables brought in line.
//
// Forking a conversation copies its last, partly filled page for the child; compacting a pool moves pages to free ones and
// points the tables at them.  Both touch every layer's K and V (and, in 8 bits, their scales), so one call takes all of them:
// a launch per tensor would cost a 36-layer model 144 of them.
//
// Pure data movement: 2 bytes of traffic per byte copied.  A page of a tensor is cut into pieces of kPieceBytes; a CTA takes
// one piece of one tensor (blockIdx.y: its entry of the parameters is then read by all threads at once; found by a search
// among the pieces of all tensors, four pages of 144 tensors took 30 us instead of 13).  A CTA looks through the pairs for one
// that forbids its own while its loads are in flight: at 4096 pairs it reads as much of them as it copies, from the L2 (K and V
// in 8 bits with their scales, 8 kv heads, pages of 256 tokens: 710 us, 0.94 of a plain copy's rate; of 64 tokens, where a page
// is half a piece, 218 us, 0.77).  Several pieces a CTA, each with its own look, are the same within 3 %.
#include "common.cuh"

#include <algorithm>

namespace nvllm {
namespace pages {

constexpr int kThreads = 256;
constexpr int kUnroll = 8;
constexpr int kPieceBytes = kThreads * kUnroll * 16;  // 32 KB
constexpr int kFew = 16, kMany = 512;                 // tensors of a launch: the parameters are of one of two sizes

__device__ int g_error_flag = 0;  // bit 7 (128): a pair was not carried out

struct Cache {
    uint8_t* base;
    int rows, row_bytes;  // of a page; bytes of a row
};
struct Common {
    const int32_t *src, *dst, *tokens;
    int n, block_size;
    int64_t NB;
    int pieces;        // of the largest page
    int copy_ctas;     // per tensor, n * pieces; CTAs behind them take the tables
    int32_t* tables;
    int64_t table_entries;
};
template <int kCaches>
struct Params : Common {
    Cache caches[kCaches];
};

__device__ __forceinline__ bool in_pool(const Common& p, int page) { return page >= 0 && page < p.NB; }

// Whether pair j stands in the way of another pair, (s, d) at place i: it reads the page that i would write, or writes the same
// page later in the list.  With these left out no page is both read and written, and none is written twice.
__device__ __forceinline__ bool forbids(const Common& p, int j, int i, int d) {
    if (j == i) return false;
    const int sj = __ldg(p.src + j), dj = __ldg(p.dst + j);
    return in_pool(p, sj) && in_pool(p, dj) && (sj == d || (dj == d && j > i));
}

template <int kCaches>
__global__ void __launch_bounds__(kThreads) copy_pages_kernel(const __grid_constant__ Params<kCaches> p) {
    const int tid = threadIdx.x;
    griddep_wait();
    griddep_launch_dependents();
    // The tables: an entry that names a source names its destination now.  A thread goes through the list for its entry, and once more for
    // the pair that names it, the threads of a warp one after the other: 64 x 32 entries that all name one of 96 pairs 270 us, of
    // 4096 pairs 12 ms; entries that name none cost nothing beside the copy.
    if ((int)blockIdx.x >= p.copy_ctas) {
        const int64_t at = (int64_t)(blockIdx.x - p.copy_ctas) * kThreads + tid;
        if (blockIdx.y > 0 || at >= p.table_entries) return;
        const int page = p.tables[at];
        if (!in_pool(p, page)) return;
        for (int i = 0; i < p.n; ++i) {
            if (__ldg(p.src + i) != page) continue;
            const int d = __ldg(p.dst + i);
            bool ok = in_pool(p, d);
            for (int j = 0; ok && j < p.n; ++j) ok = !forbids(p, j, i, d);
            if (ok) {
                p.tables[at] = d;
                return;
            }
        }
        return;
    }
    const Cache cache = p.caches[blockIdx.y];
    const int64_t page_bytes = (int64_t)cache.rows * cache.row_bytes;
    const bool wide = (((uintptr_t)cache.base | (uintptr_t)cache.row_bytes) & 15) == 0;
    const int i = (int)blockIdx.x / p.pieces;
    const int64_t off = (int64_t)((int)blockIdx.x - i * p.pieces) * kPieceBytes;
    if (off >= page_bytes) return;
    const int s = __ldg(p.src + i), d = __ldg(p.dst + i);
    if (!in_pool(p, s) || !in_pool(p, d) || s == d) return;
    int64_t live = page_bytes;
    if (p.tokens != nullptr) {
        const int64_t t = max(0, min(__ldg(p.tokens + i), p.block_size));
        live = (t * cache.rows + p.block_size - 1) / p.block_size * cache.row_bytes;
    }
    const int bytes = (int)max((int64_t)0, min((int64_t)kPieceBytes, live - off));  // pages may have more than 2^31
    if (bytes == 0 && off > 0) return;  // a page's first piece looks at the pair even where nothing is live
    const uint8_t* const from = cache.base + s * page_bytes + off;
    uint8_t* const to = cache.base + d * page_bytes + off;
    uint4 x[kUnroll];
    if (wide) {
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            const int at = (k * kThreads + tid) * 16;
            if (at < bytes) x[k] = __ldg(reinterpret_cast<const uint4*>(from + at));
        }
    }
    bool bad = false;
    for (int j = tid; j < p.n; j += kThreads) bad |= forbids(p, j, i, d);
    if (__syncthreads_or(bad)) {
        if (tid == 0) atomicOr(&g_error_flag, 128);
        return;
    }
    if (wide) {
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            const int at = (k * kThreads + tid) * 16;
            if (at < bytes) *reinterpret_cast<uint4*>(to + at) = x[k];
        }
    } else {  // scales of few heads: rows of 4 or 8 bytes
        for (int at = tid * 4; at < bytes; at += kThreads * 4)
            *reinterpret_cast<uint32_t*>(to + at) = __ldg(reinterpret_cast<const uint32_t*>(from + at));
    }
}

}  // namespace pages

int read_pages_flags(int* out) {
    NVLLM_CUDA_OK(cudaMemcpyFromSymbol(out, pages::g_error_flag, sizeof(int)));
    return NVLLM_B200_OK;
}
int clear_pages_flags() {
    const int zero = 0;
    NVLLM_CUDA_OK(cudaMemcpyToSymbol(pages::g_error_flag, &zero, sizeof(int)));
    return NVLLM_B200_OK;
}
}  // namespace nvllm

extern "C" int nvllm_b200_copy_pages(void* const* caches_host, const int32_t* page_rows_host, const int64_t* row_bytes_host,
                                     int num_caches, const int32_t* src, const int32_t* dst, const int32_t* tokens, int n,
                                     int64_t NB, int block_size, int32_t* block_tables, int64_t table_entries, void* stream) {
    using namespace nvllm;
    using namespace nvllm::pages;
    const char* who = "copy_pages";
    if (num_caches < 0 || n < 0 || NB < 0 || block_size <= 0 || table_entries < 0)
        return fail(NVLLM_B200_EINVAL, "%s: negative size (num_caches=%d n=%d NB=%lld block=%d table_entries=%lld)", who, num_caches, n,
                    (long long)NB, block_size, (long long)table_entries);
    if (NB > 0x7fffffffLL) return fail(NVLLM_B200_EUNSUPPORTED, "%s: more than 2^31-1 pages", who);
    if (num_caches > 0 && (!caches_host || !page_rows_host || !row_bytes_host)) return fail(NVLLM_B200_EINVAL, "%s: null pointer", who);
    for (int c = 0; c < num_caches; ++c) {
        const int64_t rows = page_rows_host[c], row = row_bytes_host[c];
        if (rows <= 0 || block_size % rows)
            return fail(NVLLM_B200_EUNSUPPORTED, "%s: cache %d has %lld rows a page, not a divisor of block_size %d", who, c,
                        (long long)rows, block_size);
        if (row <= 0 || row % 4 || row > 0x7fffffffLL)
            return fail(NVLLM_B200_EUNSUPPORTED, "%s: cache %d has rows of %lld bytes, not a multiple of 4", who, c, (long long)row);
        if (NB > 0 && n > 0 && !caches_host[c]) return fail(NVLLM_B200_EINVAL, "%s: null pointer", who);
        if ((uintptr_t)caches_host[c] & 3) return fail(NVLLM_B200_EINVAL, "%s: caches must be 4-byte aligned", who);
    }
    if (n == 0 || NB == 0) return NVLLM_B200_OK;
    if (!src || !dst || (table_entries > 0 && !block_tables)) return fail(NVLLM_B200_EINVAL, "%s: null pointer", who);
    if (((uintptr_t)src | (uintptr_t)dst | (uintptr_t)tokens | (uintptr_t)block_tables) & 3)
        return fail(NVLLM_B200_EINVAL, "%s: index arrays must be 4-byte aligned", who);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kThreads);
    cfg.stream = reinterpret_cast<cudaStream_t>(stream);
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    for (int c0 = 0; c0 < num_caches || c0 == 0; c0 += kMany) {
        const int count = std::min(num_caches - c0, kMany);
        Params<kMany> p = {};
        int64_t pieces = 1;
        for (int c = 0; c < count; ++c) {
            p.caches[c] = Cache{(uint8_t*)caches_host[c0 + c], page_rows_host[c0 + c], (int)row_bytes_host[c0 + c]};
            pieces = std::max(pieces, ((int64_t)page_rows_host[c0 + c] * row_bytes_host[c0 + c] + kPieceBytes - 1) / kPieceBytes);
        }
        if (pieces > 0x3fffffffLL) return fail(NVLLM_B200_EUNSUPPORTED, "%s: pages too large", who);
        p.pieces = (int)pieces;
        p.src = src;
        p.dst = dst;
        p.tokens = tokens;
        p.n = n;
        p.block_size = block_size;
        p.NB = NB;
        const int64_t copy_ctas = count > 0 ? (int64_t)n * pieces : 0;
        const bool last = c0 + kMany >= num_caches;
        p.tables = last ? block_tables : nullptr;
        p.table_entries = last ? table_entries : 0;
        const int64_t ctas = copy_ctas + (p.table_entries + kThreads - 1) / kThreads;
        if (ctas > 0x7fffffffLL) return fail(NVLLM_B200_EUNSUPPORTED, "%s: too many pages", who);
        if (ctas == 0) break;
        p.copy_ctas = (int)copy_ctas;
        cfg.gridDim = dim3((unsigned)ctas, (unsigned)std::max(count, 1));
        if (count > kFew) {
            NVLLM_CUDA_OK(cudaLaunchKernelEx(&cfg, copy_pages_kernel<kMany>, p));
        } else {
            Params<kFew> few;
            static_cast<Common&>(few) = p;
            std::copy(p.caches, p.caches + kFew, few.caches);
            NVLLM_CUDA_OK(cudaLaunchKernelEx(&cfg, copy_pages_kernel<kFew>, few));
        }
    }
    return NVLLM_B200_OK;
}
