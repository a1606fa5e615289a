// copy_pages: pages of a paged cache copied to other pages, in many tensors at once, and block tables brought in line.
//
// Forking a conversation copies its last, partly filled page for the child; compacting a pool moves pages to free ones and
// points the tables at them.  Both touch every layer's K and V (and, in 8 bits, their scales), so one call takes all of them:
// a launch per tensor would cost a 36-layer model 144 of them.
//
// Pure data movement: 2 bytes of traffic per byte copied.  A page of a tensor is cut into pieces of kPieceBytes; a CTA takes
// one piece, or a few where there are many.  A CTA looks through the pairs for one that forbids its own (see refused) while
// its loads are in flight.
#include "common.cuh"

#include <algorithm>

namespace nvllm {
namespace pages {

constexpr int kThreads = 256;
constexpr int kUnroll = 8;
constexpr int kPieceBytes = kThreads * kUnroll * 16;  // 32 KB
constexpr int kMaxCaches = 128;                       // per launch: 2 KB of parameters

__device__ int g_error_flag = 0;  // bit 7 (128): a pair was not carried out

struct Cache {
    uint8_t* base;
    int row_bytes;
    int first_piece;  // of this cache among a pair's
};
struct Params {
    Cache caches[kMaxCaches];
    int rows[kMaxCaches];  // of a page
    int num_caches, pieces;  // pieces of a pair, over all caches
    const int32_t *src, *dst, *tokens;
    int n, block_size;
    int64_t NB;
    int64_t copy_ctas;  // CTAs behind them take the tables
    int64_t units;      // n * pieces
    int32_t* tables;
    int64_t table_entries;
};

__device__ __forceinline__ bool in_pool(const Params& p, int page) { return page >= 0 && page < p.NB; }

// Whether pair j stands in the way of another pair, (s, d) at place i: it reads the page that i would write, or writes the same
// page later in the list.  With these left out no page is both read and written, and none is written twice.
__device__ __forceinline__ bool forbids(const Params& p, int j, int i, int d) {
    if (j == i) return false;
    const int sj = __ldg(p.src + j), dj = __ldg(p.dst + j);
    return in_pool(p, sj) && in_pool(p, dj) && (sj == d || (dj == d && j > i));
}

__global__ void __launch_bounds__(kThreads) copy_pages_kernel(const __grid_constant__ Params p) {
    const int tid = threadIdx.x, lane = tid & 31;
    griddep_wait();
    griddep_launch_dependents();
    if ((int64_t)blockIdx.x >= p.copy_ctas) {  // the tables: an entry that names a source names its destination now
        const int64_t at = ((int64_t)blockIdx.x - p.copy_ctas) * kThreads + tid;
        if (at >= p.table_entries) return;
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
    for (int64_t u = blockIdx.x; u < p.units; u += p.copy_ctas) {
        const int i = (int)(u / p.pieces), piece = (int)(u - (int64_t)i * p.pieces);
        const int s = __ldg(p.src + i), d = __ldg(p.dst + i);
        if (!in_pool(p, s) || !in_pool(p, d) || s == d) continue;
        int c = -1;  // the last cache that begins at or before the piece
#pragma unroll
        for (int w = 0; w < kMaxCaches; w += 32)
            c += __popc(__ballot_sync(0xffffffffu, w + lane < p.num_caches && p.caches[w + lane].first_piece <= piece));
        const Cache cache = p.caches[c];
        const int rows = p.rows[c];
        const int64_t page_bytes = (int64_t)rows * cache.row_bytes;
        int64_t live = page_bytes;
        if (p.tokens != nullptr) {
            const int64_t t = max(0, min(__ldg(p.tokens + i), p.block_size));
            live = (t * rows + p.block_size - 1) / p.block_size * cache.row_bytes;
        }
        const int64_t off = (int64_t)(piece - cache.first_piece) * kPieceBytes;
        const int bytes = (int)min((int64_t)kPieceBytes, live - off);
        if (bytes <= 0 && off > 0) continue;  // the cache's first piece looks at the pair even where nothing is live
        const uint8_t* const from = cache.base + s * page_bytes + off;
        uint8_t* const to = cache.base + d * page_bytes + off;
        const bool wide = (((uintptr_t)cache.base | (uintptr_t)cache.row_bytes) & 15) == 0;
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
            continue;
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
    int c0 = 0;
    do {
        Params p = {};
        int64_t pieces = 0;
        for (; c0 < num_caches && p.num_caches < kMaxCaches; ++c0) {
            const int64_t page = (int64_t)page_rows_host[c0] * row_bytes_host[c0];
            const int64_t mine = (page + kPieceBytes - 1) / kPieceBytes;
            if (pieces + mine > 0x3fffffffLL) {
                if (p.num_caches == 0) return fail(NVLLM_B200_EUNSUPPORTED, "%s: page of %lld bytes too large", who, (long long)page);
                break;
            }
            p.caches[p.num_caches] = Cache{(uint8_t*)caches_host[c0], (int)row_bytes_host[c0], (int)pieces};
            p.rows[p.num_caches++] = page_rows_host[c0];
            pieces += mine;
        }
        p.pieces = (int)pieces;
        p.src = src;
        p.dst = dst;
        p.tokens = tokens;
        p.n = n;
        p.block_size = block_size;
        p.NB = NB;
        p.units = (int64_t)n * pieces;
        // A piece per CTA; with very many, up to 16 of them, so that the look through a long list of pairs is shared.
        const int64_t wave = (int64_t)sm_count() * 64;
        const int64_t each = std::max<int64_t>(1, std::min<int64_t>(16, p.units / wave));
        p.copy_ctas = (p.units + each - 1) / each;
        if (c0 == num_caches) p.tables = block_tables, p.table_entries = table_entries;
        const int64_t ctas = p.copy_ctas + (p.table_entries + kThreads - 1) / kThreads;
        if (ctas > 0x7fffffffLL) return fail(NVLLM_B200_EUNSUPPORTED, "%s: too many pages", who);
        if (ctas == 0) break;
        cfg.gridDim = dim3((unsigned)ctas);
        NVLLM_CUDA_OK(cudaLaunchKernelEx(&cfg, copy_pages_kernel, p));
    } while (c0 < num_caches);
    return NVLLM_B200_OK;
}
