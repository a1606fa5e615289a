// What the prefill kernels have in common (varlen_prefill.cu: packed keys or bf16 pages; paged_prefill_q8.cu: 8-bit pages): the
// tcgen05 wrappers, the (token, head) rows of a Q tile, the items of the work list and how items are cut into runs.
#pragma once

#include "store_kvcache.cuh"

#include <algorithm>

namespace nvllm {
namespace prefill {

constexpr int kD = 128;
constexpr int kTileQ = 128;            // rows per Q tile
constexpr int kTileKV = 128;
constexpr int kPanelBytes = 128 * 128;  // 128 rows x 64 dims bf16, 128B-swizzled
constexpr int kTileBytes = 2 * kPanelBytes;
constexpr int kMaxLevels = 4096;       // K/V tiles per sequence the plan kernel can rank items by
constexpr uint32_t kTmemCols = 512;
constexpr float kRescaleThreshold = 8.0f;  // log2 units

// A (sequence, token block) pair, longest causal span first: {first query token of the sequence, its query length, first
// token of the block, sequence index} and {first key token (packed keys), key length, 0, 0}.
struct Record {
    int4 q, k;
};

// What a Q tile holds: `tokens` consecutive tokens of `heads` neighbouring q heads of one kv head, token after token, and what
// the item's second tile holds beside it.  All heads of a kv head see the same keys, so the narrower the block of tokens, the
// fewer rows lie behind a sequence's end and the more of a diagonal tile is behind every row (skipped, see key_steps).
struct Pack {
    int heads, tokens;  // of a tile
    int dq, dh;         // tile B: dq tokens further, or dh heads further
    int span;           // tokens of an item
    int per_kv;         // items per kv head and token block
};
// A kv head's G q heads in one item, half of them per tile: both tiles then see the same keys and finish together.  An odd
// number goes into both tiles, which take tokens in turn (B may see one K/V tile more).  Groups of more than eight heads are
// cut into equal parts.  `lone`: items of tile A alone, twice as many (see lone_tiles).
inline Pack make_pack(int G, bool lone = false) {
    int w = std::min(G, 8);
    while (G % w) --w;
    Pack k;
    k.heads = w % 2 ? w : w / 2;
    k.tokens = kTileQ / k.heads;
    k.dq = w % 2 ? k.tokens : 0;
    k.dh = w % 2 ? 0 : k.heads;
    k.span = w % 2 ? 2 * k.tokens : k.tokens;
    k.per_kv = G / w;
    if (lone) k.dq = 1 << 28, k.dh = 0, k.span = k.tokens, k.per_kv = G / k.heads;  // no tokens behind dq: no tile B
    return k;
}

struct Params {
    const int4* items;  // record 0: {number of pairs, items claimed, head groups, 0}; then the two halves of every Record
    const int32_t* block_tables;  // [B, MB] page ids, or nullptr for packed keys/values
    int MB, block_size;
    __nv_bfloat16* out;
    int H, G;
    Pack pack;
    int per_pair;  // items per (sequence, token block)
    int wide;      // out is aligned to 32 bytes
    float scale_log2;
};

// Few items with many keys each (a short question behind a long cached conversation): the K/V tiles of an item are cut into
// up to `splits` contiguous runs, one per CTA, which leave partial results that prefill_combine_kernel puts together.
struct SplitParams : Params {
    float* partials;  // [CTA][Q tile][kPartialFloats]
    int splits;
    int ctas;  // the launch's
};
constexpr int kPartialFloats = kTileQ * kD + 2 * kTileQ;  // O[128][128] relative to m, then m[128] (log2 units) and l[128]
// K/V tiles per run.  A row that sees none of a run's keys would have no maximum.  An item's first token sees all of its tiles
// but one (two where the item has more tokens than a tile keys).
__host__ __device__ __forceinline__ int min_run(int span) { return span > kTileKV ? 3 : 2; }
// Items of fewer tiles stay whole: they take less time than the partial results and the combining launch (about 6 us).  The
// rule looks at an item's own tiles, so that packed keys and keys in pages give the same bits.  20 new tokens behind 1200 cached
// ones, 16 / 2 heads: whole 27.6 us, cut 19.6; 100 behind 8000, 32 / 8: 130 and 35.
constexpr int kSplitTiles = 8;
constexpr int kMaxSplits = 16;  // runs per item
// A sequence without a cached prefix is cut only if it has more keys: below, whole items leave the launch short (no plan kernel, the
// scatter in it).  One prompt of 1200, 8 / 2 heads, whole 25.2 us, cut 27.5; of 1500, 8 / 1, whole 34.6, cut 28.0.
constexpr int kWholeKeys = 11 * kTileKV;
// The launch has a CTA for every run that the host could foresee.  Where the device's lengths make more items than that (a
// captured launch whose lengths were rewritten), the items stay whole and the CTAs claim them one by one.
__device__ __forceinline__ int splits_of(const SplitParams& p, int pairs) {
    return (long long)pairs * p.per_pair * p.splits <= p.ctas ? p.splits : 1;
}
__device__ __forceinline__ int runs_of(const Params& p, int splits, int n_a, int prefix, int len_k) {
    return n_a < kSplitTiles || (prefix == 0 && len_k <= kWholeKeys) ? 1 : min(splits, n_a / min_run(p.pack.span));
}

__device__ __forceinline__ Record record_of(const Params& p, int pair) {
    return Record{__ldg(p.items + 1 + 2 * pair), __ldg(p.items + 2 + 2 * pair)};
}
__device__ __forceinline__ int claim_item(const Params& p) {
    return (int)gridDim.x + atomicAdd(&const_cast<int4*>(p.items)->y, 1);
}
// The item list's header, read once per thread.
struct List {
    int pairs, groups;
};
__device__ __forceinline__ List list_of(const Params& p) {
    const int4 h = p.items[0];
    return List{h.x, h.z};
}
__device__ __forceinline__ int items_of(const Params& p, const List& l) { return l.pairs * p.per_pair; }
__device__ __forceinline__ int items_of(const SplitParams& p, const List& l) {
    return l.pairs * p.per_pair * splits_of(p, l.pairs);
}

// Items of which the last ones are cut: `whole` in front stay as they are, of those behind every one is `splits` runs.
struct Cut {
    int whole, splits;
};
__device__ __forceinline__ Cut cut_of(const SplitParams& p, const List& l) { return Cut{0, splits_of(p, l.pairs)}; }

// ------------------------------------------------------------------------------------------
// tcgen05 wrappers
// ------------------------------------------------------------------------------------------
__device__ __forceinline__ void tmem_alloc(uint32_t* smem_dst, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem_dst)),
                 "r"(ncols)
                 : "memory");
}
__device__ __forceinline__ void tmem_relinquish() {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}

// D[tmem] (+)= A[smem] * B[smem]
__device__ __forceinline__ void mma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(acc)
        : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
        "}\n" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(acc)
        : "memory");
}

// 32 lanes x 32 consecutive 32-bit columns: thread i of the warp gets lane (base + i), columns c..c+31.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
        "%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,"
        "%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
// 32 lanes x 16 columns, from the first 16 words of r.
template <int N>
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[N]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
            taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// Packed fp32 pairs (one instruction, two lanes of math) and the three-input max of sm_100.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Shared-memory matrix descriptor, 128-byte swizzle, version 1 (sm_100).
__device__ __forceinline__ uint64_t make_desc(uint32_t smem_addr, uint32_t lbo_bytes, uint32_t sbo_bytes) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr >> 4) & 0x3FFF);
    d |= (uint64_t)((lbo_bytes >> 4) & 0x3FFF) << 16;
    d |= (uint64_t)((sbo_bytes >> 4) & 0x3FFF) << 32;
    d |= (uint64_t)1 << 46;  // descriptor version
    d |= (uint64_t)2 << 61;  // SWIZZLE_128B
    return d;
}
// K-major operand tile [128 rows][128 dims] stored as two 64-dim panels; k-step = 16 dims.
__device__ __forceinline__ uint64_t kmajor_desc(uint32_t tile_addr, int ks) {
    return make_desc(tile_addr + (ks >> 2) * kPanelBytes + (ks & 3) * 32, 16, 1024);
}
// MN-major operand: V tile [128 tokens][128 dims] as two 64-dim panels; N = dims, K = tokens; k-step = 16 tokens.
__device__ __forceinline__ uint64_t mnmajor_desc(uint32_t tile_addr, int ks) {
    return make_desc(tile_addr + ks * 16 * 128, kPanelBytes, 1024);
}

constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 4) << 24);
constexpr uint32_t idesc_qk(uint32_t keys) { return kIdesc | ((keys >> 3) << 17); }
constexpr uint32_t kIdescPV = kIdesc | ((128u >> 3) << 17) | (1u << 16);  // B operand MN-major

struct Item {
    int seq_start, len, q0, head;      // first query token of the sequence, query length, first token of the block, first head
    int k_start, len_k, prefix, kvh;   // first key token (packed keys), key length, len_k - len, kv head
    int n_a, n_b, n_kv, b;             // KV tiles seen by Q tile A, by Q tile B (0: no such rows; else n_a or n_a + 1), the
                                       // larger (0: nothing to do; -1: no more items), sequence
    int kv0;                           // a run of a split item: its first KV tile (len_k and prefix count from there on), else -1
};
// Keys up to the last one that a row of Q tile x sees, counted from the item's first K/V tile.
__device__ __forceinline__ int visible_keys(const Params& p, const Item& it, int x) {
    return it.prefix + min(it.len, it.q0 + x * p.pack.dq + p.pack.tokens);
}
// Steps of 16 keys of the tile's n-th and last K/V tile that hold any of them: what its two products go through.
__device__ __forceinline__ int key_steps(int keys, int n) { return (min(kTileKV, keys - (n - 1) * kTileKV) + 15) >> 4; }

// Item r (of per_pair) of a (sequence, token block).
__device__ __forceinline__ Item make_item(const Params& p, const Record& rec, int r) {
    Item it;
    it.kvh = r / p.pack.per_kv;
    it.head = it.kvh * p.G + (r - it.kvh * p.pack.per_kv) * (p.G / p.pack.per_kv);
    const int4 q = rec.q, k = rec.k;
    it.seq_start = q.x;
    it.len = q.y;
    it.q0 = q.z;
    it.b = q.w;
    it.k_start = k.x;
    it.len_k = k.y;
    it.prefix = it.len_k - it.len;  // >= 0: the plan kernel publishes no items otherwise
    it.n_a = (visible_keys(p, it, 0) - 1) / kTileKV + 1;
    it.n_b = it.len - it.q0 > p.pack.dq ? (visible_keys(p, it, 1) - 1) / kTileKV + 1 : 0;
    it.n_kv = max(it.n_a, it.n_b);
    it.kv0 = -1;
    return it;
}
// Items go by head group (see head_groups), in a group by pair.
__device__ __forceinline__ Item load_item(const Params& p, const List& l, int idx) {
    int per = p.per_pair, first = 0;
    if (l.groups > 1) {
        per /= l.groups;
        first = idx / (l.pairs * per) * per;
        idx -= first * l.pairs;
    }
    const int pair = idx / per;
    return make_item(p, record_of(p, pair), first + idx - pair * per);
}
// Run c of an item that is cut into up to `splits`; one with nothing to do (n_kv = 0) where it has fewer.
__device__ __forceinline__ void take_run(const Params& p, Item& it, int c, int splits) {
    const int runs = runs_of(p, splits, it.n_a, it.prefix, it.len_k);
    if (c >= runs) {
        it.n_a = it.n_b = it.n_kv = 0;
        return;
    }
    if (runs == 1) return;
    const int j0 = it.n_a * c / runs, j1 = c + 1 == runs ? it.n_kv : it.n_a * (c + 1) / runs;
    it.kv0 = j0;
    it.n_a = min(it.n_a, j1) - j0;
    it.n_b = it.n_b > 0 ? min(it.n_b, j1) - j0 : 0;
    it.n_kv = j1 - j0;
    it.len_k -= j0 * kTileKV;
    it.prefix -= j0 * kTileKV;
}
__device__ __forceinline__ Item load_item(const SplitParams& p, const List& l, int idx) {
    const int splits = splits_of(p, l.pairs), c = idx % splits;
    Item it = load_item(static_cast<const Params&>(p), l, idx / splits);
    take_run(p, it, c, splits);
    return it;
}

// A few rounds of items, each an SM's work for a long time: those of the last round, which leaves SMs idle, are cut into runs as well.  `ctas`:
// the launch's, which claim the items in their order and then the runs.  (8-bit pages only: packed bf16 keys and bf16 keys in pages
// are to give the same bits.)  Whole and cut, 32 / 8 heads: 1280 new tokens (160 items) behind 30 000 1044 and 637 us, behind 8000 304 and 225,
// behind 2500 121 and 117; 640 (80 items) behind 8000 157 and 143; 2560 (320) 473 and 410; 20 x 64 behind 3000 126 and 113.  Twice the room
// for results lets 2048 (256) be cut, too: 345 instead of 335, for at the power cap what idle SMs leave makes the others faster.
struct TailParams : Params {
    float* partials;  // [kTailSlots * ctas][Q tile][kPartialFloats]
    int ctas;
};
constexpr int kTailRounds = 3;  // there is a quarter to be gained at most behind more
constexpr int kTailSlots = 2;
constexpr int kTailRuns = 8;
// In K/V tiles' time: what a run costs beside its own (start, first scores, its results to memory), and the launch that combines them.
constexpr int kRunCost = 2, kCombineCost = 4;
// Runs for each of n items (fewer than CTAs) of so many K/V tiles: the number that ends first, 1 where that is the items as they are.
__host__ __device__ __forceinline__ int tail_runs(int n, int tiles, int ctas) {
    int best = 1, least = tiles < 2 * kSplitTiles ? 0 : tiles;
    for (int s = 2; s <= kTailRuns && n * s <= kTailSlots * ctas; ++s) {
        const int t = (n * s + ctas - 1) / ctas * ((tiles + s - 1) / s + kRunCost) + kCombineCost;
        if (t < least) least = t, best = s;
    }
    return best;
}
__device__ __forceinline__ Cut cut_of(const TailParams& p, const List& l) {
    const int total = items_of(static_cast<const Params&>(p), l), whole = total / p.ctas * p.ctas, n = total - whole;
    if (n == 0 || total > kTailRounds * p.ctas) return Cut{total, 1};
    const int runs = tail_runs(n, load_item(static_cast<const Params&>(p), l, whole).n_kv, p.ctas);
    return runs == 1 ? Cut{total, 1} : Cut{whole, runs};
}

// The output is marked as evicted first, so that it does not push keys and values out of the L2 (16 prompts of 128..4096 tokens, 32 / 8
// heads, with Q's loads marked too: 931 -> 912 us as one head group).  The GEMM that reads it next does not notice: attention and an
// o_proj-shaped GEMM together, outputs of 4 to 268 MB, take 0 to 0.4 % less with the mark.
__device__ __forceinline__ void store_32bytes(void* dst, const uint32_t (&w)[8]) {
    asm volatile("st.global.L1::no_allocate.L2::evict_first.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst), "r"(w[0]),
                 "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// ------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------
// Runs per item: as many as leave one run per SM; 1 where no item can have enough tiles.
inline int splits_for(int64_t items, int64_t max_tiles, int sms, int span) {
    if (items <= 0 || 2 * items > sms || max_tiles < kSplitTiles) return 1;
    return (int)std::min<int64_t>(std::min<int64_t>(sms / items, kMaxSplits), max_tiles / min_run(span));
}
// Whether split items are of one Q tile, which has its SM's exponentials to itself and takes no turns, rather than of two.  They are
// twice as many, so where the SMs do not suffice a run has more K/V tiles: worth up to three more where a tile's live rows fill more
// than a warp, none where they do not.  60 new tokens, 32 / 8 heads, behind 3000 cached ones (two / three tiles a run) 24.0 -> 21.3 us,
// behind 6500 (four / six) 29.5 -> 26.0, behind 12 000 (six / eleven, so still of two) 36.0, else 36.3; 16 / 8 heads there 32.7, else 35.6.
inline bool lone_tiles(int64_t max_tiles, int splits, int lone_splits, int64_t live_rows) {
    const int more = live_rows > 32 ? 3 : 0;
    return (max_tiles + lone_splits - 1) / lone_splits <= (max_tiles + splits - 1) / splits + more;
}
inline size_t partials_bytes(int sms) { return (size_t)sms * 2 * kPartialFloats * 4; }
// Whether `items` of up to max_tiles K/V tiles (bounds of what the device will find) leave a last round that is worth cutting.
inline bool tail_worth(int64_t items, int64_t max_tiles, int sms) {
    return 2 * items > sms && items <= (int64_t)kTailRounds * sms && items % sms && tail_runs((int)(items % sms), (int)max_tiles, sms) > 1;
}

// Keys and values in 8-bit pages: the main kernel is another one (paged_prefill_q8.cu).  `split`, `tail`: for runs, or null.
struct Bytes {
    const float *k_scale, *v_scale;
    int NB;
};
int launch_bytes(const Params& p, const SplitParams* split, const TailParams* tail, const Bytes& in, const void* q, const void* k, const void* v, int64_t slots,
                 int KVH, cudaLaunchConfig_t cfg);

}  // namespace prefill
}  // namespace nvllm
