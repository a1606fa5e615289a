// paged_decode_q8: flash decoding over the 8-bit paged cache (e4m3 values, an fp32 scale for every 64 slots and kv head).
//
//   out[b,h,:] = sum_t p_t vs_t V_t / sum_t p_t,   p_t = exp(scale * ks_t * q . K_t - max)
//
// The op is bound by the bytes of the live K and V rows, half as many as in bf16.  It walks them as the bf16 kernel does
// (paged_decode.cu: chunks of equal cost, persistent CTAs, a ring of 64-token tiles filled by TMA, partial results combined by
// whoever draws the last ticket); a tile is a block of the scales, so that there is one K and one V scale per tile.  What differs
// is the arithmetic between shared memory and the tensor cores:
//
//  * e4m3 -> fp16 is exact and one instruction for two values, so both products run in fp16 with fp32 accumulation
//    (mma.m16n8k16).  The bytes reach the registers by ldmatrix as if two of them were one 16-bit element:
//      S^T = K Q^T   a register holds dims 4 quad .. + 3 of a token.  The order of the dims within a k-step is free as long as
//                    Q has the same one, so the two converted pairs are the k-low and the k-high part of the fragment.
//      O^T += V^T P^T (transposed ldmatrix) a register holds dims 2u, 2u + 1 of tokens 2 quad, 2 quad + 1: one byte permutation
//                    puts the tokens side by side, and even dims become rows 0..7 of the fragment, odd ones rows 8..15.
//  * q is bf16 and may exceed fp16: every row is divided by the power of two in front of its largest magnitude, which goes
//    into the factor of its scores.  (A component below 2^-14 of that loses bits, at most 2^-25 of the largest one.)
//  * The V scale multiplies a tile's 16 x 8 products on their way into the fp32 accumulators: folding it into the fp16
//    probabilities would cost range where the blocks of a sequence differ in magnitude.
//  * The probabilities are fp16 (half a step is 2^-11; in bf16 it would be 2^-8), taken relative to 2^-kBias of the running
//    maximum.  Where a head's are all below 2^kLow in a tile they are taken relative to the tile's maximum instead, and the
//    products scaled back with the V scale: what underflows is then below 2^-20 of the tile's largest, which shares its V scale.
//  * The scales come with the tile: two 4-byte cp.async of the producer, whose completion the tile's barrier counts too.
#include "paged_decode.cuh"
#include "store_kvcache_q8.cuh"

namespace nvllm {
namespace q8 {
size_t store_workspace_bytes(int64_t T);
int check_store(const char* who, const Store& s, int64_t D, int src_dtype);
int launch_store(const char* who, const Store& s, int src_dtype, void* workspace, size_t workspace_bytes, cudaStream_t stream);
}  // namespace q8

namespace decode_q8 {

using namespace decode;

// CTAs per SM and their stages.  Under the power limit the SM clock falls and with it what the consumer warps, bound by the latency
// of their own chains, get done: three CTAs with three stages each hold as many bytes in flight as two with five, and give every
// scheduler a third warp (64 sequences of 512..8192 tokens, 32 / 8 heads, at 1.69 GHz: 103 us with two, 97 with three; 256 of
// 16..16384, 64 / 8: 229 and 214; four with two stages do not fit the registers: 144 and 307).
constexpr int kCtas = 3;
constexpr int kStages = 3;
constexpr int kItemCost = 3;                          // cost of a sequence boundary in tile units
constexpr int kMinUnits = 6;                          // units per CTA from which on more CTAs pay
constexpr int kTileBytes = kTile * kD;                // one K or V tile, 128B-swizzled
constexpr int kQBytes = kMaxG * kD * 2;
constexpr int kStageBytes = 2 * kTileBytes + kQBytes;
constexpr int kMiscBytes = 1024 + kThreads * 8;
constexpr int kSmemBytes = kStages * kStageBytes + kOsBytes + kMiscBytes;
static_assert(kSmemBytes + 1024 <= 228 * 1024 / kCtas, "CTAs per SM");
static_assert(kTile == q8::kGrain, "a tile has one scale");
constexpr float kBias = 10.f;                         // log2 units: the largest probability is stored as 2^kBias ...
constexpr float kStale = 4.f;                         // ... or up to 2^(kBias + kStale) until the maximum moves (fp16: 2^16)
constexpr float kLow = -4.f;

__device__ int g_error_flag = 0;  // bit 0 / 1: producer / consumer timed out

struct Params8 : Params {
    const float *k_scale, *v_scale;  // [num_slots / 64, KVH]
};

// D(16x8,f32) = A(16x16,f16,row) * B(16x8,f16,col) (+ D)
__device__ __forceinline__ void mma_add(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_new(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t lo_half2(uint32_t w) { return q8::e4m3x2_to_half2(w & 0xffffu); }
__device__ __forceinline__ uint32_t hi_half2(uint32_t w) { return q8::e4m3x2_to_half2(w >> 16); }
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void load_scale(float* dst, const float* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// An arrival that the barrier counts as one of its own, once this thread's cp.async before it have landed.
__device__ __forceinline__ void arrive_behind_scales(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__global__ void __launch_bounds__(kThreads, kCtas)
paged_decode_q8_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const Params8 p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    // swizzled tiles first: their addresses are multiples of 8 KB; the q rows of all stages behind them
    uint8_t* const q_rows = smem + kStages * 2 * kTileBytes;
    float* Os = reinterpret_cast<float*>(smem + kStages * kStageBytes);
    uint8_t* misc = smem + kStages * kStageBytes + kOsBytes;
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(misc);            // [kStages]
    uint64_t* empty_bar = full_bar + kStages;                          // [kStages]
    int* sm_i = reinterpret_cast<int*>(misc + 96);                     // scan sums [5], abort [6], ticket [7]
    volatile int* sm_abort = sm_i + 6;
    float2* sm_scale = reinterpret_cast<float2*>(misc + 128);          // [kStages] K and V scale of a tile
    float* sm_ml = reinterpret_cast<float*>(misc + 256);               // [2 parities][m|l][4 warps][8 rows]
    TileMeta* sm_meta = reinterpret_cast<TileMeta*>(misc + 768);       // [kStages]
    long long* sm_seg = reinterpret_cast<long long*>(misc + 1024);     // [kThreads] unit at which a thread's sequences start

    const int tid = threadIdx.x;
    const int warp = tid >> 5, lane = tid & 31;
    const int kvh = blockIdx.x % p.KVH;
    const int chunk = blockIdx.x / p.KVH;
    const int max_ctx = p.MB * p.block_size;

    if (smem_u32(smem) & 1023) {
        if (tid == 0) atomicOr(&g_error_flag, 1);
        griddep_wait();
        return;
    }
    if (tid == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full_bar + s, 2);  // the tiles' bytes, the scales
            mbar_init(empty_bar + s, kConsumerWarps);
        }
        fence_mbar_init();
        *sm_abort = 0;
        prefetch_tensormap(&tm_k);
        prefetch_tensormap(&tm_v);
    }
    griddep_launch_dependents();

    // What may be read before the kernel in front has finished is as in the bf16 kernel: it writes tickets and, in a decode
    // step, the rows and scales of the blocks that hold the step's slots.  A tile is such a block, or it is settled memory.
    int my_slots[kEarlySlots];
    const bool early = p.slot_mapping == nullptr || p.B <= 32 * kEarlySlots;
    if (warp == kConsumerWarps && p.slot_mapping != nullptr && early) {
#pragma unroll
        for (int i = 0; i < kEarlySlots; ++i)
            my_slots[i] = lane + 32 * i < p.B ? __ldg(p.slot_mapping + lane + 32 * i) : -1;
    }

    // ---- total cost units per head, and where on the line every thread's share of the sequences starts ----
    const int per = (p.B + kThreads - 1) / kThreads;
    {
        const int b_lo = min(p.B, tid * per), b_hi = min(p.B, b_lo + per);
        int mine = 0;
        for (int b = b_lo; b < b_hi; ++b) {
            const int tb = tiles_of(clamp_ctx(__ldg(p.context_lens + b), max_ctx));
            mine += units_of(tb, p.item_cost);
            if (tb == 0 && b % (int)gridDim.x == (int)blockIdx.x) {
                uint4* orow = reinterpret_cast<uint4*>(p.out + (size_t)b * p.H * kD);
                for (int i = 0; i < p.H * (kD * 2 / 16); ++i) orow[i] = make_uint4(0, 0, 0, 0);
            }
        }
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) sm_i[warp] = incl;
        __syncthreads();
        long long warp_off = 0;
        for (int w = 0; w < warp; ++w) warp_off += sm_i[w];
        sm_seg[tid] = warp_off + incl - mine;
        __syncthreads();
    }
    long long total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) total += sm_i[w];
    const Cut cut = make_cut(total, p.num_groups, kMinUnits);
    if (total == 0 || chunk >= cut.groups) {  // uniform across the CTA
        griddep_wait();
        return;
    }

    if (warp == kConsumerWarps) {
        // =========================== producer warp ===========================
        const uint64_t pol = policy_evict_first();
        Walk walk;
        walk.x0 = cut.bound(chunk);
        walk.x1 = cut.bound(chunk + 1);
        {
            int s = -1;  // last segment that starts at or before x0
#pragma unroll
            for (int w = 0; w < kWarps; ++w) s += __popc(__ballot_sync(0xffffffffu, sm_seg[32 * w + lane] <= walk.x0));
            walk.b = s * per;
            walk.fv = sm_seg[s];
        }
        // Lane 0 walks the tiles; the others help to compare a tile with the step's slots until the wait has been passed.
        Item item;
        int left = 0, valid = 0;  // tiles left of `item`, live tokens from the next tile on
        int bi = 0, off = 0;      // its page and the offset in the page
        int phys = 0, next = 0;   // that page's block and the following page's (requested one page ahead)
        const int32_t* bt = p.block_tables;
        int pf_b = -1, pf_ctx = 0, pf_phys = 0;  // the next sequence's length and first page, fetched one item ahead
        bool waited = false, ok = true;
        uint32_t it = 0, stage = 0, parity = 1;
#pragma unroll 1
        while (true) {
            int slot = -1, flags = 0;
            if (lane == 0) {
                if (left == 0 && next_item(walk, p, max_ctx, item, pf_b, pf_ctx)) {
                    left = item.n;
                    flags = kFirst;
                    valid = item.ctx - item.t0 * kTile;
                    bi = item.t0 == 0 ? 0 : item.t0 * kTile / p.block_size;
                    off = item.t0 * kTile - bi * p.block_size;
                    bt = p.block_tables + (size_t)item.b * p.MB;
                    phys = item.b == pf_b && bi == 0 ? pf_phys : __ldg(bt + bi);
                    next = bi + 1 < p.MB ? __ldg(bt + bi + 1) : 0;
                    if (walk.b < p.B) {
                        pf_b = walk.b;
                        pf_ctx = __ldg(p.context_lens + walk.b);
                        pf_phys = __ldg(p.block_tables + (size_t)walk.b * p.MB);
                    }
                }
                if (left > 0) {
                    slot = (phys < 0 ? 0 : (phys >= p.NB ? p.NB - 1 : phys)) * p.block_size + off;
                    if (--left == 0) flags |= item.n == item.tb ? kLast | kWhole : kLast;
                }
            }
            if (!waited) {
                const int first_slot = __shfl_sync(0xffffffffu, slot, 0);
                bool stop = !early || first_slot < 0 || it == kStages;
                if (p.slot_mapping != nullptr) {
#pragma unroll
                    for (int i = 0; i < kEarlySlots; ++i) {
                        if (32 * i >= p.B) break;
                        stop |= (uint32_t)(my_slots[i] - first_slot) < (uint32_t)kTile;
                    }
                }
                if (__any_sync(0xffffffffu, stop)) {
                    griddep_wait();
                    waited = true;
                    if (lane != 0) return;
                }
            }
            if (lane == 0) {
                uint8_t* st = smem + stage * 2 * kTileBytes;
                uint64_t* bar = full_bar + stage;
                if (it >= kStages && !wait_or_abort(sm_abort, empty_bar + stage, parity)) {
                    ok = false;
                    break;
                }
                if (slot < 0) {
                    sm_meta[stage].flags = kDone;
                    mbar_arrive(bar);
                    mbar_arrive(bar);
                    break;
                }
                sm_meta[stage].valid = valid;
                sm_meta[stage].flags = flags;
                sm_meta[stage].b = item.b;
                if ((flags & (kLast | kWhole)) == kLast) {
                    const long long first = item.fv + p.item_cost;  // unit of the sequence's tile 0
                    sm_meta[stage].part = (chunk * p.KVH + kvh) * 2 + (item.t0 == 0 ? 1 : 0);
                    sm_meta[stage].gf = item.t0 == 0 ? chunk : cut.chunk_of(first);
                    sm_meta[stage].gl = item.t0 + item.n == item.tb ? chunk : cut.chunk_of(first + item.tb - 1);
                }
                const size_t grain = (size_t)(slot / kTile) * p.KVH + kvh;
                load_scale(&sm_scale[stage].x, p.k_scale + grain);
                load_scale(&sm_scale[stage].y, p.v_scale + grain);
                arrive_behind_scales(bar);
                mbar_expect_tx(bar, 2 * kTileBytes + ((flags & kFirst) ? (uint32_t)p.G * kD * 2 : 0u));
                tma_load_3d_hint(st, &tm_k, bar, 0, slot, kvh, pol);
                tma_load_3d_hint(st + kTileBytes, &tm_v, bar, 0, slot, kvh, pol);
                if (flags & kFirst)
                    bulk_load(q_rows + stage * kQBytes, p.q + ((size_t)item.b * p.H + (size_t)kvh * p.G) * kD, (uint32_t)p.G * kD * 2, bar);
                valid -= kTile;
                off += kTile;
                if (off == p.block_size) {
                    off = 0;
                    phys = next;
                    ++bi;
                    next = bi + 1 < p.MB ? __ldg(bt + bi + 1) : 0;
                }
            }
            ++it;
            if (++stage == kStages) stage = 0, parity ^= 1u;
        }
        if (!ok) {
            *sm_abort = 1;
            atomicOr(&g_error_flag, 1);
            for (uint32_t j = (it >= kStages ? it - kStages : 0); j < it; ++j)  // loads in flight land before the memory is released
                (void)mbar_wait(full_bar + (j % kStages), (j / kStages) & 1u, polls_of_ms(90));
        }
        return;
    }

    // ============================= consumer warps =============================
    const int grp = lane >> 2;
    const int quad = lane & 3;
    const int mi = lane >> 3;        // which 8x8 matrix this lane addresses in ldmatrix.x4
    const int r8 = lane & 7;
    const int tok_base = warp * 16;
    const int ctid = tid;            // 0..127 among consumers
    uint32_t item = 0;
    uint32_t qb[8][2];               // Q^T: dims 16 ks + 4 quad (+ 1), (+ 2, + 3) of head grp
    float qf0 = 0.f, qf1 = 0.f;      // factors of the scores of heads 2 quad, 2 quad + 1
    float o[8][4];                   // O^T: dims 16 j + 2 grp and + 1 of the lane's two heads
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;  // per head (m less kBias); the sums are this lane's tokens only
    bool waited = false;             // for the kernel in front, which clears the tickets
    const uint32_t row_k = (uint32_t)(tok_base + (mi & 1) * 8 + r8) * 128;  // this lane's ldmatrix row

    for (uint32_t next = 0, parity = 0;;) {
        const uint32_t stage = next;
        if (!wait_or_abort(sm_abort, full_bar + stage, parity)) {
            *sm_abort = 1;
            atomicOr(&g_error_flag, 2);
            break;
        }
        if (++next == kStages) next = 0, parity ^= 1u;
        uint8_t* st = smem + stage * 2 * kTileBytes;
        const int2 head = *reinterpret_cast<const int2*>(sm_meta + stage);
        const int flags = head.y;
        if (flags & kDone) break;
        const float2 scale = sm_scale[stage];
        if (flags & kFirst) {
            const uint2* qs = reinterpret_cast<const uint2*>(q_rows + stage * kQBytes);
            uint32_t top = 0;
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                const uint2 w = grp < p.G ? qs[grp * 32 + ks * 4 + quad] : make_uint2(0u, 0u);
                qb[ks][0] = w.x, qb[ks][1] = w.y;
                top = max(top, max(max(w.x & 0x7fffu, w.x >> 16 & 0x7fffu), max(w.y & 0x7fffu, w.y >> 16 & 0x7fffu)));
            }
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const uint32_t e = min(max(top >> 7, 1u), 253u);  // biased exponent of the row's largest magnitude
            const float down = __uint_as_float((254u - e) << 23);
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    qb[ks][i] = pack_half(__uint_as_float(qb[ks][i] << 16) * down, __uint_as_float(qb[ks][i] & 0xffff0000u) * down);
            const float up = __uint_as_float(e << 23) * p.scale_log2;
            qf0 = __shfl_sync(0xffffffffu, up, 8 * quad);
            qf1 = __shfl_sync(0xffffffffu, up, 8 * quad + 4);
            m0 = m1 = -INFINITY;
            l0 = l1 = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        }
        const int valid = head.x - tok_base;  // live tokens in this warp's 16-token slice
        if (valid > 0) {
            const uint32_t kbase = smem_u32(st);
            const uint32_t vbase = kbase + kTileBytes;
            if (valid < 16) {
                // rows past the context end may hold anything, NaN too: 0 * garbage must not reach the accumulators
                for (int idx = lane; idx < (16 - valid) * 8; idx += 32)
                    *reinterpret_cast<uint4*>(st + kTileBytes + (tok_base + valid + (idx >> 3)) * 128 + (idx & 7) * 16) = make_uint4(0, 0, 0, 0);
                fence_proxy_async_smem();  // order these generic writes before the stage's next TMA refill
                __syncwarp();
            }
            // ---- S^T = K Q^T for 16 tokens, in two accumulators (half the chain) ----
            float sa[4] = {0.f, 0.f, 0.f, 0.f}, sb[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < 8; c += 2) {  // 16-byte chunks of the rows
                uint32_t a[4];
                ldsm_x4(kbase + row_k + (((c + (mi >> 1)) ^ r8) << 4), a);
                mma_add(sa, lo_half2(a[0]), lo_half2(a[1]), hi_half2(a[0]), hi_half2(a[1]), qb[c][0], qb[c][1]);
                mma_add(sb, lo_half2(a[2]), lo_half2(a[3]), hi_half2(a[2]), hi_half2(a[3]), qb[c + 1][0], qb[c + 1][1]);
            }
            // ---- online softmax (log2 domain), against a maximum that may be stale by up to 2^kStale ----
            const float f0 = qf0 * scale.x, f1 = qf1 * scale.x;
            const float s00 = sa[0] + sb[0], s01 = sa[1] + sb[1], s10 = sa[2] + sb[2], s11 = sa[3] + sb[3];
            const bool in0 = grp < valid, in1 = grp + 8 < valid;
            float x00 = in0 ? fmaf(s00, f0, -m0) : -INFINITY, x01 = in0 ? fmaf(s01, f1, -m1) : -INFINITY;
            float x10 = in1 ? fmaf(s10, f0, -m0) : -INFINITY, x11 = in1 ? fmaf(s11, f1, -m1) : -INFINITY;
            if (__any_sync(0xffffffffu, fmaxf(fmaxf(x00, x01), fmaxf(x10, x11)) > kStale + kBias)) {
                float r0 = fmaxf(in0 ? s00 * f0 : -INFINITY, in1 ? s10 * f0 : -INFINITY);
                float r1 = fmaxf(in0 ? s01 * f1 : -INFINITY, in1 ? s11 * f1 : -INFINITY);
#pragma unroll
                for (int step = 4; step < 32; step <<= 1) {
                    r0 = fmaxf(r0, __shfl_xor_sync(0xffffffffu, r0, step));
                    r1 = fmaxf(r1, __shfl_xor_sync(0xffffffffu, r1, step));
                }
                r0 = fmaxf(m0, r0 - kBias), r1 = fmaxf(m1, r1 - kBias);
                const float d0 = fast_exp2(m0 - r0), d1 = fast_exp2(m1 - r1);
                m0 = r0, m1 = r1;
                l0 *= d0, l1 *= d1;
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j][0] *= d0, o[j][1] *= d1, o[j][2] *= d0, o[j][3] *= d1;
                x00 = in0 ? fmaf(s00, f0, -m0) : -INFINITY, x01 = in0 ? fmaf(s01, f1, -m1) : -INFINITY;
                x10 = in1 ? fmaf(s10, f0, -m0) : -INFINITY, x11 = in1 ? fmaf(s11, f1, -m1) : -INFINITY;
            }
            // A head whose probabilities are all small here: relative to its largest of the tile, u.
            float w0 = scale.y, w1 = scale.y;  // of the lane's two heads: what the products with V are multiplied by
            const uint32_t same = 0x11111111u << quad;  // lanes with the same two heads
            const uint32_t fair0 = __ballot_sync(0xffffffffu, fmaxf(x00, x10) > kLow);
            const uint32_t fair1 = __ballot_sync(0xffffffffu, fmaxf(x01, x11) > kLow);
            float g0 = 1.f, g1 = 1.f;
            if (__any_sync(0xffffffffu, (fair0 & same) == 0 || (fair1 & same) == 0)) {
                float u0 = fmaxf(x00, x10), u1 = fmaxf(x01, x11);
#pragma unroll
                for (int step = 4; step < 32; step <<= 1) {
                    u0 = fmaxf(u0, __shfl_xor_sync(0xffffffffu, u0, step));
                    u1 = fmaxf(u1, __shfl_xor_sync(0xffffffffu, u1, step));
                }
                u0 = u0 <= kLow && u0 > -INFINITY ? u0 - kBias : 0.f, u1 = u1 <= kLow && u1 > -INFINITY ? u1 - kBias : 0.f;
                x00 -= u0, x01 -= u1, x10 -= u0, x11 -= u1;
                g0 = fast_exp2(u0), g1 = fast_exp2(u1);
                w0 *= g0, w1 *= g1;
            }
            x00 = fast_exp2(x00), x01 = fast_exp2(x01), x10 = fast_exp2(x10), x11 = fast_exp2(x11);
            l0 = fmaf(x00 + x10, g0, l0);
            l1 = fmaf(x01 + x11, g1, l1);
            // P^T as the B operand: tokens along k, head grp as the column
            const uint32_t p0 = transpose_8x8(pack_half(x00, x01)), p1 = transpose_8x8(pack_half(x10, x11));
            // ---- O^T += vs V^T P^T: 8 row tiles of 16 dims, tokens of a head by the tile's V scale ----
#pragma unroll
            for (int c = 0; c < 8; c += 2) {
                uint32_t a[4];
                ldsm_x4_t(vbase + row_k + (((c + (mi >> 1)) ^ r8) << 4), a);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t t0 = __byte_perm(a[2 * i], 0, 0x3120), t1 = __byte_perm(a[2 * i + 1], 0, 0x3120);
                    float t[4];
                    mma_new(t, lo_half2(t0), hi_half2(t0), lo_half2(t1), hi_half2(t1), p0, p1);
                    o[c + i][0] = fmaf(t[0], w0, o[c + i][0]), o[c + i][1] = fmaf(t[1], w1, o[c + i][1]);
                    o[c + i][2] = fmaf(t[2], w0, o[c + i][2]), o[c + i][3] = fmaf(t[3], w1, o[c + i][3]);
                }
            }
        }
        TileMeta tm;
        if (flags & kLast) tm = sm_meta[stage];
        __syncwarp();
        if (lane == 0) mbar_arrive(empty_bar + stage);
        if (!(flags & kLast)) continue;

        // ---- merge the four warps' (m, l, O) and emit the item ----
        float* sm_m = sm_ml + (item & 1u) * (2 * kConsumerWarps * kMaxG);
        float* sm_l = sm_m + kConsumerWarps * kMaxG;
        ++item;
#pragma unroll
        for (int step = 4; step < 32; step <<= 1) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, step);
            l1 += __shfl_xor_sync(0xffffffffu, l1, step);
        }
        if (grp == 0) {
            *reinterpret_cast<float2*>(sm_m + warp * kMaxG + 2 * quad) = make_float2(m0, m1);
            *reinterpret_cast<float2*>(sm_l + warp * kMaxG + 2 * quad) = make_float2(l0, l1);
        }
        named_barrier_sync(1, kConsumerWarps * 32);
        {
            // fixed order (bitwise reproducible): warps 0,1 store, warps 2,3 add, readers sum the two
            float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
            for (int w = 0; w < kConsumerWarps; ++w) {
                const float2 v = *reinterpret_cast<const float2*>(sm_m + w * kMaxG + 2 * quad);
                t0 = fmaxf(t0, v.x), t1 = fmaxf(t1, v.y);
            }
            const float f0 = (m0 == -INFINITY) ? 0.f : fast_exp2(m0 - t0), f1 = (m1 == -INFINITY) ? 0.f : fast_exp2(m1 - t1);
            float* d0 = Os + (warp & 1) * (kMaxG * kOsStride) + 2 * quad * kOsStride + 2 * grp;
            float* d1 = d0 + kOsStride;
            if (warp < 2) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    *reinterpret_cast<float2*>(d0 + 16 * j) = make_float2(o[j][0] * f0, o[j][2] * f0);
                    *reinterpret_cast<float2*>(d1 + 16 * j) = make_float2(o[j][1] * f1, o[j][3] * f1);
                }
            }
            named_barrier_sync(1, kConsumerWarps * 32);
            if (warp >= 2) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float2 a = *reinterpret_cast<float2*>(d0 + 16 * j), b = *reinterpret_cast<float2*>(d1 + 16 * j);
                    a.x += o[j][0] * f0, a.y += o[j][2] * f0, b.x += o[j][1] * f1, b.y += o[j][3] * f1;
                    *reinterpret_cast<float2*>(d0 + 16 * j) = a;
                    *reinterpret_cast<float2*>(d1 + 16 * j) = b;
                }
            }
        }
        named_barrier_sync(1, kConsumerWarps * 32);
        // thread t finishes row t / 16, dims 8 (t % 16) .. + 7
        const int r = ctid >> 4, c8 = (ctid & 15) * 8;
        if (r < p.G) {
            float mt = -INFINITY;
#pragma unroll
            for (int w = 0; w < kConsumerWarps; ++w) mt = fmaxf(mt, sm_m[w * kMaxG + r]);
            float lt = 0.f;
#pragma unroll
            for (int w = 0; w < kConsumerWarps; ++w) {
                const float mw = sm_m[w * kMaxG + r];
                if (mw != -INFINITY) lt += sm_l[w * kMaxG + r] * fast_exp2(mw - mt);
            }
            const float* s0 = Os + r * kOsStride + c8;
            const float* s1 = s0 + kMaxG * kOsStride;
            const float4 x0 = *reinterpret_cast<const float4*>(s0), x1 = *reinterpret_cast<const float4*>(s0 + 4);
            const float4 y0 = *reinterpret_cast<const float4*>(s1), y1 = *reinterpret_cast<const float4*>(s1 + 4);
            float4 a = make_float4(x0.x + y0.x, x0.y + y0.y, x0.z + y0.z, x0.w + y0.w);
            float4 b = make_float4(x1.x + y1.x, x1.y + y1.y, x1.z + y1.z, x1.w + y1.w);
            if (tm.flags & kWhole) {
                const float inv = 1.f / lt;  // at least 2^(kBias - kStale) / 2: the row's maximum has been added
                uint4 w;
                w.x = pack_bf16(a.x * inv, a.y * inv);
                w.y = pack_bf16(a.z * inv, a.w * inv);
                w.z = pack_bf16(b.x * inv, b.y * inv);
                w.w = pack_bf16(b.z * inv, b.w * inv);
                *reinterpret_cast<uint4*>(p.out + ((size_t)tm.b * p.H + (size_t)kvh * p.G + r) * kD + c8) = w;
            } else {
                float* part = p.partials + (size_t)tm.part * partial_floats(p.G);
                *reinterpret_cast<float4*>(part + r * kD + c8) = a;
                *reinterpret_cast<float4*>(part + r * kD + c8 + 4) = b;
                if (c8 == 0) {
                    part[p.G * kD + r] = mt == -INFINITY ? 0.f : mt;  // only where all scores are NaN, and then o is: not to be left out
                    part[p.G * kD + kMaxG + r] = lt;
                }
            }
        }
        if (!(tm.flags & kWhole)) {
            if (!waited) griddep_wait();
            waited = true;
            // publish the partial, then take a ticket for this (sequence, kv head): the last one combines, nobody waits
            named_barrier_sync(1, kConsumerWarps * 32);
            if (ctid == 0) sm_i[7] = (int)atomic_add_acq_rel(p.tickets + (size_t)tm.b * p.KVH + kvh, 1u);
            named_barrier_sync(1, kConsumerWarps * 32);
            if (sm_i[7] == tm.gl - tm.gf) merge_sequence(p, tm.b, kvh, tm.gf, tm.gl, ctid);
        }
    }
}

// In front of the kernel above: clears the tickets and, in a decode step of up to kScanStep sequences, stores the step's rows
// (blocks [0, store_blocks): a token and kv head each).
template <typename SrcT>
__global__ void __launch_bounds__(q8::kStoreThreads)
decode_q8_prepare_kernel(unsigned int* __restrict__ tickets, int num_tickets, int store_blocks, const q8::Store s) {
    __shared__ q8::StoreShared sh;
    griddep_wait();  // the kernel in front may still be reading these tickets or the cache rows written below
    griddep_launch_dependents();
    if ((int)blockIdx.x < store_blocks) {
        q8::store_token<SrcT>(sh, s, blockIdx.x / s.KVH, blockIdx.x % s.KVH);
    } else {
        const int i = ((int)blockIdx.x - store_blocks) * q8::kStoreThreads + threadIdx.x;
        if (i < num_tickets) tickets[i] = 0u;
    }
}

static int grid() { return kCtas * sm_count(); }

static int ensure_smem_attr() {
    static std::mutex mu;
    static bool done[64];
    int dev = 0;
    NVLLM_CUDA_OK(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lock(mu);
    if (dev >= 0 && dev < 64 && !done[dev]) {
        NVLLM_CUDA_OK(cudaFuncSetAttribute(paged_decode_q8_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
        done[dev] = true;
    }
    return NVLLM_B200_OK;
}

static size_t workspace_bytes_for(int B, int H, int KVH, bool step) {
    return ticket_bytes(B, KVH) + partial_bytes(grid(), H / KVH) + (step && B > q8::kScanStep ? q8::store_workspace_bytes(B) : 0) + 256;
}

// `step`: the store of a decode step (T = B), or null.
static int run(const char* who, const DecodeArgs& a, const float* k_scale, const float* v_scale, const q8::Store* step, int src_dtype,
               void* workspace, size_t workspace_bytes) {
    int rc = check_decode_args(who, a);
    if (rc) return rc;
    if (step && (rc = q8::check_store(who, *step, a.D, src_dtype))) return rc;
    if (a.B == 0) return NVLLM_B200_OK;
    if ((rc = check_decode_pointers(who, a))) return rc;
    if (!k_scale || !v_scale) return fail(NVLLM_B200_EINVAL, "%s: null pointer", who);
    if (((uintptr_t)k_scale | (uintptr_t)v_scale) & 3) return fail(NVLLM_B200_EINVAL, "%s: scales must be 4-byte aligned", who);
    const size_t need = workspace_bytes_for(a.B, a.H, a.KVH, step != nullptr);
    if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255))
        return fail(NVLLM_B200_EWORKSPACE, "%s: workspace of %zu bytes (256-byte aligned) required, got %zu", who, need,
                    workspace ? workspace_bytes : (size_t)0);
    if ((rc = ensure_smem_attr())) return rc;
    CUtensorMap tm_k, tm_v;
    const int64_t num_slots = (int64_t)a.NB * a.block_size;
    if ((rc = cached_cache_map(&tm_k, a.k_cache, num_slots, a.KVH, true))) return rc;
    if ((rc = cached_cache_map(&tm_v, a.v_cache, num_slots, a.KVH, true))) return rc;

    uint8_t* const ws = static_cast<uint8_t*>(workspace);
    Params8 p;
    p.q = (const __nv_bfloat16*)a.q;
    p.block_tables = a.block_tables;
    p.context_lens = a.context_lens;
    p.slot_mapping = step ? step->slots : nullptr;
    p.q_in_flight = 0;
    p.out = (__nv_bfloat16*)a.out;
    p.tickets = (unsigned int*)ws;
    p.partials = (float*)(ws + ticket_bytes(a.B, a.KVH));
    p.B = a.B;
    p.H = a.H;
    p.KVH = a.KVH;
    p.G = a.H / a.KVH;
    p.NB = a.NB;
    p.block_size = a.block_size;
    p.MB = a.MB;
    p.num_groups = grid() / a.KVH;
    p.item_cost = kItemCost;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.k_scale = k_scale;
    p.v_scale = v_scale;

    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.stream = reinterpret_cast<cudaStream_t>(a.stream);
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;

    const int num_tickets = a.B * a.KVH;
    const int clear_blocks = (num_tickets + q8::kStoreThreads - 1) / q8::kStoreThreads;
    const bool inside = step && a.B <= q8::kScanStep;
    if (step && !inside &&
        (rc = q8::launch_store(who, *step, src_dtype, ws + ticket_bytes(a.B, a.KVH) + partial_bytes(grid(), p.G),
                               q8::store_workspace_bytes(a.B), cfg.stream)))
        return rc;
    const int store_blocks = inside ? num_tickets : 0;
    cfg.gridDim = dim3((unsigned)(store_blocks + clear_blocks));
    cfg.blockDim = dim3(q8::kStoreThreads);
    NVLLM_CUDA_OK(cudaLaunchKernelEx(
        &cfg, src_dtype == NVLLM_B200_DTYPE_F32 ? decode_q8_prepare_kernel<float> : decode_q8_prepare_kernel<__nv_bfloat16>, p.tickets,
        num_tickets, store_blocks, inside ? *step : q8::Store{}));
    cfg.gridDim = dim3((unsigned)(p.num_groups * a.KVH));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmemBytes;
    NVLLM_CUDA_OK(cudaLaunchKernelEx(&cfg, paged_decode_q8_kernel, tm_k, tm_v, p));
    return NVLLM_B200_OK;
}

}  // namespace decode_q8

int read_decode_q8_flags(int* out) {
    NVLLM_CUDA_OK(cudaMemcpyFromSymbol(out, decode_q8::g_error_flag, sizeof(int)));
    return NVLLM_B200_OK;
}
int clear_decode_q8_flags() {
    const int zero = 0;
    NVLLM_CUDA_OK(cudaMemcpyToSymbol(decode_q8::g_error_flag, &zero, sizeof(int)));
    return NVLLM_B200_OK;
}
}  // namespace nvllm

extern "C" size_t nvllm_b200_paged_decode_q8_workspace_bytes(int B, int H, int KVH) {
    if (B < 0 || H <= 0 || KVH <= 0 || H % KVH != 0) return 256;
    return nvllm::decode_q8::workspace_bytes_for(B, H, KVH, true);
}

extern "C" int nvllm_b200_paged_decode_q8(const void* q, const void* k_cache, const void* v_cache, const float* k_scale,
                                          const float* v_scale, const int32_t* block_tables, const int32_t* context_lens, void* out,
                                          void* workspace, size_t workspace_bytes, int B, int H, int KVH, int D, int NB,
                                          int block_size, int MB, float scale, void* stream) {
    const nvllm::decode::DecodeArgs a = {q, k_cache, v_cache, block_tables, context_lens, out, B, H, KVH, D, NB, block_size, MB, scale,
                                         stream};
    return nvllm::decode_q8::run("paged_decode_q8", a, k_scale, v_scale, nullptr, NVLLM_B200_DTYPE_BF16, workspace, workspace_bytes);
}

extern "C" int nvllm_b200_decode_step_q8(const void* q, const void* k, const void* v, void* k_cache, void* v_cache, float* k_scale,
                                         float* v_scale, const int32_t* slot_mapping, const int32_t* block_tables,
                                         const int32_t* context_lens, void* out, void* workspace, size_t workspace_bytes, int B, int H,
                                         int KVH, int D, int NB, int block_size, int MB, float scale, int src_dtype, void* stream) {
    const nvllm::decode::DecodeArgs a = {q, k_cache, v_cache, block_tables, context_lens, out, B, H, KVH, D, NB, block_size, MB, scale,
                                         stream};
    const nvllm::q8::Store s = {k, v, (uint8_t*)k_cache, (uint8_t*)v_cache, k_scale, v_scale, slot_mapping, B, KVH,
                                (int64_t)NB * block_size};
    return nvllm::decode_q8::run("decode_step_q8", a, k_scale, v_scale, &s, src_dtype, workspace, workspace_bytes);
}
