// paged_prefill_q8: causal attention of new tokens over their whole sequences in the 8-bit paged cache, on the sm_100a tensor
// cores.
//
// Work items, tiles, runs and the softmax warps are those of the bf16 kernel (varlen_prefill.cu, and see there); what differs is
// how bytes become operands.  Converting a whole K/V tile to bf16 in the SM would double what goes through its shared memory,
// which the two products fill to nine tenths already, so as little as possible is converted:
//
//  * Q.K^T takes K as it is, e4m3 from TMA (tcgen05.mma kind::f8f6f4, K = 32 per instruction), and Q as the sum of two e4m3 tiles.
//    bf16 has eight significant bits, e4m3 four: with a row divided by the power of two that brings its largest magnitude to
//    224 .. 448, hi = e4m3(q) and lo = e4m3(q - hi) give every q from 1/4 on exactly (2^-9.8 of the largest or less) and a smaller
//    one to within half of e4m3's least step, 2^-10 (2^-17.8 of the largest).  Twice as many products at twice the rate: the time of
//    the bf16 product, with no conversion of K at all.
//  * The row's power of two and the K scale of each half of a tile (a scale has 64 slots) go into the factor that the softmax
//    multiplies its scores by anyway.
//  * O += P.V runs in fp16 (P would lose its small probabilities in e4m3): e4m3 -> fp16 is exact and one instruction for two
//    values.  A warpgroup of its own fetches V bytes into its registers a tile ahead, writes fp16 tiles (rows behind the
//    sequence's end as zeros) and splits Q between two items.  The V scale goes into the exponent of the probabilities, relative
//    to the unit that O is in: the first tile's scale, moved -- O rescaled, as when the maximum grows -- when a tile's is larger or less
//    than 2^-kUnitRange of it.  The sums of the probabilities take the exponent back, once per half of a tile.
//
// Softmax steps are of 64 keys, with two score buffers per Q tile; a step's P lies over its own scores.
//
// What bounds it, at 2048 tokens x 32 heads behind 16384 keys (640 us; 585 GFLOP, 352 us at the measured bf16 rate; the bf16 kernel
// takes 520, and 256 items on 148 SMs cost either an eighth): the MMAs and the chain from a step's scores to its P.V.  A
// 128 x 64 x 32 byte product reads 6 KB of shared memory, 48 cycles for 32 of arithmetic.  Left out one by one (wrong results, to see
// what counts): the lower part of Q 575 us, three quarters of P.V 555, both and the rest of Q.K^T 520; the exponentials 641 and
// without all of the products 408; the conversion 636; the V loads 627.
// Measured instead, each against the form of its time: V bytes staged by TMA and written as bf16 668 (12 sequences of 17..700 tokens
// behind 500..5000: 303; as it is now 240 to 283, by box and clock); steps of 128 keys and one score buffer 638 (276) when steps of 64
// took 649 (262), with a commit per P.V and K slots given back by the issuers; the next step's scores taken into registers before this
// one's exponentials 767 (324); sixteen softmax warps, two threads a row 707 (291); a share of the exponentials as polynomials 686 (an
// eighth) .. 744 (a quarter); probabilities against the maximum of the steps before while this one's is found, taken again where it grew
// 657 (267); V converted by integer operations instead of cvt 654.
//
// Per CTA (16 warps = 4 warpgroups; registers 96 | 160 | 160 | 96 of the launch's 128 each):
//   warp 0       TMA producer: K bytes, four slots; slot and scales of a tile, looked up a tile ahead, into a ring
//   warps 1, 2   MMA issuers of Q tiles A and B
//   warp 3       item records
//   warps 4-11   softmax, as in the bf16 kernel
//   warps 12-15  Q: bf16 -> two e4m3 tiles and the rows' factors.  V: e4m3 -> fp16, three slots
// Every mbarrier wait is bounded; on timeout the CTA raises a device error flag, lets its copies land and releases its
// tensor memory before it exits.
#include "q8.cuh"
#include "varlen_prefill.cuh"

#include <mutex>
#include <type_traits>

namespace nvllm {
namespace prefill_q8 {

using namespace prefill;

__device__ int g_error_flag = 0;  // bit 2 (4): a pipeline wait timed out, or no room in tensor memory

constexpr int kThreads = 512;
constexpr int kByteTile = 128 * 128;     // 128 rows of 128 bytes, 128B-swizzled
constexpr int kSlots = 4;                // of K bytes
constexpr int kVSlots = 3;               // of V in fp16
constexpr int kStep = 64;                // keys of a softmax step: half a K/V tile, a block of scales
constexpr int kInfos = 8;                // ring of what a tile is: nobody is as far ahead of a reader (see the producer)
constexpr int kK = 2 * kTileBytes;       // offsets: Q (A: hi, lo; B: hi, lo), K, V
constexpr int kV = kK + kSlots * kByteTile;
constexpr int kSmemTiles = kV + kVSlots * kTileBytes;  // 224 KB
constexpr int kItemRing = 2;
constexpr int kItemReaders = 3 + 8 + 4;  // TMA producer, two MMA issuers, eight softmax warps, four converting warps
constexpr int kRegsControl = 96, kRegsSoftmax = 160, kRegsConvert = 96;
static_assert(kRegsControl + 2 * kRegsSoftmax + kRegsConvert == 4 * 128, "what setmaxnreg asks for is what the launch has");

constexpr float kTiny = 1.17549435e-38f;
// log2 units: a row's largest probability is 2^kBias, or up to 2^(kBias + kRescaleThreshold) until the maximum moves (fp16: 2^16);
// one of 2^-21 of it is still a normal fp16 number.
constexpr float kBias = 7.f;
constexpr float kUnitRange = 8.f;
// A V scale below 2^-kScaleRange of the largest one before it in the run counts as that (a block of zeros has the least scale there
// is): its values are nothing beside what p * v may be off by, and O, in units of it, would leave fp32.
constexpr float kScaleRange = 64.f;

struct Source {
    const __nv_bfloat16* q;
    const uint8_t* v;                // [NB * block_size, KVH, 128] e4m3
    const float *k_scale, *v_scale;  // [NB * block_size / 64, KVH]
    int NB, KVH;
};
struct Whole : Params {
    Source in;
};
struct Split : SplitParams {
    Source in;
};
struct Tail : TailParams {
    Source in;
};
struct Work : Item {
    int part;  // of a run: the place of its results
};

struct Shared {
    float q_factor[2][2][kTileQ];  // [item parity][Q tile][row]: what a row was divided by
    float4 scale[kInfos];          // of a tile: K scales of the first and second half, log2 of the V scales
    int token[kInfos];             // its first slot
    Work items[kItemRing];         // the items of this CTA, written ahead by warp 3
    uint64_t item_full[kItemRing], item_empty[kItemRing];
    uint64_t q_full, q_empty;
    uint64_t factor_full[2];       // of the item parity: the softmax may come to an item when Q of the next one is there already
    uint64_t k_full[kSlots], k_empty[kSlots];
    uint64_t v_full[kVSlots], v_empty[kVSlots];
    uint64_t info_full[kInfos];
    uint64_t s_full[2][2], p_full[2][2];  // [Q tile][step parity]
    uint64_t o_done[2][2];               // [Q tile][an item's last step but one (or only one), its last one]
    uint64_t o_empty[2];
    uint32_t odd_values[2];              // of the item parity: 1 + the item of which V held NaN behind a row's limit (see add_nan)
    uint32_t tmem_base;
    volatile int abort_flag;
};
constexpr int kSmemBytes = kSmemTiles + sizeof(Shared);
static_assert(kSmemBytes <= 227 * 1024, "shared memory of a CTA");

__device__ __forceinline__ bool wait_or_abort(Shared* sh, uint64_t* bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    if (sh->abort_flag) return false;
    if (mbar_wait(bar, parity)) return true;
    sh->abort_flag = 1;
    atomicOr(&g_error_flag, 4);
    return false;
}

__device__ __forceinline__ bool next_item(Shared* sh, uint32_t k, Work& it) {
    const uint32_t slot = k % kItemRing;
    if (!wait_or_abort(sh, &sh->item_full[slot], (k / kItemRing) & 1u)) return false;
    it = sh->items[slot];
    return it.n_kv >= 0;
}

// 16 bytes global -> shared, or zeros.
__device__ __forceinline__ void copy_16(uint32_t to, const void* from, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// D[tmem] (+)= A[smem] * B[smem], both e4m3, K = 32
__device__ __forceinline__ void mma_bytes(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(acc)
        : "memory");
}
constexpr uint32_t kIdescBytes = (1u << 4) | ((128u >> 4) << 24);  // e4m3 x e4m3 -> fp32, M = 128, both K-major
constexpr uint32_t kIdescHalf = (1u << 4) | (1u << 16) | ((128u >> 3) << 17) | ((128u >> 4) << 24);  // fp16, V MN-major
constexpr uint32_t idesc_bytes(uint32_t keys) { return kIdescBytes | ((keys >> 3) << 17); }

// Steps of Q tile x in an item, and how many keys its last one has (of the item's last row).
__device__ __forceinline__ int keys_of(const Params& p, const Item& it, int x, int n_x) { return min(visible_keys(p, it, x), n_x * kTileKV); }
__device__ __forceinline__ int steps_of(int keys) { return (keys + kStep - 1) / kStep; }

// One step of a row: 64 scores -> running maximum, perhaps O rescaled, fp16 P over the first half of the scores' columns.
// DIAG: key c of this step is visible iff c <= lim (which may be negative, or 63 and more), and the limits of the warp's rows
// lie in warp_lo .. warp_hi; keys behind every limit may hold anything.  alive: the warp's rows in front of the sequence's
// end; the others have no vote on when to rescale, or the live rows' bits would depend on them.
// c0: factor of the scores (positive); the maxima are of the products, in log2 units.  v0: log2 of the V scale; unit: of the one
// that O is in units of.  o_bar: the P.V in front of this step's.
template <bool DIAG>
__device__ __forceinline__ bool softmax_step(Shared* sh, const uint32_t t_s, const uint32_t t_o, const int lim, const int warp_lo,
                                             const int warp_hi, const bool first, uint64_t* o_bar, const uint32_t o_parity, const float c0,
                                             const float v0, const uint32_t alive, float& m_run, float& m_used, float& unit, float& l,
                                             uint64_t* p_bar) {
    uint32_t v[2][32];
    tmem_ld32(t_s, v[0]);
    tmem_ld32(t_s + 32, v[1]);
    tmem_wait_ld();
    float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        if (DIAG) {
            if (32 * c > warp_hi) continue;  // nothing of this chunk is visible to any row of the warp
            if (32 * c + 31 > warp_lo) {     // mask in place so that the second pass needs no select
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (c * 32 + i > lim) v[c][i] = 0xFF800000u;
            }
        }
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
            mx0 = max3(mx0, __uint_as_float(v[c][i]), __uint_as_float(v[c][i + 1]));
            mx1 = max3(mx1, __uint_as_float(v[c][i + 2]), __uint_as_float(v[c][i + 3]));
            mx2 = max3(mx2, __uint_as_float(v[c][i + 4]), __uint_as_float(v[c][i + 5]));
            mx3 = max3(mx3, __uint_as_float(v[c][i + 6]), __uint_as_float(v[c][i + 7]));
        }
    }
    m_run = fmaxf(m_run, fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)) * c0);
    if (first) {
        m_used = m_run;  // finite for live rows: key 0 of the sequence is visible to every row and sits in the first step
        unit = v0;
    } else {
        const bool grow = m_run - m_used > kRescaleThreshold;
        const bool other_unit = v0 > unit || v0 < unit - kUnitRange;  // for all rows alike
        if ((__ballot_sync(0xffffffffu, grow) & alive) || other_unit) {
            // O holds sums relative to m_used in the old unit: bring it to m_run and the new one before this step's P.V is added.
            if (!wait_or_abort(sh, o_bar, o_parity)) return false;
            tc_fence_after();
            const float f = fast_exp2(m_used - m_run);
            const float fo = other_unit ? fast_exp2(m_used - m_run + (unit - v0)) : f;
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
                uint32_t ov[16];
                tmem_ld16(t_o + c * 16, ov);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * fo);
                tmem_st16(t_o + c * 16, ov);
            }
            tmem_wait_st();
            l *= f;
            m_used = m_run;
            if (other_unit) unit = v0;
        }
    }
    // p = 2^(s*c0 - m + the V scale's exponent) as fp16 pairs, written over the S columns (all of them are in registers by
    // now): chunk c (scores 32c .. 32c + 31) becomes packed columns 16c .. 16c + 15.
    const float n = kBias - m_used + (v0 - unit);
    const float back = fast_exp2(unit - v0);
    const uint64_t scale2 = pack2(c0, c0), neg2 = pack2(n, n);
    uint64_t acc_a = pack2(0.f, 0.f), acc_b = pack2(0.f, 0.f);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        if (DIAG && 32 * c > warp_hi) {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[c][i] = 0u;
        } else {
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                float x0, x1, x2, x3;
                unpack2(fma2(pack2(__uint_as_float(v[c][2 * i]), __uint_as_float(v[c][2 * i + 1])), scale2, neg2), x0, x1);
                unpack2(fma2(pack2(__uint_as_float(v[c][2 * i + 2]), __uint_as_float(v[c][2 * i + 3])), scale2, neg2), x2, x3);
                const float e0 = fast_exp2(x0), e1 = fast_exp2(x1);  // 2^-inf = 0 for masked keys
                const float e2 = fast_exp2(x2), e3 = fast_exp2(x3);
                acc_a = add2(acc_a, pack2(e0, e1));
                acc_b = add2(acc_b, pack2(e2, e3));
                v[c][i] = pack_half(e0, e1);  // in place: word i <= 2i has been consumed
                v[c][i + 1] = pack_half(e2, e3);
            }
        }
        tmem_st16(t_s + c * 16, v[c]);
    }
    tmem_wait_st();
    tc_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(p_bar);
    float s0, s1, s2, s3;
    unpack2(acc_a, s0, s1);
    unpack2(acc_b, s2, s3);
    l = fmaf((s0 + s1) + (s2 + s3), back, l);
    return true;
}

// K/V tiles in front of the first one of which the item's first row does not see every key.
__device__ __forceinline__ int plain_tiles(const Item& it) { return (it.prefix + it.q0 + 1) / kTileKV; }

// Whether a byte of w is NaN: its bit 7.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return (w & 0x7f7f7f7fu) + 0x01010101u; }

// P is 0 for a key behind a row's limit, but 0 * NaN is NaN: a NaN there would reach rows that do not see it.  In the tiles that hold
// such keys V has 0 in its place, and here O gets it back in the rows that do see it: every row reads the bytes again for itself, up to
// its own limit.  Called by a warp of the softmax for its rows, of Q tile x and its token tok each.  Only what is not finite is stored
// as NaN, so this is rare; a call, which costs the others nothing (in the loops that read O it made eight runs of four steps, 25.2 us,
// half a microsecond longer).
__device__ __noinline__ void add_nan(const Params& p, const Source& in, const Work& it, int x, int tok, uint32_t t_o) {
    const int q_pos = it.q0 + x * p.pack.dq, tiles = x == 0 ? it.n_a : it.n_b;
    const int seen = tok < min(p.pack.tokens, it.len - q_pos) ? it.prefix + q_pos + tok + 1 : 0;  // keys of the row
#pragma unroll 1
    for (int c = 0; c < 8; ++c) {  // 16 dims at a time
        uint32_t odd[4] = {0u, 0u, 0u, 0u};
        for (int j = plain_tiles(it); j < tiles; ++j) {
            const int off = (max(it.kv0, 0) + j) * kTileKV;
            const int page = __ldg(p.block_tables + (size_t)it.b * p.MB + min(off / p.block_size, p.MB - 1));
            const int token = min(max(page, 0), in.NB - 1) * p.block_size + off % p.block_size;
            const uint8_t* at = in.v + ((size_t)token * in.KVH + it.kvh) * kD + c * 16;
            const int keys = min(kTileKV, seen - j * kTileKV);
            for (int i = 0; i < keys; ++i, at += (size_t)in.KVH * kD) {
                const uint4 w = __ldg(reinterpret_cast<const uint4*>(at));
                odd[0] |= nan_bytes(w.x), odd[1] |= nan_bytes(w.y), odd[2] |= nan_bytes(w.z), odd[3] |= nan_bytes(w.w);
            }
        }
        __syncwarp();
        uint32_t ov[16];
        tmem_ld16(t_o + c * 16, ov);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) ov[i] = odd[i >> 2] >> (8 * (i & 3) + 7) & 1u ? 0x7fffffffu : ov[i];
        tmem_st16(t_o + c * 16, ov);
    }
    tmem_wait_st();
}

template <class P>
__global__ void __launch_bounds__(kThreads, 1)
paged_prefill_q8_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ P p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    Shared* sh = reinterpret_cast<Shared*>(smem + kSmemTiles);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (smem_u32(smem) & 1023) {  // the swizzled tiles need it; the alignment above asks for it
        if (tid == 0) atomicOr(&g_error_flag, 4);
        griddep_wait();
        return;
    }
    if (tid == 0) {
        for (int s = 0; s < kItemRing; ++s) {
            mbar_init(&sh->item_full[s], 1);
            mbar_init(&sh->item_empty[s], kItemReaders);
        }
        mbar_init(&sh->q_full, 4);    // the converting warps
        mbar_init(&sh->q_empty, 2);   // both MMA issuers
        mbar_init(&sh->factor_full[0], 4);
        mbar_init(&sh->factor_full[1], 4);
        for (int s = 0; s < kSlots; ++s) {
            mbar_init(&sh->k_full[s], 1);
            mbar_init(&sh->k_empty[s], 2);  // from each Q tile: its softmax, or its issuer where it has no step there
        }
        for (int s = 0; s < kVSlots; ++s) {
            mbar_init(&sh->v_full[s], 4);
            mbar_init(&sh->v_empty[s], 2);
        }
        for (int s = 0; s < kInfos; ++s) mbar_init(&sh->info_full[s], 1);
        for (int x = 0; x < 2; ++x) {
            for (int b = 0; b < 2; ++b) {
                mbar_init(&sh->s_full[x][b], 1);
                mbar_init(&sh->p_full[x][b], kTileQ / 32);
                mbar_init(&sh->o_done[x][b], 1);
            }
            mbar_init(&sh->o_empty[x], kTileQ / 32);
        }
        sh->odd_values[0] = sh->odd_values[1] = 0u;
        sh->abort_flag = 0;
        sh->tmem_base = 0xFFFFFFFFu;
        fence_mbar_init();
        prefetch_tensormap(&tm_k);
    }
    __syncthreads();
    if (warp == 1) {
        tmem_alloc(&sh->tmem_base, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh->tmem_base;

    griddep_wait();  // the plan kernel's item list (and the caller's q and cache) must be visible from here on

    if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsControl));
    if (warp == 0) {
        // =============================== TMA producer ===============================
        if (lane == 0) {
            uint32_t t = 0, i = 0;  // tiles, items
            bool ok = true;
            Work it = {};
            int token = 0;
            float4 scale;
            float least = 0.f;  // log2 of the smallest V scale that counts
            // First slot of K/V tile j and its scales: one per 64 slots, of which the second may lie behind the last key.
            auto locate = [&](int j) {
                const int off = (max(it.kv0, 0) + j) * kTileKV;
                const int page = __ldg(p.block_tables + (size_t)it.b * p.MB + min(off / p.block_size, p.MB - 1));
                token = min(max(page, 0), p.in.NB - 1) * p.block_size + off % p.block_size;
                const size_t at = (size_t)(token / q8::kGrain) * p.in.KVH + it.kvh;
                const bool second = it.len_k - j * kTileKV > q8::kGrain;
                scale.x = __ldg(p.in.k_scale + at);
                scale.y = second ? __ldg(p.in.k_scale + at + p.in.KVH) : 1.f;
                scale.z = log2f(fmaxf(__ldg(p.in.v_scale + at), kTiny));
                scale.w = second ? log2f(fmaxf(__ldg(p.in.v_scale + at + p.in.KVH), kTiny)) : scale.z;
                if (j > 0) scale.z = fmaxf(scale.z, least);
                least = j > 0 ? fmaxf(least, scale.z - kScaleRange) : scale.z - kScaleRange;
                scale.w = fmaxf(scale.w, least);
                least = fmaxf(least, scale.w - kScaleRange);
            };
            while (ok && next_item(sh, i, it)) {
                mbar_arrive(&sh->item_empty[i % kItemRing]);
                locate(0);
                for (int j = 0; j < it.n_kv; ++j, ++t) {
                    const int slot = t % kSlots, here = token;
                    const uint32_t empty = ((t / kSlots) & 1u) ^ 1u;
                    const float4 mine = scale;
                    if (j + 1 < it.n_kv) locate(j + 1);
                    if (!(ok = wait_or_abort(sh, &sh->k_empty[slot], empty))) break;
                    // Q.K^T(t - 4) is complete, so P.V(t - 5) has been issued: softmax and conversion have read what there is
                    // about tile t - 5, and the entry of t - 8 is free.
                    sh->scale[t % kInfos] = mine;
                    sh->token[t % kInfos] = here;
                    mbar_arrive(&sh->info_full[t % kInfos]);
                    mbar_expect_tx(&sh->k_full[slot], kByteTile);
                    tma_load_3d(smem + kK + slot * kByteTile, &tm_k, &sh->k_full[slot], 0, it.kvh, here);
                }
                ++i;
            }
            if (sh->abort_flag)  // loads in flight land before the memory is released
                for (uint32_t u = t >= kSlots ? t - kSlots : 0; u < t; ++u)
                    (void)mbar_wait(&sh->k_full[u % kSlots], (u / kSlots) & 1u, polls_of_ms(90));
        }
    } else if (warp == 3) {
        // ============================== item records ================================
        if (lane == 0) {
            const List list = list_of(p);
            Cut cut = {items_of(static_cast<const Params&>(p), list), 1};
            int total = cut.whole;
            if constexpr (!std::is_same<P, Whole>::value) {
                cut = cut_of(p, list);
                total = cut.whole + (total - cut.whole) * cut.splits;
            }
            if (tmem == 0xFFFFFFFFu) total = 0;
            uint32_t k = 0;
            int idx = blockIdx.x;
            while (true) {
                const uint32_t slot = k % kItemRing;
                if (!wait_or_abort(sh, &sh->item_empty[slot], ((k / kItemRing) & 1u) ^ 1u)) break;
                Work it;
                do {
                    if (k > 0 || idx != (int)blockIdx.x) idx = claim_item(p);
                    it.n_kv = -1;
                    if (idx < total) {
                        const int run = idx - cut.whole, c = run < 0 ? 0 : run % cut.splits;
                        static_cast<Item&>(it) = load_item(static_cast<const Params&>(p), list, run < 0 ? idx : cut.whole + run / cut.splits);
                        it.part = run;
                        if (run >= 0) take_run(p, it, c, cut.splits);
                    }
                    if (it.n_kv == 0) idx = total;  // nothing to do there: claim another one
                } while (it.n_kv == 0);
                sh->items[slot] = it;
                mbar_arrive(&sh->item_full[slot]);
                if (it.n_kv < 0) break;
                ++k;
            }
        }
    } else {
        // ============================== MMA issuers ===============================
        // One issuing thread per Q tile.  S has two buffers of a step each: Q.K^T of step h + 2 is issued right behind P.V of step h,
        // whose P it overwrites (a thread's MMAs run in order), so the scores of a step are there before the softmax of the one in
        // front of it is done, and with S(h + 2) there P.V(h) is complete as well: only an item's last two are committed by
        // themselves.  A poll and a commit cost this thread about a hundred cycles each, so a K slot is given back by a softmax
        // warp and a tile is waited for once (2048 tokens x 32 heads behind 16384 keys: 655 -> 640 us).
        // The last step's products leave out the keys behind every row.
        if (lane == 0) {
            const int x = warp - 1;
            const uint32_t s_t = tmem + x * 128, o_t = tmem + 256 + x * 128;
            const uint64_t q_desc = make_desc(smem_u32(smem + x * kTileBytes), 16, 1024);
            const uint64_t k_desc0 = make_desc(smem_u32(smem + kK), 16, 1024), v_desc0 = mnmajor_desc(smem_u32(smem + kV), 0);
            uint32_t kt = 0;    // K/V tiles consumed before this item
            uint32_t g = 0;     // steps of this Q tile before this item (buffers and barrier phases)
            uint32_t used = 0;  // items in which this Q tile was active (o_empty phases)
            uint32_t i = 0;     // items
            bool ok = true;
            auto k_full = [&](uint32_t t) { return wait_or_abort(sh, &sh->k_full[t % kSlots], (t / kSlots) & 1u); };
            auto v_full = [&](uint32_t t) { return wait_or_abort(sh, &sh->v_full[t % kVSlots], (t / kVSlots) & 1u); };
            Work it;
            while (ok && next_item(sh, i, it)) {
                mbar_arrive(&sh->item_empty[i % kItemRing]);
                const int n_x = x == 0 ? it.n_a : it.n_b, keys = keys_of(p, it, x, n_x), steps = n_x > 0 ? steps_of(keys) : 0;
                const int last = (keys - (steps - 1) * kStep + 15) >> 4;  // 16-key parts of the last step that hold any
                if (!(ok = wait_or_abort(sh, &sh->q_full, i & 1u))) break;
                auto qk = [&](int h) -> bool {
                    const uint32_t t = kt + (h >> 1), b = (g + h) & 1u;
                    if ((h & 1) == 0 && !k_full(t)) return false;
                    tc_fence_after();
                    const uint64_t kd = k_desc0 + (t % kSlots) * (uint32_t)(kByteTile >> 4) + (h & 1) * (uint32_t)(kStep * 128 >> 4);
                    const uint32_t idesc = idesc_bytes(h + 1 < steps ? kStep : 16 * last);
#pragma unroll
                    for (int part = 0; part < 2; ++part)  // the two tiles that Q is the sum of
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks)
                            mma_bytes(s_t + b * kStep, q_desc + (uint32_t)((part * kByteTile + ks * 32) >> 4), kd + (uint32_t)((ks * 32) >> 4),
                                      idesc, part + ks > 0);
                    tc_commit(&sh->s_full[x][b]);
                    if (h + 1 == steps) tc_commit(&sh->q_empty);
                    return true;
                };
                if (steps == 0) mbar_arrive(&sh->q_empty);  // this tile never reads the Q buffer of this item
                if (steps > 0) ok = qk(0);
                if (ok && steps > 1) ok = qk(1);
                for (int h = 0; ok && h < steps; ++h) {
                    const uint32_t t = kt + (h >> 1), b = (g + h) & 1u;
                    if ((h & 1) == 0 && !(ok = v_full(t))) break;
                    if (h == 0 && used > 0 && !(ok = wait_or_abort(sh, &sh->o_empty[x], (used - 1) & 1u))) break;
                    if (!(ok = wait_or_abort(sh, &sh->p_full[x][b], ((g + h) >> 1) & 1u))) break;
                    tc_fence_after();
                    const uint64_t vd = v_desc0 + (t % kVSlots) * (uint32_t)(kTileBytes >> 4) + (h & 1) * (uint32_t)(kStep * 128 >> 4);
                    const int parts = h + 1 < steps ? 4 : last;
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks)
                        if (ks < parts)
                            mma_ts(o_t, s_t + b * kStep + ks * 8, vd + (uint32_t)((ks * 16 * 128) >> 4), kIdescHalf, (h > 0 || ks > 0));
                    if (h + 2 == steps || steps == 1) tc_commit(&sh->o_done[x][0]);
                    if (h + 1 == steps) tc_commit(&sh->o_done[x][1]);
                    if ((h & 1) || h + 1 == steps) tc_commit(&sh->v_empty[t % kVSlots]);
                    if (h + 2 < steps) ok = qk(h + 2);
                }
                // tiles that only the other Q tile has steps in
                for (int j = (steps + 1) >> 1; ok && j < it.n_kv; ++j) {
                    const uint32_t t = kt + j;
                    if (!(ok = k_full(t))) break;
                    mbar_arrive(&sh->k_empty[t % kSlots]);
                    if (!(ok = v_full(t))) break;
                    mbar_arrive(&sh->v_empty[t % kVSlots]);
                }
                g += steps;
                used += steps > 0 ? 1 : 0;
                kt += it.n_kv;
                ++i;
            }
        }
    }
    } else if (warp < 12) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        // ============================ softmax warpgroups ============================
        const int x = (warp - 4) >> 2;              // 0: tile A, 1: tile B
        const int quarter = warp & 3;               // tensor-memory lane quarter this warp may touch
        const int row = quarter * 32 + lane;        // row within the Q tile: a token and a head
        const int tok = row / p.pack.heads, tok_head = row - tok * p.pack.heads;
        const int tok_lo = quarter * 32 / p.pack.heads, tok_hi = (quarter * 32 + 31) / p.pack.heads;  // the warp's tokens
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        const uint32_t t_s = tmem + x * 128 + lane_base;
        const uint32_t t_o = tmem + 256 + x * 128 + lane_base;
        uint32_t g = 0;   // steps of this Q tile in the items before this one (buffers and barrier phases)
        uint32_t kt = 0;  // K/V tiles of the items before this one
        uint32_t used = 0;  // of them, those in which this Q tile was active
        bool ok = true;
        Work it;
        for (uint32_t k = 0; ok && next_item(sh, k, it); ++k) {
            const int n_x = x == 0 ? it.n_a : it.n_b;
            const uint32_t kt0 = kt, g0 = g;
            kt += it.n_kv;
            if (n_x == 0) {
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh->item_empty[k % kItemRing]);
                continue;
            }
            const int steps = steps_of(keys_of(p, it, x, n_x));
            g += steps;
            const int q_pos = it.q0 + x * p.pack.dq;      // first token of this Q tile
            const int first_lim = it.prefix + q_pos;      // last key visible to it
            const int live = min(p.pack.tokens, it.len - q_pos);  // tokens of the tile in front of the sequence's end
            float m_run = -INFINITY, m_used = -INFINITY, unit = 0.f, l = 0.f;
            if (!(ok = wait_or_abort(sh, &sh->factor_full[k & 1], (k >> 1) & 1u))) break;
            const float factor = sh->q_factor[k & 1][x][row] * p.scale_log2;
            const uint32_t alive = __ballot_sync(0xffffffffu, tok < live);
            // Steps whose last key the tile's first row may still see need no mask; the others are masked per element.  The two
            // kinds run in two separate loops so that each loop body is straight-line code.
            float4 scale = {};
            auto step = [&](const int h, auto kind) -> bool {
                constexpr bool kDiag = decltype(kind)::value == 1, kDead = decltype(kind)::value == 2;
                const uint32_t t = kt0 + (h >> 1), b = (g0 + h) & 1u, phase = ((g0 + h) >> 1) & 1u;
                if (!kDead && (h & 1) == 0) {  // what the tile is, for its two steps
                    if (!wait_or_abort(sh, &sh->info_full[t % kInfos], (t / kInfos) & 1u)) return false;
                    scale = sh->scale[t % kInfos];
                }
                float c0 = ((h & 1) ? scale.y : scale.x) * factor;
                c0 = c0 < kTiny ? kTiny : c0;  // a normal number: a masked score, -inf, times 0 would be NaN
                const float v0 = (h & 1) ? scale.w : scale.z;
                if (!wait_or_abort(sh, &sh->s_full[x][b], phase)) return false;
                tc_fence_after();
                if (((h & 1) || h + 1 == steps) && quarter == 0 && lane == 0) mbar_arrive(&sh->k_empty[t % kSlots]);
                if constexpr (kDead) {  // nothing but the hand-over: P and O of these rows may hold anything
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh->p_full[x][b]);
                    return true;
                }
                const int lim = first_lim - h * kStep;
                return softmax_step<kDiag>(sh, t_s + b * kStep, t_o, kDiag ? lim + min(tok, live - 1) : 0, kDiag ? lim + min(tok_lo, live - 1) : 0,
                                           kDiag ? lim + min(tok_hi, live - 1) : 0, h == 0, h + 1 < steps ? &sh->s_full[x][b ^ 1] : &sh->o_done[x][0],
                                           h + 1 < steps ? ((g0 + h + 1) >> 1) & 1u : used & 1u, c0,
                                           v0, alive, m_run, m_used, unit, l, &sh->p_full[x][b]);
            };
            const int n_plain = min(steps, (first_lim + 1) / kStep);  // steps h with 64 h + 63 <= first_lim
            int h = 0;
            const bool dead = tok_lo >= live;  // the whole warp lies behind the sequence's last row
            if (dead) {
                for (; ok && h < steps; ++h) ok = step(h, std::integral_constant<int, 2>{});
            } else {
                for (; ok && h < n_plain; ++h) ok = step(h, std::integral_constant<int, 0>{});
                for (; ok && h < steps; ++h) ok = step(h, std::integral_constant<int, 1>{});
            }
            if (!ok) break;
            // ---- epilogue: O / l -> bf16 -> global, then hand O back to the MMA thread ----
            if (!(ok = wait_or_abort(sh, &sh->o_done[x][1], used & 1u))) break;
            tc_fence_after();
            ++used;
            const float in_units = fast_exp2(unit);
            // (Written in front of v_full, which the last P.V has waited for; item k + 2 is not there before the end of this one.)
            if (!dead && sh->odd_values[k & 1] == k + 1) add_nan(p, p.in, sh->items[k % kItemRing], x, tok, t_o);
            if constexpr (!std::is_same<P, Whole>::value) {
                if (it.kv0 >= 0) {  // a run of a split item: its O, maximum and sum as they are
                    float* part = p.partials + ((size_t)it.part * 2 + x) * kPartialFloats;
                    if (!dead) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            uint32_t ov[32];
                            tmem_ld32(t_o + c * 32, ov);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * in_units);
#pragma unroll
                            for (int i = 0; i < 8 && tok < live; ++i)
                                *reinterpret_cast<uint4*>(part + row * kD + c * 32 + i * 4) =
                                    make_uint4(ov[4 * i], ov[4 * i + 1], ov[4 * i + 2], ov[4 * i + 3]);
                        }
                        part[kTileQ * kD + row] = m_used;
                        part[kTileQ * kD + kTileQ + row] = l;
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&sh->o_empty[x]);
                        mbar_arrive(&sh->item_empty[k % kItemRing]);
                    }
                    continue;
                }
            }
            const float inv = in_units / l;
            const int head = it.head + x * p.pack.dh + tok_head;
            __nv_bfloat16* orow = p.out + ((size_t)(it.seq_start + q_pos + tok) * p.H + head) * kD;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if (dead) break;
                uint32_t ov[32];
                tmem_ld32(t_o + c * 32, ov);
                tmem_wait_ld();
                if (tok < live && p.wide) {  // whole sectors: half the store instructions
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t w[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            w[e] = pack_bf16(__uint_as_float(ov[16 * i + 2 * e]) * inv, __uint_as_float(ov[16 * i + 2 * e + 1]) * inv);
                        store_32bytes(orow + c * 32 + i * 16, w);
                    }
                } else if (tok < live) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint4 w;
                        w.x = pack_bf16(__uint_as_float(ov[8 * i + 0]) * inv, __uint_as_float(ov[8 * i + 1]) * inv);
                        w.y = pack_bf16(__uint_as_float(ov[8 * i + 2]) * inv, __uint_as_float(ov[8 * i + 3]) * inv);
                        w.z = pack_bf16(__uint_as_float(ov[8 * i + 4]) * inv, __uint_as_float(ov[8 * i + 5]) * inv);
                        w.w = pack_bf16(__uint_as_float(ov[8 * i + 6]) * inv, __uint_as_float(ov[8 * i + 7]) * inv);
                        *reinterpret_cast<uint4*>(orow + c * 32 + i * 8) = w;
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sh->o_empty[x]);
                mbar_arrive(&sh->item_empty[k % kItemRing]);  // only now: the next claim waits for it
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsConvert));
        // ============================ converting warps =============================
        const int w = warp - 12, r4 = lane >> 3, part = lane & 7;  // four rows of 128 bytes (16 per lane) at a time
        uint32_t t = 0;
        bool ok = true;
        Work it;
        for (uint32_t k = 0; ok && next_item(sh, k, it); ++k) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->item_empty[k % kItemRing]);
            // ---- Q: the item's rows, split in place: the two halves of a thread's 32 bytes go where their upper and lower parts will
            // be.  Sixteen rows at a time over the warps, those behind the sequence's end left out: they hold anything, and so do their
            // scores (five drafted tokens of sequences of 16 / 2 heads: a run waited 5 us for 128 rows by 32 a warp, two for 40) ----
            if (k > 0 && !(ok = wait_or_abort(sh, &sh->q_empty, (k - 1) & 1u))) break;
            const int q_tiles = it.n_b > 0 ? 2 : 1;
            for (int x = 0; x < q_tiles; ++x) {
                const int q_pos = it.q0 + x * p.pack.dq, live = min(p.pack.tokens, it.len - q_pos);
                const int groups = min(8, (live * p.pack.heads + 15) >> 4);  // of 16 rows, that hold live ones
#pragma unroll 4
                for (int s = 0; s < groups; ++s) {
                    const int row = s * 16 + w * 4 + r4, tok = row / p.pack.heads;
                    const int head = it.head + x * p.pack.dh + row - tok * p.pack.heads;
                    const bool in = tok < live;
                    const uint4* from = reinterpret_cast<const uint4*>(p.in.q) +
                                        (in ? ((size_t)(it.seq_start + q_pos + tok) * p.H + head) * (kD / 8) + part * 2 : 0);
                    const uint32_t to = smem_u32(smem) + x * kTileBytes + row * 128 + ((part ^ (row & 7)) << 4);
                    copy_16(to, from, in);
                    copy_16(to + kByteTile, from + 1, in);
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            for (int x = 0; x < q_tiles; ++x) {
                const int live = min(p.pack.tokens, it.len - (it.q0 + x * p.pack.dq));
                const int groups = min(8, (live * p.pack.heads + 15) >> 4);
#pragma unroll 1
                for (int s = 0; s < groups; ++s) {
                    const int row = s * 16 + w * 4 + r4;
                    uint4* const at = reinterpret_cast<uint4*>(smem + x * kTileBytes + row * 128 + ((part ^ (row & 7)) << 4));
                    uint4* const at_lo = at + kByteTile / 16;
                    const uint4 a = *at, b = *at_lo;
                    const uint32_t in[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
                    uint32_t top = 0;
#pragma unroll
                    for (int e = 0; e < 8; ++e) top = __vmaxu2(top, in[e] & 0x7fff7fffu);
                    top = max(top & 0xffffu, top >> 16);
#pragma unroll
                    for (int step = 1; step < 8; step <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, step));
                    const q8::RowPower power(top);
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) q8::split_row(in[2 * c], in[2 * c + 1], power.down, hi[c], lo[c]);
                    *at = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    *at_lo = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    if (part == 0) sh->q_factor[k & 1][x][row] = power.up;
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sh->factor_full[k & 1]);
                mbar_arrive(&sh->q_full);
            }
            // ---- V, tile by tile: the bytes of the next one are on their way while this one is written ----
            uint4 in[8];
            auto fetch = [&](int j) {
                if (!wait_or_abort(sh, &sh->info_full[t % kInfos], (t / kInfos) & 1u)) return false;
                const int own = it.len_k - j * kTileKV;
                const uint8_t* from = p.in.v + ((size_t)(sh->token[t % kInfos] + w * 32 + r4) * p.in.KVH + it.kvh) * kD + part * 16;
#pragma unroll
                for (int s = 0; s < 8; ++s) {
                    in[s] = make_uint4(0u, 0u, 0u, 0u);  // behind the sequence's end: 0 * garbage would poison the row
                    if (w * 32 + s * 4 + r4 < own) in[s] = __ldg(reinterpret_cast<const uint4*>(from + (size_t)s * 4 * p.in.KVH * kD));
                }
                return true;
            };
            ok = fetch(0);
            for (int j = 0; ok && j < it.n_kv; ++j) {
                const int vs = t % kVSlots;
                if (!(ok = wait_or_abort(sh, &sh->v_empty[vs], ((t / kVSlots) & 1u) ^ 1u))) break;
                uint8_t* to = smem + kV + vs * kTileBytes + (part >> 2) * kPanelBytes + (w * 32 + r4) * 128;
                uint32_t odd = 0;
                if (j >= plain_tiles(it)) {
#pragma unroll
                    for (int s = 0; s < 8; ++s) odd |= nan_bytes(in[s].x) | nan_bytes(in[s].y) | nan_bytes(in[s].z) | nan_bytes(in[s].w);
                }
#pragma unroll
                for (int s = 0; s < 8; ++s) {
                    const uint4 lo = make_uint4(q8::e4m3x2_to_half2(in[s].x & 0xffffu), q8::e4m3x2_to_half2(in[s].x >> 16),
                                                q8::e4m3x2_to_half2(in[s].y & 0xffffu), q8::e4m3x2_to_half2(in[s].y >> 16));
                    const uint4 hi = make_uint4(q8::e4m3x2_to_half2(in[s].z & 0xffffu), q8::e4m3x2_to_half2(in[s].z >> 16),
                                                q8::e4m3x2_to_half2(in[s].w & 0xffffu), q8::e4m3x2_to_half2(in[s].w >> 16));
                    // Dims 16 part .. + 15 are chunks 2 (part % 4) and + 1 of a panel's row.  Lanes of the second panel take
                    // theirs in the other order, so that eight lanes always write eight different banks' chunks.
                    const int r7 = (s * 4 + r4) & 7, first = 2 * (part & 3) + (part >> 2), second = first ^ 1;
                    *reinterpret_cast<uint4*>(to + s * 512 + ((first ^ r7) << 4)) = part < 4 ? lo : hi;
                    *reinterpret_cast<uint4*>(to + s * 512 + ((second ^ r7) << 4)) = part < 4 ? hi : lo;
                }
                if (odd & 0x80808080u) {
                    sh->odd_values[k & 1] = k + 1;
#pragma unroll 1
                    for (int i = 0; i < 128; ++i) {  // what this thread has written
                        uint16_t* const h = reinterpret_cast<uint16_t*>(to + (i >> 4) * 512 + (((2 * (part & 3) + (i >> 3 & 1)) ^ ((i >> 4) * 4 + r4 & 7)) << 4)) + (i & 7);
                        if ((*h & 0x7fffu) == 0x7fffu) *h = 0;
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh->v_full[vs]);
                ++t;
                if (j + 1 < it.n_kv) ok = fetch(j + 1);
            }
        }
    }

    // ---- teardown: everyone meets here, then the allocating warp frees tensor memory ----
    tc_fence_before();
    __syncthreads();
    if (warp == 1 && tmem != 0xFFFFFFFFu) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

static int ensure_attr() {
    static std::mutex mu;
    static bool done[64];
    int dev = 0;
    NVLLM_CUDA_OK(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lock(mu);
    if (dev >= 0 && dev < 64 && !done[dev]) {
        for (const void* f : {(const void*)paged_prefill_q8_kernel<Whole>, (const void*)paged_prefill_q8_kernel<Split>, (const void*)paged_prefill_q8_kernel<Tail>}) {
            cudaFuncAttributes a;
            NVLLM_CUDA_OK(cudaFuncGetAttributes(&a, f));
            if (a.numRegs != 128) return fail(NVLLM_B200_ECUDA, "paged_prefill_q8: built with %d registers, not the 128 it shares out", a.numRegs);
            NVLLM_CUDA_OK(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
        }
        done[dev] = true;
    }
    return NVLLM_B200_OK;
}

static int make_byte_map(CUtensorMap* map, const void* base, int heads, int64_t tokens) {
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return fail(NVLLM_B200_EDRIVER, "cuTensorMapEncodeTiled entry point not available");
    cuuint64_t dims[3] = {(cuuint64_t)kD, (cuuint64_t)heads, (cuuint64_t)tokens};
    cuuint64_t strides[2] = {(cuuint64_t)kD, (cuuint64_t)heads * kD};
    cuuint32_t box[3] = {kD, 1, kTileKV};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, estr,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(NVLLM_B200_EDRIVER, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
    return NVLLM_B200_OK;
}

}  // namespace prefill_q8

namespace prefill {
int launch_bytes(const Params& p, const SplitParams* split, const TailParams* tail, const Bytes& in, const void* q, const void* k, const void* v, int64_t slots,
                 int KVH, cudaLaunchConfig_t cfg) {
    using namespace prefill_q8;
    int rc = ensure_attr();
    if (rc) return rc;
    CUtensorMap tm_k;
    if ((rc = make_byte_map(&tm_k, k, KVH, slots))) return rc;
    const Source src = {(const __nv_bfloat16*)q, (const uint8_t*)v, in.k_scale, in.v_scale, in.NB, KVH};
    cfg.blockDim = dim3(prefill_q8::kThreads);
    cfg.dynamicSmemBytes = prefill_q8::kSmemBytes;
    if (split) {
        Split s;
        static_cast<SplitParams&>(s) = *split;
        s.in = src;
        NVLLM_CUDA_OK(cudaLaunchKernelEx(&cfg, paged_prefill_q8_kernel<Split>, tm_k, s));
    } else if (tail) {
        Tail s;
        static_cast<TailParams&>(s) = *tail;
        s.in = src;
        NVLLM_CUDA_OK(cudaLaunchKernelEx(&cfg, paged_prefill_q8_kernel<Tail>, tm_k, s));
    } else {
        Whole s;
        static_cast<Params&>(s) = p;
        s.in = src;
        NVLLM_CUDA_OK(cudaLaunchKernelEx(&cfg, paged_prefill_q8_kernel<Whole>, tm_k, s));
    }
    return NVLLM_B200_OK;
}
}  // namespace prefill

int read_prefill_q8_flags(int* out) {
    NVLLM_CUDA_OK(cudaMemcpyFromSymbol(out, prefill_q8::g_error_flag, sizeof(int)));
    return NVLLM_B200_OK;
}
int clear_prefill_q8_flags() {
    const int zero = 0;
    NVLLM_CUDA_OK(cudaMemcpyToSymbol(prefill_q8::g_error_flag, &zero, sizeof(int)));
    return NVLLM_B200_OK;
}
}  // namespace nvllm
