// Latent attention, expanded form (vk_latent_prefill): a chunk of new tokens
// over the latent cache, with keys and values per head
//
//   k_h,j = [W_k,h c_j | r_j]  (128 + rope elements),  v_h,j = W_v,h c_j  (128)
//   out_t = sum_{j <= pos_t} softmax_j(scale * q_t . k_j) v_j
//
// A (query, key, head) triple costs 2 * (256 + rope) flop here against
// 2 * (2 latent + rope) absorbed (640 and 2,176 at 512 + 64), and a cached token
// and head 2 * 256 * latent once for the expansion: from ~170 new tokens on the
// expanded form does less.  Two kernels per group of heads:
//
//  * latent_expand_kernel: [256 cached tokens] x [128 rows of W] as a tcgen05 GEMM.
//    What bounds it is the way from L2 into an SM (at most 64 bytes a cycle, and
//    ~1,000 to 2,000 cycles long), so every byte of W serves two 128-row tiles: the
//    gathered rows stay on the SM for all heads of the CTA, row tile 0 in shared
//    memory (128 KiB at 512), row tile 1 in TMEM (256 columns), as the A operands of
//    its MMAs.  With one row tile a CTA the same GEMM took 150 us at 8 x 2048 tokens
//    and 32 heads, with two 141.  Output rows [token][head][128 K | 128 V] in the
//    workspace, rounded to the cache's 16-bit type (relative 2^-8 in bf16 and 2^-11
//    in fp16 at most, as a cache of keys and values holds them: in fp32 they would
//    be twice the workspace and its traffic, and no operand of kind::f16); rows behind the
//    sequence are stored as zeros, so the attention reads no stale bytes.
//  * latent_prefill_kernel: causal attention, one CTA per (256 query rows, head,
//    sequence): the rows are two 128-row tiles whose softmax steps alternate on
//    one tensor core (S_A, S_B, then P V of one tile while the other's softmax
//    runs), P in TMEM as the A operand, rounded to the cache's type (vk_latent.cuh,
//    struct Weights), its sum kept in fp32 unrounded.  K and V move through one ring of eight
//    16 KiB units (128 keys x 64 elements): a key tile takes three for K (two of
//    W_k c from the workspace, one of r from the pages) and two for V.  K and V
//    of whole 32 + 16 KiB tiles would not fit twice beside 96 KiB of queries;
//    units let the next K load while the last V is read.
//
// Measured, 512 + 64, 32 heads: 8 chunks of 2048 tokens 500 us (596 in a long run
// under the 1000 W cap, at 1.62 GHz), 141 of them the expansion and 359 the attention.  The
// expansion is bound by shared memory: a stage of 64 latent elements takes 660 cycles,
// 640 of them reads of operands at 128 bytes a cycle.  A step of the attention (a key
// tile against two row tiles) takes ~3,700 cycles, 2,300 to 2,560 of them MMAs: each row
// tile's S, softmax (~1,900 cycles: maximum 285, exponentials and P 1,430, TMEM the
// rest) and P V follow one another, and the issuing thread pays 150 to 200 cycles for
// every barrier and commit between them.  Not kept: a share of the exponentials by a
// polynomial on the FMA pipe (no gain), two issuing threads (16% slower), waiting for
// the next tile's loads between the halves of P V (3% slower).
#include <atomic>

#include "vk_internal.h"
#include "vk_latent.cuh"
#include "vk_ptx.cuh"
#include "vk_rotary.cuh"
#include "vk_tc.cuh"

namespace vk {

constexpr int kLpKeys = 128;
constexpr int kLpRows = 128;           // rows of a tile; a CTA has two
constexpr int kLpHead = 128;           // elements of W_k,h c and of v
constexpr int kLpUnit = kLpKeys * 128;  // 16 KiB
constexpr int kLpSmemMax = 232448;

struct LpParams {
    const int32_t* bt;
    const int32_t* pos;
    const int32_t* offsets;  // NULL: tokens / B each
    uint32_t* err;
    char* ws;     // [nb * lpad][heads][256]
    char* out;    // [tokens][H][128]
    int bt_stride, B, b0, nb, tokens, H, heads, h0, layer, num_pages, P, latent, rope, lpad, max_tokens, max_len, stages, per_cta;
    int q_tiles, splits;   // attention: 256-row tiles of the longest chunk, key ranges a CTA's tile is cut into
    float* part_o;         // splits > 1: [q tile of (b, head)][split][256][128] unnormalised O
    float2* part_ml;       // and its (reference of the weights, their sum) [..][256]
    float scale_log2;
};

struct LpSeq {
    int row0, n, pos;  // first row of the chunk, its tokens, position of its first token
};

// The chunk of sequence b; n = 0 when there is nothing to do or the arguments
// are out of range (recorded by the caller's `record` thread).
__device__ __forceinline__ LpSeq lp_seq(const LpParams& p, int b, bool record) {
    LpSeq s;
    int64_t end;
    if (p.offsets) {
        s.row0 = __ldg(p.offsets + b);
        end = __ldg(p.offsets + b + 1);
    } else {
        const int per = p.tokens / p.B;
        s.row0 = b * per;
        end = s.row0 + per;
    }
    s.pos = __ldg(p.pos + b);
    const int64_t n = end - s.row0;
    s.n = static_cast<int>(n);
    if (n <= 0 || s.row0 < 0 || end > p.tokens || n > p.max_tokens || s.pos < 0 || s.pos + n > p.max_len ||
        s.pos + n > static_cast<int64_t>(p.bt_stride) * p.P) {
        if (n != 0 && record) atomicOr(p.err, VK_ERR_SEQ_LEN);
        s.n = 0;
    }
    return s;
}

// ------------------------------------------------------------------ expansion

// A TMA load holds its issuing warp for ~500 cycles per 16 KiB (and a 2 KiB box
// ~70), about what the MMAs of the stage take: two warps issue.
constexpr int kLeLoaders = 2;
constexpr int kLeThreads = 384;   // 8 epilogue warps, two MMA warps, two TMA warps
constexpr int kLeTokens = 256;    // cached rows of a CTA: row tiles 0 and 1 of 128
constexpr int kLeStage = 16384;   // 128 rows of W x 64
constexpr int kLeMaxStages = 10;

template <typename T>
__global__ void __launch_bounds__(kLeThreads, 1) latent_expand_kernel(const __grid_constant__ CUtensorMap tmap,
                                                                      const __grid_constant__ CUtensorMap tmapw,
                                                                      const __grid_constant__ CUtensorMap tmapkv,
                                                                      const __grid_constant__ LpParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = smem_u32(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // the attention may start its launch: it reads what this kernel writes only behind
    // griddepcontrol.wait
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int bl = blockIdx.z, b = p.b0 + bl, key0 = blockIdx.y * kLeTokens;
    const LpSeq sq = lp_seq(p, b, threadIdx.x == 0 && blockIdx.x == 0 && key0 == 0 && p.h0 == 0);
    const int len = sq.pos + sq.n;
    if (sq.n == 0 || key0 >= len) return;
    const bool two = key0 + kLpKeys < len;  // row tile 1 has rows
    const int hfirst = blockIdx.x * p.per_cta, nh = min(p.per_cta, p.heads - hfirst);
    const int lch = p.latent >> 6;
    const uint32_t s_b = sbase + lch * kLpUnit, s_out = s_b + p.stages * kLeStage;  // s_out: [row tile][128 rows][128 B]
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + lch * kLpUnit + (p.stages + 2) * kLeStage);
    uint64_t* a_full = bars;                       // [2] row tile 1's, then row tile 0's latent rows landed
    uint64_t* a_moved = bars + 2;                  // row tile 1's rows are in TMEM
    uint64_t* b_full = bars + 3;                   // [stages]
    uint64_t* b_empty = b_full + kLeMaxStages;     // [stages]
    uint64_t* acc_full = b_empty + kLeMaxStages;   // [row tile]
    uint64_t* acc_empty = acc_full + 2;            // [row tile]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    if (threadIdx.x == 0) {
        for (int i = 0; i < p.stages; ++i) {
            mbar_init(smem_u32(&b_full[i]), 1);
            mbar_init(smem_u32(&b_empty[i]), two ? 2 : 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&a_full[i]), kLeLoaders);
            mbar_init(smem_u32(&acc_full[i]), 1);
            mbar_init(smem_u32(&acc_empty[i]), 4);
        }
        mbar_init(smem_u32(a_moved), 4);
        mbar_fence_init();
    }
    if (warp == 9) {
        tmem_alloc(smem_u32(tmem_slot), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;  // columns 0..255: row tile 1's latent rows; 256, 384: the accumulators

    if (warp == 8 || warp == 10) {
        const int me = warp == 8 ? 0 : 1;
        const uint64_t pol = l2_evict_last_policy();
        const int npages = (len + p.P - 1) / p.P, ppt = kLpKeys / p.P;
        bool ok = true;
        // stages in the order (head, K rows then V rows, 64 columns of W), every other one mine
        int st = me, it = me;
        uint32_t ph = 1;
        const int total = nh * lch * 2, lead = min(p.stages, total);
        auto load_b = [&](bool wait) {
            if (wait) ok = mbar_wait(smem_u32(&b_empty[st]), ph, p.err);
            if (!ok) return;
            const uint32_t bar = smem_u32(&b_full[st]);
            const int hh = it / lch;  // half-head
            mbar_expect_tx(bar, kLeStage);
            tma_load_2d(s_b + st * kLeStage, &tmapw, (it - hh * lch) * 64, (p.h0 + hfirst) * 256 + hh * 128, bar, pol);
            it += kLeLoaders;
            st += kLeLoaders;
            if (st >= p.stages) {
                st -= p.stages;
                ph ^= 1;
            }
        };
        // the gathered rows: row tile 1 through the same shared memory first
        auto load_a = [&](int tile) {
            const int first = key0 / p.P + tile * ppt, cnt = min(ppt, npages - first);
            int page = 0;
            if (lane < cnt) {
                page = __ldg(p.bt + static_cast<int64_t>(b) * p.bt_stride + first + lane);
                if (page < 0 || page >= p.num_pages) {
                    atomicOr(p.err, VK_ERR_PAGE_ID);
                    page = 0;
                }
            }
            const int mine = (lch - me + kLeLoaders - 1) / kLeLoaders;  // chunks me, me + 2, ...
            const uint32_t bar = smem_u32(&a_full[tile ^ 1]);
            if (lane == 0) mbar_expect_tx(bar, mine * cnt * p.P * 128);
            __syncwarp();
            for (int k = me; k < lch; k += kLeLoaders)
                if (lane < cnt)
                    tma_load_2d(sbase + k * kLpUnit + lane * p.P * 128, &tmap, k * 64, (p.layer * p.num_pages + page) * p.P, bar, pol);
        };
        if (two) load_a(1);
        if (lane == 0)
            while (it < lead) load_b(false);
        __syncwarp();
        if (two) ok = wait_all(smem_u32(a_moved), 0, p.err);
        if (ok) load_a(0);
        if (lane == 0) {
            while (it < total && ok) load_b(true);
            if (!ok) {  // a wait gave up: no copy of this warp may land behind the CTA's end (bounded as well)
                if (two) mbar_wait(smem_u32(&a_full[0]), 0, p.err);
                for (int k = max(me, it - p.stages); k < it; ++k)
                    if ((k - me) % kLeLoaders == 0) mbar_wait(smem_u32(&b_full[k % p.stages]), (k / p.stages) & 1, p.err);
            }
        }
    } else if (warp == 9 || warp == 11) {
        // MMA issuers, one per row tile: an issuing thread is held until its last MMA is
        // dispatched and then needs ~200 cycles to see the next stage's barrier, most of
        // what four MMAs take; the other tile's MMAs fill that time (one warp for both
        // took 980 cycles a stage, 512 of them MMAs).
        constexpr uint32_t id = idesc_16(Elem<T>::kBf16, 128, 128, 0, 0);
        const int tile = warp == 9 ? 0 : 1;
        if ((tile == 0 || two) && elect_lane()) {
            const uint64_t d0 = umma_desc_sw128(sbase, 16, 1024);
            const uint32_t hi = static_cast<uint32_t>(d0 >> 32), a_lo = static_cast<uint32_t>(d0), b_lo = a_lo + ((s_b - sbase) >> 4);
            const uint32_t d = tmem + 256 + tile * 128;
            int st = 0, ph = 0;
            bool ok = mbar_wait(tile ? smem_u32(a_moved) : smem_u32(&a_full[1]), 0, p.err);
            tc_fence_after();
            for (int hh = 0; hh < 2 * nh && ok; ++hh) {  // K half, V half of each head
                if (hh > 0) ok = mbar_wait(smem_u32(&acc_empty[tile]), (hh - 1) & 1, p.err);
                for (int c = 0; c < lch && ok; ++c) {
                    ok = mbar_wait(smem_u32(&b_full[st]), ph, p.err);
                    if (ok) {
                        tc_fence_after();
                        const uint32_t bl = b_lo + st * (kLeStage >> 4);
                        if (tile) {
#pragma unroll
                            for (int ks = 0; ks < 4; ++ks) umma_ts_lo(d, tmem + c * 32 + ks * 8, bl + ks * 2, hi, id, ks ? 1 : c != 0);
                        } else {
                            const uint32_t al = a_lo + c * (kLpUnit >> 4);
#pragma unroll
                            for (int ks = 0; ks < 4; ++ks) umma_ss_lo(d, al + ks * 2, hi, bl + ks * 2, hi, id, ks ? 1 : c != 0);
                        }
                        umma_commit(smem_u32(&b_empty[st]));
                        if (c == lch - 1) umma_commit(smem_u32(&acc_full[tile]));
                    }
                    if (++st == p.stages) {
                        st = 0;
                        ph ^= 1;
                    }
                }
            }
        }
    } else if (warp < 4 || two) {
        // Epilogue: warps 0-3 row tile 0, warps 4-7 row tile 1, a row per thread, out
        // through shared memory by TMA (rows stored straight from registers, 32 bytes
        // each at the workspace's pitch, kept the load/store queue busy for 2,000 to
        // 3,700 cycles a head, and MMAs and loads of those warps waited behind them).
        const int tile = warp >> 2, r = threadIdx.x & 127;
        const bool inside = key0 + tile * kLpKeys + r < len;
        const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const uint32_t stage = s_out + tile * kLeStage;
        constexpr uint32_t kExp = 0x7f800000u;
        bool ok = true;
        if (tile) {  // row tile 1's latent rows, shared memory -> TMEM (two elements a column)
            ok = wait_all(smem_u32(&a_full[0]), 0, p.err);
            for (int c = 0; c < lch; ++c) {
                float w[32];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(w[4 * i]), "=f"(w[4 * i + 1]), "=f"(w[4 * i + 2]), "=f"(w[4 * i + 3])
                                 : "r"(sbase + c * kLpUnit + swz128(r, i)));
                tmem_st32(lane_base + c * 32, w);
            }
            tmem_wait_st();
            fence_async_smem();  // these reads before the next tile's TMA writes
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(a_moved));
        }
        bool bad = false;
        for (int hh = 0; hh < 2 * nh; ++hh) {
            ok = ok && wait_all(smem_u32(&acc_full[tile]), hh & 1, p.err);
            tc_fence_after();
            uint32_t w[64], all = kExp;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float v[2][32];
                tmem_ld32(lane_base + 256 + tile * 128 + c * 64, v[0]);
                tmem_ld32(lane_base + 256 + tile * 128 + c * 64 + 32, v[1]);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const float x = v[i >> 4][2 * (i & 15)], y = v[i >> 4][2 * (i & 15) + 1];
                    w[c * 32 + i] = inside ? Elem<T>::pack_sat(x, y) : 0u;
                    all &= __float_as_uint(x) & __float_as_uint(y);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&acc_empty[tile]));
            // A key whose every element is NaN or infinite comes from such a latent.  Rows
            // that may not see it multiply its value by a weight of zero, so the value is
            // stored as zeros and the key as NaN: a row that sees it gets its NaN through
            // S.  (For the same reason a finite value beyond the type's range is stored as
            // the largest number, not as infinity.)
            if ((hh & 1) == 0) bad = inside && (all & kExp) == kExp;
            if (bad) {
                const uint32_t fill = hh & 1 ? 0u : 0x7fff7fffu;
#pragma unroll
                for (int i = 0; i < 64; ++i) w[i] = fill;
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {  // 64 columns at a time through this tile's 16 KiB
                if (r == 0) bulk_wait_read();
                asm volatile("barrier.cta.sync %0, 128;" ::"r"(1 + tile) : "memory");
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + swz128(r, i)), "r"(w[c * 32 + 4 * i]),
                                 "r"(w[c * 32 + 4 * i + 1]), "r"(w[c * 32 + 4 * i + 2]), "r"(w[c * 32 + 4 * i + 3])
                                 : "memory");
                fence_async_smem();
                asm volatile("barrier.cta.sync %0, 128;" ::"r"(1 + tile) : "memory");
                if (r == 0 && ok) {
                    tma_store_2d(&tmapkv, stage, hfirst * 256 + hh * 128 + c * 64, bl * p.lpad + key0 + tile * kLpKeys);
                    bulk_commit();
                }
            }
        }
        if (r == 0) bulk_wait();
    }
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ------------------------------------------------------------------ attention

constexpr int kLaThreads = 384;  // 8 softmax warps, MMA warp, three TMA warps
constexpr int kLaQ = 0;                              // [2 tiles][3 chunks][128 rows][128 B]
constexpr int kLaRing = 2 * 3 * kLpUnit;             // 96 KiB
constexpr int kLaUnits = 8;
constexpr int kLaBar = kLaRing + kLaUnits * kLpUnit;  // 224 KiB
constexpr int kLaSmem = kLaBar + 256 + 1024;
static_assert(kLaSmem <= kLpSmemMax, "latent prefill shared memory");

template <typename T, bool SPLIT>  // SPLIT: the CTA has one of p.splits ranges of the keys
__global__ void __launch_bounds__(kLaThreads, 1) latent_prefill_kernel(const __grid_constant__ CUtensorMap tmap,
                                                                       const __grid_constant__ CUtensorMap tmapq,
                                                                       const __grid_constant__ CUtensorMap tmapkv,
                                                                       const __grid_constant__ LpParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = smem_u32(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int bl = SPLIT ? blockIdx.z / p.splits : blockIdx.z, split = SPLIT ? blockIdx.z % p.splits : 0, hl = blockIdx.y;
    const int b = p.b0 + bl, h = p.h0 + hl;
    const LpSeq sq = lp_seq(p, b, false);
    const int qt = p.q_tiles - 1 - static_cast<int>(blockIdx.x), q0 = qt * 2 * kLpRows;  // most keys first
    if (q0 >= sq.n) {  // (this grid must not end before the expansion does)
        asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    const int pos0 = sq.pos;
    const int rowsA = min(kLpRows, sq.n - q0), rowsB = max(0, min(kLpRows, sq.n - q0 - kLpRows));
    const int lenA = pos0 + q0 + rowsA, lenB = rowsB > 0 ? pos0 + q0 + kLpRows + rowsB : 0;
    // this CTA's key tiles kt0 .. kt0 + ntiles - 1; row tile A (B) sees the first ntA (ntB)
    const int kv_len = max(lenA, lenB), all = (kv_len + kLpKeys - 1) / kLpKeys;
    const int kt0 = SPLIT ? static_cast<int>(static_cast<int64_t>(split) * all / p.splits) : 0;
    const int ntiles = SPLIT ? static_cast<int>(static_cast<int64_t>(split + 1) * all / p.splits) - kt0 : all;
    const int ntA = max(0, min(ntiles, (lenA + kLpKeys - 1) / kLpKeys - kt0));
    const int ntB = max(0, min(ntiles, (lenB + kLpKeys - 1) / kLpKeys - kt0));

    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kLaBar);
    uint64_t* k_full = bars;       // [2] the three K units of a tile landed
    uint64_t* v_full = bars + 2;   // [2]
    // even and odd key tiles have barriers of their own: the tile after the one the
    // producer waits for may complete first, and one barrier would then be a phase ahead
    uint64_t* v_empty = bars + 4;  // [2] both row tiles' P V of a key tile done
    uint64_t* s_full = bars + 6;   // [row tile][2] S done; row tile B's (or the last to see the keys): K has been read too
    uint64_t* p_full = bars + 10;  // [row tile][half of the keys] P written, before the first O rescaled
    uint64_t* o_full = bars + 14;  // [row tile] the last P V done
    uint64_t* q_full = bars + 16;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 17);
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&k_full[i]), 3);  // the two units of W_k c and the rotary parts
            mbar_init(smem_u32(&v_full[i]), 2);
            mbar_init(smem_u32(&v_empty[i]), 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(smem_u32(&s_full[i]), 1);
            mbar_init(smem_u32(&p_full[i]), 4);
        }
        mbar_init(smem_u32(&o_full[0]), 1);
        mbar_init(smem_u32(&o_full[1]), 1);
        mbar_init(smem_u32(q_full), 1);
        mbar_fence_init();
        // rows past the chunk read the next rows of q or zeros and are not stored
        prefetch_tmap(&tmapq);
        mbar_expect_tx(smem_u32(q_full), 2 * 3 * kLpUnit);
        const uint64_t pol = l2_evict_first_policy();
        for (int t = 0; t < 2; ++t)
            for (int c = 0; c < 3; ++c)
                tma_load_3d(sbase + kLaQ + (t * 3 + c) * kLpUnit, &tmapq, c * 64, h, sq.row0 + q0 + t * kLpRows,
                            smem_u32(q_full), pol);
    }
    if (warp == 9) {
        tmem_alloc(smem_u32(tmem_slot), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 8 || warp == 10) {
        // ------------------------------------------------------------ TMA: W c of K and V, one unit of each
        // (a load holds its warp for ~500 cycles per 16 KiB: three warps share a tile)
        // units 5j .. 5j+2 take the ring slots of tile j-2's last K unit and its V,
        // units 5j+3, 5j+4 those of tile j-1's first two K units
        if (lane == 0) {
            const uint64_t pol = l2_evict_last_policy();  // other row tiles read the same K and V
            const int wrow = bl * p.lpad + kt0 * kLpKeys, u = warp == 8 ? 0 : 1;
            int landed = -1;  // the last tile whose K and V are on their way
            bool ok = true;
            asm volatile("griddepcontrol.wait;" ::: "memory");
            for (int j = 0; j < ntiles; ++j) {
                if (j >= 2) ok = ok && mbar_wait(smem_u32(&v_empty[j & 1]), ((j >> 1) - 1) & 1, p.err);
                if (!ok) break;
                const uint32_t kbar = smem_u32(&k_full[j & 1]), vbar = smem_u32(&v_full[j & 1]);
                mbar_expect_tx(kbar, kLpUnit);
                tma_load_2d(sbase + kLaRing + ((5 * j + u) & 7) * kLpUnit, &tmapkv, hl * 256 + u * 64, wrow + j * kLpKeys,
                            kbar, pol);
                if (j >= 1) ok = mbar_wait(smem_u32(&s_full[(j - 1 < ntB ? 2 : 0) + ((j - 1) & 1)]), ((j - 1) >> 1) & 1, p.err);
                if (!ok) break;
                mbar_expect_tx(vbar, kLpUnit);
                tma_load_2d(sbase + kLaRing + ((5 * j + 3 + u) & 7) * kLpUnit, &tmapkv, hl * 256 + kLpHead + u * 64,
                            wrow + j * kLpKeys, vbar, pol);
                landed = j;
            }
            if (!ok)  // a wait gave up: no copy of this warp may land behind the CTA's end (bounded as well)
                for (int j = max(0, landed - 1); j <= min(landed + 1, ntiles - 1); ++j) {
                    mbar_wait(smem_u32(&k_full[j & 1]), (j >> 1) & 1, p.err);
                    if (j <= landed) mbar_wait(smem_u32(&v_full[j & 1]), (j >> 1) & 1, p.err);
                }
        }
    } else if (warp == 11) {
        // ------------------------------------------------------------ TMA: rotary parts from the pages
        // (a warp of its own: eight 16-token pages take ~600 cycles to issue)
        const uint64_t pol = l2_evict_last_policy();
        const int ppt = kLpKeys / p.P, npages = (kv_len + p.P - 1) / p.P - kt0 * ppt;  // from the first tile's on
        const int32_t* btrow = p.bt + static_cast<int64_t>(b) * p.bt_stride + kt0 * ppt;
        auto page_of = [&](int j) {  // a page of the tile per lane
            int page = lane < ppt && j * ppt + lane < npages ? __ldg(btrow + j * ppt + lane) : 0;
            if (page < 0 || page >= p.num_pages) {
                atomicOr(p.err, VK_ERR_PAGE_ID);
                page = 0;
            }
            return page;
        };
        bool ok = true;
        int next = page_of(0);
        for (int j = 0; j < ntiles; ++j) {
            const int page = next, cnt = min(ppt, npages - j * ppt);
            if (j + 1 < ntiles) next = page_of(j + 1);
            if (j >= 2) ok = wait_all(smem_u32(&v_empty[j & 1]), ((j >> 1) - 1) & 1, p.err);
            if (!ok) break;
            const uint32_t kbar = smem_u32(&k_full[j & 1]);
            if (lane == 0) mbar_expect_tx(kbar, cnt * p.P * 128);
            if (lane < cnt)
                tma_load_2d(sbase + kLaRing + ((5 * j + 2) & 7) * kLpUnit + lane * p.P * 128, &tmap, p.latent,
                            (p.layer * p.num_pages + page) * p.P, kbar, pol);
        }
    } else if (warp == 9) {
        // ------------------------------------------------------------ MMA issuer
        // S_A0, S_B0, PV_A0, S_A1, PV_B0, S_B1, ...: one thread, so its MMAs execute in
        // order, P is read before the next S overwrites it, and each step's products
        // are done as early as they can be (a second issuing warp, one per row tile,
        // made the steps interleave and was 16% slower).  Unrolled runs on 32-bit
        // descriptor words: ~40 cycles an MMA (60 on 64-bit ones).
        constexpr uint32_t id_s = idesc_16(Elem<T>::kBf16, 128, 128, 0, 0);
        constexpr uint32_t id_pv = idesc_16(Elem<T>::kBf16, 128, 128, 0, 1), id_half = idesc_16(Elem<T>::kBf16, 128, 64, 0, 1);
        if (elect_lane()) {
            bool ok = mbar_wait(smem_u32(q_full), 0, p.err);
            int k_waited = -1, v_waited = -1;
            const int rsteps = p.rope >> 4;
            const uint64_t dk0 = umma_desc_sw128(sbase + kLaRing, 16, 1024), dv0 = umma_desc_sw128(sbase + kLaRing, kLpUnit, 1024);
            const uint32_t k_hi = static_cast<uint32_t>(dk0 >> 32), k_lo = static_cast<uint32_t>(dk0);
            const uint32_t v_hi = static_cast<uint32_t>(dv0 >> 32), v_lo = static_cast<uint32_t>(dv0);
            const uint32_t q_lo = k_lo - (kLaRing >> 4);
            constexpr uint32_t kUnit16 = kLpUnit >> 4;
            auto issue_s = [&](int t, int j) {
                if (j > k_waited) {
                    ok = ok && mbar_wait(smem_u32(&k_full[j & 1]), (j >> 1) & 1, p.err);
                    k_waited = j;
                }
                if (ok) {
                    tc_fence_after();
                    const uint32_t ql = q_lo + t * 3 * kUnit16, d = tmem + t * 128;
#pragma unroll
                    for (int u = 0; u < 3; ++u) {
                        const uint32_t kl = k_lo + ((5 * j + u) & 7) * kUnit16;
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks)
                            if (u < 2 || ks < rsteps) umma_ss_lo(d, ql + u * kUnit16 + ks * 2, k_hi, kl + ks * 2, k_hi, id_s, (u | ks) != 0);
                    }
                    umma_commit(smem_u32(&s_full[2 * t + (j & 1)]));
                }
            };
            auto issue_pv = [&](int t, int j) {
                if (j > v_waited) {
                    ok = ok && mbar_wait(smem_u32(&v_full[j & 1]), (j >> 1) & 1, p.err);
                    v_waited = j;
                }
                // in two halves of the keys: the first runs behind the second's exponentials
                const uint32_t d = tmem + 256 + t * 128, a = tmem + t * 128;
                const int slot = (5 * j + 3) & 7;
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    ok = ok && mbar_wait(smem_u32(&p_full[2 * t + hf]), j & 1, p.err);
                    if (!ok) return;
                    tc_fence_after();
                    const uint32_t acc = j > 0 || hf > 0;
                    if (slot < 7) {  // both 64-column units side by side: one MMA spans them
                        const uint32_t vl = v_lo + slot * kUnit16;
#pragma unroll
                        for (int ks = 4 * hf; ks < 4 * hf + 4; ++ks)
                            umma_ts_lo(d, a + ks * 8, vl + ks * 128, v_hi, id_pv, ks & 3 ? 1 : acc);
                    } else {
#pragma unroll 1
                        for (int u = 0; u < 2; ++u) {
                            const uint32_t vl = v_lo + ((slot + u) & 7) * kUnit16;
#pragma unroll
                            for (int ks = 4 * hf; ks < 4 * hf + 4; ++ks)
                                umma_ts_lo(d + u * 64, a + ks * 8, vl + ks * 128, v_hi, id_half, ks & 3 ? 1 : acc);
                        }
                    }
                }
                // a commit costs this thread ~200 cycles, the second of two in a row more:
                // three a step (six took 3,700 cycles a step)
                if (t == 1 || j >= ntB) umma_commit(smem_u32(&v_empty[j & 1]));
                if (j == (t ? ntB : ntA) - 1) umma_commit(smem_u32(&o_full[t]));
            };
            if (ntA > 0) issue_s(0, 0);
            if (ntB > 0) issue_s(1, 0);
            for (int j = 0; j < ntiles && ok; ++j) {
                if (j < ntA) {
                    issue_pv(0, j);
                    if (j + 1 < ntA) issue_s(0, j + 1);
                }
                if (j < ntB) {
                    issue_pv(1, j);
                    if (j + 1 < ntB) issue_s(1, j + 1);
                }
            }
        }
    } else {
        // ------------------------------------------------------------ softmax, one query row per thread
        const int t = warp >> 2, r = threadIdx.x & 127, qrow = q0 + t * kLpRows + r;
        const bool valid_row = qrow < sq.n;
        const int qpos = pos0 + qrow, ntt = t ? ntB : ntA;
        const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const uint32_t s_col = t * 128, o_col = 256 + t * 128;
        const float sc = p.scale_log2;
        float m_ref = -INFINITY, l = 0.f;
        bool alive = true;
        for (int j = 0; j < ntt; ++j) {
            if (!wait_all(smem_u32(&s_full[2 * t + (j & 1)]), (j >> 1) & 1, p.err)) { alive = false; break; }
            tc_fence_after();
            const int key0 = (kt0 + j) * kLpKeys;
            float v[kLpKeys / 32][32];
#pragma unroll
            for (int c = 0; c < kLpKeys / 32; ++c) tmem_ld32(lane_base + s_col + c * 32, v[c]);
            tmem_wait_ld();
            if (key0 + kLpKeys - 1 > pos0 + q0 + t * kLpRows) {
                const int lim = qpos - key0;
#pragma unroll
                for (int c = 0; c < kLpKeys / 32; ++c)
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (c * 32 + i > lim) v[c][i] = -INFINITY;
            }
            float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < kLpKeys / 32; ++c)
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    mx4[0] = max3(mx4[0], v[c][i], v[c][i + 1]);
                    mx4[1] = max3(mx4[1], v[c][i + 2], v[c][i + 3]);
                    mx4[2] = max3(mx4[2], v[c][i + 4], v[c][i + 5]);
                    mx4[3] = max3(mx4[3], v[c][i + 6], v[c][i + 7]);
                }
            const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * sc;
            float alpha = 1.f;
            if (mx > m_ref + (Weights<T>::kMargin + Weights<T>::kLag) || m_ref == -INFINITY) {
                const float m_new = fmaxf(m_ref, mx - Weights<T>::kMargin);
                alpha = m_ref == -INFINITY ? 0.f : ex2(m_ref - m_new);
                m_ref = m_new;
            }
            const float mneg = m_ref == -INFINITY ? 0.f : -m_ref;
            const uint64_t sc2 = f2(sc, sc), mneg2 = f2(mneg, mneg);
            uint64_t sum2[4] = {0, 0, 0, 0};
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
#pragma unroll
                for (int c = 2 * hf; c < 2 * hf + 2; ++c) {
                    uint32_t pk[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        float a0, a1;
                        f2_get(f2_fma(f2(v[c][i], v[c][i + 1]), sc2, mneg2), a0, a1);
                        a0 = ex2(a0);
                        a1 = ex2(a1);
                        sum2[(i >> 1) & 3] = f2_add(sum2[(i >> 1) & 3], f2(a0, a1));
                        pk[i >> 1] = Elem<T>::pack(a0, a1);
                    }
                    tmem_st16(lane_base + s_col + c * 16, pk);
                }
                // with half of the S row's registers dead
                if (hf == 0 && j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
                    for (int c = 0; c < kLpHead / 32; ++c) {
                        float o[32];
                        tmem_ld32(lane_base + o_col + c * 32, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] *= alpha;
                        tmem_st32(lane_base + o_col + c * 32, o);
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&p_full[2 * t + hf]));
            }
            {
                float s0, s1;
                f2_get(f2_add(f2_add(sum2[0], sum2[1]), f2_add(sum2[2], sum2[3])), s0, s1);
                l = l * alpha + (s0 + s1);
            }
        }
        const int64_t part = SPLIT ? ((((static_cast<int64_t>(bl) * p.heads + hl) * p.q_tiles + qt) * p.splits + split) * 256 + t * kLpRows + r) : 0;
        if (SPLIT) p.part_ml[part] = make_float2(m_ref, l);  // (-inf, 0) where no key is seen
        if (alive && ntt > 0 && wait_all(smem_u32(&o_full[t]), 0, p.err)) {
            tc_fence_after();
            const float inv = 1.f / l;
            char* dst = SPLIT ? reinterpret_cast<char*>(p.part_o + part * kLpHead)
                              : p.out + 2 * ((static_cast<int64_t>(sq.row0) + (valid_row ? qrow : 0)) * p.H + h) * kLpHead;
#pragma unroll
            for (int c = 0; c < kLpHead / 32; ++c) {
                float o[32];
                tmem_ld32(lane_base + o_col + c * 32, o);
                tmem_wait_ld();
                if (!valid_row) continue;
                if constexpr (SPLIT) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<float4*>(dst + 4 * (c * 32 + i)) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i += 8)
                        *reinterpret_cast<uint4*>(dst + 2 * (c * 32 + i)) =
                            make_uint4(Elem<T>::pack(o[i] * inv, o[i + 1] * inv), Elem<T>::pack(o[i + 2] * inv, o[i + 3] * inv),
                                       Elem<T>::pack(o[i + 4] * inv, o[i + 5] * inv), Elem<T>::pack(o[i + 6] * inv, o[i + 7] * inv));
                }
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Joins the key ranges of a query row: a warp per (row, head), four elements a lane.
template <typename T>
__global__ void __launch_bounds__(128) latent_prefill_merge_kernel(const __grid_constant__ LpParams p) {
    const int lane = threadIdx.x & 31, bl = blockIdx.z, hl = blockIdx.y, qrow = blockIdx.x * 4 + (threadIdx.x >> 5);
    const LpSeq sq = lp_seq(p, p.b0 + bl, false);
    if (qrow >= sq.n) return;
    const int64_t part0 = ((static_cast<int64_t>(bl) * p.heads + hl) * p.q_tiles + (qrow >> 8)) * p.splits;
    float2 ml = make_float2(-INFINITY, 0.f);  // lane s: split s (at most 16)
    if (lane < p.splits) ml = p.part_ml[(part0 + lane) * 256 + (qrow & 255)];
    float m = ml.x;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    m = __shfl_sync(0xffffffffu, m, 0);
    const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - m);
    float l = f * ml.y;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    l = __shfl_sync(0xffffffffu, l, 0);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < p.splits; ++s) {
        const float w = __shfl_sync(0xffffffffu, f, s);
        if (w == 0.f) continue;  // a range that the row does not see has no O
        const float4 x = *reinterpret_cast<const float4*>(p.part_o + ((part0 + s) * 256 + (qrow & 255)) * kLpHead + lane * 4);
        acc = make_float4(fmaf(w, x.x, acc.x), fmaf(w, x.y, acc.y), fmaf(w, x.z, acc.z), fmaf(w, x.w, acc.w));
    }
    const float inv = 1.f / l;
    char* dst = p.out + 2 * ((static_cast<int64_t>(sq.row0) + qrow) * p.H + p.h0 + hl) * kLpHead;
    *reinterpret_cast<uint2*>(dst + lane * 8) = make_uint2(Elem<T>::pack(acc.x * inv, acc.y * inv), Elem<T>::pack(acc.z * inv, acc.w * inv));
}

// Partials of split query tiles: at most one CTA per SM.
constexpr int kLpMaxSplits = 16;
static size_t lp_part_bytes(const vk_pool* pool) { return static_cast<size_t>(pool->num_sms) * 256 * (kLpHead * 4 + 8); }

// What the workspace holds the keys and values of at once: as many heads of all
// sequences as fit 1 GiB, else as many sequences' one head, one at least; in even groups.
constexpr int64_t kLpWorkspace = 1ll << 30;
constexpr int kLpMaxLen = 65535 * kLpKeys;  // (row tiles are a grid's y)
struct LpGroup {
    int heads, seqs;
};
static int64_t lp_pad(int32_t max_seq_len) { return (static_cast<int64_t>(max_seq_len) + kLpKeys - 1) / kLpKeys * kLpKeys; }
static LpGroup lp_group(int64_t lpad, int B, int H) {
    auto even = [](int n, int64_t most) {
        const int groups = static_cast<int>((n + most - 1) / most);
        return (n + groups - 1) / groups;
    };
    const int64_t fit = max(kLpWorkspace / (lpad * 512), static_cast<int64_t>(1));  // (sequence, head) pairs
    return {even(H, max(fit / B, static_cast<int64_t>(1))), even(B, fit)};
}

template <typename T>
static vk_status launch_latent_prefill(vk_pool* pool, LpParams p, const CUtensorMap& tq, const CUtensorMap& tw, const CUtensorMap& tkv,
                                       cudaStream_t st) {
    static std::atomic<uint64_t> attr_set{0};  // a bit per device; host threads may call at once
    const uint64_t bit = 1ull << (pool->device & 63);
    if (!(attr_set.load(std::memory_order_acquire) & bit)) {
        cudaError_t e = cudaFuncSetAttribute(latent_expand_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kLpSmemMax);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(latent_prefill_kernel<T, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kLaSmem);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(latent_prefill_kernel<T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kLaSmem);
        if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(latent prefill)");
        attr_set.fetch_or(bit, std::memory_order_release);
    }
    const int lch = p.latent / 64;
    p.stages = min(kLeMaxStages, (kLpSmemMax - 2048 - lch * kLpUnit) / kLeStage - 2);  // 4, 6, 8, 10 at 512 .. 128
    const size_t smem = static_cast<size_t>(lch) * kLpUnit + static_cast<size_t>(p.stages + 2) * kLeStage + 2048;
    // Heads per CTA: the count whose waves of CTAs are done first, at ~10 units of time a
    // head and ~6 for a CTA's start (its gathered rows are read once for all its heads).
    const int row_tiles = (p.lpad + kLeTokens - 1) / kLeTokens;
    int64_t best = 0;
    p.per_cta = 1;
    for (int n = 1; n <= p.heads; ++n) {
        const int64_t ctas = static_cast<int64_t>(p.nb) * row_tiles * ((p.heads + n - 1) / n);
        const int64_t cost = (ctas + pool->num_sms - 1) / pool->num_sms * (10 * n + 6);
        if (n == 1 || cost < best) {
            best = cost;
            p.per_cta = n;
        }
    }
    latent_expand_kernel<T><<<dim3((p.heads + p.per_cta - 1) / p.per_cta, row_tiles, p.nb), kLeThreads, smem, st>>>(pool->tmap16, tw, tkv, p);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "latent_expand_kernel launch");
    // Too few CTAs for the GPU: each (query tile, head, sequence) is cut along its keys,
    // into ranges of six key tiles or more (200 new tokens behind 30k, 8 heads: 598 us
    // without, 134 with; 1,030 behind none in two ranges: 44 instead of 35).
    p.q_tiles = (p.max_tokens + 2 * kLpRows - 1) / (2 * kLpRows);
    const int64_t base = static_cast<int64_t>(p.q_tiles) * p.heads * p.nb;
    p.splits = static_cast<int>(max(static_cast<int64_t>(1), min(min(static_cast<int64_t>(kLpMaxSplits), pool->num_sms / base),
                                                                  static_cast<int64_t>(p.max_len / (6 * kLpKeys)))));
    const dim3 grid(p.q_tiles, p.heads, p.nb * p.splits);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kLaThreads);
    cfg.dynamicSmemBytes = kLaSmem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = p.splits > 1 ? cudaLaunchKernelEx(&cfg, latent_prefill_kernel<T, true>, pool->tmap16, tq, tkv, p)
                     : cudaLaunchKernelEx(&cfg, latent_prefill_kernel<T, false>, pool->tmap16, tq, tkv, p);
    if (e != cudaSuccess) return cuda_fail(e, "latent_prefill_kernel launch");
    if (p.splits > 1) {
        latent_prefill_merge_kernel<T><<<dim3((p.max_tokens + 3) / 4, p.heads, p.nb), 128, 0, st>>>(p);
        e = cudaGetLastError();
        if (e != cudaSuccess) return cuda_fail(e, "latent_prefill_merge_kernel launch");
    }
    return VK_OK;
}

}  // namespace vk

using namespace vk;

extern "C" size_t vk_latent_prefill_workspace_size(const vk_pool* pool, int32_t batch, int32_t max_seq_len, int32_t num_heads) {
    if (!pool || !is_latent(pool) || batch <= 0 || max_seq_len <= 0 || max_seq_len > kLpMaxLen || num_heads <= 0) return 0;
    const int64_t lpad = lp_pad(max_seq_len);
    const LpGroup group = lp_group(lpad, batch, num_heads);
    return static_cast<size_t>(lpad) * group.seqs * 512 * group.heads + lp_part_bytes(pool);
}

extern "C" vk_status vk_latent_prefill(vk_pool* pool, int32_t layer, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                       const void* w_kv, int64_t w_stride, void* out, const int32_t* block_tables,
                                       int32_t bt_stride, const int32_t* positions, const int32_t* offsets, int32_t batch,
                                       int32_t tokens, int32_t max_tokens, int32_t max_seq_len, int32_t num_heads, float scale,
                                       void* workspace, size_t workspace_bytes, void* stream) {
    if (!pool) return fail(VK_INVALID_ARG, "pool is NULL");
    if (!is_latent(pool)) return fail(VK_UNSUPPORTED, "latent prefill needs a latent pool");
    if (layer < 0 || layer >= pool->cfg.num_layers) return fail(VK_INVALID_ARG, "layer out of range");
    if (batch < 0 || tokens < 0 || num_heads <= 0 || bt_stride <= 0) return fail(VK_INVALID_ARG, "bad batch/tokens/heads/bt_stride");
    if (!(scale >= 0.f) || scale > 3.0e38f) return fail(VK_INVALID_ARG, "scale must be finite, > 0 or 0 for 1/sqrt(128 + rope_dim)");
    if (batch == 0 || tokens == 0) return VK_OK;
    if (!q || !w_kv || !out || !block_tables || !positions) return fail(VK_INVALID_ARG, "NULL array");
    if (!offsets && tokens % batch) return fail(VK_INVALID_ARG, "without offsets, tokens must be a multiple of batch");
    if (max_tokens <= 0 || max_seq_len <= 0) return fail(VK_INVALID_ARG, "max_tokens and max_seq_len must be > 0");
    if (!offsets && (max_tokens < tokens / batch || max_seq_len < tokens / batch))
        return fail(VK_INVALID_ARG, "max_tokens or max_seq_len is smaller than the chunk");
    if (max_tokens > max_seq_len) max_tokens = max_seq_len;  // no chunk is longer than its sequence
    if (max_seq_len > static_cast<int64_t>(bt_stride) * pool->cfg.page_tokens)
        return fail(VK_INVALID_ARG, "max_seq_len exceeds the block table capacity");
    if (batch > 65535 || num_heads > 65535) return fail(VK_INVALID_ARG, "batch and num_heads must be <= 65535");
    if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(w_kv) | reinterpret_cast<uintptr_t>(out)) & 15) ||
        q_token_stride % 8 || q_head_stride % 8 || w_stride % 8)
        return fail(VK_INVALID_ARG, "q, w_kv and out must be 16-byte aligned, strides multiples of 8");
    if (q_token_stride < 0 || q_head_stride < 0 || w_stride < pool->latent_dim)
        return fail(VK_INVALID_ARG, "q strides must be >= 0, w_stride >= latent_dim");
    if (max_seq_len > kLpMaxLen) return fail(VK_INVALID_ARG, "max_seq_len too large");
    const size_t need = vk_latent_prefill_workspace_size(pool, batch, max_seq_len, num_heads);
    if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 127))
        return fail(VK_INVALID_ARG, "workspace missing, too small or not 128-byte aligned");
    LpParams p{};
    p.bt = block_tables;
    p.pos = positions;
    p.offsets = offsets;
    p.err = pool->d_err;
    p.ws = static_cast<char*>(workspace);
    p.out = static_cast<char*>(out);
    p.bt_stride = bt_stride;
    p.B = batch;
    p.tokens = tokens;
    p.H = num_heads;
    p.layer = layer;
    p.num_pages = pool->num_pages;
    p.P = pool->cfg.page_tokens;
    p.latent = pool->latent_dim;
    p.rope = pool->rope_dim;
    p.lpad = static_cast<int>(lp_pad(max_seq_len));
    p.max_tokens = max_tokens;
    p.max_len = max_seq_len;
    const int width = kLpHead + p.rope;
    p.scale_log2 = (scale > 0.f ? scale : 1.0f / sqrtf(static_cast<float>(width))) * 1.4426950408889634f;
    const LpGroup group = lp_group(p.lpad, batch, num_heads);
    p.part_o = reinterpret_cast<float*>(p.ws + static_cast<size_t>(p.lpad) * group.seqs * 512 * group.heads);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + static_cast<size_t>(pool->num_sms) * 256 * kLpHead);

    const CUtensorMapDataType type = pool->kv_format == VK_KV_LATENT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    alignas(64) CUtensorMap tq, tw, tkv;
    auto encode = tmap_encode_fn();
    if (!encode) return fail(VK_CUDA_ERROR, "cuTensorMapEncodeTiled unavailable");
    const cuuint32_t estr[3] = {1, 1, 1};
    {
        // a stride of a dimension of one element is never used: any valid one will do
        const cuuint64_t hs = static_cast<cuuint64_t>(num_heads > 1 ? q_head_stride : width + 8) * 2 & ~cuuint64_t(15);
        const cuuint64_t ts = static_cast<cuuint64_t>(tokens > 1 ? q_token_stride : width + 8) * 2 & ~cuuint64_t(15);
        const cuuint64_t dims[3] = {static_cast<cuuint64_t>(width), static_cast<cuuint64_t>(num_heads), static_cast<cuuint64_t>(tokens)};
        const cuuint64_t strides[2] = {hs, ts};
        const cuuint32_t box[3] = {64, 1, kLpRows};
        if (encode(&tq, type, 3, const_cast<void*>(q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return fail(VK_INVALID_ARG, "q's shape or strides cannot be addressed by TMA");
    }
    {
        const cuuint64_t dims[2] = {static_cast<cuuint64_t>(p.latent), static_cast<cuuint64_t>(num_heads) * 256};
        const cuuint64_t strides[1] = {static_cast<cuuint64_t>(w_stride) * 2};
        const cuuint32_t box[2] = {64, 128};
        if (encode(&tw, type, 2, const_cast<void*>(w_kv), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return fail(VK_INVALID_ARG, "w_kv's shape or stride cannot be addressed by TMA");
    }
    DeviceGuard g(pool->device);
    // the last groups may have fewer heads or sequences; rows keep their own pitch, so each has its own map
    for (int b0 = 0; b0 < batch; b0 += group.seqs)
        for (int h0 = 0; h0 < num_heads; h0 += group.heads) {
            p.b0 = b0;
            p.nb = min(group.seqs, batch - b0);
            p.h0 = h0;
            p.heads = min(group.heads, num_heads - h0);
            const cuuint64_t dims[2] = {static_cast<cuuint64_t>(p.heads) * 256, static_cast<cuuint64_t>(p.nb) * p.lpad};
            const cuuint64_t strides[1] = {static_cast<cuuint64_t>(p.heads) * 512};
            const cuuint32_t box[2] = {64, kLpKeys};
            if (encode(&tkv, type, 2, workspace, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
                return fail(VK_CUDA_ERROR, "cuTensorMapEncodeTiled failed for the workspace");
            const vk_status s = pool->kv_format == VK_KV_LATENT_BF16
                                    ? launch_latent_prefill<__nv_bfloat16>(pool, p, tq, tw, tkv, as_stream(stream))
                                    : launch_latent_prefill<__half>(pool, p, tq, tw, tkv, as_stream(stream));
            if (s != VK_OK) return s;
        }
    return VK_OK;
}
