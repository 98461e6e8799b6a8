// Latent attention, absorbed form (vk_latent_decode): every query row of a
// sequence (its T new tokens x H heads) attends the cached rows x_j = [c_j | r_j]
//
//   s_j = scale * (ql . c_j + qr . r_j),  out = sum_j softmax(s)_j c_j
//
// so the cache row is key and value at once and is read from HBM once for up to
// 64 rows.  Floor: (latent + rope) * 2 bytes a cached token; 2 * (2 latent +
// rope) flop a token and row, which 64 rows keep below the memory time.
//
// One persistent CTA per SM.  The cached tokens of all units (sequence, group
// of 64 rows) are cut into 64-key tiles, laid end to end and dealt in equal
// contiguous ranges, from the device's own lengths (no host plan: a captured
// graph replays with other lengths).  A unit that several CTAs share leaves
// fp32 partials (O, m, l) that latent_merge_kernel joins.
//
//  * warps 4 and 7-9 stream tiles with 2-D TMA boxes (64 elements x one page's
//    rows, 128-byte swizzle) into a ring of as many stages as fit (2 at 512 + 64);
//  * warp 5 issues  S[64 rows x 64 keys] = Q K^T  (tcgen05.mma, M 64, K-major
//    both) and warp 6  O^T[latent x 64 rows] += V^T P^T  as M = 128 blocks of
//    latent elements: an MMA costs its thread ~40 cycles to issue, more than the
//    tensor core takes, so two threads issue (one lane each: waits and issue by the
//    whole warp were 6% slower).  The transposed output keeps all 128 lanes at work with 64
//    rows (O itself would be M = 64 at half the rate) and needs 256 TMEM columns
//    instead of 512, so S has two buffers beside it: S of tile i+1 is issued
//    before O of tile i and the tensor core works through the softmax.  V^T is
//    the K tile itself read MN-major, P^T is P read K-major: nothing is copied;
//  * warps 0-3: softmax with running maximum and sum.  Row r of S lies in lane
//    (r/16)*32 + r%16 of TMEM (M = 64 fills 16 lanes of each warp's quarter); the
//    matrix-fragment load spreads them over all 32 threads (2 rows x 16 keys
//    each), and P goes to shared memory by stmatrix.  O is rescaled only when a
//    row's maximum grows by more than 2^8 (all warps vote).
//
// P is rounded to the cache's 16-bit type for the second product, the type that
// the tensor core takes beside it: relative 2^-8 (bf16) or 2^-11 (fp16) a weight at
// most, the same step as the output's own rounding, absolute 2^-32 of the row's
// largest weight among fp16's subnormals (struct Weights); the sum of the weights is
// taken from the unrounded fp32 values.
//
// Measured, 512 + 64, 64 rows: 24 sequences of ~16k tokens 89 us at 1.965 GHz, 0.75 of
// the measured copy rate, and 107 us in a long run, where the 1000 W cap leaves 1.62 GHz:
// the time follows the SM clock.  Between its ends a CTA takes a 64-key tile in 2,980
// cycles (7.2 TB/s at 1.965 GHz), and those cycles bound it.
// 64 x ~2k tokens 49 us, 0.53: the merge kernel takes 6-7 us of that, a CTA's start
// (lengths, queries, first pages, first tile) 12,000 cycles and a change of units
// 10,500, of which half is the next queries waiting behind the tiles in flight.
// Measured and not kept: the output written by the TMA warps behind the next unit's
// first tiles (no faster), queries loaded into the ring ahead of the tiles (52 us: the
// MMA threads lose more to moving buffers than the change of units gains), queries
// prefetched to L2 (50.3), P V products cut to the live 16-key blocks of the last tile
// (a predicate per MMA: 10% slower), L2 prefetch ahead of the ring (4-12% slower),
// programmatic launch of this kernel behind the last (no gain).
//
// Rows of the last tile behind the sequence are zeroed in shared memory before
// the second product (0 * NaN is NaN), and keys that only some of the T tokens
// may see have non-finite elements cleared there.  A row that does see such a
// key gets its NaN through S where the score is +inf or NaN; a score of -inf is a
// weight of 0, and 0 * inf is NaN in the infinite element alone, as in a tile that all
// rows see: those elements are written behind the output (ld_broken_keys).
#include <atomic>

#include "vk_internal.h"
#include "vk_latent.cuh"
#include "vk_latent_deal.h"
#include "vk_ptx.cuh"
#include "vk_rotary.cuh"
#include "vk_tc.cuh"

namespace vk {

constexpr int kLdKeys = 64;       // keys of a tile
constexpr int kLdThreads = 320;   // 4 softmax warps, four TMA warps, two MMA warps
constexpr int kLdMaxStages = 8;
constexpr int kLdParts = 5;       // barriers of a stage: pairs of chunks of the latent, the rotary chunk
constexpr int kLdChunk = kLdKeys * 128;  // 64 keys x 64 elements, 128-byte rows
constexpr int kLdAux = 1536;             // barriers, alpha, 1/l, schedule
constexpr int kLdSmemMax = 232448;
// A unit's prologue and epilogue (q load, output) in tiles, for the deal (2 to 4 are
// within 2% of one another, 1 and 6 slower).
constexpr int kLdUnitCost = 3;

struct LdParams {
    const char* base;  // the layer's region
    const char* ql;
    const char* qr;
    int64_t ql_token, ql_head, qr_token, qr_head;  // strides in elements
    char* out;
    float* lse;
    const int32_t* bt;
    const int32_t* lens;
    uint32_t* err;
    float4* ws_o;    // partial O: ld_part()
    float2* ws_ml;   // [2 * CTAs][64]: reference of the weights (log2 domain), sum
    int2* ws_unit;   // [units]: first and last CTA of a split unit, or (-1, -1)
    int bt_stride, B, T, H, groups, layer, num_pages, P, latent, rope, nch, stages, capacity, ctas;
    float scale_log2;
};

__device__ __forceinline__ int ld_len(const LdParams& p, int b) {
    const int len = __ldg(p.lens + b);
    return len < 0 || len > p.capacity ? 0 : len;
}

// 1 / l of a row.  A row that sees no key has l = 0 and gives zeros; one whose every
// score is -inf has l = 0 too, and 0 / 0 of the formula is NaN.
__device__ __forceinline__ float ld_inverse(float l, bool sees) {
    return l != 0.f ? 1.f / l : sees ? __uint_as_float(0x7fffffffu) : 0.f;
}

struct LdPiece {
    int b, g, t0, t1, tiles, len;
    int64_t unit_start;
    __device__ __forceinline__ bool whole() const { return t0 == 0 && t1 == tiles; }
};

// The pieces of one CTA's range [v, v1) of the laid-out units; a unit spans its
// tiles, then kLdUnitCost.
struct LdWalk {
    int64_t v, v1, unit_start;
    int b, g, len, tiles;

    __device__ __forceinline__ bool next(const LdParams& p, LdPiece& o) {
        while (v < v1) {
            const int64_t unit_end = unit_start + tiles + kLdUnitCost;
            const int64_t ve = v1 < unit_end ? v1 : unit_end;
            o.b = b;
            o.g = g;
            o.len = len;
            o.tiles = tiles;
            o.unit_start = unit_start;
            o.t0 = static_cast<int>(v - unit_start);
            o.t1 = static_cast<int>(ve - unit_start < tiles ? ve - unit_start : tiles);
            v = ve;
            if (v == unit_end) {
                unit_start = unit_end;
                if (++g == p.groups) {
                    g = 0;
                    ++b;
                    len = b < p.B ? ld_len(p, b) : 0;
                    tiles = (len + kLdKeys - 1) / kLdKeys;
                }
            }
            if (o.t0 < o.t1 || (o.t0 == 0 && o.tiles == 0)) return true;  // an empty unit: its rows are zeros
        }
        return false;
    }
    __device__ __forceinline__ bool next_real(const LdParams& p, LdPiece& o) {
        while (next(p, o))
            if (o.t0 < o.t1) return true;
        return false;
    }
};

// Partial O of a slot as [16 row quads][latent / 128][128 elements] of four rows
// each: what a thread reads from TMEM, stored and loaded 16 bytes at a time.
template <int LCH>
__device__ __forceinline__ int64_t ld_part(int slot, int quad, int mb, int d) {
    return ((static_cast<int64_t>(slot) * 16 + quad) * (LCH / 2) + mb) * 128 + d;
}

__device__ __forceinline__ void bar_softmax() { asm volatile("barrier.cta.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ bool bar_softmax_or(bool x) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, 1, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(static_cast<uint32_t>(x))
        : "memory");
    return r != 0;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}

// NaN in the output (or partial output) elements that a non-finite element of a key
// reaches: of the keys of the piece that only some tokens may see, in the rows that see
// them.  Called by the 128 softmax threads, behind the piece's output, when one of them
// cleared such an element.
template <typename T, int LCH>
__device__ __forceinline__ void ld_broken_keys(const LdParams& p, const LdPiece& c, int slot, int live) {
    bar_softmax();  // behind the stores of the other threads
    const int first = max(max(c.len - (p.T - 1), 0), c.t0 * kLdKeys), end = min(c.len, c.t1 * kLdKeys);
    const int64_t row0 = static_cast<int64_t>(c.b) * p.T * p.H + c.g * 64;
    constexpr uint32_t e = Elem<T>::kBf16 ? 0x7f80u : 0x7c00u;
#pragma unroll 1
    for (int key = first; key < end; ++key) {
        int page = __ldg(p.bt + static_cast<int64_t>(c.b) * p.bt_stride + key / p.P);
        if (page < 0 || page >= p.num_pages) page = 0;  // as the tile had it
        const uint16_t* x = reinterpret_cast<const uint16_t*>(p.base) +
                            (static_cast<int64_t>(page) * p.P + key % p.P) * (p.latent + p.rope);
        // rows from this one on see the key
        const int64_t from = (static_cast<int64_t>(key) - c.len + p.T) * p.H - c.g * 64;
#pragma unroll 1
        for (int d = threadIdx.x; d < LCH * 64; d += 128) {
            if ((__ldg(x + d) & e) != e) continue;
            for (int r = static_cast<int>(max(from, static_cast<int64_t>(0))); r < live; ++r) {
                if (c.whole()) reinterpret_cast<uint16_t*>(p.out)[(row0 + r) * (LCH * 64) + d] = 0x7fff;
                else reinterpret_cast<float*>(p.ws_o + ld_part<LCH>(slot, r >> 2, d >> 7, d & 127))[r & 3] = __uint_as_float(0x7fffffffu);
            }
        }
    }
}

template <typename T, int LCH>  // LCH: latent_dim / 64
__global__ void __launch_bounds__(kLdThreads, 1) latent_decode_kernel(const __grid_constant__ CUtensorMap tmap,
                                                                      const __grid_constant__ LdParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = smem_u32(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t stage_bytes = p.nch * kLdChunk;
    const uint32_t s_q = sbase + p.stages * stage_bytes, s_p = s_q + stage_bytes;
    uint8_t* aux = smem + (p.stages + 1) * stage_bytes + kLdChunk;
    uint64_t* bars = reinterpret_cast<uint64_t*>(aux);
    uint64_t* k_full = bars;                                // [stages][parts] a part of the tile landed
    uint64_t* k_empty = bars + kLdMaxStages * kLdParts;     // [stages][parts] its last product is done
    uint64_t* s_full = bars + 2 * kLdMaxStages * kLdParts;  // [2]
    uint64_t* p_full = s_full + 2;  // [2] S read, P written, O rescaled, last piece's O read
    uint64_t* pv_done = s_full + 4;
    uint64_t* q_full = s_full + 5;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_full + 6);
    float* alpha = reinterpret_cast<float*>(aux + 768);   // [64] rescale factors
    float* inv_l = reinterpret_cast<float*>(aux + 1024);  // [64]

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        for (int i = 0; i < p.stages * kLdParts; ++i) {
            mbar_init(smem_u32(&k_full[i]), 1);
            mbar_init(smem_u32(&k_empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&s_full[i]), 1);
            mbar_init(smem_u32(&p_full[i]), 4);
        }
        mbar_init(smem_u32(pv_done), 1);
        mbar_init(smem_u32(q_full), 4);
        mbar_fence_init();
    }
    // ---- the deal, by every warp for itself: the sequences' costs from the device's
    // lengths, their prefix sums, this CTA's range and the unit it starts in
    const int per = (p.B + 31) >> 5, b_lo = min(p.B, lane * per), b_hi = min(p.B, b_lo + per);
    int64_t mine = 0;
#pragma unroll 4
    for (int b = b_lo; b < b_hi; ++b)
        mine += static_cast<int64_t>(p.groups) * ((ld_len(p, b) + kLdKeys - 1) / kLdKeys + kLdUnitCost);
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += up;
    }
    const int64_t total = __shfl_sync(0xffffffffu, upto, 31);
    const LdDeal deal(total, gridDim.x);
    if (static_cast<int>(blockIdx.x) >= deal.n) return;  // the whole CTA: nothing allocated yet
    LdWalk walk0;
    walk0.v = deal.start(blockIdx.x);
    walk0.v1 = deal.start(blockIdx.x + 1);
    {
        const int src = __ffs(__ballot_sync(0xffffffffu, walk0.v < upto)) - 1;
        int64_t at = __shfl_sync(0xffffffffu, upto - mine, src);
        int b = src * per;
        for (;; ++b) {
            walk0.len = ld_len(p, b);
            walk0.tiles = (walk0.len + kLdKeys - 1) / kLdKeys;
            const int64_t c = static_cast<int64_t>(p.groups) * (walk0.tiles + kLdUnitCost);
            if (walk0.v < at + c) break;
            at += c;
        }
        const int span = walk0.tiles + kLdUnitCost;
        walk0.b = b;
        walk0.g = p.groups > 1 ? static_cast<int>((walk0.v - at) / span) : 0;
        walk0.unit_start = at + static_cast<int64_t>(walk0.g) * span;
    }
    const int rows = p.T * p.H, rope8 = p.rope >> 3, lat8 = LCH * 8;
    LdWalk w = walk0;  // every role walks the CTA's pieces for itself
    LdPiece c;
    // next piece with tiles; rows of empty units are written on the way
    auto advance = [&](LdPiece& o) -> bool {
        while (w.next(p, o)) {
            if (o.t0 < o.t1) return true;
            const int live = min(64, rows - o.g * 64);
            const int64_t row0 = static_cast<int64_t>(o.b) * rows + o.g * 64;
            uint4* dst = reinterpret_cast<uint4*>(p.out + 2 * row0 * p.latent);
            for (int i = threadIdx.x; i < live * lat8; i += 128) dst[i] = make_uint4(0, 0, 0, 0);
            if (p.lse && threadIdx.x < live) p.lse[row0 + threadIdx.x] = -INFINITY;
            if (threadIdx.x == 0) p.ws_unit[static_cast<int64_t>(o.b) * p.groups + o.g] = make_int2(-1, -1);
        }
        return false;
    };
    // 16 rows a warp, a row's 16-byte vectors across the lanes; one division per
    // piece, then (token, head) step along
    auto load_q = [&](const LdPiece& o) {
        int t = (o.g * 64 + warp * 16) / p.H, h = (o.g * 64 + warp * 16) % p.H;
        const char* ql = p.ql + 2 * ((static_cast<int64_t>(o.b) * p.T + t) * p.ql_token + h * p.ql_head) + lane * 16;
        const char* qr = p.qr + 2 * ((static_cast<int64_t>(o.b) * p.T + t) * p.qr_token + h * p.qr_head) + lane * 16;
        const int live = rows - o.g * 64 - warp * 16;  // rows of this warp that exist
#pragma unroll 4
        for (int k = 0; k < 16; ++k) {
            const bool on = k < live;
            const uint32_t dst = s_q + swz128(warp * 16 + k, lane & 7) + (lane >> 3) * kLdChunk;
#pragma unroll
            for (int i = 0; i < (LCH + 3) / 4; ++i)
                if (lane + 32 * i < LCH * 8) cp_async16(dst + i * 4 * kLdChunk, on ? ql + i * 512 : p.ql, on);
            if (lane < rope8)
                cp_async16(s_q + LCH * kLdChunk + swz128(warp * 16 + k, lane), on ? qr : p.qr, on);
            ql += 2 * p.ql_head;
            qr += 2 * p.qr_head;
            if (++h == p.H) {
                h = 0;
                ++t;
                ql += 2 * (p.ql_token - p.H * p.ql_head);
                qr += 2 * (p.qr_token - p.H * p.qr_head);
            }
        }
    };
    auto q_landed = [&]() {
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(q_full));
    };

    // The first queries are on their way before any tile is: behind the tiles of all
    // SMs they took 2 us longer to arrive.
    bool have = false;
    if (warp < 4) {
        have = advance(c);
        if (have) load_q(c);
    } else if (warp == 5) {
        tmem_alloc(smem_u32(tmem_slot), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 4 || (warp >= 7 && warp <= 5 + LCH / 2)) {
        const int g = warp == 4 ? 0 : warp - 6;
        // ------------------------------------------------------------ TMA producers
        // Warp g of latent / 128 brings part g of every tile (two chunks of 64 elements;
        // the first warp the rotary chunk too): a part of 16-token pages takes eight
        // copies, ~70 cycles each to issue, and all 36 of a tile from one warp took
        // longer than the tile (24 x 16k tokens: 116 us with one warp, 96 with several).
        int st = 0;
        uint32_t ph = 1;      // parity of the stage's release before this fill
        bool ok = true, filled = false;  // filled: every stage has been, releases to wait for
        if (lane == 0) prefetch_tmap(&tmap);
        const uint64_t pol = p.groups > 1 ? l2_evict_last_policy() : l2_evict_first_policy();
        const int ppt = kLdKeys / p.P;  // pages of a full tile
        const int i = lane >> 1;  // lane: page i of the tile, chunk lane % 2 of the part
        while (ok && w.next_real(p, c)) {
            const int32_t* row = p.bt + static_cast<int64_t>(c.b) * p.bt_stride;
            const int npages = (c.len + p.P - 1) / p.P;
            // block-table entries win .. win+63, two a lane
            int win = c.t0 * ppt;
            auto entry = [&](int k) {
                int e = k < npages ? __ldg(row + k) : 0;
                if (e < 0 || e >= p.num_pages) {
                    atomicOr(p.err, VK_ERR_PAGE_ID);
                    e = 0;
                }
                return e;
            };
            int e0 = entry(win + lane), e1 = entry(win + 32 + lane);
            for (int t = c.t0; t < c.t1 && ok; ++t) {
                const int first = t * ppt, cnt = min(ppt, npages - first);
                if (first + cnt > win + 32) {  // tiles do not straddle windows: 32 is a multiple of ppt
                    win += 32;
                    e0 = e1;
                    e1 = entry(win + 32 + lane);
                }
                const int page = __shfl_sync(0xffffffffu, e0, (first - win + min(i, cnt - 1)) & 31);
                const int y = (p.layer * p.num_pages + page) * p.P;
                auto bring = [&](int part, int chunks) {
                    if (filled) ok = ok && wait_all(smem_u32(&k_empty[st * kLdParts + part]), ph, p.err);
                    if (!ok) return;
                    const uint32_t bar = smem_u32(&k_full[st * kLdParts + part]);
                    if (lane == 0) mbar_expect_tx(bar, chunks * cnt * p.P * 128);
                    const int ch = 2 * part + (lane & 1);
                    if (i < cnt && (lane & 1) < chunks)
                        tma_load_2d(sbase + st * stage_bytes + ch * kLdChunk + i * p.P * 128, &tmap, ch * 64, y, bar, pol);
                };
                bring(g, 2);
                if (g == 0) bring(LCH / 2, 1);
                if (++st == p.stages) {
                    st = 0;
                    ph ^= 1;
                    filled = true;
                }
            }
        }
        if (!ok)  // a wait gave up: no copy of this warp may land behind the CTA's end (bounded as well)
            for (int k = 0; k < p.stages; ++k)
                if (k < st || filled) {
                    const uint32_t par = k < st ? ph ^ 1 : ph;
                    mbar_wait(smem_u32(&k_full[k * kLdParts + g]), par, p.err);
                    if (g == 0) mbar_wait(smem_u32(&k_full[k * kLdParts + LCH / 2]), par, p.err);
                }
    } else if (warp == 5) {
        // ------------------------------------------------------------ S = Q K^T
        int si = 0, piece = 0, st = 0, ph = 0;
        bool ok = true;
        constexpr uint32_t id_s = idesc_16(Elem<T>::kBf16, 64, 64, 0, 0);
        const uint64_t dk0 = umma_desc_sw128(sbase, 16, 1024);
        const uint32_t k_hi = static_cast<uint32_t>(dk0 >> 32), k_lo = static_cast<uint32_t>(dk0);
        const uint32_t q_lo = k_lo + ((s_q - sbase) >> 4);
        const int rsteps = p.rope >> 4;
        if (elect_lane()) {
            while (ok && w.next_real(p, c)) {
                ok = mbar_wait(smem_u32(q_full), piece & 1, p.err);
                ++piece;
                for (int t = c.t0; t < c.t1 && ok; ++t, ++si) {
                    if (si >= 2) ok = mbar_wait(smem_u32(&p_full[si & 1]), ((si >> 1) - 1) & 1, p.err);  // S's buffer has been read
                    const uint32_t kl = k_lo + st * (stage_bytes >> 4);
                    const uint32_t d = tmem + 256 + (si & 1) * 64;
#pragma unroll
                    for (int g = 0; g < LCH / 2; ++g) {
                        ok = ok && mbar_wait(smem_u32(&k_full[st * kLdParts + g]), ph, p.err);
                        if (ok) {
                            tc_fence_after();
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                const uint32_t off = ((2 * g + (k >> 2)) * kLdChunk + (k & 3) * 32) >> 4;
                                umma_ss_lo(d, q_lo + off, k_hi, kl + off, k_hi, id_s, (g | k) != 0);
                            }
                        }
                    }
                    ok = ok && mbar_wait(smem_u32(&k_full[st * kLdParts + LCH / 2]), ph, p.err);
                    if (ok) {
                        tc_fence_after();
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks) {
                            const uint32_t off = (LCH * kLdChunk + ks * 32) >> 4;
                            if (ks < rsteps) umma_ss_lo(d, q_lo + off, k_hi, kl + off, k_hi, id_s, 1);
                        }
                        umma_commit(smem_u32(&s_full[si & 1]));
                        umma_commit(smem_u32(&k_empty[st * kLdParts + LCH / 2]));
                    }
                    if (++st == p.stages) {
                        st = 0;
                        ph ^= 1;
                    }
                }
            }
        }
    } else if (warp == 6) {
        // ------------------------------------------------------------ O^T += V^T P^T
        int pi = 0, st = 0, ph = 0;
        bool ok = true;
        constexpr uint32_t id_pv = idesc_16(Elem<T>::kBf16, 128, 64, 1, 0);
        const uint64_t dv0 = umma_desc_sw128(sbase, kLdChunk, 1024), dp0 = umma_desc_sw128(s_p, 16, 1024);
        const uint32_t v_hi = static_cast<uint32_t>(dv0 >> 32), v_lo = static_cast<uint32_t>(dv0);
        const uint32_t p_hi = static_cast<uint32_t>(dp0 >> 32), p_lo = static_cast<uint32_t>(dp0);
        if (elect_lane()) {
            while (ok && w.next_real(p, c)) {
                for (int t = c.t0; t < c.t1 && ok; ++t, ++pi) {
#pragma unroll
                    for (int g = 0; g < LCH / 2; ++g)  // long complete: S has read them
                        ok = ok && mbar_wait(smem_u32(&k_full[st * kLdParts + g]), ph, p.err);
                    ok = ok && mbar_wait(smem_u32(&p_full[pi & 1]), (pi >> 1) & 1, p.err);
                    if (ok) {
                        tc_fence_after();
                        const uint32_t vl = v_lo + st * (stage_bytes >> 4);
                        const uint32_t acc = t != c.t0;
#pragma unroll
                        for (int mb = 0; mb < LCH / 2; ++mb) {
#pragma unroll
                            for (int ks = 0; ks < kLdKeys / 16; ++ks)
                                umma_ss_lo(tmem + mb * 64, vl + ((mb * 2 * kLdChunk + ks * 2048) >> 4), v_hi, p_lo + ks * 2, p_hi, id_pv,
                                           ks ? 1 : acc);
                            umma_commit(smem_u32(&k_empty[st * kLdParts + mb]));
                        }
                        umma_commit(smem_u32(pv_done));
                    }
                    if (++st == p.stages) {
                        st = 0;
                        ph ^= 1;
                    }
                }
            }
        }
    } else if (warp < 4) {
        // ------------------------------------------------------------ softmax and output
        LdPiece nx;
        // this thread's rows of the group: r and r + 8; its keys of a tile: 8j + kq and the next
        const int r = warp * 16 + (lane >> 2), kq = 2 * (lane & 3);
        const uint32_t lane_base = tmem + (static_cast<uint32_t>(warp * 32) << 16);
        if (blockIdx.x == 0)
            for (int b = threadIdx.x; b < p.B; b += 128)
                if (__ldg(p.lens + b) != ld_len(p, b)) atomicOr(p.err, VK_ERR_SEQ_LEN);
        int it = 0, st = 0;
        bool fail = false;
        if (have) q_landed();
        while (have) {
            float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // log2 domain; l: this thread's keys
            int lim[2];  // keys that the row sees
            bool live_row[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int row = c.g * 64 + r + 8 * u;
                live_row[u] = row < rows;
                lim[u] = c.len - (p.T - 1 - (live_row[u] ? row / p.H : p.T - 1));
            }
            const int lim0 = c.len - (p.T - 1);  // keys that every token sees
            bool broken = false;                 // this thread cleared a non-finite element
            for (int t = c.t0; t < c.t1; ++t, ++it) {
                const int key0 = t * kLdKeys;
                fail = !wait_all(smem_u32(&s_full[it & 1]), (it >> 1) & 1, p.err) || fail;
                tc_fence_after();
                float a[32];
                tmem_ld_16x64(lane_base + 256 + (it & 1) * 64, a);
                tmem_wait_ld();
                const bool tail = key0 + kLdKeys > lim0;
                if (tail) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (key0 + (i >> 2) * 8 + kq + (i & 1) >= lim[(i >> 1) & 1]) a[i] = -INFINITY;
                }
                float al[2];
                bool resc = false;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        x0 = max3(x0, a[4 * j + 2 * u], a[4 * j + 2 * u + 1]);
                        x1 = max3(x1, a[4 * j + 4 + 2 * u], a[4 * j + 4 + 2 * u + 1]);
                    }
                    float top = fmaxf(x0, x1) * p.scale_log2;
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    al[u] = 1.f;
                    if (top > m[u] + (Weights<T>::kMargin + Weights<T>::kLag) || m[u] == -INFINITY) {
                        const float mn = fmaxf(m[u], top - Weights<T>::kMargin);
                        al[u] = m[u] == -INFINITY ? 0.f : ex2(m[u] - mn);
                        m[u] = mn;
                        resc = resc || live_row[u];
                    }
                }
                // before the unit's first product O holds nothing to rescale
                resc = resc && t > c.t0;
                const bool any = bar_softmax_or(resc || fail);
                if (any && bar_softmax_or(fail)) goto done;
                uint32_t pk[16];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float mneg = m[u] == -INFINITY ? 0.f : -m[u];
                    float sum[2] = {0.f, 0.f};
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float e0 = ex2(fmaf(a[4 * j + 2 * u], p.scale_log2, mneg));
                        const float e1 = ex2(fmaf(a[4 * j + 2 * u + 1], p.scale_log2, mneg));
                        sum[j & 1] += e0 + e1;
                        pk[2 * j + u] = Elem<T>::pack(e0, e1);
                    }
                    l[u] = l[u] * al[u] + (sum[0] + sum[1]);
                }
                if (tail) {  // V rows: zeros behind the sequence, finite where some token may not look
                    const int lo = max(0, lim0 - key0), nrow = kLdKeys - lo;
                    for (int i = threadIdx.x; i < nrow * lat8; i += 128) {
                        const int kr = lo + i / lat8, v = i % lat8;
                        const uint32_t addr = sbase + st * stage_bytes + (v >> 3) * kLdChunk + swz128(kr, v & 7);
                        uint4 x = make_uint4(0, 0, 0, 0);
                        if (key0 + kr < c.len) {
                            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                         : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                                         : "r"(addr));
                            const uint4 y = x;
                            x = make_uint4(finite_word<T>(x.x), finite_word<T>(x.y), finite_word<T>(x.z), finite_word<T>(x.w));
                            broken = broken || ((x.x ^ y.x) | (x.y ^ y.y) | (x.z ^ y.z) | (x.w ^ y.w));
                        }
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w)
                                     : "memory");
                    }
                }
                // P's buffer is free, and O complete, once the previous tile's product is done
                if (it > 0) fail = !wait_all(smem_u32(pv_done), (it - 1) & 1, p.err) || fail;
                if (any) {
                    tc_fence_after();
                    if ((lane & 3) == 0) {
                        alpha[r] = al[0];
                        alpha[r + 8] = al[1];
                    }
                    bar_softmax();
                    for (int col = 0; col < (LCH * 32); col += 32) {
                        float o[32];
                        tmem_ld32(lane_base + col, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] *= alpha[(col & 32) + i];
                        tmem_st32(lane_base + col, o);
                    }
                    tmem_wait_st();
                }
                // P: 8x8 blocks (rows +0 / +8, key blocks j and j + 1); lane i gives the address
                // of row i % 8 of block i / 8
#pragma unroll
                for (int j = 0; j < 8; j += 2)
                    stsm_x4(s_p + swz128(warp * 16 + (lane & 15), j + (lane >> 4)), pk[2 * j], pk[2 * j + 1], pk[2 * j + 2],
                            pk[2 * j + 3]);
                fence_async_smem();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&p_full[it & 1]));
                if (++st == p.stages) st = 0;
            }
            // the last S of this piece has been read: the next piece's queries may land
            have = advance(nx);
            if (have) {
                load_q(nx);
                q_landed();
            }
            const bool whole = c.whole();
            const int64_t row0 = static_cast<int64_t>(c.b) * rows + c.g * 64;
            const int slot = 2 * blockIdx.x + (c.t0 == 0 ? 1 : 0);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
                l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
                if ((lane & 3) == 0) {
                    const int rr = r + 8 * u;
                    inv_l[rr] = ld_inverse(l[u], lim[u] > 0);
                    if (!whole) p.ws_ml[slot * 64 + rr] = make_float2(m[u], l[u]);
                    else if (p.lse && live_row[u])
                        p.lse[row0 + rr] = l[u] == 0.f ? -INFINITY : Weights<T>::log2_sum(m[u], l[u]) * 0.69314718055994531f;
                }
            }
            if (threadIdx.x == 0 && c.t0 == 0) {
                int2 u = make_int2(-1, -1);
                if (!whole)
                    u = make_int2(blockIdx.x, deal.owner(c.unit_start + c.tiles - 1));
                p.ws_unit[static_cast<int64_t>(c.b) * p.groups + c.g] = u;
            }
            fail = !wait_all(smem_u32(pv_done), (it - 1) & 1, p.err) || fail;
            const bool odd = bar_softmax_or(fail || broken);
            if (odd && bar_softmax_or(fail)) goto done;
            tc_fence_after();
            const int live = min(64, rows - c.g * 64);
            // rolled loops: a CTA runs this once or twice, and unrolled code would arrive
            // through cold instruction fetches
#pragma unroll 1
            for (int k = 0; k < LCH; ++k) {
                const int mb = k >> 1, hc = k & 1;  // 128 latent elements, 32 rows
                if (hc * 32 >= live) continue;
                if (whole) {
                    // O^T fragments, scaled, transposed on the way to shared memory (P's
                    // buffer: [32 rows][128 elements], 16-byte chunks XOR row % 8)
#pragma unroll 1
                    for (int half = 0; half < 2; ++half) {
                        float o[16];
                        tmem_ld_16x32(lane_base + (static_cast<uint32_t>(half * 16) << 16) + mb * 64 + hc * 32, o);
                        tmem_wait_ld();
                        uint32_t w2[8];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float2 i2 = *reinterpret_cast<const float2*>(inv_l + hc * 32 + 8 * j + kq);
#pragma unroll
                            for (int u = 0; u < 2; ++u)
                                w2[2 * j + u] = Elem<T>::pack(i2.x == 0.f ? 0.f : o[4 * j + 2 * u] * i2.x,
                                                              i2.y == 0.f ? 0.f : o[4 * j + 2 * u + 1] * i2.y);
                        }
#pragma unroll
                        for (int j = 0; j < 4; j += 2) {
                            const int rr = 8 * (j + (lane >> 4)) + (lane & 7), ch = warp * 4 + half * 2 + ((lane >> 3) & 1);
                            stsm_x4_t(s_p + rr * 256 + ((ch ^ (rr & 7)) << 4), w2[2 * j], w2[2 * j + 1], w2[2 * j + 2], w2[2 * j + 3]);
                        }
                    }
                    bar_softmax();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int rr = (threadIdx.x >> 4) + 8 * i, ch = threadIdx.x & 15;
                        uint4 x;
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                     : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                                     : "r"(s_p + rr * 256 + ((ch ^ (rr & 7)) << 4)));
                        if (hc * 32 + rr < live)
                            *reinterpret_cast<uint4*>(p.out + 2 * ((row0 + hc * 32 + rr) * (LCH * 64) + mb * 128) + ch * 16) = x;
                    }
                    bar_softmax();
                } else {
                    // four rows of one latent element a 16-byte store (ld_part)
                    float o[32];
                    tmem_ld32(lane_base + mb * 64 + hc * 32, o);
                    tmem_wait_ld();
                    float4* dst = p.ws_o + ld_part<LCH>(slot, hc * 8, mb, warp * 32 + lane);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (hc * 32 + 4 * i < live)
                            dst[i * (LCH / 2) * 128] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                }
            }
            tc_fence_before();
            if (odd) ld_broken_keys<T, LCH>(p, c, slot, live);
            c = nx;
        }
    done:;
    }
    __syncthreads();
    if (warp == 5) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Joins the partials of units that several CTAs share.  A thread has one latent
// element (of each of MBS blocks of 128) of four rows; KG groups of D threads take
// the pieces in turn and meet in shared memory.  Bound by latency: the pieces'
// weights come from one round of loads, a piece per thread, while the first
// partials are already on their way.  The order of the sums is fixed by the
// pieces, so results repeat bit for bit.
//   many units, few pieces each: MBS = latent / 128, D 128, KG 1 (one wave)
//   few units, up to a piece per SM: MBS 1, D 64, KG 16 (more SMs, short loops)
constexpr int kLdMaxPieces = 256;  // CTAs of a launch
template <typename T, int LCH, int MBS, int D, int KG>
__global__ void __launch_bounds__(D * KG) latent_merge_kernel(const __grid_constant__ LdParams p) {
    __shared__ float4 part[KG > 1 ? KG : 1][KG > 1 ? D : 1];
    __shared__ float4 wts[kLdMaxPieces];
    __shared__ float4 m_warp[kLdMaxPieces / 32], l_warp[kLdMaxPieces / 32];
    constexpr int kSplit = LCH * 64 / (MBS * 128) * (128 / D);  // blocks per row quad
    const int lane = threadIdx.x & 31, kg = threadIdx.x / D;
    const int64_t unit = blockIdx.x;
    const int quad = blockIdx.y / kSplit, e0 = blockIdx.y % kSplit * D + threadIdx.x % D;  // element in its blocks
    const int b = static_cast<int>(unit / p.groups), g = static_cast<int>(unit % p.groups);
    const int rows = p.T * p.H, row_in = g * 64 + quad * 4;
    if (row_in >= rows) return;
    const int len = ld_len(p, b);  // an input of the launch before: no need to wait for it
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int2 u = p.ws_unit[unit];
    if (!ld_joinable(u.x, u.y, p.ctas)) return;
    // piece i of CTA u.x + i: the first tile's piece in the odd slot, the others in even ones
    auto slot_of = [&](int i) { return 2 * (u.x + i) + (i == 0 ? 1 : 0); };
    const int pieces = u.y - u.x + 1;
    constexpr int kAhead = KG > 1 ? 5 : 16 / MBS;  // pieces in flight
    float4 o[kAhead][MBS];
    auto fetch = [&](int i0) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (i0 + j * KG < pieces) {
#pragma unroll
                for (int k = 0; k < MBS; ++k)
                    o[j][k] = __ldcs(p.ws_o + ld_part<LCH>(slot_of(i0 + j * KG), quad, k + (MBS == 1 ? e0 >> 7 : 0), e0 & 127));
            }
    };
    fetch(kg);
    // Weights: a thread per piece, the block's maxima and sums through the warps.
    constexpr int kThreads = D * KG, kPer = kLdMaxPieces > kThreads ? kLdMaxPieces / kThreads : 1;
    const int warp = threadIdx.x >> 5, used = min(kThreads / 32, (pieces + 31) >> 5);  // warps that hold pieces
    float4 x[kPer], y[kPer], m = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY), l = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int i = threadIdx.x + j * kThreads;
        x[j] = y[j] = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);  // (m, l) of rows 0, 1 and 2, 3
        if (i < pieces) {
            const float4* ml = reinterpret_cast<const float4*>(p.ws_ml + slot_of(i) * 64 + quad * 4);
            x[j] = ml[0];
            y[j] = ml[1];
        }
        m = make_float4(fmaxf(m.x, x[j].x), fmaxf(m.y, x[j].z), fmaxf(m.z, y[j].x), fmaxf(m.w, y[j].z));
    }
    if (warp < used) {
#pragma unroll
        for (int s = 16; s > 0; s >>= 1)
            m = make_float4(fmaxf(m.x, __shfl_xor_sync(0xffffffffu, m.x, s)), fmaxf(m.y, __shfl_xor_sync(0xffffffffu, m.y, s)),
                            fmaxf(m.z, __shfl_xor_sync(0xffffffffu, m.z, s)), fmaxf(m.w, __shfl_xor_sync(0xffffffffu, m.w, s)));
        if (lane == 0) m_warp[warp] = m;
    }
    __syncthreads();
    m = m_warp[0];
    for (int k = 1; k < used; ++k)
        m = make_float4(fmaxf(m.x, m_warp[k].x), fmaxf(m.y, m_warp[k].y), fmaxf(m.z, m_warp[k].z), fmaxf(m.w, m_warp[k].w));
    if (warp < used) {
        auto weight = [](float mi, float mm) { return ex2(mi - (mm == -INFINITY ? 0.f : mm)); };
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int i = threadIdx.x + j * kThreads;
            // a piece whose keys a row may not see has weight, O and l of zero
            const float4 f = make_float4(weight(x[j].x, m.x), weight(x[j].z, m.y), weight(y[j].x, m.z), weight(y[j].z, m.w));
            if (i < pieces) {
                wts[i] = f;
                l = make_float4(fmaf(f.x, x[j].y, l.x), fmaf(f.y, x[j].w, l.y), fmaf(f.z, y[j].y, l.z), fmaf(f.w, y[j].w, l.w));
            }
        }
#pragma unroll
        for (int s = 16; s > 0; s >>= 1)
            l = make_float4(l.x + __shfl_xor_sync(0xffffffffu, l.x, s), l.y + __shfl_xor_sync(0xffffffffu, l.y, s),
                            l.z + __shfl_xor_sync(0xffffffffu, l.z, s), l.w + __shfl_xor_sync(0xffffffffu, l.w, s));
        if (lane == 0) l_warp[warp] = l;
    }
    __syncthreads();
    l = l_warp[0];
    for (int k = 1; k < used; ++k) l = make_float4(l.x + l_warp[k].x, l.y + l_warp[k].y, l.z + l_warp[k].z, l.w + l_warp[k].w);
    float4 acc[MBS];
#pragma unroll
    for (int k = 0; k < MBS; ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = kg; i0 < pieces; i0 += kAhead * KG) {
        if (i0 != kg) fetch(i0);
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (i0 + j * KG < pieces) {
                const float4 f = wts[i0 + j * KG];
#pragma unroll
                for (int k = 0; k < MBS; ++k)
                    acc[k] = make_float4(fmaf(f.x, o[j][k].x, acc[k].x), fmaf(f.y, o[j][k].y, acc[k].y),
                                         fmaf(f.z, o[j][k].z, acc[k].z), fmaf(f.w, o[j][k].w, acc[k].w));
            }
    }
    if constexpr (KG > 1) {
        part[kg][threadIdx.x % D] = acc[0];
        __syncthreads();
        if (kg) return;
#pragma unroll
        for (int k = 1; k < KG; ++k) {
            const float4 a = part[k][threadIdx.x];
            acc[0] = make_float4(acc[0].x + a.x, acc[0].y + a.y, acc[0].z + a.z, acc[0].w + a.w);
        }
    }
    const int64_t row = static_cast<int64_t>(b) * rows + row_in;
    const float lv[4] = {l.x, l.y, l.z, l.w}, mv[4] = {m.x, m.y, m.z, m.w};
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if (row_in + r >= rows) break;
        const float inv = ld_inverse(lv[r], len - (p.T - 1 - (row_in + r) / p.H) > 0);
#pragma unroll
        for (int k = 0; k < MBS; ++k) {
            const float a = r == 0 ? acc[k].x : r == 1 ? acc[k].y : r == 2 ? acc[k].z : acc[k].w;
            reinterpret_cast<T*>(p.out)[(row + r) * (LCH * 64) + k * 128 + e0] = Elem<T>::down(inv == 0.f ? 0.f : a * inv);
        }
        if (p.lse && blockIdx.y % kSplit == 0 && threadIdx.x == 0)
            p.lse[row + r] = lv[r] == 0.f ? -INFINITY : Weights<T>::log2_sum(mv[r], lv[r]) * 0.69314718055994531f;
    }
}

static size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

template <typename T, int LCH>
static vk_status launch_latent_decode(vk_pool* pool, const LdParams& p, cudaStream_t st) {
    static std::atomic<uint64_t> attr_set{0};  // a bit per device; host threads may call at once
    const uint64_t bit = 1ull << (pool->device & 63);
    const size_t smem = static_cast<size_t>(p.stages + 1) * p.nch * kLdChunk + kLdChunk + kLdAux + 1024;
    cudaError_t e = cudaSuccess;
    if (!(attr_set.load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(latent_decode_kernel<T, LCH>, cudaFuncAttributeMaxDynamicSharedMemorySize, kLdSmemMax);
        if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(latent_decode)");
        attr_set.fetch_or(bit, std::memory_order_release);
    }
    latent_decode_kernel<T, LCH><<<p.ctas, kLdThreads, smem, st>>>(pool->tmap16, p);
    e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "latent_decode_kernel launch");
    const int64_t units = static_cast<int64_t>(p.B) * p.groups;
    const int quads = (min(64, p.T * p.H) + 3) / 4;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (units * quads <= pool->num_sms / 2) {
        cfg.gridDim = dim3(static_cast<unsigned>(units), static_cast<unsigned>(quads * LCH));
        cfg.blockDim = dim3(1024);
        e = cudaLaunchKernelEx(&cfg, latent_merge_kernel<T, LCH, 1, 64, 16>, p);
    } else {
        cfg.gridDim = dim3(static_cast<unsigned>(units), static_cast<unsigned>(quads));
        cfg.blockDim = dim3(128);
        e = cudaLaunchKernelEx(&cfg, latent_merge_kernel<T, LCH, LCH / 2, 128, 1>, p);
    }
    return e == cudaSuccess ? VK_OK : cuda_fail(e, "latent_merge_kernel launch");
}

template <typename T>
static vk_status launch_latent_decode(vk_pool* pool, const LdParams& p, cudaStream_t st) {
    switch (pool->latent_dim) {
        case 512: return launch_latent_decode<T, 8>(pool, p, st);
        case 384: return launch_latent_decode<T, 6>(pool, p, st);
        case 256: return launch_latent_decode<T, 4>(pool, p, st);
        default: return launch_latent_decode<T, 2>(pool, p, st);
    }
}

}  // namespace vk

using namespace vk;

extern "C" size_t vk_latent_decode_workspace_size(const vk_pool* pool, int32_t batch, int32_t tokens_per_seq,
                                                  int32_t num_heads) {
    if (!pool || !is_latent(pool) || batch <= 0 || tokens_per_seq <= 0 || num_heads <= 0) return 0;
    const int64_t rows = static_cast<int64_t>(tokens_per_seq) * num_heads, units = batch * ((rows + 63) / 64);
    if (rows > (1 << 20) || units > (1 << 24)) return 0;
    const size_t slots = 2 * static_cast<size_t>(pool->num_sms);
    return align256(slots * 64 * pool->latent_dim * 4) + align256(slots * 64 * 8) + align256(static_cast<size_t>(units) * 8);
}

extern "C" vk_status vk_latent_decode(vk_pool* pool, int32_t layer, const void* q_latent, int64_t ql_token_stride,
                                      int64_t ql_head_stride, const void* q_rope, int64_t qr_token_stride,
                                      int64_t qr_head_stride, void* out, float* lse, const int32_t* block_tables,
                                      int32_t bt_stride, const int32_t* seq_lens, int32_t batch, int32_t tokens_per_seq,
                                      int32_t num_heads, float scale, void* workspace, size_t workspace_bytes, void* stream) {
    if (!pool) return fail(VK_INVALID_ARG, "pool is NULL");
    if (!is_latent(pool)) return fail(VK_UNSUPPORTED, "latent decode needs a latent pool");
    if (layer < 0 || layer >= pool->cfg.num_layers) return fail(VK_INVALID_ARG, "layer out of range");
    if (batch < 0 || tokens_per_seq < 0 || num_heads <= 0 || bt_stride <= 0) return fail(VK_INVALID_ARG, "bad batch/tokens/heads/bt_stride");
    if (!(scale > 0.f) || scale > 3.0e38f) return fail(VK_INVALID_ARG, "scale must be > 0 and finite");
    if (batch == 0 || tokens_per_seq == 0) return VK_OK;
    if (!q_latent || !q_rope || !out || !block_tables || !seq_lens) return fail(VK_INVALID_ARG, "NULL array");
    if (((reinterpret_cast<uintptr_t>(q_latent) | reinterpret_cast<uintptr_t>(q_rope) | reinterpret_cast<uintptr_t>(out)) & 15) ||
        ql_token_stride % 8 || ql_head_stride % 8 || qr_token_stride % 8 || qr_head_stride % 8)
        return fail(VK_INVALID_ARG, "q_latent, q_rope and out must be 16-byte aligned, strides multiples of 8");
    const size_t need = vk_latent_decode_workspace_size(pool, batch, tokens_per_seq, num_heads);
    if (need == 0) return fail(VK_INVALID_ARG, "too many rows: tokens_per_seq * num_heads <= 2^20, batch * ceil(rows/64) <= 2^24");
    if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15))
        return fail(VK_INVALID_ARG, "workspace missing, too small or not 16-byte aligned");
    LdParams p;
    p.base = pool->base + static_cast<uint64_t>(layer) * pool->seg_stride;
    p.ql = static_cast<const char*>(q_latent);
    p.qr = static_cast<const char*>(q_rope);
    p.ql_token = ql_token_stride;
    p.ql_head = ql_head_stride;
    p.qr_token = qr_token_stride;
    p.qr_head = qr_head_stride;
    p.out = static_cast<char*>(out);
    p.lse = lse;
    p.bt = block_tables;
    p.lens = seq_lens;
    p.err = pool->d_err;
    p.bt_stride = bt_stride;
    p.B = batch;
    p.T = tokens_per_seq;
    p.H = num_heads;
    p.groups = (tokens_per_seq * num_heads + 63) / 64;
    p.layer = layer;
    p.num_pages = pool->num_pages;
    p.P = pool->cfg.page_tokens;
    p.ctas = min(pool->num_sms, kLdMaxPieces);
    const int64_t capacity = static_cast<int64_t>(bt_stride) * p.P;
    p.capacity = static_cast<int>(capacity < 0x7fffff00 ? capacity : 0x7fffff00);  // (rounded up to tiles in int32)
    p.latent = pool->latent_dim;
    p.rope = pool->rope_dim;
    p.nch = p.latent / 64 + 1;
    const int stage = p.nch * kLdChunk;
    p.stages = (kLdSmemMax - 1024 - kLdAux - kLdChunk - stage) / stage;  // 2, 2, 4, 8 at 512, 384, 256, 128
    if (p.stages > kLdMaxStages) p.stages = kLdMaxStages;
    p.scale_log2 = scale * 1.4426950408889634f;
    const size_t slots = 2 * static_cast<size_t>(pool->num_sms);
    char* ws = static_cast<char*>(workspace);
    p.ws_o = reinterpret_cast<float4*>(ws);
    ws += align256(slots * 64 * p.latent * 4);
    p.ws_ml = reinterpret_cast<float2*>(ws);
    ws += align256(slots * 64 * 8);
    p.ws_unit = reinterpret_cast<int2*>(ws);
    DeviceGuard g(pool->device);
    return pool->kv_format == VK_KV_LATENT_BF16 ? launch_latent_decode<__nv_bfloat16>(pool, p, as_stream(stream))
                                                : launch_latent_decode<__half>(pool, p, as_stream(stream));
}
