// Append to a latent pool (vk_latent_append): root-mean-square norm of the
// latent, rotation of the shared key part, and the row written through the
// block table.
//
//   row = [ c / sqrt(mean(c^2) + eps) * w  |  R(pos) k ]
//
// Floor: 2 * (latent + rope) * 2 bytes a token.  One warp per token: the row stays in
// registers between the sum of squares (fp32, one shuffle tree) and the scaled
// store, so it is read once and written once, the latent in 16-byte vectors.
// Bound by latency: 2.6 us for a decode step; 17.6k tokens of 512 + 64 take 11.3 us,
// 3.6 TB/s (the memory alone 6.3): ~20% of the time is the launch, the rest three
// dependent loads a warp (sequence and position, page; the row meanwhile).  At 32
// registers (one spilled) all 64 warps fit an SM: 11.3 us against 11.8 at 44.  Blocks of
// 8 and 16 warps measured 12.0 and 12.2 us, two and four rows a warp 14.0 and 14.6
// where one took 13.6.
#include "vk_internal.h"
#include "vk_rotary.cuh"

namespace vk {

struct LatentAppendParams {
    char* base;            // the layer's region
    const char* latent;
    const char* k_rope;
    const char* weight;    // NULL: no norm
    int64_t latent_stride, rope_stride;  // elements
    const int32_t* bt;
    const int32_t* pos;
    const int32_t* offsets;
    uint32_t* err;
    int bt_stride, B, tokens, latent_dim, rope_dim, P_log2, num_pages;
    float eps, inv_dim;
};

constexpr int kLaWarps = 4;

// The sequence of a row, the last b with offsets[b] <= row, and that offset, by a
// 32-ary search of the warp (one round of loads for up to 32 sequences); -1 behind
// the last sequence.
__device__ __forceinline__ int sequence_of(const int32_t* offsets, const int32_t* positions, int B, int row, int lane, int* first,
                                           int* position) {
    const int end = __ldg(offsets + B);
    int lo = 0, n = B, at = 0, pos = 0;
    do {
        const int step = (n + 31) >> 5;
        const int v = lane * step < n ? __ldg(offsets + lo + lane * step) : 0;
        const int pv = lane * step < n ? __ldg(positions + lo + lane * step) : 0;  // beside it: one load less in the chain
        const unsigned le = __ballot_sync(0xffffffffu, lane * step < n && v <= row);
        const int k = le ? 31 - __clz(le) : 0;
        at = __shfl_sync(0xffffffffu, v, k);
        pos = __shfl_sync(0xffffffffu, pv, k);
        lo += k * step;
        n = min(step, n - k * step);
    } while (n > 1);
    *first = at;
    *position = pos;
    return row < end ? lo : -1;
}

template <typename T>
__global__ void __launch_bounds__(kLaWarps * 32, 64 / kLaWarps) latent_append_kernel(
    const __grid_constant__ RotaryTable rot, const __grid_constant__ LatentAppendParams p) {
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kLaWarps + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    // the turns of the pairs, read from the kernel's parameters once a block: a warp's 32
    // addresses in the constant cache are served one after another (a read per warp: 13.0 us)
    __shared__ uint64_t turn[32];
    if (threadIdx.x < rot.pairs) turn[threadIdx.x] = rot.turn[threadIdx.x];
    __syncthreads();
    if (row >= p.tokens) return;
    // the row's loads go out first; the lookups (three dependent loads: sequence,
    // position, page) run behind them
    const int vecs = p.latent_dim >> 3;  // 16-byte vectors of the latent: 16..64, two a lane at most
    // of the rotary part a lane has one pair (rope_dim <= 64): elements 2i and 2i+1, or
    // i and i + rope_dim/2 in the half layout
    const int pairs = p.rope_dim >> 1;
    const bool half = rot.pairs && rot.half;
    const uint4* src = reinterpret_cast<const uint4*>(p.latent + 2 * (row * p.latent_stride));
    const char* ksrc = p.k_rope + 2 * (row * p.rope_stride);
    uint4 c[2], wv[2];
    uint32_t k = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const bool in = lane + 32 * i < vecs;
        c[i] = in ? __ldg(src + lane + 32 * i) : make_uint4(0, 0, 0, 0);
        wv[i] = in && p.weight ? __ldg(reinterpret_cast<const uint4*>(p.weight) + lane + 32 * i) : make_uint4(0, 0, 0, 0);
    }
    if (lane < pairs) {
        if (half)
            k = __ldg(reinterpret_cast<const uint16_t*>(ksrc) + lane) |
                static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t*>(ksrc) + lane + pairs)) << 16;
        else
            k = __ldg(reinterpret_cast<const uint32_t*>(ksrc) + lane);
    }
    int b, first, start;
    if (p.offsets) {
        b = sequence_of(p.offsets, p.pos, p.B, static_cast<int>(row), lane, &first, &start);
        if (b < 0 || (b == 0 && row < first)) return;  // a row of no sequence
    } else {
        const int per = p.tokens / p.B;
        b = static_cast<int>(static_cast<uint32_t>(row) / static_cast<uint32_t>(per));
        first = b * per;
        start = __ldg(p.pos + b);
    }
    const int64_t pos = static_cast<int64_t>(start) + (row - first);
    if (row < first || pos < 0 || (pos >> p.P_log2) >= p.bt_stride) {
        if (lane == 0) atomicOr(p.err, VK_ERR_TABLE_INDEX);
        return;
    }
    const int32_t page = __ldg(p.bt + static_cast<int64_t>(b) * p.bt_stride + (pos >> p.P_log2));
    if (page < 0 || page >= p.num_pages) {
        if (lane == 0) atomicOr(p.err, VK_ERR_PAGE_ID);
        return;
    }
    const int64_t slot = (static_cast<int64_t>(page) << p.P_log2) + (pos & ((1 << p.P_log2) - 1));
    uint4* dst = reinterpret_cast<uint4*>(p.base + 2 * slot * (p.latent_dim + p.rope_dim));
    if (p.weight) {
        float x[2][8], sum = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            unpack16<T>(c[i], x[i]);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = fmaf(x[i][j], x[i][j], sum);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const float inv = rsqrtf(sum * p.inv_dim + p.eps);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float w[8];
            unpack16<T>(wv[i], w);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[i][j] = x[i][j] * inv * w[j];
            c[i] = pack16<T>(x[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (lane + 32 * i < vecs) dst[lane + 32 * i] = c[i];
    if (lane < pairs) {
        if (rot.pairs) {
            const float2 x = Elem<T>::unpack(k);
            const float2 r = rotary_turn(x.x, x.y, rotary_cos_sin(turn[lane], rot.magnitude, static_cast<int>(pos)));
            k = Elem<T>::pack(r.x, r.y);
        }
        char* kdst = reinterpret_cast<char*>(dst + vecs);
        if (half) {
            reinterpret_cast<uint16_t*>(kdst)[lane] = static_cast<uint16_t>(k);
            reinterpret_cast<uint16_t*>(kdst)[lane + pairs] = static_cast<uint16_t>(k >> 16);
        } else {
            reinterpret_cast<uint32_t*>(kdst)[lane] = k;
        }
    }
}

}  // namespace vk

using namespace vk;

extern "C" vk_status vk_latent_append(vk_pool* pool, int32_t layer, const void* latent, int64_t latent_stride,
                                      const void* k_rope, int64_t rope_stride, const void* norm_weight, float eps,
                                      const vk_rotary* rotary, const int32_t* block_tables, int32_t bt_stride,
                                      const int32_t* positions, const int32_t* offsets, int32_t batch, int32_t tokens,
                                      void* stream) {
    if (!pool) return fail(VK_INVALID_ARG, "pool is NULL");
    if (!is_latent(pool)) return fail(VK_UNSUPPORTED, "latent append needs a latent pool");
    if (layer < 0 || layer >= pool->cfg.num_layers) return fail(VK_INVALID_ARG, "layer out of range");
    if (batch < 0 || tokens < 0 || bt_stride <= 0) return fail(VK_INVALID_ARG, "bad batch/tokens/bt_stride");
    if (batch == 0 || tokens == 0) return VK_OK;
    if (!latent || !k_rope || !block_tables || !positions) return fail(VK_INVALID_ARG, "NULL array");
    if (!offsets && tokens % batch) return fail(VK_INVALID_ARG, "without offsets, tokens must be a multiple of batch");
    if (((reinterpret_cast<uintptr_t>(latent) | reinterpret_cast<uintptr_t>(k_rope) | reinterpret_cast<uintptr_t>(norm_weight)) & 15) ||
        latent_stride % 8 || rope_stride % 8)
        return fail(VK_INVALID_ARG, "latent, k_rope and norm_weight must be 16-byte aligned, row strides multiples of 8");
    if (norm_weight && !(eps >= 0.f)) return fail(VK_INVALID_ARG, "eps must be >= 0");
    RotaryTable none{};
    const RotaryTable* rot = rotary ? rotary_table(rotary) : &none;
    if (rotary && 2 * rot->pairs != pool->rope_dim) return fail(VK_INVALID_ARG, "the rotary's rotary_dim must be the pool's rope_dim");
    LatentAppendParams p;
    p.base = pool->base + static_cast<uint64_t>(layer) * pool->seg_stride;
    p.latent = static_cast<const char*>(latent);
    p.k_rope = static_cast<const char*>(k_rope);
    p.weight = static_cast<const char*>(norm_weight);
    p.latent_stride = latent_stride;
    p.rope_stride = rope_stride;
    p.bt = block_tables;
    p.pos = positions;
    p.offsets = offsets;
    p.err = pool->d_err;
    p.bt_stride = bt_stride;
    p.B = batch;
    p.tokens = tokens;
    p.latent_dim = pool->latent_dim;
    p.rope_dim = pool->rope_dim;
    p.P_log2 = pool->cfg.page_tokens == 16 ? 4 : pool->cfg.page_tokens == 32 ? 5 : 6;
    p.num_pages = pool->num_pages;
    p.eps = eps;
    p.inv_dim = 1.f / static_cast<float>(pool->latent_dim);
    DeviceGuard g(pool->device);
    const unsigned blocks = static_cast<unsigned>((static_cast<int64_t>(tokens) + kLaWarps - 1) / kLaWarps);
    if (pool->kv_format == VK_KV_LATENT_BF16)
        latent_append_kernel<__nv_bfloat16><<<blocks, kLaWarps * 32, 0, as_stream(stream)>>>(*rot, p);
    else
        latent_append_kernel<__half><<<blocks, kLaWarps * 32, 0, as_stream(stream)>>>(*rot, p);
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? VK_OK : cuda_fail(e, "latent_append_kernel launch");
}
