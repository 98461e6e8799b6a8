// Append to a latent pool (vk_latent_append): root-mean-square norm of the
// latent, rotation of the shared key part, and the row written through the
// block table.
//
//   row = [ c / sqrt(mean(c^2) + eps) * w  |  R(pos) k ]
//
// Bound by memory for chunks (2 * (latent + rope) * 2 bytes a token) and by
// latency for a decode step.  One warp per token: the row stays in registers
// between the sum of squares (fp32, one shuffle tree) and the scaled store, so
// it is read once and written once, in 16-byte vectors.
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
    int bt_stride, B, tokens, latent_dim, rope_dim, P, num_pages;
    float eps;
};

constexpr int kLaWarps = 4;  // tokens per block: 16k tokens still give every SM several blocks

// The sequence of a row: the last b with offsets[b] <= row, or -1 behind the end.
__device__ __forceinline__ int sequence_of(const int32_t* offsets, int B, int row) {
    if (row >= __ldg(offsets + B)) return -1;
    int lo = 0, hi = B - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (__ldg(offsets + mid) <= row) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

template <typename T>
__global__ void __launch_bounds__(kLaWarps * 32) latent_append_kernel(const __grid_constant__ RotaryTable rot,
                                                                      const LatentAppendParams p) {
    const int row = blockIdx.x * kLaWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row >= p.tokens) return;
    // the row's loads go out first; the page lookup runs behind them
    const int vecs = p.latent_dim >> 3;  // 16-byte vectors of the latent: 16..64, two a lane at most
    const uint4* src = reinterpret_cast<const uint4*>(p.latent + 2 * (row * p.latent_stride));
    uint4 c[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        c[i] = lane + 32 * i < vecs ? __ldg(src + lane + 32 * i) : make_uint4(0, 0, 0, 0);
    const uint4* ksrc = reinterpret_cast<const uint4*>(p.k_rope + 2 * (row * p.rope_stride));
    const int kvecs = p.rope_dim >> 3;
    // half layout: a lane takes vector j of both halves; else vector j alone
    const int half = rot.pairs && rot.half ? kvecs >> 1 : 0;
    const int kitems = half ? half : kvecs;
    uint4 k0 = make_uint4(0, 0, 0, 0), k1 = k0;
    if (lane < kitems) {
        k0 = __ldg(ksrc + lane);
        if (half) k1 = __ldg(ksrc + lane + half);
    }
    int b, t;
    if (p.offsets) {
        b = sequence_of(p.offsets, p.B, row);
        if (b < 0) return;
        t = row - __ldg(p.offsets + b);
    } else {
        const int per = p.tokens / p.B;
        b = row / per;
        t = row % per;
    }
    const int64_t pos = static_cast<int64_t>(__ldg(p.pos + b)) + t;
    if (t < 0 || pos < 0 || pos / p.P >= p.bt_stride) {
        if (lane == 0) atomicOr(p.err, VK_ERR_TABLE_INDEX);
        return;
    }
    const int32_t page = __ldg(p.bt + static_cast<int64_t>(b) * p.bt_stride + pos / p.P);
    if (page < 0 || page >= p.num_pages) {
        if (lane == 0) atomicOr(p.err, VK_ERR_PAGE_ID);
        return;
    }
    const int width = p.latent_dim + p.rope_dim;
    uint4* dst = reinterpret_cast<uint4*>(p.base + 2 * (static_cast<uint64_t>(page) * p.P + pos % p.P) * width);
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
        const float inv = 1.f / sqrtf(sum / p.latent_dim + p.eps);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (lane + 32 * i >= vecs) continue;
            float w[8];
            unpack16<T>(__ldg(reinterpret_cast<const uint4*>(p.weight) + lane + 32 * i), w);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[i][j] = x[i][j] * inv * w[j];
            c[i] = pack16<T>(x[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (lane + 32 * i < vecs) dst[lane + 32 * i] = c[i];
    if (lane < kitems) {
        if (rot.pairs) {
            float u[8];
            unpack16<T>(k0, u);
            if (half) {
                float w[8];
                unpack16<T>(k1, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float2 r = rotary_turn(u[j], w[j], rotary_cos_sin(rot, lane * 8 + j, static_cast<int>(pos)));
                    u[j] = r.x;
                    w[j] = r.y;
                }
                k1 = pack16<T>(w);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const float2 r = rotary_turn(u[j], u[j + 1], rotary_cos_sin(rot, lane * 4 + (j >> 1), static_cast<int>(pos)));
                    u[j] = r.x;
                    u[j + 1] = r.y;
                }
            }
            k0 = pack16<T>(u);
        }
        dst[vecs + lane] = k0;
        if (half) dst[vecs + lane + half] = k1;
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
    p.P = pool->cfg.page_tokens;
    p.num_pages = pool->num_pages;
    p.eps = eps;
    DeviceGuard g(pool->device);
    const unsigned blocks = static_cast<unsigned>((static_cast<int64_t>(tokens) + kLaWarps - 1) / kLaWarps);
    if (pool->kv_format == VK_KV_LATENT_BF16)
        latent_append_kernel<__nv_bfloat16><<<blocks, kLaWarps * 32, 0, as_stream(stream)>>>(*rot, p);
    else
        latent_append_kernel<__half><<<blocks, kLaWarps * 32, 0, as_stream(stream)>>>(*rot, p);
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? VK_OK : cuda_fail(e, "latent_append_kernel launch");
}
