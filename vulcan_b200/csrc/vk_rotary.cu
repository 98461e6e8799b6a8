// Rotary positions as an operator of its own (vk_rotary_*): q, and k when
// given, in one launch; interleaved or half layout, the leading rotary_dim
// elements of each head, frequencies scaled for long contexts.
//
//   y[a_i] = x[a_i] cos - x[b_i] sin,   y[b_i] = x[a_i] sin + x[b_i] cos
//
// with (a_i, b_i) = (2i, 2i+1) or (i, i + rotary_dim/2), angle = pos * f_i, cos
// and sin times the magnitude; computed in fp32, rounded once to the type.
//
// Floor: 4 bytes an element of a 16-bit tensor.  16,384 tokens of 32 + 32 heads of 128
// take 92 us, 0.90 of the measured copy rate (101 in a long run); blocks of 128 threads,
// one vector (a pair of vectors in the half layout) a thread, were the fastest of 64 to
// 512 threads and 1 to 4 vectors.  64 tokens: 2.5 us, the launch.
#include <algorithm>
#include <cmath>
#include <new>

#include "vk_internal.h"
#include "vk_rotary.cuh"

struct vk_rotary {
    vk::RotaryTable table{};
    int device = 0;
};

namespace vk {

struct RotaryView {
    const char* x;
    char* y;
    int64_t x_token, x_head, y_token, y_head;  // strides in elements
    int heads;
};

struct RotaryParams {
    RotaryView v[2];  // q, k
    const int32_t* pos;
    int tokens, head_dim;
    int items;      // work items of one token: (q heads + k heads) * per_head
    int per_head;   // items of one head: rotated ones, then copied ones
    int rotated;    // rotated items of one head
    int slices;     // blocks per token
};

constexpr int kRotThreads = 128;

// Block (token, slice of its items): the token's cos and sin once into shared
// memory (sincospi of each pair, shared by every head), then one item per
// thread (two or four in flight measured the same or slower).  An item is 16 bytes of one head (interleaved), the two 16-byte halves of 4 or 8
// pairs (half layout), or 16 bytes behind rotary_dim to copy; with VEC 0 a single
// pair or element, for pointers and strides that are not 16-byte multiples.  The
// loads go out before the cos/sin are computed.
template <typename T, int HALF, int VEC>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const __grid_constant__ RotaryTable tab,
                                                             const __grid_constant__ RotaryParams p) {
    __shared__ float2 cs[kRotaryMaxPairs];
    const int token = blockIdx.x / p.slices, slice = blockIdx.x % p.slices;
    const int item = slice * kRotThreads + threadIdx.x, half = tab.pairs;
    const bool live = item < p.items;
    const T* x = nullptr;
    T* y = nullptr;
    int j = 0;
    bool rot = false;
    if (live) {
        const int head = item / p.per_head;
        j = item % p.per_head;
        rot = j < p.rotated;
        const bool is_k = head >= p.v[0].heads;
        const RotaryView& v = is_k ? p.v[1] : p.v[0];
        const int h = is_k ? head - p.v[0].heads : head;
        x = reinterpret_cast<const T*>(v.x) + token * v.x_token + h * v.x_head;
        y = reinterpret_cast<T*>(v.y) + token * v.y_token + h * v.y_head;
    }
    if constexpr (VEC != 0) {
        constexpr int N = Elem<T>::kVec;
        // element of the item's first vector; (half layout, rotated) the second is `half` on
        const int e0 = rot || !HALF ? j * N : 2 * half + (j - p.rotated) * N;
        uint4 a, b;
        if (live) {
            a = *reinterpret_cast<const uint4*>(x + e0);
            if (HALF && rot) b = *reinterpret_cast<const uint4*>(x + half + e0);
            y += e0;
        }
        for (int i = threadIdx.x; i < half; i += kRotThreads) cs[i] = rotary_cos_sin(tab, i, __ldg(p.pos + token));
        __syncthreads();
        if (!live) return;
        if (rot) {
            float u[N];
            unpack16<T>(a, u);
            if constexpr (HALF) {
                float w[N];
                unpack16<T>(b, w);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float2 r = rotary_turn(u[i], w[i], cs[e0 + i]);
                    u[i] = r.x;
                    w[i] = r.y;
                }
                *reinterpret_cast<uint4*>(y + half) = pack16<T>(w);
            } else {
#pragma unroll
                for (int i = 0; i < N; i += 2) {
                    const float2 r = rotary_turn(u[i], u[i + 1], cs[(e0 + i) >> 1]);
                    u[i] = r.x;
                    u[i + 1] = r.y;
                }
            }
            a = pack16<T>(u);
        }
        *reinterpret_cast<uint4*>(y) = a;
    } else {
        for (int i = threadIdx.x; i < half; i += kRotThreads) cs[i] = rotary_cos_sin(tab, i, __ldg(p.pos + token));
        __syncthreads();
        if (!live) return;
        if (rot) {
            const int ea = HALF ? j : 2 * j, eb = HALF ? j + half : 2 * j + 1;
            const float2 r = rotary_turn(Elem<T>::up(x[ea]), Elem<T>::up(x[eb]), cs[j]);
            y[ea] = Elem<T>::down(r.x);
            y[eb] = Elem<T>::down(r.y);
        } else {
            const int e = 2 * half + (j - p.rotated);
            y[e] = x[e];
        }
    }
}

const RotaryTable* rotary_table(const vk_rotary* r) { return &r->table; }

template <typename T, int HALF>
static vk_status launch_rotary(const vk_rotary* r, const RotaryParams& p, bool vec, cudaStream_t st) {
    const int64_t blocks = static_cast<int64_t>(p.tokens) * p.slices;
    if (blocks > 0x7fffffff) return fail(VK_INVALID_ARG, "rotary: too many tokens for one launch");
    const dim3 grid(static_cast<unsigned>(blocks));
    if (vec) rotary_kernel<T, HALF, 1><<<grid, kRotThreads, 0, st>>>(r->table, p);
    else rotary_kernel<T, HALF, 0><<<grid, kRotThreads, 0, st>>>(r->table, p);
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? VK_OK : cuda_fail(e, "rotary_kernel launch");
}

// Angle per position of each pair, scaled for long contexts.  In long double (64 bits
// of mantissa or more): at position 2^31 the 2^-53 of a double is 2^-22 rad.
constexpr long double kTwoPi = 6.283185307179586476925286766559005768L;
static vk_status rotary_frequencies(const vk_rotary_cfg& c, long double* f, double* magnitude) {
    const int n = c.rotary_dim / 2;
    const long double theta = c.theta_base, factor = c.factor, original_len = c.original_len, low = c.low, high = c.high;
    for (int i = 0; i < n; ++i) f[i] = std::pow(theta, -2.0L * i / c.rotary_dim);
    *magnitude = c.magnitude > 0 ? c.magnitude : 1.0;
    if (c.scaling == VK_ROTARY_LINEAR) {
        for (int i = 0; i < n; ++i) f[i] /= factor;
    } else if (c.scaling == VK_ROTARY_BY_PARTS) {
        // the pair that makes `turns` turns within original_len positions
        auto pair_of = [&](long double turns) {
            return c.rotary_dim * std::log(original_len / (turns * kTwoPi)) / (2.0L * std::log(theta));
        };
        // the ramp may end behind the last pair: cut there, it would give pairs that make
        // more than `low` turns the whole factor
        const long double last = std::min(std::ceil(pair_of(low)), static_cast<long double>(c.rotary_dim - 1));
        const long double first = std::min(std::max(std::floor(pair_of(high)), 0.0L), last);
        for (int i = 0; i < n; ++i) {
            const long double ramp = std::min(std::max((i - first) / std::max(last - first, 0.001L), 0.0L), 1.0L);
            f[i] = f[i] * (1.0L - ramp) + f[i] / factor * ramp;
        }
        if (!(c.magnitude > 0)) *magnitude = c.factor > 1.0 ? 0.1 * std::log(c.factor) + 1.0 : 1.0;
    } else if (c.scaling == VK_ROTARY_BY_WAVELENGTH) {
        for (int i = 0; i < n; ++i) {
            const long double blend = std::min(std::max((original_len * f[i] / kTwoPi - low) / (high - low), 0.0L), 1.0L);
            f[i] = (1.0L - blend) * f[i] / factor + blend * f[i];
        }
    }
    for (int i = 0; i < n; ++i)
        if (!(f[i] >= 0.0L) || f[i] >= 3.0L) return fail(VK_INVALID_ARG, "rotary: a frequency is outside [0, 3) rad per position");
    return VK_OK;
}

// Whether two (token, head) rows of n elements may lie on one another: rows of either
// index apart by n or more, and those of one index within one step of the other.
static bool rotary_shares(int64_t token, int64_t tokens, int64_t head, int64_t heads, int64_t n) {
    token = token < 0 ? -token : token;
    head = head < 0 ? -head : head;
    if (tokens <= 1) return heads > 1 && head < n;
    if (heads <= 1) return token < n;
    return head < n || token < n || ((token - n) / head < heads - 1 && (head - n) / token < tokens - 1);
}

static vk_status check_rotary_cfg(const vk_rotary_cfg* c) {
    if (!c) return fail(VK_INVALID_ARG, "rotary: cfg is NULL");
    if (c->rotary_dim <= 0 || (c->rotary_dim & 1) || c->rotary_dim > 2 * kRotaryMaxPairs)
        return fail(VK_INVALID_ARG, "rotary_dim must be even, in 2..256");
    if (c->layout != VK_ROTARY_INTERLEAVED && c->layout != VK_ROTARY_HALF) return fail(VK_INVALID_ARG, "unknown rotary layout");
    if (!(c->theta_base > 1.0) || !std::isfinite(c->theta_base)) return fail(VK_INVALID_ARG, "theta_base must be > 1");
    if (c->scaling < VK_ROTARY_PLAIN || c->scaling > VK_ROTARY_BY_WAVELENGTH) return fail(VK_INVALID_ARG, "unknown rotary scaling");
    if (!std::isfinite(c->magnitude) || c->magnitude < 0) return fail(VK_INVALID_ARG, "magnitude must be >= 0 (0: the scaling's own)");
    if (c->scaling != VK_ROTARY_PLAIN && (!(c->factor > 0) || !std::isfinite(c->factor)))
        return fail(VK_INVALID_ARG, "the scaling's factor must be > 0");
    if (c->scaling >= VK_ROTARY_BY_PARTS &&
        (!(c->original_len > 0) || !std::isfinite(c->original_len) || !(c->low > 0) || !(c->high > c->low) ||
         !std::isfinite(c->high)))
        return fail(VK_INVALID_ARG, "the scaling needs original_len > 0 and 0 < low < high");
    return VK_OK;
}

}  // namespace vk

using namespace vk;

extern "C" vk_status vk_rotary_create(const vk_rotary_cfg* cfg, vk_rotary** out) {
    if (!out) return fail(VK_INVALID_ARG, "out is NULL");
    *out = nullptr;
    vk_status s = check_rotary_cfg(cfg);
    if (s != VK_OK) return s;
    long double f[kRotaryMaxPairs];
    double magnitude = 1.0;
    s = rotary_frequencies(*cfg, f, &magnitude);
    if (s != VK_OK) return s;
    auto* r = new (std::nothrow) vk_rotary();
    if (!r) return fail(VK_INVALID_ARG, "out of host memory");
    r->device = cfg->device;
    r->table.pairs = cfg->rotary_dim / 2;
    r->table.half = cfg->layout == VK_ROTARY_HALF;
    r->table.magnitude = static_cast<float>(magnitude);
    for (int i = 0; i < r->table.pairs; ++i)  // f / (2 pi) < 1/2: the scaled value fits 63 bits
        r->table.turn[i] = static_cast<uint64_t>(std::llround(std::ldexp(f[i] / kTwoPi, 64)));
    *out = r;
    return VK_OK;
}

extern "C" vk_status vk_rotary_destroy(vk_rotary* r) {
    delete r;
    return VK_OK;
}

extern "C" vk_status vk_rotary_frequencies(const vk_rotary_cfg* cfg, double* out, double* magnitude) {
    vk_status s = check_rotary_cfg(cfg);
    if (s != VK_OK) return s;
    if (!out || !magnitude) return fail(VK_INVALID_ARG, "NULL array");
    long double f[kRotaryMaxPairs];
    s = rotary_frequencies(*cfg, f, magnitude);
    if (s != VK_OK) return s;
    for (int i = 0; i < cfg->rotary_dim / 2; ++i) out[i] = static_cast<double>(f[i]);
    return VK_OK;
}

extern "C" vk_status vk_rotary_apply(const vk_rotary* r, int32_t dtype, const vk_rotary_view* q, const vk_rotary_view* k,
                                     int32_t head_dim, const int32_t* positions, int32_t tokens, void* stream) {
    if (!r) return fail(VK_INVALID_ARG, "rotary is NULL");
    if (dtype != VK_F16 && dtype != VK_BF16 && dtype != VK_F32) return fail(VK_INVALID_ARG, "unknown dtype");
    if (!q) return fail(VK_INVALID_ARG, "q is NULL");
    const int rotary_dim = 2 * r->table.pairs;
    if (head_dim < rotary_dim) return fail(VK_INVALID_ARG, "head_dim is smaller than rotary_dim");
    if (tokens < 0) return fail(VK_INVALID_ARG, "tokens must be >= 0");
    const int esize = dtype == VK_F32 ? 4 : 2, n = 16 / esize;
    RotaryParams p{};
    int64_t heads = 0;
    // 16-byte vectors need every pointer and stride on 16 bytes and, in the half
    // layout, the second half of a head too
    bool vec = head_dim % n == 0 && rotary_dim % n == 0 && (!r->table.half || r->table.pairs % n == 0), copies = false;
    const vk_rotary_view* views[2] = {q, k};
    for (int i = 0; i < 2; ++i) {
        const vk_rotary_view* v = views[i];
        if (!v || v->heads == 0) continue;
        if (v->heads < 0) return fail(VK_INVALID_ARG, "heads must be >= 0");
        if (tokens && (!v->x || !v->y)) return fail(VK_INVALID_ARG, "NULL array");
        if ((reinterpret_cast<uintptr_t>(v->x) | reinterpret_cast<uintptr_t>(v->y)) & (esize - 1))
            return fail(VK_INVALID_ARG, "x and y must be aligned to their elements");
        if (v->x == v->y && (v->x_token != v->y_token || v->x_head != v->y_head))
            return fail(VK_INVALID_ARG, "in place needs equal strides of x and y");
        if (rotary_shares(v->y_token, tokens, v->y_head, v->heads, head_dim))
            return fail(VK_INVALID_ARG, "the heads and tokens of y may not share elements");
        vec = vec && !((reinterpret_cast<uintptr_t>(v->x) | reinterpret_cast<uintptr_t>(v->y)) & 15) && v->x_token % n == 0 &&
              v->x_head % n == 0 && v->y_token % n == 0 && v->y_head % n == 0;
        copies = copies || v->x != v->y;
        p.v[i] = {static_cast<const char*>(v->x), static_cast<char*>(v->y), v->x_token, v->x_head, v->y_token, v->y_head, v->heads};
        heads += v->heads;
    }
    if (tokens == 0 || heads == 0) return VK_OK;
    if (p.v[0].heads && p.v[1].heads && (p.v[0].y == p.v[1].y || p.v[0].y == p.v[1].x || p.v[1].y == p.v[0].x))
        return fail(VK_INVALID_ARG, "an output may not be a tensor of the other of q and k");
    if (!positions) return fail(VK_INVALID_ARG, "NULL array");
    if (vec) {
        p.rotated = rotary_dim / n / (r->table.half ? 2 : 1);
        p.per_head = p.rotated + (copies ? (head_dim - rotary_dim) / n : 0);
    } else {
        p.rotated = r->table.pairs;
        p.per_head = p.rotated + (copies ? head_dim - rotary_dim : 0);
    }
    if (heads * p.per_head > 0x3fffffff) return fail(VK_INVALID_ARG, "too many heads");
    p.items = static_cast<int>(heads * p.per_head);
    p.slices = (p.items + kRotThreads - 1) / kRotThreads;
    p.pos = positions;
    p.tokens = tokens;
    p.head_dim = head_dim;
    DeviceGuard g(r->device);
    cudaStream_t st = as_stream(stream);
    const bool half = r->table.half;
    switch (dtype) {
        case VK_F16: return half ? launch_rotary<__half, 1>(r, p, vec, st) : launch_rotary<__half, 0>(r, p, vec, st);
        case VK_BF16: return half ? launch_rotary<__nv_bfloat16, 1>(r, p, vec, st) : launch_rotary<__nv_bfloat16, 0>(r, p, vec, st);
        default: return half ? launch_rotary<float, 1>(r, p, vec, st) : launch_rotary<float, 0>(r, p, vec, st);
    }
}
