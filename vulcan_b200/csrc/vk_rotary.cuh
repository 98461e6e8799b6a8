// Rotary positions of the standalone rotation and of the latent cache's append:
// the angle of a pair at a position, right to fp32 at any position.
//
// Pair i of the R rotated elements turns by pos * f_i.  In fp32 that product
// has lost its fraction of a turn by position 2^20 (one ulp is 0.06 rad); in
// fp64 it would be right but slow.  Instead the host stores f_i / (2 pi) as a
// 64-bit fixed-point fraction of a turn, and the device multiplies modulo 2^64:
// whole turns fall off the top by themselves, and the fraction is off by at
// most pos * 2^-65 turns and the host's relative error of f_i (a few 2^-64; four
// roundings in long double), together below 2^-29 rad at any int32 position.  The
// whole fraction, as a signed count of 2^-64 turns, goes to sincospi in fp32:
// its top 32 bits alone were 1.5e-9 rad off, a thousandth of the sine of slow pairs
// at the first positions.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace vk {

constexpr int kRotaryMaxPairs = 128;  // rotary_dim <= 256

// By value in kernel parameters: no device table, so none to allocate or order.
struct RotaryTable {
    uint64_t turn[kRotaryMaxPairs];  // round(f_i / (2 pi) * 2^64)
    float magnitude;                 // multiplies cos and sin
    int pairs;                       // rotary_dim / 2; 0: no rotation
    int half;                        // 0: pairs (2i, 2i+1); 1: pairs (i, i + rotary_dim/2)
};

__device__ __forceinline__ float2 rotary_cos_sin(uint64_t turn, float magnitude, int pos) {
    const uint64_t phase = static_cast<uint64_t>(static_cast<int64_t>(pos)) * turn;
    // 2 * turns, in [-1, 1], by halves (a 64-bit conversion made 16k tokens of 64 heads 6% slower)
    const float turns2 = fmaf(static_cast<float>(static_cast<uint32_t>(phase)), 0x1p-63f,
                              static_cast<float>(static_cast<int32_t>(phase >> 32)) * 0x1p-31f);
    float s, c;
    sincospif(turns2, &s, &c);
    return make_float2(c * magnitude, s * magnitude);
}

__device__ __forceinline__ float2 rotary_cos_sin(const RotaryTable& t, int pair, int pos) {
    return rotary_cos_sin(t.turn[pair], t.magnitude, pos);
}

__device__ __forceinline__ float2 rotary_turn(float a, float b, float2 cs) {
    return make_float2(a * cs.x - b * cs.y, a * cs.y + b * cs.x);
}

// Element type: conversions to fp32 and back (round to nearest even), alone and
// for the 16-byte vectors that the kernels move.
template <typename T>
struct Elem;
template <>
struct Elem<__half> {
    static constexpr int kVec = 8;
    static constexpr bool kBf16 = false;
    static __device__ __forceinline__ float up(__half x) { return __half2float(x); }
    static __device__ __forceinline__ __half down(float x) { return __float2half_rn(x); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    // beyond the type's range: its largest number
    static __device__ __forceinline__ uint32_t pack_sat(float a, float b) {
        uint32_t w;
        asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
        return w;
    }
    static __device__ __forceinline__ float2 unpack(uint32_t w) {
        return __half22float2(*reinterpret_cast<const __half2*>(&w));
    }
};
template <>
struct Elem<__nv_bfloat16> {
    static constexpr int kVec = 8;
    static constexpr bool kBf16 = true;
    static __device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
    static __device__ __forceinline__ __nv_bfloat16 down(float x) { return __float2bfloat16_rn(x); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ uint32_t pack_sat(float a, float b) {
        uint32_t w;
        asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
        return w;
    }
    static __device__ __forceinline__ float2 unpack(uint32_t w) {
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
};
template <>
struct Elem<float> {
    static constexpr int kVec = 4;
    static __device__ __forceinline__ float up(float x) { return x; }
    static __device__ __forceinline__ float down(float x) { return x; }
};

template <typename T>
__device__ __forceinline__ void unpack16(const uint4& v, float (&x)[Elem<T>::kVec]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if constexpr (Elem<T>::kVec == 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = Elem<T>::unpack(w[i]);
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
    }
}

template <typename T>
__device__ __forceinline__ uint4 pack16(const float (&x)[Elem<T>::kVec]) {
    if constexpr (Elem<T>::kVec == 8)
        return make_uint4(Elem<T>::pack(x[0], x[1]), Elem<T>::pack(x[2], x[3]), Elem<T>::pack(x[4], x[5]),
                          Elem<T>::pack(x[6], x[7]));
    else
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
}

}  // namespace vk
