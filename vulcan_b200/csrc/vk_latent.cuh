// Shared by the kernels of the latent cache.
#pragma once

#include "vk_ptx.cuh"
#include "vk_rotary.cuh"

namespace vk {

// Bounded mbarrier wait of a whole warp, with one answer for all its lanes.
__device__ __forceinline__ bool wait_all(uint32_t bar, uint32_t parity, uint32_t* err) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, err));
}

// 3-input max (one instruction on sm_100)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Two fp32 values in one 64-bit register pair, one instruction for both (sm_100).
__device__ __forceinline__ uint64_t f2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void f2_get(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// The unnormalised weights of both attentions are 2^(s - m) (s: scores in the log2
// domain), with m a reference below the row's running maximum by kMargin or, while the
// maximum has grown since m was taken, by up to kMargin + kLag: a growth by more than
// kLag moves m and rescales O.  The weights are rounded to the cache's type for the
// second product.  fp16 has normal numbers from 2^-14 to 2^16 only: with m at the maximum
// itself, the weights of keys 2^-25 below it became 0 there and still counted in full in
// the fp32 sum, and 131,072 such keys lost 0.4% of the mass to one dominant key.  Weights up to
// 2^(kMargin + kLag) = 2^15 use the range above 1: relative 2^-11 down to 2^-21 of the
// maximum, absolute 2^-32 of it below (131,072 keys: 2^-15 of the mass at most).  A margin of
// 11 with a lag of 4 is 2^4 more exact there, but rescales O so much more often that 24 x
// 16k tokens whose scores have a deviation of 3 took 108 us for 95.  bf16 has fp32's range and
// needs no margin.
template <typename T>
struct Weights {
    static constexpr float kMargin = Elem<T>::kBf16 ? 0.f : 7.f;
    static constexpr float kLag = 8.f;
    // log2 of the sum of 2^s from the reference and the sum of the weights
    static __device__ __forceinline__ float log2_sum(float m, float l) {
        constexpr float unit = Elem<T>::kBf16 ? 1.f : 0x1p-7f;
        return (m + kMargin) + log2f(l * unit);
    }
};

// 0 in the place of each non-finite 16-bit element of a word.
template <typename T>
__device__ __forceinline__ uint32_t finite_word(uint32_t w) {
    constexpr uint32_t e = Elem<T>::kBf16 ? 0x7f80u : 0x7c00u;
    if ((w & e) == e) w &= 0xffff0000u;
    if ((w & (e << 16)) == (e << 16)) w &= 0x0000ffffu;
    return w;
}

}  // namespace vk
