// Shared by the kernels of the latent cache.
#pragma once

#include "vk_ptx.cuh"

namespace vk {

// Bounded mbarrier wait of a whole warp, with one answer for all its lanes.
__device__ __forceinline__ bool wait_all(uint32_t bar, uint32_t parity, uint32_t* err) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, err));
}

}  // namespace vk
