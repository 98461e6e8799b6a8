// How latent decode deals its work to CTAs, and what its merge may join.  Plain
// arithmetic, compiled for the host too: tests/cpp/test_latent_deal.cpp runs it
// without a GPU.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define VK_HD __host__ __device__ __forceinline__
#else
#define VK_HD inline
#endif

namespace vk {

// n CTAs share `total`: the first `rem` take q + 1, the others q; a range may be a
// single tile (1 x 200 tokens: 12.5 us so, 14.7 with four at least: tiles in parallel
// and a merge beat tiles in turn).  (64-bit divisions cost hundreds of cycles of every
// launch; totals below 2^32 need none.)
struct LdDeal {
    int64_t q, rem;
    int n;
    VK_HD LdDeal(int64_t total, int ctas) {
        n = static_cast<int>(ctas < total ? ctas : total);
        q = div(total, n);
        rem = total - q * n;
    }
    static VK_HD int64_t div(int64_t a, int64_t b) {
        return (a | b) >> 32 ? a / b : static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b));
    }
    VK_HD int64_t start(int c) const { return c * q + (c < rem ? c : rem); }
    VK_HD int owner(int64_t v) const {  // the CTA whose range holds v
        const int64_t head = rem * (q + 1);
        return static_cast<int>(v < head ? div(v, q + 1) : rem + div(v - head, q));
    }
};

// Whether a unit's entry (first, last CTA) names pieces to join.  A unit that one CTA
// has whole is (-1, -1).  A CTA that gives up on a wait leaves its units' entries
// unwritten, and the workspace needs no initial value: an entry may hold anything
// then, so only CTAs of the launch (and with them slots of the workspace) pass.
VK_HD bool ld_joinable(int first, int last, int ctas) { return first >= 0 && last > first && last < ctas; }

}  // namespace vk
