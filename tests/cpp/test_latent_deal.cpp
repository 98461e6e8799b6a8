// The deal of latent decode on the host: every position of the laid-out work has
// one owner, the entry of a unit that several CTAs share may be joined, and no
// other entry may be.
#include <climits>
#include <cstdio>
#include <random>
#include <vector>

#include "vk_latent_deal.h"

static int g_failures = 0;
#define CHECK(x)                                                              \
    do {                                                                      \
        if (!(x)) {                                                           \
            if (++g_failures < 20) std::printf("line %d: %s\n", __LINE__, #x); \
        }                                                                     \
    } while (0)

static void check_deal(const std::vector<int64_t>& units, int ctas) {
    int64_t total = 0;
    for (int64_t u : units) total += u;
    const vk::LdDeal deal(total, ctas);
    CHECK(deal.n >= 1 && deal.n <= ctas && deal.start(0) == 0 && deal.start(deal.n) == total);
    for (int c = 0; c < deal.n; ++c) CHECK(deal.start(c) < deal.start(c + 1));
    int64_t at = 0;
    for (int64_t u : units) {
        const int first = deal.owner(at), last = deal.owner(at + u - 1);
        CHECK(first >= 0 && last < deal.n);
        CHECK(deal.start(first) <= at && at < deal.start(first + 1));
        CHECK(deal.start(last) <= at + u - 1 && at + u - 1 < deal.start(last + 1));
        CHECK(vk::ld_joinable(first, last, ctas) == (first != last));
        at += u;
    }
}

int main() {
    std::mt19937_64 rng(1);
    for (int ctas : {1, 2, 3, 147, 148, 256}) {
        check_deal({1}, ctas);
        check_deal({3}, ctas);
        check_deal({int64_t(1) << 40, 3, int64_t(1) << 33}, ctas);
        for (int k = 0; k < 300; ++k) {
            std::vector<int64_t> units(1 + rng() % 400);
            for (auto& u : units) u = 1 + rng() % (k % 2 ? 40 : 3000);
            check_deal(units, ctas);
        }
        // what unwritten memory may hold
        for (int i = 0; i < 20000; ++i) {
            const int first = static_cast<int>(rng()), last = static_cast<int>(rng());
            CHECK(!vk::ld_joinable(first, last, ctas) || (first >= 0 && first < last && last < ctas));
        }
        for (int bad : {INT_MIN, -2, -1, ctas, ctas + 1, 0x7f7f7f7f, INT_MAX}) {
            CHECK(!vk::ld_joinable(bad, bad, ctas));
            CHECK(!vk::ld_joinable(0, bad, ctas));
            CHECK(!vk::ld_joinable(bad, ctas - 1, ctas));
        }
        CHECK(!vk::ld_joinable(1, 0, ctas) && !vk::ld_joinable(0, 0, ctas));
    }
    std::printf("%d failures\n", g_failures);
    return g_failures != 0;
}
