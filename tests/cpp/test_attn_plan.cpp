// The arithmetic of infer_amd/csrc/iq_attn_plan.h on the CPU: pages of
// tokens, and the split of a batch's tokens over workgroups.
#include <cstdio>
#include <random>
#include <vector>

#include "../../infer_amd/csrc/iq_attn_plan.h"

static long failures = 0;
#define CHECK(x) \
    do { if (!(x)) { failures++; if (failures < 10) std::printf("%s:%d %s\n", __FILE__, __LINE__, #x); } } while (0)

// The work items of a batch as the kernel enumerates them.
static void check_batch(const std::vector<int32_t>& lens, uint32_t heads, int64_t cap, uint32_t target) {
    uint32_t total = 0;
    for (const int32_t n : lens) total += iq::attn_tiles(n);
    const uint32_t least = iq::attn_chunk_tiles(total, heads, target);
    uint32_t c = least;
    for (int i = 0; i < iq::kAttnTries; i++) {
        uint64_t all = 0;
        for (const int32_t n : lens) all += iq::attn_chunks(iq::attn_tiles(n), c);
        if (all * heads <= target) break;
        c = iq::attn_more_tiles(c, least);
    }
    CHECK(c >= uint32_t(iq::kAttnWaves));
    int64_t items = 0, partials = 0;
    for (const int32_t n : lens) {
        const uint32_t tiles = iq::attn_tiles(n), k = iq::attn_chunks(tiles, c);
        CHECK(k >= 1 && uint64_t(k) * c >= tiles && (k == 1 || uint64_t(k - 1) * c < tiles));  // no chunk is empty
        items += int64_t(k) * heads;
        if (k > 1) partials += int64_t(k) * heads;
    }
    CHECK(items <= iq::attn_max_items(int64_t(lens.size()), heads, cap, target));
    CHECK(partials <= iq::attn_max_partials(target));
    // a table of at most one chunk has no partial results (the join is not launched)
    if (iq::attn_tiles(int32_t(cap)) <= uint32_t(iq::kAttnWaves)) CHECK(partials == 0);
}

int main() {
    std::mt19937_64 rng(7);
    for (uint32_t d = 1; d < 70000; d += d < 2100 ? 1 : 997) {
        const iq::PageDiv p = iq::page_div(d);
        for (uint64_t q = 0; q < 40; q++)
            for (int64_t o = -1; o <= 1; o++) {
                const int64_t n = int64_t(q < 20 ? q * d : (rng() % 0x7fffffffu) / d * d) + o;
                if (n >= 0 && n < 0x7fffffff) CHECK(iq::page_of(uint32_t(n), p) == uint32_t(n) / d);
            }
        CHECK(iq::page_of(0x7fffffffu, p) == 0x7fffffffu / d);
    }
    for (uint32_t d : {0x7fffffffu, 0x40000000u, 0x40000001u, 0x3fffffffu}) {
        const iq::PageDiv p = iq::page_div(d);
        for (uint32_t n : {0u, 1u, d - 1, d, d + 1 > 0x7fffffffu ? d : d + 1, 0x7fffffffu})
            CHECK(iq::page_of(n, p) == n / d);
    }
    for (int it = 0; it < 20000; it++) {
        const uint32_t heads = 1 + rng() % 64, target = 1 + rng() % 1024;
        const int B = 1 + int(rng() % (it % 10 ? 40 : 1024));
        const int64_t cap = 1 + int64_t(rng() % (it % 3 ? 5000 : 300000));
        std::vector<int32_t> lens(size_t(B), 0);
        for (auto& n : lens) n = rng() % 4 ? int32_t(rng() % uint64_t(cap + 1)) : (rng() % 2 ? int32_t(cap) : int32_t(rng() % 2));
        check_batch(lens, heads, cap, target);
    }
    check_batch({0x7fff0000}, 8, 0x7fff0000, 512);
    std::printf("%ld failures\n", failures);
    return failures != 0;
}
