// The split that the attention kernels make (iq_attn_plan.h) on the CPU: a
// sequence's chunks by a reciprocal, the choice of a chunk's size, and with
// these that every token lies in one chunk, none is empty, and all stay within
// the grid and the partial results that the host plans for.
#include <cmath>
#include <cstdio>
#include <random>
#include <vector>

#include "../../infer_amd/csrc/iq_attn_plan.h"

static long failures = 0;
#define CHECK(x) \
    do { if (!(x)) { failures++; if (failures < 10) std::printf("%s:%d %s\n", __FILE__, __LINE__, #x); } } while (0)

constexpr uint32_t kMostTiles = (0x7fff0000u + 31) / 32;

// Reciprocals as they may come out: an estimate off by up to 2^-23 of itself
// before the Newton step, and what is behind it off by up to 2^-46.
static std::vector<double> reciprocals(uint32_t c) {
    std::vector<double> r;
    for (double e : {0.0, 0x1p-23, -0x1p-23, 0x1.8p-24, -0x1p-30}) r.push_back(iq::attn_rcp(c, 1.0 / c * (1 + e)));
    for (double e : {0x1p-46, -0x1p-46}) r.push_back(1.0 / c * (1 + e));
    return r;
}

static void check_quotients(uint32_t c, std::mt19937_64& rng) {
    const std::vector<double> rs = reciprocals(c);
    // 2^-46, and three roundings of half a step, 2^-53: of 1 / c, of its product
    // with 1 + e (or, where a Newton step squares these two away, of the step's
    // result), of r * c: 2^-46 (1 + 3 / 128)
    for (double r : rs) CHECK(std::fabs(r * c - 1) <= 0x1.06p-46);
    auto check = [&](int64_t tiles) {
        if (tiles < 0 || tiles > int64_t(kMostTiles)) return;
        for (double r : rs) CHECK(iq::attn_chunks_by(uint32_t(tiles), c, r) == iq::attn_chunks(uint32_t(tiles), c));
    };
    const int64_t most = kMostTiles / c;
    for (int i = 0; i < 60; i++) {
        const int64_t k = i < 20 ? i : i < 40 ? most - (i - 20) : int64_t(rng() % uint64_t(most + 1));
        for (int o = -1; o <= 1; o++) check(k * c + o);
    }
    check(kMostTiles);
}

// The work items of a batch as find_item enumerates them; seen: the tokens that
// a sequence sees at most.
static void check_batch(const std::vector<int32_t>& lens, uint32_t heads, int32_t seen, uint32_t target, std::mt19937_64& rng) {
    const uint32_t B = uint32_t(lens.size());
    auto tiles_of = [&](int32_t n) { return n < 0 ? 0u : iq::attn_tiles(std::min(n, seen)); };
    auto rcp = [&](uint32_t c) {
        const std::vector<double> r = reciprocals(c);
        return r[rng() % r.size()];
    };
    uint32_t total = 0;
    for (const int32_t n : lens) total += tiles_of(n);
    const uint32_t least = iq::attn_chunk_tiles(total, heads, target);
    uint32_t c = least;
    if (B * heads <= target) {
        uint32_t items[iq::kAttnTries] = {}, size = least;
        for (int i = 0; i < iq::kAttnTries; i++) {
            const double r = rcp(size);
            for (const int32_t n : lens) items[i] += iq::attn_chunks_by(tiles_of(n), size, r);
            size = iq::attn_more_tiles(size, least);
        }
        c = iq::attn_pick_tiles(least, items, heads, target);
        CHECK(c >= least && c <= size);
        if (c != size) {  // one that was tried: its items run at once, those of the sizes before it do not
            uint64_t all = 0;
            for (const int32_t n : lens) all += iq::attn_chunks(tiles_of(n), c);
            CHECK(all * heads <= target);
            for (uint32_t before = least; before < c; before = iq::attn_more_tiles(before, least)) {
                all = 0;
                for (const int32_t n : lens) all += iq::attn_chunks(tiles_of(n), before);
                CHECK(all * heads > target);
            }
        }
    }
    CHECK(c >= uint32_t(iq::kAttnWaves));
    const double r = rcp(c);
    int64_t items = 0, partials = 0;
    for (const int32_t n : lens) {
        const uint32_t tiles = tiles_of(n), k = iq::attn_chunks_by(tiles, c, r);
        CHECK(k >= 1 && uint64_t(k) * c >= tiles && (k == 1 || uint64_t(k - 1) * c < tiles));  // no chunk is empty
        items += int64_t(k) * heads;
        if (k > 1) partials += int64_t(k) * heads;
    }
    CHECK(items <= iq::attn_max_items(B, heads, seen, target));
    CHECK(partials <= iq::attn_max_partials(target));
    // where a sequence sees at most one chunk there are no partial results (the join is not launched)
    if (iq::attn_tiles(seen) <= uint32_t(iq::kAttnWaves)) CHECK(partials == 0);
}

int main() {
    std::mt19937_64 rng(9);
    for (uint32_t c = 1; c < 3000; c++) check_quotients(c, rng);
    for (int it = 0; it < 20000; it++) check_quotients(1 + uint32_t(std::exp2(26.0 * double(rng() % 1000003) / 1000003)), rng);
    for (uint32_t c : {kMostTiles - 1, kMostTiles, (1u << 26) - 1, 1u << 25, (1u << 25) + 1}) check_quotients(c, rng);
    for (int it = 0; it < 20000; it++) {
        const uint32_t heads = 1 + rng() % 64, target = it % 2 ? 256 * (1 + rng() % 4) : 1 + rng() % 1024;
        const int B = 1 + int(rng() % (it % 10 ? 40 : 1024));
        const int32_t cap = 1 + int32_t(rng() % (it % 3 ? 5000 : 300000));
        const int32_t seen = it % 4 ? cap : 1 + int32_t(rng() % uint32_t(cap));
        std::vector<int32_t> lens(size_t(B), 0);
        for (auto& n : lens) n = rng() % 4 ? int32_t(rng() % uint64_t(cap + 1)) : rng() % 2 ? cap : int32_t(rng() % 3) - 1;
        check_batch(lens, heads, seen, target, rng);
    }
    check_batch({0x7fff0000}, 8, 0x7fff0000, 512, rng);
    check_batch({0x7fff0000}, 1, 0x7fff0000, 1, rng);
    check_batch({0x7fff0000, 0x7fff0000 - 31, 1, 0}, 4, 0x7fff0000, 1024, rng);
    std::printf("%ld failures\n", failures);
    return failures != 0;
}
