// The arithmetic of infer_amd/csrc/iq_extend_plan.h on the CPU: every new token
// in exactly one unit, and nothing out of range whatever the starts hold.
#include <cstdio>
#include <random>
#include <vector>

#include "../../infer_amd/csrc/iq_extend_plan.h"

static long failures = 0;
#define CHECK(x) \
    do { if (!(x)) { failures++; if (failures < 10) std::printf("%s:%d %s\n", __FILE__, __LINE__, #x); } } while (0)

// Units as extend_kernel enumerates them; `sound`: the starts are ascending from 0 to T.
static void check(const std::vector<int32_t>& starts, const std::vector<int32_t>& lens, int32_t T, int32_t cap, int32_t span,
                  bool sound) {
    const int64_t B = int64_t(lens.size()), grid = iq::max_units(T, B, span);
    const iq::PageDiv div = iq::page_div(uint32_t(span));
    std::vector<int> seen(size_t(T), 0);
    int64_t all = 0;
    for (int64_t b = 0; b < B; b++) {
        const int32_t len = lens[size_t(b)];
        const iq::NewTokens n = iq::new_tokens(starts[size_t(b)], starts[size_t(b) + 1], len, T, cap);
        CHECK(n.count >= 0 && (n.count == 0 || (n.row >= 0 && n.row + int64_t(n.count) <= T)));
        const uint32_t units = iq::units_of(len, n.count, div);
        all += units;
        int64_t tokens = 0;
        for (uint32_t i = 0; i < units && i < 4000; i++) {
            const iq::Unit u = iq::unit_at(i, len, n, span, div);
            CHECK(u.count > 0 && u.count <= span && u.begin >= 0 && u.begin % span == 0 && u.tok >= u.begin);
            CHECK(u.tok >= len && int64_t(u.tok) + u.count <= int64_t(u.begin) + span && int64_t(u.tok) + u.count <= cap);
            CHECK(u.row >= n.row && u.row - n.row == u.tok - len);
            CHECK((u.tok > u.begin) == (i == 0 && len % span != 0));  // only the first unit has older tokens
            for (int32_t k = 0; k < u.count; k++) seen[size_t(u.row) + size_t(k)]++;
            tokens += u.count;
        }
        if (units <= 4000) CHECK(tokens == n.count);
        // past the last unit there is nothing, however far (a batch's sum that wrapped)
        for (uint32_t far : {0u, 1u, 77u, 0x7fffffffu, 0xffffffffu - units}) CHECK(iq::unit_at(units + far, len, n, span, div).count == 0);
    }
    if (!sound) return;
    CHECK(all <= grid);
    for (int64_t b = 0; b < B; b++) {
        const int32_t len = lens[size_t(b)];
        for (int64_t t = starts[size_t(b)]; t < starts[size_t(b) + 1]; t++)
            CHECK(seen[size_t(t)] == (len >= 0 && len + (t - starts[size_t(b)]) < cap ? 1 : 0));
    }
}

int main() {
    std::mt19937_64 rng(11);
    auto below = [&](int64_t n) { return int64_t(rng() % uint64_t(n)); };
    for (int it = 0; it < 20000; it++) {
        const int64_t B = 1 + below(it % 9 ? 12 : 300);
        const int32_t span = int32_t(1 + below(it % 3 ? 20 : 200)), cap = int32_t(span * (1 + below(30)));
        std::vector<int32_t> starts{0}, lens;
        for (int64_t b = 0; b < B; b++) {
            const int kind = int(below(6));
            lens.push_back(kind == 0 ? -1 - int32_t(below(1000)) : kind == 1 ? cap + int32_t(below(3)) - 1 : int32_t(below(cap)));
            starts.push_back(starts.back() + (below(3) ? int32_t(below(it % 2 ? 4 : 3 * span)) : 0));
        }
        const int32_t T = starts.back() + int32_t(below(3));
        if (T < 1) continue;
        check(starts, lens, T, cap, span, true);
        for (auto& s : starts)
            if (below(4) == 0) s = int32_t(rng());
        check(starts, lens, T, cap, span, false);
    }
    check({0, 50}, {0x7ffeffff - 20}, 50, 0x7fff0000, 64, true);
    check({0, 50}, {0x7ffeffff}, 50, 0x7fff0000, 1, true);
    check({-0x7fffffff - 1, 0x7fffffff, 0}, {0x7fffffff, -0x7fffffff - 1}, 9, 0x7fff0000, 7, false);
    std::printf("%ld failures\n", failures);
    return failures != 0;
}
