// infer_amd/csrc/iq_overlap.h on the CPU: outputs against the rows of a cache
// of any strides, byte by byte.
#include <cstdio>
#include <random>
#include <vector>

#include "../../infer_amd/csrc/iq_overlap.h"

static long failures = 0, met = 0, between = 0;
#define CHECK(x) \
    do { if (!(x)) { failures++; if (failures < 10) std::printf("%s:%d %s\n", __FILE__, __LINE__, #x); } } while (0)

int main() {
    std::mt19937_64 rng(5);
    auto below = [&](int64_t n) { return int64_t(rng() % uint64_t(n)); };
    char* const base = reinterpret_cast<char*>(uintptr_t(1) << 40);  // (nothing is read)
    for (int it = 0; it < 40000; it++) {
        // rows that nest in a random order, with gaps or not, and a stride of 0 over a single thing
        int64_t n[3], stride[3];
        const int64_t row = 1 + below(6);
        int order[3] = {0, 1, 2};
        std::shuffle(order, order + 3, rng);
        int64_t span = row;
        for (int i : order) {
            n[i] = 1 + below(4);
            stride[i] = n[i] == 1 ? 0 : span + (below(2) ? below(8) : 0);
            span += (n[i] - 1) * stride[i];
        }
        std::vector<bool> mine(size_t(span), false);
        for (int64_t x = 0; x < n[0]; x++)
            for (int64_t y = 0; y < n[1]; y++)
                for (int64_t z = 0; z < n[2]; z++)
                    for (int64_t e = 0; e < row; e++) mine[size_t(x * stride[0] + y * stride[1] + z * stride[2] + e)] = true;
        for (int k = 0; k < 20; k++) {
            const int64_t at = below(span + 24) - 12, bytes = 1 + below(below(2) ? 5 : span + 8);
            bool want = false;
            for (int64_t e = std::max<int64_t>(at, 0); e < std::min(at + bytes, span); e++) want |= mine[size_t(e)];
            CHECK(iq::meets_rows(base + at, bytes, base, n, stride, row) == want);
            met += want;
            between += !want && at >= 0 && at + bytes <= span;
        }
    }
    CHECK(met > 10000 && between > 10000);
    {
        // strides that do not nest: whatever lies in the range counts, nothing outside it
        const int64_t n[3] = {4, 5, 2}, stride[3] = {24, 16, 64};
        CHECK(iq::meets_rows(base + 1, 1, base, n, stride, 1) && !iq::meets_rows(base - 4, 4, base, n, stride, 1));
        CHECK(!iq::meets_rows(base + 3 * 24 + 4 * 16 + 64 + 1, 9, base, n, stride, 1));
    }
    {
        // the largest pool there can be on paper
        const int64_t big = int64_t(1) << 30, n[3] = {0x7fffffff, 0x7fffffff, 1024}, stride[3] = {4 * big, 4 * big, 4 * big};
        CHECK(iq::meets_rows(base + 5, 1 << 20, base, n, stride, 4) && !iq::meets_rows(base - 8, 8, base, n, stride, 4));
        const int64_t one[3] = {0x7fffffff, 1, 1}, far[3] = {4 * big, 0, 0};
        CHECK(iq::meets_rows(base + 4 * big, 1, base, one, far, 4) && !iq::meets_rows(base + 4 * big + 4, 4 * big - 4, base, one, far, 4));
        CHECK(iq::meets_rows(base + 4 * big + 4, 4 * big - 3, base, one, far, 4));
    }
    {
        const int64_t n[3] = {1, 1, 1}, stride[3] = {0, 0, 0};  // no output
        CHECK(!iq::meets_rows(nullptr, 1 << 20, nullptr, n, stride, 4));
    }
    std::printf("%ld failures\n", failures);
    return failures != 0;
}
