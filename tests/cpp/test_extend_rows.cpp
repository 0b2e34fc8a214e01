// The way of threads through a block's older rows (iq_extend_plan.h) on the
// CPU: every piece of every row once, also where rows times pieces passes 32
// bits.
#include <cstdio>
#include <random>
#include <vector>

#include "../../infer_amd/csrc/iq_extend_plan.h"

static long failures = 0;
#define CHECK(x) \
    do { if (!(x)) { failures++; if (failures < 10) std::printf("%s:%d %s\n", __FILE__, __LINE__, #x); } } while (0)

int main() {
    // whole walks
    for (int32_t threads : {4, 8, 16, 32, 256})
        for (int32_t per = 1; per <= 16; per++)
            for (int32_t rows : {0, 1, 2, 15, 16, 17, 63, 255, 300}) {
                std::vector<int> seen(size_t(rows) * size_t(per), 0);
                const iq::Piece step = iq::piece_of(threads, per);
                for (int32_t t = 0; t < threads; t++)
                    for (iq::Piece p = iq::piece_of(t, per); p.row < rows; p = iq::piece_behind(p, step, per)) {
                        CHECK(p.row >= 0 && p.col >= 0 && p.col < per);
                        seen[size_t(p.row) * size_t(per) + size_t(p.col)]++;
                    }
                for (int n : seen) CHECK(n == 1);
            }
    // single steps anywhere, up to the last of the most rows there can be: the
    // piece behind number i is number i + threads (in 64 bits)
    std::mt19937_64 rng(3);
    for (int32_t threads : {4, 8, 16, 32, 256})
        for (int32_t per = 1; per <= 16; per++) {
            const iq::Piece step = iq::piece_of(threads, per);
            for (int32_t rows : {(1 << 27) - 1, 1 << 27, (1 << 27) + 3, 1 << 28, 0x7ffeffff}) {
                const int64_t all = int64_t(rows) * per;
                for (int it = 0; it < 2000; it++) {
                    const int64_t i = it < 500 ? all - 1 - it : int64_t(rng() % uint64_t(all));
                    const iq::Piece p{int32_t(i / per), int32_t(i % per)}, q = iq::piece_behind(p, step, per);
                    CHECK(int64_t(q.row) * per + q.col == i + threads && q.col >= 0 && q.col < per);
                    CHECK((q.row < rows) == (i + threads < all));  // the walk's end
                }
            }
        }
    std::printf("%ld failures\n", failures);
    return failures != 0;
}
