// iq_overlap.h -- whether memory that a call writes meets memory that it reads:
// plain C++, shared by the entry points and the CPU tests (g++ compiles it on
// its own).
#pragma once

#include <algorithm>
#include <cstdint>

namespace iq {

inline bool ranges_overlap(const void* a, int64_t abytes, const void* b, int64_t bbytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && x < y + uintptr_t(bbytes) && y < x + uintptr_t(abytes);
}

// Whether the `bytes` bytes from `a` on meet one of n[0] x n[1] x n[2] rows of
// `row` bytes, `stride` bytes apart, from `base` on.  An output may lie between
// a pool's rows (of a larger tensor): only the rows themselves count, where
// each stride spans what lies below it; else whatever lies in between does too.
// (128 bits: the last row's offset may pass 64, if only on paper.)
inline bool meets_rows(const void* a, int64_t bytes, const void* base, const int64_t (&n)[3], const int64_t (&stride)[3],
                       int64_t row) {
    typedef __int128 wide;
    if (!a) return false;
    int order[3] = {0, 1, 2};
    std::sort(order, order + 3, [&](int x, int y) { return stride[x] > stride[y]; });
    wide extent[4] = {0, 0, 0, row};  // of what a level spans
    for (int i = 2; i >= 0; i--) extent[i] = wide(n[order[i]] - 1) * stride[order[i]] + extent[i + 1];
    auto meets = [&](auto&& self, int level, wide lo) -> bool {
        const wide hi = lo + bytes;
        if (hi <= 0 || lo >= extent[level]) return false;
        if (level == 3) return true;
        const wide step = stride[order[level]], below = extent[level + 1], last = n[order[level]] - 1;
        if (last == 0) return self(self, level + 1, lo);
        if (below > step) return true;
        // the things that reach past lo and begin before hi; one between two others is covered
        const wide from = lo < below ? 0 : (lo - below) / step + 1, to = (hi - 1) / step < last ? (hi - 1) / step : last;
        if (to - from >= 2) return true;
        for (wide i = from; i <= to; i++)
            if (self(self, level + 1, lo - i * step)) return true;
        return false;
    };
    return meets(meets, 0, wide(reinterpret_cast<uintptr_t>(a)) - wide(reinterpret_cast<uintptr_t>(base)));
}

}  // namespace iq
