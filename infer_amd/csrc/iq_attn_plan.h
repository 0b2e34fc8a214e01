// iq_attn_plan.h -- a token's page, and how a batch's cached tokens are split
// over workgroups: arithmetic shared by the kernels of iq_kv.hip and
// iq_attn.hip, their host side and the CPU tests (plain C++: g++ compiles it
// on its own).
//
// Lengths are known on the device only.  Every sequence is cut into chunks
// of the same number of 32-token tiles, C: the least share of the batch's
// total, or up to 7/4 of it, with which all chunks of all key/value head tiles
// are at most `target` work items, so that a long sequence beside short ones
// gets as many workgroups as its share of the tokens and all of them run at
// once.  A sequence always has one chunk at least (an empty one's writes its
// zeros), so many sequences may still be more than `target` items.
#pragma once

#include <algorithm>
#include <cstdint>

#if defined(__HIPCC__)
#define IQ_HD __host__ __device__ inline
#else
#define IQ_HD inline
#endif

namespace iq {

// Division by a page size: n / d = (n * mul) >> (31 + shift) for every n <
// 2^31, where 2^(shift - 1) < d <= 2^shift and mul = ceil(2^(31 + shift) / d)
// (mul * d exceeds 2^(31 + shift) by less than d <= 2^shift, n times that by
// less than 2^(31 + shift)).
struct PageDiv {
    uint32_t mul, shift;
};
inline PageDiv page_div(uint32_t d) {
    PageDiv p{0, 0};
    while ((uint64_t(1) << p.shift) < d) p.shift++;
    p.mul = uint32_t(((uint64_t(1) << (31 + p.shift)) + d - 1) / d);
    return p;
}
IQ_HD uint32_t page_of(uint32_t n, PageDiv p) { return uint32_t((uint64_t(n) * p.mul) >> (31 + p.shift)); }

constexpr int kAttnTile = 32;   // tokens a wave multiplies at a time
constexpr int kAttnWaves = 4;   // waves of a workgroup: a chunk's tiles are dealt to them in turn

IQ_HD uint32_t attn_tiles(int32_t len) { return (uint32_t(len) + kAttnTile - 1) / kAttnTile; }

// Tiles of a chunk, `total` tiles of all sequences with `heads` head tiles
// each (total * heads < 2^31): the least, and the next one to try.
constexpr int kAttnTries = 6;
IQ_HD uint32_t attn_chunk_tiles(uint32_t total, uint32_t heads, uint32_t target) {
    const uint32_t c = (total * heads + target - 1) / target;
    return c < uint32_t(kAttnWaves) ? uint32_t(kAttnWaves) : c;
}
IQ_HD uint32_t attn_more_tiles(uint32_t c, uint32_t least) { return c + (least + 7) / 8; }

// Of the sizes tried, least and kAttnTries - 1 behind it, with items[i] chunks
// of all sequences each: the first that is at most `target` work items, or the
// one behind the last.
IQ_HD uint32_t attn_pick_tiles(uint32_t least, const uint32_t (&items)[kAttnTries], uint32_t heads, uint32_t target) {
    uint32_t c = least;
    for (int i = 0; i < kAttnTries; i++) {
        if (items[i] * heads <= target) break;
        c = attn_more_tiles(c, least);
    }
    return c;
}

// A sequence's chunks; the kernels have them from attn_chunks_by.
IQ_HD uint32_t attn_chunks(uint32_t tiles, uint32_t c) { return tiles <= c ? 1 : (tiles + c - 1) / c; }

// The same with 1 / c: (tiles - 1/2) / c + 1 lies at least 1 / 2c from a whole
// number, and its error (2^-46 of at most 2^26 / c, from a reciprocal of 23 bits,
// `near`, and a Newton step) is far less.  An integer division takes five times
// as long.
IQ_HD double attn_rcp(uint32_t c, double near) {
    const double x = double(c);
    return __builtin_fma(near, __builtin_fma(-x, near, 1.0), near);
}
IQ_HD uint32_t attn_chunks_by(uint32_t tiles, uint32_t c, double rcp) {
    return tiles <= c ? 1 : uint32_t(__builtin_fma(double(tiles) - 0.5, rcp, 1.0));
}

// Bounds over all lengths up to `cap` tokens: work items, and those of
// sequences with more than one chunk (which have a partial result each).
// chunks <= tiles / C + 1 each, C >= total * heads / target; a sequence of
// more than one chunk has tiles > C, so at most 2 tiles / C of them.
inline int64_t attn_max_items(int64_t B, int64_t heads, int64_t cap, int64_t target) {
    const int64_t most = (int64_t(attn_tiles(int32_t(cap))) + kAttnWaves - 1) / kAttnWaves;
    return std::min(B * heads * most, target + B * heads);
}
inline int64_t attn_max_partials(int64_t target) { return 2 * target; }

}  // namespace iq
