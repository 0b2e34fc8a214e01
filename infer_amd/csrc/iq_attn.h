// iq_attn.h -- what the attention kernels of iq_attn.hip (16-bit caches) and
// iq_attn8.hip (8-bit ones) share: a batch's tokens split over workgroups,
// fp32 operands cut into 16-bit terms, and the join of the chunks' results.
#pragma once

#include <algorithm>

#include "iq_attn_plan.h"
#include "iq_kv.h"

namespace iq {

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));

struct AttnArgs {
    KvView c;
    KvTable t;
    const float* q;
    float* out;
    int hq, group, B;
    int ht;           // 16-head tiles of a group
    uint32_t nh;      // hk * ht
    uint32_t target;
    int lines;        // heads share cache lines
    float mul;        // scale * log2(e): scores in powers of two
    float* ml;        // [partials][16][2]: a chunk's maximum and sum of every head
    float* part;      // [partials][16][d]
    uint2* plan;      // [B]: chunks, first partial
    float* sc;        // scores [B][hk][cap][group] for the weights, or null
    float* fin;       // [B][hq][2]: maximum and sum of every head, for the weights
    int32_t sinks, visible;  // a window: a sequence's first tokens that are seen, and all that are
    KvScales scales;  // of an 8-bit cache
};

// The maximum of no scores: finite, so that scores of -inf (products past
// fp32's range) and runs without scores count nothing instead of giving NaN.
constexpr float kNone = -3.4e38f;

// 1 / a head's sum.  It is 0 only where every score is -inf: the head's values
// are then 0 times 0 (or NaN, where a value is not finite), its weights 0.
__device__ __forceinline__ float inv_sum(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }

// What a kernel is built for: chunks of whole sequences' tokens, of the tokens
// seen under a window, or whole sequences (under a window or not).  The last as
// an argument instead cost the others 0.3 us of 17 (8-bit, 32 of up to 8192).
enum AttnMode { kAll, kWindow, kWhole };

struct Item {
    int b, n;            // sequence and its length (as given)
    int seen;            // tokens that it sees: n, or under a window fewer
    uint32_t j, c, chunks, first;  // chunk, tiles of a chunk, chunks of the sequence, its first partial
};

__device__ __forceinline__ double chunk_rcp(uint32_t c) { return attn_rcp(c, __builtin_amdgcn_rcp(double(c))); }

// The (sequence, chunk) number w of the batch's plan; false past the last.
// Every wave finds it from the lengths by itself (64 sequences a step).  Under
// a window a sequence counts as the tokens that it sees.  Sizes of a chunk past
// the first are tried at once: one after the other, 24 sequences of 16 heads
// took 2.6 us here.
template <int MODE>
__device__ __forceinline__ bool find_item(const AttnArgs& a, uint32_t w, Item* it) {
    constexpr bool WIN = MODE != kAll;
    if constexpr (MODE == kWhole) {
        if (w >= uint32_t(a.B)) return false;
        const int len = a.t.lens[w];
        *it = Item{int(w), len, min(len, a.visible), 0, attn_tiles(a.visible), 1, 0};
        return true;
    }
    const int lane = threadIdx.x & 63;
    auto length = [&](int b) { return b < a.B ? a.t.lens[b] : 0; };
    auto tiles_of = [&](int n) { return n < 0 || n > a.t.cap ? 0u : attn_tiles(WIN ? min(n, a.visible) : n); };
    int n = length(lane);
    const int n0 = n;
    uint32_t total = lane_of(wave_scan(tiles_of(n)), 63);
    for (int b0 = 64; b0 < a.B; b0 += 64) total += lane_of(wave_scan(tiles_of(length(b0 + lane))), 63);
    const uint32_t least = attn_chunk_tiles(total, a.nh, a.target);
    uint32_t c = least;
    double rcp = chunk_rcp(c);
    auto items_of = [&](int b0, uint32_t size, double r) {
        const uint32_t t = tiles_of(b0 ? length(b0 + lane) : n0);
        return lane_of(wave_scan(b0 + lane < a.B ? attn_chunks_by(t, size, r) : 0), 63);
    };
    if (uint32_t(a.B) * a.nh <= a.target) {
        uint32_t items[kAttnTries] = {};
        for (int b0 = 0; b0 < a.B; b0 += 64) items[0] += items_of(b0, c, rcp);
        if (items[0] * a.nh > a.target) {
            for (int b0 = 0; b0 < a.B; b0 += 64) {
                uint32_t size = least;
#pragma unroll
                for (int i = 1; i < kAttnTries; i++) {
                    size = attn_more_tiles(size, least);
                    items[i] += items_of(b0, size, chunk_rcp(size));
                }
            }
            c = attn_pick_tiles(least, items, a.nh, a.target);
            rcp = chunk_rcp(c);
        }
    }
    uint32_t before = 0, first = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        if (b0) n = length(b0 + lane);
        const uint32_t k = b0 + lane < a.B ? attn_chunks_by(tiles_of(n), c, rcp) : 0;
        const uint32_t upto = wave_scan(k), many = k > 1 ? k : 0, pupto = wave_scan(many);
        const uint64_t past = __ballot(w < before + upto);
        if (past) {
            const int l = __builtin_ctzll(past);
            it->b = b0 + l;
            it->n = __builtin_amdgcn_readlane(n, l);
            it->seen = WIN ? min(it->n, a.visible) : it->n;
            it->chunks = lane_of(k, l);
            it->j = w - before - (lane_of(upto, l) - it->chunks);
            it->first = first + lane_of(pupto, l) - lane_of(many, l);
            it->c = c;
            return true;
        }
        before += lane_of(upto, 63);
        first += lane_of(pupto, 63);
    }
    return false;
}

// ------------------------------------------------------- operands of q and p
template <int TYPE>
struct Terms;

// x = t0 + t1 + t2 exactly, each the upper 16 bits of what is left.
template <>
struct Terms<IQ_KV_BF16> {
    static constexpr int N = 3;
    static constexpr float kUp = 0.0f;
    static __device__ __forceinline__ void cut(const float (&x)[8], s16x8_t (&t)[N]) {
        float r[8];
#pragma unroll
        for (int i = 0; i < 8; i++) r[i] = x[i];
#pragma unroll
        for (int k = 0; k < N; k++) {
            u32x4_t u;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t lo = __float_as_uint(r[2 * i]), hi = __float_as_uint(r[2 * i + 1]);
                u[i] = __builtin_amdgcn_perm(hi, lo, 0x07060302u);
                if (k + 1 < N) {
                    r[2 * i] -= __uint_as_float(lo & 0xffff0000u);
                    r[2 * i + 1] -= __uint_as_float(hi & 0xffff0000u);
                }
            }
            t[k] = __builtin_bit_cast(s16x8_t, u);
        }
    }
    static __device__ __forceinline__ float4_t mma(s16x8_t a, s16x8_t b, float4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b),
                                                       c, 0, 0, 0);
    }
};

// x = t0 + t1, off by at most 2^-23 of x (each term rounds to 11 bits), and by
// 2^-25 where t1 is subnormal.  p is scaled by 2^12 (and its sum with it), which
// makes the latter 2^-37 of the largest p.
template <>
struct Terms<IQ_KV_F16> {
    static constexpr int N = 2;
    static constexpr float kUp = 12.0f;
    static __device__ __forceinline__ void cut(const float (&x)[8], s16x8_t (&t)[N]) {
        half8_t h, l;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            h[i] = _Float16(x[i]);
            l[i] = _Float16(x[i] - float(h[i]));
        }
        t[0] = __builtin_bit_cast(s16x8_t, h);
        t[1] = __builtin_bit_cast(s16x8_t, l);
    }
    static __device__ __forceinline__ float4_t mma(s16x8_t a, s16x8_t b, float4_t c) {
        return mfma16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c);
    }
};

// The split kernel of an 8-bit cache (iq_attn8.hip), and for how many workgroups
// of it a CU the batch is split (no more than run at once).
void launch_attn8(const AttnArgs& a, AttnMode mode, unsigned grid, hipStream_t s);
int attn8_groups(int head_dim);

}  // namespace iq
