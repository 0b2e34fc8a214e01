// iq_kv8.hip -- tokens added behind what sequences have cached, with head norms
// and rotary embedding, to caches of any type (8-bit ones with a scale for each
// block of tokens and head), and cached tokens read back.
//
// Both move bytes; what they take beyond that is latency.  One token each of 16
// sequences (28 query and 2 x 4 cached heads, e4m3) 4.0 us, of which an empty launch
// is 1.4 and three dependent loads (length, page id, scale) most of the rest; 945
// tokens in runs (int8, blocks of 32) 9.7 us for 32 MB, 2.5 us and 4.8 TB/s by what
// 2950 take (23.2), a large copy's rate; 684 with norms (12 + 2 x 2 heads, e4m3,
// blocks of 8) 5.9.  Into a bf16 cache, calls of a graph: the 945 tokens 7.7 us (33 MB,
// 4.3 TB/s), 2048 in one run 15.3 (4.7 TB/s; int8 in blocks of 8 to 64 14.1 to 15.4).
// Reading back 24155 tokens of 4 e4m3 heads as bf16: 16.7 us for 74 MB (4.4 TB/s).
//
// A scale that grows has its block's older codes read and written: the 16 tokens
// 5.9 us in int8 blocks of 16 (3.3 where none grows), 13.3 in blocks of 64, 43 of 256, by
// the threads of one row; in runs, where a workgroup has them, 4 x 200 tokens behind
// half a block 10.6 either way in blocks of 16, 24.0 and 22.1 of 256.  A block of a
// head is one workgroup's: with few large ones it goes through them in many steps
// (2048 tokens in blocks of 128 20.7 us, of 256 35, of 1024 125).
#include <algorithm>

#include "iq_extend_plan.h"
#include "iq_kv.h"

namespace iq {
namespace {

// A thread has 8 values of a row of head_dim values, W threads a row (head_dim
// rounded up to 8 W): two runs of 4, the halves of 4 rotary pairs, or
// neighbours.
constexpr int kThreads = 256;
constexpr int kSpan = 16;      // tokens of a 16-bit cache's unit
constexpr int kMaxHeads = 16;  // heads of a workgroup
constexpr int kHeld = 4;       // rows that a thread can hold

// Things of `groups` workgroups each, from the one that a launch begins with:
// 32-bit divisions in the kernels, by multiplication.
struct Parts {
    int64_t first;       // thing
    uint32_t group;      // of the first workgroup
    uint32_t groups;
    PageDiv div;
};
struct Part {
    int64_t thing;
    uint32_t group;
};
__device__ __forceinline__ Part part_of(const Parts& p, uint32_t block) {
    const uint32_t x = p.group + block, n = page_of(x, p.div);
    return {p.first + n, x - n * p.groups};
}

struct ExtendArgs {
    const float *q, *k, *v;
    const uint16_t *q_norm, *k_norm;
    const int64_t* pos;
    const double* freqs;
    float* qo;
    float eps;
    double inv_d;  // 1 / head_dim
    int hq, rot, B;
    int64_t T;
    KvView c;
    KvScales sc;
    KvTable t;
    const int32_t* starts;
    int span;             // tokens of a unit
    PageDiv span_div;
    Parts cached;         // units x groups of their heads (one token each: tokens x groups of all heads)
    Parts queries;        // tokens x groups of query heads, behind them
    int heads;            // of a unit's group
    PageDiv heads_div, last_div;  // by heads, and by those of the last group
    uint32_t rest;        // workgroups of this launch that are the cache's
};

template <int W, typename V, typename F>
__device__ __forceinline__ V over_row(V v, F f) {
#pragma unroll
    for (int o = W / 2; o > 0; o /= 2) v = f(v, __shfl_xor(v, o));
    return v;
}

// The uth unit of the batch, false past the last.  Every wave finds it from
// the lengths and starts by itself (64 sequences a step).
__device__ __forceinline__ bool find_unit(const ExtendArgs& a, uint32_t u, int* seq, Unit* unit) {
    const int lane = threadIdx.x & 63;
    uint32_t before = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const int b = min(b0 + lane, a.B - 1), len = a.t.lens[b];
        NewTokens n = new_tokens(a.starts[b], a.starts[b + 1], len, int32_t(a.T), a.t.cap);
        if (b0 + lane >= a.B) n.count = 0;
        const uint32_t k = units_of(len, n.count, a.span_div), upto = before + wave_scan(k);
        const uint64_t past = __ballot(u < upto);
        if (past) {
            const int l = __builtin_ctzll(past);
            const NewTokens mine{__builtin_amdgcn_readlane(n.row, l), __builtin_amdgcn_readlane(n.count, l)};
            *seq = b0 + l;
            *unit = unit_at(u - (lane_of(upto, l) - lane_of(k, l)), __builtin_amdgcn_readlane(len, l), mine, a.span, a.span_div);
            return unit->count > 0;
        }
        before = lane_of(upto, 63);
    }
    return false;
}

// 4 values of any alignment (their own).
typedef float float4u_t __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t ushort4u_t __attribute__((ext_vector_type(4), aligned(2)));

// A thread's two runs of 4 values of a row.  A thread past the row's end (on
// false) reads the row's first ones and takes them as 0.
struct Runs {
    int e0, e1;
    bool turn, on;
};
__device__ __forceinline__ Runs runs_of(int i, int rot, int d) {
    Runs r;
    r.on = i * 2 < d;
    if (!r.on) i = 0;
    r.turn = i < rot / 2;
    r.e0 = r.turn ? i : rot + (i - rot / 2) * 2;
    r.e1 = r.turn ? i + rot / 2 : r.e0 + 4;
    return r;
}

__device__ __forceinline__ void load_row(const float* src, const Runs& p, float (&x)[8]) {
    const float4u_t a = *reinterpret_cast<const float4u_t*>(src + p.e0), b = *reinterpret_cast<const float4u_t*>(src + p.e1);
#pragma unroll
    for (int r = 0; r < 4; r++) {
        x[r] = p.on ? a[r] : 0.0f;
        x[4 + r] = p.on ? b[r] : 0.0f;
    }
}

__device__ __forceinline__ void store_row(float* dst, const Runs& p, const float (&x)[8]) {
    if (!p.on) return;
    *reinterpret_cast<float4u_t*>(dst + p.e0) = float4u_t{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<float4u_t*>(dst + p.e1) = float4u_t{x[4], x[5], x[6], x[7]};
}

// x / sqrt(mean(x^2) + eps) * norm; the squares and their root in 64 bits: no x
// in fp32's range over- or underflows.  inv_d = 1 / d.
template <int W>
__device__ __forceinline__ void norm_row(float (&x)[8], const Runs& p, const uint16_t* norm, float eps, double inv_d) {
    const ushort4u_t n0 = *reinterpret_cast<const ushort4u_t*>(norm + p.e0), n1 = *reinterpret_cast<const ushort4u_t*>(norm + p.e1);
    double ss = 0.0;
#pragma unroll
    for (int r = 0; r < 8; r++) ss = fma(double(x[r]), double(x[r]), ss);
    ss = over_row<W>(ss, [](double u, double v) { return u + v; });
    // 1 / sqrt by a Newton step, which is no number at 0 and infinity
    const double mean = fma(ss, inv_d, double(eps)), r0 = __builtin_amdgcn_rsq(mean);
    const double r1 = fma(0.5 * r0, fma(-mean * r0, r0, 1.0), r0), inv = r1 == r1 ? r1 : r0;
#pragma unroll
    for (int r = 0; r < 8; r++) x[r] = float(x[r] * inv) * bf16_to_f32(r < 4 ? n0[r] : n1[r - 4]);
}

// Cosine and sine of pos * freq.  The angle is reduced to a part of a quarter turn
// in 64 bits (in 32 a far position's has lost its last bits), y in -pi/4..pi/4;
// there the series up to y^9 and y^10 are off by less than 2^-29.
__device__ __forceinline__ float2 angle(double pos, double freq) {
    double t = pos * freq * 0.15915494309189533577;
    t = (t - rint(t)) * 4.0;
    const double quarter = rint(t);
    const float y = float(t - quarter) * 1.57079632679489661923f, z = y * y;
    const float s = y * fmaf(z, fmaf(z, fmaf(z, fmaf(z, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), 1.0f);
    const float c = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
    const int q = int(quarter);
    const float a = q & 1 ? s : c, b = q & 1 ? c : s;
    return make_float2((q + 1) & 2 ? -a : a, q & 2 ? -b : b);
}

// The pairs turned by w.
__device__ __forceinline__ void turn_row(float (&x)[8], const Runs& p, const float2 (&w)[4]) {
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const float u = x[r], v = x[4 + r];
        x[r] = p.turn ? u * w[r].x - v * w[r].y : u;
        x[4 + r] = p.turn ? v * w[r].x + u * w[r].y : v;
    }
}

template <int W>
__device__ __forceinline__ uint32_t largest(const float (&x)[8]) {  // |x|'s bits: NaN above infinity
    uint32_t big = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) big = max(big, __float_as_uint(fabsf(x[i])));
    return over_row<W>(big, [](uint32_t u, uint32_t v) { return max(u, v); });
}

template <int TYPE>
constexpr float kMostCode = TYPE == IQ_KV_I8 ? 127.0f : 448.0f;

// A thread's values as codes (or 16-bit values), to nearest even; s: the
// block's scale.
template <int TYPE>
__device__ __forceinline__ void put8(char* row, const Runs& p, const float (&x)[8], float s) {
#pragma unroll
    for (int half = 0; half < 2; half++) {
        const int e = half ? p.e1 : p.e0;
        if constexpr (TYPE == IQ_KV_I8 || TYPE == IQ_KV_E4M3) {
            float c[4];
#pragma unroll
            for (int r = 0; r < 4; r++)  // (no scale: zeros, and what a NaN block holds)
                c[r] = s > 0.0f ? fminf(fmaxf(x[half * 4 + r] / s, -kMostCode<TYPE>), kMostCode<TYPE>) : 0.0f;
            uint32_t u;
            if constexpr (TYPE == IQ_KV_I8) {
                u = 0;
#pragma unroll
                for (int r = 0; r < 4; r++) u |= (uint32_t(int(rintf(c[r]))) & 255u) << (8 * r);
            } else {
                const int v = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
                u = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], v, true));
            }
            *reinterpret_cast<uint32_t*>(row + e) = u;
        } else {
            uint2 u;
            u.x = f32_to_kv<TYPE>(x[half * 4]) | uint32_t(f32_to_kv<TYPE>(x[half * 4 + 1])) << 16;
            u.y = f32_to_kv<TYPE>(x[half * 4 + 2]) | uint32_t(f32_to_kv<TYPE>(x[half * 4 + 3])) << 16;
            *reinterpret_cast<uint2*>(row + 2 * e) = u;
        }
    }
}

// The scale of a block with scale `old` (0: a new one) that receives values up
// to the one with these bits, and how often it doubles.
template <int TYPE>
__device__ __forceinline__ float new_scale(float old, uint32_t bits, int* up) {
    const float big = __uint_as_float(bits);
    *up = 0;
    if (!(big < INFINITY) || !(fabsf(old) < INFINITY)) return __builtin_nanf("");
    if (!(old > 0.0f)) return big > 0.0f ? fmaxf(big / kMostCode<TYPE>, 0x1p-126f) : 0.0f;
    // the ratio in 64 bits: exact where it is 1, 2, 4, ...
    const double ratio = double(big) / (double(kMostCode<TYPE>) * double(old));
    if (!(ratio > 1.0)) return old;
    int e;
    const double f = frexp(ratio, &e);
    *up = f == 0.5 ? e - 1 : e;
    return ldexpf(old, *up);
}

// 4 codes halved `up` times, to nearest even.
template <int TYPE>
__device__ __forceinline__ uint32_t halved4(uint32_t u, int up) {
    float c[4];
    if constexpr (TYPE == IQ_KV_I8) {
#pragma unroll
        for (int r = 0; r < 4; r++) c[r] = ldexpf(float(int8_t(u >> (8 * r))), -up);
        uint32_t v = 0;
#pragma unroll
        for (int r = 0; r < 4; r++) v |= (uint32_t(int(rintf(c[r]))) & 255u) << (8 * r);
        return v;
    } else {
        c[0] = ldexpf(__builtin_amdgcn_cvt_f32_fp8(u, 0), -up);
        c[1] = ldexpf(__builtin_amdgcn_cvt_f32_fp8(u, 1), -up);
        c[2] = ldexpf(__builtin_amdgcn_cvt_f32_fp8(u, 2), -up);
        c[3] = ldexpf(__builtin_amdgcn_cvt_f32_fp8(u, 3), -up);
        const int v = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
        return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], v, true));
    }
}

// `rows` rows of 16 byte pieces from `base`, halved, by `threads` threads.
template <int TYPE>
__device__ __forceinline__ void halve_rows(char* base, int rows, int d, uint32_t stride, int up, int first, int threads) {
    const int per = d / 16;
    const Piece step = piece_of(threads, per);
#pragma unroll 4
    for (Piece p = piece_of(first, per); p.row < rows; p = piece_behind(p, step, per)) {
        u32x4_t* at = reinterpret_cast<u32x4_t*>(base + uint64_t(uint32_t(p.row)) * stride + p.col * 16);
        u32x4_t x = *at;
#pragma unroll
        for (int c = 0; c < 4; c++) x[c] = halved4<TYPE>(x[c], up);
        *at = x;
    }
}

// One token a sequence: a workgroup per kRows rows of a token (query, key, value
// heads), W threads a row, which have all that the row's block needs: no barrier,
// and nothing between the loads that they could wait for (rows, angles and the
// chain of length, page id and scale are requested together).
template <int TYPE, int W>
__global__ __launch_bounds__(kThreads) void extend_one_kernel(ExtendArgs a) {
    constexpr bool kCodes = TYPE == IQ_KV_I8 || TYPE == IQ_KV_E4M3;
    constexpr int kSize = kCodes ? 1 : 2, kRows = kThreads / W;
    const int tid = threadIdx.x, d = a.c.d, heads = a.hq + 2 * a.c.hk;
    const Part part = part_of(a.cached, blockIdx.x);
    const uint32_t t = uint32_t(part.thing);
    const int h = int(part.group) * kRows + tid / W;
    if (h >= heads) return;
    const bool is_q = h < a.hq, is_k = !is_q && h < a.hq + a.c.hk;
    const uint32_t j = uint32_t(is_q ? h : is_k ? h - a.hq : h - a.hq - a.c.hk);
    const int n = a.t.lens[t];
    const Runs p = runs_of(tid % W * 4, is_q || is_k ? a.rot : 0, d);
    const int64_t at = (int64_t(t) * (is_q ? a.hq : a.c.hk) + j) * d;
    float x[8];
    load_row((is_q ? a.q : is_k ? a.k : a.v) + at, p, x);
    double pos = 0.0, freqs[4] = {};
    if (p.turn) {
        pos = double(a.pos[t]);
#pragma unroll
        for (int r = 0; r < 4; r++) freqs[r] = a.freqs[p.e0 + r];
    }
    const bool inside = n >= 0 && n < a.t.cap;
    const uint32_t tok = inside ? uint32_t(n) : 0, page = page_of(tok, a.c.div), slot = tok - page * uint32_t(a.c.ps);
    const int32_t id = a.t.table[t * a.t.ld + page];
    const bool live = inside && id >= 0 && id < a.c.pages;
    const uint32_t pid = live ? uint32_t(id) : 0;
    int older = 0;
    float* scale = nullptr;
    float old = 0.0f;
    if constexpr (kCodes) {
        scale = (is_k ? a.sc.k : a.sc.v) + kv_scale(a.sc, pid, slot, is_q ? 0 : j);
        older = int(slot - page_of(slot, a.sc.div) * uint32_t(a.sc.block));
        old = *scale;
        if (older == 0) old = 0.0f;
    }
    float2 turn[4];
    if (p.turn) {
#pragma unroll
        for (int r = 0; r < 4; r++) turn[r] = angle(pos, freqs[r]);
    }
    const uint16_t* norm = is_q ? a.q_norm : is_k ? a.k_norm : nullptr;
    if (norm) norm_row<W>(x, p, norm, a.eps, a.inv_d);
    turn_row(x, p, turn);
    if (is_q) {
        store_row(a.qo + at, p, x);
        return;
    }
    if (!live) return;
    char* row = const_cast<char*>(is_k ? a.c.k : a.c.v) + kSize * kv_element(a.c, pid, slot, j);
    if constexpr (kCodes) {
        int up;
        const float s = new_scale<TYPE>(old, largest<W>(x), &up);
        if (p.on) put8<TYPE>(row, p, x, s);
        if (tid % W == 0 && (older == 0 || !(s == old))) *scale = s;
        if (up) halve_rows<TYPE>(row - uint64_t(uint32_t(older)) * a.c.sstr, older, d, a.c.sstr, up, tid % W, W);
    } else {
        if (p.on) put8<TYPE>(row, p, x, 0.0f);
    }
}

// Runs of tokens: one workgroup per unit (a block's new tokens, or kSpan tokens of
// a 16-bit cache) and group of its heads (key heads, then value heads), and one per
// token and up to 2 kRows query heads.  An 8-bit cache's workgroup makes its rows,
// finds each head's largest value, settles the scales, and stores the rows (made
// a second time if there are more than its threads hold); where a scale grew, it
// halves the older tokens' codes.  No other workgroup touches these rows and
// scales.
template <int TYPE, int W>
__global__ __launch_bounds__(kThreads) void extend_kernel(ExtendArgs a) {
    constexpr bool kCodes = TYPE == IQ_KV_I8 || TYPE == IQ_KV_E4M3;
    constexpr int kSize = kCodes ? 1 : 2, kRows = kThreads / W;
    __shared__ __align__(16) float2 cs[128];
    __shared__ uint32_t most[kMaxHeads];
    __shared__ float scale[kMaxHeads];
    __shared__ int ups[kMaxHeads];
    const int tid = threadIdx.x, d = a.c.d, mine = tid / W;
    const Runs pk = runs_of(tid % W * 4, a.rot, d), pv = runs_of(tid % W * 4, 0, d);
    if (blockIdx.x >= a.rest) {
        // (two rows a thread, requested ahead of the angles that they share)
        const Part part = part_of(a.queries, blockIdx.x - a.rest);
        const int64_t t = part.thing;
        const int h0 = int(part.group) * 2 * kRows + mine;
        const int64_t at = (t * a.hq + h0) * d, next = int64_t(kRows) * d;
        float x[2][8];
#pragma unroll
        for (int i = 0; i < 2; i++)
            if (h0 + i * kRows < a.hq) load_row(a.q + at + i * next, pk, x[i]);
        if (tid < a.rot / 2) cs[tid] = angle(double(a.pos[t]), a.freqs[tid]);
        __syncthreads();
        float2 turn[4];
#pragma unroll
        for (int r = 0; r < 4; r++) turn[r] = pk.turn ? cs[pk.e0 + r] : make_float2(1.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            if (h0 + i * kRows >= a.hq) break;
            if (a.q_norm) norm_row<W>(x[i], pk, a.q_norm, a.eps, a.inv_d);
            turn_row(x[i], pk, turn);
            store_row(a.qo + at + i * next, pk, x[i]);
        }
        return;
    }
    Unit u;
    int seq;
    const Part part = part_of(a.cached, blockIdx.x);
    if (!find_unit(a, uint32_t(part.thing), &seq, &u)) return;
    const int g0 = int(part.group) * a.heads, G = min(a.heads, 2 * a.c.hk - g0), rows = u.count * G;
    const PageDiv by_heads = G == a.heads ? a.heads_div : a.last_div;
    const int32_t* table = a.t.table + seq * a.t.ld;
    auto head = [&](int h) { return uint32_t(h < a.c.hk ? h : h - a.c.hk); };
    auto pool = [&](int h) { return const_cast<char*>(h < a.c.hk ? a.c.k : a.c.v); };
    auto page_id = [&](int tok) { return table[page_of(uint32_t(tok), a.c.div)]; };
    auto there = [&](int32_t id) { return id >= 0 && id < a.c.pages; };
    // Row r of the unit, a token's head: its values and position (requested ahead of
    // what waits for the page), and from these what is stored.
    struct Raw {
        float x[8];
        int64_t pos;
        int k, h;  // token of the unit, head of the 2 hk
    };
    const bool turns = a.rot > 0 && g0 < a.c.hk && pk.turn;
    double freqs[4] = {};
    if (turns) {
#pragma unroll
        for (int r = 0; r < 4; r++) freqs[r] = a.freqs[pk.e0 + r];
    }
    auto get = [&](int r, Raw& y) {
        y.k = int(page_of(uint32_t(r), by_heads));
        y.h = g0 + r - y.k * G;
        const int64_t t = int64_t(u.row) + y.k;
        load_row((y.h < a.c.hk ? a.k : a.v) + (t * a.c.hk + head(y.h)) * d, y.h < a.c.hk ? pk : pv, y.x);
        y.pos = turns ? a.pos[t] : 0;
    };
    auto make = [&](Raw& y) {
        if (y.h >= a.c.hk) return;
        float2 turn[4];
#pragma unroll
        for (int i = 0; i < 4; i++) turn[i] = angle(double(y.pos), freqs[i]);
        if (a.k_norm) norm_row<W>(y.x, pk, a.k_norm, a.eps, a.inv_d);
        turn_row(y.x, pk, turn);
    };
    const int32_t first_id = kCodes ? page_id(u.begin) : 0;  // (a block lies in one page)
    const uint32_t slot0 = uint32_t(u.begin) - page_of(uint32_t(u.begin), a.c.div) * uint32_t(a.c.ps);
    auto store = [&](const Raw& y) {
        const int h = y.h, tok = u.tok + y.k;
        const Runs& p = h < a.c.hk ? pk : pv;
        uint32_t slot = slot0 + uint32_t(tok - u.begin);
        int32_t id = first_id;
        if constexpr (!kCodes) {
            slot = uint32_t(tok) - page_of(uint32_t(tok), a.c.div) * uint32_t(a.c.ps);
            id = page_id(tok);
            if (!there(id)) return;
        }
        if (p.on) put8<TYPE>(pool(h) + kSize * kv_element(a.c, uint32_t(id), slot, head(h)), p, y.x, kCodes ? scale[h - g0] : 0.0f);
    };
    if constexpr (!kCodes) {
        for (int r = mine; r < rows; r += kRows) {
            Raw y;
            get(r, y);
            make(y);
            store(y);
        }
        return;
    }
    Raw held[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; i++)
        if (mine + i * kRows < rows) get(mine + i * kRows, held[i]);
    if (!there(first_id)) return;
    float* at = nullptr;
    float old = 0.0f;
    if (tid < G) {
        most[tid] = 0;
        at = (g0 + tid < a.c.hk ? a.sc.k : a.sc.v) + kv_scale(a.sc, uint32_t(first_id), slot0, head(g0 + tid));
        if (u.tok > u.begin) old = *at;
    }
    __syncthreads();
    auto note = [&](const Raw& y) {
        const uint32_t big = largest<W>(y.x);
        if (tid % W == 0) atomicMax(&most[y.h - g0], big);
    };
#pragma unroll
    for (int i = 0; i < kHeld; i++) {
        if (mine + i * kRows < rows) {
            make(held[i]);
            note(held[i]);
        }
    }
    for (int r = mine + kHeld * kRows; r < rows; r += kRows) {
        Raw y;
        get(r, y);
        make(y);
        note(y);
    }
    __syncthreads();
    if (tid < G) {
        int up;
        const float s = new_scale<TYPE>(old, most[tid], &up);
        scale[tid] = s;
        ups[tid] = up;
        if (u.tok == u.begin || !(s == old)) *at = s;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kHeld; i++)
        if (mine + i * kRows < rows) store(held[i]);
    for (int r = mine + kHeld * kRows; r < rows; r += kRows) {
        Raw y;
        get(r, y);
        make(y);
        store(y);
    }
    if (u.tok == u.begin) return;
    for (int h = g0; h < g0 + G; h++) {
        if (ups[h - g0] == 0) continue;
        halve_rows<TYPE>(pool(h) + kv_element(a.c, uint32_t(first_id), slot0, head(h)), u.tok - u.begin, d, a.c.sstr,
                         ups[h - g0], tid, kThreads);
    }
}

// -------------------------------------------------------------------- read
struct ReadArgs {
    KvView c;
    KvScales sc;
    KvTable t;               // (lens: first tokens, or null)
    const int32_t* starts;
    int B, rows;             // rows of a workgroup, at most kReadRows
    int64_t T, r0;           // first row of this launch
    char *k, *v;
};

constexpr int kReadRows = 16;

// N values from their codes (or 16-bit values), N * their size bytes.
template <int TYPE, int N>
__device__ __forceinline__ void numbers(const char* src, float s, float (&y)[N]) {
    if constexpr (TYPE == IQ_KV_I8 || TYPE == IQ_KV_E4M3) {
        uint32_t x[N / 4];
        __builtin_memcpy(x, __builtin_assume_aligned(src, N), N);
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            if constexpr (TYPE == IQ_KV_I8) {
#pragma unroll
                for (int r = 0; r < 4; r++) y[i * 4 + r] = float(int8_t(x[i] >> (8 * r))) * s;
            } else {
                y[i * 4 + 0] = __builtin_amdgcn_cvt_f32_fp8(x[i], 0) * s;
                y[i * 4 + 1] = __builtin_amdgcn_cvt_f32_fp8(x[i], 1) * s;
                y[i * 4 + 2] = __builtin_amdgcn_cvt_f32_fp8(x[i], 2) * s;
                y[i * 4 + 3] = __builtin_amdgcn_cvt_f32_fp8(x[i], 3) * s;
            }
        }
    } else {
        uint32_t x[N / 2];
        __builtin_memcpy(x, __builtin_assume_aligned(src, 2 * N), 2 * N);
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            y[i * 2] = kv_to_f32<TYPE>(uint16_t(x[i]));
            y[i * 2 + 1] = kv_to_f32<TYPE>(uint16_t(x[i] >> 16));
        }
    }
}

// One workgroup per `rows` rows of the outputs.  Its first wave finds the rows'
// places, a lane each (a row's sequence is the number of sequences that end at or
// before it); then a thread has one 16-byte column of the outputs' rows, k's and v's
// (or several, where a row has more than the workgroup threads), and goes
// through the rows, so that neighbouring threads write neighbouring bytes.
template <int TYPE, int OUT>
__global__ __launch_bounds__(kThreads) void read_kernel(ReadArgs a) {
    constexpr bool kCodes = TYPE == IQ_KV_I8 || TYPE == IQ_KV_E4M3;
    constexpr int kSize = kCodes ? 1 : 2, kOut = OUT == IQ_READ_F32 ? 4 : 2, N = 16 / kOut;
    struct Place {
        int64_t at, scale;  // at: -1 NaN, -2 none
    };
    __shared__ Place places[kReadRows];
    const int tid = threadIdx.x, lane = tid & 63;
    const int64_t r0 = a.r0 + int64_t(blockIdx.x) * a.rows;
    if (tid < 64) {
        int b = 0;
        for (int b0 = 0; b0 < a.B; b0 += 64) {
            const int end = a.starts[min(b0 + lane, a.B - 1) + 1];
            for (int r = 0; r < a.rows; r++) {
                const int n = __popcll(__ballot(b0 + lane < a.B && end <= r0 + r));
                if (lane == r) b += n;
            }
        }
        if (lane < a.rows) {
            const int64_t row = r0 + lane;
            Place p{-2, 0};
            const int start = a.starts[min(b, a.B)];
            if (row < a.T && b < a.B && row >= start) {
                const int64_t tok = (a.t.lens ? int64_t(a.t.lens[b]) : 0) + (row - start);
                p.at = -1;
                if (tok >= 0 && tok < a.t.cap) {
                    const uint32_t g = page_of(uint32_t(tok), a.c.div), slot = uint32_t(tok) - g * uint32_t(a.c.ps);
                    const int32_t id = a.t.table[b * a.t.ld + g];
                    if (id >= 0 && id < a.c.pages) {
                        p.at = kv_element(a.c, uint32_t(id), slot, 0);
                        if (kCodes) p.scale = kv_scale(a.sc, uint32_t(id), slot, 0);
                    }
                }
            }
            places[lane] = p;
        }
    }
    __syncthreads();
    const int per = a.c.d / N, half = a.c.hk * per, pools = (a.k != nullptr) + (a.v != nullptr);
    const int cols = half * pools, way = min(cols, kThreads), lanes = kThreads / way;
    if (tid >= way * lanes) return;
    for (int x = tid % way; x < cols; x += way) {
        const bool is_v = x >= half || !a.k;
        const int u = x >= half ? x - half : x, h = u / per, e = (u - h * per) * N;
        const char* src = (is_v ? a.c.v : a.c.k) + kSize * (int64_t(uint64_t(uint32_t(h)) * a.c.hstr) + e);
        const float* scales = (is_v ? a.sc.v : a.sc.k) + int64_t(uint64_t(uint32_t(h)) * a.sc.hstr);
        char* to = (is_v ? a.v : a.k) + (r0 * half + u) * 16;
#pragma unroll 4
        for (int r = tid / way; r < a.rows; r += lanes) {
            const Place p = places[r];
            if (p.at == -2) continue;
            const int64_t from = p.at < 0 ? 0 : p.at;
            const float s = p.at < 0 ? __builtin_nanf("") : kCodes ? scales[p.scale] : 1.0f;
            float y[N];
            numbers<TYPE, N>(src + kSize * from, s, y);
            // (the product is fp32's: without this its rounding is merged with fp16's)
#pragma unroll
            for (int k = 0; k < N; k++) asm("" : "+v"(y[k]));
            u32x4_t out;
            if constexpr (OUT == IQ_READ_F32) {
#pragma unroll
                for (int k = 0; k < 4; k++) out[k] = __float_as_uint(y[k]);
            } else {
                constexpr int T16 = OUT == IQ_READ_BF16 ? IQ_KV_BF16 : IQ_KV_F16;
#pragma unroll
                for (int k = 0; k < 4; k++) out[k] = f32_to_kv<T16>(y[2 * k]) | uint32_t(f32_to_kv<T16>(y[2 * k + 1])) << 16;
            }
            if (!kCodes && p.at < 0) {  // (codes: the scale)
                constexpr uint32_t nan = OUT == IQ_READ_F32 ? 0x7fc00000u : OUT == IQ_READ_BF16 ? 0x7fc07fc0u : 0x7e007e00u;
                out = u32x4_t{nan, nan, nan, nan};
            }
            *reinterpret_cast<u32x4_t*>(to + int64_t(r) * half * 16) = out;
        }
    }
}

template <int TYPE, int W>
void launch_rows(const ExtendArgs& a, unsigned grid, hipStream_t s) {
    if (a.starts) extend_kernel<TYPE, W><<<grid, kThreads, 0, s>>>(a);
    else extend_one_kernel<TYPE, W><<<grid, kThreads, 0, s>>>(a);
}

template <int TYPE>
void launch_extend(const ExtendArgs& a, unsigned grid, hipStream_t s) {
    if (a.c.d <= 32) launch_rows<TYPE, 4>(a, grid, s);
    else if (a.c.d <= 64) launch_rows<TYPE, 8>(a, grid, s);
    else if (a.c.d <= 128) launch_rows<TYPE, 16>(a, grid, s);
    else launch_rows<TYPE, 32>(a, grid, s);
}

template <int TYPE>
void launch_read(const ReadArgs& a, int out, unsigned grid, hipStream_t s) {
    if (out == IQ_READ_F32) read_kernel<TYPE, IQ_READ_F32><<<grid, kThreads, 0, s>>>(a);
    else if (out == IQ_READ_BF16) read_kernel<TYPE, IQ_READ_BF16><<<grid, kThreads, 0, s>>>(a);
    else read_kernel<TYPE, IQ_READ_F16><<<grid, kThreads, 0, s>>>(a);
}

constexpr int64_t kMostRows = 0x7fff0000;

}  // namespace
}  // namespace iq

extern "C" {

int iq_kv_extend(const float* q, const float* k, const float* v, int64_t T, int q_heads, const uint16_t* q_norm,
                 const uint16_t* k_norm, float eps, const int64_t* positions, const double* freqs, int rot_dim,
                 const iq_kv* kv, const iq_kv_scales* scales, const int32_t* table, int64_t table_ld,
                 int64_t max_pages, const int32_t* lens, const int32_t* starts, int B, float* q_out, void* stream) {
    iq::ExtendArgs a{};
    int rc = iq::check_any_kv(kv, scales, &a.c, &a.sc);
    if (rc) return rc;
    rc = iq::check_table(a.c, table, table_ld, max_pages, lens, B, &a.t);
    if (rc) return rc;
    if (T < 1 || q_heads < 0 || q_heads > 16384 || (!starts && T != B)) return IQ_ESHAPE;
    if (rot_dim < 0 || rot_dim > a.c.d || rot_dim % 8) return IQ_ESHAPE;
    if ((q_norm || k_norm) && !(eps >= 0.0f && std::isfinite(eps))) return IQ_ESHAPE;
    if (T > iq::kMostRows) return IQ_ETOOLARGE;
    if (!k || !v || (q_heads && (!q || !q_out)) || (rot_dim && (!positions || !freqs))) return IQ_ENULL;
    const int64_t qb = T * q_heads * a.c.d * 4, kb = T * a.c.hk * a.c.d * 4;
    if (q_heads && ((q_out != q && iq::ranges_overlap(q, qb, q_out, qb)) || iq::ranges_overlap(k, kb, q_out, qb) ||
                    iq::ranges_overlap(v, kb, q_out, qb) || iq::meets_cache(q_out, qb, a.c, a.sc)))
        return IQ_EALIAS;
    const bool codes = iq::is_kv8(kv->type);
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_norm = q_norm;
    a.k_norm = k_norm;
    a.eps = eps;
    a.inv_d = 1.0 / a.c.d;
    a.pos = positions;
    a.freqs = freqs;
    a.qo = q_out;
    a.hq = q_heads;
    a.rot = rot_dim;
    a.B = B;
    a.T = T;
    a.starts = starts;
    a.span = codes ? a.sc.block : iq::kSpan;
    a.span_div = iq::page_div(uint32_t(a.span));
    const int rows = iq::kThreads / (a.c.d <= 32 ? 4 : a.c.d <= 64 ? 8 : a.c.d <= 128 ? 16 : 32);
    // workgroups: the cache's units (or tokens), then the query heads
    int64_t cached, all;
    auto parts = [](iq::Parts* p, int64_t n, int64_t groups) {
        p->groups = uint32_t(groups);
        p->div = iq::page_div(p->groups);
        return n * groups;
    };
    if (starts) {
        // as many heads as fill a workgroup's threads once, of the tokens that a unit has
        a.heads = std::min({2 * a.c.hk, iq::kMaxHeads, std::max(1, rows / std::min(a.span, rows))});
        const int groups = (2 * a.c.hk + a.heads - 1) / a.heads;
        a.heads_div = iq::page_div(uint32_t(a.heads));
        a.last_div = iq::page_div(uint32_t(2 * a.c.hk - (groups - 1) * a.heads));
        cached = parts(&a.cached, iq::max_units(T, B, a.span), groups);
        all = cached + (q_heads ? parts(&a.queries, T, (q_heads + 2 * rows - 1) / (2 * rows)) : 0);
    } else {
        cached = all = parts(&a.cached, T, (q_heads + 2 * a.c.hk + rows - 1) / rows);
    }
    const hipStream_t s = static_cast<hipStream_t>(stream);
    for (int64_t w0 = 0; w0 < all; w0 += iq::kMaxGrid256) {
        const unsigned grid = unsigned(std::min(all - w0, iq::kMaxGrid256));
        auto begin = [](iq::Parts* p, int64_t w) {
            p->first = w / p->groups;
            p->group = uint32_t(w % p->groups);
        };
        a.rest = uint32_t(std::max<int64_t>(0, std::min<int64_t>(cached - w0, grid)));
        if (a.rest) begin(&a.cached, w0);
        if (a.rest < grid) begin(&a.queries, std::max<int64_t>(0, w0 - cached));
        switch (kv->type) {
            case IQ_KV_BF16: iq::launch_extend<IQ_KV_BF16>(a, grid, s); break;
            case IQ_KV_F16: iq::launch_extend<IQ_KV_F16>(a, grid, s); break;
            case IQ_KV_I8: iq::launch_extend<IQ_KV_I8>(a, grid, s); break;
            default: iq::launch_extend<IQ_KV_E4M3>(a, grid, s);
        }
    }
    return int(hipGetLastError());
}

int iq_kv_read(const iq_kv* kv, const iq_kv_scales* scales, const int32_t* table, int64_t table_ld, int64_t max_pages,
               const int32_t* first, const int32_t* starts, int B, int64_t T, int out_type, void* k_out, void* v_out,
               void* stream) {
    iq::ReadArgs a{};
    int rc = iq::check_any_kv(kv, scales, &a.c, &a.sc);
    if (rc) return rc;
    rc = iq::check_table(a.c, table, table_ld, max_pages, starts, B, &a.t);
    if (rc) return rc;
    if (out_type < IQ_READ_F32 || out_type > IQ_READ_F16) return IQ_EKIND;
    if (T < 1) return IQ_ESHAPE;
    if (T > iq::kMostRows) return IQ_ETOOLARGE;
    if (!k_out && !v_out) return IQ_ENULL;
    const int64_t bytes = T * a.c.hk * a.c.d * (out_type == IQ_READ_F32 ? 4 : 2);
    if (reinterpret_cast<uintptr_t>(k_out) % 16 || reinterpret_cast<uintptr_t>(v_out) % 16) return IQ_ESHAPE;
    if (iq::ranges_overlap(k_out, bytes, v_out, bytes)) return IQ_EALIAS;
    if (iq::meets_cache(k_out, bytes, a.c, a.sc) || iq::meets_cache(v_out, bytes, a.c, a.sc)) return IQ_EALIAS;
    a.t.lens = first;
    a.starts = starts;
    a.B = B;
    a.T = T;
    a.k = static_cast<char*>(k_out);
    a.v = static_cast<char*>(v_out);
    // few rows: fewer a workgroup, so that they fill the card
    a.rows = T < int64_t(iq::kReadRows) * 4 * iq::device_cu_count() ? 4 : iq::kReadRows;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    for (; a.r0 < T; a.r0 += iq::kMaxGrid256 * a.rows) {
        const unsigned grid = unsigned(std::min((T - a.r0 + a.rows - 1) / a.rows, iq::kMaxGrid256));
        switch (kv->type) {
            case IQ_KV_BF16: iq::launch_read<IQ_KV_BF16>(a, out_type, grid, s); break;
            case IQ_KV_F16: iq::launch_read<IQ_KV_F16>(a, out_type, grid, s); break;
            case IQ_KV_I8: iq::launch_read<IQ_KV_I8>(a, out_type, grid, s); break;
            default: iq::launch_read<IQ_KV_E4M3>(a, out_type, grid, s);
        }
    }
    return int(hipGetLastError());
}

}  // extern "C"
