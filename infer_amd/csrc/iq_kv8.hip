// iq_kv8.hip -- tokens added behind what sequences have cached, with head norms
// and rotary embedding, to caches of any type (8-bit ones with a scale for each
// block of tokens and head), and cached tokens read back.
#include <algorithm>

#include "iq_kv.h"

namespace iq {
namespace {

// A thread has 8 values of a row of head_dim values, W threads a row (head_dim
// rounded up to 8 W): two runs of 4, the halves of 4 rotary pairs, or
// neighbours.
constexpr int kThreads = 256;
constexpr int kSpan = 16;     // tokens of a 16-bit cache's unit
constexpr int kChunk = 16;    // tokens whose angles a workgroup holds
constexpr int kMaxHeads = 16; // heads of a workgroup

struct ExtendArgs {
    const float *q, *k, *v;
    const uint16_t *q_norm, *k_norm;
    const int64_t* pos;
    const double* freqs;
    float* qo;
    float eps;
    int hq, rot, B;
    int64_t T;
    KvView c;
    KvScales sc;
    KvTable t;
    const int32_t* starts;
    int span;             // tokens of a unit
    PageDiv span_div;
    uint32_t groups;      // of the 2 hk rows that a token has in the cache
    int heads;            // of a group
    uint32_t qgroups;     // of 16 query heads
    int64_t cached;       // workgroups of the cache's part, then T * qgroups
    int64_t w0;           // first workgroup of this launch
};

template <int W, typename V, typename F>
__device__ __forceinline__ V over_row(V v, F f) {
#pragma unroll
    for (int o = W / 2; o > 0; o /= 2) v = f(v, __shfl_xor(v, o));
    return v;
}

// A new token run of one sequence inside one span of its tokens.
struct Unit {
    int b, tok, count;  // its first token, and how many
    int begin;          // the span's first token
    int64_t row;        // of the first token's q, k, v
};

__device__ __forceinline__ bool find_unit(const ExtendArgs& a, uint32_t u, Unit* it) {
    if (!a.starts) {
        it->b = int(u);
        it->tok = a.t.lens[u];
        it->count = 1;
        it->row = u;
        if (it->tok < 0 || it->tok >= a.t.cap) return false;
        it->begin = int(page_of(uint32_t(it->tok), a.span_div)) * a.span;
        return true;
    }
    const int lane = threadIdx.x & 63;
    uint32_t before = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const int b = min(b0 + lane, a.B - 1);
        const int T = int(a.T), s0 = min(max(a.starts[b], 0), T), s1 = min(a.starts[b + 1], T), L = a.t.lens[b];
        const int n = L < 0 || L >= a.t.cap || b0 + lane >= a.B ? 0 : min(s1 - s0, a.t.cap - L);
        const uint32_t f = page_of(uint32_t(max(L, 0)), a.span_div);
        const uint32_t k = n > 0 ? page_of(uint32_t(L + n - 1), a.span_div) - f + 1 : 0;
        const uint32_t upto = before + wave_scan(k);
        const uint64_t past = __ballot(u < upto);
        if (past) {
            const int l = __builtin_ctzll(past);
            const int len = __builtin_amdgcn_readlane(L, l), cnt = __builtin_amdgcn_readlane(n, l);
            const int s = int(lane_of(f, l) + (u - (lane_of(upto, l) - lane_of(k, l))));
            it->b = b0 + l;
            it->begin = s * a.span;
            it->tok = max(len, it->begin);
            // (in 64 bits: the span behind the last token may end past 2^31)
            it->count = int(min(int64_t(len) + cnt, int64_t(it->begin) + a.span) - it->tok);
            it->row = int64_t(__builtin_amdgcn_readlane(s0, l)) + (it->tok - len);
            return true;
        }
        before = lane_of(upto, 63);
    }
    return false;
}

// A thread's two runs of 4 values of a row.
struct Runs {
    int e0, e1;
    bool turn, on;
};
__device__ __forceinline__ Runs runs_of(int i, int rot, int d) {
    Runs r;
    r.turn = i < rot / 2;
    r.e0 = r.turn ? i : rot + (i - rot / 2) * 2;
    r.e1 = r.turn ? i + rot / 2 : r.e0 + 4;
    r.on = i * 2 < d;
    return r;
}

// One head's row: loaded, normed (norm may be null), turned by cs.
template <int W>
__device__ __forceinline__ void make_row(const float* src, const Runs& p, const uint16_t* norm, float eps, int d,
                                         const float2* cs, float (&y0)[4], float (&y1)[4]) {
    float x0[4], x1[4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        x0[r] = p.on ? src[p.e0 + r] : 0.0f;
        x1[r] = p.on ? src[p.e1 + r] : 0.0f;
    }
    if (norm) {
        // squares and their root in 64 bits: no x in fp32's range over- or underflows
        double ss = 0.0;
#pragma unroll
        for (int r = 0; r < 4; r++) ss += double(x0[r]) * x0[r] + double(x1[r]) * x1[r];
        ss = over_row<W>(ss, [](double u, double v) { return u + v; });
        const double inv = 1.0 / sqrt(ss / d + double(eps));
#pragma unroll
        for (int r = 0; r < 4; r++) {
            x0[r] = float(x0[r] * inv) * bf16_to_f32(p.on ? norm[p.e0 + r] : 0);
            x1[r] = float(x1[r] * inv) * bf16_to_f32(p.on ? norm[p.e1 + r] : 0);
        }
    }
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const float2 w = p.turn ? cs[p.e0 + r] : make_float2(1.0f, 0.0f);
        y0[r] = p.turn ? x0[r] * w.x - x1[r] * w.y : x0[r];
        y1[r] = p.turn ? x1[r] * w.x + x0[r] * w.y : x1[r];
    }
}

// The cosines and sines of `tokens` tokens from row t on (at most kChunk).  The
// angle is reduced to a fraction of a turn in 64 bits: in 32 a far position's
// has lost its last bits.
__device__ __forceinline__ void make_angles(const ExtendArgs& a, int64_t t, int tokens, float2 (*cs)[128]) {
    const int half = a.rot / 2;
    for (int i = threadIdx.x; i < tokens * half; i += kThreads) {
        const int k = i / half, e = i - k * half;
        const double turns = double(a.pos[t + k]) * a.freqs[e] * 0.15915494309189533577;
        const float r = float((turns - rint(turns)) * 6.28318530717958647693);
        cs[k][e] = make_float2(cosf(r), sinf(r));
    }
}

template <int TYPE>
constexpr float kMostCode = TYPE == IQ_KV_I8 ? 127.0f : 448.0f;

// 4 values as codes (or 16-bit values), to nearest even; s: the block's scale.
template <int TYPE>
__device__ __forceinline__ void put4(char* at, const float (&y)[4], float s) {
    if constexpr (TYPE == IQ_KV_I8 || TYPE == IQ_KV_E4M3) {
        float c[4];
#pragma unroll
        for (int r = 0; r < 4; r++)  // (no scale: zeros, and what a NaN block holds)
            c[r] = s > 0.0f ? fminf(fmaxf(y[r] / s, -kMostCode<TYPE>), kMostCode<TYPE>) : 0.0f;
        uint32_t u;
        if constexpr (TYPE == IQ_KV_I8) {
            u = 0;
#pragma unroll
            for (int r = 0; r < 4; r++) u |= (uint32_t(int(rintf(c[r]))) & 255u) << (8 * r);
        } else {
            int v = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
            u = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], v, true));
        }
        *reinterpret_cast<uint32_t*>(at) = u;
    } else {
        uint2 u;
        u.x = f32_to_kv<TYPE>(y[0]) | uint32_t(f32_to_kv<TYPE>(y[1])) << 16;
        u.y = f32_to_kv<TYPE>(y[2]) | uint32_t(f32_to_kv<TYPE>(y[3])) << 16;
        *reinterpret_cast<uint2*>(at) = u;
    }
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

// One workgroup per unit (a block's new tokens, or kSpan tokens of a 16-bit
// cache) and group of its heads (key heads, then value heads), and one per token
// and 16 query heads.  An 8-bit cache's workgroup makes the rows, finds each
// head's largest value, settles the scales, and stores the rows (made a second
// time if there are more than its threads hold); where a scale grew, it halves
// the older tokens' codes.  No other workgroup touches these rows and scales.
template <int TYPE, int W>
__global__ __launch_bounds__(kThreads) void extend_kernel(ExtendArgs a) {
    constexpr bool kCodes = TYPE == IQ_KV_I8 || TYPE == IQ_KV_E4M3;
    constexpr int kSize = kCodes ? 1 : 2, kRows = kThreads / W;
    __shared__ float2 cs[kChunk][128];
    __shared__ uint32_t most[kMaxHeads];
    __shared__ float scale[kMaxHeads];
    __shared__ int ups[kMaxHeads];
    const int tid = threadIdx.x, d = a.c.d, i4 = tid % W * 4;
    const int64_t w = a.w0 + blockIdx.x;
    if (w >= a.cached) {
        const int64_t t = (w - a.cached) / a.qgroups;
        const int h0 = int((w - a.cached) % a.qgroups) * 16, h1 = min(h0 + 16, a.hq);
        make_angles(a, t, 1, cs);
        __syncthreads();
        const Runs p = runs_of(i4, a.rot, d);
        for (int h = h0 + tid / W; h < h1; h += kRows) {
            const int64_t at = (t * a.hq + h) * d;
            float y0[4], y1[4];
            make_row<W>(a.q + at, p, a.q_norm, a.eps, d, cs[0], y0, y1);
            if (!p.on) continue;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                a.qo[at + p.e0 + r] = y0[r];
                a.qo[at + p.e1 + r] = y1[r];
            }
        }
        return;
    }
    Unit u;
    if (!find_unit(a, uint32_t(w / a.groups), &u)) return;
    const int g0 = int(w % a.groups) * a.heads, G = min(a.heads, 2 * a.c.hk - g0), rows = u.count * G;
    const int32_t* table = a.t.table + u.b * a.t.ld;
    // the page and slot of a token; -1 without a page
    auto place = [&](int tok, uint32_t* slot) -> int {
        const uint32_t p = page_of(uint32_t(tok), a.c.div);
        *slot = uint32_t(tok) - p * uint32_t(a.c.ps);
        const int32_t id = table[p];
        return id >= 0 && id < a.c.pages ? id : -1;
    };
    uint32_t slot0 = 0;
    int page = 0;
    float old = 0.0f;
    float* my_scale = nullptr;
    if constexpr (kCodes) {  // (a block lies in one page)
        page = place(u.begin, &slot0);
        if (page < 0) return;
        if (tid < G) {
            const int h = g0 + tid;
            my_scale = (h < a.c.hk ? a.sc.k : a.sc.v) + kv_scale(a.sc, uint32_t(page), slot0, uint32_t(h < a.c.hk ? h : h - a.c.hk));
            if (u.tok > u.begin) old = *my_scale;
            most[tid] = 0;
        }
    }
    const Runs pk = runs_of(i4, a.rot, d), pv = runs_of(i4, 0, d);
    float y0[4], y1[4];
    auto angles = [&](int c0) {
        if (a.rot && g0 < a.c.hk) make_angles(a, u.row + c0, min(kChunk, u.count - c0), cs);
        __syncthreads();
    };
    auto make = [&](int c0, int r) {  // row r of the chunk of tokens from c0 on
        const int k = r / G, h = g0 + r - k * G;
        const int64_t t = u.row + c0 + k;
        if (h < a.c.hk) make_row<W>(a.k + (t * a.c.hk + h) * d, pk, a.k_norm, a.eps, d, cs[k], y0, y1);
        else make_row<W>(a.v + (t * a.c.hk + h - a.c.hk) * d, pv, nullptr, 0.0f, d, cs[k], y0, y1);
    };
    auto store = [&](int c0, int r) {
        const int k = r / G, h = g0 + r - k * G, tok = u.tok + c0 + k;
        uint32_t slot;
        int id = page;
        if constexpr (kCodes) slot = slot0 + uint32_t(tok - u.begin);
        else id = place(tok, &slot);
        const Runs& p = h < a.c.hk ? pk : pv;
        if (id < 0 || !p.on) return;
        char* to = const_cast<char*>(h < a.c.hk ? a.c.k : a.c.v) +
                   kSize * kv_element(a.c, uint32_t(id), slot, uint32_t(h < a.c.hk ? h : h - a.c.hk));
        const float s = kCodes ? scale[h - g0] : 0.0f;
        put4<TYPE>(to + kSize * p.e0, y0, s);
        put4<TYPE>(to + kSize * p.e1, y1, s);
    };
    const int mine = tid / W;
    if constexpr (!kCodes) {
        angles(0);  // (kSpan <= kChunk)
        for (int r = mine; r < rows; r += kRows) {
            make(0, r);
            store(0, r);
        }
        return;
    }
    for (int c0 = 0; c0 < u.count; c0 += kChunk) {
        if (c0) __syncthreads();  // (the angles before are no longer read)
        angles(c0);
        const int n = min(kChunk, u.count - c0) * G;
        for (int r = mine; r < n; r += kRows) {
            make(c0, r);
            uint32_t big = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) big = max(big, max(__float_as_uint(fabsf(y0[i])), __float_as_uint(fabsf(y1[i]))));
            big = over_row<W>(big, [](uint32_t x, uint32_t y) { return max(x, y); });
            if (tid % W == 0) atomicMax(&most[r % G], big);
        }
    }
    __syncthreads();
    if (tid < G) {
        const float big = __uint_as_float(most[tid]);
        float s = old;
        int up = 0;
        if (!(big < INFINITY) || !(fabsf(old) < INFINITY)) {
            s = __builtin_nanf("");
        } else if (!(old > 0.0f)) {
            s = big > 0.0f ? fmaxf(big / kMostCode<TYPE>, 0x1p-126f) : 0.0f;
        } else {
            // the ratio in 64 bits: exact where it is 1, 2, 4, ...
            const double ratio = double(big) / (double(kMostCode<TYPE>) * double(old));
            if (ratio > 1.0) {
                int e;
                const double f = frexp(ratio, &e);
                up = f == 0.5 ? e - 1 : e;
                s = ldexpf(old, up);
            }
        }
        scale[tid] = s;
        ups[tid] = up;
        if (!(s == old) || u.tok == u.begin) *my_scale = s;
    }
    __syncthreads();
    const bool held = rows <= kRows && u.count <= kChunk;
    for (int c0 = 0; c0 < u.count; c0 += kChunk) {
        if (u.count > kChunk) {
            __syncthreads();
            angles(c0);
        }
        const int n = min(kChunk, u.count - c0) * G;
        for (int r = mine; r < n; r += kRows) {
            if (!held) make(c0, r);
            store(c0, r);
        }
    }
    if (u.tok > u.begin) {
        for (int h = 0; h < G; h++) {
            const int up = ups[h], hh = g0 + h;
            if (up == 0) continue;
            char* base = const_cast<char*>(hh < a.c.hk ? a.c.k : a.c.v) +
                         kv_element(a.c, uint32_t(page), slot0, uint32_t(hh < a.c.hk ? hh : hh - a.c.hk));
            const int per = d / 16;
            for (int i = tid; i < (u.tok - u.begin) * per; i += kThreads) {
                const int r = i / per;
                u32x4_t* at = reinterpret_cast<u32x4_t*>(base + uint64_t(r) * a.c.sstr + (i - r * per) * 16);
                u32x4_t x = *at;
#pragma unroll
                for (int c = 0; c < 4; c++) x[c] = halved4<TYPE>(x[c], up);
                *at = x;
            }
        }
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

template <int TYPE>
void launch_extend(const ExtendArgs& a, unsigned grid, hipStream_t s) {
    if (a.c.d <= 32) extend_kernel<TYPE, 4><<<grid, kThreads, 0, s>>>(a);
    else if (a.c.d <= 64) extend_kernel<TYPE, 8><<<grid, kThreads, 0, s>>>(a);
    else if (a.c.d <= 128) extend_kernel<TYPE, 16><<<grid, kThreads, 0, s>>>(a);
    else extend_kernel<TYPE, 32><<<grid, kThreads, 0, s>>>(a);
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
                    iq::ranges_overlap(v, kb, q_out, qb)))
        return IQ_EALIAS;
    const bool codes = iq::is_kv8(kv->type);
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_norm = q_norm;
    a.k_norm = k_norm;
    a.eps = eps;
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
    // as many heads as fill a workgroup's threads once, of the tokens that a unit has
    const int rows = iq::kThreads / (a.c.d <= 32 ? 4 : a.c.d <= 64 ? 8 : a.c.d <= 128 ? 16 : 32);
    const int tokens = starts ? std::min(a.span, rows) : 1;
    a.heads = std::min({2 * a.c.hk, iq::kMaxHeads, std::max(1, rows / tokens)});
    a.groups = uint32_t((2 * a.c.hk + a.heads - 1) / a.heads);
    a.qgroups = uint32_t((q_heads + 15) / 16);
    // n tokens touch at most (n - 1) / span + 2 units
    const int64_t units = starts ? T / a.span + 2 * std::min<int64_t>(B, T) : B;
    a.cached = units * a.groups;
    const int64_t all = a.cached + T * a.qgroups;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    for (; a.w0 < all; a.w0 += iq::kMaxGrid256) {
        const unsigned grid = unsigned(std::min(all - a.w0, iq::kMaxGrid256));
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
