// iq_logprob.hip -- log probabilities, entropy and top alternatives of rows
// of logits.
//
// One pass over the logits: every lane keeps a running maximum m, s = sum
// e^(x - m) and u = sum e^(x - m) (x - m), from which log softmax(x) = (x -
// m) - log s and the entropy log s - u / s follow (both free of cancellation:
// u / s <= 0), and every wave keeps its `top` largest logits in order, one a
// lane.  A logit enters that list only if it is above the list's last one:
// 16 logits a lane are compared by their maximum, which the sums need
// anyway, so the list costs one comparison a batch except for the few
// batches that hold a candidate (about top * ln(V / top) in a random row).
// Rows are split over workgroups when they are few; a second launch joins a
// row's parts.  The read of the logits bounds it.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "../../include/iq.h"
#include "iq_internal.h"

namespace iq {
namespace {

constexpr int kWaves = 4, kBatch = 1024;  // waves of a workgroup, logits of a wave's step (16 a lane)
constexpr int kMaxTop = 64;

struct LogprobArgs {
    const float* x;
    int64_t ld;
    uint32_t V;
    const int64_t* tokens;
    int top;
    float *lp, *ent;
    int64_t* ids;
    float* tlp;
    uint32_t chunks, size;  // parts of a row, logits of a part (whole batches)
    float4* stat;           // [rows][chunks]: m, s, u
    uint2* list;            // [rows][chunks][top]: key, id
};

// Order of the logits: by value (-0 as 0), NaN largest.  0 is below every
// logit and stands for "none".
__device__ __forceinline__ uint32_t logit_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

constexpr float kLog2e = 1.44269504088896340736f;

// e^x for x <= 0
__device__ __forceinline__ float exp_neg(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// A row's (or a part's) maximum and sums.  m is at least the lowest finite
// number, so that -inf - m is -inf and counts nothing; NaN and +inf make s
// NaN.  Distances below -200 (e^x is 0 there) are cut where they are
// factors: 0 times -inf would be NaN.
struct Stat {
    float m, s, u;
    __device__ __forceinline__ void clear() {
        m = -FLT_MAX;
        s = u = 0.0f;
    }
    __device__ __forceinline__ void raise(float to) {  // to >= m
        const float dm = m - to, f = exp_neg(dm);
        u = (u + s * fmaxf(dm, -200.0f)) * f;
        s *= f;
        m = to;
    }
    __device__ __forceinline__ void join(Stat o) {
        const float to = fmaxf(m, o.m);
        raise(to);
        o.raise(to);
        s += o.s;
        u += o.u;
    }
};

// Whether (k, i) ranks before (l, j): key descending, id ascending.
__device__ __forceinline__ bool before(uint32_t k, uint32_t i, uint32_t l, uint32_t j) {
    return k > l || (k == l && i < j);
}

// The wave's largest logits by (key descending, id ascending), entry i in
// lane i; key 0: none.
struct List {
    uint32_t key, id;    // this lane's entry
    uint32_t last, lid;  // entry top - 1, uniform
    __device__ __forceinline__ void clear() {
        key = last = 0;
        id = lid = 0xffffffffu;
    }
    __device__ __forceinline__ void find_last(int top) {
        last = uint32_t(__builtin_amdgcn_readlane(int(key), top - 1));
        lid = uint32_t(__builtin_amdgcn_readlane(int(id), top - 1));
    }
    // The lanes' candidates (k, i), one after the other; k == 0: none.
    __device__ __forceinline__ void add(uint32_t k, uint32_t i, int top) {
        const int lane = threadIdx.x & 63;
        uint64_t more = __ballot(k != 0 && before(k, i, last, lid));
        while (more) {
            const int from = __builtin_ctzll(more);
            const uint32_t nk = uint32_t(__builtin_amdgcn_readlane(int(k), from));
            const uint32_t ni = uint32_t(__builtin_amdgcn_readlane(int(i), from));
            // entries before the new one stay, the others move up a lane
            const uint32_t pk = uint32_t(__builtin_amdgcn_update_dpp(0, int(key), 0x138, 0xf, 0xf, false));  // wave_shr:1
            const uint32_t pi = uint32_t(__builtin_amdgcn_update_dpp(0, int(id), 0x138, 0xf, 0xf, false));
            const int at = __builtin_popcountll(__ballot(before(key, id, nk, ni)));
            key = lane < at ? key : (lane == at ? nk : pk);
            id = lane < at ? id : (lane == at ? ni : pi);
            find_last(top);
            more &= more - 1;
            more &= __ballot(before(k, i, last, lid));
        }
    }
    // The first batch, 16 candidates a lane, into the empty list.  Inserting
    // them one by one would take some 5 top steps; instead a bound that at
    // least `top` of them reach is found by bisection, first over the lanes'
    // largest (counted by one ballot a step), then, while more than a wave's
    // lanes reach it, over all; those that do go to a lane each (through
    // `room`, the wave's own 64 places in LDS) and to the place that the
    // number of greater ones says.
    template <class Id>
    __device__ __forceinline__ void fill(const uint32_t (&k)[16], Id id_of, int top, uint2* room) {
        const int lane = threadIdx.x & 63;
        uint32_t lm = k[0];
#pragma unroll
        for (int i = 1; i < 16; i++) lm = max(lm, k[i]);
        uint32_t lo = 0;
        for (int bit = 31; bit >= 0; bit--) {
            const uint32_t to = lo | (1u << bit);
            const int n = __builtin_popcountll(__ballot(lm >= to));
            if (n >= top) lo = to;
            if (n == top) break;
        }
        lo = max(lo, 1u);
        auto count = [&](uint32_t to) {
            int n = 0;
#pragma unroll
            for (int i = 0; i < 16; i++) n += __builtin_popcountll(__ballot(k[i] >= to));
            return n;
        };
        int c = count(lo);
        uint32_t hi = 0xffffffffu;
        while (c > 64 && hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            const int n = count(mid);
            if (n >= top) {
                lo = mid;
                c = n;
            } else {
                hi = mid;
            }
        }
        if (c > 64) {  // (many equal ones)
#pragma unroll
            for (int i = 0; i < 16; i++) add(k[i] >= lo ? k[i] : 0, id_of(i), top);
            return;
        }
        const uint64_t below = lane ? (~uint64_t(0) >> (64 - lane)) : 0;
        int at = 0;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const uint64_t in = __ballot(k[i] >= lo);
            if (k[i] >= lo) room[at + __builtin_popcountll(in & below)] = make_uint2(k[i], id_of(i));
            at += __builtin_popcountll(in);
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
        uint2 e = make_uint2(0, 0xffffffffu);
        if (lane < c) e = room[lane];
        int rank = 0;
        for (int i = 0; i < c; i++)
            rank += before(uint32_t(__builtin_amdgcn_readlane(int(e.x), i)), uint32_t(__builtin_amdgcn_readlane(int(e.y), i)), e.x, e.y);
        if (lane >= c) rank = lane;
        key = uint32_t(__builtin_amdgcn_ds_permute(rank * 4, int(e.x)));
        id = uint32_t(__builtin_amdgcn_ds_permute(rank * 4, int(e.y)));
        find_last(top);
    }
    // Up to 16 candidates a lane into the list; `nan`: some may be NaN.
    template <class Key, class Id>
    __device__ __forceinline__ void batch(Key key_of, Id id_of, uint32_t most, bool nan, int top, uint2* room) {
        if (!__any(most >= last || nan)) return;
        uint32_t k[16];
#pragma unroll
        for (int i = 0; i < 16; i++) k[i] = key_of(i);
        if (last == 0 && lane_key0() == 0) {
            fill(k, id_of, top, room);
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++) add(k[i], id_of(i), top);
        }
    }
    __device__ __forceinline__ uint32_t lane_key0() const { return uint32_t(__builtin_amdgcn_readfirstlane(int(key))); }
};

__device__ __forceinline__ Stat wave_join(Stat st) {
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        Stat p;
        p.m = __shfl_xor(st.m, o);
        p.s = __shfl_xor(st.s, o);
        p.u = __shfl_xor(st.u, o);
        st.join(p);
    }
    return st;
}

// Shared memory of a workgroup: a wave's room, then its list.
struct Shared {
    Stat st[kWaves];
    uint2 room[kWaves][kMaxTop];
    uint2 out[kMaxTop];
};

// The workgroup's waves joined, in wave order; the list is wave 0's.  Of the
// waves' sorted lists an entry's place is its own index and the number of
// entries of the other lists that rank before it.
template <bool TOP>
__device__ __forceinline__ void block_join(Stat& st, List& li, int top, Shared& sh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    st = wave_join(st);
    if (lane == 0) sh.st[wave] = st;
    if (TOP) {
        sh.room[wave][lane] = make_uint2(li.key, li.id);
        if (wave == 0) sh.out[lane] = make_uint2(0, 0xffffffffu);
    }
    __syncthreads();
    st = sh.st[0];
#pragma unroll
    for (int w = 1; w < kWaves; w++) st.join(sh.st[w]);
    if (TOP) {
        int at = lane;
#pragma unroll
        for (int o = 1; o < kWaves; o++) {
            const uint2* l = sh.room[(wave + o) % kWaves];
            for (int i = 0; i < top; i++) at += before(l[i].x, l[i].y, li.key, li.id);
        }
        if (lane < top && at < top && li.key) sh.out[at] = make_uint2(li.key, li.id);
        __syncthreads();
        li.key = sh.out[lane].x;
        li.id = sh.out[lane].y;
    }
}

// Wave 0 writes row t's results.
template <bool TOP>
__device__ __forceinline__ void finish(const LogprobArgs& a, int64_t t, const Stat& st, const List& li) {
    if (threadIdx.x >= 64) return;
    const int lane = threadIdx.x;
    const float nan = __builtin_nanf("");
    const float lz = st.s > 0.0f ? logf(st.s) : nan;  // (NaN, or no finite logit: no distribution)
    if (lane == 0) {
        if (a.lp) {
            const int64_t k = a.tokens[t];
            a.lp[t] = k >= 0 && k < int64_t(a.V) ? (a.x[t * a.ld + k] - st.m) - lz : nan;
        }
        if (a.ent) a.ent[t] = lz - st.u / st.s;
    }
    if (TOP && lane < a.top) {
        a.ids[t * a.top + lane] = li.id;
        a.tlp[t * a.top + lane] = (key_logit(li.key) - st.m) - lz;
    }
}

template <bool TOP>
__global__ __launch_bounds__(64 * kWaves) void logprob_kernel(LogprobArgs a) {
    __shared__ Shared sh;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t t = blockIdx.x / a.chunks;
    const uint32_t chunk = blockIdx.x % a.chunks;
    const float* x = a.x + t * a.ld;
    const uint32_t end = min(uint64_t(a.V), uint64_t(chunk + 1) * a.size);
    Stat st;
    List li;
    st.clear();
    li.clear();
    for (uint32_t b = chunk * a.size + wave * kBatch; b < end; b += kWaves * kBatch) {
        float v[16];
        const bool whole = b + kBatch <= end;
        if (whole) {
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int i = 0; i < 4; i++) v[4 * r + i] = x[b + r * 256 + lane * 4 + i];
        } else {
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t at = b + r * 256 + lane * 4 + i;
                    v[4 * r + i] = at < end ? x[at] : -INFINITY;
                }
        }
        float mx = v[0];
#pragma unroll
        for (int i = 1; i < 16; i++) mx = fmaxf(mx, v[i]);
        if (__any(mx > st.m)) st.raise(fmaxf(st.m, mx));
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float d = v[i] - st.m, e = exp_neg(d);
            st.s += e;
            st.u = fmaf(e, fmaxf(d, -200.0f), st.u);
        }
        if constexpr (TOP) {
            // (a NaN does not show in the maximum, but in the sum)
            auto id_of = [&](int i) { return b + i / 4 * 256 + lane * 4 + i % 4; };
            li.batch([&](int i) { return id_of(i) < end ? logit_key(v[i]) : 0u; }, id_of, logit_key(mx), !(st.s >= 0.0f),
                     a.top, sh.room[wave]);
        }
    }
    block_join<TOP>(st, li, a.top, sh);
    if (a.chunks == 1) {
        finish<TOP>(a, t, st, li);
        return;
    }
    if (threadIdx.x == 0) a.stat[blockIdx.x] = make_float4(st.m, st.s, st.u, 0.0f);
    if (TOP && wave == 0 && lane < a.top) a.list[int64_t(blockIdx.x) * a.top + lane] = make_uint2(li.key, li.id);
}

template <bool TOP>
__global__ __launch_bounds__(64 * kWaves) void logprob_join_kernel(LogprobArgs a) {
    __shared__ Shared sh;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t t = blockIdx.x;
    Stat st;
    List li;
    st.clear();
    li.clear();
    for (uint32_t c = threadIdx.x; c < a.chunks; c += 64 * kWaves) {
        const float4 f = a.stat[t * a.chunks + c];
        st.join(Stat{f.x, f.y, f.z});
    }
    if constexpr (TOP) {
        const uint32_t n = a.chunks * a.top;
        const uint2* l = a.list + t * n;
        for (uint32_t b = wave * kBatch; b < n; b += kWaves * kBatch) {
            uint2 e[16];
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const uint32_t at = b + i * 64 + lane;
                e[i] = at < n ? l[at] : make_uint2(0, 0);
                most = max(most, e[i].x);
            }
            li.batch([&](int i) { return e[i].x; }, [&](int i) { return e[i].y; }, most, false, a.top, sh.room[wave]);
        }
    }
    block_join<TOP>(st, li, a.top, sh);
    finish<TOP>(a, t, st, li);
}

}  // namespace
}  // namespace iq

extern "C" {

int iq_logprobs(const float* logits, int64_t ld, int64_t T, int64_t V, const int64_t* tokens, int top,
                float* logprob, float* entropy, int64_t* top_ids, float* top_logprobs, void* stream) {
    if (T < 1 || V < 1 || ld < V || top < 0 || top > iq::kMaxTop || top > V) return IQ_ESHAPE;
    if (!logits || !tokens != !logprob || (top && (!top_ids || !top_logprobs))) return IQ_ENULL;
    if (!logprob && !entropy && !top) return IQ_ENULL;
    if (V > 0x7fffffff - 65536 || T > 0x7fffffff) return IQ_ETOOLARGE;
    iq::LogprobArgs a{logits, ld, uint32_t(V), tokens, top, logprob, entropy, top_ids, top_logprobs};
    // about eight workgroups a CU, parts of four batches at least
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t target = 8 * int64_t(iq::device_cu_count());
    int64_t chunks = std::max<int64_t>(1, std::min((target + T - 1) / T, (V + 4095) / 4096));
    const int64_t size = ((V + chunks - 1) / chunks + iq::kBatch - 1) / iq::kBatch * iq::kBatch;
    chunks = (V + size - 1) / size;
    a.chunks = uint32_t(chunks);
    a.size = uint32_t(size);
    if (chunks > 1) {
        iq::Workspace* ws = nullptr;
        const hipError_t e = iq::get_workspace(s, &ws);
        if (e != hipSuccess) return e == hipErrorOutOfMemory ? IQ_ENOMEM : int(e);
        if (T * chunks * (4 + 2 * int64_t(top)) > ws->part_floats) return IQ_ETOOLARGE;
        a.stat = reinterpret_cast<float4*>(ws->partials);
        a.list = reinterpret_cast<uint2*>(ws->partials + T * chunks * 4);
    }
    const unsigned grid = unsigned(T * chunks);
    if (top) iq::logprob_kernel<true><<<grid, 64 * iq::kWaves, 0, s>>>(a);
    else iq::logprob_kernel<false><<<grid, 64 * iq::kWaves, 0, s>>>(a);
    if (chunks > 1) {
        if (top) iq::logprob_join_kernel<true><<<unsigned(T), 64 * iq::kWaves, 0, s>>>(a);
        else iq::logprob_join_kernel<false><<<unsigned(T), 64 * iq::kWaves, 0, s>>>(a);
    }
    return int(hipGetLastError());
}

}  // extern "C"
