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
// row's parts.  The read of the logits bounds it: 999 rows of 152064 take 138
// us (4.4 TB/s); 32 rows with the top 20 13.7 us and 6.4 to join, one row 7.1
// and 4.7 (latency).
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
    uint64_t* list;         // [rows][chunks][top]
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

// A logit's place in the ranking: key descending, then id ascending; 0: none.
__device__ __forceinline__ uint64_t entry(uint32_t key, uint32_t id) { return uint64_t(key) << 32 | uint32_t(~id); }
__device__ __forceinline__ uint64_t lane_of64(uint64_t v, int lane) {
    return uint64_t(uint32_t(__builtin_amdgcn_readlane(int(v >> 32), lane))) << 32 |
           uint32_t(__builtin_amdgcn_readlane(int(v), lane));
}

// The wave's largest logits in order, entry i in lane i.
struct List {
    uint64_t e;      // this lane's entry
    uint64_t floor;  // an entry that `top` others of the row reach
    uint64_t last;   // entry top - 1 or the floor: what a candidate has to pass; uniform
    __device__ __forceinline__ void clear() { e = floor = last = 0; }
    __device__ __forceinline__ void find_last(int top) {
        const uint64_t l = lane_of64(e, top - 1);
        last = l > floor ? l : floor;
    }
    __device__ __forceinline__ uint32_t last_key() const { return uint32_t(last >> 32); }
    // The lanes' candidates, one after the other (0: none).
    __device__ __forceinline__ void add(uint64_t c, int top) {
        const int lane = threadIdx.x & 63;
        uint64_t more = __ballot(c > last);
        while (more) {
            const uint64_t n = lane_of64(c, __builtin_ctzll(more));
            // entries before the new one stay, the others move up a lane
            const uint32_t ph = uint32_t(__builtin_amdgcn_update_dpp(0, int(e >> 32), 0x138, 0xf, 0xf, false));  // wave_shr:1
            const uint32_t pl = uint32_t(__builtin_amdgcn_update_dpp(0, int(e), 0x138, 0xf, 0xf, false));
            const int at = __builtin_popcountll(__ballot(e > n));
            e = lane < at ? e : (lane == at ? n : uint64_t(ph) << 32 | pl);
            find_last(top);
            more &= more - 1;
            more &= __ballot(c > last);
        }
    }
    // A wave's first batch, 16 candidates a lane, into the empty list (where
    // first_batch below cannot): a bound that at least `top` of them reach is
    // found by bisection, first over the lanes' largest (counted by one
    // ballot a step, until no more than 24 lanes reach it), then, while more
    // than a wave's lanes do, over all; those that do go to a lane each
    // (through `room`, the wave's own 64 places in LDS) and from there to the
    // place that the number of greater ones says.
    template <class Id>
    __device__ __forceinline__ void fill(const uint32_t (&k)[16], Id id_of, int top, uint64_t* room) {
        const int lane = threadIdx.x & 63;
        room[lane] = 0;
        uint32_t lm = k[0];
#pragma unroll
        for (int i = 1; i < 16; i++) lm = max(lm, k[i]);
        uint32_t lo = 0;
        const int few = max(top, 24);
        for (int bit = 31; bit >= 0; bit--) {
            const uint32_t to = lo | (1u << bit);
            const int n = __builtin_popcountll(__ballot(lm >= to));
            if (n >= top) {
                lo = to;
                if (n <= few) break;
            }
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
            for (int i = 0; i < 16; i++) add(k[i] >= lo ? entry(k[i], id_of(i)) : 0, top);
            return;
        }
        int at = 0;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const uint64_t in = __ballot(k[i] >= lo);
            if (k[i] >= lo)
                room[at + __builtin_amdgcn_mbcnt_hi(uint32_t(in >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(in), 0))] =
                    entry(k[i], id_of(i));
            at += __builtin_popcountll(in);
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
        const uint64_t mine = room[lane];
        int rank = 0;
        for (int i = 0; i < c; i += 8)
#pragma unroll
            for (int r = 0; r < 8; r++) rank += room[i + r] > mine;
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
        if (lane < c) room[rank] = mine;  // (the places from c on stay 0)
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
        e = room[lane];
        find_last(top);
    }
    // Up to 16 candidates a lane into the list, `most` their largest key;
    // `nan`: some may be NaN, which does not show in it.
    template <class Key, class Id>
    __device__ __forceinline__ void batch(Key key_of, Id id_of, uint32_t most, bool nan, int top, uint64_t* room) {
        if (!__any(most >= last_key() || nan)) return;
        uint32_t k[16];
#pragma unroll
        for (int i = 0; i < 16; i++) k[i] = key_of(i);
        if (last == 0 && lane_of64(e, 0) == 0) {
            fill(k, id_of, top, room);
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++) add(k[i] ? entry(k[i], id_of(i)) : 0, top);
        }
    }
};

// Maximum and sum over a wave's lanes, in every lane (DPP: row_shr 1, 2, 4,
// 8, then the rows' last lanes into the next rows; lane 63 has the result).
template <int CTRL, int ROWS>
__device__ __forceinline__ float from_lane(float v, float none) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(none), __float_as_int(v), CTRL, ROWS, 0xf, false));
}
template <class Op>
__device__ __forceinline__ float wave_reduce(float v, float none, Op op) {
    v = op(v, from_lane<0x111, 0xf>(v, none));
    v = op(v, from_lane<0x112, 0xf>(v, none));
    v = op(v, from_lane<0x114, 0xf>(v, none));
    v = op(v, from_lane<0x118, 0xf>(v, none));
    v = op(v, from_lane<0x142, 0xa>(v, none));
    v = op(v, from_lane<0x143, 0xc>(v, none));
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ Stat wave_join(Stat st) {
    st.raise(wave_reduce(st.m, -FLT_MAX, [](float x, float y) { return fmaxf(x, y); }));
    st.s = wave_reduce(st.s, 0.0f, [](float x, float y) { return x + y; });
    st.u = wave_reduce(st.u, 0.0f, [](float x, float y) { return x + y; });
    return st;
}

// Shared memory of a workgroup: first_batch's, then a wave's room, then its list.
struct Shared {
    Stat st[kWaves];
    uint32_t most[64 * kWaves];  // the lanes' largest keys
    uint64_t room[kWaves][kMaxTop];
    uint64_t out[kMaxTop];
    uint32_t nan[kWaves];
    uint32_t lo, count;
};

// The workgroup's first batch, 16 candidates a lane of all its waves.
// Inserting them one by one would take some 5 top steps a wave (32 rows of
// 152064, top 20: 53 us a launch; a bound and a sorted list for every wave,
// 15).  Instead wave 0 bisects for a bound that `top` of the 256 lanes'
// largest keys reach (at most 24, if top allows), the few candidates that
// reach it (`reach(i, bound)`) are collected in LDS, and each goes to the
// place that the number of greater ones says: wave 0's list, and the floor of
// the other waves'.  False, with nothing changed, where more than 256 reach
// it (many equal ones, or a large `top`) or there may be NaN: the waves then
// fill lists of their own.
template <class Reach, class Entry>
__device__ __forceinline__ bool first_batch(List& li, uint32_t most, bool nan, int top, Shared& sh, Reach reach,
                                            Entry entry_of) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint64_t* found = &sh.room[0][0];
    sh.most[tid] = most;
    found[tid] = 0;
    if (wave == 0) sh.out[lane] = 0;
    const bool any = __any(nan);
    if (lane == 0) sh.nan[wave] = any;
    __syncthreads();
    if (wave == 0) {
        uint32_t k[kWaves];
#pragma unroll
        for (int w = 0; w < kWaves; w++) k[w] = sh.most[w * 64 + lane];
        uint32_t lo = 0;
        const int few = max(top, 24);
        for (int bit = 31; bit >= 0; bit--) {
            const uint32_t to = lo | (1u << bit);
            int n = 0;
#pragma unroll
            for (int w = 0; w < kWaves; w++) n += __builtin_popcountll(__ballot(k[w] >= to));
            if (n >= top) {
                lo = to;
                if (n <= few) break;
            }
        }
        if (lane == 0) {
            sh.lo = max(lo, 1u);
            sh.count = 0;
        }
    }
    __syncthreads();
    const uint32_t lo = sh.lo;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        if (reach(i, lo)) {
            const uint32_t at = atomicAdd(&sh.count, 1u);
            if (at < 64 * kWaves) found[at] = entry_of(i);
        }
    }
    __syncthreads();
    const int c = int(sh.count);
    if (c > 64 * kWaves || sh.nan[0] | sh.nan[1] | sh.nan[2] | sh.nan[3]) {
        __syncthreads();  // (the rooms become the waves' own)
        return false;
    }
    const uint64_t mine = found[tid];
    if (tid < c) {
        int rank = 0;
        for (int i = 0; i < c; i += 8)
#pragma unroll
            for (int r = 0; r < 8; r++) rank += found[i + r] > mine;
        if (rank < kMaxTop) sh.out[rank] = mine;
    }
    __syncthreads();
    if (wave == 0) li.e = sh.out[lane];
    li.floor = sh.out[top - 1];
    li.find_last(top);
    __syncthreads();
    return true;
}
static_assert(kWaves == 4, "first_batch ors four flags");

// The workgroup's waves joined, in wave order; the list is wave 0's.  Of the
// waves' sorted lists an entry's place is its own index and the number of
// entries of the other lists that rank before it.  `done`: it is wave 0's already.
template <bool TOP>
__device__ __forceinline__ void block_join(Stat& st, List& li, int top, Shared& sh, bool done) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    st = wave_join(st);
    if (lane == 0) sh.st[wave] = st;
    if (TOP && !done) {
        sh.room[wave][lane] = lane < top ? li.e : 0;
        if (wave == 0) sh.out[lane] = 0;
    }
    __syncthreads();
    st = sh.st[0];
#pragma unroll
    for (int w = 1; w < kWaves; w++) st.join(sh.st[w]);
    if (TOP && !done) {
        int at = lane;
        const uint64_t mine = li.e;
#pragma unroll
        for (int o = 1; o < kWaves; o++) {
            const uint64_t* l = sh.room[(wave + o) % kWaves];
            for (int i = 0; i < top; i += 4)
#pragma unroll
                for (int r = 0; r < 4; r++) at += l[i + r] > mine;
        }
        if (lane < top && at < top && mine) sh.out[at] = mine;
        __syncthreads();
        li.e = sh.out[lane];
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
        a.ids[t * a.top + lane] = uint32_t(~li.e);
        a.tlp[t * a.top + lane] = (key_logit(uint32_t(li.e >> 32)) - st.m) - lz;
    }
}

// Workgroups a CU that a call is split into (and that its registers allow for:
// with the list and five a CU, 96 of them and one that is spilled, 8 bytes of
// scratch memory a lane).
constexpr int kPerCu = 4, kPerCuTop = 5;

template <bool TOP>
__global__ __launch_bounds__(64 * kWaves, 5) void logprob_kernel(LogprobArgs a) {
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
    const uint32_t b0 = chunk * a.size;
    bool done = false;
    for (uint32_t b = b0 + wave * kBatch; b < end || b < b0 + kWaves * kBatch; b += kWaves * kBatch) {
        float v[16];  // past the end: -inf
        if (b + kBatch <= end) {
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
            // (a NaN shows in the sum)
            auto id_of = [&](int i) { return b + i / 4 * 256 + lane * 4 + i % 4; };
            if (b < b0 + kWaves * kBatch) {
                // (the bound as a logit: keys up to -inf's are all logits)
                done = first_batch(
                    li, b + lane * 4 < end ? logit_key(mx) : 0, !(st.s >= 0.0f), a.top, sh,
                    [&](int i, uint32_t lo) {
                        return v[i] >= (lo <= 0x007fffffu ? -INFINITY : key_logit(lo)) && id_of(i) < end;
                    },
                    [&](int i) { return entry(logit_key(v[i]), id_of(i)); });
                if (done) continue;
            } else {
                done = false;
            }
            li.batch([&](int i) { return id_of(i) < end ? logit_key(v[i]) : 0u; }, id_of, logit_key(mx), !(st.s >= 0.0f),
                     a.top, sh.room[wave]);
        }
    }
    done = done && end - b0 <= kWaves * kBatch;
    block_join<TOP>(st, li, a.top, sh, done);
    if (a.chunks == 1) {
        finish<TOP>(a, t, st, li);
        return;
    }
    if (threadIdx.x == 0) a.stat[blockIdx.x] = make_float4(st.m, st.s, st.u, 0.0f);
    if (TOP && wave == 0 && lane < a.top) a.list[int64_t(blockIdx.x) * a.top + lane] = li.e;
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
    bool done = false;
    if constexpr (TOP) {
        const uint32_t n = a.chunks * a.top;
        const uint64_t* l = a.list + t * n;
        for (uint32_t b = wave * kBatch; b < n || b < kWaves * kBatch; b += kWaves * kBatch) {
            uint64_t e[16];
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const uint32_t at = b + i * 64 + lane;
                e[i] = at < n ? l[at] : 0;
                most = max(most, uint32_t(e[i] >> 32));
            }
            if (b < kWaves * kBatch) {
                done = first_batch(li, most, false, a.top, sh,
                                   [&](int i, uint32_t lo) { return uint32_t(e[i] >> 32) >= lo; }, [&](int i) { return e[i]; });
                if (done) continue;
            }
            li.batch([&](int i) { return uint32_t(e[i] >> 32); }, [&](int i) { return uint32_t(~e[i]); }, most, false, a.top,
                     sh.room[wave]);
        }
    }
    block_join<TOP>(st, li, a.top, sh, done && a.chunks * a.top <= kWaves * kBatch);
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
    // workgroups for every CU, parts of four batches at least (32 rows of 152064,
    // top 20, in 4 / 8 / 19 / 38 parts: 38.6 / 27.1 / 21.8 / 19.3 us; 999 rows, no
    // list, in 1 / 2 / 4: 138.3 / 143.5 / 145.6)
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t target = (top ? iq::kPerCuTop : iq::kPerCu) * int64_t(iq::device_cu_count());
    int64_t chunks = std::max<int64_t>(1, std::min(target / T, (V + 4095) / 4096));
    // whole steps of a workgroup where they are few, of a wave where many
    int64_t size = (V + chunks - 1) / chunks;
    const int64_t whole = size > 16 * iq::kBatch ? iq::kBatch : iq::kWaves * iq::kBatch;
    size = (size + whole - 1) / whole * whole;
    chunks = (V + size - 1) / size;
    a.chunks = uint32_t(chunks);
    a.size = uint32_t(size);
    if (chunks > 1) {
        iq::Workspace* ws = nullptr;
        const hipError_t e = iq::get_workspace(s, &ws);
        if (e != hipSuccess) return e == hipErrorOutOfMemory ? IQ_ENOMEM : int(e);
        if (T * chunks * (4 + 2 * int64_t(top)) > ws->part_floats) return IQ_ETOOLARGE;
        a.stat = reinterpret_cast<float4*>(ws->partials);
        a.list = reinterpret_cast<uint64_t*>(ws->partials + T * chunks * 4);
    }
    // (more rows than a grid can have are more than the CUs: a part each)
    const int64_t rows = chunks > 1 ? T : iq::kMaxGrid256;
    for (int64_t t0 = 0; t0 < T; t0 += rows) {
        const unsigned grid = unsigned(std::min(T - t0, rows) * chunks);
        a.x = logits + t0 * ld;
        a.tokens = tokens ? tokens + t0 : nullptr;
        a.lp = logprob ? logprob + t0 : nullptr;
        a.ent = entropy ? entropy + t0 : nullptr;
        a.ids = top ? top_ids + t0 * top : nullptr;
        a.tlp = top ? top_logprobs + t0 * top : nullptr;
        if (top) iq::logprob_kernel<true><<<grid, 64 * iq::kWaves, 0, s>>>(a);
        else iq::logprob_kernel<false><<<grid, 64 * iq::kWaves, 0, s>>>(a);
    }
    if (chunks > 1) {
        if (top) iq::logprob_join_kernel<true><<<unsigned(T), 64 * iq::kWaves, 0, s>>>(a);
        else iq::logprob_join_kernel<false><<<unsigned(T), 64 * iq::kWaves, 0, s>>>(a);
    }
    return int(hipGetLastError());
}

}  // extern "C"
