// iq_kv.hip -- the paged key/value cache: tokens added to it (with rotary
// embedding) and evicted from it by accumulated attention weight.
#include <algorithm>

#include "iq_kv.h"

namespace iq {
namespace {

// ------------------------------------------------------------------ append
// One workgroup per token and block of 16 heads (query heads, then key, then
// value heads).  The token's angles are made once per workgroup: pos * f is
// reduced to a fraction of a turn in 64 bits (a far position's angle has
// lost its last bits in 32: 131072 rad in fp32 is known to 0.008) and its
// sine and cosine taken in 32.  A thread then turns 4 pairs of one head
// (two 16-byte loads, two 16- or 8-byte stores; without rotation, or past
// rot_dim, it moves the values as they are).
struct AppendArgs {
    const float *q, *k, *v;
    const int64_t *pos, *slots;
    const double* freqs;
    float* qo;
    int hq, rot;
    KvView c;
};

template <int TYPE>
__device__ __forceinline__ void store_kv4(uint16_t* p, const float (&y)[4]) {
    uint2 u;
    u.x = f32_to_kv<TYPE>(y[0]) | uint32_t(f32_to_kv<TYPE>(y[1])) << 16;
    u.y = f32_to_kv<TYPE>(y[2]) | uint32_t(f32_to_kv<TYPE>(y[3])) << 16;
    *reinterpret_cast<uint2*>(p) = u;
}

constexpr int kAppendHeads = 16;

template <int TYPE>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
    __shared__ float2 cs[128];
    const int64_t t = blockIdx.x;
    const int d = a.c.d, half = a.rot / 2;
    if (int(threadIdx.x) < half) {
        const double turns = double(a.pos[t]) * a.freqs[threadIdx.x] * 0.15915494309189533577;
        const float r = float((turns - rint(turns)) * 6.28318530717958647693);
        cs[threadIdx.x] = make_float2(cosf(r), sinf(r));
    }
    __syncthreads();
    const int heads = a.hq + 2 * a.c.hk;
    const int64_t slot = a.slots[t];
    const bool live = slot >= 0 && slot < a.c.pages * a.c.ps;
    const int64_t page = live ? slot / a.c.ps : 0;
    const int64_t base = page * a.c.pstr + (live ? slot % a.c.ps : 0) * a.c.sstr;
    const int per = d / 8;  // 4-pair units of a head
    const int h0 = blockIdx.y * kAppendHeads, h1 = min(h0 + kAppendHeads, heads);
    for (int u = threadIdx.x; u < (h1 - h0) * per; u += 256) {
        const int h = h0 + u / per, i = u % per * 4;
        const bool is_q = h < a.hq, is_k = !is_q && h < a.hq + a.c.hk;
        if (!is_q && !live) continue;
        const int j = is_q ? h : (is_k ? h - a.hq : h - a.hq - a.c.hk);
        const float* src = is_q ? a.q + (t * a.hq + j) * d : (is_k ? a.k : a.v) + (t * a.c.hk + j) * d;
        // the two runs of 4 values: a pair's halves, or two neighbours
        const int rot = (is_q || is_k) ? a.rot : 0;
        int e0, e1;
        const bool turn = i < rot / 2;
        if (turn) {
            e0 = i;
            e1 = i + rot / 2;
        } else {
            e0 = rot + (i - rot / 2) * 2;
            e1 = e0 + 4;
        }
        float x0[4], x1[4], y0[4], y1[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            x0[r] = src[e0 + r];
            x1[r] = src[e1 + r];
        }
#pragma unroll
        for (int r = 0; r < 4; r++) {
            if (turn) {
                const float2 w = cs[i + r];
                y0[r] = x0[r] * w.x - x1[r] * w.y;
                y1[r] = x1[r] * w.x + x0[r] * w.y;
            } else {
                y0[r] = x0[r];
                y1[r] = x1[r];
            }
        }
        if (is_q) {
            float* dst = a.qo + (t * a.hq + j) * d;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                dst[e0 + r] = y0[r];
                dst[e1 + r] = y1[r];
            }
        } else {
            uint16_t* dst = reinterpret_cast<uint16_t*>(const_cast<char*>(is_k ? a.c.k : a.c.v)) + base + j * a.c.hstr;
            store_kv4<TYPE>(dst + e0, y0);
            store_kv4<TYPE>(dst + e1, y1);
        }
    }
}

// ---------------------------------------------------------------- eviction
// Of a (sequence, key/value head)'s n cached tokens `budget` stay: the newest
// `recent`, and the cut = budget - recent of the largest sums among the old =
// n - recent others.  Keys are rotated when they are appended and attention
// does not depend on the order of its tokens, so the kept rows below cut need
// not move: the i-th free place below cut takes the i-th kept row above it
// (as many as there are: cut - (kept below)), and only the newest rows,
// whose order says which are the newest at the next call, move down by n -
// budget.  That is what the call has to move; keeping the order of all rows
// would move everything behind the first evicted one.
//
// evict_plan_kernel (one workgroup per sequence and head) finds the cut-th
// largest sum by three histogram passes over its bits (11 + 11 + 10, highest
// first) and writes the lists of free places and of rows that fill them.
// evict_move_kernel moves rows: a workgroup has one sequence, head, K or V
// (or the sums) and a slice of the row, and goes through the moves in order,
// a chunk at a time: read, barrier, write.  No write of a chunk meets a read
// of a later one: free places lie below cut and every source at or above
// it, and the newest rows, after all of those, move down in ascending order.
struct EvictArgs {
    KvView c;
    KvTable t;
    int b0;                // first sequence of this launch
    int64_t budget, recent;
    float* w;
    int64_t wld;
    int32_t* new_lens;
    int32_t* count;        // [sequences][hk]: free places to fill, -1: nothing to evict
    int32_t* dst;          // [sequences][hk][m]
    int32_t* src;
    int64_t m;
    int slices, units;     // slices of a row, 16-byte units of a slice
    int holes_done;        // the free places are filled by an earlier launch
};

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64, kBins = 2048, kCopies = 4;

// Order of the sums: NaN lowest, then by value (-0 as 0).
__device__ __forceinline__ uint32_t sum_key(float w) {
    const uint32_t u = __float_as_uint(w + 0.0f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0;
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ int wave_incl_scan(int v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(v, o);
        if (lane >= o) v += u;
    }
    return v;
}

// Exclusive prefix of v over the workgroup's threads and its total.
__device__ __forceinline__ int block_excl_scan(int v, int* total, int* sh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int inc = wave_incl_scan(v);
    __syncthreads();  // (sh may still be read from a previous scan)
    if (lane == 63) sh[wave] = inc;
    __syncthreads();
    int before = 0, sum = 0;
    for (int i = 0; i < kPlanWaves; i++) {
        const int s = sh[i];
        if (i < wave) before += s;
        sum += s;
    }
    *total = sum;
    return before + inc - v;
}

__global__ __launch_bounds__(kPlanThreads) void evict_plan_kernel(EvictArgs a) {
    __shared__ int hist[kCopies][kBins];
    __shared__ int sh[kPlanWaves];
    __shared__ int found[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int h = blockIdx.x, b = a.b0 + int(blockIdx.y), row = int(blockIdx.y) * a.c.hk + h;
    const int n = a.t.lens[b];
    bool bad = n < 0 || n > a.t.cap;
    if (!bad) {
        const int np = (n + a.c.ps - 1) / a.c.ps;
        bool mine = false;
        for (int i = tid; i < np; i += kPlanThreads) {
            const int p = a.t.table[b * a.t.ld + i];
            mine |= p < 0 || p >= a.c.pages;
        }
        bad = __syncthreads_or(mine);
    }
    const bool idle = bad || n <= a.budget;
    if (h == 0 && tid == 0) a.new_lens[b] = idle ? n : int(a.budget);
    if (idle) {
        if (tid == 0) a.count[row] = -1;
        return;
    }
    const int old = n - int(a.recent), cut = int(a.budget - a.recent);
    const float* w = a.w + (int64_t(b) * a.c.hk + h) * a.wld;
    if (cut == 0) {
        if (tid == 0) a.count[row] = 0;
        return;
    }
    // the cut-th largest key (1 <= cut < old)
    uint32_t prefix = 0;
    int want = cut, shift = 32;
    int equal = 0;
    for (int pass = 0; pass < 3; pass++) {
        const int bits = pass < 2 ? 11 : 10;
        for (int i = tid; i < kCopies * kBins; i += kPlanThreads) (&hist[0][0])[i] = 0;
        __syncthreads();
        shift -= bits;
        for (int i = tid; i < old; i += kPlanThreads) {
            const uint32_t k = sum_key(w[i]);
            const bool in = pass == 0 || (k >> (shift + bits)) == prefix;
            if (in) atomicAdd(&hist[lane % kCopies][(k >> shift) & ((1u << bits) - 1)], 1);
        }
        __syncthreads();
        const int hi = kBins - 1 - 2 * tid, lo = hi - 1;
        int nh = 0, nl = 0;
#pragma unroll
        for (int c = 0; c < kCopies; c++) {
            nh += hist[c][hi];
            nl += hist[c][lo];
        }
        int total;
        const int before = block_excl_scan(nh + nl, &total, sh);
        if (before < want && want <= before + nh + nl) {
            const bool first = want <= before + nh;
            found[0] = first ? hi : lo;
            found[1] = want - before - (first ? 0 : nh);
            found[2] = first ? nh : nl;
        }
        __syncthreads();
        prefix = (prefix << bits) | uint32_t(found[0]);
        want = found[1];
        equal = found[2];
    }
    // keys above `prefix` stay, of the equal ones the first `want`.  Every wave
    // has a run of slots, 64 at a time in order.
    const int seg = ((old + kPlanWaves - 1) / kPlanWaves + 63) / 64 * 64;
    const int s0 = min(wave * seg, old), s1 = min(s0 + seg, old);
    int eq_before = 0;
    if (equal > want) {
        int mine = 0;
        for (int i = s0 + lane; i < s1; i += 64) mine += sum_key(w[i]) == prefix;
        for (int o = 32; o; o >>= 1) mine += __shfl_xor(mine, o);
        __syncthreads();
        if (lane == 0) sh[wave] = mine;
        __syncthreads();
        for (int i = 0; i < wave; i++) eq_before += sh[i];
        __syncthreads();
    }
    const uint64_t below = lane ? (~uint64_t(0) >> (64 - lane)) : 0;
    int32_t* dst = a.dst + row * a.m;
    int32_t* src = a.src + row * a.m;
    int holes = 0, highs = 0;  // of the waves before, then running
    for (int pass = 0; pass < 2; pass++) {
        int nhole = 0, nhigh = 0, eq = eq_before;
        for (int i0 = s0; i0 < s1; i0 += 64) {
            const int i = i0 + lane;
            const uint32_t k = i < s1 ? sum_key(w[i]) : 0;
            const bool same = i < s1 && k == prefix;
            const uint64_t eqm = __ballot(same);
            const bool keep = i < s1 && (k > prefix || (same && eq + __popcll(eqm & below) < want));
            eq += __popcll(eqm);
            const bool hole = i < s1 && !keep && i < cut, high = keep && i >= cut;
            const uint64_t hm = __ballot(hole), gm = __ballot(high);
            if (pass == 1) {
                if (hole) dst[holes + nhole + __popcll(hm & below)] = i;
                if (high) src[highs + nhigh + __popcll(gm & below)] = i;
            }
            nhole += __popcll(hm);
            nhigh += __popcll(gm);
        }
        if (pass == 0) {
            if (lane == 0) {
                hist[0][wave] = nhole;
                hist[1][wave] = nhigh;
            }
            __syncthreads();
            int all = 0;
            for (int i = 0; i < kPlanWaves; i++) {
                if (i < wave) {
                    holes += hist[0][i];
                    highs += hist[1][i];
                }
                all += hist[0][i];
            }
            if (tid == 0) a.count[row] = all;
        }
    }
}

// Byte offset of (token t of sequence b, head h) in either pool (page ids
// were checked by the plan).
__device__ __forceinline__ int64_t kv_offset(const KvView& c, const KvTable& t, int b, int h, int tok) {
    const int p = tok / c.ps;
    return 2 * (t.table[b * t.ld + p] * c.pstr + int64_t(tok - p * c.ps) * c.sstr + h * c.hstr);
}

constexpr int kMoveThreads = 256, kMoveUnroll = 8;

// grid: x = (K, V) x slices of a row, then one for the sums; y = head; z =
// sequence.
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictArgs a) {
    const int h = blockIdx.y, b = a.b0 + int(blockIdx.z), row = int(blockIdx.z) * a.c.hk + h;
    const int holes = a.count[row];
    if (holes < 0) return;
    const int n = a.t.lens[b], recent = int(a.recent), cut = int(a.budget) - recent, tid = threadIdx.x;
    const int32_t* dst = a.dst + row * a.m;
    const int32_t* src = a.src + row * a.m;
    const int first = a.holes_done ? holes : 0;
    auto from = [&](int i) { return i < holes ? src[i] : n - recent + (i - holes); };
    auto to = [&](int i) { return i < holes ? dst[i] : cut + (i - holes); };
    if (int(blockIdx.x) == 2 * a.slices) {
        float* w = a.w + (int64_t(b) * a.c.hk + h) * a.wld;
        for (int m0 = 0; m0 < holes + recent; m0 += kMoveThreads * kMoveUnroll) {
            float x[kMoveUnroll];
#pragma unroll
            for (int r = 0; r < kMoveUnroll; r++) {
                const int i = m0 + r * kMoveThreads + tid;
                x[r] = i < holes + recent ? w[from(i)] : 0.0f;
            }
            __builtin_amdgcn_s_waitcnt(0);  // (the values are here before another wave writes)
            __syncthreads();
#pragma unroll
            for (int r = 0; r < kMoveUnroll; r++) {
                const int i = m0 + r * kMoveThreads + tid;
                if (i < holes + recent) w[to(i)] = x[r];
            }
        }
        __syncthreads();
        for (int i = int(a.budget) + tid; i < n; i += kMoveThreads) w[i] = 0.0f;
        return;
    }
    char* pool = const_cast<char*>(int(blockIdx.x) < a.slices ? a.c.k : a.c.v);
    const int u0 = int(blockIdx.x) % a.slices * a.units, nu = min(a.units, a.c.d / 8 - u0);
    const int64_t total = int64_t(holes + recent) * nu;
    for (int64_t m0 = int64_t(first) * nu; m0 < total; m0 += kMoveThreads * kMoveUnroll) {
        u32x4_t x[kMoveUnroll];
#pragma unroll
        for (int r = 0; r < kMoveUnroll; r++) {
            const int64_t i = m0 + r * kMoveThreads + tid;
            if (i < total) {
                const int m = int(i / nu), u = int(i % nu);
                x[r] = *reinterpret_cast<const u32x4_t*>(pool + kv_offset(a.c, a.t, b, h, from(m)) + (u0 + u) * 16);
            }
        }
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kMoveUnroll; r++) {
            const int64_t i = m0 + r * kMoveThreads + tid;
            if (i < total) {
                const int m = int(i / nu), u = int(i % nu);
                *reinterpret_cast<u32x4_t*>(pool + kv_offset(a.c, a.t, b, h, to(m)) + (u0 + u) * 16) = x[r];
            }
        }
    }
}

}  // namespace
}  // namespace iq

extern "C" {

int iq_kv_append(const float* q, const float* k, const float* v, const int64_t* positions, const int64_t* slots,
                 int64_t T, int q_heads, const double* freqs, int rot_dim, const iq_kv* kv, float* q_out,
                 void* stream) {
    iq::AppendArgs a{};
    const int rc = iq::check_kv(kv, &a.c);
    if (rc) return rc;
    if (T < 1 || q_heads < 0 || q_heads > 16384 || rot_dim < 0 || rot_dim > kv->head_dim || rot_dim % 8) return IQ_ESHAPE;
    if (!k || !v || !slots || (q_heads && (!q || !q_out)) || (rot_dim && (!positions || !freqs))) return IQ_ENULL;
    if (T > 0x7fffffff) return IQ_ETOOLARGE;
    const int64_t qn = T * q_heads * a.c.d * 4, kn = T * a.c.hk * a.c.d * 4;
    if (q_heads) {
        if (q_out != q && iq::ranges_overlap(q_out, qn, q, qn)) return IQ_EALIAS;
        if (iq::ranges_overlap(q_out, qn, k, kn) || iq::ranges_overlap(q_out, qn, v, kn)) return IQ_EALIAS;
    }
    a.q = q;
    a.k = k;
    a.v = v;
    a.pos = positions;
    a.slots = slots;
    a.freqs = freqs;
    a.qo = q_out;
    a.hq = q_heads;
    a.rot = rot_dim;
    const dim3 grid(static_cast<unsigned>(T), (q_heads + 2 * a.c.hk + iq::kAppendHeads - 1) / iq::kAppendHeads);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (kv->type == IQ_KV_BF16) iq::append_kernel<IQ_KV_BF16><<<grid, 256, 0, s>>>(a);
    else iq::append_kernel<IQ_KV_F16><<<grid, 256, 0, s>>>(a);
    return int(hipGetLastError());
}

int iq_kv_evict(const iq_kv* kv, const int32_t* table, int64_t table_ld, int64_t max_pages, const int32_t* lens,
                int B, int64_t budget, int64_t recent, float* weights, int64_t weights_ld, int32_t* new_lens,
                void* stream) {
    iq::EvictArgs a{};
    int rc = iq::check_kv(kv, &a.c);
    if (rc) return rc;
    rc = iq::check_table(a.c, table, table_ld, max_pages, lens, B, &a.t);
    if (rc) return rc;
    if (!weights || !new_lens) return IQ_ENULL;
    if (budget < 1 || recent < 0 || recent > budget || weights_ld < a.t.cap) return IQ_ESHAPE;
    if (iq::ranges_overlap(new_lens, 4 * int64_t(B), lens, 4 * int64_t(B))) return IQ_EALIAS;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    iq::Workspace* ws = nullptr;
    const hipError_t e = iq::get_workspace(s, &ws);
    if (e != hipSuccess) return e == hipErrorOutOfMemory ? IQ_ENOMEM : int(e);
    // the move lists of a launch's sequences lie in the workspace's partial
    // sums; as many sequences a launch as fit
    const int64_t m = std::max<int64_t>(1, std::min<int64_t>(budget - recent, a.t.cap - budget));
    const int64_t per_seq = int64_t(a.c.hk) * (2 * m + 1);
    const int64_t fit = ws->part_floats / per_seq;
    if (fit < 1) return IQ_ETOOLARGE;
    a.budget = budget;
    a.recent = recent;
    a.w = weights;
    a.wld = weights_ld;
    a.new_lens = new_lens;
    a.m = m;
    const int step = int(std::min<int64_t>(B, fit));
    a.count = reinterpret_cast<int32_t*>(ws->partials);
    a.dst = a.count + int64_t(step) * a.c.hk;
    a.src = a.dst + int64_t(step) * a.c.hk * m;
    const int row_units = a.c.d / 8;
    a.units = row_units;
    a.slices = 1;
    for (a.b0 = 0; a.b0 < B; a.b0 += step) {
        const int nb = std::min(step, B - a.b0);
        iq::evict_plan_kernel<<<dim3(unsigned(a.c.hk), unsigned(nb)), iq::kPlanThreads, 0, s>>>(a);
        // (a cache that cannot hold more than the budget has nothing to move)
        if (a.t.cap > budget)
            iq::evict_move_kernel<<<dim3(unsigned(2 * a.slices + 1), unsigned(a.c.hk), unsigned(nb)),
                                    iq::kMoveThreads, 0, s>>>(a);
    }
    return int(hipGetLastError());
}

}  // extern "C"
