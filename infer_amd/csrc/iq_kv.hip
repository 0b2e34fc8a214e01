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
// rot_dim, it moves the values as they are).  1021 tokens of 12 + 2 x 2 heads
// of 128: 6.6 us (2.4 TB/s); 16 tokens of 28 + 2 x 4: 3.6 us, a launch and two
// load latencies.
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
    const int64_t base = kv_element(a.c, uint32_t(page), live ? uint32_t(slot - page * a.c.ps) : 0, 0);
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
            uint16_t* dst = reinterpret_cast<uint16_t*>(const_cast<char*>(is_k ? a.c.k : a.c.v)) + base + uint64_t(j) * a.c.hstr;
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
// evict_plan_kernel (one workgroup per sequence and head) holds up to 32768
// sums in LDS (longer rows are read again), finds the cut-th largest by
// histograms of its bits (12 + 12 + 8, highest first; few share the upper 24,
// and are ranked by counting) and writes the lists of free places and of the
// rows that fill them.
//
// The rows are moved by two kernels.  The free places lie below cut and every
// source at or above it, so evict_fill_kernel moves those rows in any order.
// evict_shift_kernel then moves the newest ones (and the sums).  Where they
// move by less than their number, places and sources overlap: a thread takes
// every by-th row in ascending order, or, where `by` gives too few threads
// work, one workgroup goes through a slice of all rows, a chunk at a time:
// read, barrier, write; a chunk's writes lie below every later chunk's reads.
// With many sequences and heads that kernel does both, and
// one launch is saved: the free places come first in its list.
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
    int slices, ushift;    // slices of a row, of 1 << ushift 16-byte units
    int blocks;            // workgroups along the rows, where they are not one's
    int filled;            // the free places are filled by an earlier launch
};

constexpr int kPlanWaves = 16, kPlanThreads = 64 * kPlanWaves;
constexpr int kBinBits = 12, kBins = 1 << kBinBits, kFew = 64;
constexpr int kHeldSums = 32768;  // keys that a workgroup holds (128 KiB of LDS)

// Order of the sums: NaN lowest, then by value (-0 as 0).
__device__ __forceinline__ uint32_t sum_key(float w) {
    const uint32_t u = __float_as_uint(w + 0.0f);
    const uint32_t k = u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u);
    return w != w ? 0 : k;
}

// Exclusive prefix of v over the workgroup's W waves of threads and its total.
template <int W>
__device__ __forceinline__ uint32_t block_excl_scan(uint32_t v, uint32_t* total, uint32_t* sh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t inc = wave_scan(v);
    __syncthreads();  // (sh may still be read from a previous scan)
    if (lane == 63) sh[wave] = inc;
    __syncthreads();
    uint32_t before = 0, sum = 0;
#pragma unroll
    for (int i = 0; i < W; i++) {
        const uint32_t s = sh[i];
        if (i < wave) before += s;
        sum += s;
    }
    *total = sum;
    return before + inc - v;
}

// The lanes of the 64 slots from i on that lie below `end`.
__device__ __forceinline__ uint64_t lanes_below(int i, int end) {
    const int c = end - i;
    return c >= 64 ? ~uint64_t(0) : (c <= 0 ? 0 : (uint64_t(1) << c) - 1);
}

__device__ __forceinline__ uint32_t lanes_before(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi(uint32_t(mask >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(mask), 0));
}

// The keys lie in LDS.  A wave goes through a run of them in slot order, 64 in
// a round, so that ranks are a scan over the waves and counts of ballots.  The
// loops are kept short on purpose: with the keys in
// registers they have to be unrolled, and instructions that are executed once
// cost more to fetch than they take (32768 sums: 28 us with 32 keys a lane, 22.5
// so; 2112 sums: 8.8 and 7.8).
__global__ __launch_bounds__(kPlanThreads) void evict_plan_kernel(EvictArgs a) {
    extern __shared__ __align__(16) uint32_t lds[];
    uint32_t* hist = lds;
    uint32_t* keys = lds + kBins;
    __shared__ uint64_t cand[kFew];
    __shared__ uint32_t sh[kPlanWaves];
    __shared__ uint32_t found[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = blockIdx.x, b = a.b0 + int(blockIdx.y), row = int(blockIdx.y) * a.c.hk + h;
    const int n = a.t.lens[b];
    const bool fits = n >= 0 && n <= a.t.cap, over = fits && n > a.budget;
    const int old = n - int(a.recent), cut = int(a.budget - a.recent);
    const float* w = a.w + (int64_t(b) * a.c.hk + h) * a.wld;
    // this block of sums from slot i0 on: rounds of a wave, its first slot
    int rounds = 0, w0 = 0;
    const uint32_t* own = nullptr;  // its keys
    auto hold = [&](int i0) {
        const int count = min(old - i0, kHeldSums);
        rounds = (count + kPlanThreads - 1) / kPlanThreads;
        w0 = i0 + wave * rounds * 64;
        own = keys + wave * rounds * 64 + lane;
        __syncthreads();  // (the block before is done with)
#pragma unroll 8
        for (int r = 0; r < rounds; r++) {
            const int i = r * kPlanThreads + tid;
            keys[i] = sum_key(w[i0 + min(i, count - 1)]);  // (past the end: not counted)
        }
        __syncthreads();
    };
    if (over && cut) hold(0);
    bool bad = !fits;
    if (over) {
        const int np = int(page_of(uint32_t(n - 1), a.c.div)) + 1;
        bool mine = false;
        for (int i = tid; i < np; i += kPlanThreads) {
            const int p = a.t.table[b * a.t.ld + i];
            mine |= p < 0 || p >= a.c.pages;
        }
        bad = __syncthreads_or(mine);
    }
    const bool idle = bad || !over;
    if (h == 0 && tid == 0) a.new_lens[b] = idle ? n : int(a.budget);
    if (idle || cut == 0) {
        if (tid == 0) a.count[row] = idle ? -1 : 0;
        return;
    }
    const bool all = old <= kHeldSums;
    // The cut-th largest key (1 <= cut < old): its upper bits, 12 + 12 + 8,
    // until the keys that share them are all wanted or few.
    uint32_t prefix = 0, want = uint32_t(cut), equal = 0;
    int shift = 32;
    for (int pass = 0; pass < 3; pass++) {
        const int bits = pass < 2 ? kBinBits : 32 - 2 * kBinBits;
        reinterpret_cast<uint4*>(hist)[tid] = make_uint4(0, 0, 0, 0);
        if (tid == 0) found[3] = 0;
        __syncthreads();
        shift -= bits;
        for (int i0 = 0; i0 < old; i0 += kHeldSums) {
            if (!all) hold(i0);
#pragma unroll 4
            for (int r = 0; r < rounds; r++) {
                const uint32_t k = own[r * 64];
                if (pass == 0) {
                    if (w0 + r * 64 + lane < old) atomicAdd(&hist[k >> (32 - kBinBits)], 1u);
                } else if ((k >> (shift + bits)) == prefix && w0 + r * 64 + lane < old) {
                    atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1)], 1u);
                }
            }
        }
        __syncthreads();
        // bins from the highest down, four a thread
        const int b0 = kBins - 4 * (tid + 1);
        const uint4 q = *reinterpret_cast<const uint4*>(&hist[b0]);
        uint32_t total, before = block_excl_scan<kPlanWaves>(q.x + q.y + q.z + q.w, &total, sh);
        const uint32_t nb[4] = {q.w, q.z, q.y, q.x};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (before < want && want <= before + nb[i]) {
                found[0] = uint32_t(b0 + 3 - i);
                found[1] = want - before;
                found[2] = nb[i];
            }
            before += nb[i];
        }
        __syncthreads();
        prefix = (prefix << bits) | found[0];
        want = found[1];
        equal = found[2];
        if (equal == want || equal <= kFew) break;
    }
    // Which sums stay: keys above `least`, and of those equal to it the ones
    // up to slot `upto`.
    uint32_t least = prefix << shift;
    int upto = 0x7fffffff;
    if (equal > want && equal <= kFew) {
        // few keys share the bits: each one's rank among them (key descending,
        // slot ascending) is the number of greater ones
        for (int i0 = 0; i0 < old; i0 += kHeldSums) {
            if (!all) hold(i0);
#pragma unroll 4
            for (int r = 0; r < rounds; r++) {
                const uint32_t k = own[r * 64];
                const int i = w0 + r * 64 + lane;
                if ((k >> shift) == prefix && i < old) cand[atomicAdd(&found[3], 1u)] = uint64_t(k) << 32 | uint32_t(~i);
            }
        }
        __syncthreads();
        if (tid < int(equal)) {
            const uint64_t mine = cand[tid];
            uint32_t rank = 0;
            for (int i = 0; i < int(equal); i++) rank += cand[i] > mine;
            if (rank == want - 1) {
                found[0] = uint32_t(mine >> 32);
                found[1] = uint32_t(~mine);
            }
        }
        __syncthreads();
        least = found[0];
        upto = int(found[1]);
    } else if (equal > want) {
        // many equal ones (all 32 bits are known): the slot of the want-th
        uint32_t eqs = 0;  // in the blocks before
        for (int i0 = 0; i0 < old; i0 += kHeldSums) {
            if (!all) hold(i0);
            uint32_t total, eq = 0;
            for (int r = 0; r < rounds; r++)
                eq += uint32_t(__popcll(__ballot(own[r * 64] == least) & lanes_below(w0 + r * 64, old)));
            eq = block_excl_scan<kPlanWaves>(lane == 0 ? eq : 0, &total, sh);
            eq = eqs + uint32_t(__builtin_amdgcn_readfirstlane(int(eq)));
            for (int r = 0; r < rounds; r++) {
                const uint64_t same = __ballot(own[r * 64] == least) & lanes_below(w0 + r * 64, old);
                if ((same >> lane & 1) && eq + lanes_before(same) == want - 1) found[1] = uint32_t(w0 + r * 64 + lane);
                eq += uint32_t(__popcll(same));
            }
            eqs += total;
        }
        __syncthreads();
        upto = int(found[1]);
    }
    int32_t* dst = a.dst + row * a.m;
    int32_t* src = a.src + row * a.m;
    uint32_t holes = 0, highs = 0;  // of the blocks before
    for (int i0 = 0; i0 < old; i0 += kHeldSums) {
        if (!all) hold(i0);
        // the lanes of round r whose place becomes free, and whose row has to
        // move (few instructions: the CU's one scalar unit, and its vector
        // units together, start one a cycle for all sixteen waves)
        const uint64_t bound = uint64_t(least) << 32 | uint32_t(~upto);
        auto masks = [&](int r, uint64_t& to, uint64_t& from) {
            const int i = w0 + r * 64 + lane;
            const uint64_t stay = __ballot((uint64_t(own[r * 64]) << 32 | uint32_t(~i)) >= bound && i < old);
            const uint64_t low = __ballot(i < cut);
            to = low & ~stay;
            from = stay & ~low;
        };
        // (a block has at most 32768 of either: two counts in a word)
        uint32_t total, count = 0;
        for (int r = 0; r < rounds; r++) {
            uint64_t to, from;
            masks(r, to, from);
            count += uint32_t(__popcll(to)) + (uint32_t(__popcll(from)) << 16);
        }
        uint32_t at = block_excl_scan<kPlanWaves>(lane == 0 ? count : 0, &total, sh);
        at = uint32_t(__builtin_amdgcn_readfirstlane(int(at)));
        int32_t* hole = dst + holes + (at & 0xffffu);
        int32_t* high = src + highs + (at >> 16);
        for (int r = 0; r < rounds; r++) {
            const int i = w0 + r * 64 + lane;
            uint64_t to, from;
            masks(r, to, from);
            if (to) {
                if (to >> lane & 1) hole[lanes_before(to)] = i;
                hole += __popcll(to);
            }
            if (from) {
                if (from >> lane & 1) high[lanes_before(from)] = i;
                high += __popcll(from);
            }
        }
        holes += total & 0xffffu;
        highs += total >> 16;
    }
    if (tid == 0) a.count[row] = int32_t(holes);
}

// Byte offsets in either pool of N tokens of sequence b, head h (page ids were
// checked by the plan; their loads go out together).
template <int N>
__device__ __forceinline__ void kv_offsets(const KvView& c, const KvTable& t, int b, int h, const int (&tok)[N],
                                           int64_t (&at)[N]) {
    const int32_t* table = t.table + b * t.ld;
    uint32_t p[N], id[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        p[i] = page_of(uint32_t(tok[i]), c.div);
        id[i] = uint32_t(table[p[i]]);
    }
#pragma unroll
    for (int i = 0; i < N; i++) at[i] = 2 * kv_element(c, id[i], uint32_t(tok[i]) - p[i] * uint32_t(c.ps), uint32_t(h));
}

constexpr int kMoveThreads = 256, kMoveUnroll = 4;

// Moves rows [m0, m1) of a list (m1 - m0 at most 2^31 less a chunk; none:
// nothing is read, a list's entries before its first are not its own), a
// slice's 16-byte units of each from `u0` on, a chunk of 4 units a thread at a
// time: read, then written.  ORDERED: no thread writes a chunk before all have
// its values; the next chunk is requested before this one is written (the
// call on one sequence of 20027 tokens, all but 64 kept, 12889 of them the
// newest: 145 us without that and with loads that wait for one another).
template <int TH, bool ORDERED, class From, class To>
__device__ __forceinline__ void move_rows(const EvictArgs& a, char* pool, int b, int h, int m0, int m1, int u0,
                                          int ushift, From from, To to) {
    if (m0 >= m1) return;  // (the same for the whole workgroup: no barrier is left out by some)
    const int rows = TH >> ushift, r0 = int(threadIdx.x) >> ushift;
    const int u = u0 + (int(threadIdx.x) & ((1 << ushift) - 1));
    const int left = u < a.c.d / 8 ? m1 - r0 : 0;  // rows from m on are this thread's while m < left
    struct Chunk {
        u32x4_t x[kMoveUnroll];
        int64_t go[kMoveUnroll];
    };
    // (past the end the last row again, not written: no branch between the
    // loads of the rows, which would wait for one another; likewise a unit past
    // the row)
    if (u < a.c.d / 8) pool += u * 16;
    auto read = [&](int m, Chunk& c) {
        int f[kMoveUnroll], t[kMoveUnroll];
        int64_t at[kMoveUnroll];
#pragma unroll
        for (int r = 0; r < kMoveUnroll; r++) {
            const int i = min(m + r * rows + r0, m1 - 1);
            f[r] = from(i);
            t[r] = to(i);
        }
        kv_offsets(a.c, a.t, b, h, f, at);
        kv_offsets(a.c, a.t, b, h, t, c.go);
#pragma unroll
        for (int r = 0; r < kMoveUnroll; r++) c.x[r] = *reinterpret_cast<const u32x4_t*>(pool + at[r]);
    };
    const int step = rows * kMoveUnroll;
    Chunk c, next;
    read(m0, c);
    for (; m0 < m1; m0 += step) {
        if (ORDERED) {
#pragma unroll
            for (int r = 0; r < kMoveUnroll; r++) asm volatile("" : "+v"(c.x[r]));  // (waits for the values)
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        }
        if (m0 + step < m1) read(m0 + step, next);
#pragma unroll
        for (int r = 0; r < kMoveUnroll; r++)
            if (m0 + r * rows < left) *reinterpret_cast<u32x4_t*>(pool + c.go[r]) = c.x[r];
        c = next;
    }
}

constexpr int kSumBlocks = 4;

// grid: x = (K, V) x slices x blocks of rows, then kSumBlocks for the sums; y =
// head; z = sequence
__global__ __launch_bounds__(kMoveThreads, 4) void evict_fill_kernel(EvictArgs a) {
    const int h = blockIdx.y, b = a.b0 + int(blockIdx.z), row = int(blockIdx.z) * a.c.hk + h;
    const int holes = a.count[row];
    const int per = (kMoveThreads >> a.ushift) * kMoveUnroll;
    const int32_t* dst = a.dst + row * a.m;
    const int32_t* src = a.src + row * a.m;
    const int sums = int(blockIdx.x) - 2 * a.slices * a.blocks;
    if (sums >= 0) {
        float* w = a.w + (int64_t(b) * a.c.hk + h) * a.wld;
        for (int i = sums * kMoveThreads + int(threadIdx.x); i < holes; i += kSumBlocks * kMoveThreads) w[dst[i]] = w[src[i]];
        return;
    }
    const int block = int(blockIdx.x) / (2 * a.slices), sl = int(blockIdx.x) % (2 * a.slices);
    const int m0 = block * per;
    if (m0 >= holes) return;
    char* pool = const_cast<char*>(sl < a.slices ? a.c.k : a.c.v);
    move_rows<kMoveThreads, false>(a, pool, b, h, m0, min(holes, m0 + per), (sl % a.slices) << a.ushift, a.ushift,
                     [&](int i) { return src[i]; }, [&](int i) { return dst[i]; });
}

// grid: x = (K, V) x slices x blocks of rows, then one for the sums; y = head;
// z = sequence
template <int TH>
__global__ __launch_bounds__(TH, TH == kMoveThreads ? 4 : 1) void evict_shift_kernel(EvictArgs a) {
    const int h = blockIdx.y, b = a.b0 + int(blockIdx.z), row = int(blockIdx.z) * a.c.hk + h;
    const int holes = a.count[row];
    if (holes < 0) return;
    const int n = a.t.lens[b], recent = int(a.recent), cut = int(a.budget) - recent, tid = threadIdx.x;
    const int32_t* dst = a.dst + row * a.m;
    const int32_t* src = a.src + row * a.m;
    // (past the free places entry 0 is named, which is there to be read even
    // where no place is free, and is not used then; the compiler puts the load
    // behind a branch all the same)
    auto from = [&](int i) {
        const int s = src[i < holes ? i : 0];
        return i < holes ? s : n - recent + (i - holes);
    };
    auto to = [&](int i) {
        const int s = dst[i < holes ? i : 0];
        return i < holes ? s : cut + (i - holes);
    };
    const int moves = holes + recent;  // (at most the budget)
    if (int(blockIdx.x) == 2 * a.slices * a.blocks) {
        float* w = a.w + (int64_t(b) * a.c.hk + h) * a.wld;
        for (int m0 = a.filled ? holes : 0; m0 < moves; m0 += TH * kMoveUnroll) {
            float x[kMoveUnroll];
            int f[kMoveUnroll], t[kMoveUnroll];
#pragma unroll
            for (int r = 0; r < kMoveUnroll; r++) {
                const int i = min(m0 + r * TH + tid, moves - 1);
                f[r] = from(i);
                t[r] = to(i);
            }
#pragma unroll
            for (int r = 0; r < kMoveUnroll; r++) x[r] = w[f[r]];
            __builtin_amdgcn_s_waitcnt(0);  // (the values are here before another wave writes)
            __syncthreads();
#pragma unroll
            for (int r = 0; r < kMoveUnroll; r++)
                if (m0 + r * TH + tid < moves) w[t[r]] = x[r];
        }
        __syncthreads();
        for (int i = int(a.budget) + tid; i < n; i += TH) w[i] = 0.0f;
        return;
    }
    const int block = int(blockIdx.x) / (2 * a.slices), sl = int(blockIdx.x) % (2 * a.slices);
    char* pool = const_cast<char*>(sl < a.slices ? a.c.k : a.c.v);
    const int u0 = (sl % a.slices) << a.ushift, rows = TH >> a.ushift, per = rows * kMoveUnroll;
    const int by = n - int(a.budget);  // how far the newest rows move
    if (a.filled && by >= recent) {
        // their places and sources do not meet: any order
        for (int m0 = holes + block * per; m0 < moves; m0 += a.blocks * per)
            move_rows<TH, false>(a, pool, b, h, m0, min(moves, m0 + per), u0, a.ushift, from, to);
    } else if (a.filled && by >= rows) {
        // row i goes where row i - by was read: the rows of one remainder
        // modulo `by` are a thread's, in ascending order, reads first
        const int u = u0 + (tid & ((1 << a.ushift) - 1));
        if (u >= a.c.d / 8) return;
        pool += u * 16;
        for (int c = block * rows + (tid >> a.ushift); c < by; c += a.blocks * rows)
            for (int64_t i = c; i < recent; i += int64_t(by) * kMoveUnroll) {
                u32x4_t x[kMoveUnroll];
                int f[kMoveUnroll], t[kMoveUnroll];
                int64_t at[kMoveUnroll], go[kMoveUnroll];
#pragma unroll
                for (int r = 0; r < kMoveUnroll; r++) {
                    const int m = int(min(i + int64_t(r) * by, int64_t(recent) - 1));
                    f[r] = n - recent + m;
                    t[r] = cut + m;
                }
                kv_offsets(a.c, a.t, b, h, f, at);
                kv_offsets(a.c, a.t, b, h, t, go);
#pragma unroll
                for (int r = 0; r < kMoveUnroll; r++) x[r] = *reinterpret_cast<const u32x4_t*>(pool + at[r]);
#pragma unroll
                for (int r = 0; r < kMoveUnroll; r++)
                    if (i + int64_t(r) * by < recent) *reinterpret_cast<u32x4_t*>(pool + go[r]) = x[r];
            }
    } else {
        // one workgroup a slice, or two with half of it each
        const int halves = a.blocks > 1 && a.ushift > 0;
        if (block > halves) return;
        const int ushift = a.ushift - halves;
        move_rows<TH, true>(a, pool, b, h, a.filled ? holes : 0, moves, u0 + (block << ushift), ushift, from, to);
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
        if (iq::meets_cache(q_out, qn, a.c, iq::KvScales{})) return IQ_EALIAS;
    }
    a.freqs = freqs;
    a.hq = q_heads;
    a.rot = rot_dim;
    const int64_t qrow = int64_t(q_heads) * a.c.d, krow = int64_t(a.c.hk) * a.c.d;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    for (int64_t t0 = 0; t0 < T; t0 += iq::kMaxGrid256) {
        a.q = q ? q + t0 * qrow : nullptr;
        a.k = k + t0 * krow;
        a.v = v + t0 * krow;
        a.pos = positions ? positions + t0 : nullptr;
        a.slots = slots + t0;
        a.qo = q_out ? q_out + t0 * qrow : nullptr;
        const dim3 grid(static_cast<unsigned>(std::min<int64_t>(T - t0, iq::kMaxGrid256)),
                        (q_heads + 2 * a.c.hk + iq::kAppendHeads - 1) / iq::kAppendHeads);
        if (kv->type == IQ_KV_BF16) iq::append_kernel<IQ_KV_BF16><<<grid, 256, 0, s>>>(a);
        else iq::append_kernel<IQ_KV_F16><<<grid, 256, 0, s>>>(a);
    }
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
    // a workgroup's slice of the rows: 128 bytes, a cache line (16 x 4 heads of
    // 2112 tokens 16.3 us, 64 x 2 of 8000 of which 7000 move down 231; with 64
    // bytes, which read every line twice, 19.0 and 287)
    const int row_units = a.c.d / 8;
    a.ushift = row_units >= 8 ? 3 : row_units >= 4 ? 2 : (row_units >= 2 ? 1 : 0);
    a.slices = (row_units + (1 << a.ushift) - 1) >> a.ushift;
    const int64_t per = (iq::kMoveThreads >> a.ushift) * iq::kMoveUnroll;
    iq::allow_big_lds<iq::evict_plan_kernel>();
    for (a.b0 = 0; a.b0 < B; a.b0 += step) {
        const int nb = std::min(step, B - a.b0);
        const unsigned hk = unsigned(a.c.hk), nz = unsigned(nb);
        const size_t held = size_t(std::min<int64_t>((a.t.cap + 1023) / 1024 * 1024, iq::kHeldSums));
        iq::evict_plan_kernel<<<dim3(hk, nz), iq::kPlanThreads, (iq::kBins + held) * 4, s>>>(a);
        // (a cache that cannot hold more than the budget has nothing to move)
        if (a.t.cap <= budget) continue;
        // fewer than two workgroups a CU in an ordered move, and more than a
        // chunk or two of rows: spread over blocks of rows
        const int64_t wgs = int64_t(2) * a.slices * a.c.hk * nb;
        a.filled = wgs < 2 * iq::device_cu_count() && (m > per || recent > 4 * per);
        a.blocks = 1;
        if (a.filled) {
            a.blocks = int(std::min<int64_t>((m + per - 1) / per, 65536));
            iq::evict_fill_kernel<<<dim3(2 * unsigned(a.slices * a.blocks) + iq::kSumBlocks, hk, nz), iq::kMoveThreads, 0, s>>>(a);
            // (four times the threads: an ordered move has few workgroups)
            a.blocks = int(std::max<int64_t>(1, std::min<int64_t>((recent + 4 * per - 1) / (4 * per), 64)));
            iq::evict_shift_kernel<1024><<<dim3(2 * unsigned(a.slices * a.blocks) + 1, hk, nz), 1024, 0, s>>>(a);
        } else {
            iq::evict_shift_kernel<iq::kMoveThreads><<<dim3(2 * unsigned(a.slices) + 1, hk, nz), iq::kMoveThreads, 0, s>>>(a);
        }
    }
    return int(hipGetLastError());
}

}  // extern "C"
