// iq_attn.hip -- attention of one new token a sequence over a paged cache.
//
// With g query heads on a key/value head, every cached element is used by g
// products of each kind, and an element is 2 bytes: on the vector units that
// is 7 multiply-adds for Qwen2.5-7B where HBM delivers one element per two
// cycles and lane, too many beside the unpacking; on the matrix cores the up
// to 16 heads of a group are the 16 columns of one product and cost nothing.
// What bounds the operator is the read of the cache: 131072 tokens, 4 heads of
// 128 in bf16 take 52.8 us (5.1 TB/s; a device copy reaches 4.7, a plain read
// 6.2), every byte read once, the matrix cores busy for 13 % of it; 32 sequences
// of up to 8192 tokens, 2 heads, 20.4 us (4.2 TB/s).  A join adds 4 to 5 us.
// Under a window a sequence is its visible tokens: 16 of up to 16384 that see
// 4100 each, 4 heads, 19.1 us (4.1 TB/s).
//
//   scores  S^T[token][head] = K[token][d] . q^T[d][head]
//   sums    O^T[d][head]    += V^T[d][token] . P^T[token][head]
//
// both as 16 x 16 x 32 MFMAs on the 16-bit cache as it is.  q and p are fp32:
// for a bf16 cache each is cut exactly into three bf16 terms (8 + 8 + 8 bits)
// and multiplied three times, for fp16 into two fp16 terms (22 bits, scaled
// so that nothing becomes subnormal): the products stay at fp32 precision and
// still take a small part of the matrix cores' time.
//
// A wave takes 32 tokens at a time: their K and V rows come in whole rows (16
// bytes a lane, 16 lanes a row at d = 128) into registers while the previous
// tile is multiplied, then through the wave's own part of LDS (no barrier)
// into operand order: K rows by 16-byte reads, V transposed by
// ds_read_b64_tr_b16.  The scores' result order (head = lane % 16, tokens
// 4 (lane / 16) + 0..3 of either half) is used as the second product's
// operand order, so P never leaves its lane.  Maximum and sum run along
// (one pass); a new maximum rescales the 16 x d sums.
//
// The batch's tokens are split into chunks of equal size over all sequences
// (iq_attn_plan.h); a workgroup of 4 waves has one chunk of one head tile,
// joins its waves in LDS, and writes the result if the sequence has no other
// chunk, else the chunk's maximum, sum and unnormalised rows, which
// attn_join_kernel adds up.  Nothing is kept between calls and no order of
// additions depends on timing.
#include "iq_attn.h"

namespace iq {
namespace {

// DP: head_dim rounded up to 32, 64, 128 or 256.  MODE: AttnMode.  Under a window
// (WIN) of a sequence longer than a.visible only the first a.sinks tokens and the
// newest others are seen; they are numbered without the gap.
template <int TYPE, int DP, int MODE>
__global__ __launch_bounds__(64 * kAttnWaves, DP > 128 ? 1 : 2) void attn_kernel(AttnArgs a) {
    using T = Terms<TYPE>;
    constexpr bool WIN = MODE != kAll;
    constexpr int CH = DP / 8, RPI = 64 / CH, NI = kAttnTile / RPI;  // 16-byte chunks of a row, rows of a load, loads
    constexpr int KC = DP / 32, VT = DP / 16;                       // steps of the first product, tiles of the second
    constexpr int ROWB = DP * 2, KVB = kAttnTile * ROWB;
    __shared__ __align__(16) char lds[kAttnWaves][2 * KVB];
    __shared__ float wm[kAttnWaves][16], wl[kAttnWaves][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, col = lane & 15;
    Item it;
    // Heads that share cache lines (see the host side) go to one XCD for a
    // chunk: workgroups are dealt to the 8 of them in turn.
    const uint32_t turn = a.lines ? 8 : 1, round = blockIdx.x / (turn * a.nh), in = blockIdx.x % (turn * a.nh);
    const uint32_t hidx = in / turn;
    if (!find_item<MODE>(a, round * turn + in % turn, &it)) return;
    const int b = it.b, n = it.n, d = a.c.d;
    const int j = int(hidx) / a.ht, h0 = int(hidx) % a.ht * 16, gh = min(16, a.group - h0);
    float* out = a.out + (int64_t(b) * a.hq + j * a.group + h0) * d;
    if (MODE != kWhole && hidx == 0 && it.j == 0 && threadIdx.x == 0) a.plan[b] = make_uint2(it.chunks, it.first);
    if (n <= 0 || n > a.t.cap) {
        const float x = n == 0 ? 0.0f : __builtin_nanf("");
        for (int i = threadIdx.x; i < gh * d; i += 64 * kAttnWaves) out[i] = x;
        return;
    }
    const int t0 = int(it.j * it.c) * kAttnTile, t1 = t0 + min(it.seen - t0, int(it.c) * kAttnTile);
    const int ntiles = (t1 - t0 + kAttnTile - 1) / kAttnTile;

    // token r of a tile and its page's id (0 past the end), and from these the
    // element offset of its (page, slot), 0 where there is none
    bool poison = false;
    const int32_t* table = a.t.table + b * a.t.ld;
    auto token = [&](int tile) {
        const int tok = t0 + tile * kAttnTile + (lane & 31);
        return WIN && tok >= a.sinks ? tok + (n - it.seen) : tok;
    };
    auto page_id = [&](int tile) -> int32_t {
        return t0 + tile * kAttnTile + (lane & 31) < t1 ? table[page_of(uint32_t(token(tile)), a.c.div)] : 0;
    };
    auto row_offset = [&](int tile, int32_t id) -> int64_t {
        const uint32_t tok = uint32_t(token(tile)), s = tok - page_of(tok, a.c.div) * uint32_t(a.c.ps);
        const bool live = t0 + tile * kAttnTile + (lane & 31) < t1, ok = id >= 0 && id < a.c.pages;
        poison |= live && !ok;
        return live && ok ? kv_element(a.c, uint32_t(id), s, 0) : 0;
    };
    // chunks past the row's end repeat its first one (q is 0 there, and the
    // sums of those columns are not written)
    const int ch = lane % CH, chsrc = ch * 8 < d ? ch : 0;
    const int64_t lane_off = int64_t(uint64_t(j) * a.c.hstr) + chsrc * 8;
    const uint16_t* kp = reinterpret_cast<const uint16_t*>(a.c.k) + lane_off;
    const uint16_t* vp = reinterpret_cast<const uint16_t*>(a.c.v) + lane_off;
    u32x4_t kr[NI], vr[NI];
    auto load = [&](int64_t off) {
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int64_t o = __shfl(off, i * RPI + lane / CH);
            kr[i] = *reinterpret_cast<const u32x4_t*>(kp + o);
            vr[i] = *reinterpret_cast<const u32x4_t*>(vp + o);
        }
    };
    // Chunk c of row r lies at chunk c ^ swizzle(r) of the row's place: the 16
    // rows that a K read, and the 4 x 4 rows of which a V read takes 32 bytes,
    // then fall on different banks.
    constexpr int RPB = 256 / ROWB > 1 ? 256 / ROWB : 1;  // rows across the banks
    auto ksw = [](int r) { return (r / RPB) & (CH < 16 ? CH - 1 : 15); };
    auto vsw = [](int r) { return ((r / RPB) & (CH < 16 ? CH / 2 - 1 : 7)) * 2; };
    char* kl = lds[wave];
    char* vl = lds[wave] + KVB;

    // The chain of loads that nothing shortens is length, page id, rows: q,
    // needed last, is requested behind the first page ids and cut while the
    // first rows come.
    const int32_t id0 = page_id(wave);
    int32_t next_id = page_id(wave + kAttnWaves);
    // q: column = head, 8 values of each 32-value step a lane
    s16x8_t qt[KC][T::N];
    float mul = a.mul;
    {
        const float* q = a.q + (int64_t(b) * a.hq + j * a.group + h0 + (col < gh ? col : 0)) * d;
        float x[KC][8];
        float big = 0.0f;
#pragma unroll
        for (int c = 0; c < KC; c++) {
            const int e = c * 32 + g * 8;
#pragma unroll
            for (int i = 0; i < 8; i++) x[c][i] = q[(e < d ? e : 0) + i];
        }
        if (wave < ntiles) load(row_offset(wave, id0));
#pragma unroll
        for (int c = 0; c < KC; c++) {
            const bool in = col < gh && c * 32 + g * 8 < d;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[c][i] = in ? x[c][i] : 0.0f;
                big = fmaxf(big, fabsf(x[c][i]));
            }
        }
        if constexpr (TYPE == IQ_KV_F16) {
            // the head's largest value to 2^13..2^14, undone on the scores
            big = fmaxf(big, __shfl_xor(big, 16));
            big = fmaxf(big, __shfl_xor(big, 32));
            const int e = max(int(__float_as_uint(big) >> 23), 27) - 127;
            const float up = __uint_as_float(uint32_t(127 + 13 - e) << 23);
            mul *= __uint_as_float(uint32_t(127 - 13 + e) << 23);
#pragma unroll
            for (int c = 0; c < KC; c++)
#pragma unroll
                for (int i = 0; i < 8; i++) x[c][i] *= up;
        }
#pragma unroll
        for (int c = 0; c < KC; c++) T::cut(x[c], qt[c]);
    }

    float4_t o[VT];
#pragma unroll
    for (int i = 0; i < VT; i++) o[i] = float4_t{0, 0, 0, 0};
    float m = kNone, l = 0.0f;
    float* sc = a.sc ? a.sc + ((int64_t(b) * a.c.hk + j) * a.t.cap) * a.group + h0 + col : nullptr;

    for (int tile = wave; tile < ntiles; tile += kAttnWaves) {
        const int tk = t0 + tile * kAttnTile;  // first token
        const bool whole = tk + kAttnTile <= t1;
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int r = i * RPI + lane / CH;
            *reinterpret_cast<u32x4_t*>(kl + r * ROWB + (ch ^ ksw(r)) * 16) = kr[i];
            // (a row past the end may hold anything: 0 times NaN is NaN)
            const u32x4_t zero = {0, 0, 0, 0};
            *reinterpret_cast<u32x4_t*>(vl + r * ROWB + (ch ^ vsw(r)) * 16) = whole || tk + r < t1 ? vr[i] : zero;
        }
        if (tile + kAttnWaves < ntiles) {
            // (the id behind it first: a wait for it then leaves the tile's loads in flight)
            const int64_t off = row_offset(tile + kAttnWaves, next_id);
            next_id = page_id(tile + 2 * kAttnWaves);
            load(off);
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
        float s[8];
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
            float4_t acc = {0, 0, 0, 0};
            const int r = hf * 16 + col;
#pragma unroll
            for (int c = 0; c < KC; c++) {
                const s16x8_t kv = *reinterpret_cast<const s16x8_t*>(kl + r * ROWB + ((c * 4 + g) ^ ksw(r)) * 16);
#pragma unroll
                for (int k = 0; k < T::N; k++) acc = T::mma(kv, qt[c][k], acc);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int tok = tk + hf * 16 + g * 4 + i;
                float x = acc[i] * mul;
                if (!whole && tok >= t1) x = -INFINITY;
                s[hf * 4 + i] = x;
            }
        }
        if (sc && col < gh) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int tok = tk + (i >> 2) * 16 + g * 4 + (i & 3);
                if (tok < t1) sc[int64_t(tok) * a.group] = s[i];
            }
        }
        float mx = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        if (__any(mx > m)) {
            const float mn = fmaxf(m, mx), al = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= al;
#pragma unroll
            for (int i = 0; i < VT; i++) o[i] *= al;
        }
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            // (not s - (m - 12): from 2^26 on m - 12 is rounded to m - 16 and more,
            // p becomes 2^16, past fp16's range, and the waves' scales differ)
            const float e = s[i] - m;
            p[i] = __builtin_amdgcn_exp2f(T::kUp != 0.0f ? e + T::kUp : e);
            l += p[i];
        }
        s16x8_t pt[T::N];
        T::cut(p, pt);
        // (all VT tiles of columns, also past head_dim: a branch around those costs whole
        // heads 1 to 4 %, 24 sequences of up to 2047, 16 heads of 256 120.5 -> 125.9 us, of
        // 128 40.5 -> 40.8, and gains the others about 1 % at most, 16 heads of 80 31.9 -> 31.8, of
        // 144 110.2 -> 109.0, of 160 110.3 -> 110.8)
#pragma unroll
        for (int v = 0; v < VT; v++) {
            // rows 4g..4g+3 of either half: lane 4r + c of 16 gives row r's
            // 8-byte piece c, lane i gets the 4 rows' value of column i
            s16x8_t av;
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                const int r = hf * 16 + g * 4 + col / 4;
                const int at = r * ROWB + ((v * 2 + (col & 3) / 2) ^ vsw(r)) * 16 + (col & 1) * 8;
                const s16x4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    reinterpret_cast<__attribute__((address_space(3))) s16x4_t*>(
                        (__attribute__((address_space(3))) char*)(vl) + at));
#pragma unroll
                for (int i = 0; i < 4; i++) av[hf * 4 + i] = x[i];
            }
#pragma unroll
            for (int k = 0; k < T::N; k++) o[v] = T::mma(av, pt[k], o[v]);
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
    }
    // the waves' results; the tiles' places are free once every wave is here
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (__any(poison)) l = __builtin_nanf("");
    __syncthreads();
    constexpr int OST = DP + 4;
    static_assert(16 * OST * 4 <= 2 * KVB, "a wave's sums fit its tiles' place");
    float* ol = reinterpret_cast<float*>(lds[wave]);
#pragma unroll
    for (int v = 0; v < VT; v++) *reinterpret_cast<float4_t*>(ol + col * OST + v * 16 + g * 4) = o[v];
    if (g == 0) {
        wm[wave][col] = m;
        wl[wave][col] = l;
    }
    __syncthreads();
    const bool alone = it.chunks == 1;
    const int64_t slot = (int64_t(it.first) + it.j) * a.nh + hidx;
    for (int i = threadIdx.x; i < gh * (d / 4); i += 64 * kAttnWaves) {
        const int h = i / (d / 4), e = i % (d / 4) * 4;
        float M = wm[0][h];
#pragma unroll
        for (int w = 1; w < kAttnWaves; w++) M = fmaxf(M, wm[w][h]);
        float L = 0.0f;
        float4_t x = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kAttnWaves; w++) {
            const float f = __builtin_amdgcn_exp2f(wm[w][h] - M);
            L += wl[w][h] * f;
            x += *reinterpret_cast<const float4_t*>(reinterpret_cast<const float*>(lds[w]) + h * OST + e) * f;
        }
        float* to;
        if (alone) {
            const float inv = inv_sum(L);
            x *= inv;
            to = out + h * d + e;
        } else {
            to = a.part + slot * 16 * d + h * d + e;
        }
        if (e == 0) {
            float* f = alone ? a.fin + (int64_t(b) * a.hq + j * a.group + h0 + h) * 2 : a.ml + slot * 32 + h * 2;
            f[0] = M;
            f[1] = L;
        }
#pragma unroll
        for (int r = 0; r < 4; r++) to[r] = x[r];
    }
}

// Chunk i's maximum and sum of a head, of the sequence whose plan is pl.
__device__ __forceinline__ float2 chunk_ml(const AttnArgs& a, uint2 pl, int head, uint32_t i) {
    const int hg = head % a.group;
    const int64_t slot = (int64_t(pl.y) + i) * a.nh + head / a.group * a.ht + hg / 16;
    return reinterpret_cast<const float2*>(a.ml)[slot * 16 + hg % 16];
}

// One workgroup per (head, sequence): the chunks' rows, each times 2^(its
// maximum - the largest so far), in chunk order within TH / (d / 4 rounded to
// a power of two) runs that are then added in order.  TH: 1024 threads for
// few sequences with many chunks each (one of 20000 tokens, 2 key/value heads:
// 17.4 us with 256, 15.6 so; their runs are added in pairs down to 8), else 256.
template <int TH>
__device__ __forceinline__ void join_head(const AttnArgs& a, int b, int head) {
    __shared__ float4_t xs[TH];
    __shared__ float2 ms[TH];
    const int d = a.c.d, tid = threadIdx.x;
    const uint2 pl = a.plan[b];
    if (pl.x < 2) return;
    const int j = head / a.group, hg = head % a.group, hidx = j * a.ht + hg / 16, h = hg % 16;
    const float* part = a.part + (int64_t(pl.y) * a.nh + hidx) * 16 * d + h * d;
    int w = 2;  // 16-byte pieces of a row, to a power of two
    while (w * 4 < d) w *= 2;
    const int e = tid % w * 4, run = tid / w, runs = TH / w, n = int(pl.x);
    float M = kNone, L = 0.0f;
    float4_t x = {0, 0, 0, 0};
    auto add = [&](float2 v, float4_t y) {
        const float mn = fmaxf(M, v.x), f = __builtin_amdgcn_exp2f(M - mn), k = __builtin_amdgcn_exp2f(v.x - mn);
        M = mn;
        L = L * f + v.y * k;
        x = x * f + y * k;
    };
    if (e < d) {
        int i = run;
        for (; i + 3 * runs < n; i += 4 * runs) {
            float2 v[4];
            float4_t y[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                v[r] = chunk_ml(a, pl, head, uint32_t(i + r * runs));
                y[r] = *reinterpret_cast<const float4_t*>(part + int64_t(i + r * runs) * a.nh * 16 * d + e);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) add(v[r], y[r]);
        }
        for (; i < n; i += runs)
            add(chunk_ml(a, pl, head, uint32_t(i)), *reinterpret_cast<const float4_t*>(part + int64_t(i) * a.nh * 16 * d + e));
    }
    xs[tid] = x;
    ms[tid] = make_float2(M, L);
    __syncthreads();
    if constexpr (TH > 256) {
        for (int s = runs / 2; s > 4; s /= 2) {
            if (run < s) {
                add(ms[tid + s * w], xs[tid + s * w]);
                xs[tid] = x;
                ms[tid] = make_float2(M, L);
            }
            __syncthreads();
        }
    }
    if (run == 0 && e < d) {
        for (int r = 1; r < min(TH > 256 ? min(runs, 8) : runs, n); r++) add(ms[r * w + tid], xs[r * w + tid]);
        const float inv = inv_sum(L);
        float* out = a.out + (int64_t(b) * a.hq + head) * d + e;
#pragma unroll
        for (int r = 0; r < 4; r++) out[r] = x[r] * inv;
    }
}

template <int TH>
__global__ __launch_bounds__(TH) void attn_join_kernel(AttnArgs a) {
    join_head<TH>(a, blockIdx.y, blockIdx.x);
}

// The same with further workgroups that add the weights: for TH tokens of a
// key/value head, weights[b][j][t] += sum over the group's heads, in order,
// of 2^(score - maximum) / sum.  The heads' maxima and sums over the chunks
// are made here again, 16 heads x TH / 16 runs of chunks at a time.
template <int TH>
__global__ __launch_bounds__(TH) void attn_weights_kernel(AttnArgs a, float* weights, int64_t wld, float up) {
    constexpr int RUNS = TH / 16;
    __shared__ float2 run_ml[16][RUNS + 1];
    __shared__ float2 head_ml[16];  // maximum, 1 / sum
    const int b = blockIdx.y, tid = threadIdx.x;
    if (int(blockIdx.x) < a.hq) {
        join_head<TH>(a, b, blockIdx.x);
        return;
    }
    const int n = a.t.lens[b];
    const uint32_t w = blockIdx.x - uint32_t(a.hq);
    const int j = int(w % uint32_t(a.c.hk)), t0 = int(w / uint32_t(a.c.hk)) * TH, t = t0 + tid;
    if (n > a.t.cap || t0 >= n) return;
    const uint2 pl = a.plan[b];
    const int64_t row = int64_t(b) * a.c.hk + j;
    const float* s = a.sc + (row * a.t.cap + min(t, n - 1)) * a.group;
    float sum = 0.0f;
    for (int h0 = 0; h0 < a.group; h0 += 16) {
        const int gh = min(16, a.group - h0), h = tid & 15, run = tid >> 4;
        float M = -INFINITY, L = 0.0f;
        auto add = [&](float2 v) {
            const float mn = fmaxf(M, v.x);
            L = L * __builtin_amdgcn_exp2f(M - mn) + v.y * __builtin_amdgcn_exp2f(v.x - mn);
            M = mn;
        };
        if (h < gh) {
            if (pl.x < 2) {
                if (run == 0) add(reinterpret_cast<const float2*>(a.fin)[int64_t(b) * a.hq + j * a.group + h0 + h]);
            } else {
                for (uint32_t i = uint32_t(run); i < pl.x; i += RUNS) add(chunk_ml(a, pl, j * a.group + h0 + h, i));
            }
        }
        __syncthreads();
        run_ml[h][run] = make_float2(M, L);
        __syncthreads();
        if (tid < gh) {
            const int runs = pl.x < 2 ? 1 : int(min(pl.x, uint32_t(RUNS)));
            M = run_ml[tid][0].x;
            L = run_ml[tid][0].y;
            for (int r = 1; r < runs; r++) add(run_ml[tid][r]);
            head_ml[tid] = make_float2(M, inv_sum(L));
        }
        __syncthreads();
        // (2^(score - maximum) of a head whose sum is 0: the maximum is kNone, the
        // scores -inf, 2^-inf = 0)
        for (int i = 0; i < gh; i++) sum += __builtin_amdgcn_exp2f((s[h0 + i] - head_ml[i].x) + up) * head_ml[i].y;
    }
    if (t < n) weights[row * wld + t] += sum;
}

template <int TYPE, int MODE>
void launch_mode(const AttnArgs& a, unsigned grid, hipStream_t s) {
    if (a.c.d <= 32) attn_kernel<TYPE, 32, MODE><<<grid, 64 * kAttnWaves, 0, s>>>(a);
    else if (a.c.d <= 64) attn_kernel<TYPE, 64, MODE><<<grid, 64 * kAttnWaves, 0, s>>>(a);
    else if (a.c.d <= 128) attn_kernel<TYPE, 128, MODE><<<grid, 64 * kAttnWaves, 0, s>>>(a);
    else attn_kernel<TYPE, 256, MODE><<<grid, 64 * kAttnWaves, 0, s>>>(a);
}

template <int TYPE>
void launch_attn(const AttnArgs& a, AttnMode mode, unsigned grid, hipStream_t s) {
    (mode == kWhole ? launch_mode<TYPE, kWhole> : mode == kWindow ? launch_mode<TYPE, kWindow> : launch_mode<TYPE, kAll>)(a, grid, s);
}

// The most tiles of a batch whose sequences are each one chunk: where more tiles
// in a row (0.4 us each) cost less than the search for a chunk, its sums' way
// through memory, the second launch and, with more pairs (sequence, kv head) than
// CUs, a second round of workgroups.  Split and whole, us a call in a graph, by
// sequences x tiles, 4 key/value heads:
//   int8, 128     1 x 8 8.9, 7.0   1 x 12 9.0, 8.5     1 x 16 9.1, 9.9   32 x 16 11.7, 10.4
//                 32 x 32 15.0, 16.5   64 x 16 13.3, 11.1   64 x 32 19.1, 17.0   128 x 32 31.1, 27.9
//   int8, 32      1 x 12 7.3, 5.5  1 x 16 7.4, 6.3     32 x 32 10.7, 9.9 64 x 32 12.7, 10.3
//   int8, 256     1 x 8 11.3, 11.3 1 x 12 11.5, 14.9   32 x 16 16.9, 19.2
//                 64 x 16 22.2, 20.3   64 x 32 34.0, 32.5   (e4m3: 1 x 8 10.9, 10.3)
//   bf16 under a window
//        32       1 x 8 7.5, 5.2   1 x 12 7.7, 6.1     32 x 16 8.8, 7.2  64 x 32 13.3, 11.9
//        64       1 x 8 8.1, 6.2   1 x 12 8.2, 7.4     1 x 13 8.3, 8.5   64 x 32 19.8, 15.9
//        128      1 x 8 9.5, 8.4   1 x 12 9.6, 10.3    32 x 16 14.5, 13.5
//                 64 x 16 21.1, 16.9   64 x 32 30.4, 26.1   256 x 32 107, 102
//        256      1 x 4 10.4, 9.9  1 x 8 13.0, 14.3    32 x 16 24.9, 26.9   64 x 32 55.3, 53.3
// Where the rule takes the slower side: whole, few pairs of 256 in 16 bits (1 x 8);
// split, heads of 32 and 64 a few tiles past the bounds and many pairs just past 32
// (bf16 of 64, 32 x 17 11.0, 10.1, 128 x 33 31.2, 26.8).
// With more tiles a long sequence among short ones would be waited for (2048
// tokens: 9.2 us split, 22.7 whole).  It goes by the table's width, the lengths
// being on the device: in a wide table a short sequence is split and pays 2 us for
// it (17 tokens 5.6, in a table of 128 pages of 16 and more 7.7).  (16-bit caches
// without a window keep the order of their sums, the split's.)
int64_t whole_tiles(int64_t pairs, int cus, int d, int bytes) {
    if (pairs >= cus) return 32;
    if (2 * pairs >= cus && d <= 128) return 16;
    return d * bytes <= 128 ? 12 : 8;
}

// The call behind either entry point; a: cache, scales and table, checked.
int attn_decode(AttnArgs a, const float* q, int B, int q_heads, float scale, int64_t window, int64_t sinks, float* out,
                float* weights, int64_t weights_ld, hipStream_t s) {
    if (!q || !out) return IQ_ENULL;
    a.mul = scale * 1.44269504088896340736f;
    if (q_heads < 1 || q_heads > 16384 || q_heads % a.c.hk || !std::isfinite(a.mul)) return IQ_ESHAPE;
    if (window < 0 || sinks < 0) return IQ_ESHAPE;
    if (weights && weights_ld < a.t.cap) return IQ_ESHAPE;
    const int64_t row = int64_t(q_heads) * a.c.d;
    if (ranges_overlap(q, B * row * 4, out, B * row * 4) || meets_cache(out, B * row * 4, a.c, a.scales)) return IQ_EALIAS;
    Workspace* ws = nullptr;
    const hipError_t e = get_workspace(s, &ws);
    if (e != hipSuccess) return e == hipErrorOutOfMemory ? IQ_ENOMEM : int(e);
    const bool bits8 = a.c.type == IQ_KV_I8 || a.c.type == IQ_KV_E4M3;
    a.hq = q_heads;
    a.group = q_heads / a.c.hk;
    a.ht = (a.group + 15) / 16;
    a.nh = uint32_t(a.c.hk * a.ht);
    // what a sequence sees at most; a window that no sequence can reach is none
    const bool win = window > 0 && window < a.t.cap && sinks < a.t.cap - window;
    a.sinks = win ? int32_t(sinks) : 0;
    a.visible = win ? int32_t(window + sinks) : a.t.cap;
    // as many work items as run at once: 4, 3, 2 or 1 workgroups a CU by the
    // registers (d <= 64) and the LDS of an instance.  Both launches with 1, 2, 3
    // and 4 a CU: d = 128, 131072 tokens 56.5, 57.3, 61.1, 62 us, 32 sequences of up
    // to 8192 23.8, 24.2, 27.3, 27.4; d = 64, 24 of up to 2047, 16 heads 16.0,
    // 16.5, 16.9, 18.3; d = 32, 8 of 16384 46.9, 38.3, 37.7, 38.6.  (The choice goes
    // into the order of a result's sums; 8-bit caches have their own.)
    const int groups = bits8 ? attn8_groups(a.c.d) : a.c.d <= 32 ? 4 : a.c.d <= 64 ? 3 : a.c.d <= 128 ? 2 : 1;
    const int cus = device_cu_count();
    a.target = uint32_t(groups * cus);
    // Neighbouring heads' rows meet in a cache line, or several head tiles read
    // the same rows: one XCD's L2 then serves them (8 sequences of 16384, 8 heads
    // of 32: 49.7 -> 38.8 us; of 8192, heads of 80: 50.1 -> 44.6).  Whole lines
    // are better spread (131072 tokens, 4 heads of 128: 61.9 and 64.0).
    a.lines = a.nh > 1 && (a.ht > 1 || (bits8 ? 1 : 2) * a.c.hstr % 128 != 0);
    const int64_t capt = attn_tiles(a.visible);
    // the workspace's partial sums: plan | final (maximum, sum) | chunks' | rows;
    // its GEMM operand area: the scores that the weights are made of
    const int64_t slots = attn_max_partials(a.target);
    int64_t step = B;
    step = std::min<int64_t>(step, (int64_t(1) << 30) / (capt * a.nh));
    if (weights) step = std::min<int64_t>(step, int64_t(ws->gx_bytes / 4) / (int64_t(a.t.cap) * q_heads));
    const int64_t room = ws->part_floats - 2 * kMaxSeqs - slots * 16 * (2 + a.c.d) - 63;
    step = std::min<int64_t>(step, room / (2 * q_heads));
    if (step < 1) return IQ_ETOOLARGE;
    const int64_t fin = (step * q_heads * 2 + 63) / 64 * 64;
    a.plan = reinterpret_cast<uint2*>(ws->partials);
    a.fin = ws->partials + 2 * kMaxSeqs;
    a.ml = a.fin + fin;
    a.part = a.ml + slots * 32;
    a.sc = weights ? static_cast<float*>(ws->gx) : nullptr;
    const KvTable t = a.t;
    for (int b0 = 0; b0 < B; b0 += int(step)) {
        a.B = int(std::min<int64_t>(step, B - b0));
        a.q = q + b0 * row;
        a.out = out + b0 * row;
        a.t.table = t.table + b0 * t.ld;
        a.t.lens = t.lens + b0;
        const int64_t pairs = int64_t(a.B) * a.nh;
        const bool whole = (bits8 || win) && capt <= whole_tiles(pairs, cus, a.c.d, bits8 ? 1 : 2);
        int64_t grid = whole ? pairs : attn_max_items(a.B, a.nh, a.visible, a.target);
        if (a.lines) grid = (grid / a.nh + 7) / 8 * 8 * a.nh;
        const AttnMode mode = whole ? kWhole : win ? kWindow : kAll;
        if (bits8) launch_attn8(a, mode, unsigned(grid), s);
        else if (a.c.type == IQ_KV_BF16) launch_attn<IQ_KV_BF16>(a, mode, unsigned(grid), s);
        else launch_attn<IQ_KV_F16>(a, mode, unsigned(grid), s);
        if (whole) continue;
        // (a sequence has at most target / nh chunks and one more)
        const bool many = a.B <= 4 && std::min<int64_t>(capt / kAttnWaves, a.target / a.nh) > 64;
        const int th = many ? 1024 : 256;
        const dim3 heads{unsigned(q_heads), unsigned(a.B)};
        if (weights) {
            float* w = weights + int64_t(b0) * a.c.hk * weights_ld;
            const float up = a.c.type == IQ_KV_F16 ? Terms<IQ_KV_F16>::kUp : Terms<IQ_KV_BF16>::kUp;
            const dim3 all{unsigned(q_heads + (int64_t(a.t.cap) + th - 1) / th * a.c.hk), unsigned(a.B)};
            if (many) attn_weights_kernel<1024><<<all, 1024, 0, s>>>(a, w, weights_ld, up);
            else attn_weights_kernel<256><<<all, 256, 0, s>>>(a, w, weights_ld, up);
        } else if (capt > kAttnWaves) {  // (else no sequence has two chunks)
            if (many) attn_join_kernel<1024><<<heads, 1024, 0, s>>>(a);
            else attn_join_kernel<256><<<heads, 256, 0, s>>>(a);
        }
    }
    return int(hipGetLastError());
}

}  // namespace
}  // namespace iq

extern "C" {

int iq_attn_decode(const float* q, const iq_kv* kv, const int32_t* table, int64_t table_ld, int64_t max_pages,
                   const int32_t* lens, int B, int q_heads, float scale, float* out, float* weights,
                   int64_t weights_ld, void* stream) {
    iq::AttnArgs a{};
    int rc = iq::check_kv(kv, &a.c);
    if (rc) return rc;
    rc = iq::check_table(a.c, table, table_ld, max_pages, lens, B, &a.t);
    if (rc) return rc;
    return iq::attn_decode(a, q, B, q_heads, scale, 0, 0, out, weights, weights_ld, static_cast<hipStream_t>(stream));
}

int iq_attn_decode_window(const float* q, const iq_kv* kv, const iq_kv_scales* scales, const int32_t* table,
                          int64_t table_ld, int64_t max_pages, const int32_t* lens, int B, int q_heads, float scale,
                          int64_t window, int64_t sinks, float* out, void* stream) {
    iq::AttnArgs a{};
    int rc = iq::check_any_kv(kv, scales, &a.c, &a.scales);
    if (rc) return rc;
    rc = iq::check_table(a.c, table, table_ld, max_pages, lens, B, &a.t);
    if (rc) return rc;
    return iq::attn_decode(a, q, B, q_heads, scale, window, sinks, out, nullptr, 0, static_cast<hipStream_t>(stream));
}

}  // extern "C"
