// iq_attn.hip -- attention of one new token a sequence over a paged cache.
//
// With g query heads on a key/value head, every cached element is used by g
// products of each kind, and an element is 2 bytes: on the vector units that
// is 7 multiply-adds for Qwen2.5-7B where HBM delivers one element per two
// cycles and lane, too many beside the unpacking; on the matrix cores the up
// to 16 heads of a group are the 16 columns of one product and cost nothing.
// What bounds the operator is the read of the cache: 131072 tokens, 4 heads of
// 128 in bf16 take 57 us (4.71 TB/s; a device copy reaches 4.74), every byte
// read once, the matrix cores busy for 12 % of it; 32 sequences of up to 8192
// tokens, 2 heads, 21 us (4.1 TB/s).  A join adds 4 to 5 us.
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
#include <algorithm>

#include "iq_attn_plan.h"
#include "iq_kv.h"

namespace iq {
namespace {

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
};

// The maximum of no scores: finite, so that scores of -inf (products past
// fp32's range) and runs without scores count nothing instead of giving NaN.
constexpr float kNone = -3.4e38f;

// 1 / a head's sum.  It is 0 only where every score is -inf: the head's values
// are then 0 times 0 (or NaN, where a value is not finite), its weights 0.
__device__ __forceinline__ float inv_sum(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }

struct Item {
    int b, n;            // sequence and its length (as given)
    uint32_t j, c, chunks, first;  // chunk, tiles of a chunk, chunks of the sequence, its first partial
};

// The (sequence, chunk) number w of the batch's plan; false past the last.
// Every wave finds it from the lengths by itself (64 sequences a step).
__device__ bool find_item(const AttnArgs& a, uint32_t w, Item* it) {
    const int lane = threadIdx.x & 63;
    auto length = [&](int b) { return b < a.B ? a.t.lens[b] : 0; };
    auto tiles_of = [&](int n) { return n < 0 || n > a.t.cap ? 0u : attn_tiles(n); };
    int n = length(lane);
    const int n0 = n;
    uint32_t total = lane_of(wave_scan(tiles_of(n)), 63);
    for (int b0 = 64; b0 < a.B; b0 += 64) total += lane_of(wave_scan(tiles_of(length(b0 + lane))), 63);
    const uint32_t least = attn_chunk_tiles(total, a.nh, a.target);
    uint32_t c = least;
    for (int i = 0; i < kAttnTries && uint32_t(a.B) * a.nh <= a.target; i++) {
        uint32_t items = 0;
        for (int b0 = 0; b0 < a.B; b0 += 64)
            items += lane_of(wave_scan(b0 + lane < a.B ? attn_chunks(tiles_of(b0 ? length(b0 + lane) : n0), c) : 0), 63);
        if (items * a.nh <= a.target) break;
        c = attn_more_tiles(c, least);
    }
    uint32_t before = 0, first = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        if (b0) n = length(b0 + lane);
        const uint32_t k = b0 + lane < a.B ? attn_chunks(tiles_of(n), c) : 0;
        const uint32_t upto = wave_scan(k), many = k > 1 ? k : 0, pupto = wave_scan(many);
        const uint64_t past = __ballot(w < before + upto);
        if (past) {
            const int l = __builtin_ctzll(past);
            it->b = b0 + l;
            it->n = __builtin_amdgcn_readlane(n, l);
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

// DP: head_dim rounded up to 32, 64, 128 or 256.
template <int TYPE, int DP>
__global__ __launch_bounds__(64 * kAttnWaves, DP > 128 ? 1 : 2) void attn_kernel(AttnArgs a) {
    using T = Terms<TYPE>;
    constexpr int CH = DP / 8, RPI = 64 / CH, NI = kAttnTile / RPI;  // 16-byte chunks of a row, rows of a load, loads
    constexpr int KC = DP / 32, VT = DP / 16;                       // steps of the first product, tiles of the second
    constexpr int ROWB = DP * 2, KVB = kAttnTile * ROWB;
    __shared__ __align__(16) char lds[kAttnWaves][2 * KVB];
    __shared__ float wm[kAttnWaves][16], wl[kAttnWaves][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, col = lane & 15;
    Item it;
    // Heads that share cache lines (see the host side) go to one XCD for a
    // chunk: workgroups are dealt to the 8 of them in turn.
    const uint32_t turn = a.lines ? 8 : 1, round = blockIdx.x / (turn * a.nh), in = blockIdx.x % (turn * a.nh);
    const uint32_t hidx = in / turn;
    if (!find_item(a, round * turn + in % turn, &it)) return;
    const int b = it.b, n = it.n, d = a.c.d;
    const int j = int(hidx) / a.ht, h0 = int(hidx) % a.ht * 16, gh = min(16, a.group - h0);
    float* out = a.out + (int64_t(b) * a.hq + j * a.group + h0) * d;
    if (hidx == 0 && it.j == 0 && threadIdx.x == 0) a.plan[b] = make_uint2(it.chunks, it.first);
    if (n <= 0 || n > a.t.cap) {
        const float x = n == 0 ? 0.0f : __builtin_nanf("");
        for (int i = threadIdx.x; i < gh * d; i += 64 * kAttnWaves) out[i] = x;
        return;
    }
    const int t0 = int(it.j * it.c) * kAttnTile, t1 = t0 + min(n - t0, int(it.c) * kAttnTile);
    const int ntiles = (t1 - t0 + kAttnTile - 1) / kAttnTile;

    // row r of a tile: element offset of its (page, slot), 0 where there is none
    bool poison = false;
    const int32_t* table = a.t.table + b * a.t.ld;
    auto row_offset = [&](int tile) -> int64_t {
        const int tok = t0 + tile * kAttnTile + (lane & 31);
        if (tok >= t1) return 0;
        const uint32_t p = page_of(uint32_t(tok), a.c.div), s = uint32_t(tok) - p * uint32_t(a.c.ps);
        const int32_t id = table[p];
        const bool ok = id >= 0 && id < a.c.pages;
        poison |= !ok;
        return ok ? kv_element(a.c, uint32_t(id), s, 0) : 0;
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
    const int64_t off0 = row_offset(wave);
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
        if (wave < ntiles) load(off0);
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

    int64_t off_next = wave + kAttnWaves < ntiles ? row_offset(wave + kAttnWaves) : 0;
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
            load(off_next);
            if (tile + 2 * kAttnWaves < ntiles) off_next = row_offset(tile + 2 * kAttnWaves);
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
#pragma unroll
        for (int v = 0; v < VT; v++) {
            if (v * 16 >= d) continue;
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

template <int TYPE>
void launch_attn(const AttnArgs& a, unsigned grid, hipStream_t s) {
    if (a.c.d <= 32) attn_kernel<TYPE, 32><<<grid, 64 * kAttnWaves, 0, s>>>(a);
    else if (a.c.d <= 64) attn_kernel<TYPE, 64><<<grid, 64 * kAttnWaves, 0, s>>>(a);
    else if (a.c.d <= 128) attn_kernel<TYPE, 128><<<grid, 64 * kAttnWaves, 0, s>>>(a);
    else attn_kernel<TYPE, 256><<<grid, 64 * kAttnWaves, 0, s>>>(a);
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
    if (!q || !out) return IQ_ENULL;
    a.mul = scale * 1.44269504088896340736f;
    if (q_heads < 1 || q_heads > 16384 || q_heads % a.c.hk || !std::isfinite(a.mul)) return IQ_ESHAPE;
    if (weights && weights_ld < a.t.cap) return IQ_ESHAPE;
    const int64_t row = int64_t(q_heads) * a.c.d;
    if (iq::ranges_overlap(q, B * row * 4, out, B * row * 4)) return IQ_EALIAS;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    iq::Workspace* ws = nullptr;
    const hipError_t e = iq::get_workspace(s, &ws);
    if (e != hipSuccess) return e == hipErrorOutOfMemory ? IQ_ENOMEM : int(e);
    a.hq = q_heads;
    a.group = q_heads / a.c.hk;
    a.ht = (a.group + 15) / 16;
    a.nh = uint32_t(a.c.hk * a.ht);
    // as many work items as run at once: 4, 3, 2 or 1 workgroups a CU by the
    // registers (d <= 64) and the LDS of an instance.  Measured for d = 128 on
    // 131072 tokens / 32 sequences of up to 8192: 1 a CU 69.9 / 30.4 us, 2 61.8
    // / 24.7, 3 69.1 / 27.8, 4 66.0 / 29.4; for d = 64 (24 of up to 2047, 16
    // heads) 18.1, 19.0, 17.2, 18.8.
    a.target = uint32_t((a.c.d <= 32 ? 4 : a.c.d <= 64 ? 3 : a.c.d <= 128 ? 2 : 1) * iq::device_cu_count());
    // Neighbouring heads' rows meet in a cache line, or several head tiles read
    // the same rows: one XCD's L2 then serves them (8 sequences of 16384, 8 heads
    // of 32: 49.7 -> 38.8 us; of 8192, heads of 80: 50.1 -> 44.6).  Whole lines
    // are better spread (131072 tokens, 4 heads of 128: 61.9 and 64.0).
    a.lines = a.nh > 1 && (a.ht > 1 || 2 * a.c.hstr % 128 != 0);
    const int64_t capt = iq::attn_tiles(a.t.cap);
    // the workspace's partial sums: plan | final (maximum, sum) | chunks' | rows;
    // its GEMM operand area: the scores that the weights are made of
    const int64_t slots = iq::attn_max_partials(a.target);
    int64_t step = B;
    step = std::min<int64_t>(step, (int64_t(1) << 30) / (capt * a.nh));
    if (weights) step = std::min<int64_t>(step, int64_t(ws->gx_bytes / 4) / (int64_t(a.t.cap) * q_heads));
    const int64_t room = ws->part_floats - 2 * iq::kMaxSeqs - slots * 16 * (2 + a.c.d) - 63;
    step = std::min<int64_t>(step, room / (2 * q_heads));
    if (step < 1) return IQ_ETOOLARGE;
    const int64_t fin = (step * q_heads * 2 + 63) / 64 * 64;
    a.plan = reinterpret_cast<uint2*>(ws->partials);
    a.fin = ws->partials + 2 * iq::kMaxSeqs;
    a.ml = a.fin + fin;
    a.part = a.ml + slots * 32;
    a.sc = weights ? static_cast<float*>(ws->gx) : nullptr;
    for (int b0 = 0; b0 < B; b0 += int(step)) {
        a.B = int(std::min<int64_t>(step, B - b0));
        a.q = q + b0 * row;
        a.out = out + b0 * row;
        a.t.table = table + b0 * table_ld;
        a.t.lens = lens + b0;
        int64_t grid = iq::attn_max_items(a.B, a.nh, a.t.cap, a.target);
        if (a.lines) grid = (grid / a.nh + 7) / 8 * 8 * a.nh;
        if (kv->type == IQ_KV_BF16) iq::launch_attn<IQ_KV_BF16>(a, unsigned(grid), s);
        else iq::launch_attn<IQ_KV_F16>(a, unsigned(grid), s);
        // (a sequence has at most target / nh chunks and one more)
        const bool many = a.B <= 4 && std::min<int64_t>(capt / iq::kAttnWaves, a.target / a.nh) > 64;
        const int th = many ? 1024 : 256;
        const dim3 heads{unsigned(q_heads), unsigned(a.B)};
        if (weights) {
            float* w = weights + int64_t(b0) * a.c.hk * weights_ld;
            const float up = kv->type == IQ_KV_F16 ? iq::Terms<IQ_KV_F16>::kUp : iq::Terms<IQ_KV_BF16>::kUp;
            const dim3 all{unsigned(q_heads + (int64_t(a.t.cap) + th - 1) / th * a.c.hk), unsigned(a.B)};
            if (many) iq::attn_weights_kernel<1024><<<all, 1024, 0, s>>>(a, w, weights_ld, up);
            else iq::attn_weights_kernel<256><<<all, 256, 0, s>>>(a, w, weights_ld, up);
        } else if (capt > iq::kAttnWaves) {  // (else no sequence has two chunks)
            if (many) iq::attn_join_kernel<1024><<<heads, 1024, 0, s>>>(a);
            else iq::attn_join_kernel<256><<<heads, 256, 0, s>>>(a);
        }
    }
    return int(hipGetLastError());
}

}  // extern "C"
