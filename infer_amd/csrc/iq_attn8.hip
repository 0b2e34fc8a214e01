// iq_attn8.hip -- attention of one new token a sequence over a paged cache of
// 8-bit codes with a scale for each block of tokens and key/value head.
//
// As iq_attn.hip, which launches it and joins its chunks, with the scores and
// sums
//   S^T[token][head] = (scale * ks[token]) (K[token][d] . q^T[d][head])
//   O^T[d][head]    += V^T[d][token] . (vs[token] P^T[token][head])
// on the codes as they are: both code types are exact in bf16 (8 bits of a
// mantissa hold -127..127; e4m3 is a part of bf16), so a tile's rows go through
// LDS as bytes and become bf16 operands in registers.  A key's scale multiplies
// its score, a value's its weight before that is cut into three bf16 terms,
// which have fp32's range, so that scales from 2^-86 on lose nothing.
//
// What bounds it is the read of the cache: 131072 tokens of 4 int8 heads of 128 in
// 31 us (4.3 TB/s over all, 5.2 behind the first tile, where a plain read reaches
// 5.5 on as many bytes), every byte read once, the vector units busy for 45 % of it
// (int8 to bf16: 1.5 operations a code; e4m3: 0.5), the matrix cores for 18 %, no
// bank conflicts.  The rest is a launch with its chain of length, page id and
// rows (4.2 us; 5.6 for 24 sequences of up to 2047, 16 heads of 64), a tile's products
// (1.2 to 1.5) and the chunk's end (1): 32 sequences of up to 8192, 2 e4m3 heads, 15.1 us
// (2.9 TB/s).  Two tiles ahead instead of one gain nothing (131072 tokens,
// both launches, 33.2 and 33.9 us).
//
// K: a lane's 16 bytes are two 8-value operands, so the 32-value steps of the
// product go over bytes 16 g .. 16 g + 7 and 16 g + 8 .. 16 g + 15 of 64, and q is
// laid out alike.  V: ds_read_b64_tr_b8 gives a lane one column of 8 rows, the
// tokens 4 g + 0..3 of either half, which is P's order.
#include "iq_attn.h"

namespace iq {
namespace {

typedef int i32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

// 8 codes to bf16, exactly.
template <int TYPE>
__device__ __forceinline__ s16x8_t codes_bf16(uint32_t lo, uint32_t hi) {
    u32x4_t r;
    if constexpr (TYPE == IQ_KV_I8) {
        uint32_t x, y;
        bf16_int8_x4(lo, x, y);
        r[0] = x;
        r[1] = y;
        bf16_int8_x4(hi, x, y);
        r[2] = x;
        r[3] = y;
    } else {
        auto two = [](uint32_t v, auto up) {
            return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, 1.0f, decltype(up)::value));
        };
        r[0] = two(lo, std::false_type{});
        r[1] = two(lo, std::true_type{});
        r[2] = two(hi, std::false_type{});
        r[3] = two(hi, std::true_type{});
    }
    return __builtin_bit_cast(s16x8_t, r);
}

// DP: head_dim rounded up to 32, 64, 128 or 256.
template <int TYPE, int DP, int MODE>
__global__ __launch_bounds__(64 * kAttnWaves, DP > 128 ? 1 : 2) void attn8_kernel(AttnArgs a) {
    using T = Terms<IQ_KV_BF16>;
    constexpr bool WIN = MODE != kAll;
    constexpr int CH = DP / 16, RPI = 64 / CH, NI = kAttnTile / RPI;  // 16-byte chunks of a row, rows of a load, loads
    constexpr int KC = DP / 32, VT = DP / 16;                         // steps of the first product, tiles of the second
    constexpr int KVB = kAttnTile * DP;
    constexpr int OST = DP + 4;  // floats from head to head of a wave's sums
    constexpr int WB = 2 * KVB > 16 * OST * 4 ? 2 * KVB : 16 * OST * 4;
    __shared__ __align__(16) char lds[kAttnWaves][WB];
    __shared__ __align__(16) float tile_ks[kAttnWaves][kAttnTile], tile_vs[kAttnWaves][kAttnTile];
    __shared__ float wm[kAttnWaves][16], wl[kAttnWaves][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, col = lane & 15;
    Item it;
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

    // Token r of a tile and its page's id, and from these the element offset of
    // its (page, slot) and its scales'; 0 where there is none.  Past the last token
    // it is the last one again: its score is masked, and no row has to be.
    bool poison = false;
    const int32_t* table = a.t.table + b * a.t.ld;
    struct Row {
        int64_t at, scale;
    };
    auto token = [&](int tile) {
        const int tok = min(t0 + tile * kAttnTile + (lane & 31), t1 - 1);
        return uint32_t(WIN && tok >= a.sinks ? tok + (n - it.seen) : tok);
    };
    auto page_id = [&](int tile) { return table[page_of(token(tile), a.c.div)]; };
    auto row_of = [&](int tile, int32_t id) -> Row {
        const uint32_t tok = token(tile), s = tok - page_of(tok, a.c.div) * uint32_t(a.c.ps);
        const bool ok = id >= 0 && id < a.c.pages;
        poison |= !ok;
        const uint32_t p = ok ? uint32_t(id) : 0;
        return {kv_element(a.c, p, s, 0), kv_scale(a.scales, p, s, uint32_t(j))};
    };
    // chunks past the row's end repeat its first one (q is 0 there, and the
    // sums of those columns are not written)
    const int ch = lane % CH, chsrc = ch * 16 < d ? ch : 0;
    const int64_t lane_off = int64_t(uint64_t(j) * a.c.hstr) + chsrc * 16;
    const char* kp = a.c.k + lane_off;
    const char* vp = a.c.v + lane_off;
    struct Tile {
        u32x4_t k[NI], v[NI];
        float ks, vs;
    };
    Tile ahead;
    auto load = [&](Tile& t, Row r) {
        t.ks = a.scales.k[r.scale];
        t.vs = a.scales.v[r.scale];
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int64_t o = __shfl(r.at, i * RPI + lane / CH);
            t.k[i] = *reinterpret_cast<const u32x4_t*>(kp + o);
            t.v[i] = *reinterpret_cast<const u32x4_t*>(vp + o);
        }
    };
    // Chunk c of row r lies at chunk c ^ swizzle(r) of the row's place.  A K
    // read takes a chunk of 16 rows; half a wave's V read one of the rows 0..7
    // and 16..23 (or 8 on): each then meets every bank equally often.
    constexpr int RPB = 256 / DP > 1 ? 256 / DP : 1;  // rows across the banks
    auto ksw = [](int r) { return (r / RPB) & (CH < 16 ? CH - 1 : 15); };
    auto vsw = [](int r) { return (((r & 7) + (r >> 4) * 8) / RPB) & (CH - 1); };
    char* kl = lds[wave];
    char* vl = lds[wave] + KVB;

    const int32_t id0 = page_id(wave);
    int32_t next_id = page_id(wave + kAttnWaves);
    // q: column = head, 8 values of each 32-value step a lane
    s16x8_t qt[KC][T::N];
    {
        const float* q = a.q + (int64_t(b) * a.hq + j * a.group + h0 + (col < gh ? col : 0)) * d;
        // steps 2 i and 2 i + 1 take the halves of a lane's 16 bytes
        auto first_of = [&](int c) { return DP == 32 ? g * 8 : (c >> 1) * 64 + g * 16 + (c & 1) * 8; };
        float x[KC][8];
#pragma unroll
        for (int c = 0; c < KC; c++) {
            const int e = first_of(c);
#pragma unroll
            for (int i = 0; i < 8; i++) x[c][i] = q[(e < d ? e : 0) + i];
        }
        load(ahead, row_of(wave, id0));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int c = 0; c < KC; c++) {
            const bool in = col < gh && first_of(c) < d;
#pragma unroll
            for (int i = 0; i < 8; i++) x[c][i] = in ? x[c][i] : 0.0f;
            T::cut(x[c], qt[c]);
        }
    }

    float4_t o[VT];
#pragma unroll
    for (int i = 0; i < VT; i++) o[i] = float4_t{0, 0, 0, 0};
    float m = kNone, l = 0.0f;

    for (int tile = wave; tile < ntiles; tile += kAttnWaves) {
        const int tk = t0 + tile * kAttnTile;  // first token
        const bool whole = tk + kAttnTile <= t1;
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int r = i * RPI + lane / CH;
            *reinterpret_cast<u32x4_t*>(kl + r * DP + (ch ^ ksw(r)) * 16) = ahead.k[i];
            *reinterpret_cast<u32x4_t*>(vl + r * DP + (ch ^ vsw(r)) * 16) = ahead.v[i];
        }
        if (lane < kAttnTile) {
            // (an infinite one becomes NaN, by the sum with 0 times it: its negative
            // products, -inf, would weigh nothing)
            tile_ks[wave][lane] = fmaf(ahead.ks, a.mul, ahead.ks * 0.0f);
            tile_vs[wave][lane] = ahead.vs;
        }
        // the next tile's loads, and the id behind it ahead of them: a wait for it
        // then leaves them in flight (131072 tokens of 4 int8 heads: 35.7 and 31.1 us)
        if (tile + kAttnWaves < ntiles) {
            const Row r = row_of(tile + kAttnWaves, next_id);
            next_id = page_id(tile + 2 * kAttnWaves);
            load(ahead, r);
            __builtin_amdgcn_sched_barrier(0);
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
        float s[8], w[8];
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
            float4_t acc = {0, 0, 0, 0};
            const int r = hf * 16 + col;
            if constexpr (DP == 32) {
                const uint2 kv = *reinterpret_cast<const uint2*>(kl + r * DP + ((g >> 1) ^ ksw(r)) * 16 + (g & 1) * 8);
                const s16x8_t kx = codes_bf16<TYPE>(kv.x, kv.y);
#pragma unroll
                for (int k = 0; k < T::N; k++) acc = T::mma(kx, qt[0][k], acc);
            } else {
#pragma unroll
                for (int c = 0; c < KC / 2; c++) {
                    const u32x4_t kv = *reinterpret_cast<const u32x4_t*>(kl + r * DP + ((c * 4 + g) ^ ksw(r)) * 16);
                    const s16x8_t k0 = codes_bf16<TYPE>(kv[0], kv[1]), k1 = codes_bf16<TYPE>(kv[2], kv[3]);
#pragma unroll
                    for (int k = 0; k < T::N; k++) acc = T::mma(k0, qt[2 * c][k], acc);
#pragma unroll
                    for (int k = 0; k < T::N; k++) acc = T::mma(k1, qt[2 * c + 1][k], acc);
                }
            }
            const float4_t k4 = *reinterpret_cast<const float4_t*>(&tile_ks[wave][hf * 16 + g * 4]);
            const float4_t v4 = *reinterpret_cast<const float4_t*>(&tile_vs[wave][hf * 16 + g * 4]);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int tok = tk + hf * 16 + g * 4 + i;
                float x = acc[i] * k4[i];
                if (!whole && tok >= t1) x = -INFINITY;
                s[hf * 4 + i] = x;
                w[hf * 4 + i] = v4[i];
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
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float p = __builtin_amdgcn_exp2f(s[i] - m);
            l += p;
            w[i] *= p;
        }
        s16x8_t pt[T::N];
        T::cut(w, pt);
#pragma unroll
        for (int v = 0; v < VT; v++) {
            // rows 4g..4g+3 of either half: lane 2r + c of 16 gives row r's
            // 8-byte piece c, lane i gets the 8 rows' value of column i
            const int r8 = col >> 1, r = (r8 >> 2) * 16 + g * 4 + (r8 & 3);
            const int at = r * DP + (v ^ vsw(r)) * 16 + (col & 1) * 8;
            const i32x2_t x = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                reinterpret_cast<__attribute__((address_space(3))) i32x2_t*>(
                    (__attribute__((address_space(3))) char*)(vl) + at));
            const s16x8_t av = codes_bf16<TYPE>(uint32_t(x[0]), uint32_t(x[1]));
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
            x *= inv_sum(L);
            to = out + h * d + e;
        } else {
            to = a.part + slot * 16 * d + h * d + e;
        }
        if (e == 0 && !alone) {
            float* f = a.ml + slot * 32 + h * 2;
            f[0] = M;
            f[1] = L;
        }
#pragma unroll
        for (int r = 0; r < 4; r++) to[r] = x[r];
    }
}

template <int TYPE, int MODE>
void launch_mode(const AttnArgs& a, unsigned grid, hipStream_t s) {
    if (a.c.d <= 32) attn8_kernel<TYPE, 32, MODE><<<grid, 64 * kAttnWaves, 0, s>>>(a);
    else if (a.c.d <= 64) attn8_kernel<TYPE, 64, MODE><<<grid, 64 * kAttnWaves, 0, s>>>(a);
    else if (a.c.d <= 128) attn8_kernel<TYPE, 128, MODE><<<grid, 64 * kAttnWaves, 0, s>>>(a);
    else attn8_kernel<TYPE, 256, MODE><<<grid, 64 * kAttnWaves, 0, s>>>(a);
}

template <int TYPE>
void launch(const AttnArgs& a, AttnMode mode, unsigned grid, hipStream_t s) {
    (mode == kWhole ? launch_mode<TYPE, kWhole> : mode == kWindow ? launch_mode<TYPE, kWindow> : launch_mode<TYPE, kAll>)(a, grid, s);
}

}  // namespace

// Measured with 1, 2 and 3 a CU, both launches: 131072 tokens of 4 int8 heads of
// 128 33.1, 35.3, 37 us, 32 sequences of up to 8192 (e4m3) 17.3, 18.4, 20; 8 of 8192
// with heads of 256 39, 46, 55; heads of 64 (24 of up to 2047) 16.0, 16.9, 15.5;
// of 32 (8 of 16384) 32.5, 26.0, 25.5.  Where one a CU keeps enough rows in
// flight, more of them only add chunks.
int attn8_groups(int head_dim) { return head_dim <= 64 ? 3 : 1; }

void launch_attn8(const AttnArgs& a, AttnMode mode, unsigned grid, hipStream_t s) {
    if (a.c.type == IQ_KV_I8) launch<IQ_KV_I8>(a, mode, grid, s);
    else launch<IQ_KV_E4M3>(a, mode, grid, s);
}

}  // namespace iq
