// iq_attn.hip -- attention of one new token a sequence over a paged cache.
#include "iq_kv.h"

namespace iq {
namespace {

struct AttnArgs {
    KvView c;
    KvTable t;
    const float* q;
    float* out;
    float* w;
    int64_t wld;
    float* ml;  // [B][hq][2]: running maximum and sum of every head
    int hq, group;
    float scale;
};

// The score of token tok (or -inf past the end).
template <int TYPE>
__device__ float score(const AttnArgs& a, const float* q, int b, int j, int tok, bool* bad) {
    const int p = tok / a.c.ps, id = a.t.table[b * a.t.ld + p];
    if (id < 0 || id >= a.c.pages) {
        *bad = true;
        return 0.0f;
    }
    const uint16_t* k = reinterpret_cast<const uint16_t*>(a.c.k) + id * a.c.pstr + int64_t(tok - p * a.c.ps) * a.c.sstr +
                        j * a.c.hstr;
    float s = 0.0f;
    for (int i = 0; i < a.c.d; i++) s = fmaf(kv_to_f32<TYPE>(k[i]), q[i], s);
    return s * a.scale;
}

// One wave per (head, sequence), 64 tokens at a time.
template <int TYPE>
__global__ __launch_bounds__(64) void attn_simple_kernel(AttnArgs a) {
    __shared__ float q[256], ps[64];
    __shared__ int64_t off[64];
    const int h = blockIdx.x, b = blockIdx.y, j = h / a.group, lane = threadIdx.x, d = a.c.d;
    const int n = a.t.lens[b];
    for (int i = lane; i < d; i += 64) q[i] = a.q[(int64_t(b) * a.hq + h) * d + i];
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o[4] = {0, 0, 0, 0};
    bool bad = n < 0 || n > a.t.cap;
    for (int t0 = 0; !bad && t0 < n; t0 += 64) {
        const int tok = t0 + lane;
        const float s = tok < n ? score<TYPE>(a, q, b, j, tok, &bad) : -INFINITY;
        if (__any(bad)) {
            bad = true;
            break;
        }
        float mx = s;
        for (int x = 32; x; x >>= 1) mx = fmaxf(mx, __shfl_xor(mx, x));
        const float mn = fmaxf(m, mx), al = expf(m - mn), p = expf(s - mn);
        float sum = p;
        for (int x = 32; x; x >>= 1) sum += __shfl_xor(sum, x);
        l = l * al + sum;
        m = mn;
        ps[lane] = p;
        if (tok < n) {
            const int pg = tok / a.c.ps;
            off[lane] = a.t.table[b * a.t.ld + pg] * a.c.pstr + int64_t(tok - pg * a.c.ps) * a.c.sstr + j * a.c.hstr;
        }
        __syncthreads();
        for (int r = 0; r < 4; r++) o[r] *= al;
        for (int i = 0; i < min(64, n - t0); i++) {
            const uint16_t* v = reinterpret_cast<const uint16_t*>(a.c.v) + off[i];
            for (int r = 0; r < 4; r++)
                if (r * 64 + lane < d) o[r] = fmaf(ps[i], kv_to_f32<TYPE>(v[r * 64 + lane]), o[r]);
        }
        __syncthreads();
    }
    const float inv = bad ? __builtin_nanf("") : (n == 0 ? 0.0f : 1.0f / l);
    for (int r = 0; r < 4; r++)
        if (r * 64 + lane < d) a.out[(int64_t(b) * a.hq + h) * d + r * 64 + lane] = n == 0 ? 0.0f : o[r] * inv;
    if (a.w && lane == 0) {
        a.ml[(int64_t(b) * a.hq + h) * 2] = m;
        a.ml[(int64_t(b) * a.hq + h) * 2 + 1] = bad ? __builtin_nanf("") : l;
    }
}

template <int TYPE>
__global__ __launch_bounds__(256) void weights_simple_kernel(AttnArgs a) {
    const int j = blockIdx.x, b = blockIdx.y, d = a.c.d;
    const int n = a.t.lens[b];
    if (n < 0 || n > a.t.cap) return;
    for (int tok = threadIdx.x; tok < n; tok += 256) {
        float sum = 0.0f;
        for (int g = 0; g < a.group; g++) {
            const int64_t h = int64_t(b) * a.hq + j * a.group + g;
            bool bad = false;
            const float s = score<TYPE>(a, a.q + h * d, b, j, tok, &bad);
            sum += expf(s - a.ml[2 * h]) / a.ml[2 * h + 1];
        }
        a.w[(int64_t(b) * a.c.hk + j) * a.wld + tok] += sum;
    }
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
    if (q_heads < 1 || q_heads > 16384 || q_heads % a.c.hk || !std::isfinite(scale)) return IQ_ESHAPE;
    if (weights && weights_ld < a.t.cap) return IQ_ESHAPE;
    const int64_t bytes = int64_t(B) * q_heads * a.c.d * 4;
    if (iq::ranges_overlap(q, bytes, out, bytes)) return IQ_EALIAS;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    iq::Workspace* ws = nullptr;
    const hipError_t e = iq::get_workspace(s, &ws);
    if (e != hipSuccess) return e == hipErrorOutOfMemory ? IQ_ENOMEM : int(e);
    a.q = q;
    a.out = out;
    a.w = weights;
    a.wld = weights_ld;
    a.ml = ws->partials;
    a.hq = q_heads;
    a.group = q_heads / a.c.hk;
    a.scale = scale;
    if (int64_t(B) * q_heads * 2 > ws->part_floats) return IQ_ETOOLARGE;
    const dim3 g1(static_cast<unsigned>(q_heads), static_cast<unsigned>(B)), g2(static_cast<unsigned>(a.c.hk), static_cast<unsigned>(B));
    if (kv->type == IQ_KV_BF16) {
        iq::attn_simple_kernel<IQ_KV_BF16><<<g1, 64, 0, s>>>(a);
        if (weights) iq::weights_simple_kernel<IQ_KV_BF16><<<g2, 256, 0, s>>>(a);
    } else {
        iq::attn_simple_kernel<IQ_KV_F16><<<g1, 64, 0, s>>>(a);
        if (weights) iq::weights_simple_kernel<IQ_KV_F16><<<g2, 256, 0, s>>>(a);
    }
    return int(hipGetLastError());
}

}  // extern "C"
