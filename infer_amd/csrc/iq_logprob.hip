// iq_logprob.hip -- log probabilities, entropy and top alternatives of rows
// of logits.
#include <cmath>

#include "../../include/iq.h"
#include "iq_kv.h"

namespace iq {
namespace {

struct LogprobArgs {
    const float* x;
    int64_t ld, V;
    const int64_t* tokens;
    int top;
    float *lp, *ent;
    int64_t* ids;
    float* tlp;
};

// Order of the logits: by value (-0 as 0), NaN largest.
__device__ __forceinline__ uint32_t logit_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__global__ __launch_bounds__(1024) void logprob_simple_kernel(LogprobArgs a) {
    __shared__ float sm[16], ss[16], su[16];
    __shared__ unsigned long long sb[16];
    const int64_t t = blockIdx.x;
    const float* x = a.x + t * a.ld;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    float m = -INFINITY;
    bool bad = false;
    for (int64_t i = tid; i < a.V; i += 1024) {
        m = fmaxf(m, x[i]);
        bad |= !(x[i] < INFINITY);
    }
    bad = __syncthreads_or(bad);
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if (lane == 0) sm[wave] = m;
    __syncthreads();
    for (int i = 0; i < 16; i++) m = fmaxf(m, sm[i]);
    float s = 0.0f, u = 0.0f;
    for (int64_t i = tid; i < a.V; i += 1024) {
        const float dx = x[i] - m, e = expf(dx);
        s += e;
        if (e > 0.0f) u += e * dx;
    }
    for (int o = 32; o; o >>= 1) {
        s += __shfl_xor(s, o);
        u += __shfl_xor(u, o);
    }
    if (lane == 0) {
        ss[wave] = s;
        su[wave] = u;
    }
    __syncthreads();
    s = u = 0.0f;
    for (int i = 0; i < 16; i++) {
        s += ss[i];
        u += su[i];
    }
    const float nan = __builtin_nanf("");
    const float lz = bad || m == -INFINITY ? nan : logf(s);
    if (tid == 0) {
        if (a.lp) {
            const int64_t k = a.tokens[t];
            a.lp[t] = k >= 0 && k < a.V ? x[k] - m - lz : nan;
        }
        if (a.ent) a.ent[t] = lz - u / s;
    }
    unsigned long long last = ~0ull;
    for (int r = 0; r < a.top; r++) {
        unsigned long long best = 0;
        for (int64_t i = tid; i < a.V; i += 1024) {
            const unsigned long long k = (static_cast<unsigned long long>(logit_key(x[i])) << 32) | (0xffffffffu - uint32_t(i));
            if ((r == 0 || k < last) && k > best) best = k;
        }
        for (int o = 32; o; o >>= 1) {
            const unsigned long long k = __shfl_xor(best, o);
            if (k > best) best = k;
        }
        __syncthreads();
        if (lane == 0) sb[wave] = best;
        __syncthreads();
        for (int i = 0; i < 16; i++)
            if (sb[i] > best) best = sb[i];
        last = best;
        if (tid == 0) {
            const uint32_t id = 0xffffffffu - uint32_t(best);
            a.ids[t * a.top + r] = id;
            a.tlp[t * a.top + r] = x[id] - m - lz;
        }
    }
}

}  // namespace
}  // namespace iq

extern "C" {

int iq_logprobs(const float* logits, int64_t ld, int64_t T, int64_t V, const int64_t* tokens, int top,
                float* logprob, float* entropy, int64_t* top_ids, float* top_logprobs, void* stream) {
    if (T < 1 || V < 1 || ld < V || top < 0 || top > 64 || top > V) return IQ_ESHAPE;
    if (!logits || !tokens != !logprob || (top && (!top_ids || !top_logprobs))) return IQ_ENULL;
    if (!logprob && !entropy && !top) return IQ_ENULL;
    if (V > 0x7fffffff - 65536 || T > 0x7fffffff) return IQ_ETOOLARGE;
    iq::LogprobArgs a{logits, ld, V, tokens, top, logprob, entropy, top_ids, top_logprobs};
    iq::logprob_simple_kernel<<<static_cast<unsigned>(T), 1024, 0, static_cast<hipStream_t>(stream)>>>(a);
    return int(hipGetLastError());
}

}  // extern "C"
