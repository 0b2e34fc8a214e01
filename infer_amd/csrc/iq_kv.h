// iq_kv.h -- the paged key/value cache as the kernels of iq_kv.hip (append,
// eviction) and iq_attn.hip (attention) see it, and the host's checks of it.
#pragma once

#include <cmath>

#include "../../include/iq.h"
#include "iq_attn_plan.h"
#include "iq_internal.h"

namespace iq {

// Kernel-argument copy of iq_kv, strides in elements of 2 bytes (at most
// 2^30, so that a product with an index is one 32 x 32 bit multiplication).
struct KvView {
    int32_t type, hk, d, ps;
    int64_t pages;
    uint32_t pstr, sstr, hstr;
    const char* k;
    const char* v;
    PageDiv div;  // by ps
};

// A batch's block table: row b's page ids at table + b * ld, at most
// max_pages of them; cap = max_pages * ps tokens a sequence can hold.
struct KvTable {
    const int32_t* table;
    int64_t ld;
    const int32_t* lens;
    int32_t max_pages, cap;
};

constexpr int kMaxSeqs = 1024;

// Element offset of (page id, slot, head) in either pool, id in [0, pages).
__device__ __forceinline__ int64_t kv_element(const KvView& c, uint32_t id, uint32_t slot, uint32_t head) {
    return int64_t(uint64_t(id) * c.pstr + uint64_t(slot) * c.sstr + uint64_t(head) * c.hstr);
}

// Element of a 16-bit cache as fp32, and back (to nearest even).
template <int TYPE>
__device__ __forceinline__ float kv_to_f32(uint16_t u) {
    if constexpr (TYPE == IQ_KV_BF16) return bf16_to_f32(u);
    else return float(__builtin_bit_cast(_Float16, u));
}
template <int TYPE>
__device__ __forceinline__ uint16_t f32_to_kv(float f) {
    if constexpr (TYPE == IQ_KV_BF16) return f32_to_bf16(f);
    else return __builtin_bit_cast(uint16_t, _Float16(f));
}

// Inclusive prefix sum over a wave's lanes (DPP: no LDS).
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ uint32_t dpp_add(uint32_t v) {
    return v + uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, ROW_MASK, 0xf, true));
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v = dpp_add<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8: within 16 lanes
    v = dpp_add<0x112, 0xf>(v);
    v = dpp_add<0x114, 0xf>(v);
    v = dpp_add<0x118, 0xf>(v);
    v = dpp_add<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
    v = dpp_add<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
    return v;
}
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int lane) {
    return uint32_t(__builtin_amdgcn_readlane(int(v), lane));
}

inline bool ranges_overlap(const void* a, int64_t abytes, const void* b, int64_t bbytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && x < y + uintptr_t(bbytes) && y < x + uintptr_t(abytes);
}

// The limits keep every byte offset (below 2 * 3 * 2^31 * 2^30) inside 64 bits
// and every page id inside an int32.
inline int check_kv(const iq_kv* kv, KvView* out) {
    if (!kv) return IQ_ENULL;
    if (kv->type != IQ_KV_BF16 && kv->type != IQ_KV_F16) return IQ_EKIND;
    if (kv->kv_heads < 1 || kv->kv_heads > 1024 || kv->page_size < 1) return IQ_ESHAPE;
    if (kv->head_dim < 8 || kv->head_dim > 256 || kv->head_dim % 8) return IQ_ESHAPE;
    if (kv->pages < 1 || kv->pages > 0x7fffffff) return IQ_ESHAPE;
    // (a stride over a single page, slot or head is not used)
    const int64_t count[3] = {kv->pages, kv->page_size, kv->kv_heads};
    int64_t stride[3] = {kv->page_stride, kv->slot_stride, kv->head_stride};
    for (int i = 0; i < 3; i++) {
        if (count[i] == 1) stride[i] = 0;
        else if (stride[i] < 8 || stride[i] > int64_t(1) << 30 || stride[i] % 8) return IQ_ESHAPE;
    }
    if (!kv->k || !kv->v) return IQ_ENULL;
    if (reinterpret_cast<uintptr_t>(kv->k) % 16 || reinterpret_cast<uintptr_t>(kv->v) % 16) return IQ_ESHAPE;
    out->type = kv->type;
    out->hk = kv->kv_heads;
    out->d = kv->head_dim;
    out->ps = kv->page_size;
    out->pages = kv->pages;
    out->pstr = uint32_t(stride[0]);
    out->sstr = uint32_t(stride[1]);
    out->hstr = uint32_t(stride[2]);
    out->k = static_cast<const char*>(kv->k);
    out->v = static_cast<const char*>(kv->v);
    out->div = page_div(uint32_t(kv->page_size));
    return IQ_OK;
}

inline int check_table(const KvView& c, const int32_t* table, int64_t ld, int64_t max_pages, const int32_t* lens,
                       int B, KvTable* out) {
    if (!table || !lens) return IQ_ENULL;
    if (B < 1 || B > kMaxSeqs || max_pages < 1 || ld < max_pages || ld > 0x7fffffff) return IQ_ESHAPE;
    if (max_pages * int64_t(c.ps) > 0x7fff0000) return IQ_ETOOLARGE;
    out->table = table;
    out->ld = ld;
    out->lens = lens;
    out->max_pages = int32_t(max_pages);
    out->cap = int32_t(max_pages * c.ps);
    return IQ_OK;
}

}  // namespace iq
