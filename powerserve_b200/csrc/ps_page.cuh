// ps_page.cuh - caches in 8 bits and in pages: what their kernels share (layout: include/ps_cuda.h, "paged caches in 8 bits").
#pragma once
#include "ps_ptx.cuh"
#include "ps_serve.h"

#include <cuda_bf16.h>

#define PG_SEQS 256     // sequences of a launch: their table is a kernel parameter
#define PG_BLOCK PS_CUDA_BLOCK_TOKENS

struct PgPool {         // of one layer, or (edit, compact) of the first of all
    int8_t *codes;
    float *scales;
    int n_pages, P, shift, G, hs;   // P = 2^shift slots of a page
    int *err;
    PS_HD int64_t page_codes() const { return (int64_t)P * hs; }
    // number of a page's, head's K (0) or V (1): times P hs codes, times P / 16 scales
    PS_HD int64_t at(int page, int g, int kv) const { return ((int64_t)page * G + g) * 2 + kv; }
    PS_D bool has(int page) const {
        const bool ok = (unsigned)page < (unsigned)n_pages;
        if (!ok) *err = PS_ERR_PAGE;
        return ok;
    }
};
PS_D float pg_num(float x) { return x; }
PS_D float pg_num(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> PS_D T pg_to(float x);
template <> PS_D float pg_to<float>(float x) { return x; }
template <> PS_D __nv_bfloat16 pg_to<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
// number / scale as a code (a block without numbers, or with an infinite one, has none to tell apart)
PS_D int pg_code(float x, float scale) {
    const float q = scale > 0.f ? __fdiv_rn(x, scale) : 0.f;
    return q == q ? max(-127, min(127, __float2int_rn(fmaxf(-127.f, fminf(127.f, q))))) : 0;
}
// a code under another scale, f = old / new, at most 1
PS_D int pg_recode(int code, float f) { return __float2int_rn((float)code * f); }
PS_D float pg_follow(float old, float now) { return now > 0.f ? __fdiv_rn(old, now) : 0.f; }
PS_D float pg_warp_max(float v) { // of numbers that are not negative: no number counts as 0 before
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
PS_D int pg_byte(const uint4 &v, int i) { // i-th signed byte
    const uint32_t w = i < 8 ? (i < 4 ? v.x : v.y) : (i < 12 ? v.z : v.w);
    return (int8_t)(w >> (8 * (i & 3)));
}
