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
// Whole numbers of eight bits by sums with 1.5 2^23: the sum's last bits are the whole number, rounded to the nearest, even where two are
#define PG_MAGIC 12582912.f
// Sixteen numbers / scale as codes, packed.  A code is the quotient, rounded to float32, rounded to a whole number.  The product with the scale's inverse is off by less than 2^-16 of a code, so only where one of
// the sixteen is that near to a middle h of two codes (or no number), more is asked: x - h scale, whose sign an fma gives exactly, says on which side of h the quotient is, and whether it rounds to h itself,
// where the even code is taken.  (bfloat16 numbers often lie in the middle: their largest has eight bits.  Divisions instead: 6 385 tokens 36 us, divisions for every number 63; 33 now.)
PS_D uint32_t pg_pack(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410); } // of their lowest bytes
struct PgDivide {
    float scale, inv, near;
    PS_D PgDivide(float s) : scale(s), inv(s > 0.f ? 1.f / s : 0.f), near(s > 0x1p-120f && s < 0x1p120f ? 0.5f - 0x1p-16f : -1.f) {} // (scales near float32's ends: their inverses are no good)
    PS_D int middle(float x, float c) const { // c: the code, or the one beside it
        const float off = fmaf(x, inv, -c), h = c + copysignf(0.5f, off), above = fmaf(-h, scale, x);
        if (x != x) return 0;
        if (fabsf(off) < near) return (int)c;
        const float step = __uint_as_float((__float_as_uint(h) & 0x7f800000u) - (24u << 23)); // half a step of float32 at h
        const float half = fabsf(h) == 0.5f && above * h < 0.f ? 0.5f * step : step;           // (below a power of two its steps are half as long)
        if (fabsf(above) <= half * scale) return 2 * __float2int_rn(0.5f * h);                // the even one of h - 1/2, h + 1/2
        return (int)(above > 0.f ? h + 0.5f : h - 0.5f);
    }
    PS_D int divided(float x) const {
        const float q = scale > 0.f ? __fdiv_rn(x, scale) : 0.f;
        return q == q ? __float2int_rn(fmaxf(-127.f, fminf(127.f, q))) : 0;
    }
    PS_D uint4 operator()(const float (&x)[16]) const {
        uint32_t t[16];
        float worst = 0.f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float m = fmaf(x[i], inv, PG_MAGIC), off = fmaf(x[i], inv, -(m - PG_MAGIC));
            t[i] = __float_as_uint(m);
            asm("max.NaN.f32 %0, %1, %2;" : "=f"(worst) : "f"(worst), "f"(fabsf(off)));
        }
        if (!(worst < near)) {
#pragma unroll
            for (int i = 0; i < 16; i++) t[i] = (uint32_t)(near > 0.f ? middle(x[i], __uint_as_float(t[i]) - PG_MAGIC) : divided(x[i]));
        }
        return make_uint4(pg_pack(t[0], t[1], t[2], t[3]), pg_pack(t[4], t[5], t[6], t[7]), pg_pack(t[8], t[9], t[10], t[11]), pg_pack(t[12], t[13], t[14], t[15]));
    }
};
// a byte's code under another scale, f = old / new, at most 1: in the lowest byte
PS_D uint32_t pg_recode(uint32_t codes, int byte, float f) {
    const float x = __uint_as_float(__byte_perm(codes ^ 0x80808080u, 0x4b000000u, 0x7540 + byte)) - 8388736.f; // (the code + 128 as the last bits of 2^23)
    return __float_as_uint(__fadd_rn(__fmul_rn(x, f), PG_MAGIC));
}
PS_D uint32_t pg_recode4(uint32_t codes, float f) { return pg_pack(pg_recode(codes, 0, f), pg_recode(codes, 1, f), pg_recode(codes, 2, f), pg_recode(codes, 3, f)); }
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
