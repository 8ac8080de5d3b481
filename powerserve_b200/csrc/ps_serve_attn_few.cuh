// ps_serve_attn_few.cuh - ps_serve_attn.cuh's attention for head sizes 64 and 128 and up to sixteen query rows of a kv head (a token or a few each): the products are as in
// ps_serve_attn_tc.cuh - fp16 parts, three MMAs for one of 32 bits - but by mma.sync on fragments that come straight from memory, without shared memory
// or barriers on the way.  With so few rows the tensor cores have little to do (a fifth of what mma.sync can), and what counts is bytes under way: a warp works
// alone on sixteen slots at a time, four warps a CTA, two or three CTAs an SM, each warp with 8 KB of K and V on the way while it computes.
// Which element of a row a thread holds is free (a sum's order is), so a thread takes neighbours: of K eight elements of a slot's row, of V four slots of a channel;
// slots are dealt to the columns of the scores so that a thread's scores are, as they lie, its fragment of the weights for the second product.
// A tile's output is added up in 32 bits outside the MMAs, after a factor of its own for every group (sixteen slots of 64 channels of V).
#pragma once
#include "ps_serve_attn_tc.cuh"

#define SV_FEW_ROWS 16

PS_D void sv_mma(float (&d)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// N neighbouring elements as floats.  mode: they begin at a 16-byte boundary (bfloat16: 2 N); live: of V, the slots that count
template <int N> PS_D void sv_read(float (&x)[N], const float *p, int mode, uint32_t live) {
    if (mode) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 v = __ldcs(reinterpret_cast<const float4 *>(p + i));
            x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = live >> i & 1 ? __ldcs(p + i) : 0.f;
    }
}
template <int N> PS_D void sv_read(uint32_t (&x)[N / 2], const __nv_bfloat16 *p, int mode, uint32_t live) {
    if (mode && N == 8) {
        const uint4 v = __ldcs(reinterpret_cast<const uint4 *>(p));
        x[0] = v.x; x[1] = v.y; x[N / 2 - 2] = v.z; x[N / 2 - 1] = v.w;
    } else if (mode) {
        const uint2 v = __ldcs(reinterpret_cast<const uint2 *>(p));
        x[0] = v.x; x[1] = v.y;
    } else {
        const uint16_t *u = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
        for (int i = 0; i < N; i += 2) x[i / 2] = (live >> i & 1 ? (uint32_t)__ldcs(u + i) : 0u) | (live >> i & 2 ? (uint32_t)__ldcs(u + i + 1) << 16 : 0u);
    }
}
// a thread's share of a group: 32 elements (head size 64, K: 16)
template <typename T, int N> struct SvShare;
template <int N> struct SvShare<float, N> {
    float x[N];
    PS_D float at(int i) const { return x[i]; }
    PS_D void keep(int i, bool yes) { x[i] = yes ? x[i] : 0.f; }
};
template <int N> struct SvShare<__nv_bfloat16, N> {
    uint32_t x[N / 2];
    PS_D float at(int i) const { return __uint_as_float(i & 1 ? x[i / 2] & 0xffff0000u : x[i / 2] << 16); }
    PS_D void keep(int i, bool yes) { if (!yes) x[i / 2] &= i & 1 ? 0x0000ffffu : 0xffff0000u; }
};
template <int M, int N> PS_D void sv_read_at(SvShare<float, N> &s, int i, const float *p, int mode, uint32_t live) {
    float v[M];
    sv_read<M>(v, p, mode, live);
#pragma unroll
    for (int e = 0; e < M; e++) s.x[i + e] = v[e];
}
template <int M, int N> PS_D void sv_read_at(SvShare<__nv_bfloat16, N> &s, int i, const __nv_bfloat16 *p, int mode, uint32_t live) {
    uint32_t v[M / 2];
    sv_read<M>(v, p, mode, live);
#pragma unroll
    for (int e = 0; e < M / 2; e++) s.x[i / 2 + e] = v[e];
}
template <typename T, int N> PS_D float sv_group_scale(const SvShare<T, N> &s, float &inv) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < N; i += 2) top = fmaxf(fmaxf(top, fabsf(s.at(i))), fabsf(s.at(i + 1)));
    return sv_scale(__reduce_max_sync(0xffffffffu, __float_as_uint(top)), inv);
}

template <typename T, int D>
__global__ void __launch_bounds__(128, 2) sv_k_attn_few(const __grid_constant__ SvAttn a) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int KS = D / 16, VG = D / 64;   // steps of the first product; groups of 64 channels
    __shared__ uint4 s_q[2][KS][32];          // the queries' fragments
    __shared__ float s_qinv[SV_FEW_ROWS], s_m[4][SV_FEW_ROWS], s_l[4][SV_FEW_ROWS], s_o[4][SV_FEW_ROWS][D + 4];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, c = lane & 3, n8 = lane >> 2;
    const int si = sv_find(a, blockIdx.x), split = blockIdx.x - a.seq[si].unit0, g = blockIdx.y;
    const SvSeq &s = a.seq[si];
    const int rows = s.n_tok * a.R, rp = sv_rp(rows), past = s.n_kv - s.n_tok;
    const int j_begin = split * a.tps * SV_TILE, j_end = min(s.n_kv, j_begin + a.tps * SV_TILE);
    const int64_t kvd = (int64_t)a.G * D;
    const T *kc = static_cast<const T *>(s.k) + (int64_t)g * D + 8 * c, *vc = static_cast<const T *>(s.v) + ((int64_t)g * D + n8) * s.n_ctx + 4 * c;
    SvShare<T, D / 4> ka, kb;                 // K rows of two times eight slots
    SvShare<T, 32> va[VG];                    // V of 64 channels each.  (Head size 128: K's two and V's two take turns in the same registers)
    // column n of score tile t is slot 4 (n / 2) + 2 t + n % 2: a thread's two columns of both tiles are slots 4 c .. 4 c + 3
    auto live_of = [&](int j) -> uint32_t { // (of sixteen slots)
        const int k = j + (lane & 15);
        return __ballot_sync(0xffffffffu, k < j_end && !(s.hidden && s.hidden[k])) & 0xffffu;
    };
    auto load_k = [&](SvShare<T, D / 4> &r, int j, int t, uint32_t live) {
        const int slot = 4 * (n8 >> 1) + 2 * t + (n8 & 1);
        const bool in = live >> slot & 1;
#pragma unroll
        for (int i = 0; i < D / 32; i++) {
            if (in) sv_read_at<8>(r, 8 * i, kc + (int64_t)(j + slot) * kvd + 32 * i, s.k_mode, 0xffu);
            else
#pragma unroll
                for (int e = 0; e < 8; e++) r.keep(8 * i + e, false);
        }
    };
    auto load_v = [&](SvShare<T, 32> &r, int j, int v, uint32_t live) {
        const uint32_t in = live >> (4 * c) & 0xfu;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (in) sv_read_at<4>(r, 4 * i, vc + (int64_t)(64 * v + 8 * i) * s.n_ctx + j, s.v_mode, in);
            if (in != 0xfu)
#pragma unroll
                for (int e = 0; e < 4; e++) r.keep(4 * i + e, in >> e & 1);
        }
    };
    int j = j_begin + 16 * warp;
    uint32_t live = live_of(j);
    load_k(ka, j, 0, live);
    load_k(kb, j, 1, live);
    // queries: a warp takes four rows' scales, then every thread its fragments
    for (int r = 4 * warp; r < 4 * warp + 4; r++) {
        float top = 0.f;
        if (r < rows)
            for (int d = lane; d < D; d += 32) top = fmaxf(top, fabsf(a.q[((int64_t)(s.tok0 + r / a.R) * a.n_heads + g * a.R + r % a.R) * D + d] * a.scale));
        float inv;
        sv_scale(__reduce_max_sync(0xffffffffu, __float_as_uint(top)), inv);
        if (lane == 0) s_qinv[r] = inv;
    }
    __syncthreads();
    for (int i = tid; i < KS * 32; i += 128) {
        const int ks = i >> 5, l = i & 31, d = 32 * (ks >> 1) + 8 * (l & 3) + 4 * (ks & 1);
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; e++) { // row, row + 8, then the next two elements of both
            const int r = (l >> 2) + 8 * (e & 1);
            float x0 = 0.f, x1 = 0.f;
            if (r < rows) {
                const float *q = a.q + ((int64_t)(s.tok0 + r / a.R) * a.n_heads + g * a.R + r % a.R) * D + d + (e & 2);
                const float f = 1.f / s_qinv[r]; // (a power of two)
                x0 = q[0] * a.scale * f;
                x1 = q[1] * a.scale * f;
            }
            sv_cut(x0, x1, hi[e], lo[e]);
        }
        s_q[0][ks][l] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        s_q[1][ks][l] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
    __syncthreads();
    const float qinv0 = s_qinv[n8], qinv1 = s_qinv[n8 + 8];
    float o[D / 8][4], m0 = SV_NONE, m1 = SV_NONE, l0 = 0.f, l1 = 0.f;
#pragma unroll
    for (int i = 0; i < D / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

    auto scores = [&](const SvShare<T, D / 4> &r, float (&z)[4]) {
        float inv;
        const float f = sv_group_scale(r, inv);
        float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            uint32_t h0, h1, x0, x1;
            const int i = 8 * (ks >> 1) + 4 * (ks & 1);
            sv_cut(r.at(i) * f, r.at(i + 1) * f, h0, x0);
            sv_cut(r.at(i + 2) * f, r.at(i + 3) * f, h1, x1);
            const uint4 qh = s_q[0][ks][lane], ql = s_q[1][ks][lane];
            sv_mma(d, ql, h0, h1);
            if (F32) sv_mma(d, qh, x0, x1);
            sv_mma(d, qh, h0, h1);
        }
        const float f0 = qinv0 * inv, f1 = qinv1 * inv;
        z[0] = d[0] * f0; z[1] = d[1] * f0; z[2] = d[2] * f1; z[3] = d[3] * f1;
    };
    auto output = [&](const SvShare<T, 32> &r, int v, const uint4 &ph, const uint4 &pl, float f0, float f1) {
        float inv;
        const float f = sv_group_scale(r, inv);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            uint32_t h0, h1, x0, x1;
            sv_cut(r.at(4 * i) * f, r.at(4 * i + 1) * f, h0, x0);
            sv_cut(r.at(4 * i + 2) * f, r.at(4 * i + 3) * f, h1, x1);
            float d[4] = {0.f, 0.f, 0.f, 0.f};
            sv_mma(d, pl, h0, h1);
            if (F32) sv_mma(d, ph, x0, x1);
            sv_mma(d, ph, h0, h1);
            float (&to)[4] = o[8 * v + i];
            to[0] = fmaf(to[0], f0, d[0] * inv); to[1] = fmaf(to[1], f0, d[1] * inv);
            to[2] = fmaf(to[2], f1, d[2] * inv); to[3] = fmaf(to[3], f1, d[3] * inv);
        }
    };

    for (; j < j_end; j += 64) {
        const int next = j + 64;
        float z[2][4];
        scores(ka, z[0]);
        load_v(va[0], j, 0, live);
        scores(kb, z[1]);
        if (VG == 2) load_v(va[VG - 1], j, 1, live);
        const uint32_t next_live = next < j_end ? live_of(next) : 0u;
        // which of its four slots the thread's rows see
        uint32_t see0 = live >> (4 * c) & 0xfu, see1 = see0;
        if (j + 16 > past)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int back = j + 4 * c + e - past;
                if (back >= 0 && back < s.n_tok) {
                    if (n8 < rows && !sv_sees(s, n8 / a.R, back)) see0 &= ~(1u << e);
                    if (n8 + 8 < rows && !sv_sees(s, (n8 + 8) / a.R, back)) see1 &= ~(1u << e);
                }
            }
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                if (!(see0 >> (2 * t + e) & 1)) z[t][e] = SV_NONE;
                if (!(see1 >> (2 * t + e) & 1)) z[t][2 + e] = SV_NONE;
            }
        if (s.scores) {
            float4 *to = reinterpret_cast<float4 *>(s.scores) + ((int64_t)g * sv_quads(s.n_kv) + j / 4 + c) * rp;
            if (n8 < rows) to[n8] = make_float4(z[0][0], z[0][1], z[1][0], z[1][1]);
            if (n8 + 8 < rows) to[n8 + 8] = make_float4(z[0][2], z[0][3], z[1][2], z[1][3]);
        }
        float t0 = fmaxf(fmaxf(z[0][0], z[0][1]), fmaxf(z[1][0], z[1][1])), t1 = fmaxf(fmaxf(z[0][2], z[0][3]), fmaxf(z[1][2], z[1][3]));
        t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 1)); t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 2));
        t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 1)); t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 2));
        t0 = fmaxf(t0, m0);
        t1 = fmaxf(t1, m1);
        const float r0 = t0 == SV_NONE ? 0.f : t0, r1 = t1 == SV_NONE ? 0.f : t1, f0 = sv_ex2(m0 - r0), f1 = sv_ex2(m1 - r1);
        m0 = t0;
        m1 = t1;
        // 2^15 p, and so its sum (the thread's; the four threads of a row are joined at the end)
        float p[2][4];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            p[t][0] = sv_ex2(z[t][0] + (15.f - r0)); p[t][1] = sv_ex2(z[t][1] + (15.f - r0));
            p[t][2] = sv_ex2(z[t][2] + (15.f - r1)); p[t][3] = sv_ex2(z[t][3] + (15.f - r1));
        }
        l0 = fmaf(l0, f0, (p[0][0] + p[0][1]) + (p[1][0] + p[1][1]));
        l1 = fmaf(l1, f1, (p[0][2] + p[0][3]) + (p[1][2] + p[1][3]));
        uint4 ph, pl;
        sv_cut(p[0][0], p[0][1], ph.x, pl.x);
        sv_cut(p[0][2], p[0][3], ph.y, pl.y);
        sv_cut(p[1][0], p[1][1], ph.z, pl.z);
        sv_cut(p[1][2], p[1][3], ph.w, pl.w);
        output(va[0], 0, ph, pl, f0, f1);
        live = next_live;
        if (next < j_end) load_k(ka, next, 0, live);
        if (VG == 2) output(va[VG - 1], VG - 1, ph, pl, f0, f1);
        if (next < j_end) load_k(kb, next, 1, live);
    }
    // the warps' parts
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1); l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1); l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    if (c == 0) {
        s_m[warp][n8] = m0; s_m[warp][n8 + 8] = m1;
        s_l[warp][n8] = l0; s_l[warp][n8 + 8] = l1;
    }
#pragma unroll
    for (int i = 0; i < D / 8; i++) {
        *reinterpret_cast<float2 *>(&s_o[warp][n8][8 * i + 2 * c]) = make_float2(o[i][0], o[i][1]);
        *reinterpret_cast<float2 *>(&s_o[warp][n8 + 8][8 * i + 2 * c]) = make_float2(o[i][2], o[i][3]);
    }
    __syncthreads();
    float2 *ml = reinterpret_cast<float2 *>(s.part + (int64_t)s.splits * a.G * rows * D);
    for (int i = tid; i < rows * D; i += 128) {
        const int r = i / D, d = i % D;
        float m = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r])), l = 0.f, v = 0.f;
        const float ref = m == SV_NONE ? 0.f : m;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float f = sv_ex2(s_m[w][r] - ref);
            l = fmaf(s_l[w][r], f, l);
            v = fmaf(s_o[w][r][d], f, v);
        }
        if (d == 0) ml[((int64_t)split * a.G + g) * rows + r] = make_float2(m, l * (1.f / 32768.f));
        if (s.splits == 1) a.out[((int64_t)(s.tok0 + r / a.R) * a.n_heads + g * a.R + r % a.R) * D + d] = l > 0.f ? v / l : 0.f;
        else s.part[(((int64_t)split * a.G + g) * rows + r) * D + d] = v * (1.f / 32768.f);
    }
}
