// ps_serve_attn_few.cuh - ps_serve_attn.cuh's attention for head sizes 64 and 128 and up to eight query rows of a kv head (a token of each sequence): the products are as in
// ps_serve_attn_tc.cuh - fp16 parts, three MMAs for one of 32 bits - but by mma.sync on fragments that come straight from memory, without shared memory
// or barriers on the way.  With so few rows the tensor cores have little to do, and what counts is bytes under way: a warp works alone on sixteen slots at a time,
// four warps a CTA, three CTAs an SM, each warp with 8 KB of K and V on the way while it computes.
// The cache is the MMAs' 16-row side, the queries are the eight columns: S^T = K Q^T, O^T = V^T P^T.  Which element of a row a thread holds is free (a sum's order is), so
// a thread takes neighbours: of K eight elements of a slot's row, of V four slots of a channel; row m of a score tile is slot 4 (m % 8 / 2) + m % 2 + 2 (m / 8) so that
// those four slots are its columns in the second product.  The weights change places by movmatrix.
// A group's sum (sixteen slots of 64 channels) is added up in 32 bits outside the MMAs, after a factor of its own.  The MMAs' accumulators truncate: the scores' small products have one of their own,
// those of the outputs come first, while their accumulator, which starts from zero for every sixteen slots, is small.
// Bound by loads under way: 128 to 168 registers a thread hold them, and the tail of a launch by its last CTAs. Eight kv heads of 128, four heads each, float32: 8 sequences of 16 000 slots
// 215 us = 4.9 TB/s, 64 of 2 041 234 us = 4.6, 64 of 256 to 2 041 118 us = 3.7; heads of 64: 5.2 TB/s; bfloat16 3.2 (the same instructions for half the bytes). The kernel for 128 rows
// took 194 us where this one takes 118. Few splits are a cluster that joins them: one sequence of 1 000 slots 18.5 us, 20.5 with a launch to join.
#pragma once
#include "ps_serve_attn_tc.cuh"

#define SV_FEW_ROWS 8

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
// a thread's share of a group
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

PS_D uint32_t sv_turn(uint32_t x) { // an 8 x 8 matrix of halves, transposed
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// CL: a sequence's splits are a cluster (that code in one kernel with the other: 64 sessions 125 -> 129 us)
template <typename T, int D, bool CL>
__global__ void __launch_bounds__(128, sizeof(T) == 4 && D == 128 ? 3 : 4) sv_k_attn_few(const __grid_constant__ SvAttn a) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int KS = D / 16, HALF = D / 64; // steps of the first product; items of 64 channels
    __shared__ uint4 s_q[KS][32];             // the queries' fragments: hi, hi, lo, lo
    __shared__ float s_top[SV_FEW_ROWS], s_sum[SV_FEW_ROWS]; // the CTA's rows, for its cluster
    __shared__ float s_qinv[SV_FEW_ROWS], s_m[4][SV_FEW_ROWS], s_l[4][SV_FEW_ROWS];
    __shared__ __align__(16) float s_o[4][SV_FEW_ROWS][D + 4];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, c = lane & 3, n8 = lane >> 2;
    const int si = sv_find(a, blockIdx.x), split = blockIdx.x - a.seq[si].unit0, g = blockIdx.y;
    const SvSeq &s = a.seq[si];
    const int rows = s.n_tok * a.R, rp = sv_rp(rows), past = s.n_kv - s.n_tok;
    const int j_begin = split * a.tps * SV_TILE, j_end = min(s.n_kv, j_begin + a.tps * SV_TILE);
    const int64_t kvd = (int64_t)a.G * D;
    const int slot0 = 4 * (n8 >> 1) + (n8 & 1);   // the thread's score rows: this slot and the one two further on
    const T *kc = static_cast<const T *>(s.k) + (int64_t)g * D + 8 * c + slot0 * kvd, *vc = static_cast<const T *>(s.v) + ((int64_t)g * D + n8) * s.n_ctx + 4 * c;
    SvShare<T, 32> x, y;                          // two items under way: K's halves, then V's (head size 64: K, then V)
    auto live_of = [&](int j) -> uint32_t { // (of sixteen slots)
        const int k = j + (lane & 15);
        return __ballot_sync(0xffffffffu, k < j_end && !(s.hidden && s.hidden[k])) & 0xffffu;
    };
    auto load_k = [&](SvShare<T, 32> &r, int j, int half, uint32_t live) {
#pragma unroll
        for (int i = 0; i < 4; i++) { // (slot, 32 channels)
            const bool in = live >> (slot0 + (i & 2)) & 1;
            if (in) sv_read_at<8>(r, 8 * i, kc + (int64_t)(j + (i & 2)) * kvd + 64 * half + 32 * (i & 1), s.k_mode, 0xffu);
            else
#pragma unroll
                for (int e = 0; e < 8; e++) r.keep(8 * i + e, false);
        }
    };
    auto load_v = [&](SvShare<T, 32> &r, int j, int half, uint32_t live) {
        const uint32_t in = live >> (4 * c) & 0xfu;
        const T *p = vc + (int64_t)(64 * half) * s.n_ctx + j;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (in) sv_read_at<4>(r, 4 * i, p + (int64_t)(8 * i) * s.n_ctx, s.v_mode, in);
            if (in != 0xfu)
#pragma unroll
                for (int e = 0; e < 4; e++) r.keep(4 * i + e, in >> e & 1);
        }
    };
    int j = j_begin + 16 * warp;
    uint32_t live = live_of(j);
    load_k(x, j, 0, live);
    if (HALF == 2) load_k(y, j, 1, live);
    // queries: a warp takes two rows' scales, then every thread its fragments
    for (int r = 2 * warp; r < 2 * warp + 2; r++) {
        float top = 0.f;
        if (r < rows)
            for (int d = lane; d < D; d += 32) top = fmaxf(top, fabsf(a.q[((int64_t)(s.tok0 + r / a.R) * a.n_heads + g * a.R + r % a.R) * D + d] * a.scale));
        float inv;
        sv_scale(__reduce_max_sync(0xffffffffu, __float_as_uint(top)), inv);
        if (lane == 0) s_qinv[r] = inv;
    }
    __syncthreads();
    for (int i = tid; i < KS * 32; i += 128) {
        const int ks = i >> 5, l = i & 31, r = l >> 2, d = 32 * (ks >> 1) + 8 * (l & 3) + 4 * (ks & 1);
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (r < rows) {
            const float *q = a.q + ((int64_t)(s.tok0 + r / a.R) * a.n_heads + g * a.R + r % a.R) * D + d;
            const float f = 1.f / s_qinv[r]; // (a power of two)
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = q[e] * a.scale * f;
        }
        uint4 w;
        sv_cut(v[0], v[1], w.x, w.z);
        sv_cut(v[2], v[3], w.y, w.w);
        s_q[ks][l] = w;
    }
    __syncthreads();
    const float qinv0 = s_qinv[2 * c], qinv1 = s_qinv[2 * c + 1];
    const int row0 = 2 * c, row1 = 2 * c + 1;
    float o[D / 16][4], m0 = SV_NONE, m1 = SV_NONE, l0 = 0.f, l1 = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

    auto scores = [&](const SvShare<T, 32> &r, int half, float (&z)[4]) {
        float inv;
        const float f = sv_group_scale(r, inv);
        float d[4] = {0.f, 0.f, 0.f, 0.f}, low[4] = {0.f, 0.f, 0.f, 0.f}; // (the accumulators truncate: small products have one of their own)
#pragma unroll
        for (int k = 0; k < 4; k++) { // 32-channel group, half of it
            uint4 hi, lo;
            const int i = 8 * (k >> 1) + 4 * (k & 1);
            sv_cut(r.at(i) * f, r.at(i + 1) * f, hi.x, lo.x);
            sv_cut(r.at(16 + i) * f, r.at(17 + i) * f, hi.y, lo.y);
            sv_cut(r.at(i + 2) * f, r.at(i + 3) * f, hi.z, lo.z);
            sv_cut(r.at(18 + i) * f, r.at(19 + i) * f, hi.w, lo.w);
            const uint4 q = s_q[4 * half + k][lane];
            sv_mma(low, hi, q.z, q.w);
            if (F32) sv_mma(low, lo, q.x, q.y);
            sv_mma(d, hi, q.x, q.y);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) z[e] = half ? fmaf(d[e] + low[e], inv, z[e]) : (d[e] + low[e]) * inv;
    };
    auto output = [&](const SvShare<T, 32> &r, int half, uint32_t ph0, uint32_t ph1, uint32_t pl0, uint32_t pl1) {
        float inv;
        const float f = sv_group_scale(r, inv);
#pragma unroll
        for (int i = 0; i < 4; i++) { // sixteen channels
            uint4 hi, lo;
            sv_cut(r.at(8 * i) * f, r.at(8 * i + 1) * f, hi.x, lo.x);
            sv_cut(r.at(8 * i + 4) * f, r.at(8 * i + 5) * f, hi.y, lo.y);
            sv_cut(r.at(8 * i + 2) * f, r.at(8 * i + 3) * f, hi.z, lo.z);
            sv_cut(r.at(8 * i + 6) * f, r.at(8 * i + 7) * f, hi.w, lo.w);
            float d[4] = {0.f, 0.f, 0.f, 0.f};
            sv_mma(d, hi, pl0, pl1);
            if (F32) sv_mma(d, lo, ph0, ph1);
            sv_mma(d, hi, ph0, ph1);
            float (&to)[4] = o[4 * half + i];
#pragma unroll
            for (int e = 0; e < 4; e++) to[e] = fmaf(d[e], inv, to[e]);
        }
    };

    for (; j < j_end; j += 64) {
        const int next = j + 64;
        float z[4];
        scores(x, 0, z);
        load_v(x, j, 0, live);
        if (HALF == 2) {
            scores(y, 1, z);
            load_v(y, j, 1, live);
        }
        const uint32_t next_live = next < j_end ? live_of(next) : 0u;
        if (HALF == 1 && next < j_end) load_k(y, next, 0, next_live);
        // which of its two slots the thread's two rows see
        uint32_t see = (live >> slot0 & 1) * 3u | (live >> (slot0 + 2) & 1) * 12u;
        if (j + 16 > past)
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int back = j + slot0 + 2 * t - past;
                if (back >= 0 && back < s.n_tok) {
                    if (row0 < rows && !sv_sees(s, row0 / a.R, back)) see &= ~(1u << (2 * t));
                    if (row1 < rows && !sv_sees(s, row1 / a.R, back)) see &= ~(2u << (2 * t));
                }
            }
#pragma unroll
        for (int e = 0; e < 4; e++) z[e] = see >> e & 1 ? z[e] * (e & 1 ? qinv1 : qinv0) : SV_NONE;
        if (s.scores) {
            float *to = s.scores + ((((int64_t)g * sv_quads(s.n_kv) + j / 4 + (n8 >> 1)) * rp) * 4) + (n8 & 1);
            if (row0 < rows) { to[row0 * 4] = z[0]; to[row0 * 4 + 2] = z[2]; }
            if (row1 < rows) { to[row1 * 4] = z[1]; to[row1 * 4 + 2] = z[3]; }
        }
        float t0 = fmaxf(z[0], z[2]), t1 = fmaxf(z[1], z[3]);
#pragma unroll
        for (int i = 4; i < 32; i *= 2) {
            t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, i));
            t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, i));
        }
        t0 = fmaxf(t0, m0);
        t1 = fmaxf(t1, m1);
        const float r0 = t0 == SV_NONE ? 0.f : t0, r1 = t1 == SV_NONE ? 0.f : t1, f0 = sv_ex2(m0 - r0), f1 = sv_ex2(m1 - r1);
        m0 = t0;
        m1 = t1;
        // 2^15 p, and so its sum (the thread's; those of a row are joined at the end).  The factor comes after: 15 in the exponent would cost the large weights four bits
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; e++) p[e] = sv_ex2(z[e] - (e & 1 ? r1 : r0)) * 32768.f;
        l0 = fmaf(l0, f0, p[0] + p[2]);
        l1 = fmaf(l1, f1, p[1] + p[3]);
        uint32_t ph0, pl0, ph1, pl1;
        sv_cut(p[0], p[1], ph0, pl0);
        sv_cut(p[2], p[3], ph1, pl1);
        ph0 = sv_turn(ph0); pl0 = sv_turn(pl0); ph1 = sv_turn(ph1); pl1 = sv_turn(pl1);
        if (__any_sync(0xffffffffu, f0 != 1.f || f1 != 1.f))
#pragma unroll
            for (int i = 0; i < D / 16; i++) { o[i][0] *= f0; o[i][1] *= f1; o[i][2] *= f0; o[i][3] *= f1; }
        output(x, 0, ph0, ph1, pl0, pl1);
        live = next_live;
        if (HALF == 2) {
            if (next < j_end) load_k(x, next, 0, live);
            output(y, 1, ph0, ph1, pl0, pl1);
            if (next < j_end) load_k(y, next, 1, live);
        } else x = y;
    }
    // the warps' parts
#pragma unroll
    for (int i = 4; i < 32; i *= 2) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, i);
        l1 += __shfl_xor_sync(0xffffffffu, l1, i);
    }
    if (n8 == 0) {
        s_m[warp][row0] = m0; s_m[warp][row1] = m1;
        s_l[warp][row0] = l0; s_l[warp][row1] = l1;
    }
#pragma unroll
    for (int i = 0; i < D / 16; i++) {
        s_o[warp][row0][16 * i + n8] = o[i][0]; s_o[warp][row1][16 * i + n8] = o[i][1];
        s_o[warp][row0][16 * i + 8 + n8] = o[i][2]; s_o[warp][row1][16 * i + 8 + n8] = o[i][3];
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
        if (CL) { // (who writes an element of s_o[0] is the only one that reads it)
            s_o[0][r][d] = v;
            if (d == 0) { s_top[r] = m; s_sum[r] = l; }
            continue;
        }
        if (d == 0) {
            if (s.splits == 1) sv_put_lse(s, (int64_t)g * rows + r, m, l * (1.f / 32768.f));
            else ml[((int64_t)split * a.G + g) * rows + r] = make_float2(m, l * (1.f / 32768.f));
        }
        if (s.splits == 1) a.out[((int64_t)(s.tok0 + r / a.R) * a.n_heads + g * a.R + r % a.R) * D + d] = l == 0.f ? 0.f : v / l; // (a sum that is no number: so is the row)
        else s.part[(((int64_t)split * a.G + g) * rows + r) * D + d] = v * (1.f / 32768.f);
    }
    if (CL) sv_join_cluster<D>(a, s, g, 0, rows, rows, &s_o[0][0][0], D + 4, s_top, s_sum);
}
