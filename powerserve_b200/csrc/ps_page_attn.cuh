// ps_page_attn.cuh - attention of a step's tokens over caches in 8 bits and in pages.
//
//   z[t][h][j] = scale q[t][h] . k[j][g(h)],   p = soft-max over the slots j that token t sees,   out[t][h] = sum_j p[t][h][j] v[g(h)][j]
#pragma once
#include "ps_page.cuh"

struct PgAttnSeq {
    const int32_t *table;
    const uint8_t *hidden, *mask;
    int n_kv, n_tok, tok0, unit0;
};
struct PgAttn {
    PgAttnSeq seq[PG_SEQS];
    PgPool pool;
    const void *q;
    void *out;
    int n_seqs, n_heads, R;
    float scale; // times log2 e
};
PS_D bool pg_sees(const PgAttnSeq &s, int t, int back) { return back < 0 || (s.mask ? s.mask[t * s.n_tok + back] != 0 : back <= t); }

// right and simple: sixteen query rows, 32 slots at a time, everything in 32 bits on the CUDA cores
template <typename T>
__global__ void __launch_bounds__(128) pg_k_attn(const __grid_constant__ PgAttn a) {
    extern __shared__ float pg_sm[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, hs = a.pool.hs, g = blockIdx.y;
    const PgAttnSeq &s = a.seq[blockIdx.x];
    const int rows = s.n_tok * a.R, r0 = blockIdx.z * 16, B = a.pool.P / PG_BLOCK;
    if (r0 >= rows) return;
    const int kp = hs + 1;
    float *sq = pg_sm, *sk = sq + 16 * hs, *sv = sk + 32 * kp, *sp = sv + hs * 33, *sc = sp + 16 * 33;
    const T *q = static_cast<const T *>(a.q);
    T *out = static_cast<T *>(a.out);
    for (int i = tid; i < 16 * hs; i += 128) {
        const int r = r0 + i / hs, t = r / a.R, h = g * a.R + r % a.R;
        sq[i] = r < rows ? pg_num(q[((int64_t)(s.tok0 + t) * a.n_heads + h) * hs + i % hs]) * a.scale : 0.f;
    }
    float acc[2][16], m[4], l[4];
#pragma unroll
    for (int r = 0; r < 16; r++) acc[0][r] = acc[1][r] = 0.f;
#pragma unroll
    for (int r = 0; r < 4; r++) { m[r] = -INFINITY; l[r] = 0.f; }
    const int past = s.n_kv - s.n_tok;
    for (int j0 = 0; j0 < s.n_kv; j0 += 32) {
        __syncthreads();
        for (int i = tid; i < 2 * 32 * hs; i += 128) {
            const int kv = i / (32 * hs), e = i % (32 * hs), j = j0 + (kv ? e & 31 : e / hs), d = kv ? e >> 5 : e % hs;
            float x = 0.f;
            if (j < s.n_kv && !(s.hidden && s.hidden[j])) {
                const int page = s.table[j >> a.pool.shift], o = j & (a.pool.P - 1);
                if (a.pool.has(page)) {
                    const int64_t at = a.pool.at(page, g, kv);
                    x = (float)a.pool.codes[at * a.pool.page_codes() + (kv ? ((int64_t)(o / 16) * hs + d) * 16 + o % 16 : ((int64_t)(o / 8) * (hs / 16) + d / 16) * 128 + (o % 8) * 16 + d % 16)] *
                        a.pool.scales[at * B + o / PG_BLOCK];
                }
            }
            if (kv) sv[d * 33 + (j - j0)] = x;
            else sk[(j - j0) * kp + d] = x;
        }
        __syncthreads();
        const int j = j0 + lane;
        const bool in = j < s.n_kv && !(s.hidden && s.hidden[j]) && a.pool.has(s.table[j >> a.pool.shift]);
        float z[4] = {0.f, 0.f, 0.f, 0.f};
        for (int d = 0; d < hs; d++) {
            const float kv = sk[lane * kp + d];
#pragma unroll
            for (int r = 0; r < 4; r++) z[r] = fmaf(sq[(warp * 4 + r) * hs + d], kv, z[r]);
        }
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int row = r0 + warp * 4 + r;
            if (!in || row >= rows || !pg_sees(s, row / a.R, j - past)) z[r] = -INFINITY;
            float mx = z[r];
#pragma unroll
            for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float mn = fmaxf(m[r], mx), ref = mn == -INFINITY ? 0.f : mn, f = exp2f(m[r] - ref), p = exp2f(z[r] - ref);
            float sum = p;
#pragma unroll
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            l[r] = l[r] * f + sum;
            m[r] = mn;
            sp[(warp * 4 + r) * 33 + lane] = p;
            if (lane == 0) sc[warp * 4 + r] = f;
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const int d = tid + 128 * c;
            if (d >= hs) break;
#pragma unroll
            for (int r = 0; r < 16; r++) acc[c][r] *= sc[r];
            for (int jj = 0; jj < 32; jj++) {
                const float v = sv[d * 33 + jj];
#pragma unroll
                for (int r = 0; r < 16; r++) acc[c][r] = fmaf(sp[r * 33 + jj], v, acc[c][r]);
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 4; r++)
        if (lane == 0) sc[warp * 4 + r] = l[r] == 0.f ? 0.f : 1.f / l[r];
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 2; c++) {
        const int d = tid + 128 * c;
        if (d >= hs) break;
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const int row = r0 + r;
            if (row >= rows) break;
            out[((int64_t)(s.tok0 + row / a.R) * a.n_heads + g * a.R + row % a.R) * hs + d] = pg_to<T>(acc[c][r] * sc[r]);
        }
    }
}
inline size_t pg_attn_smem(int hs) { return 4 * ((size_t)16 * hs + 32 * (hs + 1) + (size_t)hs * 33 + 16 * 33 + 16); }
