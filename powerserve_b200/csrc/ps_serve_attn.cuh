// ps_serve_attn.cuh - attention of a step's tokens over the caches of several sequences.
//
//   z[t][h][j] = scale q[t][h] . k[j][g(h)],   p = soft-max over the slots j that token t sees,   out[t][h] = sum_j p[t][h][j] v[g(h)][j]
//   weight[g][j] += sum over tokens t and heads h of g of p[t][h][j]
//
// A sequence's query rows of one kv head (n_tok tokens x the heads that share it) go together, so that its K rows and V^T columns are read once.
// The slots are cut into splits; a split leaves its rows' running maximum, sum and unnormalised output in the workspace, and sv_k_join joins
// them.  Where weights are gathered, the scores (32 bits) go to the workspace too, and sv_k_weights sums exp(z - log-sum) over the rows.
#pragma once
#include "ps_ptx.cuh"

#include <cooperative_groups.h>
#include <cuda_bf16.h>

#define SV_SEQS 64      // sequences of a launch: their table is a kernel parameter
#define SV_TILE 64      // slots of a tile
#define SV_LOG2E 1.4426950408889634f
#define SV_NONE (-INFINITY)

struct SvSeq {
    const void *k, *v;
    float *weight;
    const uint8_t *hidden, *mask;
    float *scores;          // [kv head][quad of slots][rp][4], or null: quads up to a whole tile, -inf where a row does not see the slot
    float *part;            // [split][kv head][row][hs]; then [split][kv head][row] pairs of maximum and sum
    float *lse;             // [kv head][row] log2 of the row's sum, for the weights; or null
    int n_ctx, n_kv, n_tok, tok0;
    int k_mode, v_mode;     // head sizes 64 and 128: rows begin at 16-byte boundaries
    int splits, unit0;      // unit0: number of the sequence's first split among all of the launch
};
struct SvAttn {
    SvSeq seq[SV_SEQS];
    const float *q;
    float *out;
    int n_seqs, hs, n_heads, G, R, tps; // R: heads that share a kv head; tps: tiles of a split
    int cluster;                        // above 1: every sequence has as many splits, and they are a cluster's CTAs
    int q_vec, out_vec;                 // aligned to 16 bytes
    float scale;                        // times log2 e
    int *err;
};

PS_D float sv_ld(const float *p, int64_t i) { return p[i]; }
PS_D float sv_ld(const __nv_bfloat16 *p, int64_t i) { return __bfloat162float(p[i]); }
PS_D float sv_ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
PS_HD int sv_rp(int rows) { return (rows + 3) & ~3; }
PS_HD int64_t sv_quads(int n_kv) { return (int64_t)((n_kv + SV_TILE - 1) / SV_TILE) * (SV_TILE / 4); }
PS_D int sv_find(const SvAttn &a, int unit) {
    int s = 0;
    while (s + 1 < a.n_seqs && unit >= a.seq[s + 1].unit0) s++;
    return s;
}
// slot j, token t: back = j - (n_kv - n_tok) is the slot's number among the step's own tokens (negative: the past)
PS_D bool sv_sees(const SvSeq &s, int t, int back) { return back < 0 || (s.mask ? s.mask[t * s.n_tok + back] != 0 : back <= t); }

PS_D void sv_put_lse(const SvSeq &s, int64_t at, float top, float sum) { // (a row that sees nothing adds nothing)
    if (s.lse) s.lse[at] = sum > 0.f ? top + log2f(sum) : INFINITY;
}
// The splits of a sequence are a cluster: each CTA's rows r0 .. r0 + rows of `all` lie unnormalised in its shared memory (o: ld floats a row), 2^15 times their maxima's reference as everywhere;
// the CTAs take shares of the elements and read them from one another
template <int D> PS_D void sv_join_cluster(const SvAttn &a, const SvSeq &s, int g, int r0, int rows, int all, float *o, int ld, float *top, float *sum) {
    cooperative_groups::cluster_group cl = cooperative_groups::this_cluster();
    cl.sync();
    const int C = a.cluster;
    for (int i = cl.block_rank() * blockDim.x + threadIdx.x; i < rows * (D / 4); i += C * blockDim.x) {
        const int r = i / (D / 4), d = i % (D / 4) * 4, row = r0 + r;
        float t[8], m = SV_NONE, l = 0.f;
        float4 x[8], v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int c = 0; c < 8; c++) {
            t[c] = SV_NONE;
            if (c < C) {
                t[c] = cl.map_shared_rank(top, c)[r];
                x[c] = *reinterpret_cast<const float4 *>(cl.map_shared_rank(o, c) + r * ld + d);
            }
            m = fmaxf(m, t[c]);
        }
        const float ref = m == SV_NONE ? 0.f : m;
#pragma unroll
        for (int c = 0; c < 8; c++)
            if (c < C) {
                const float f = sv_ex2(t[c] - ref);
                l = fmaf(cl.map_shared_rank(sum, c)[r], f, l);
                v.x = fmaf(x[c].x, f, v.x); v.y = fmaf(x[c].y, f, v.y); v.z = fmaf(x[c].z, f, v.z); v.w = fmaf(x[c].w, f, v.w);
            }
        if (d == 0) sv_put_lse(s, (int64_t)g * all + row, m, l * (1.f / 32768.f));
        const float inv = l > 0.f ? 1.f / l : 0.f;
        float *to = a.out + ((int64_t)(s.tok0 + row / a.R) * a.n_heads + g * a.R + row % a.R) * D + d;
        if (a.out_vec) *reinterpret_cast<float4 *>(to) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
        else { to[0] = v.x * inv; to[1] = v.y * inv; to[2] = v.z * inv; to[3] = v.w * inv; }
    }
    cl.sync(); // (nobody leaves while its rows are read)
}

// ---------------------------------------------------------------------------------------------------- any head size
// For head sizes that are not 64 or 128, right and simple: scalar products, element by element. Bound by instructions (a load and a division for every element, no more than a CTA's own tile under way): 64 sequences of
// 2 041 slots, a token each, 8 kv heads, four heads each, float32: of 32 746 us = 0.36 TB/s, of 96 1 870, of 160 3 100, of 256 9 170 us (heads of 64 and 128 in kernels of their own: 103 and 232).  Sixteen query rows, 32 slots at a time, everything in 32-bit arithmetic on the CUDA cores.  Thread (slot, row group) takes four scores; a warp
// takes the soft-max of four rows; then a thread owns channels d, d + 128 of all sixteen rows.
template <typename T>
__global__ void __launch_bounds__(128) sv_k_attn(const __grid_constant__ SvAttn a) {
    extern __shared__ float sv_sm[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, hs = a.hs;
    const int si = sv_find(a, blockIdx.x), split = blockIdx.x - a.seq[si].unit0, g = blockIdx.y;
    const SvSeq &s = a.seq[si];
    const int rows = s.n_tok * a.R, r0 = blockIdx.z * 16;
    if (r0 >= rows) return;
    const int kp = hs + 1;
    float *sq = sv_sm, *sk = sq + 16 * hs, *sv = sk + 32 * kp, *sp = sv + hs * 33, *sc = sp + 16 * 33;
    const T *kc = static_cast<const T *>(s.k) + (int64_t)g * hs, *vc = static_cast<const T *>(s.v) + (int64_t)g * hs * s.n_ctx;
    const int64_t kvd = (int64_t)a.G * hs;
    for (int i = tid; i < 16 * hs; i += 128) {
        const int r = r0 + i / hs, t = r / a.R, h = g * a.R + r % a.R;
        sq[i] = r < rows ? a.q[((int64_t)(s.tok0 + t) * a.n_heads + h) * hs + i % hs] * a.scale : 0.f;
    }
    float acc[2][16], m[4], l[4];
#pragma unroll
    for (int r = 0; r < 16; r++) acc[0][r] = acc[1][r] = 0.f;
#pragma unroll
    for (int r = 0; r < 4; r++) { m[r] = SV_NONE; l[r] = 0.f; }
    const int j_end = min(s.n_kv, (split + 1) * a.tps * SV_TILE), past = s.n_kv - s.n_tok, rp = sv_rp(rows);
    for (int j0 = split * a.tps * SV_TILE; j0 < j_end; j0 += 32) {
        __syncthreads();
        // what a slot that is hidden, or behind the last one, holds may be anything: it is not read into the products
        for (int i = tid; i < 32 * hs; i += 128) {
            const int j = j0 + i / hs, d = i % hs;
            sk[(i / hs) * kp + d] = j < j_end && !(s.hidden && s.hidden[j]) ? sv_ld(kc, j * kvd + d) : 0.f;
        }
        for (int i = tid; i < 32 * hs; i += 128) {
            const int j = j0 + (i & 31), d = i >> 5;
            sv[d * 33 + (i & 31)] = j < j_end && !(s.hidden && s.hidden[j]) ? sv_ld(vc, (int64_t)d * s.n_ctx + j) : 0.f;
        }
        __syncthreads();
        const int j = j0 + lane;
        const bool in = j < j_end && !(s.hidden && s.hidden[j]);
        float z[4] = {0.f, 0.f, 0.f, 0.f};
        for (int d = 0; d < hs; d++) {
            const float kv = sk[lane * kp + d];
#pragma unroll
            for (int r = 0; r < 4; r++) z[r] = fmaf(sq[(warp * 4 + r) * hs + d], kv, z[r]);
        }
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int row = r0 + warp * 4 + r;
            if (!in || row >= rows || !sv_sees(s, row / a.R, j - past)) z[r] = SV_NONE;
            if (s.scores && row < rows && j < j_end) s.scores[(((int64_t)g * sv_quads(s.n_kv) + j / 4) * rp + row) * 4 + j % 4] = z[r];
            float mx = z[r];
#pragma unroll
            for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float mn = fmaxf(m[r], mx), ref = mn == SV_NONE ? 0.f : mn, f = exp2f(m[r] - ref), p = exp2f(z[r] - ref);
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
    float *ml = s.part + (int64_t)s.splits * a.G * rows * hs;
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int row = r0 + warp * 4 + r;
        if (lane == 0 && row < rows) {
            if (s.splits == 1) sv_put_lse(s, (int64_t)g * rows + row, m[r], l[r]);
            else reinterpret_cast<float2 *>(ml)[((int64_t)split * a.G + g) * rows + row] = make_float2(m[r], l[r]);
            sc[warp * 4 + r] = s.splits == 1 ? (l[r] > 0.f ? 1.f / l[r] : 0.f) : 1.f;
        }
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 2; c++) {
        const int d = tid + 128 * c;
        if (d >= hs) break;
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const int row = r0 + r;
            if (row >= rows) break;
            if (s.splits == 1) a.out[((int64_t)(s.tok0 + row / a.R) * a.n_heads + g * a.R + row % a.R) * hs + d] = acc[c][r] * sc[r];
            else s.part[(((int64_t)split * a.G + g) * rows + row) * hs + d] = acc[c][r];
        }
    }
}
inline size_t sv_attn_smem(int hs) { return 4 * ((size_t)16 * hs + 32 * (hs + 1) + (size_t)hs * 33 + 16 * 33 + 16); }

// ---------------------------------------------------------------------------------------------------- joining the splits
// A warp a row of kv head y: a lane a split takes maxima and sums at once, then eight splits' outputs are under way at a time. Its start overlaps the end of the kernel before; bound by
// latency (two dependent rounds of loads): 16 splits of 48 rows of 8 heads 5 us. (Joined by the CTA that comes last, one for all of a head's rows, 30.)
__global__ void __launch_bounds__(256) sv_k_join(const __grid_constant__ SvAttn a) {
    ps_grid_dep_wait();
    ps_grid_dep_launch();
    const int tid = threadIdx.x, lane = tid & 31, hs = a.hs, g = blockIdx.y;
    const SvSeq &s = a.seq[blockIdx.z];
    const int rows = s.n_tok * a.R, row = blockIdx.x * 8 + (tid >> 5);
    if (row >= rows || s.splits == 1) return;
    const float2 *ml = reinterpret_cast<const float2 *>(s.part + (int64_t)s.splits * a.G * rows * hs);
    const int64_t at = (int64_t)g * rows + row, step = (int64_t)a.G * rows;
    float mx = SV_NONE;
    for (int i = lane; i < s.splits; i += 32) mx = fmaxf(mx, ml[i * step + at].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float ref = mx == SV_NONE ? 0.f : mx;
    float l = 0.f, acc[8] = {};
    for (int i0 = 0; i0 < s.splits; i0 += 32) {
        float f = 0.f;
        if (i0 + lane < s.splits) {
            const float2 p = ml[(i0 + lane) * step + at];
            f = exp2f(p.x - ref);
            l = fmaf(p.y, f, l);
        }
        for (int i = 0; i < min(32, s.splits - i0); i += 8) {
            float v[8][8];
#pragma unroll
            for (int e = 0; e < 8; e++)
#pragma unroll
                for (int c = 0; c < 8; c++)
                    if (c * 32 < hs && i0 + i + e < s.splits) v[e][c] = s.part[((i0 + i + e) * step + at) * hs + c * 32 + lane];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float fe = __shfl_sync(0xffffffffu, f, i + e);
#pragma unroll
                for (int c = 0; c < 8; c++)
                    if (c * 32 < hs && i0 + i + e < s.splits) acc[c] = fmaf(v[e][c], fe, acc[c]);
            }
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) sv_put_lse(s, at, mx, l);
    const float inv = l > 0.f ? 1.f / l : 0.f;
    float *to = a.out + ((int64_t)(s.tok0 + row / a.R) * a.n_heads + g * a.R + row % a.R) * hs;
#pragma unroll
    for (int c = 0; c < 8; c++)
        if (c * 32 < hs) to[c * 32 + lane] = acc[c] * inv;
}

// x: 256 slots of a sequence's kv head y: their weights.  PER lanes take rows, four slots each, two such quads at a time; then the lanes exchange halves of their eight sums
// until each has sums of its own (nine shuffles for 32 lanes instead of forty), the old weights are there by then.  Bound by memory: two sequences of 32 700 slots, 128 rows
// of each of 8 kv heads: 268 MB in 47 us = 5.7 TB/s (one old weight at a time and forty shuffles: 92 us)
#define SV_FIN_SLOTS 256
template <int PER> PS_D void sv_weights(const SvSeq &s, const float *lse, int rows, int g, int j0) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, at = lane % PER, rp = sv_rp(rows);
    constexpr int AT = 32 / PER, N = PER >= 8 ? 1 : 8 / PER; // quads of a warp; sums that a lane ends with
    const float4 *z0 = reinterpret_cast<const float4 *>(s.scores) + ((int64_t)g * sv_quads(s.n_kv) + j0 / 4) * rp;
    float *w0 = s.weight + (int64_t)g * s.n_ctx + j0;
    const int n = s.n_kv - j0;
    int first = 0; // number of the first sum that the lane ends with: quad, slot
#pragma unroll
    for (int o = PER / 2, half = 4; o && half; o /= 2, half /= 2) first += at & o ? half : 0;
    const bool writes = PER <= 8 || at % (PER > 8 ? PER / 8 : 1) == 0;
    for (int b = warp * 2 * AT; b < SV_FIN_SLOTS / 4 && 4 * b < n; b += 16 * AT) {
        const int q[2] = {b + lane / PER, b + AT + lane / PER};
        const bool in[2] = {q[0] < SV_FIN_SLOTS / 4 && 4 * q[0] < n, q[1] < SV_FIN_SLOTS / 4 && 4 * q[1] < n};
        float old[N], v[8] = {};
#pragma unroll
        for (int e = 0; e < N; e++) {
            const int i = first + e, slot = 4 * (i >= 4 ? q[1] : q[0]) + i % 4;
            old[e] = writes && (i >= 4 ? in[1] : in[0]) && slot < n ? w0[slot] : 0.f;
        }
#pragma unroll 4
        for (int row = at; row < rows; row += PER) {
            const float4 none = make_float4(SV_NONE, SV_NONE, SV_NONE, SV_NONE);
            const float4 a = in[0] ? __ldcs(z0 + (int64_t)q[0] * rp + row) : none, c = in[1] ? __ldcs(z0 + (int64_t)q[1] * rp + row) : none;
            const float l = lse[row];
            v[0] += sv_ex2(a.x - l); v[1] += sv_ex2(a.y - l); v[2] += sv_ex2(a.z - l); v[3] += sv_ex2(a.w - l);
            v[4] += sv_ex2(c.x - l); v[5] += sv_ex2(c.y - l); v[6] += sv_ex2(c.z - l); v[7] += sv_ex2(c.w - l);
        }
#pragma unroll
        for (int o = PER / 2, half = 4; o; o /= 2, half /= 2) {
            if (half) {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (e < half) {
                        const float keep = at & o ? v[e + half] : v[e], give = at & o ? v[e] : v[e + half];
                        v[e] = keep + __shfl_xor_sync(0xffffffffu, give, o);
                    }
            } else v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
        }
#pragma unroll
        for (int e = 0; e < N; e++) {
            const int i = first + e, slot = 4 * (i >= 4 ? q[1] : q[0]) + i % 4;
            if (writes && (i >= 4 ? in[1] : in[0]) && slot < n) w0[slot] = old[e] + v[e];
        }
    }
}
__global__ void __launch_bounds__(256) sv_k_weights(const __grid_constant__ SvAttn a) {
    extern __shared__ float sv_lse[];
    ps_grid_dep_wait();
    const int g = blockIdx.y, j0 = blockIdx.x * SV_FIN_SLOTS;
    const SvSeq &s = a.seq[blockIdx.z];
    const int rows = s.n_tok * a.R;
    if (!s.scores || j0 >= s.n_kv) return;
    for (int row = threadIdx.x; row < rows; row += 256) sv_lse[row] = s.lse[(int64_t)g * rows + row];
    __syncthreads();
    if (rows > 16) sv_weights<32>(s, sv_lse, rows, g, j0);
    else if (rows > 8) sv_weights<16>(s, sv_lse, rows, g, j0);
    else if (rows > 4) sv_weights<8>(s, sv_lse, rows, g, j0);
    else if (rows > 2) sv_weights<4>(s, sv_lse, rows, g, j0);
    else if (rows > 1) sv_weights<2>(s, sv_lse, rows, g, j0);
    else sv_weights<1>(s, sv_lse, rows, g, j0);
}
