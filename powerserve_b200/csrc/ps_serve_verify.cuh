// ps_serve_verify.cuh - drafted tokens against the target's distribution p and the draft's q, from given random numbers.
//
// Beginning at node 0, the children of the last accepted node are asked in order: child i with token c is accepted where u_i < p(c) / q(c); where not, p becomes max(p - q, 0), normalised.
// With p_0 = p and T_0 = 1, the k-th rejection leaves p_k = max(p - t_k q, 0) / T_k with t_k+1 = t_k + T_k and T_k+1 = sum max(p - t_k+1 q, 0) (as max(max(x - a, 0) - b, 0) = max(x - a - b, 0)
// for b >= 0): so a rejection costs one pass over the two rows, whatever came before, and no row is written.  Without a draft's rows q is one at c: p loses c, and T is a sum of whole numbers less one of them.
//
// sv_k_stats finds for every row what its settings leave of it (ps_serve_sample.cuh): a border and a mass.  Then sv_k_verify: a cluster a sequence walks its tree - every CTA the same walk, whose
// tests ask for a few weights - and meets for the passes: a sum for each rejection, and the draw.  Weights and sums are whole numbers, as there, so what is accepted does not depend on the launch.
#pragma once
#include "ps_serve_sample.cuh"

#define SV_VERIFY_SEQS 1024 // sequences of a launch: their first nodes are a kernel parameter
#define SV_P_ONE 0x1p58     // a residual's unit: sums stay below 2^59

struct SvStats {
    SvSample s;
    const int32_t *parents; // or null; a row whose node nobody has for a parent is left out
    int first[SV_VERIFY_SEQS + 1], n_seqs;
};
struct SvVerify {
    const SvRowStats *target, *draft;
    int32_t *ids, *path, *n_path;
    const int32_t *parents, *tokens;
    const float *logits, *draft_logits, *u;
    const ps_cuda_sampler *samplers, *draft_samplers;
    int64_t row_stride;
    int vocab, chunk;
    int first[SV_VERIFY_SEQS + 1];
};

__global__ void __launch_bounds__(SV_SMP_THREADS, 2) sv_k_stats(const __grid_constant__ SvStats a) {
    if (a.parents) {
        const int row = blockIdx.x / cooperative_groups::this_cluster().num_blocks();
        int lo = 0, hi = a.n_seqs - 1; // the last sequence that begins at or before the row
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (a.first[mid] <= row) lo = mid;
            else hi = mid - 1;
        }
        int child = 0;
        for (int i = row + 1 + (int)threadIdx.x; i < a.first[lo + 1]; i += SV_SMP_THREADS) child |= a.parents[i] == row - a.first[lo];
        if (!__syncthreads_or(child)) return; // (the whole cluster)
    }
    sv_sample<true>(a.s);
}

// a row's distribution
struct SvDist {
    const float *x;
    SvScale log2w;
    unsigned long long kappa, min_w, all;
    int only;
    double inv;         // of `all`
    PS_D void load(const float *row, const SvRowStats &st, const ps_cuda_sampler &p) {
        x = row; kappa = st.kappa; all = st.all; only = st.only;
        min_w = p.min_p > 0.f ? (unsigned long long)ceil((double)fminf(p.min_p, 1.f) * (double)SV_ONE) : 0;
        log2w.top = st.top;
        log2w.s = 1.4426950408889634 / (double)p.temperature;
        log2w.off = -(double)st.top * log2w.s;
        if (st.top == INFINITY) { log2w.s = 0.0; log2w.off = -INFINITY; }
        if (all == 0) all = SV_ONE, kappa = ~0ull; // (one token has all of it, or none)
        else only = -1;
        inv = 1.0 / (double)all;
    }
    PS_D unsigned long long of(const double *pow2, float v, int i) const { // (without branches, so that several are under way at once)
        const bool in = v > -INFINITY && sv_key(v, i) >= kappa;
        const unsigned long long w = sv_weight(pow2, log2w(v));
        return i == only ? SV_ONE : in && w >= min_w ? w : 0;
    }
    PS_D unsigned long long operator()(const double *pow2, int i) const { return of(pow2, x[i], i); }
};

__global__ void __launch_bounds__(SV_SMP_THREADS, 2) sv_k_verify(const __grid_constant__ SvVerify a) {
    namespace cg = cooperative_groups;
    constexpr int WARPS = SV_SMP_THREADS / 32;
    __shared__ double pow2[32], s_pc[PS_CUDA_TREE_TOKENS], s_qc[PS_CUDA_TREE_TOKENS];
    __shared__ unsigned long long mail[2][16], warp_sum[WARPS], s_w[PS_CUDA_TREE_TOKENS], s_all[PS_CUDA_TREE_TOKENS];
    __shared__ int s_parent[PS_CUDA_TREE_TOKENS], s_token[PS_CUDA_TREE_TOKENS], s_path[PS_CUDA_TREE_TOKENS], s_gone[PS_CUDA_TREE_TOKENS];
    __shared__ float s_u[PS_CUDA_TREE_TOKENS];
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = cl.block_rank(), C = cl.num_blocks();
    const int seq = blockIdx.x / C, base = a.first[seq], n = a.first[seq + 1] - base;
    int turn = 0;
    if (tid < 32) pow2[tid] = exp2(tid / 32.0);
    __syncthreads();
    auto target = [&](SvDist &d, int i) { d.load(a.logits + (int64_t)(base + i) * a.row_stride, a.target[base + i], a.samplers[base + i]); };
    auto draft = [&](SvDist &d, int i) { d.load(a.draft_logits + (int64_t)(base + i) * a.row_stride, a.draft[base + i], a.draft_samplers[base + i]); };
    // what the tests ask for: a thread a node, all at once
    if (tid < n) {
        const int i = tid, up = a.parents[base + i], c = a.tokens[base + i];
        const unsigned long long all = a.target[base + i].all;
        s_parent[i] = up;
        s_u[i] = a.u[base + i];
        s_all[i] = all ? all : SV_ONE;
        const bool in = i > 0 && up >= 0 && up < i && c >= 0 && c < a.vocab;
        s_token[i] = in ? c : -1;
        if (in) {
            SvDist d;
            target(d, up);
            const unsigned long long w = d(pow2, c);
            s_w[i] = w;
            s_pc[i] = (double)w * d.inv;
            if (a.draft_logits) {
                draft(d, up);
                s_qc[i] = (double)d(pow2, c) * d.inv;
            }
        }
    }
    __syncthreads();
    SvDist p, q;
    int cur = 0, n_path = 1, n_gone = 0;
    double t = 0.0, T = 1.0;
    unsigned long long left = s_all[0]; // without a draft: mass of what p still has
    bool have = false;                  // p and q are row cur's
    const int i0 = min(rank * a.chunk, a.vocab), i1 = min(i0 + a.chunk, a.vocab);
    const int run = ((i1 - i0 + WARPS - 1) / WARPS + 31) & ~31, w0 = min(i0 + warp * run, i1), w1 = min(w0 + run, i1); // the warp's tokens
    // what tokens i + 32 e still have, in whole numbers: E weights of a row are under way at a time
    auto masses = [&](int i, auto &m) {
        constexpr int E = sizeof(m) / sizeof(m[0]);
        float x[E], y[E];
#pragma unroll
        for (int e = 0; e < E; e++) x[e] = i + 32 * e < w1 ? p.x[i + 32 * e] : -INFINITY;
        if (t > 0.0)
#pragma unroll
            for (int e = 0; e < E; e++) y[e] = i + 32 * e < w1 ? q.x[i + 32 * e] : -INFINITY;
#pragma unroll
        for (int e = 0; e < E; e++) m[e] = i + 32 * e < w1 ? p.of(pow2, x[e], i + 32 * e) : 0;
        if (t > 0.0)
#pragma unroll
            for (int e = 0; e < E; e++) {
                const double r = i + 32 * e < w1 ? (double)m[e] * p.inv - t * ((double)q.of(pow2, y[e], i + 32 * e) * q.inv) : 0.0;
                m[e] = r > 0.0 ? (unsigned long long)(r * SV_P_ONE) : 0;
            }
        for (int g = 0; g < n_gone; g++)
#pragma unroll
            for (int e = 0; e < E; e++)
                if (s_gone[g] == i + 32 * e) m[e] = 0;
    };
    auto warp_mass = [&]() {
        if (!have) {
            target(p, cur);
            if (t > 0.0) draft(q, cur);
            have = true;
        }
        unsigned long long sum = 0;
        for (int i = w0 + lane; i < w1; i += 128) {
            unsigned long long m[4];
            masses(i, m);
#pragma unroll
            for (int e = 0; e < 4; e++) sum += m[e];
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        return sum;
    };
    // the CTAs' sums to every CTA; its own warps' stay in warp_sum
    auto meet = [&](unsigned long long of_warp) -> const unsigned long long * {
        __syncthreads();
        if (lane == 0) warp_sum[warp] = of_warp;
        __syncthreads();
        turn ^= 1;
        if (tid < C) {
            unsigned long long block = 0;
            for (int w = 0; w < WARPS; w++) block += warp_sum[w];
            cl.map_shared_rank(&mail[turn][0], tid)[rank] = block;
        }
        cl.sync();
        return mail[turn];
    };
    for (int i = 1; i < n; i++) {
        const int c = s_token[i];
        if (s_parent[i] != cur || c < 0) continue;
        bool yes;
        if (a.draft_logits) yes = (double)s_u[i] * T * s_qc[i] < s_pc[i] - t * s_qc[i];
        else {
            const unsigned long long w = s_w[i];
            bool gone = false;
            for (int g = 0; g < n_gone; g++) gone |= s_gone[g] == c;
            yes = !gone && (double)s_u[i] * (double)left < (double)w;
            if (!yes && !gone && w && left > w) { // (p stays where nothing would be left)
                __syncthreads();
                if (tid == 0) s_gone[n_gone] = c;
                n_gone++;
                left -= w;
                __syncthreads();
            }
        }
        if (yes) {
            if (tid == 0) s_path[n_path] = i;
            n_path++;
            cur = i;
            left = s_all[i];
            t = 0.0; T = 1.0; n_gone = 0; have = false;
        } else if (a.draft_logits) {
            const double t_was = t;
            if (t == 0.0) have = false; // (q is asked for, too)
            t += T;
            const unsigned long long *m = meet(warp_mass());
            unsigned long long sum = 0;
            for (int o = 0; o < C; o++) sum += m[o];
            if (sum) T = (double)sum * (1.0 / SV_P_ONE);
            else t = t_was;
        }
    }
    // the next token
    const unsigned long long mine = warp_mass();
    const unsigned long long *m = meet(mine);
    unsigned long long before = 0, block = 0, all = 0;
    for (int o = 0; o < C; o++) {
        if (o < rank) before += m[o];
        if (o == rank) block = m[o];
        all += m[o];
    }
    if (rank == 0) {
        for (int i = tid; i < n; i += SV_SMP_THREADS) a.path[base + i] = i == 0 ? 0 : i < n_path ? s_path[i] : -1;
        if (tid == 0) {
            a.n_path[seq] = n_path;
            if (all == 0) a.ids[seq] = -1;
        }
    }
    if (all == 0) return;
    const float u = s_u[0];
    unsigned long long goal = u > 0.f ? (unsigned long long)((double)fminf(u, 1.f) * (double)all) : 0;
    goal = min(goal, all - 1);
    if (goal < before || goal >= before + block) return;
    for (int w = 0; w < warp; w++) before += warp_sum[w];
    if (goal < before || goal >= before + mine) return;
    for (int i = w0; i < w1; i += 64) {
        unsigned long long w[2];
        masses(i + lane, w);
#pragma unroll
        for (int e = 0; e < 2; e++) {
            unsigned long long inc = w[e];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned long long v = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += v;
            }
            const unsigned ball = __ballot_sync(0xffffffffu, goal < before + inc);
            if (ball) {
                if (lane == __ffs(ball) - 1) a.ids[seq] = i + 32 * e + lane;
                return;
            }
            before += __shfl_sync(0xffffffffu, inc, 31);
        }
    }
}
