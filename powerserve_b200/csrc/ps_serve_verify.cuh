// ps_serve_verify.cuh - drafted tokens against the target's distribution p and the draft's q, from given random numbers.
//
// Beginning at node 0, the children of the last accepted node are asked in order: child i with token c is accepted where u_i < p(c) / q(c); where not, p becomes max(p - q, 0), normalised.
// With p_0 = p and T_0 = 1, the k-th rejection leaves p_k = max(p - t_k q, 0) / T_k with t_k+1 = t_k + T_k and T_k+1 = sum max(p - t_k+1 q, 0) (as max(max(x - a, 0) - b, 0) = max(x - a - b, 0)
// for b >= 0): so a rejection costs one pass over the two rows, whatever came before, and no row is written.  Without a draft's rows q is one at c: p loses c, and T is a sum of whole numbers less one of them.
//
// sv_k_stats finds for every row what its settings leave of it (ps_serve_sample.cuh): a border and a mass.  (Rows that were looked at only when the walk came to them, by the cluster of the walk: 780 us for 64 sequences of
// five nodes, of whose rows two thirds are looked at, where 580 took all of them at once.)  Then sv_k_verify: a cluster a sequence walks its tree - every CTA the same walk, whose tests ask for a few weights - and meets
// for the passes: a sum for each rejection that a sibling or the draw asks about, and the draw.  Weights and sums are whole numbers, as there, so what is accepted does not depend on the launch.
// 64 sequences of five nodes, rows and drafts' rows of 128 256 with mixed settings: 95 us for rows by a CTA each, 283 for those left to clusters (a row a microsecond, bound by the cluster's exchanges), 81 for the walks.
// Masses of whole rows are sums of the weights that a draw sees, of 2^-44: p sums to one, and a top-p has the border that ps_cuda_sample finds.  (By float32 exponentials, off by 2^-20: 86 and 272 us.)
#pragma once
#include "ps_serve_sample.cuh"

#define SV_VERIFY_SEQS 1024 // sequences of a launch: their first nodes are a kernel parameter
#define SV_P_ONE 0x1p58     // a residual's unit: sums stay below 2^59

struct SvStats { // [0]: the target's, [1]: the draft's, whose rows come behind the target's
    const float *logits[2];
    const ps_cuda_sampler *samplers[2];
    SvRowStats *stats[2];
    int vec[2];
    uint8_t *todo;          // [row] not 0: the row is left to the clusters; or null, and all are
    const int32_t *parents;
    int64_t row_stride;
    int vocab, chunk;       // chunk: tokens of a cluster's CTA
    int first[SV_VERIFY_SEQS + 1], n_seqs;
    PS_D SvSample sample(int d) const {
        SvSample s{};
        s.logits = logits[d]; s.samplers = samplers[d]; s.stats = stats[d]; s.row_stride = row_stride; s.vocab = vocab; s.chunk = chunk; s.vec = vec[d];
        return s;
    }
    // whether anybody asks for the draft's row
    PS_D bool has_child(int row) const {
        int lo = 0, hi = n_seqs - 1; // the last sequence that begins at or before the row
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (first[mid] <= row) lo = mid;
            else hi = mid - 1;
        }
        int child = 0;
        for (int i = row + 1 + (int)threadIdx.x; i < first[lo + 1]; i += SV_SMP_THREADS) child |= parents[i] == row - first[lo];
        return __syncthreads_or(child) != 0;
    }
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

// settings whose rows a CTA alone hardly ever decides: many tokens, the border of a mass that thousands of tokens share, or a min-p that leaves tokens which are not listed
PS_D bool sv_hard(const ps_cuda_sampler &p, int vocab) {
    const bool use_k = p.top_k > 0 && p.top_k < vocab;
    return p.temperature > 0.f && (use_k ? p.top_k > SV_SMP_THREADS / 2 : (p.top_p < 1.f || p.min_p > 0.f) && !(p.min_p >= 0x1p-16f));
}
// a cluster a row.  Where sv_k_rows runs before it, its end overlaps this one's start: what it leaves for certain is not waited for
__global__ void __launch_bounds__(SV_SMP_THREADS, 2) sv_k_stats(const __grid_constant__ SvStats a) {
    const int row = blockIdx.x / cooperative_groups::this_cluster().num_blocks(), nodes = a.first[a.n_seqs], d = row >= nodes;
    const bool hard = a.todo && sv_hard(a.samplers[d][row - d * nodes], a.vocab);
    if (a.todo && !hard) {
        ps_grid_dep_wait();
        if (!a.todo[row]) return; // (the whole cluster)
    }
    if (!a.todo || hard)
        if (d && !a.has_child(row - nodes)) {
            ps_grid_dep_wait();
            return;
        }
    const SvSample s = a.sample(d);
    sv_sample<true>(s, row - d * nodes);
    ps_grid_dep_wait(); // (who comes after this kernel comes after the one before, too)
}

// A CTA a row, for many rows: the row is read twice, once from memory and once from L2, and only the likely tokens are kept.  What they do not decide (more than 1 024 of them, or fewer than top_k asks for) is left
// to the clusters, which keep the row: those have 37 rows under way at a time, this 296
__global__ void __launch_bounds__(SV_SMP_THREADS, 2) sv_k_rows(const __grid_constant__ SvStats a) {
    __shared__ SvSmpShared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nodes = a.first[a.n_seqs], d = (int)blockIdx.x >= nodes, row = blockIdx.x - d * nodes;
    ps_grid_dep_launch();
    if (tid == 0) a.todo[blockIdx.x] = 0;
    if (sv_hard(a.samplers[d][row], a.vocab) || (d && !a.has_child(row))) return;
    const float *from = a.logits[d] + row * a.row_stride;
    const int n4 = a.vec[d] ? a.vocab / 4 : 0;
    // f(logit, number) of the CTA's tokens, four at a time; no number is -inf
    auto each = [&](auto f) {
#pragma unroll 4
        for (int i = tid; i < n4; i += SV_SMP_THREADS) {
            const float4 v = __ldg(reinterpret_cast<const float4 *>(from) + i);
            f(v.x == v.x ? v.x : -INFINITY, 4 * i);
            f(v.y == v.y ? v.y : -INFINITY, 4 * i + 1);
            f(v.z == v.z ? v.z : -INFINITY, 4 * i + 2);
            f(v.w == v.w ? v.w : -INFINITY, 4 * i + 3);
        }
#pragma unroll 4
        for (int i = 4 * n4 + tid; i < a.vocab; i += SV_SMP_THREADS) {
            const float v = __ldg(from + i);
            f(v == v ? v : -INFINITY, i);
        }
    };
    float most = -INFINITY, least = INFINITY;
    each([&](float v, int) {
        most = fmaxf(most, v);
        least = fminf(least, v > -INFINITY ? v : INFINITY);
    });
    if (tid < 32) sh.pow2[tid] = exp2(tid / 32.0);
    if (tid == 0) sh.n_list = 0;
    SvSmpRow r{};
    r.vocab = a.vocab;
    r.p = a.samplers[d][row];
    const uint32_t mine = most > -INFINITY ? sv_rank(most) : 0, of_warp = __reduce_max_sync(0xffffffffu, mine), low = __reduce_min_sync(0xffffffffu, sv_rank(least));
    if (lane == 0) { sh.warp_most[warp] = of_warp; sh.warp_listed[warp] = low; }
    __syncthreads();
    const uint32_t best = __reduce_max_sync(0xffffffffu, sh.warp_most[lane & 15]), worst = __reduce_min_sync(0xffffffffu, sh.warp_listed[lane & 15]);
    SvRowStats *to = a.stats[d] + row;
    r.log2w.top = sv_unrank(best);
    if (best == 0 || !(r.p.temperature > 0.f)) { // one token, the lowest that has the largest logit, or none
        unsigned long long at = 0;
        if (best)
            each([&](float v, int i) {
                if (v == r.log2w.top) at = max(at, (unsigned long long)~(uint32_t)i);
            });
        at = sv_block<true>(sh, at);
        if (tid == 0) *to = SvRowStats{0, 0, r.log2w.top, best ? (int)~(uint32_t)at : -1};
        return;
    }
    // a number that top_k tokens reach: the top_k-th largest of the threads' largest
    uint32_t reach = 0;
    if (r.p.top_k >= 1 && r.p.top_k <= SV_SMP_THREADS && r.p.top_k < a.vocab) {
        unsigned long long *sorted = reinterpret_cast<unsigned long long *>(sh.lists);
        sorted[tid] = mine;
        sv_sort(sorted, SV_SMP_THREADS);
        reach = (uint32_t)sorted[r.p.top_k - 1];
        __syncthreads();
    }
    sv_settings(r, sv_unrank(worst), reach);
    const bool filters = r.use_k || r.use_p || r.min_w, last = r.min_w >= SV_ONE >> (int)SV_SMP_SPAN; // last: min-p takes out all that is not listed
    const bool mass = !filters || (r.use_p && !r.use_k);
    unsigned long long whole = 0;
    auto list = [&](float v, int i) {
        if (v >= r.cut && v > -INFINITY) {
            const uint32_t n = atomicAdd(&sh.n_list, 1u);
            if (n < SV_SMP_BINS) sh.list[n] = sv_key(v, i);
        }
    };
    auto weigh = [&](float v) {
        const unsigned long long w = sv_weight(sh, r.log2w(v));
        whole += v > -INFINITY ? w : 0;
    };
    // (a loop for each case, so that several weights are under way at once)
    if (!filters) each([&](float v, int) { weigh(v); });
    else if (!mass) each(list);
    else each([&](float v, int i) { list(v, i); weigh(v); });
    whole = sv_block<false>(sh, whole);
    __syncthreads();
    if (!filters) {
        if (tid == 0) *to = SvRowStats{0, whole, r.log2w.top, 0};
        return;
    }
    const int n = (int)min(sh.n_list, (uint32_t)SV_SMP_BINS + 1);
    // (beside a smaller min-p, top-p without top-k is not asked here: sv_hard)
    const bool known = n <= SV_SMP_BINS && (r.use_k ? n >= r.p.top_k || (last && !r.use_p) : last);
    if (!known) {
        if (tid == 0) a.todo[blockIdx.x] = 1;
        return;
    }
    SvSample s = a.sample(d);
    sv_few<true>(s, row, r, sh, n, whole);
}

// a row's distribution
struct SvDist {
    const float *x;
    SvScale log2w;
    unsigned long long kappa, min_w, all;
    int only;
    float cut;          // tokens with smaller logits have nothing (that is nearly all of them where there are filters)
    double inv;         // of `all`
    PS_D void load(const float *row, const SvRowStats &st, const ps_cuda_sampler &p) {
        x = row; kappa = st.kappa; all = st.all; only = st.only;
        min_w = p.min_p > 0.f ? (unsigned long long)ceil((double)fminf(p.min_p, 1.f) * (double)SV_ONE) : 0;
        log2w.top = st.top;
        log2w.s = 1.4426950408889634 / (double)p.temperature;
        log2w.off = -(double)st.top * log2w.s;
        if (st.top == INFINITY) { log2w.s = 0.0; log2w.off = -INFINITY; }
        const double least = min_w ? fmax(log2((double)min_w) - 44.0, -46.0) - 1e-6 : -46.0; // log2 of the least weight
        cut = st.top == INFINITY ? INFINITY : fmaxf(__double2float_rd((double)st.top + least / log2w.s), kappa ? sv_logit(kappa) : -INFINITY);
        if (all == 0) all = SV_ONE, kappa = ~0ull, cut = INFINITY; // (one token has all of it, or none)
        else only = -1;
        inv = 1.0 / (double)all;
    }
    PS_D unsigned long long of(const double *pow2, float v, int i) const { // (without branches, so that several are under way at once)
        const bool in = v > -INFINITY && sv_key(v, i) >= kappa;
        const unsigned long long w = sv_weight(pow2, log2w(v));
        return i == only ? SV_ONE : in && w >= min_w ? w : 0;
    }
    // the same as a number, for a test: below 2^-20 a whole number of 2^-44 says too little about p(c) / q(c)
    PS_D double operator()(const double *pow2, int i, unsigned long long &w) const {
        const float v = x[i];
        w = of(pow2, v, i);
        return i == only ? (double)SV_ONE : v > -INFINITY && sv_key(v, i) >= kappa && sv_weight(pow2, log2w(v)) >= min_w ? exp2(log2w(v)) * (double)SV_ONE : 0.0;
    }
};

// how many of the warp's tokens come before token c.  (Hardly ever asked for: no registers of the walk's are kept for it)
__device__ __noinline__ unsigned sv_above(const float *row, int c, int w0, int w1) {
    const unsigned long long key = sv_key(row[c], c);
    unsigned above = 0;
    for (int i = w0 + (threadIdx.x & 31); i < w1; i += 32) {
        const float v = row[i];
        above += v > -INFINITY && sv_key(v, i) > key;
    }
    return __reduce_add_sync(0xffffffffu, above);
}

__global__ void __launch_bounds__(SV_SMP_THREADS, 2) sv_k_verify(const __grid_constant__ SvVerify a) {
    namespace cg = cooperative_groups;
    constexpr int WARPS = SV_SMP_THREADS / 32;
    __shared__ double pow2[32], s_pc[PS_CUDA_TREE_TOKENS], s_qc[PS_CUDA_TREE_TOKENS];
    __shared__ unsigned long long mail[2][16], warp_sum[WARPS], s_w[PS_CUDA_TREE_TOKENS], s_all[PS_CUDA_TREE_TOKENS];
    __shared__ int s_parent[PS_CUDA_TREE_TOKENS], s_token[PS_CUDA_TREE_TOKENS], s_path[PS_CUDA_TREE_TOKENS], s_gone[PS_CUDA_TREE_TOKENS], s_last[PS_CUDA_TREE_TOKENS]; // s_last: a node's last child
    __shared__ float s_u[PS_CUDA_TREE_TOKENS];
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = cl.block_rank(), C = cl.num_blocks();
    const int seq = blockIdx.x / C, base = a.first[seq], n = a.first[seq + 1] - base;
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    int turn = 0;
    if (tid < 32) pow2[tid] = exp2(tid / 32.0);
    __syncthreads();
    auto target = [&](SvDist &d, int i) { d.load(a.logits + (int64_t)(base + i) * a.row_stride, a.target[base + i], a.samplers[base + i]); };
    auto draft = [&](SvDist &d, int i) { d.load(a.draft_logits + (int64_t)(base + i) * a.row_stride, a.draft[base + i], a.draft_samplers[base + i]); };
    for (int i = tid; i < n; i += SV_SMP_THREADS) {
        const int up = a.parents[base + i], c = a.tokens[base + i];
        s_parent[i] = up;
        s_u[i] = a.u[base + i];
        s_token[i] = i > 0 && up >= 0 && up < i && c >= 0 && c < a.vocab ? c : -1; // (-1: never accepted)
        s_last[i] = -1;
    }
    __syncthreads();
    if (tid < n && s_token[tid] >= 0) atomicMax(&s_last[s_parent[tid]], tid);
    // what the tests ask for: a thread a node, all at once
    if (tid < n) {
        const int i = tid;
        const unsigned long long all = a.target[base + i].all;
        s_all[i] = all ? all : SV_ONE;
        if (s_token[i] >= 0) {
            SvDist d;
            target(d, s_parent[i]);
            unsigned long long w;
            const double x = d(pow2, s_token[i], w);
            s_w[i] = w;
            s_pc[i] = a.draft_logits ? x * d.inv : x;
            if (a.draft_logits) {
                draft(d, s_parent[i]);
                s_qc[i] = d(pow2, s_token[i], w) * d.inv;
            }
        }
    }
    __syncthreads();
    SvDist p, q;
    int cur = 0, n_path = 1, n_gone = 0;
    double t = 0.0, T = 1.0, before = 0.0; // before: t before the last rejection
    unsigned long long left = s_all[0]; // without a draft: mass of what p still has
    bool have = false;                  // p and q are row cur's
    const int i0 = min(rank * a.chunk, a.vocab), i1 = min(i0 + a.chunk, a.vocab);
    const int run = ((i1 - i0 + WARPS - 1) / WARPS + 31) & ~31, w0 = min(i0 + warp * run, i1), w1 = min(w0 + run, i1); // the warp's tokens
    // what tokens i + 32 e still have, in whole numbers: E weights of a row are under way at a time
    auto masses = [&](int i, auto &m) {
        constexpr int E = sizeof(m) / sizeof(m[0]);
        float x[E], y[E];
        bool some = false;
#pragma unroll
        for (int e = 0; e < E; e++) {
            x[e] = i + 32 * e < w1 ? p.x[i + 32 * e] : -INFINITY;
            some |= x[e] >= p.cut || i + 32 * e == p.only;
            m[e] = 0;
        }
        if (!__any_sync(0xffffffffu, some)) return;
        if (t > 0.0)
#pragma unroll
            for (int e = 0; e < E; e++) y[e] = i + 32 * e < w1 ? q.x[i + 32 * e] : -INFINITY;
#pragma unroll
        for (int e = 0; e < E; e++) m[e] = i + 32 * e < w1 ? p.of(pow2, x[e], i + 32 * e) : 0;
        if (t > 0.0)
#pragma unroll
            for (int e = 0; e < E; e++) {
                const double r = m[e] ? (double)m[e] * p.inv - t * ((double)q.of(pow2, y[e], i + 32 * e) * q.inv) : 0.0;
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
        for (int i = w0; i < w1; i += 128) {
            unsigned long long m[4];
            masses(i + lane, m);
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
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); // (all CTAs are there, so `meet` may write to them)
    for (int i = 1; i < n; i++) {
        const int c = s_token[i];
        if (s_parent[i] != cur || c < 0) continue;
        bool yes;
        if (a.draft_logits) yes = (double)s_u[i] * T * s_qc[i] < s_pc[i] - t * s_qc[i];
        else {
            const unsigned long long w = s_w[i];
            bool gone = false;
            for (int g = 0; g < n_gone; g++) gone |= s_gone[g] == c;
            yes = !gone && (double)s_u[i] * (double)left < s_pc[i];
            if (!yes && !gone && w && left > w) { // (p stays where nothing would be left)
                __syncthreads();
                if (tid == 0) s_gone[n_gone] = c;
                n_gone++;
                left -= w;
                __syncthreads();
            }
        }
        if (yes && s_w[i] == 0) { // a token below 2^-46 of the likeliest, by u = 0 or a q as small: where the border of a top-k lies down there, the row's record leaves all of them in (no draw asks)
            const ps_cuda_sampler &set = a.samplers[base + cur];
            if (set.top_k > 0 && set.top_k < a.vocab) {
                const unsigned long long *m = meet(sv_above(a.logits + (int64_t)(base + cur) * a.row_stride, c, w0, w1));
                unsigned long long rank_c = 0;
                for (int o = 0; o < C; o++) rank_c += m[o];
                yes = rank_c < (unsigned long long)set.top_k;
            }
        }
        if (yes) {
            if (tid == 0) s_path[n_path] = i;
            n_path++;
            cur = i;
            left = s_all[i];
            t = 0.0; T = 1.0; n_gone = 0; have = false;
        } else if (a.draft_logits) {
            before = t;
            if (t == 0.0) have = false; // (q is asked for, too)
            t += T;
            if (s_last[cur] > i) { // (a sibling asks for T)
                const unsigned long long *m = meet(warp_mass());
                unsigned long long sum = 0;
                for (int o = 0; o < C; o++) sum += m[o];
                if (sum) T = (double)sum * (1.0 / SV_P_ONE);
                else t = before;
            }
        }
    }
    // the next token
    unsigned long long mine, start, block, all;
    for (int again = 0;; again++) {
        mine = warp_mass();
        const unsigned long long *m = meet(mine);
        start = block = all = 0;
        for (int o = 0; o < C; o++) {
            if (o < rank) start += m[o];
            if (o == rank) block = m[o];
            all += m[o];
        }
        if (all || t == 0.0 || again) break;
        t = before; // (nothing is left of p: it stays what it was)
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
    if (goal < start || goal >= start + block) return;
    for (int w = 0; w < warp; w++) start += warp_sum[w];
    if (goal < start || goal >= start + mine) return;
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
            const unsigned ball = __ballot_sync(0xffffffffu, goal < start + inc);
            if (ball) {
                if (lane == __ffs(ball) - 1) a.ids[seq] = i + 32 * e + lane;
                return;
            }
            start += __shfl_sync(0xffffffffu, inc, 31);
        }
    }
}
