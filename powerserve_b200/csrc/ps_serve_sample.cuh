// ps_serve_sample.cuh - one token of each row of logits: temperature, top-k, top-p, min-p, and a given random number.
//
// w_i = exp((x_i - max) / T).  The tokens in the order (logit, lower token): the first top_k; of these the shortest beginning that holds top_p of
// their mass; of these the ones with w >= min_p.  The token is the first one, in the vocabulary's order, where the kept tokens' running mass is
// over u times all of it.  A weight is a whole number of 2^-44: sums do not depend on their order, so the result does not depend on the launch.
//
// A cluster of CTAs takes a row.  Both borders are borders of the sorted order, which nobody sorts: a histogram over log2 w (counts and masses)
// finds the bin that the border lies in, its few members are gathered and sorted, and the border becomes a number (logit, token) to compare with.
#pragma once
#include "ps_ptx.cuh"

#include <cooperative_groups.h>

#define SV_SMP_THREADS 512
#define SV_SMP_BINS 2048
#define SV_SMP_LIST 2048
#define SV_SMP_CLUSTER 8
#define SV_ONE (1ull << 44)

struct SvSample {
    const float *logits;
    const ps_cuda_sampler *samplers;
    const float *u;
    int32_t *ids;
    float *probs;
    int64_t row_stride;
    int vocab, chunk;       // tokens of a CTA
};
struct SvSmpShared {
    unsigned long long mass[SV_SMP_BINS], list[SV_SMP_LIST], mail[2][4][16], red[32];
    uint32_t count[SV_SMP_BINS];
    unsigned long long border[4];
    uint32_t n_list;
};

PS_D unsigned long long sv_key(float x, int i) { // (logit, lower token first) as a number; no number and -inf: nothing
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (unsigned long long)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (uint32_t)~i;
}
PS_D double sv_log2w(float x, float top, double s) { return x == top ? 0.0 : ((double)x - (double)top) * s; }
PS_D unsigned long long sv_weight(double t) { return t > -46.0 ? (unsigned long long)(exp2(t) * (double)SV_ONE + 0.5) : 0ull; }

template <bool MAX> PS_D unsigned long long sv_block(SvSmpShared &sh, unsigned long long v) { // sum or maximum over the block
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto join = [](unsigned long long x, unsigned long long y) { return MAX ? (x > y ? x : y) : x + y; };
#pragma unroll
    for (int o = 16; o; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if (lane == 0) sh.red[warp] = v;
    __syncthreads();
    v = lane < SV_SMP_THREADS / 32 ? sh.red[lane] : 0;
#pragma unroll
    for (int o = 16; o; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
// every CTA's numbers to every CTA: mail[turn][kind][rank].  Two turns are enough: who writes the turn after next has passed a barrier that all reach
// with the last but one read
struct SvMail {
    cooperative_groups::cluster_group cl;
    SvSmpShared &sh;
    int turn, rank, size;
    PS_D SvMail(SvSmpShared &s) : cl(cooperative_groups::this_cluster()), sh(s), turn(0), rank(cl.block_rank()), size(cl.num_blocks()) {}
    PS_D const unsigned long long (*post(unsigned long long a, unsigned long long b = 0, unsigned long long c = 0, unsigned long long d = 0))[16] {
        turn ^= 1;
        if ((int)threadIdx.x < size) {
            unsigned long long (*to)[16] = cl.map_shared_rank(&sh, threadIdx.x)->mail[turn];
            to[0][rank] = a; to[1][rank] = b; to[2][rank] = c; to[3][rank] = d;
        }
        cl.sync();
        return sh.mail[turn];
    }
};

// sorts the n numbers of sh.list, largest first
PS_D void sv_sort(SvSmpShared &sh, int n) {
    int p2 = 2;
    while (p2 < n) p2 *= 2;
    for (int i = n + threadIdx.x; i < p2; i += SV_SMP_THREADS) sh.list[i] = 0;
    __syncthreads();
    for (int k = 2; k <= p2; k *= 2)
        for (int j = k / 2; j; j /= 2) {
            for (int i = threadIdx.x; i < p2 / 2; i += SV_SMP_THREADS) {
                const int lo = (i / j) * 2 * j + i % j, hi = lo + j;
                const unsigned long long x = sh.list[lo], y = sh.list[hi];
                if ((x < y) == ((lo & k) == 0)) { sh.list[lo] = y; sh.list[hi] = x; }
            }
            __syncthreads();
        }
}

template <bool KEPT> // the row's logits fit the cluster's shared memory
__global__ void __launch_bounds__(SV_SMP_THREADS) sv_k_sample(const __grid_constant__ SvSample a) {
    extern __shared__ float sv_x[];
    __shared__ SvSmpShared sh;
    SvMail mail(sh);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = mail.rank, C = mail.size;
    const int64_t row = blockIdx.x / C;
    const float *x0 = a.logits + row * a.row_stride;
    const int i0 = min(rank * a.chunk, a.vocab), n = min(a.chunk, a.vocab - i0);
    auto at = [&](int i) {
        const float x = KEPT ? sv_x[i] : x0[i0 + i];
        return x == x ? x : -INFINITY;
    };
    // ---- the largest logit and the lowest token that has it
    unsigned long long best = 0;
    for (int i = tid; i < n; i += SV_SMP_THREADS) {
        float x = x0[i0 + i];
        if (KEPT) sv_x[i] = x;
        if (x > -INFINITY) best = max(best, sv_key(x, i0 + i));
    }
    best = sv_block<true>(sh, best);
    mail.cl.sync(); // (all CTAs are there)
    {
        const unsigned long long(*m)[16] = mail.post(best);
        for (int r = 0; r < C; r++) best = max(best, m[0][r]);
    }
    const ps_cuda_sampler p = a.samplers[row];
    const int first = (int)~(uint32_t)best;
    if (best == 0 || !(p.temperature > 0.f)) { // (the whole cluster goes; nothing of a CTA that has gone is read)
        if (rank == 0 && tid == 0) {
            a.ids[row] = best ? first : -1;
            if (a.probs) a.probs[row] = best ? 1.f : 0.f;
        }
        mail.cl.sync();
        return;
    }
    const uint32_t bk = (uint32_t)(best >> 32);
    const float top = __uint_as_float(bk & 0x80000000u ? bk & 0x7fffffffu : ~bk);
    const double s = 1.4426950408889634 / (double)p.temperature;
    const bool use_k = p.top_k > 0 && p.top_k < a.vocab, use_p = p.top_p < 1.f;
    const unsigned long long min_w = p.min_p > 0.f ? (unsigned long long)ceil((double)fminf(p.min_p, 1.f) * (double)SV_ONE) : 0;
    // ---- the borders: tokens whose number is below `kappa` are out
    unsigned long long kappa = 0;
    if (use_k || use_p) {
        bool done_k = !use_k, done_p = !use_p;
        unsigned long long held = 0; // mass of the top-k tokens
        for (int level = 0; level < 2 && !(done_k && done_p); level++) {
            // level 0 looks at the likely tokens alone; level 1 at all that weigh something
            const double span = level ? 46.0 : 12.0, per = SV_SMP_BINS / span;
            auto bin_of = [&](double t) { return t > -span ? min((int)(-t * per), SV_SMP_BINS - 1) : -1; };
            for (int i = tid; i < SV_SMP_BINS; i += SV_SMP_THREADS) { sh.count[i] = 0; sh.mass[i] = 0; }
            __syncthreads();
            unsigned long long out = 0;
            for (int i = tid; i < n; i += SV_SMP_THREADS) {
                const double t = sv_log2w(at(i), top, s);
                const int b = bin_of(t);
                if (b >= 0) {
                    atomicAdd(&sh.count[b], 1u);
                    if (use_p) atomicAdd(&sh.mass[b], sv_weight(t));
                } else if (use_p && !use_k) out += sv_weight(t);
            }
            out = sv_block<false>(sh, out);
            mail.cl.sync();
            // a CTA joins its slice of the bins
            const int per_cta = SV_SMP_BINS / C, b0 = rank * per_cta;
            unsigned long long sc = 0, sm = 0;
            for (int b = b0 + tid; b < b0 + per_cta; b += SV_SMP_THREADS) {
                uint32_t c = 0;
                unsigned long long m = 0;
                for (int r = 0; r < C; r++) {
                    const SvSmpShared *o = mail.cl.map_shared_rank(&sh, r);
                    c += o->count[b];
                    m += o->mass[b];
                }
                sh.count[b] = c; // (this slice of this CTA's own bins: nobody else reads it)
                sh.mass[b] = m;
                sc += c;
                sm += m;
            }
            sc = sv_block<false>(sh, sc);
            sm = sv_block<false>(sh, sm);
            unsigned long long slice_c[16], slice_m[16], all_m = 0, win_m = 0, win_c = 0;
            {
                const unsigned long long(*m)[16] = mail.post(sc, sm, out);
                for (int r = 0; r < C; r++) {
                    slice_c[r] = m[0][r]; slice_m[r] = m[1][r];
                    win_c += m[0][r]; win_m += m[1][r]; all_m += m[1][r] + m[2][r];
                }
            }
            if (!use_k) held = all_m;
            for (int which = 0; which < 2; which++) { // top-k, then top-p
                if (which ? done_p || !done_k : done_k) continue;
                const unsigned long long need = which ? max(1ull, (unsigned long long)ceil((double)fmaxf(p.top_p, 0.f) * (double)held)) : (unsigned long long)p.top_k;
                if (need > (which ? win_m : win_c)) {
                    if (level) { // fewer tokens than top_k weigh anything: all of them stay
                        if (!which) held = win_m;
                        if (which) done_p = true; else done_k = true;
                    }
                    continue;
                }
                unsigned long long before = 0, before_m = 0;
                int owner = 0;
                for (; owner < C - 1; owner++) {
                    const unsigned long long v = which ? slice_m[owner] : slice_c[owner];
                    if (need <= before + v) break;
                    before += v;
                    before_m += slice_m[owner];
                }
                // the owner's warp 0 walks its slice
                if (rank == owner && warp == 0) {
                    unsigned long long run = before, run_m = before_m;
                    int hit = -1;
                    for (int b = b0; b < b0 + per_cta && hit < 0; b += 32) {
                        const bool in = b + lane < b0 + per_cta;
                        unsigned long long m = in ? sh.mass[b + lane] : 0, v = which ? m : in ? sh.count[b + lane] : 0, inc = v, inc_m = m;
#pragma unroll
                        for (int o = 1; o < 32; o <<= 1) {
                            const unsigned long long u = __shfl_up_sync(0xffffffffu, inc, o), um = __shfl_up_sync(0xffffffffu, inc_m, o);
                            if (lane >= o) { inc += u; inc_m += um; }
                        }
                        const unsigned ball = __ballot_sync(0xffffffffu, need <= run + inc);
                        if (ball) {
                            const int f = __ffs(ball) - 1;
                            hit = b + f;
                            run += __shfl_sync(0xffffffffu, inc - v, f);
                            run_m += __shfl_sync(0xffffffffu, inc_m - m, f);
                        } else {
                            run += __shfl_sync(0xffffffffu, inc, 31);
                            run_m += __shfl_sync(0xffffffffu, inc_m, 31);
                        }
                    }
                    if (lane == 0) { sh.border[0] = hit; sh.border[1] = run; sh.border[2] = run_m; sh.border[3] = hit >= 0 ? sh.count[hit] : 0; }
                }
                if (tid == 0) sh.n_list = 0;
                __syncthreads();
                unsigned long long bin, in_bin;
                {
                    const unsigned long long(*m)[16] = mail.post(sh.border[0], sh.border[1], sh.border[2], sh.border[3]);
                    bin = m[0][owner]; before = m[1][owner]; before_m = m[2][owner]; in_bin = m[3][owner];
                }
                unsigned long long k_at, m_at; // the border's number, and the mass down to it
                if (in_bin <= SV_SMP_LIST) {
                    SvSmpShared *to = mail.cl.map_shared_rank(&sh, 0);
                    for (int i = tid; i < n; i += SV_SMP_THREADS) {
                        const float x = at(i);
                        if (bin_of(sv_log2w(x, top, s)) == (int)bin) to->list[atomicAdd(&to->n_list, 1u)] = sv_key(x, i0 + i);
                    }
                    mail.cl.sync();
                    if (rank == 0) {
                        sv_sort(sh, (int)in_bin);
                        if (warp == 0) {
                            unsigned long long run = before, run_m = before_m, key = 0;
                            bool found = false;
                            for (int b = 0; b < (int)in_bin && !found; b += 32) {
                                const unsigned long long k = b + lane < (int)in_bin ? sh.list[b + lane] : 0;
                                const uint32_t kb = (uint32_t)(k >> 32);
                                const unsigned long long m = k ? sv_weight(sv_log2w(__uint_as_float(kb & 0x80000000u ? kb & 0x7fffffffu : ~kb), top, s)) : 0, v = which ? m : k != 0;
                                unsigned long long inc = v, inc_m = m;
#pragma unroll
                                for (int o = 1; o < 32; o <<= 1) {
                                    const unsigned long long u = __shfl_up_sync(0xffffffffu, inc, o), um = __shfl_up_sync(0xffffffffu, inc_m, o);
                                    if (lane >= o) { inc += u; inc_m += um; }
                                }
                                const unsigned ball = __ballot_sync(0xffffffffu, need <= run + inc);
                                const int f = ball ? __ffs(ball) - 1 : 31;
                                run += __shfl_sync(0xffffffffu, inc, f);
                                run_m += __shfl_sync(0xffffffffu, inc_m, f);
                                key = __shfl_sync(0xffffffffu, k, f);
                                found = ball != 0;
                            }
                            if (lane == 0) { sh.border[0] = key; sh.border[1] = run_m; }
                        }
                        __syncthreads();
                    }
                    const unsigned long long(*m)[16] = mail.post(sh.border[0], sh.border[1]);
                    k_at = m[0][0];
                    m_at = m[1][0];
                } else { // a bin with thousands of members (equal logits, or nearly): the border's number bit by bit, a sum over the row for each
                    k_at = 0;
                    m_at = 0;
                    for (int bit = 63; bit >= -1; bit--) { // (at -1: the mass down to the number that was found)
                        const unsigned long long probe = bit >= 0 ? k_at | 1ull << bit : k_at;
                        unsigned long long c = 0, m = 0;
                        for (int i = tid; i < n; i += SV_SMP_THREADS) {
                            const float x = at(i);
                            if (x > -INFINITY && sv_key(x, i0 + i) >= probe) {
                                c++;
                                if (which || bit < 0) m += sv_weight(sv_log2w(x, top, s));
                            }
                        }
                        c = sv_block<false>(sh, c);
                        m = sv_block<false>(sh, m);
                        const unsigned long long(*t)[16] = mail.post(c, m);
                        c = m = 0;
                        for (int r = 0; r < C; r++) { c += t[0][r]; m += t[1][r]; }
                        if (bit < 0) m_at = m;
                        else if ((which ? m : c) >= need) k_at = probe;
                    }
                }
                kappa = max(kappa, k_at);
                if (which) done_p = true;
                else { done_k = true; held = m_at; }
            }
        }
    }
    // ---- the kept mass: a warp owns a run of tokens
    const int run = ((n + SV_SMP_THREADS / 32 - 1) / (SV_SMP_THREADS / 32) + 31) & ~31, w0 = min(warp * run, n), w1 = min(w0 + run, n);
    auto mass_at = [&](int i) -> unsigned long long {
        const float x = at(i);
        if (!(x > -INFINITY) || sv_key(x, i0 + i) < kappa) return 0;
        const unsigned long long w = sv_weight(sv_log2w(x, top, s));
        return w >= min_w ? w : 0;
    };
    unsigned long long mine = 0;
    for (int i = w0 + lane; i < w1; i += 32) mine += mass_at(i);
#pragma unroll
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    const unsigned long long block = sv_block<false>(sh, lane == 0 ? mine : 0);
    unsigned long long before = 0, all = 0;
    {
        const unsigned long long(*m)[16] = mail.post(block);
        for (int r = 0; r < C; r++) {
            if (r < rank) before += m[0][r];
            all += m[0][r];
        }
    }
    const float u = a.u[row];
    unsigned long long goal = u > 0.f ? (unsigned long long)((double)fminf(u, 1.f) * (double)all) : 0;
    goal = min(goal, all - 1); // (the largest logit weighs 2^44, so `all` is not zero)
    if (goal >= before && goal < before + block) {
        // (red still holds the warps' masses)
        for (int w = 0; w < warp; w++) before += sh.red[w];
        if (goal >= before && goal < before + mine) {
            for (int i = w0; i < w1; i += 32) {
                const unsigned long long m = i + lane < w1 ? mass_at(i + lane) : 0;
                unsigned long long inc = m;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned long long v = __shfl_up_sync(0xffffffffu, inc, o);
                    if (lane >= o) inc += v;
                }
                const unsigned ball = __ballot_sync(0xffffffffu, goal < before + inc);
                if (ball) {
                    const int f = __ffs(ball) - 1;
                    if (lane == f) {
                        a.ids[row] = i0 + i + lane;
                        if (a.probs) a.probs[row] = (float)((double)m / (double)all);
                    }
                    break;
                }
                before += __shfl_sync(0xffffffffu, inc, 31);
            }
        }
    }
    mail.cl.sync(); // nobody goes while its mail may still be read or written
}
