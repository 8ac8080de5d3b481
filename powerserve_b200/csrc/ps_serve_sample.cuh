// ps_serve_sample.cuh - one token of each row of logits: temperature, top-k, top-p, min-p, and a given random number.
//
// w_i = exp((x_i - max) / T).  The tokens in the order (logit, lower token): the first top_k; of these the shortest beginning that holds top_p of
// their mass; of these the ones with w >= min_p.  The token is the first one, in the vocabulary's order, where the kept tokens' running mass is
// over u times all of it.  A weight is a whole number of 2^-44: sums do not depend on their order, so the result does not depend on the launch.
//
// A cluster of CTAs takes a row and keeps it in shared memory.  What the filters decide, they decide among the likely tokens (log2 w >= -16): these are
// listed first, in order, a list per warp, and the rest of the work looks at the lists alone.  The borders of top-k and top-p are borders of the sorted
// order, which nobody sorts: a histogram over log2 w (counts and masses) finds the bin that a border lies in, its few members are gathered and sorted, and
// the border becomes a number (logit, token) to compare with.  Rows whose lists do not fit, or whose border lies below (flat ones), go the same way over all of
// their tokens.  No filter: the running mass over all tokens.
// Bound by latency: a row is four to seven exchanges across its cluster, and two CTAs an SM hide little of one another's; then by the 45-bit exponentials, which top-p needs of all tokens
// (64-bit arithmetic: borders would move with float32's). In a captured graph, one row of 151 936: largest logit 5.3 us, min-p 9, top-p with min-p 10, no filter 11, top-k 40 with top-p 16, top-p alone 31;
// 64 rows of 128 256: 15, 25, 30, 40, 35, 98; 256 rows of 151 936: 67 (2.3 TB/s), 103, 128, 149, 121, 404. Flat rows (their border is below 2^-16 of the largest) 48 / 168 / 696.
#pragma once
#include "ps_ptx.cuh"

#include <cooperative_groups.h>

#define SV_SMP_THREADS 512
#define SV_SMP_BINS 1024
#define SV_SMP_CAP 512      // tokens of a warp's list
#define SV_SMP_OVER (1u << 20) // said of a list that did not fit; more than all others together
#define SV_SMP_SPAN 16.0    // log2 of the least weight that is listed, negative
#define SV_ONE (1ull << 44)

// What the settings leave of a row: its tokens of which the number sv_key is at least kappa and the weight at least min_p, and their mass (0: one token alone, `only`; -1: none)
struct alignas(16) SvRowStats {
    unsigned long long kappa, all;
    float top;
    int only;
};
struct SvSample {
    const float *logits;
    const ps_cuda_sampler *samplers;
    const float *u;
    int32_t *ids;
    float *probs;
    int64_t row_stride;
    int vocab, chunk;       // tokens; tokens of a CTA
    int vec;                // rows begin at 16-byte boundaries
    SvRowStats *stats;      // sv_sample<true>: what is left of a row is asked for, no token
};
struct alignas(16) SvSmpShared { // (the logits lie behind it, read and written sixteen bytes at a time)
    union {
        unsigned long long mass[SV_SMP_BINS]; // this CTA's share of the bins' masses; when those are added up:
        unsigned long long list[SV_SMP_BINS]; // members of a border's bin
    };
    unsigned long long own_mass[SV_SMP_BINS / 8], mail[2][4][16], red[32], border[4];
    double pow2[32];                          // 2^(i / 32)
    uint32_t count[SV_SMP_BINS], own_count[SV_SMP_BINS / 8], warp_listed[SV_SMP_THREADS / 32], warp_most[SV_SMP_THREADS / 32], n_list; // own: the row's, of the bins that are this CTA's
    alignas(16) uint16_t lists[SV_SMP_THREADS / 32][SV_SMP_CAP]; // places of the likely tokens among the CTA's
};
static_assert(sizeof(SvSmpShared) % 16 == 0, "the logits behind it");

PS_D uint32_t sv_rank(float x) { // larger logit, larger number (both zeros are one); above zero but for no number at all
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
PS_D float sv_unrank(uint32_t b) { return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b); }
PS_D unsigned long long sv_key(float x, int i) { return (unsigned long long)sv_rank(x) << 32 | (uint32_t)~i; } // (logit, lower token first) as a number
PS_D float sv_logit(unsigned long long key) { return sv_unrank((uint32_t)(key >> 32)); }
// log2 of a weight
struct SvScale {
    float top;
    double s, off;          // log2 e / temperature; -top times it
    PS_D double operator()(float x) const { return x == top ? 0.0 : fma((double)x, s, off); } // (x is a number above -inf)
};
// 2^t as a whole number of 2^-44: 2^t = 2^n 2^(j / 32) 2^r, |r| <= 1/64, the last by the exponential's series to the fifth power (the sixth is below 2^-48).
// Without branches, so that several are under way at once: one alone takes 300 cycles
PS_D unsigned long long sv_weight(const double *pow2, double t) {
    const double magic = 211106232532992.0;        // 1.5 2^47: its last bit is 1/32
    const double z = t + magic;
    const int j = __double2loint(z);
    const double r = t - (z - magic);
    double p = fma(r, 1.3333558146428443e-3, 9.618129107628477e-3); // ln2^5 / 120, ln2^4 / 24
    p = fma(p, r, 5.5504108664821580e-2);
    p = fma(p, r, 2.4022650695910072e-1);
    p = fma(p, r, 6.9314718055994531e-1);
    const double b = pow2[j & 31];
    const double w = fma(p * r, b, b);
    const double big = __hiloint2double(__double2hiint(w) + (((j >> 5) + 44) << 20), __double2loint(w));
    const unsigned long long n = (unsigned long long)__double_as_longlong(big + 4503599627370496.0) & 0xfffffffffffffull; // (2^52: the sum's mantissa is the whole number)
    return (uint32_t)__double2hiint(t) < 0xc0470000u ? n : 0; // above -46
}
PS_D unsigned long long sv_weight(const SvSmpShared &sh, double t) { return sv_weight(sh.pow2, t); }
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

// sorts n numbers, largest first (there is room for the next power of two)
PS_D void sv_sort(unsigned long long *list, int n) {
    int p2 = 2;
    while (p2 < n) p2 *= 2;
    for (int i = n + threadIdx.x; i < p2; i += SV_SMP_THREADS) list[i] = 0;
    __syncthreads();
    for (int k = 2; k <= p2; k *= 2)
        for (int j = k / 2; j; j /= 2) {
            for (int i = threadIdx.x; i < p2 / 2; i += SV_SMP_THREADS) {
                const int lo = (i / j) * 2 * j + i % j, hi = lo + j;
                const unsigned long long x = list[lo], y = list[hi];
                if ((x < y) == ((lo & k) == 0)) { list[lo] = y; list[hi] = x; }
            }
            __syncthreads();
        }
}

// what the parts of the kernel share about a row
struct SvSmpRow {
    SvScale log2w;
    ps_cuda_sampler p;
    unsigned long long min_w;
    float cut, low;                     // logits below `cut` are not listed; the least that counts
    int vocab, i0, n, w0, w1, listed;   // w0 .. w1: the warp's tokens; listed: of them in its list
    bool use_k, use_p;
};
// f(logit, number) of the CTA's tokens: the listed ones, or all
template <bool LIST, typename F> PS_D void sv_each(const SvSmpRow &r, const SvSmpShared &sh, const float *x, F f) {
    const int lane = threadIdx.x & 31;
    const uint16_t *l = sh.lists[threadIdx.x >> 5];
    const int from = LIST ? lane : r.w0 + lane, to = LIST ? r.listed : r.w1;
#pragma unroll 4
    for (int i = from; i < to; i += 32) {
        const int at = LIST ? l[i] : i;
        const float v = x[at];
        if (LIST || v > -INFINITY) f(v, sv_key(v, r.i0 + at));
    }
}
// the mass of all tokens of the warp
PS_D unsigned long long sv_all(const SvSmpRow &r, const SvSmpShared &sh, const float *x) {
    unsigned long long sum = 0;
    for (int i = r.w0 + (threadIdx.x & 31); i < r.w1; i += 128) {
        unsigned long long w[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float v = i + 32 * e < r.w1 ? x[i + 32 * e] : -INFINITY;
            w[e] = sv_weight(sh, r.log2w(v));
            if (!(v > -INFINITY)) w[e] = 0;
        }
        sum += w[0] + w[1] + w[2] + w[3];
    }
    return sum;
}

// The borders: tokens whose number is below `kappa` are out.  LIST: false if the lists do not decide.  `whole`: the mass of all
template <bool LIST> PS_D bool sv_borders(const SvSmpRow &r, SvSmpShared &sh, SvMail &mail, const float *x, unsigned long long whole, unsigned long long &kappa) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = mail.rank, C = mail.size;
    bool done_k = !r.use_k, done_p = !r.use_p;
    unsigned long long held = whole; // mass of the top-k tokens
    kappa = 0;
    const float low = LIST ? r.cut : r.low, per = r.log2w.top > low ? (float)SV_SMP_BINS / (r.log2w.top - low) : 0.f;
    auto bin_of = [&](float v) { return min((int)((r.log2w.top - v) * per), SV_SMP_BINS - 1); }; // (a larger logit is never in a later bin)
    const int per_cta = SV_SMP_BINS / C, b0 = rank * per_cta;
    if (!LIST) {                 // (the lists' sums are in the way)
        mail.cl.sync();
        for (int i = tid; i < SV_SMP_BINS; i += SV_SMP_THREADS) { sh.count[i] = 0; sh.mass[i] = 0; }
        for (int i = tid; i < per_cta; i += SV_SMP_THREADS) { sh.own_count[i] = 0; sh.own_mass[i] = 0; }
        mail.cl.sync();
    }
    sv_each<LIST>(r, sh, x, [&](float v, unsigned long long) {
        if (LIST || v >= low) {
            const int b = bin_of(v);
            atomicAdd(&sh.count[b], 1u);
            if (r.use_p) atomicAdd(&sh.mass[b], sv_weight(sh, r.log2w(v)));
        }
    });
    __syncthreads();
    // to the CTAs that own the bins
    for (int i = tid; i < SV_SMP_BINS; i += SV_SMP_THREADS)
        if (const uint32_t c = sh.count[i]) {
            SvSmpShared *to = mail.cl.map_shared_rank(&sh, i / per_cta);
            atomicAdd(&to->own_count[i % per_cta], c);
            if (r.use_p) atomicAdd(&to->own_mass[i % per_cta], sh.mass[i]);
        }
    mail.cl.sync();
    unsigned long long sc = 0, sm = 0;
    if (tid < per_cta) { sc = sh.own_count[tid]; sm = sh.own_mass[tid]; }
    sc = sv_block<false>(sh, sc);
    if (r.use_p) sm = sv_block<false>(sh, sm);
    unsigned long long win_m = 0, win_c = 0;
    unsigned long long slices[2][16]; // (the mail is overwritten before the second border is looked for)
    {
        const unsigned long long(*slice)[16] = mail.post(sc, sm);
#pragma unroll
        for (int o = 0; o < 16; o++) {
            slices[0][o] = o < C ? slice[0][o] : 0;
            slices[1][o] = o < C ? slice[1][o] : 0;
            win_c += slices[0][o]; win_m += slices[1][o];
        }
    }
    for (int which = 0; which < 2; which++) { // top-k, then top-p
        if (which ? done_p || !done_k : done_k) continue;
        const unsigned long long need = which ? max(1ull, (unsigned long long)ceil((double)fmaxf(r.p.top_p, 0.f) * (double)held)) : (unsigned long long)r.p.top_k;
        if (need > (which ? win_m : win_c)) {
            if (LIST) { // the border lies among what is not listed.  Where min-p takes all of that out, it decides nothing
                if (r.min_w < SV_ONE >> (int)SV_SMP_SPAN || (!which && r.use_p)) return false;
            } else if (!which) held = win_m; // fewer tokens than top_k weigh anything: all of them stay
            if (which) done_p = true; else done_k = true;
            continue;
        }
        unsigned long long before = 0, before_m = 0;
        int owner = 0;
        bool there = false;
#pragma unroll
        for (int o = 0; o < 16; o++) {
            const unsigned long long v = slices[which][o];
            there |= need <= before + v;
            if (!there) { before += v; before_m += slices[1][o]; owner++; }
        }
        // the owner's warp 0 walks its slice
        if (rank == owner && warp == 0) {
            unsigned long long run = before, run_m = before_m;
            int hit = -1;
            for (int b = 0; b < per_cta && hit < 0; b += 32) {
                const unsigned long long m = sh.own_mass[b + lane], v = which ? m : sh.own_count[b + lane];
                unsigned long long inc = v, inc_m = m;
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
            if (lane == 0) { sh.border[0] = b0 + hit; sh.border[1] = run; sh.border[2] = run_m; sh.border[3] = hit >= 0 ? sh.own_count[hit] : 0; }
        }
        if (tid == 0) sh.n_list = 0;
        __syncthreads();
        unsigned long long bin, in_bin;
        {
            const unsigned long long(*m)[16] = mail.post(sh.border[0], sh.border[1], sh.border[2], sh.border[3]);
            bin = m[0][owner]; before = m[1][owner]; before_m = m[2][owner]; in_bin = m[3][owner];
        }
        unsigned long long k_at, m_at; // the border's number, and the mass down to it
        if (in_bin <= SV_SMP_BINS) {
            SvSmpShared *to = mail.cl.map_shared_rank(&sh, 0);
            sv_each<LIST>(r, sh, x, [&](float v, unsigned long long key) {
                if ((LIST || v >= low) && bin_of(v) == (int)bin) to->list[atomicAdd(&to->n_list, 1u)] = key;
            });
            mail.cl.sync();
            if (rank == 0) {
                sv_sort(sh.list, (int)in_bin);
                if (warp == 0) {
                    unsigned long long run = before, run_m = before_m, key = 0;
                    bool found = false;
                    for (int b = 0; b < (int)in_bin && !found; b += 32) {
                        const unsigned long long k = b + lane < (int)in_bin ? sh.list[b + lane] : 0;
                        const unsigned long long m = k ? sv_weight(sh, r.log2w(sv_logit(k))) : 0, v = which ? m : k != 0;
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
        } else { // a bin with thousands of members (equal logits, or nearly): the border's number bit by bit, a sum over the members for each, from the first bit that they differ in
            unsigned long long hi = 0, lo = ~0ull;
            auto members = [&](auto f) {
                sv_each<LIST>(r, sh, x, [&](float v, unsigned long long key) {
                    if ((LIST || v >= low) && bin_of(v) == (int)bin) f(v, key);
                });
            };
            members([&](float, unsigned long long key) { hi = max(hi, key); lo = min(lo, key); });
            hi = sv_block<true>(sh, hi);
            lo = ~sv_block<true>(sh, ~lo);
            {
                const unsigned long long(*m)[16] = mail.post(hi, lo);
                for (int o = 0; o < C; o++) { hi = max(hi, m[0][o]); lo = min(lo, m[1][o]); }
            }
            const int first = hi == lo ? -1 : 63 - __clzll(hi ^ lo);
            k_at = first < 0 ? hi : first == 63 ? 0 : hi >> (first + 1) << (first + 1);
            m_at = 0;
            for (int bit = first; bit >= -1; bit--) { // (at -1: the mass down to the number that was found)
                const unsigned long long probe = bit >= 0 ? k_at | 1ull << bit : k_at;
                unsigned long long c = 0, m = 0;
                members([&](float v, unsigned long long key) {
                    if (key >= probe) {
                        c++;
                        if (which || bit < 0) m += sv_weight(sh, r.log2w(v));
                    }
                });
                c = sv_block<false>(sh, c);
                m = sv_block<false>(sh, m);
                const unsigned long long(*t)[16] = mail.post(c, m);
                c = which ? before_m : before;
                m = before_m;
                for (int o = 0; o < C; o++) { c += t[which][o]; m += t[1][o]; }
                if (bit < 0) m_at = m;
                else if (c >= need) k_at = probe;
            }
        }
        kappa = max(kappa, k_at);
        if (which) done_p = true;
        else { done_k = true; held = m_at; }
    }
    return true;
}

// the token: the warps' kept masses, and in the warp where u times all of them falls its tokens in order
template <bool LIST, bool STATS> PS_D void sv_pick(const SvSample &a, int64_t row, const SvSmpRow &r, SvSmpShared &sh, SvMail &mail, const float *x, unsigned long long kappa, bool filters) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto mass_of = [&](float v, unsigned long long key) -> unsigned long long {
        if (key < kappa) return 0;
        const unsigned long long w = sv_weight(sh, r.log2w(v));
        return w >= r.min_w ? w : 0;
    };
    unsigned long long mine = 0;
    if (!LIST && !filters) mine = sv_all(r, sh, x);
    else sv_each<LIST>(r, sh, x, [&](float v, unsigned long long key) { mine += mass_of(v, key); });
#pragma unroll
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    const unsigned long long block = sv_block<false>(sh, lane == 0 ? mine : 0);
    unsigned long long before = 0, all = 0;
    {
        const unsigned long long(*m)[16] = mail.post(block);
        for (int o = 0; o < mail.size; o++) {
            if (o < mail.rank) before += m[0][o];
            all += m[0][o];
        }
    }
    if (STATS) {
        if (mail.rank == 0 && threadIdx.x == 0) a.stats[row] = SvRowStats{kappa, all, r.log2w.top, 0};
        return;
    }
    const float u = a.u[row];
    unsigned long long goal = u > 0.f ? (unsigned long long)((double)fminf(u, 1.f) * (double)all) : 0;
    goal = min(goal, all - 1); // (the largest logit weighs 2^44, so `all` is not zero)
    if (goal < before || goal >= before + block) return;
    for (int w = 0; w < warp; w++) before += sh.red[w]; // (they still hold the warps' masses)
    if (goal < before || goal >= before + mine) return;
    const int from = LIST ? 0 : r.w0, to = LIST ? r.listed : r.w1;
    constexpr int W = LIST ? 1 : 2; // weights under way at a time (lists are short; four cost registers: 64 rows of mixed settings 70 us, 67 with two, 64 without filters 40 and 41, with one 45)
    for (int i = from; i < to; i += 32 * W) {
        unsigned long long m[W], key[W], sum = 0;
#pragma unroll
        for (int e = 0; e < W; e++) {
            const int n = i + 32 * e + lane, at = n < to ? LIST ? sh.lists[warp][n] : n : -1;
            const float v = at >= 0 ? x[at] : -INFINITY;
            key[e] = sv_key(v, r.i0 + at);
            m[e] = mass_of(v, key[e]);
            if (!(v > -INFINITY)) m[e] = 0;
            sum += m[e];
        }
        if (W > 1) {
#pragma unroll
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (goal >= before + sum) { before += sum; continue; }
        }
#pragma unroll
        for (int e = 0; e < W; e++) {
            unsigned long long inc = m[e];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned long long v2 = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += v2;
            }
            const unsigned ball = __ballot_sync(0xffffffffu, goal < before + inc);
            if (ball) {
                if (lane == __ffs(ball) - 1) {
                    a.ids[row] = (int)~(uint32_t)key[e];
                    if (a.probs) a.probs[row] = (float)((double)m[e] / (double)all);
                }
                return;
            }
            before += __shfl_sync(0xffffffffu, inc, 31);
        }
    }
}

// sum of v over the block's threads before this one, and over all
PS_D unsigned long long sv_before(SvSmpShared &sh, unsigned long long v, unsigned long long &all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
    }
    __syncthreads();
    if (lane == 31) sh.red[warp] = inc;
    __syncthreads();
    unsigned long long base = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < SV_SMP_THREADS / 32; w++) {
        if (w < warp) base += sh.red[w];
        all += sh.red[w];
    }
    return base + inc - v;
}

// Few tokens are listed: one CTA has them all in sh.list, in the vocabulary's order, and goes on alone
template <bool STATS> PS_D void sv_few(const SvSample &a, int64_t row, const SvSmpRow &r, SvSmpShared &sh, int n, unsigned long long held) {
    const int tid = threadIdx.x;
    unsigned long long kappa = 0, all, mine[2], key[2];
    if (r.use_k || r.use_p) {
        unsigned long long *sorted = reinterpret_cast<unsigned long long *>(sh.lists);
        for (int i = tid; i < n; i += SV_SMP_THREADS) sorted[i] = sh.list[i];
        sv_sort(sorted, n);
        unsigned long long sum = 0;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            key[e] = 2 * tid + e < n ? sorted[2 * tid + e] : 0;
            mine[e] = key[e] ? sv_weight(sh, r.log2w(sv_logit(key[e]))) : 0;
            sum += mine[e];
        }
        unsigned long long before = sv_before(sh, sum, all);
        int keep = n;
        if (r.use_k && r.p.top_k < n) {
            keep = r.p.top_k;
            if (tid == (keep - 1) / 2) sh.border[0] = before + mine[0] + ((keep - 1) & 1 ? mine[1] : 0);
            __syncthreads();
            held = sh.border[0];
        } else if (r.use_k) held = all;
        if (tid == 0) sh.border[1] = sorted[keep - 1];
        __syncthreads();
        if (r.use_p) { // the first token down to which the mass is enough; none: min-p takes out all that is not listed
            const unsigned long long need = max(1ull, (unsigned long long)ceil((double)fmaxf(r.p.top_p, 0.f) * (double)held));
#pragma unroll
            for (int e = 0; e < 2; e++) {
                if (need > before && need <= before + mine[e] && 2 * tid + e < keep) sh.border[1] = key[e];
                before += mine[e];
            }
            __syncthreads();
        }
        kappa = sh.border[1];
    }
    unsigned long long sum = 0;
#pragma unroll
    for (int e = 0; e < 2; e++) {
        key[e] = 2 * tid + e < n ? sh.list[2 * tid + e] : 0;
        mine[e] = key[e] && key[e] >= kappa ? sv_weight(sh, r.log2w(sv_logit(key[e]))) : 0;
        if (mine[e] < r.min_w) mine[e] = 0;
        sum += mine[e];
    }
    unsigned long long before = sv_before(sh, sum, all);
    if (STATS) {
        if (tid == 0) a.stats[row] = SvRowStats{kappa, all, r.log2w.top, 0};
        return;
    }
    const float u = a.u[row];
    unsigned long long goal = u > 0.f ? (unsigned long long)((double)fminf(u, 1.f) * (double)all) : 0;
    goal = min(goal, all - 1);
#pragma unroll
    for (int e = 0; e < 2; e++) {
        if (goal >= before && goal < before + mine[e]) {
            a.ids[row] = (int)~(uint32_t)key[e];
            if (a.probs) a.probs[row] = (float)((double)mine[e] / (double)all);
        }
        before += mine[e];
    }
}

// what a row's settings ask for, once its largest logit is known (r.log2w.top); floor: the least one; reach: a number that top_k logits reach, or 0
PS_D void sv_settings(SvSmpRow &r, float floor, uint32_t reach) {
    r.log2w.s = 1.4426950408889634 / (double)r.p.temperature;
    r.log2w.off = -(double)r.log2w.top * r.log2w.s;
    if (r.log2w.top == INFINITY) { r.log2w.s = 0.0; r.log2w.off = -INFINITY; } // (all others weigh nothing)
    r.use_k = r.p.top_k > 0 && r.p.top_k < r.vocab;
    r.use_p = r.p.top_p < 1.f;
    r.min_w = r.p.min_p > 0.f ? (unsigned long long)ceil((double)fminf(r.p.min_p, 1.f) * (double)SV_ONE) : 0;
    // what lies `span` below the top in log2 w (and what a weight's rounding to 2^-44 takes for it), rounded outwards
    auto down = [&](double span) { return r.log2w.s > 0.0 ? __double2float_rd((double)r.log2w.top - (span + 1e-8) / r.log2w.s) : -INFINITY; };
    r.low = fmaxf(down(46.0), floor);
    // (what weighs less than min_p goes in the end: it need not be listed, unless top-p asks for the mass of the top_k)
    r.cut = fmaxf(down(r.min_w >= SV_ONE >> (int)SV_SMP_SPAN && !(r.use_k && r.use_p) ? -log2((double)fminf(r.p.min_p, 1.f)) : SV_SMP_SPAN), floor);
    if (r.use_k && reach) r.cut = fmaxf(r.min_w >= SV_ONE >> (int)SV_SMP_SPAN && !r.use_p ? r.cut : floor, sv_unrank(reach));
}
// STATS: for the verification of drafted tokens, what the settings leave of the row
template <bool STATS> PS_D void sv_sample(const SvSample &a, int64_t row) {
    extern __shared__ __align__(16) uint8_t sv_smp_raw[];
    SvSmpShared &sh = *reinterpret_cast<SvSmpShared *>(sv_smp_raw);
    float *x = reinterpret_cast<float *>(sv_smp_raw + sizeof(SvSmpShared));
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    SvMail mail(sh);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, C = mail.size;
    const float *from = a.logits + row * a.row_stride;
    SvSmpRow r;
    r.vocab = a.vocab;
    r.i0 = min(mail.rank * a.chunk, a.vocab);
    r.n = min(a.chunk, a.vocab - r.i0);
    // ---- the largest logit and the lowest token that has it, and the least; no number becomes -inf
    float most = -INFINITY, least = INFINITY;
    auto take = [&](float v) {
        v = v == v ? v : -INFINITY;
        most = fmaxf(most, v);
        least = fminf(least, v > -INFINITY ? v : INFINITY);
        return v;
    };
    const int n4 = a.vec ? r.n / 4 : 0;
#pragma unroll 4
    for (int i = tid; i < n4; i += SV_SMP_THREADS) {
        float4 v = __ldcs(reinterpret_cast<const float4 *>(from + r.i0) + i);
        v.x = take(v.x); v.y = take(v.y); v.z = take(v.z); v.w = take(v.w);
        reinterpret_cast<float4 *>(x)[i] = v;
    }
#pragma unroll 4
    for (int i = 4 * n4 + tid; i < r.n; i += SV_SMP_THREADS) x[i] = take(from[r.i0 + i]);
    if (tid < 32) sh.pow2[tid] = exp2(tid / 32.0);
    for (int i = tid; i < SV_SMP_BINS; i += SV_SMP_THREADS) { sh.count[i] = 0; sh.mass[i] = 0; }
    if (tid < SV_SMP_BINS / 8) { sh.own_count[tid] = 0; sh.own_mass[tid] = 0; }
    r.p = a.samplers[row];
    // (which token it is only a greedy row asks)
    uint32_t best = most > -INFINITY ? sv_rank(most) : 0, worst = sv_rank(least);
    const uint32_t mine = best;
    best = __reduce_max_sync(0xffffffffu, best);
    worst = __reduce_min_sync(0xffffffffu, worst);
    if (lane == 0) { sh.warp_most[warp] = best; sh.warp_listed[warp] = worst; }
    __syncthreads();
    const uint32_t of_warp = sh.warp_most[lane & 15];
    best = __reduce_max_sync(0xffffffffu, of_warp);
    worst = __reduce_min_sync(0xffffffffu, sh.warp_listed[lane & 15]);
    // A bound on the top_k: the CTA's j-th largest warp maximum (or thread maximum, where top_k is larger), j = top_k / C, is one that j of its tokens reach, so
    // that what lies below all CTAs' is not among the top_k
    const int jth = r.p.top_k < a.vocab ? (r.p.top_k + C - 1) / C : 0;
    uint32_t reach = 0;
    if (jth >= 1 && jth <= SV_SMP_THREADS / 32) {
        int above = 0;
#pragma unroll
        for (int w = 0; w < SV_SMP_THREADS / 32; w++) above += sh.warp_most[w] > of_warp || (sh.warp_most[w] == of_warp && w < (lane & 15));
        reach = __shfl_sync(0xffffffffu, of_warp, __ffs(__ballot_sync(0xffffffffu, above == jth - 1)) - 1);
    } else if (jth >= 1 && jth <= SV_SMP_THREADS) {
        unsigned long long *sorted = reinterpret_cast<unsigned long long *>(sh.lists);
        sorted[tid] = mine;
        sv_sort(sorted, SV_SMP_THREADS);
        reach = (uint32_t)sorted[jth - 1];
        __syncthreads();
    }
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); // (all CTAs are there)
    {
        const unsigned long long(*m)[16] = mail.post(best, worst, reach);
        for (int o = 0; o < C; o++) { best = max(best, (uint32_t)m[0][o]); worst = min(worst, (uint32_t)m[1][o]); reach = min(reach, (uint32_t)m[2][o]); }
    }
    r.log2w.top = sv_unrank(best);
    if (best == 0 || !(r.p.temperature > 0.f)) {
        uint32_t at = 0xffffffffu;
        if (best)
            for (int i = tid; i < r.n; i += SV_SMP_THREADS)
                if (x[i] == r.log2w.top) at = min(at, (uint32_t)(r.i0 + i));
        const unsigned long long(*m)[16] = mail.post(sv_block<true>(sh, ~at));
        uint32_t most_not = 0;
        for (int o = 0; o < C; o++) most_not = max(most_not, (uint32_t)m[0][o]);
        if (mail.rank == 0 && tid == 0) {
            if (STATS) a.stats[row] = SvRowStats{0, 0, r.log2w.top, best ? (int)~most_not : -1};
            else {
                a.ids[row] = best ? (int)~most_not : -1;
                if (a.probs) a.probs[row] = best ? 1.f : 0.f;
            }
        }
        return; // (after the last barrier a CTA looks at its own memory alone)
    }
    sv_settings(r, sv_unrank(worst), reach);
    const int run = ((r.n + SV_SMP_THREADS / 32 - 1) / (SV_SMP_THREADS / 32) + 31) & ~31;
    r.w0 = min(warp * run, r.n);
    r.w1 = min(r.w0 + run, r.n);
    r.listed = 0;
    unsigned long long kappa = 0;
    const bool filters = r.use_k || r.use_p || r.min_w;
    bool listed = false;
    if (filters) {
        const bool least = r.min_w >= SV_ONE >> (int)SV_SMP_SPAN; // min-p takes out all that is not listed
        unsigned long long whole = 0;
        // Top-p needs the mass of all.  Beside such a min-p it is enough, nearly always, to know it to a thousandth: where what min-p leaves is less than top_p of it,
        // top-p takes out nothing more
        bool roughly = r.use_p && !r.use_k && least;
        const bool exactly = r.use_p && !r.use_k && !least;
        const float rs = (float)r.log2w.s;
        float rough = 0.f, rough_in = 0.f;
        if (exactly) whole = sv_block<false>(sh, sv_all(r, sh, x));
        for (int i = r.w0; i < r.w1; i += 128) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = i + 32 * e + lane < r.w1 ? x[i + 32 * e + lane] : -INFINITY;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const bool in = v[e] >= r.cut && v[e] > -INFINITY;
                const unsigned ball = __ballot_sync(0xffffffffu, in);
                const int at = r.listed + __popc(ball & ((1u << lane) - 1));
                if (in && at < SV_SMP_CAP) sh.lists[warp][at] = (uint16_t)(i + 32 * e + lane);
                r.listed += __popc(ball);
            }
            if (roughly)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float w;
                    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"((v[e] - r.log2w.top) * rs));
                    rough += w;
                    rough_in += v[e] >= r.cut ? w : 0.f;
                }
        }
        const bool over = r.listed > SV_SMP_CAP;
        if (over) r.listed = SV_SMP_CAP;
        if (lane == 0) sh.warp_listed[warp] = over ? SV_SMP_OVER : r.listed;
        __syncthreads();
        uint32_t at = 0, cta = 0;
#pragma unroll
        for (int w = 0; w < SV_SMP_THREADS / 32; w++) {
            if (w < warp) at += sh.warp_listed[w];
            cta += sh.warp_listed[w];
        }
        uint32_t total = 0;
        bool over_any = false;
        {
            unsigned long long in = 0;
            if (roughly) { // (no number, as with an infinite logit: the exact mass is asked for.  Masses are below 2^43, and sixteen times 2^59 fits 64 bits)
                whole = sv_block<false>(sh, (unsigned long long)(rough * 16777216.f));
                in = sv_block<false>(sh, (unsigned long long)(rough_in * 16777216.f) + 1);
                const bool odd = __syncthreads_or(!(rough < 1e9f)) != 0;
                if (odd) { in = 1ull << 59; whole = 0; }
            }
            const unsigned long long(*m)[16] = mail.post(cta, whole, in);
            unsigned long long all_in = 0;
            whole = 0;
            for (int o = 0; o < C; o++) {
                if (o < mail.rank) at += (uint32_t)m[0][o];
                total += (uint32_t)m[0][o];
                over_any |= m[0][o] >= SV_SMP_OVER;
                whole += m[1][o];
                all_in += m[2][o];
            }
            if (roughly) {
                if (1.002 * (double)all_in < (double)fmaxf(r.p.top_p, 0.f) * (double)whole) r.use_p = false;
                else {
                    const unsigned long long mine = sv_block<false>(sh, sv_all(r, sh, x));
                    const unsigned long long(*n)[16] = mail.post(mine);
                    whole = 0;
                    for (int o = 0; o < C; o++) whole += n[0][o];
                }
            }
        }
        const bool known = r.use_k ? total >= (uint32_t)r.p.top_k || (least && !r.use_p) : least; // what the filters leave is listed, and the mass that top-p asks for known
        if (known && total <= SV_SMP_BINS) {
            SvSmpShared *to = mail.cl.map_shared_rank(&sh, 0);
            for (int i = lane; i < r.listed; i += 32) {
                const int l = sh.lists[warp][i];
                to->list[at + i] = sv_key(x[l], r.i0 + l);
            }
            mail.cl.sync();
            if (mail.rank == 0) sv_few<STATS>(a, row, r, sh, (int)total, whole);
            return; // (nobody's memory is asked for any more)
        }
        listed = !over_any && (r.use_k || r.use_p ? sv_borders<true>(r, sh, mail, x, whole, kappa) : least);
        if (!listed && (r.use_k || r.use_p)) sv_borders<false>(r, sh, mail, x, whole, kappa);
    }
    if (listed) sv_pick<true, STATS>(a, row, r, sh, mail, x, kappa, filters);
    else sv_pick<false, STATS>(a, row, r, sh, mail, x, kappa, filters);
}
__global__ void __launch_bounds__(SV_SMP_THREADS, 2) sv_k_sample(const __grid_constant__ SvSample a) { sv_sample<false>(a, blockIdx.x / cooperative_groups::this_cluster().num_blocks()); }
