// ps_page_attn.cuh - attention of a step's tokens over caches in 8 bits and in pages, on the fifth-generation tensor cores' whole numbers.
//
//   z[t][h][j] = scale q[t][h] . k[j][g(h)],   p = soft-max over the slots j that token t sees,   out[t][h] = sum_j p[t][h][j] v[g(h)][j]
//
// The codes are the operand as they lie in the pages: nothing is converted.  What meets them is cut into digits of eight bits, lowest first.  A query row is a whole number of 24 bits times a
// factor of its own, three signed digits; a weight times its slot's V scale over the tile's largest is one of 23 bits, three digits without a sign.  The products and their sums are exact (32 bits: 2^7 2^7 256
// channels, 2^8 2^7 128 slots), and the digits' sums are put together in float32.  Digits are columns of the product, so three of them cost no more instructions than a wider N does.
//
// The cache is the MMAs' M side: scores^T[128 slots][rows x digits] = K Q^T, then out^T[channels][rows x digits] = V^T P^T, a lane of tensor memory a slot, then a channel.  A thread of the soft-max has a slot,
// so its scales are its own, the row's largest score is a reduction over the warp (redux) and over four warps (an atomic of shared memory); a weight's digits are three bytes stored.  A thread of the
// output has a channel: it adds a tile's sums to what it holds, so the accumulator sees one tile alone, and tiles have factors and references of their own.
//
// A CTA takes a run of tiles (128 slots of one kv head and up to RT of its query rows), from one sequence and head into the next: all CTAs have the same number of tiles, whatever the sequences' lengths.  A run that does
// not have all tiles of its rows leaves the sums in the workspace, and pg_k_join joins them.  Rows above RT are other CTAs', which take the same tiles at the same time (L2).
// Roles: soft-max (SG groups of four warps, tiles in turn), output (OG groups of four, likewise), and a warp each for copies (a page's K or V of a head is one run of bytes), the MMAs of either product, scales and live
// slots, and queries.  One row a head: 64 sequences of up to 2 040 slots, 8 heads of 128, 33 us + 6 of pg_k_join: 5.5 TB/s while tiles stream, the rest is the CTAs' start and end.  32 rows: 2 x 32 tokens over 32 700 slots
// 112 + 6: bound by the soft-max's instructions and waits (1 650 cycles for 128 slots x 32 rows), matrix pipe 22 %; three soft-max and two output groups, two and one take a tenth more, either one alone no better.  (At the
// 72 registers of 32 rows, 24 bytes a thread lie in local memory.)
// Weights under a tile's own reference cost 4 us of the 112, against those under the row's largest score so far, which lose bits behind a heavy slot.
#pragma once
#include "ps_page.cuh"

#define PG_TILE 128
#define PG_STAGES 8         // at most, of K's ring and of V's
#define PG_LANES 512        // runs of row tiles at most: 256 tokens of 32 heads, 16 rows a tile
#define PG_META 8
#define PG_LOW (-3.4028234663852886e38f) // below every score
#define PG_ONE 8388600.f    // a weight of 1 in whole numbers: 2^23 less what an exponential may be above 1
#define PG_Q_ONE 8355711.f  // 127 (2^16 + 2^8 + 1)

struct PgAttnSeq {
    const int32_t *table;
    const uint8_t *hidden, *mask;
    int n_kv, n_tok, tok0, tiles;
};
struct PgAttn {
    PgAttnSeq seq[PG_SEQS];
    int tile0[PG_SEQS + 1];     // tiles of all heads before a sequence; those with more rows come first, so a run of row tiles takes the sequences up to some one
    int lane_cta0[PG_LANES + 1], lane_tiles[PG_LANES];
    PgPool pool;
    const void *q;
    void *out;
    float *part;                // [CTA][2][RT][hs], then [CTA][2][RT] pairs of reference and sum
    int n_seqs, n_lanes, n_ctas, n_heads, R, stages, bf16, q_vec;
    int whole;                  // a CTA takes the tiles of one sequence and head, all of them: nothing is left to join
    float scale;                // times log2 e
};
PS_D bool pg_sees(const PgAttnSeq &s, int t, int back) { return back < 0 || (s.mask ? s.mask[t * s.n_tok + back] != 0 : back <= t); }
PS_HD int pg_run(int tiles, int n, int k) { const int r = tiles % n; return tiles / n * k + (k < r ? k : r); } // where run k of n begins: the first ones have a tile more

template <int RT_, int MT_, int SG_, int OG_> struct PgCfg {
    static constexpr int RT = RT_, MT = MT_, SG = SG_, OG = OG_; // query rows; products of 128 channels; soft-max groups, of alternate tiles; output groups, of shares of the rows
    static constexpr int N = (3 * RT + 15) / 16 * 16;          // columns of a product
    static constexpr int QW = RT > 16 ? 4 : RT > 10 ? 2 : 1;   // warps that cut queries
    static constexpr int SB = SG == 3 ? 3 : 2;                 // tiles of scores, and of weights, at a time
    static constexpr int W_OUT = 4 * SG, W_COPY = W_OUT + 4 * OG, W_MMA = W_COPY + 1, W_META = W_MMA + 2, W_Q = W_META + 1, THREADS = 32 * (W_Q + QW);
    static constexpr int COLS = N * (SB + 2 * MT), TM = COLS <= 64 ? 64 : COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
    static constexpr int P_ROW = 8 * 144, P_BYTES = N / 8 * P_ROW; // weights: sixteen slots' core matrices 144 bytes apart, so that a warp's bytes meet other banks
    static constexpr int CTAS = MT == 2 || TM > 256 ? 1 : RT > 8 ? 2 : 3; // of an SM, where shared memory allows
    static int tail(int hs) { return SB * P_BYTES + 2 * N * hs; } // shared memory behind the rings
    static_assert(COLS <= 512, "tensor memory");
};

PS_D void pg_mma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
PS_D void pg_tm_ld16(int (&v)[16], uint32_t at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]),
                   "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(at)
                 : "memory");
}
PS_D float pg_ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
PS_D float pg_redux_max(float x) { // (no number counts as nothing)
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
}
PS_D int pg_order(float x) { // whole numbers in the order of the floats; its own inverse
    const int b = __float_as_int(x);
    return b ^ (b >> 31 & 0x7fffffff);
}
PS_D float pg_unorder(int b) { return __int_as_float(b ^ (b >> 31 & 0x7fffffff)); }
// a number of each row, from shared memory
template <int RT, typename F> PS_D void pg_rows(const float *x, F f) {
#pragma unroll
    for (int c = 0; c < RT; c += 4) {
        const float4 v = *reinterpret_cast<const float4 *>(x + c);
        f(c, v.x);
        if (c + 1 < RT) f(c + 1, v.y);
        if (c + 2 < RT) f(c + 2, v.z);
        if (c + 3 < RT) f(c + 3, v.w);
    }
}
// two floats an instruction
using pg_f2 = unsigned long long;
PS_D pg_f2 pg_two(float a, float b) { pg_f2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
PS_D void pg_one(pg_f2 x, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
PS_D pg_f2 pg_mul2(pg_f2 a, pg_f2 b) { pg_f2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
PS_D pg_f2 pg_add2(pg_f2 a, pg_f2 b) { pg_f2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
PS_D pg_f2 pg_fma2(pg_f2 a, pg_f2 b, pg_f2 c) { pg_f2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
// three digits' sums, of two neighbouring columns a, b: the lower two are whole numbers of 31 bits together
PS_D pg_f2 pg_digits2(int a0, int b0, int a1, int b1, int a2, int b2) {
    return pg_fma2(pg_two((float)a2, (float)b2), pg_two(65536.f, 65536.f), pg_two((float)(a1 * 256 + a0), (float)(b1 * 256 + b0)));
}
// the digits' sums of RT rows put together, f(pair of rows, sums): sixteen rows at a time; a digit's columns begin STRIDE after the one before
template <int RT, int STRIDE, typename F> PS_D void pg_sums(uint32_t at, F f) {
    if constexpr (RT % 16 == 0) {
#pragma unroll
        for (int c = 0; c < RT; c += 16) {
            int a[16], b[16], d[16];
            pg_tm_ld16(a, at + c);
            pg_tm_ld16(b, at + STRIDE + c);
            pg_tm_ld16(d, at + 2 * STRIDE + c);
            ps_tc_ld_wait();
#pragma unroll
            for (int r = 0; r < 16; r += 2) f((c + r) / 2, pg_digits2(a[r], a[r + 1], b[r], b[r + 1], d[r], d[r + 1]));
        }
    } else {
        static_assert(RT == STRIDE, "");
        constexpr int N = (3 * RT + 15) / 16;
        int v[N][16];
#pragma unroll
        for (int c = 0; c < N; c++) pg_tm_ld16(v[c], at + 16 * c);
        ps_tc_ld_wait();
#pragma unroll
        for (int r = 0; r < RT; r += 2) {
            auto d = [&](int k, int row) { return row < RT ? v[(k * RT + row) / 16][(k * RT + row) % 16] : 0; };
            f(r / 2, pg_digits2(d(0, r), d(0, r + 1), d(1, r), d(1, r + 1), d(2, r), d(2, r + 1)));
        }
    }
}
// Fragments: lane l has, of every eight columns, the columns 2 (l % 4) and the next, of the sixteen rows l / 4 and l / 4 + 8 in this order
template <int CG> PS_D void pg_tm_frag(int (&v)[4 * CG], uint32_t at) {
    if constexpr (CG == 1)
        asm volatile("tcgen05.ld.sync.aligned.16x256b.x1.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at) : "memory");
    else if constexpr (CG == 2)
        asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                     : "r"(at)
                     : "memory");
    else
        asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
                       "=r"(v[14]), "=r"(v[15])
                     : "r"(at)
                     : "memory");
}
// bytes in such fragments to rows of sixteen bytes, one for every column: a matrix of eight columns from every eight lanes' addresses
template <int CG> PS_D void pg_put_frag(uint32_t at, const uint32_t (&w)[CG]) {
    if constexpr (CG == 1) asm volatile("stmatrix.sync.aligned.m16n8.x1.trans.shared.b8 [%0], {%1};" ::"r"(at), "r"(w[0]));
    else if constexpr (CG == 2) asm volatile("stmatrix.sync.aligned.m16n8.x2.trans.shared.b8 [%0], {%1, %2};" ::"r"(at), "r"(w[0]), "r"(w[1]));
    else asm volatile("stmatrix.sync.aligned.m16n8.x4.trans.shared.b8 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]));
}
// v[i] of lanes with the same l % 4 put together: lane l ends with that of i = (l / 4) / (8 / NR)
template <int NR, typename F> PS_D float pg_across(float (&v)[NR], F f) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 16, half = NR / 2; o >= 4; o /= 2, half /= 2) {
        if (half) {
#pragma unroll
            for (int i = 0; i < NR / 2; i++)
                if (i < half) {
                    const float keep = lane & o ? v[i + half] : v[i], give = lane & o ? v[i] : v[i + half];
                    v[i] = f(keep, __shfl_xor_sync(0xffffffffu, give, o));
                }
        } else v[0] = f(v[0], __shfl_xor_sync(0xffffffffu, v[0], o));
    }
    return v[0];
}

// A CTA's way through its tiles: runs of one sequence and head
struct PgSeg { int s, g, t0, t1; };
struct PgWalk {
    const PgAttn &a;
    int s, u, left; // u: tile within the sequence's heads
    PS_D PgWalk(const PgAttn &a_, int lane) : a(a_) {
        const int k = blockIdx.x - a.lane_cta0[lane], n = a.lane_cta0[lane + 1] - a.lane_cta0[lane];
        if (a.whole) {
            s = k / a.pool.G;
            left = a.seq[s].tiles;
            u = (k - s * a.pool.G) * left;
            return;
        }
        const int x = pg_run(a.lane_tiles[lane], n, k);
        left = pg_run(a.lane_tiles[lane], n, k + 1) - x;
        int lo = 0, hi = a.n_seqs - 1; // the last sequence that begins at or before x
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (a.tile0[mid] <= x) lo = mid;
            else hi = mid - 1;
        }
        s = lo;
        u = x - a.tile0[s];
    }
    PS_D bool next(PgSeg &o) {
        if (left <= 0) return false;
        const int tiles = a.seq[s].tiles;
        o.s = s; o.g = u / tiles; o.t0 = u - o.g * tiles;
        o.t1 = min(tiles, o.t0 + left);
        left -= o.t1 - o.t0;
        u += o.t1 - o.t0;
        if (u == tiles * a.pool.G) { u = 0; s++; }
        return true;
    }
};

struct alignas(16) PgMeta { // of a tile: by blocks of sixteen slots
    float ks[8], vq[8];     // K's scale; V's over the tile's largest, times PG_ONE
    uint32_t live[4];       // slots that are filled, not hidden, and of a page
    float vmax;             // V's largest scale over PG_ONE
};
struct PgRing { // of a number known at launch: index and the parity of the round
    int n, i = 0;
    uint32_t round = 0;
    PS_D PgRing(int n_) : n(n_) {}
    PS_D void step() {
        if (++i == n) { i = 0; round ^= 1; }
    }
};

template <int RT, int MT, int SG, int OG>
__global__ void __launch_bounds__(PgCfg<RT, MT, SG, OG>::THREADS, PgCfg<RT, MT, SG, OG>::CTAS) pg_k_attn(const __grid_constant__ PgAttn a) {
    using C = PgCfg<RT, MT, SG, OG>;
    constexpr int N = C::N, SB = C::SB;
    extern __shared__ __align__(128) uint8_t pg_raw[];
    __shared__ __align__(8) uint64_t k_full[PG_STAGES], v_full[PG_STAGES], k_free[PG_STAGES], v_free[PG_STAGES], s_full[SB], s_free[SB], p_full[SB], p_free[SB], o_full[2], o_free[2], q_full[2], fin[2], fin_free[2],
        meta_full[PG_META], meta_free[PG_META], done;
    __shared__ PgMeta s_meta[PG_META];
    __shared__ int s_ref[SG][4][RT];                                    // a tile's largest score / row factor, in order of whole numbers: four tiles' places in turn
    __shared__ __align__(16) float s_row[SG * 4 + OG * 4][2][(RT + 3) / 4 * 4]; // a warp's numbers of the rows
    __shared__ __align__(16) float s_share[SG * 4][RT % 8 == 0 ? RT : 1]; // a warp's numbers of the rows: what a tile's weights count for in the row's sum
    __shared__ float s_qs[2][RT], s_m[8][RT], s_vm[8], s_l[2][SG * 4][RT], s_mend[2][SG][RT];
    __shared__ uint32_t s_tmem;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, D = a.pool.hs, stage = PG_TILE * D;
    // shared memory: K's ring, V's ring, weights, queries (a product of 128 channels of fewer reads behind its stage, never behind the queries)
    uint8_t *sm_k = reinterpret_cast<uint8_t *>(((uintptr_t)pg_raw + 127) & ~(uintptr_t)127), *sm_v = sm_k + a.stages * stage, *sm_p = sm_v + a.stages * stage, *sm_q = sm_p + SB * C::P_BYTES;
    int rt = 0; // row tile
    while (rt + 1 < a.n_lanes && (int)blockIdx.x >= a.lane_cta0[rt + 1]) rt++;
    const int r0 = rt * RT;

    ps_grid_dep_launch(); // (the kernel that joins may take its place: it waits for the end of this one)
    // The copies' warp makes the barriers and goes on; the others meet when they and the tensor memory are there
    if (warp == C::W_COPY) {
        if (lane == 0) {
            for (int b = 0; b < PG_STAGES; b++) { ps_mbar_init(&k_full[b], 1); ps_mbar_init(&v_full[b], 1); ps_mbar_init(&k_free[b], 1); ps_mbar_init(&v_free[b], 1); }
            for (int b = 0; b < SB; b++) { ps_mbar_init(&s_full[b], 1); ps_mbar_init(&s_free[b], 4); ps_mbar_init(&p_full[b], 4); ps_mbar_init(&p_free[b], 1); }
            for (int b = 0; b < 2; b++) {
                ps_mbar_init(&o_full[b], 1); ps_mbar_init(&o_free[b], 4 * OG);
                ps_mbar_init(&q_full[b], C::QW); ps_mbar_init(&fin[b], 4 * SG); ps_mbar_init(&fin_free[b], 4 * OG);
            }
            for (int b = 0; b < PG_META; b++) { ps_mbar_init(&meta_full[b], 1); ps_mbar_init(&meta_free[b], 4); }
            ps_mbar_init(&done, 2);
            ps_fence_barrier_init();
        }
        __syncwarp();
        asm volatile("barrier.cta.arrive 15, %0;" ::"n"(C::THREADS) : "memory");
    } else {
        if (warp == C::W_MMA) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ps_smem_u32(&s_tmem)), "n"(C::TM) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
        ps_tc_fence_before();
        asm volatile("barrier.cta.sync 15, %0;" ::"n"(C::THREADS) : "memory");
        ps_tc_fence_after();
    }
    const uint32_t tm = warp == C::W_COPY ? 0u : __shfl_sync(0xffffffffu, s_tmem, 0), tm_o = tm + SB * N;
    // 32 rows: 72 registers a thread at the launch, 504 over the seven warpgroups; 3 x 88 (soft-max) + 2 x 72 (output) + 2 x 48 (the others) = 504
    auto less = [] { if constexpr (RT == 32) asm volatile("setmaxnreg.dec.sync.aligned.u32 48;"); };
    auto more = [] { if constexpr (RT == 32) asm volatile("setmaxnreg.inc.sync.aligned.u32 88;"); };
    PgWalk walk(a, rt);
    PgSeg sg;
    bool ok = true;
    // i counts the CTA's tiles, n its runs.  Whoever gives up a wait leaves his loops; the others' waits give up after him
    auto wait = [&](uint64_t *bar, uint32_t parity, int site) {
        if (ok && !ps_tc_wait_warp(bar, parity)) { *a.pool.err = site; ok = false; }
        return ok;
    };

    if (warp == C::W_COPY) {
        less();
        // ===== copies: a lane a page.  The pages' numbers come 32 at a time, before they are needed (a tile's asked for one tile ahead: 1 500 cycles a tile, whatever the other roles did)
        PgRing ring(a.stages);
        const int pages = PG_TILE >> a.pool.shift, bytes = a.pool.P * D, block = 32 / pages; // block: tiles whose pages the lanes hold
        auto numbers = [&](const PgSeg &g, int t) {
            const PgAttnSeq &s = a.seq[g.s];
            const int p = t * pages + lane;
            return t + lane / pages < g.t1 && p < (s.n_kv + a.pool.P - 1) >> a.pool.shift ? s.table[p] : -2;
        };
        int i = 0;
        PgSeg next;
        bool more = walk.next(next);
        int first = more ? numbers(next, next.t0) : -2;
        while (ok && more) {
            sg = next;
            int now = first, ahead = sg.t0 + block < sg.t1 ? numbers(sg, sg.t0 + block) : -2;
            more = walk.next(next);
            if (more) first = numbers(next, next.t0);
            int at = 0; // tile of the block
            for (int t = sg.t0; t < sg.t1; t++, i++, at++) {
                if (at == block) {
                    at = 0;
                    now = ahead;
                    if (t + block < sg.t1) ahead = numbers(sg, t + block);
                }
                int page = __shfl_sync(0xffffffffu, now, (at * pages + lane) & 31);
                if (lane >= pages) page = -2;
                const bool have = page != -2 && a.pool.has(page);
                const uint32_t tx = __popc(__ballot_sync(0xffffffffu, have)) * (uint32_t)bytes;
                const int8_t *src = have ? a.pool.codes + a.pool.at(page, sg.g, 0) * bytes : nullptr;
                for (int v = 0; v < 2; v++) {
                    uint64_t *full = (v ? v_full : k_full) + ring.i;
                    if (i >= a.stages && !wait((v ? v_free : k_free) + ring.i, ring.round ^ 1, 11)) break;
                    if (lane == 0) ps_mbar_expect_tx(full, tx);
                    __syncwarp();
                    if (have) ps_bulk_g2s((v ? sm_v : sm_k) + ring.i * stage + lane * bytes, src + (v ? bytes : 0), bytes, full);
                }
                if (!ok) break;
                ring.step();
            }
        }
        if (!ok) // (copies in flight end before the CTA does)
            for (int b = 0; b < a.stages && b < i; b++) {
                const uint32_t round = (uint32_t)((i - 1 - b) / a.stages) & 1;
                ps_tc_wait_warp(&k_full[b], round, PS_COPY_CYCLES);
                ps_tc_wait_warp(&v_full[b], round, PS_COPY_CYCLES);
            }
    } else if (warp == C::W_MMA || warp == C::W_MMA + 1) {
        less();
        // ===== MMAs: scores by one warp, outputs by another, so that neither's waits hold up the other's
        const uint32_t id = (2u << 4) | (1u << 7) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(PG_TILE >> 4) << 24), id_s = id | (1u << 10); // whole numbers; K, V, queries signed, weights not
        const uint64_t d_k = ps_tc_smem_desc(ps_smem_u32(sm_k), 128, 8 * D), d_v = ps_tc_smem_desc(ps_smem_u32(sm_v), 16 * D, 128), d_q = ps_tc_smem_desc(ps_smem_u32(sm_q), 128, 8 * D),
                       d_p = ps_tc_smem_desc(ps_smem_u32(sm_p), 144, C::P_ROW);
        const bool pv = warp == C::W_MMA + 1;
        PgRing ring(a.stages);
        int i = 0, n = 0;
        for (; ok && walk.next(sg); n++) {
            if (!pv && !wait(&q_full[n & 1], (n >> 1) & 1, 12)) break;
            const uint64_t y0 = pv ? d_p : d_q + (uint64_t)((n & 1) * (N * D >> 4));
            for (int t = sg.t0; t < sg.t1; t++, i++) {
                const int b = i % SB, o = i & 1;
                if (pv) { // (outputs of tile i - 2 are taken)
                    if (!wait(&v_full[ring.i], ring.round, 15) || !wait(&p_full[b], (i / SB) & 1, 16) || (i >= 2 && !wait(&o_free[o], ((i >> 1) - 1) & 1, 17))) break;
                } else if (!wait(&k_full[ring.i], ring.round, 13) || (i >= SB && !wait(&s_free[b], (i / SB - 1) & 1, 14))) break;
                ps_tc_fence_after();
                if (ps_elect_one()) {
                    if (pv) {
                        const uint64_t x = d_v + (uint64_t)(ring.i * (stage >> 4)), y = y0 + (uint64_t)(b * (C::P_BYTES >> 4));
#pragma unroll
                        for (int m = 0; m < MT; m++)
#pragma unroll
                            for (int c = 0; c < PG_TILE / 32; c++) pg_mma_i8(tm_o + o * MT * N + m * N, x + 128 * m + 2 * D * c, y + 18 * c, id, c != 0);
                        ps_tc_commit(&v_free[ring.i]);
                        ps_tc_commit(&p_free[b]);
                        ps_tc_commit(&o_full[o]);
                    } else {
                        const uint64_t x = d_k + (uint64_t)(ring.i * (stage >> 4));
                        for (int c = 0; c < D / 32; c++) pg_mma_i8(tm + b * N, x + 16 * c, y0 + 16 * c, id_s, c != 0);
                        ps_tc_commit(&k_free[ring.i]);
                        ps_tc_commit(&s_full[b]);
                    }
                }
                __syncwarp();
                ring.step();
            }
        }
        if (ps_elect_one()) ps_tc_commit(&done); // MMAs in flight end before the tensor memory is given back
        __syncwarp();
        if (!ps_tc_wait_warp(&done, 0)) *a.pool.err = 18;
    } else if (warp == C::W_META) {
        less();
        // ===== scales and live slots, two tiles at a time: lanes 0-15 the first's blocks, K then V, 16-31 the second's.  What two tiles need is asked for while the two before are written, their pages one step
        // earlier (asked for in turn, with a branch for every hidden byte: 1 450 cycles a tile, 3 100 with hidden slots, more than all other roles)
        const int half = lane >> 4, b = lane & 7, kv = lane >> 3 & 1, B = a.pool.P / PG_BLOCK;
        int i = 0;
        while (ok && walk.next(sg)) {
            const PgAttnSeq &s = a.seq[sg.s];
            auto page_of = [&](int t) {
                const int j = (t + half) * PG_TILE + b * PG_BLOCK;
                return t + half < sg.t1 && j < s.n_kv ? s.table[j >> a.pool.shift] : -2;
            };
            auto is_page = [&](int page) { return (unsigned)page < (unsigned)a.pool.n_pages; }; // (the copies' warp reports)
            auto scale_of = [&](int t, int page) {
                return is_page(page) ? a.pool.scales[a.pool.at(page, sg.g, kv) * B + (((t + half) * PG_TILE + b * PG_BLOCK) & (a.pool.P - 1)) / PG_BLOCK] : 0.f;
            };
            auto hidden_of = [&](int t, int (&h)[8]) {
#pragma unroll
                for (int w = 0; w < 8; w++) h[w] = s.hidden ? s.hidden[min(t * PG_TILE + 32 * w + lane, s.n_kv - 1)] : 0;
            };
            int page = page_of(sg.t0), ahead = page_of(sg.t0 + 2), hidden[8];
            float x = scale_of(sg.t0, page);
            hidden_of(sg.t0, hidden);
            for (int t = sg.t0; ok && t < sg.t1; t += 2) {
                const bool have = is_page(page);
                const float mine = x;
                const unsigned has = __ballot_sync(0xffffffffu, have);
                unsigned live[2][4];
#pragma unroll
                for (int w = 0; w < 8; w++) {
                    const int j = t * PG_TILE + 32 * w + lane;
                    live[w >> 2][w & 3] = __ballot_sync(0xffffffffu, (j < s.n_kv) & (has >> (16 * (w >> 2) + 2 * (w & 3) + (lane >> 4)) & 1) & (hidden[w] == 0));
                }
                page = ahead;
                if (t + 2 < sg.t1) {
                    x = scale_of(t + 2, page);
                    hidden_of(t + 2, hidden);
                    ahead = page_of(t + 4);
                }
                const unsigned word = half ? (b < 2 ? live[1][0] : b < 4 ? live[1][1] : b < 6 ? live[1][2] : live[1][3]) : (b < 2 ? live[0][0] : b < 4 ? live[0][1] : b < 6 ? live[0][2] : live[0][3]);
                const float scale = word >> (b & 1 ? 16 : 0) & 0xffffu ? mine : 0.f; // (a block without live slots may have any scale)
                float top = kv ? scale : 0.f;
#pragma unroll
                for (int o = 8; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if (t + h >= sg.t1) break;
                    PgMeta &m = s_meta[i % PG_META];
                    if (i >= PG_META && !wait(&meta_free[i % PG_META], ((i / PG_META) - 1) & 1, 19)) break;
                    if (half == h) {
                        if (kv) m.vq[b] = top > 0.f ? scale / top * PG_ONE : 0.f;
                        else m.ks[b] = scale;
                        if ((lane & 15) < 4) m.live[lane & 3] = (lane & 3) == 0 ? live[h][0] : (lane & 3) == 1 ? live[h][1] : (lane & 3) == 2 ? live[h][2] : live[h][3];
                        if ((lane & 15) == 8) m.vmax = top * (1.f / PG_ONE);
                    }
                    __syncwarp();
                    if (lane == 0) ps_mbar_arrive(&meta_full[i % PG_META]);
                    i++;
                }
            }
        }
    } else if (warp >= C::W_Q) {
        less();
        // ===== queries into digits, a warp a row
        int n = 0;
        for (; ok && walk.next(sg); n++) {
            const PgAttnSeq &s = a.seq[sg.s];
            const int rows = s.n_tok * a.R;
            if (n >= 2 && !wait(&fin[n & 1], ((n >> 1) - 1) & 1, 20)) break; // (all that read the queries of the run before last are through)
            uint8_t *to = sm_q + (n & 1) * (N * D);
            for (int r = warp - C::W_Q; r < RT; r += C::QW) {
                const int row = r0 + r;
                const int64_t at = row < rows ? ((int64_t)(s.tok0 + row / a.R) * a.n_heads + sg.g * a.R + row % a.R) * D : -1;
                float x[2][4], top = 0.f;
                bool none = false;
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const int d = c * 128 + lane * 4;
#pragma unroll
                    for (int e = 0; e < 4; e++) x[c][e] = 0.f;
                    if (d < D && at >= 0) {
                        if (a.bf16) {
                            const __nv_bfloat16 *p = static_cast<const __nv_bfloat16 *>(a.q) + at + d;
                            if (a.q_vec) {
                                const uint2 w = __ldg(reinterpret_cast<const uint2 *>(p));
                                x[c][0] = __uint_as_float(w.x << 16); x[c][1] = __uint_as_float(w.x & 0xffff0000u); x[c][2] = __uint_as_float(w.y << 16); x[c][3] = __uint_as_float(w.y & 0xffff0000u);
                            } else {
#pragma unroll
                                for (int e = 0; e < 4; e++) x[c][e] = __bfloat162float(p[e]);
                            }
                        } else {
                            const float *p = static_cast<const float *>(a.q) + at + d;
                            if (a.q_vec) {
                                const float4 w = __ldg(reinterpret_cast<const float4 *>(p));
                                x[c][0] = w.x; x[c][1] = w.y; x[c][2] = w.z; x[c][3] = w.w;
                            } else {
#pragma unroll
                                for (int e = 0; e < 4; e++) x[c][e] = p[e];
                            }
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        top = fmaxf(top, fabsf(x[c][e]));
                        none |= x[c][e] != x[c][e];
                    }
                }
                top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
                none = __any_sync(0xffffffffu, none) || top == INFINITY;
                // (numbers so small that the factor would leave float32's range are multiplied by 2^64 before, and all of them are as good as zeros in the end)
                const float pre = top < 0x1p-100f ? 0x1p64f : 1.f, f = top > 0.f && !none ? PG_Q_ONE / (top * pre) : 0.f, sign = a.scale < 0.f ? -f : f;
                if (lane == 0) s_qs[n & 1][r] = none ? NAN : top * fabsf(a.scale) * (1.f / PG_Q_ONE);
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const int d = c * 128 + lane * 4;
                    if (d >= D) break;
                    uint32_t w[3] = {0, 0, 0};
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        int v = __float2int_rn(fminf(fmaxf((none ? 0.f : x[c][e]) * pre * sign, -PG_Q_ONE), PG_Q_ONE));
#pragma unroll
                        for (int k = 0; k < 3; k++) {
                            const int digit = (int8_t)v;
                            w[k] |= (uint32_t)(digit & 255) << (8 * e);
                            v = (v - digit) >> 8;
                        }
                    }
#pragma unroll
                    for (int k = 0; k < 3; k++) {
                        const int col = k * RT + r;
                        *reinterpret_cast<uint32_t *>(to + (col >> 3) * 8 * D + (d >> 4) * 128 + (col & 7) * 16 + (d & 15)) = w[k];
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) ps_mbar_arrive(&q_full[n & 1]);
        }
    } else if (warp < C::W_OUT) {
        more();
        // ===== soft-max.  A warp that gave up a wait goes on to the group's next barrier, which tells the others: nobody is left alone at one.
        // RT a multiple of eight: a lane has four slots, lane / 4 and every eighth of its warp's behind it, and of every eight rows two, 2 (lane % 4) and the next; five rows: a slot and all rows.  The numbers of a
        // row (its reference, its factor) are those of the lanes whose `own` it is
        constexpr bool FRAG = RT % 8 == 0;
        constexpr int CG = FRAG ? RT / 8 : 1, NR = 2 * CG, NS = FRAG ? 4 : 1; // eights of rows; rows, slots of a lane
        const int group = warp >> 2, w = warp & 3, bar = SG == 1 ? 1 : 1 + group, quad = 2 * (lane & 3);
        const int idx = (lane >> 2) / (FRAG ? 8 / NR : 1), own = FRAG ? idx / 2 * 8 + quad + (idx & 1) : min(lane, RT - 1);
        const bool owner = FRAG ? (lane >> 2) % (FRAG ? 8 / NR : 1) == 0 : lane < RT;
        auto slot_of = [&](int e) { return w * 32 + (FRAG ? e * 8 + (lane >> 2) : lane); };
        float *mine = s_row[warp][0], *factor = s_row[warp][1];
        int i = 0, n = 0, turn = 0;
        for (; walk.next(sg); n++) {
            const PgAttnSeq &s = a.seq[sg.s];
            const int rows = min(s.n_tok * a.R - r0, RT), past = s.n_kv - s.n_tok;
            float M = PG_LOW, qs = 0.f; // row own's largest score so far, and its factor
            float l[FRAG ? 1 : RT];
            pg_f2 l2[CG], qs2[CG];
#pragma unroll
            for (int r = 0; r < (FRAG ? 1 : RT); r++) l[r] = 0.f;
#pragma unroll
            for (int c = 0; c < CG; c++) l2[c] = 0ull;
            ok = ps_bar_all(bar, 128, ok); // (a run begins: nobody of the group reads the last one's numbers any more)
            if (!ok) break;
            if (w * 32 + lane < RT)
#pragma unroll
                for (int b = 0; b < 4; b++) s_ref[group][b][w * 32 + lane] = pg_order(PG_LOW);
            ps_bar_sync(bar, 128);
            bool first = true;
            for (int t = sg.t0; t < sg.t1; t++, i++) {
                if (SG > 1 && i % SG != group) continue;
                wait(&meta_full[i % PG_META], (i / PG_META) & 1, 21);
                const PgMeta &m = s_meta[i % PG_META];
                const float ks0 = m.ks[FRAG ? 2 * w : 2 * w + (lane >> 4)], vq0 = m.vq[FRAG ? 2 * w : 2 * w + (lane >> 4)], ks1 = FRAG ? m.ks[2 * w + 1] : 0.f, vq1 = FRAG ? m.vq[2 * w + 1] : 0.f, vmax = m.vmax;
                const uint32_t live = m.live[w];
                __syncwarp();
                if (lane == 0) ps_mbar_arrive(&meta_free[i % PG_META]);
                // rows that see the lane's slots
                const bool gaps = live != ~0u || t * PG_TILE + w * 32 + 32 > past;
                uint32_t see[NS];
                if (gaps) {
#pragma unroll
                    for (int e = 0; e < NS; e++) {
                        const int back = t * PG_TILE + slot_of(e) - past;
                        see[e] = live >> (slot_of(e) & 31) & 1 ? ~0u : 0u;
                        if (see[e] && back >= 0) {
                            int tok = r0 / a.R, rest = r0 % a.R;
                            see[e] = 0;
                            for (int r = 0; r < rows; tok++, rest = 0) {
                                const int many = min(a.R - rest, rows - r);
                                if (pg_sees(s, tok, back)) see[e] |= (many == 32 ? ~0u : (1u << many) - 1) << r;
                                r += many;
                            }
                        }
                    }
                }
                wait(&s_full[i % SB], (i / SB) & 1, 22);
                ps_tc_fence_after();
                if (first) { // (they come with the first scores)
                    qs = s_qs[n & 1][own];
                    factor[own] = fmaxf(qs, 0x1p-126f); // (above zero, and a number: -inf times it is -inf)
                    __syncwarp();
                    if constexpr (FRAG) {
#pragma unroll
                        for (int c = 0; c < CG; c++) qs2[c] = *reinterpret_cast<const pg_f2 *>(factor + 8 * c + quad);
                    }
                    first = false;
                }
                // scores over the rows' factors
                const uint32_t at = tm + i % SB * N + ((uint32_t)(w * 32) << 16);
                pg_f2 y2[FRAG ? 2 : 1][2][CG];
                float y[FRAG ? 1 : RT], top;
                if constexpr (FRAG) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        int d[3][4 * CG];
#pragma unroll
                        for (int k = 0; k < 3; k++) pg_tm_frag<CG>(d[k], at + k * RT + ((uint32_t)(16 * h) << 16));
                        ps_tc_ld_wait();
                        const pg_f2 ks = h ? pg_two(ks1, ks1) : pg_two(ks0, ks0);
#pragma unroll
                        for (int c = 0; c < CG; c++)
#pragma unroll
                            for (int b = 0; b < 2; b++) {
                                const int f = 4 * c + 2 * b;
                                y2[h][b][c] = pg_mul2(pg_digits2(d[0][f], d[0][f + 1], d[1][f], d[1][f + 1], d[2][f], d[2][f + 1]), ks);
                            }
                    }
                } else
                    pg_sums<RT, RT>(at, [&](int r, pg_f2 x) {
                        float x0, x1;
                        pg_one(x, x0, x1);
                        y[2 * r] = x0 * ks0;
                        if (2 * r + 1 < RT) y[2 * r + 1] = x1 * ks0;
                    });
                ps_tc_fence_before();
                __syncwarp();
                if (lane == 0) ps_mbar_arrive(&s_free[i % SB]);
                if constexpr (FRAG) {
                    float most[NR];
                    if (gaps) {
#pragma unroll
                        for (int c = 0; c < CG; c++)
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                float x0, x1;
                                pg_one(y2[e >> 1][e & 1][c], x0, x1);
                                const uint32_t bits = see[e] >> (8 * c + quad);
                                y2[e >> 1][e & 1][c] = pg_two(bits & 1 ? x0 : -INFINITY, bits & 2 ? x1 : -INFINITY);
                            }
                    }
#pragma unroll
                    for (int c = 0; c < CG; c++) {
                        float x0[4], x1[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) pg_one(y2[e >> 1][e & 1][c], x0[e], x1[e]);
                        most[2 * c] = fmaxf(fmaxf(x0[0], x0[1]), fmaxf(x0[2], x0[3]));
                        most[2 * c + 1] = fmaxf(fmaxf(x1[0], x1[1]), fmaxf(x1[2], x1[3]));
                    }
                    top = fmaxf(PG_LOW, pg_across<NR>(most, [](float x0, float x1) { return fmaxf(x0, x1); }));
                } else {
                    if (gaps) {
#pragma unroll
                        for (int r = 0; r < RT; r++)
                            if (!(see[0] >> r & 1)) y[r] = -INFINITY;
                    }
                    top = PG_LOW;
#pragma unroll
                    for (int r = 0; r < RT; r++) {
                        const float x = pg_redux_max(y[r]);
                        if (lane == r) top = fmaxf(top, x);
                    }
                }
                int *ref = s_ref[group][turn & 3];
                if (owner) atomicMax(&ref[own], pg_order(top));
                ok = ps_bar_all(bar, 128, ok);
                if (!ok) break;
                // A tile has a reference of its own, its largest score (of the slots that the row sees), so a weight is rounded by what counts in its tile, however heavy another one's is; the row's sum has the largest so
                // far.  (Weights under the largest so far: behind a slot that has nearly all of the mass the others lost their bits, and below 2^-24 left the output but not the sum: 22 % of the output for 12 000 such.)
                const float here = pg_unorder(ref[own]);
                float top_z = here == PG_LOW ? PG_LOW : __fmul_ru(here, fmaxf(qs, 0x1p-126f)); // as the scores are, and rounded up, so that no weight is above 1
                if (fabsf(top_z) == INFINITY || (here != PG_LOW && qs != qs)) top_z = NAN;
                const float was = M, z = here == PG_LOW ? 0.f : top_z;
                M = fmaxf(was, top_z);
                turn++;
                if (w == 0 && owner) s_ref[group][(turn + 2) & 3][own] = pg_order(PG_LOW); // (the place of the tile before: all have passed a barrier since they read it, and pass another before it is used)
                if (i >= SB && !wait(&p_free[i % SB], (i / SB - 1) & 1, 23)) continue; // (the weights of tile i - SB are used up, so outputs before it are taken, and of eight places for references this one is free)
                const float share = pg_ex2(top_z - M);
                if (w == 0 && owner) {
                    s_m[i & 7][own] = top_z;
                    if (own == 0) s_vm[i & 7] = vmax;
                }
                if (__any_sync(0xffffffffu, M > was)) { // sums so far follow their references
                    if (owner) mine[own] = pg_ex2(was - M);
                    __syncwarp();
                    if constexpr (FRAG) {
#pragma unroll
                        for (int c = 0; c < CG; c++) l2[c] = pg_mul2(l2[c], *reinterpret_cast<const pg_f2 *>(mine + 8 * c + quad));
                    } else pg_rows<RT>(mine, [&](int r, float f) { l[r] *= f; });
                    __syncwarp();
                }
                if (owner) {
                    mine[own] = -z;
                    if (FRAG) s_share[warp][own] = share;
                }
                __syncwarp();
                // weights 2^23 + p, whose lower three bytes are the digits
                const uint32_t to = ps_smem_u32(sm_p) + i % SB * C::P_BYTES;
                if constexpr (FRAG) {
                    pg_f2 z2[CG];
#pragma unroll
                    for (int c = 0; c < CG; c++) z2[c] = *reinterpret_cast<const pg_f2 *>(mine + 8 * c + quad);
                    const pg_f2 one = pg_two(8388608.f, 8388608.f);
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const pg_f2 vq = h ? pg_two(vq1, vq1) : pg_two(vq0, vq0);
                        uint32_t digit[3][CG];
#pragma unroll
                        for (int c = 0; c < CG; c++) {
                            uint32_t d[4];
#pragma unroll
                            for (int b = 0; b < 2; b++) {
                                float x0, x1;
                                pg_one(pg_fma2(y2[h][b][c], qs2[c], z2[c]), x0, x1);
                                const pg_f2 p = pg_two(pg_ex2(x0), pg_ex2(x1)); // (a slot that is not seen: -inf)
                                l2[c] = pg_fma2(p, *reinterpret_cast<const pg_f2 *>(s_share[warp] + 8 * c + quad), l2[c]);
                                pg_one(pg_fma2(p, vq, one), x0, x1);
                                d[2 * b] = __float_as_uint(x0); d[2 * b + 1] = __float_as_uint(x1);
                            }
                            const uint32_t lo = __byte_perm(d[0], d[1], 0x5140), hi = __byte_perm(d[2], d[3], 0x5140);
                            digit[0][c] = __byte_perm(lo, hi, 0x5410);
                            digit[1][c] = __byte_perm(lo, hi, 0x7632);
                            digit[2][c] = __byte_perm(__byte_perm(d[0], d[1], 0x0062), __byte_perm(d[2], d[3], 0x0062), 0x5410);
                        }
#pragma unroll
                        for (int k = 0; k < 3; k++) pg_put_frag<CG>(to + (k * CG + (lane >> 3) % CG) * C::P_ROW + (2 * w + h) * 144 + (lane & 7) * 16, digit[k]);
                    }
                } else {
                    float f[8], zs[8]; // (they come before the bytes go: the compiler keeps loads behind stores)
#pragma unroll
                    for (int e = 0; e < RT; e += 4) {
                        *reinterpret_cast<float4 *>(f + e) = *reinterpret_cast<const float4 *>(factor + e);
                        *reinterpret_cast<float4 *>(zs + e) = *reinterpret_cast<const float4 *>(mine + e);
                    }
                    const uint32_t byte = to + (2 * w + (lane >> 4)) * 144 + (lane & 15);
#pragma unroll
                    for (int r = 0; r < RT; r++) {
                        const float p = pg_ex2(fmaf(y[r], f[r], zs[r]));
                        l[r] = fmaf(p, __shfl_sync(0xffffffffu, share, r), l[r]);
                        const uint32_t d = __float_as_uint(fmaf(p, vq0, 8388608.f));
#pragma unroll
                        for (int k = 0; k < 3; k++) {
                            const int col = k * RT + r;
                            asm volatile("st.shared.u8 [%0], %1;" ::"r"(byte + (col >> 3) * C::P_ROW + (col & 7) * 16), "r"(d >> (8 * k)));
                        }
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) ps_mbar_arrive(&p_full[i % SB]);
            }
            // the run's sums
            if (!ok || (n >= 2 && !wait(&fin_free[n & 1], ((n >> 1) - 1) & 1, 24))) continue;
            if constexpr (FRAG) {
                float sums[NR];
#pragma unroll
                for (int c = 0; c < CG; c++) pg_one(l2[c], sums[2 * c], sums[2 * c + 1]);
                const float x = pg_across<NR>(sums, [](float x0, float x1) { return x0 + x1; });
                if (owner) s_l[n & 1][warp][own] = x;
            } else {
#pragma unroll
                for (int r = 0; r < RT; r++) {
                    float x = l[r];
#pragma unroll
                    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
                    if (lane == r) s_l[n & 1][warp][r] = x;
                }
            }
            if (w == 0 && owner) s_mend[n & 1][group][own] = M;
            __syncwarp();
            if (lane == 0) ps_mbar_arrive(&fin[n & 1]);
        }
    } else {
        // ===== output: thread = channel (of each product), a group its share of the rows
        constexpr int RO = RT / OG;
        const int share = (warp - C::W_OUT) >> 2, w = warp & 3, ch = w * 32 + lane, own = share * RO + min(lane, RO - 1), from = r0 + share * RO;
        const uint32_t lane_at = (uint32_t)(w * 32) << 16;
        float *mine = s_row[warp][0];
        int i = 0, n = 0;
        for (; ok && walk.next(sg); n++) {
            const PgAttnSeq &s = a.seq[sg.s];
            const int rows = min(s.n_tok * a.R - from, RO);
            constexpr int H = RO / 2 + RO % 2; // pairs of rows
            pg_f2 acc[MT][H];
            float M = PG_LOW;
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int r = 0; r < H; r++) acc[m][r] = 0ull;
            for (int t = sg.t0; t < sg.t1; t++, i++) {
                if (!wait(&o_full[i & 1], (i >> 1) & 1, 25)) break;
                ps_tc_fence_after();
                float fo = 1.f, fn = 0.f;
                if (lane < RO) {
                    const float m = s_m[i & 7][own], top = fmaxf(M, m);
                    fo = pg_ex2(M - top);
                    fn = pg_ex2(m - top) * s_vm[i & 7];
                    M = top;
                }
                if (__any_sync(0xffffffffu, fo != 1.f)) {
                    __syncwarp();
                    if (lane < RO) mine[lane] = fo;
                    __syncwarp();
#pragma unroll
                    for (int r = 0; r < H; r++) {
                        const pg_f2 f = *reinterpret_cast<const pg_f2 *>(mine + 2 * r);
#pragma unroll
                        for (int m = 0; m < MT; m++) acc[m][r] = pg_mul2(acc[m][r], f);
                    }
                }
                __syncwarp();
                if (lane < RO) mine[lane] = fn;
                __syncwarp();
#pragma unroll
                for (int m = 0; m < MT; m++) pg_sums<RO, RT>(tm_o + (i & 1) * MT * N + m * N + share * RO + lane_at, [&](int r, pg_f2 x) { acc[m][r] = pg_fma2(x, *reinterpret_cast<const pg_f2 *>(mine + 2 * r), acc[m][r]); });
                ps_tc_fence_before();
                __syncwarp();
                if (lane == 0) ps_mbar_arrive(&o_free[i & 1]);
            }
            if (!ok || !wait(&fin[n & 1], (n >> 1) & 1, 26)) break;
            float L = 0.f;
            if (lane < RO) {
#pragma unroll
                for (int g = 0; g < SG; g++) {
                    float sum = 0.f;
#pragma unroll
                    for (int k = 0; k < 4; k++) sum += s_l[n & 1][g * 4 + k][own];
                    L = fmaf(sum, pg_ex2(s_mend[n & 1][g][own] - M), L);
                }
            }
            __syncwarp();
            if (lane == 0) ps_mbar_arrive(&fin_free[n & 1]);
            const bool whole = sg.t0 == 0 && sg.t1 == s.tiles;
            if (lane < RO) mine[lane] = whole ? (L == 0.f ? 0.f : 1.f / L) : 1.f;
            __syncwarp();
            const int64_t slot = (int64_t)blockIdx.x * 2 + (n > 0);
            if (!whole && w == 0 && lane < RO) reinterpret_cast<float2 *>(a.part + (int64_t)a.n_ctas * 2 * RT * D)[slot * RT + own] = make_float2(M, L);
#pragma unroll
            for (int m = 0; m < MT; m++) {
                const int d = m * 128 + ch;
                if (d >= D) break;
                if (whole) {
                    int64_t at = ((int64_t)(s.tok0 + from / a.R) * a.n_heads + sg.g * a.R + from % a.R) * D + d;
                    int rest = from % a.R;
#pragma unroll
                    for (int r = 0; r < RO; r++) {
                        if (r >= rows) break;
                        float x0, x1;
                        pg_one(acc[m][r / 2], x0, x1);
                        const float x = (r & 1 ? x1 : x0) * mine[r];
                        if (a.bf16) static_cast<__nv_bfloat16 *>(a.out)[at] = __float2bfloat16_rn(x);
                        else static_cast<float *>(a.out)[at] = x;
                        at += D;
                        if (++rest == a.R) { rest = 0; at += (int64_t)(a.n_heads - a.R) * D; }
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < RO; r++)
                        if (r < rows) {
                            float x0, x1;
                            pg_one(acc[m][r / 2], x0, x1);
                            a.part[(slot * RT + share * RO + r) * D + d] = r & 1 ? x1 : x0;
                        }
                }
            }
            __syncwarp();
        }
    }
    ps_tc_fence_before();
    __syncthreads();
    ps_tc_fence_after();
    if (warp == C::W_MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "n"(C::TM) : "memory");
}

// ---------------------------------------------------------------------------------------------------- joining the runs
// x: the beginning of a run, y: eight of its rows.  Where it lies inside the tiles of some sequence and head, and no run before it begins there, the block joins all runs that have some of them, a warp a row.  (A warp for every row of
// the call, joined or not: 64 sequences 10 us of a kernel whose 512 blocks came in waves.)  Its start overlaps the end of the kernel before
template <int RT> __global__ void __launch_bounds__(256) pg_k_join(const __grid_constant__ PgAttn a) {
    int rt = 0;
    while (rt + 1 < a.n_lanes && (int)blockIdx.x >= a.lane_cta0[rt + 1]) rt++;
    const int k = blockIdx.x - a.lane_cta0[rt], n = a.lane_cta0[rt + 1] - a.lane_cta0[rt], T = a.lane_tiles[rt], q = T / n, more = T % n;
    auto of = [&](int x) { return x < more * (q + 1) ? x / (q + 1) : more + (x - more * (q + 1)) / q; }; // the run that has tile x
    auto begins = [&](int r) { return q * r + min(r, more); };
    const int x = begins(k);
    int lo = 0, hi = a.n_seqs - 1; // the last sequence that begins at or before x
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (a.tile0[mid] <= x) lo = mid;
        else hi = mid - 1;
    }
    const PgAttnSeq &s = a.seq[lo];
    const int g = (x - a.tile0[lo]) / s.tiles, u0 = a.tile0[lo] + g * s.tiles, k0 = k - 1, k1 = of(u0 + s.tiles - 1);
    if (k == 0 || x == u0 || begins(k - 1) > u0) return;
    ps_grid_dep_wait();
    const int lane = threadIdx.x & 31, D = a.pool.hs, rows = min(s.n_tok * a.R - rt * RT, RT);
    const float2 *ml = reinterpret_cast<const float2 *>(a.part + (int64_t)a.n_ctas * 2 * RT * D);
    const int r = blockIdx.y * 8 + (threadIdx.x >> 5);
    if (r < rows) {
        auto place = [&](int run) { // a run that begins before these tiles has come to them later
            return ((int64_t)(a.lane_cta0[rt] + run) * 2 + (begins(run) < u0)) * RT + r;
        };
        float top = PG_LOW, l = 0.f, acc[8] = {};
        for (int i = k0 + lane; i <= k1; i += 32) top = fmaxf(top, ml[place(i)].x);
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        for (int i0 = k0; i0 <= k1; i0 += 32) {
            float f = 0.f;
            int64_t at = 0;
            if (i0 + lane <= k1) {
                at = place(i0 + lane);
                const float2 p = ml[at];
                f = pg_ex2(p.x - top);
                l = fmaf(p.y, f, l);
            }
            for (int i = 0; i < min(32, k1 + 1 - i0); i += 4) {
                float v[4][8];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int64_t from = __shfl_sync(0xffffffffu, at, i + e);
#pragma unroll
                    for (int c = 0; c < 8; c++)
                        if (c * 32 < D && i0 + i + e <= k1) v[e][c] = a.part[from * D + c * 32 + lane];
                }
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float fe = __shfl_sync(0xffffffffu, f, i + e);
#pragma unroll
                    for (int c = 0; c < 8; c++)
                        if (c * 32 < D && i0 + i + e <= k1) acc[c] = fmaf(v[e][c], fe, acc[c]);
                }
            }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int row = rt * RT + r;
        const int64_t to = ((int64_t)(s.tok0 + row / a.R) * a.n_heads + g * a.R + row % a.R) * D;
#pragma unroll
        for (int c = 0; c < 8; c++)
            if (c * 32 < D) {
                const float y = acc[c] * inv;
                if (a.bf16) static_cast<__nv_bfloat16 *>(a.out)[to + c * 32 + lane] = __float2bfloat16_rn(y);
                else static_cast<float *>(a.out)[to + c * 32 + lane] = y;
            }
    }
}
