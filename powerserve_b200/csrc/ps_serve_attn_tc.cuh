// ps_serve_attn_tc.cuh - ps_serve_attn.cuh's attention for head sizes 64 and 128, on the fifth-generation tensor cores, to float32's precision.
//
// Operands.  A number x is cut into two fp16 parts, the upper eleven bits of x 2^e and the others, rounded, with 2^e from the largest of its group so that the
// group fits fp16's range from the top: what is lost is below 2^-22 of x, or 2^-39 of the group's largest.  Three MMAs (lo hi, hi lo, hi hi) replace the
// 32-bit products; the missing lo lo is below 2^-20 of the product (2^-23 on average; the upper part is cut off, not rounded, so it has the product's sign).  bfloat16 caches have no lo part: two MMAs.  Groups: a query row; eight slots' K rows;
// hs / 8 channels of a tile of V.  The weights p of the soft-max, at most 1, are cut after a factor 2^15.
// The queries' parts stay in tensor memory (in shared memory they took the room of two stages).
// A tile's output leaves the tensor memory after every tile and is added up in registers, with rounding: the accumulator, which truncates, sees the
// MMAs of one tile alone.  So groups' factors and a row's maximum may differ from tile to tile, and the soft-max of a tile knows of no other tile.
//
// A CTA takes up to 128 query rows (the MMAs' M side: one row, one lane of tensor memory) of one kv head over one split.  Warps 0-3 and 4-7: soft-max of
// every other tile; 8-15: output, a row's channels in two halves; 16-23: copies and conversion; 24, 25: MMAs (26, 27 make the warpgroup whole).
// Tiles of K and of V go through rings of three shared-memory stages each (six small ones).  A converter warp brings the rows that it will cut, two tiles ahead, as they lie
// in memory, by asynchronous 16-byte copies, cuts them into parts in their place (eight rows become the same eight rows' parts in the K-major
// no-swizzle layout, in the same bytes), and the MMAs read them.  Rows are 16 bytes apart from the next so that neither reading nor writing meets a bank twice.
// (Bulk copies of rows of 256 and 512 bytes took 65 cycles each, 12 400 a tile; two warps that only copied 60 for 512 bytes, 3 500 a tile.)
// Bound by instructions: a tile of 64 slots (float32, head size 128) takes its roles 9 400, of which cutting K and V is a third; the schedulers issue in half to two thirds of all cycles, the
// matrix pipe works 22 to 31 %. Hence two floats an instruction (11 850 a tile without), scores read twice instead of a barrier between the halves of a row, and a row's reference that follows its
// maximum by steps of 2^8 only. Float32, 8 kv heads of 128, 2 sequences x 32 tokens x 4 heads over 32 700 slots: 148 us = 3.6 TB/s (536 MB; 177 us = 3.0 TB/s where the power limit lowers
// the clock), 222 with the scores of 268 MB and their weights (265). bfloat16, heads of 64, 8 x 20 tokens over up to 8 100 slots: 66 us = 1.2 TB/s; a tile is 16 KB, so its bytes are
// a fifth of the bound.
#pragma once
#include "ps_serve_attn.cuh"

#include <cuda_fp16.h>

#define SV_TC_THREADS 896
#define SV_TC_ROWS 128
#define SV_TC_TILES 256  // most tiles of a split (a word of live slots for each)

PS_D void sv_bar_wait(uint64_t *bar, uint32_t parity, bool &ok, int *err, int site) {
    if (ok && !ps_tc_wait_warp(bar, parity)) { *err = site; ok = false; }
}
// 2^e with max 2^e in [2^14, 2^15), and its inverse
PS_D float sv_scale(uint32_t max_bits, float &inv) {
    const int e = min(126, 14 + 127 - (int)(max_bits >> 23));
    inv = __uint_as_float((uint32_t)(127 - e) << 23);
    return __uint_as_float((uint32_t)(127 + e) << 23);
}
PS_D uint32_t sv_pack(float a, float b) { // fp16 of a (low half) and b
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
// two floats at a time: the kernel below is bound by the instructions that it issues
using sv_f2 = unsigned long long;
PS_D sv_f2 sv_two(float a, float b) { sv_f2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
PS_D void sv_one(sv_f2 x, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
PS_D sv_f2 sv_mul2(sv_f2 a, sv_f2 b) { sv_f2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
PS_D sv_f2 sv_add2(sv_f2 a, sv_f2 b) { sv_f2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
PS_D sv_f2 sv_fma2(sv_f2 a, sv_f2 b, sv_f2 c) { sv_f2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
PS_D void sv_cut2(sv_f2 x, uint32_t &hi, uint32_t &lo) { // hi: the upper eleven bits, as they are (no conversion back); lo: the others, rounded
    float a, b;
    sv_one(x, a, b);
    const float ha = __uint_as_float(__float_as_uint(a) & 0xffffe000u), hb = __uint_as_float(__float_as_uint(b) & 0xffffe000u);
    hi = sv_pack(ha, hb);
    sv_one(sv_fma2(sv_two(ha, hb), sv_two(-1.f, -1.f), x), a, b);
    lo = sv_pack(a, b);
}
PS_D void sv_cut(float a, float b, uint32_t &hi, uint32_t &lo) { sv_cut2(sv_two(a, b), hi, lo); }
PS_D void sv_tm_ld16(uint32_t (&v)[16], uint32_t at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]),
                   "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(at)
                 : "memory");
}
PS_D void sv_tm_st8(uint32_t at, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
template <int N> PS_D void sv_regs_more() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> PS_D void sv_regs_less() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
// eight elements of a cache as they lie in memory
struct SvRaw32 { float4 a, b; };
struct SvRaw16 { uint4 a; };
PS_D void sv_get(SvRaw32 &r, const uint8_t *p) {
    r.a = *reinterpret_cast<const float4 *>(p);
    r.b = *reinterpret_cast<const float4 *>(p + 16);
}
PS_D void sv_get(SvRaw16 &r, const uint8_t *p) { r.a = *reinterpret_cast<const uint4 *>(p); }
PS_D void sv_keep(SvRaw32 &r, uint32_t m) { // zero where the bit is not set
    r.a.x = m & 1 ? r.a.x : 0.f; r.a.y = m & 2 ? r.a.y : 0.f; r.a.z = m & 4 ? r.a.z : 0.f; r.a.w = m & 8 ? r.a.w : 0.f;
    r.b.x = m & 16 ? r.b.x : 0.f; r.b.y = m & 32 ? r.b.y : 0.f; r.b.z = m & 64 ? r.b.z : 0.f; r.b.w = m & 128 ? r.b.w : 0.f;
}
PS_D void sv_keep(SvRaw16 &r, uint32_t m) {
    uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] &= (m >> (2 * i) & 1 ? 0x0000ffffu : 0u) | (m >> (2 * i) & 2 ? 0xffff0000u : 0u);
    r.a = make_uint4(w[0], w[1], w[2], w[3]);
}
PS_D float sv_at(const SvRaw32 &r, int i) {
    const float4 &q = i < 4 ? r.a : r.b;
    return i % 4 == 0 ? q.x : i % 4 == 1 ? q.y : i % 4 == 2 ? q.z : q.w;
}
PS_D float sv_at(const SvRaw16 &r, int i) {
    const uint32_t w = i < 2 ? r.a.x : i < 4 ? r.a.y : i < 6 ? r.a.z : r.a.w;
    return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
}

template <typename T, int D> struct SvTc {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int PARTS = F32 ? 2 : 1;
    static constexpr int K_ROW = D * (int)sizeof(T) + 16, V_ROW = SV_TILE * (int)sizeof(T) + 16; // bytes from row to row of a stage
    static constexpr int K_LO = D * 16, V_LO = SV_TILE * 16;                                     // from a group's hi part to its lo part
    static constexpr int K_STAGE = SV_TILE * K_ROW, V_STAGE = D * V_ROW;
    static constexpr int STAGES = 6 * (K_STAGE + V_STAGE) < 216 * 1024 ? 6 : 3;                  // of K's ring and of V's
    static constexpr int SMEM = STAGES * (K_STAGE + V_STAGE) + 128;
    static constexpr int V_GROUPS = D / 64;                                                      // groups of eight channels that a converter takes
    using Raw = typename std::conditional<F32, SvRaw32, SvRaw16>::type;
};

template <typename T, int D, bool W>
__global__ void __launch_bounds__(SV_TC_THREADS, 1) sv_k_attn_tc(const __grid_constant__ SvAttn a) {
    using C = SvTc<T, D>;
    extern __shared__ __align__(128) uint8_t sv_tc_raw[];
    __shared__ __align__(8) uint64_t ready[2][C::STAGES], unused[2][C::STAGES], s_full[4], p_full[4], sp_free[4], o_full[2], o_empty[2], done;
    __shared__ uint32_t tmem_smem;
    __shared__ float s_top[8][SV_TC_ROWS], s_sum[8][SV_TC_ROWS], s_qtop[2][SV_TC_ROWS];
    __shared__ __align__(16) float s_kinv[16][8], s_vinv[16][8];
    __shared__ uint64_t s_live[SV_TC_TILES];
    uint8_t *sm_k = reinterpret_cast<uint8_t *>(((uintptr_t)sv_tc_raw + 127) & ~(uintptr_t)127), *sm_v = sm_k + C::STAGES * C::K_STAGE;
    constexpr int stages = C::STAGES;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int si = __shfl_sync(0xffffffffu, sv_find(a, blockIdx.x), 0), split = blockIdx.x - a.seq[si].unit0, g = blockIdx.y;
    const SvSeq &s = a.seq[si];
    const int all_rows = s.n_tok * a.R, r0 = blockIdx.z * SV_TC_ROWS, rows = min(all_rows - r0, SV_TC_ROWS);
    if (rows <= 0) return;
    const int j0 = split * a.tps * SV_TILE, j_end = min(s.n_kv, j0 + a.tps * SV_TILE), tiles = (j_end - j0 + SV_TILE - 1) / SV_TILE, past = s.n_kv - s.n_tok;

    if (tid == 0) {
        for (int b = 0; b < stages; b++)
            for (int v = 0; v < 2; v++) { ps_mbar_init(&ready[v][b], 4); ps_mbar_init(&unused[v][b], 1); }
        for (int b = 0; b < 4; b++) { ps_mbar_init(&s_full[b], 1); ps_mbar_init(&p_full[b], 4); ps_mbar_init(&sp_free[b], 1); }
        for (int b = 0; b < 2; b++) { ps_mbar_init(&o_full[b], 1); ps_mbar_init(&o_empty[b], 8); }
        ps_mbar_init(&done, 2);
        ps_fence_barrier_init();
    }
    // Copies: a converter (of K: warps 16-19, of V: 20-23) brings the quarter of a tile's rows that it will cut, sixteen bytes a lane; one group of copies a tile
    constexpr int COPIES = D * (int)sizeof(T) / 32, K_LANES = D * (int)sizeof(T) / 16, V_LANES = SV_TILE * (int)sizeof(T) / 16; // lanes of a row
    const T *src = nullptr;
    int64_t step = 0, tile_step = 0;
    uint32_t ring_at = 0;
    if (warp >= 20 && s.v_mode) {
        const int row = (warp & 3) * (D / 4) + lane / V_LANES, col = lane % V_LANES;
        src = static_cast<const T *>(s.v) + ((int64_t)g * D + row) * s.n_ctx + j0 + col * (16 / (int)sizeof(T));
        step = (int64_t)(32 / V_LANES) * s.n_ctx;
        tile_step = SV_TILE;
        ring_at = ps_smem_u32(sm_v) + row * C::V_ROW + col * 16;
    } else if (warp < 20 && s.k_mode) {
        const int row = (warp & 3) * 16 + lane / K_LANES, col = lane % K_LANES;
        const int64_t ld = (int64_t)a.G * D;
        src = static_cast<const T *>(s.k) + (int64_t)(j0 + row) * ld + (int64_t)g * D + col * (16 / (int)sizeof(T));
        step = (32 / K_LANES) * ld;
        tile_step = SV_TILE * ld;
        ring_at = ps_smem_u32(sm_k) + row * C::K_ROW + col * 16;
    }
    auto bring = [&](int t) {
        const int at = t % stages, n = j_end - j0 - t * SV_TILE;
        auto copy = [](uint32_t to, const T *p) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(p) : "memory"); };
        if (t < tiles && src) {
            const T *p = src + t * tile_step;
            if (warp >= 20) {
                const uint32_t to = ring_at + at * C::V_STAGE;
                if (n >= SV_TILE || t * SV_TILE + j0 + (lane % V_LANES) * (16 / (int)sizeof(T)) < s.n_ctx) // (a row of V is read up to its own end)
#pragma unroll
                    for (int r = 0; r < COPIES; r++, p += step) copy(to + r * (32 / V_LANES) * C::V_ROW, p);
            } else {
                const uint32_t to = ring_at + at * C::K_STAGE;
                if (n >= SV_TILE) {
#pragma unroll
                    for (int r = 0; r < COPIES; r++, p += step) copy(to + r * (32 / K_LANES) * C::K_ROW, p);
                } else {
                    const int row = (warp & 3) * 16 + lane / K_LANES;
#pragma unroll 1
                    for (int r = 0; r < COPIES && row + r * (32 / K_LANES) < n; r++, p += step) copy(to + r * (32 / K_LANES) * C::K_ROW, p);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if (warp >= 16 && warp < 24)
        for (int t = 0; t < stages - 1; t++) bring(t); // (the rings are empty)
    if (warp == 24) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(ps_smem_u32(&tmem_smem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // live slots of a tile: in the split and not hidden
    if (s.hidden && warp < 24)
        for (int t = warp; t < tiles; t += 24) {
            const int j = j0 + t * SV_TILE + lane;
            const uint32_t lo = __ballot_sync(0xffffffffu, j < j_end && !s.hidden[min(j, j_end - 1)]), hi = __ballot_sync(0xffffffffu, j + 32 < j_end && !s.hidden[min(j + 32, j_end - 1)]);
            if (lane == 0) s_live[t] = (uint64_t)hi << 32 | lo;
        }
    auto live_of = [&](int t) -> uint64_t {
        if (s.hidden) return s_live[t];
        const int n = j_end - j0 - t * SV_TILE;
        return n >= SV_TILE ? ~0ull : (1ull << n) - 1;
    };
    // which of a tile's slots token `tok` sees
    auto see_of = [&](int t, int tok, bool mine) -> uint64_t {
        const int j = j0 + t * SV_TILE;
        uint64_t see = live_of(t);
        if (j + SV_TILE > past && mine) // of the step's own slots those that this token sees
            for (int c = max(0, past - j); c < min(SV_TILE, j_end - j); c++)
                if (!sv_sees(s, tok, j + c - past)) see &= ~(1ull << c);
        return see;
    };
    // queries: warps 0-3 the first half of the channels, 4-7 the second, a thread its half of a row
    float4 qv[D / 8];
    if (warp < 8) {
        const int r = (warp & 3) * 32 + lane, row = r0 + r;
        const float *q = a.q + ((int64_t)(s.tok0 + row / a.R) * a.n_heads + g * a.R + row % a.R) * D + (warp >> 2) * (D / 2);
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < D / 8; i++) {
            qv[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < rows) {
                if (a.q_vec) qv[i] = __ldg(reinterpret_cast<const float4 *>(q) + i);
                else qv[i] = make_float4(q[4 * i], q[4 * i + 1], q[4 * i + 2], q[4 * i + 3]);
            }
            qv[i].x *= a.scale; qv[i].y *= a.scale; qv[i].z *= a.scale; qv[i].w *= a.scale;
            top = fmaxf(fmaxf(fmaxf(top, fabsf(qv[i].x)), fabsf(qv[i].y)), fmaxf(fabsf(qv[i].z), fabsf(qv[i].w)));
        }
        s_qtop[warp >> 2][r] = top;
    }
    ps_tc_fence_before();
    __syncthreads();
    ps_tc_fence_after();
    // columns of tensor memory: four tiles' scores of 64, sixteen of which become eight of the weights' hi parts and eight of lo; outputs 128 (head size 64: two); queries D / 2 + D / 2
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem_smem, 0), tm_s = tm, tm_o = tm + 4 * SV_TILE, tm_q = tm_o + 128;
    float qinv = 1.f;
    if (warp < 8) {
        const int r = (warp & 3) * 32 + lane;
        const float f = sv_scale(__float_as_uint(fmaxf(s_qtop[0][r], s_qtop[1][r])), qinv);
#pragma unroll
        for (int i = 0; i < D / 8; i += 4) {
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                sv_cut(qv[i + e].x * f, qv[i + e].y * f, hi[2 * e], lo[2 * e]);
                sv_cut(qv[i + e].z * f, qv[i + e].w * f, hi[2 * e + 1], lo[2 * e + 1]);
            }
            const uint32_t to = tm_q + (warp >> 2) * (D / 4) + 2 * i + ((uint32_t)((warp & 3) * 32) << 16);
            sv_tm_st8(to, hi);
            sv_tm_st8(to + D / 2, lo);
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    }
    ps_tc_fence_before();
    __syncthreads();
    ps_tc_fence_after();
    // A barrier is waited on only by who must have passed it before it can complete again (a phase that was missed would never end): groups' and rows' factors
    // come with the MMAs' barrier, whose issuer has waited for those who wrote them.  Scores of tile t are asked for when the outputs of tile t - 4 are there, those when tile t - 6
    // has been taken out: so eight places for maxima and sums are enough.
    // Registers: 72 a thread at the launch, 504 over the seven warpgroups; 2 x 72 (soft-max) + 2 x 88 (output) + 2 x 72 (converters) + 40 (MMAs, copies) = 504

    if (warp >= 24) {
        sv_regs_less<40>();
        if (warp < 26) {
            // ===== MMAs, scores by warp 24, outputs by warp 25: neither's waits hold up the other's.  Small products first, while the truncating accumulator is small
            const bool pv = warp == 25;
            const uint32_t idesc = (1u << 4) | ((uint32_t)((pv ? D : SV_TILE) >> 3) << 17) | ((uint32_t)(SV_TC_ROWS >> 4) << 24);
            const uint64_t desc = ps_tc_smem_desc(ps_smem_u32(pv ? sm_v : sm_k), 128, 8 * (pv ? C::V_ROW : C::K_ROW));
            for (int t = 0; t < tiles; t++) {
                const int b = t & 1, sp = t & 3, at = t % stages;
                if (!ps_tc_wait_warp(&ready[pv][at], (t / stages) & 1)) { *a.err = 12; break; }
                if (pv) { // (head size 128: there is one output, and the tile before has to be out of it; 64: the one before that)
                    constexpr int AGO = D == 128 ? 1 : 2;
                    if (!ps_tc_wait_warp(&p_full[sp], (t >> 2) & 1)) { *a.err = 15; break; }
                    if (t >= AGO && !ps_tc_wait_warp(&o_empty[(t - AGO) & 1], ((t - AGO) >> 1) & 1)) { *a.err = 13; break; }
                } else if (t >= 4 && !ps_tc_wait_warp(&sp_free[sp], ((t >> 2) - 1) & 1)) { *a.err = 14; break; } // (the weights of tile t - 4 are used up)
                ps_tc_fence_after();
                const uint64_t d = desc + (uint64_t)(at * ((pv ? C::V_STAGE : C::K_STAGE) >> 4));
                const uint32_t tile = tm_s + sp * SV_TILE;
                if (ps_elect_one()) {
                    if (pv) {
#pragma unroll
                        for (int p = 0; p < C::PARTS + 1; p++)
#pragma unroll
                            for (int j = 0; j < SV_TILE / 16; j++)
                                ps_tc_mma_f16_ta(tm_o + (D == 64 ? b * D : 0), tile + j * 16 + (p == 0 ? 8 : 0), d + (C::F32 && p == 1 ? C::V_LO >> 4 : 0) + j * 16, idesc, (p | j) != 0);
                        ps_tc_commit(&sp_free[sp]);
                        ps_tc_commit(&o_full[b]);
                    } else {
#pragma unroll
                        for (int p = 0; p < C::PARTS + 1; p++) // lo hi, hi lo, hi hi (bfloat16 caches: lo hi, hi hi)
#pragma unroll
                            for (int j = 0; j < D / 16; j++) ps_tc_mma_f16_ta(tile, tm_q + (p == 0 ? D / 2 : 0) + j * 8, d + (C::F32 && p == 1 ? C::K_LO >> 4 : 0) + j * 16, idesc, (p | j) != 0);
                        ps_tc_commit(&s_full[sp]);
                    }
                    ps_tc_commit(&unused[pv][at]);
                }
                __syncwarp();
            }
            if (ps_elect_one()) ps_tc_commit(&done); // MMAs in flight end before the tensor memory is given back
            __syncwarp();
            if (!ps_tc_wait_warp(&done, 0)) *a.err = 16;
        }
    } else if (warp >= 16) {
        // ===== converters.  lane % 8 picks one of eight rows (slots of K, channels of V), lane / 8 one of four neighbouring eights of the row; a warp's quarter of a tile in
        // two parts, of which each has a factor of its own
        auto convert = [&](auto of_v) {
            constexpr bool V = decltype(of_v)::value;
            constexpr int ITS = D / 32, ROW = V ? C::V_ROW : C::K_ROW, LO = V ? C::V_LO : C::K_LO; // ITS: eights of a thread
            constexpr int GROUPS = V ? C::V_GROUPS : 1, AT_ONCE = ITS * sizeof(typename C::Raw) <= 64 ? 2 : 1; // groups of a part; parts at a time, as registers allow
            const int sub = lane & 7, quad = lane >> 3, mode = V ? s.v_mode : s.k_mode, first = 2 * GROUPS * (warp & 3);
            uint8_t *ring = V ? sm_v : sm_k;
            for (int t = 0; t < tiles; t++) {
                const int st = t % stages;
                const uint64_t live = live_of(t);
                asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 2) : "memory");
                __syncwarp();
#pragma unroll 1
                for (int part0 = 0; part0 < 2; part0 += AT_ONCE) {
                    // eight i of the thread: K: 32 elements further along the row; V: the row's second half, then the next group of channels
                    typename C::Raw raw[AT_ONCE][ITS];
                    uint8_t *group = ring + st * (V ? C::V_STAGE : C::K_STAGE) + (first + part0 * GROUPS) * 8 * ROW;
                    if (mode) {
                        const uint8_t *from = group + sub * ROW + quad * (8 * (int)sizeof(T));
#pragma unroll
                        for (int p = 0; p < AT_ONCE; p++)
#pragma unroll
                            for (int i = 0; i < ITS; i++) sv_get(raw[p][i], from + p * GROUPS * 8 * ROW + (V ? (i >> 1) * 8 * ROW + (i & 1) * (32 * (int)sizeof(T)) : i * (32 * (int)sizeof(T))));
                    } else { // rows that no wide copy can read: element by element
                        const int j = j0 + t * SV_TILE;
#pragma unroll
                        for (int p = 0; p < AT_ONCE; p++)
#pragma unroll
                            for (int i = 0; i < ITS; i++) {
                                T x[8];
                                const int w = 2 * (warp & 3) + part0 + p, slot = V ? (quad + 4 * (i & 1)) * 8 : w * 8 + sub;
                                const T *src = V ? static_cast<const T *>(s.v) + ((int64_t)g * D + (w * C::V_GROUPS + (i >> 1)) * 8 + sub) * s.n_ctx + j + slot
                                                 : static_cast<const T *>(s.k) + (int64_t)(j + slot) * a.G * D + (int64_t)g * D + (i * 4 + quad) * 8;
#pragma unroll
                                for (int e = 0; e < 8; e++) {
                                    x[e] = T(0.f);
                                    if (live >> (V ? slot + e : slot) & 1) x[e] = src[e];
                                }
                                memcpy(&raw[p][i], x, sizeof raw[p][i]);
                            }
                    }
                    if (live != ~0ull) { // what a slot that is not live holds, or was not copied, may be anything
#pragma unroll
                        for (int p = 0; p < AT_ONCE; p++)
                            if (V || (live >> (16 * (warp & 3) + 8 * (part0 + p)) & 0xffu) != 0xffu) {
#pragma unroll
                                for (int i = 0; i < ITS; i++)
                                    sv_keep(raw[p][i], V ? (uint32_t)(live >> (8 * (quad + 4 * (i & 1)))) : live >> (16 * (warp & 3) + 8 * (part0 + p) + sub) & 1 ? 0xffu : 0u);
                            }
                    }
                    float top[AT_ONCE];
#pragma unroll
                    for (int p = 0; p < AT_ONCE; p++) {
                        top[p] = 0.f;
#pragma unroll
                        for (int i = 0; i < ITS; i++)
#pragma unroll
                            for (int e = 0; e < 8; e += 2) top[p] = fmaxf(fmaxf(top[p], fabsf(sv_at(raw[p][i], e))), fabsf(sv_at(raw[p][i], e + 1)));
                    }
                    float inv[AT_ONCE];
                    sv_f2 f[AT_ONCE];
#pragma unroll
                    for (int p = 0; p < AT_ONCE; p++) {
                        const float f1 = sv_scale(__reduce_max_sync(0xffffffffu, __float_as_uint(top[p])), inv[p]); // (and all lanes have read)
                        f[p] = sv_two(f1, f1);
                    }
#pragma unroll
                    for (int p = 0; p < AT_ONCE; p++) {
                        uint8_t *to = group + p * GROUPS * 8 * ROW + sub * 16 + quad * 128;
#pragma unroll
                        for (int i = 0; i < ITS; i++) {
                            uint32_t hi[4], lo[4];
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const sv_f2 x = sv_mul2(sv_two(sv_at(raw[p][i], 2 * e), sv_at(raw[p][i], 2 * e + 1)), f[p]);
                                if (C::F32) sv_cut2(x, hi[e], lo[e]);
                                else { // (eight bits: hi is all of it)
                                    float x0, x1;
                                    sv_one(x, x0, x1);
                                    hi[e] = sv_pack(x0, x1);
                                }
                            }
                            uint8_t *q = to + (V ? (i >> 1) * 8 * ROW + (i & 1) * 512 : i * 512);
                            *reinterpret_cast<uint4 *>(q) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                            if (C::F32) *reinterpret_cast<uint4 *>(q + LO) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                        }
                        if (lane == 0) (V ? s_vinv : s_kinv)[t & 15][2 * (warp & 3) + part0 + p] = inv[p]; // (who reads tile t - 16's is done: the rings span six tiles at most, and scores are four ahead of outputs)
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) ps_mbar_arrive(&ready[V][st]);
                // (what is asked for now has a tile's time to come)
                if (t && t + stages - 1 < tiles && !ps_tc_wait_warp(&unused[V][(t - 1) % stages], ((t - 1) / stages) & 1)) { *a.err = 11; break; }
                bring(t + stages - 1);
            }
        };
        if (warp >= 20) convert(std::true_type{});
        else convert(std::false_type{});
        asm volatile("cp.async.wait_all;" ::: "memory"); // (what is in flight ends before the CTA does, even when a wait gave up)
    } else if (warp < 8) {
        // ===== soft-max: thread = row, warps 0-3 take the even tiles, 4-7 the odd ones.  The scores are read twice (there are no registers for 64), and the weights' parts take their place
        const int r = (warp & 3) * 32 + lane, row = r0 + r, tok = row / a.R, rp = sv_rp(all_rows);
        const bool mine = r < rows, any = (warp & 3) * 32 < rows; // (any: of the warp)
        const uint32_t lane_at = (uint32_t)((warp & 3) * 32) << 16;
        bool ok = true;
        for (int t = warp >> 2; t < tiles; t += 2) {
            const int sp = t & 3;
            const uint64_t see = see_of(t, tok, mine);
            uint32_t gaps = 0; // sixteen slots of which some row of the warp does not see one
#pragma unroll
            for (int c = 0; c < 4; c++) gaps |= __any_sync(0xffffffffu, (see >> (16 * c) & 0xffffu) != 0xffffu) ? 1u << c : 0u;
            sv_bar_wait(&s_full[sp], (t >> 2) & 1, ok, a.err, 18);
            if (!ok) break;
            ps_tc_fence_after();
            if (any) {
                const uint32_t at = tm_s + sp * SV_TILE + lane_at;
                uint32_t v0[16], v1[16];
                float top[4] = {SV_NONE, SV_NONE, SV_NONE, SV_NONE};
                const float *ki = s_kinv[t & 15];
                // (a factor is never zero: -inf times it is -inf)
                auto hide = [&](uint32_t (&v)[16], int c) {
                    if (gaps >> c & 1) {
#pragma unroll
                        for (int e = 0; e < 16; e++)
                            if (!(see >> (16 * c + e) & 1)) v[e] = __float_as_uint(SV_NONE);
                    }
                };
                auto most = [&](uint32_t (&v)[16], int c) {
                    hide(v, c);
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const float f = fmaxf(qinv * ki[2 * c + h], 0x1p-126f);
                        if (W && s.scores && mine) {
                            float4 *to = reinterpret_cast<float4 *>(s.scores) + ((int64_t)g * sv_quads(s.n_kv) + (j0 + t * SV_TILE) / 4 + 4 * c + 2 * h) * rp + row;
#pragma unroll
                            for (int e = 8 * h; e < 8 * h + 8; e += 4, to += rp)
                                __stcs(to, make_float4(__uint_as_float(v[e]) * f, __uint_as_float(v[e + 1]) * f, __uint_as_float(v[e + 2]) * f, __uint_as_float(v[e + 3]) * f));
                        }
                        float m = SV_NONE;
#pragma unroll
                        for (int e = 0; e < 8; e += 2) m = fmaxf(fmaxf(m, __uint_as_float(v[8 * h + e])), __uint_as_float(v[8 * h + e + 1]));
                        top[2 * (c & 1) + h] = fmaxf(top[2 * (c & 1) + h], m * f);
                    }
                };
                sv_tm_ld16(v0, at);
                sv_tm_ld16(v1, at + 16);
                ps_tc_ld_wait();
                most(v0, 0);
                most(v1, 1);
                sv_tm_ld16(v0, at + 32);
                sv_tm_ld16(v1, at + 48);
                ps_tc_ld_wait();
                most(v0, 2);
                most(v1, 3);
                const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                // the weights are 2^15 p, and so is their sum
                const float shift = mx == SV_NONE ? 15.f : 15.f - mx;
                const sv_f2 shift2 = sv_two(shift, shift);
                sv_f2 sum = 0ull;
                auto weigh = [&](uint32_t (&v)[16], int c) {
                    const float f[2] = {fmaxf(qinv * ki[2 * c], 0x1p-126f), fmaxf(qinv * ki[2 * c + 1], 0x1p-126f)};
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        float p0, p1;
                        sv_one(sv_fma2(sv_two(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), sv_two(f[e / 4], f[e / 4]), shift2), p0, p1);
                        const sv_f2 p = sv_two(sv_ex2(p0), sv_ex2(p1));
                        sum = sv_add2(sum, p);
                        sv_cut2(p, hi[e], lo[e]);
                    }
                    sv_tm_st8(at + 16 * c, hi);
                    sv_tm_st8(at + 16 * c + 8, lo);
                };
                weigh(v0, 2);
                sv_tm_ld16(v0, at);
                weigh(v1, 3);
                sv_tm_ld16(v1, at + 16);
                ps_tc_ld_wait();
                hide(v0, 0);
                weigh(v0, 0);
                hide(v1, 1);
                weigh(v1, 1);
                s_top[t & 7][r] = mx;
                float sum0, sum1;
                sv_one(sum, sum0, sum1);
                s_sum[t & 7][r] = sum0 + sum1;
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            }
            ps_tc_fence_before();
            __syncwarp();
            if (lane == 0) ps_mbar_arrive(&p_full[sp]);
        }
    } else {
        // ===== output: thread = row, half of the channels; the row's maximum and sum so far
        sv_regs_more<88>();
        const int half = (warp - 8) >> 2, r = (warp & 3) * 32 + lane, row = r0 + r;
        const bool any = (warp & 3) * 32 < rows;
        const uint32_t lane_at = (uint32_t)((warp & 3) * 32) << 16;
        sv_f2 acc[D / 4];
        float m = SV_NONE, l = 0.f;
        bool ok = true;
#pragma unroll
        for (int c = 0; c < D / 4; c++) acc[c] = 0ull;
        for (int t = 0; t < tiles; t++) {
            const int b = t & 1;
            sv_bar_wait(&o_full[b], (t >> 1) & 1, ok, a.err, 22);
            if (!ok) break;
            ps_tc_fence_after();
            if (any) {
                // (what has been added up changes its reference when a maximum is 2^8 above it, or the first there is: seldom)
                const float top = s_top[t & 7][r];
                const bool up = top > m + 8.f;
                const float mn = up ? top : m, ref = mn == SV_NONE ? 0.f : mn, fo = up ? sv_ex2(m - ref) : 1.f, fn = sv_ex2(top - ref);
                const float4 vi = *reinterpret_cast<const float4 *>(&s_vinv[t & 15][4 * half]);
                const sv_f2 f[4] = {sv_two(fn * vi.x, fn * vi.x), sv_two(fn * vi.y, fn * vi.y), sv_two(fn * vi.z, fn * vi.z), sv_two(fn * vi.w, fn * vi.w)};
                l = fmaf(l, fo, s_sum[t & 7][r] * fn);
                m = mn;
                if (__any_sync(0xffffffffu, up)) {
#pragma unroll
                    for (int c = 0; c < D / 4; c++) acc[c] = sv_mul2(acc[c], sv_two(fo, fo));
                }
#pragma unroll
                for (int c = 0; c < D / 2; c += 16) {
                    uint32_t v[16];
                    sv_tm_ld16(v, tm_o + (D == 64 ? b * D : 0) + half * (D / 2) + c + lane_at);
                    ps_tc_ld_wait();
#pragma unroll
                    for (int e = 0; e < 16; e += 2) acc[(c + e) / 2] = sv_fma2(sv_two(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), f[(c + e) / (D / 8)], acc[(c + e) / 2]);
                }
            }
            ps_tc_fence_before();
            __syncwarp();
            if (lane == 0) ps_mbar_arrive(&o_empty[b]);
        }
        if (r < rows) {
            if (half == 0) {
                if (s.splits == 1) sv_put_lse(s, (int64_t)g * all_rows + row, m, l * (1.f / 32768.f));
                else reinterpret_cast<float2 *>(s.part + (int64_t)s.splits * a.G * all_rows * D)[((int64_t)split * a.G + g) * all_rows + row] = make_float2(m, l * (1.f / 32768.f));
            }
            const float f = s.splits == 1 ? (l > 0.f ? 1.f / l : 0.f) : 1.f / 32768.f;
            float *to = s.splits == 1 ? a.out + ((int64_t)(s.tok0 + row / a.R) * a.n_heads + g * a.R + row % a.R) * D : s.part + (((int64_t)split * a.G + g) * all_rows + row) * D;
            to += half * (D / 2);
#pragma unroll
            for (int c = 0; c < D / 2; c += 4) {
                float x[4];
                sv_one(sv_mul2(acc[c / 2], sv_two(f, f)), x[0], x[1]);
                sv_one(sv_mul2(acc[c / 2 + 1], sv_two(f, f)), x[2], x[3]);
                if (a.out_vec || s.splits > 1) *reinterpret_cast<float4 *>(to + c) = make_float4(x[0], x[1], x[2], x[3]);
                else { to[c] = x[0]; to[c + 1] = x[1]; to[c + 2] = x[2]; to[c + 3] = x[3]; }
            }
        }
    }
    ps_tc_fence_before();
    __syncthreads();
    if (warp == 24) {
        ps_tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tm) : "memory");
    }
}
