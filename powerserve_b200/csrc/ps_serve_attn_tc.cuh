// ps_serve_attn_tc.cuh - ps_serve_attn.cuh's attention for head sizes 64 and 128, on the fifth-generation tensor cores, to float32's precision.
//
// Operands.  A number x is cut into two fp16 parts, the upper eleven bits of x 2^e and the others, rounded, with 2^e from the largest of its group so that the
// group fits fp16's range from the top: what is lost is below 2^-22 of x, or 2^-39 of the group's largest.  Three MMAs (lo hi, hi lo, hi hi) replace the
// 32-bit products; the missing lo lo is below 2^-22 of the product.  bfloat16 caches have no lo part: two MMAs.  Groups: a query row; eight slots' K rows;
// hs / 8 channels of a tile of V.  The weights p of the soft-max, at most 1, are cut after a factor 2^15.
// The queries' parts stay in tensor memory (in shared memory they took the room of two stages).
// A tile's output leaves the tensor memory after every tile and is added up in registers, with rounding: the accumulator, which truncates, sees the
// MMAs of one tile alone.  So groups' factors and a row's maximum may differ from tile to tile, and the soft-max of a tile knows of no other tile.
//
// A CTA takes up to 128 query rows (the MMAs' M side: one row, one lane of tensor memory) of one kv head over one split.  Warps 0-3 and 4-7: soft-max of a
// tile's first and last 32 slots; 8-15: output, a row's channels in two halves; 16-23: copies and conversion; 24, 25: MMAs (26, 27 make the warpgroup whole).
// Tiles of K and of V go through rings of three shared-memory stages each (six small ones).  A converter warp brings the rows that it will cut, two tiles ahead, as they lie
// in memory, by asynchronous 16-byte copies, cuts them into parts in their place (eight rows become the same eight rows' parts in the K-major
// no-swizzle layout, in the same bytes), and the MMAs read them.  Rows are 16 bytes apart from the next so that neither reading nor writing meets a bank twice.
// (Bulk copies of rows of 256 and 512 bytes took 65 cycles each, 12 400 a tile; two warps that only copied 60 for 512 bytes, 3 500 a tile.)
// Bound by memory: at head size 128 a tile of 64 slots is 64 KB, some 2 850 cycles of an SM's share of the bandwidth.
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
PS_D void sv_cut(float a, float b, uint32_t &hi, uint32_t &lo) { // hi: the upper eleven bits, as they are (no conversion back); lo: the others, rounded
    const float ha = __uint_as_float(__float_as_uint(a) & 0xffffe000u), hb = __uint_as_float(__float_as_uint(b) & 0xffffe000u);
    hi = sv_pack(ha, hb);
    lo = sv_pack(a - ha, b - hb);
}
PS_D float sv_ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
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

template <typename T, int D>
__global__ void __launch_bounds__(SV_TC_THREADS, 1) sv_k_attn_tc(const __grid_constant__ SvAttn a) {
    using C = SvTc<T, D>;
    extern __shared__ __align__(128) uint8_t sv_tc_raw[];
    __shared__ __align__(8) uint64_t ready[2][C::STAGES], unused[2][C::STAGES], s_full[2], s_free[2], p_full[2], o_full[2], o_empty[2], done;
    __shared__ uint32_t tmem_smem;
    __shared__ float s_top[2][SV_TC_ROWS], s_sum[2][2][SV_TC_ROWS], s_half[2][2][SV_TC_ROWS], s_qtop[2][SV_TC_ROWS];
    __shared__ __align__(16) float s_kinv[8][8], s_vinv[8][8];
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
        for (int b = 0; b < 2; b++) { ps_mbar_init(&s_full[b], 1); ps_mbar_init(&s_free[b], 8); ps_mbar_init(&p_full[b], 8); ps_mbar_init(&o_full[b], 1); ps_mbar_init(&o_empty[b], 8); }
        ps_mbar_init(&done, 2);
        ps_fence_barrier_init();
    }
    // Copies: a converter (of K: warps 16-19, of V: 20-23) brings the quarter of a tile's rows that it will cut, sixteen bytes a lane; one group of copies a tile
    auto bring = [&](int t) {
        const int w = warp & 3, j = j0 + t * SV_TILE, at = t % stages;
        if (t < tiles) {
            if (warp >= 20) {
                if (s.v_mode) {
                    constexpr int LANES = SV_TILE * (int)sizeof(T) / 16, AT_ONCE = 32 / LANES;  // lanes of a row, rows at once
                    const int row = w * (D / 4) + lane / LANES, col = lane % LANES;
                    const uint32_t to = ps_smem_u32(sm_v + at * C::V_STAGE) + row * C::V_ROW + col * 16;
                    const T *src = static_cast<const T *>(s.v) + ((int64_t)g * D + row) * s.n_ctx + j + col * (16 / (int)sizeof(T));
                    const int64_t step = (int64_t)AT_ONCE * s.n_ctx;
                    if (j + col * (16 / (int)sizeof(T)) < s.n_ctx) // (a row of V is read up to its own end)
#pragma unroll
                        for (int r = 0; r < D / 4 / AT_ONCE; r++, src += step) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + r * AT_ONCE * C::V_ROW), "l"(src) : "memory");
                }
            } else if (s.k_mode) {
                constexpr int LANES = D * (int)sizeof(T) / 16, AT_ONCE = 32 / LANES;
                const int row = w * 16 + lane / LANES, col = lane % LANES;
                const uint32_t to = ps_smem_u32(sm_k + at * C::K_STAGE) + row * C::K_ROW + col * 16;
                const int64_t ld = (int64_t)a.G * D, step = AT_ONCE * ld;
                const T *src = static_cast<const T *>(s.k) + (int64_t)(j + row) * ld + (int64_t)g * D + col * (16 / (int)sizeof(T));
                const int n = j_end - j - row;
#pragma unroll
                for (int r = 0; r < 16 / AT_ONCE; r++, src += step)
                    if (r * AT_ONCE < n) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + r * AT_ONCE * C::K_ROW), "l"(src) : "memory");
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
    // columns of tensor memory: scores 2 x 64, weights 2 x (32 + 32), outputs 128 (head size 64: two), queries D / 2 + D / 2
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem_smem, 0), tm_s = tm, tm_p = tm + 2 * SV_TILE, tm_o = tm + 4 * SV_TILE, tm_q = tm_o + 128;
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
    // come with the MMAs' barrier, whose issuer has waited for those who wrote them.
    // Registers: 72 a thread at the launch, 504 over the seven warpgroups; 2 x 72 (soft-max) + 2 x 88 (output) + 2 x 72 (converters) + 40 (MMAs, copies) = 504

    if (warp >= 24) {
        sv_regs_less<40>();
        if (warp < 26) {
            // ===== MMAs, scores by warp 24, outputs by warp 25: neither's waits hold up the other's.  Small products first, while the truncating accumulator is small
            const bool pv = warp == 25;
            const uint32_t idesc = (1u << 4) | ((uint32_t)((pv ? D : SV_TILE) >> 3) << 17) | ((uint32_t)(SV_TC_ROWS >> 4) << 24);
            const uint64_t desc = ps_tc_smem_desc(ps_smem_u32(pv ? sm_v : sm_k), 128, 8 * (pv ? C::V_ROW : C::K_ROW));
            for (int t = 0; t < tiles; t++) {
                const int b = t & 1, at = t % stages;
                if (!ps_tc_wait_warp(&ready[pv][at], (t / stages) & 1)) { *a.err = 12; break; }
                if (pv) { // (head size 128: there is one output, and the tile before has to be out of it)
                    if (!ps_tc_wait_warp(&p_full[b], (t >> 1) & 1)) { *a.err = 15; break; }
                    if (D == 128 && t && !ps_tc_wait_warp(&o_empty[b ^ 1], ((t - 1) >> 1) & 1)) { *a.err = 13; break; }
                } else if (t >= 2 && !ps_tc_wait_warp(&s_free[b], ((t >> 1) - 1) & 1)) { *a.err = 14; break; } // (the scores of tile t - 2 have been read)
                ps_tc_fence_after();
                const uint64_t d = desc + (uint64_t)(at * ((pv ? C::V_STAGE : C::K_STAGE) >> 4));
                if (ps_elect_one()) {
                    if (pv) {
                        const uint32_t pa = tm_p + b * SV_TILE;
#pragma unroll
                        for (int p = 0; p < C::PARTS + 1; p++)
#pragma unroll
                            for (int j = 0; j < SV_TILE / 16; j++)
                                ps_tc_mma_f16_ta(tm_o + (D == 64 ? b * D : 0), pa + (p == 0 ? SV_TILE / 2 : 0) + j * 8, d + (C::F32 && p == 1 ? C::V_LO >> 4 : 0) + j * 16, idesc, (p | j) != 0);
                    } else {
                        const uint32_t to = tm_s + b * SV_TILE;
#pragma unroll
                        for (int p = 0; p < C::PARTS + 1; p++) // lo hi, hi lo, hi hi (bfloat16 caches: lo hi, hi hi)
#pragma unroll
                            for (int j = 0; j < D / 16; j++) ps_tc_mma_f16_ta(to, tm_q + (p == 0 ? D / 2 : 0) + j * 8, d + (C::F32 && p == 1 ? C::K_LO >> 4 : 0) + j * 16, idesc, (p | j) != 0);
                    }
                    ps_tc_commit(&unused[pv][at]);
                    ps_tc_commit(pv ? &o_full[b] : &s_full[b]);
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
        const int sub = lane & 7, quad = lane >> 3;
        const bool is_v = warp >= 20;
        for (int t = 0; t < tiles; t++) {
            const int st = t % stages;
            asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 2) : "memory");
            __syncwarp();
#pragma unroll 1
            for (int part = 0; part < 2; part++) {
            const int w = 2 * (warp & 3) + part;
            constexpr int ITS = D / 32; // eights of a thread
            const int mode = is_v ? s.v_mode : s.k_mode, j = j0 + t * SV_TILE;
            const uint64_t live = live_of(t);
            uint8_t *group = is_v ? sm_v + st * C::V_STAGE + w * C::V_GROUPS * 8 * C::V_ROW : sm_k + st * C::K_STAGE + w * 8 * C::K_ROW;
            // eight i of the thread: K: 32 elements further along the row; V: the row's second half, then the next group of channels
            typename C::Raw raw[ITS];
            if (mode) {
                const uint8_t *from = group + sub * (is_v ? C::V_ROW : C::K_ROW) + quad * (8 * (int)sizeof(T));
#pragma unroll
                for (int i = 0; i < ITS; i++) sv_get(raw[i], from + (is_v ? (i >> 1) * 8 * C::V_ROW + (i & 1) * (32 * (int)sizeof(T)) : i * (32 * (int)sizeof(T))));
            } else { // rows that no bulk copy can read: element by element
#pragma unroll
                for (int i = 0; i < ITS; i++) {
                    T x[8];
                    const int slot = is_v ? (quad + 4 * (i & 1)) * 8 : w * 8 + sub;
                    const T *src = is_v ? static_cast<const T *>(s.v) + ((int64_t)g * D + (w * C::V_GROUPS + (i >> 1)) * 8 + sub) * s.n_ctx + j + slot
                                        : static_cast<const T *>(s.k) + (int64_t)(j + slot) * a.G * D + (int64_t)g * D + (i * 4 + quad) * 8;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        x[e] = T(0.f);
                        if (live >> (is_v ? slot + e : slot) & 1) x[e] = src[e];
                    }
                    memcpy(&raw[i], x, sizeof raw[i]);
                }
            }
            float x[ITS][8], top = 0.f;
            if (live == ~0ull) {
#pragma unroll
                for (int i = 0; i < ITS; i++)
#pragma unroll
                    for (int e = 0; e < 8; e++) x[i][e] = sv_at(raw[i], e);
            } else { // what a slot that is not live holds, or was not copied, may be anything
#pragma unroll
                for (int i = 0; i < ITS; i++) {
                    const uint32_t m = is_v ? (uint32_t)(live >> (8 * (quad + 4 * (i & 1)))) : live >> (w * 8 + sub) & 1 ? 0xffu : 0u;
#pragma unroll
                    for (int e = 0; e < 8; e++) x[i][e] = m >> e & 1 ? sv_at(raw[i], e) : 0.f;
                }
            }
#pragma unroll
            for (int i = 0; i < ITS; i++)
#pragma unroll
                for (int e = 0; e < 8; e += 2) top = fmaxf(fmaxf(top, fabsf(x[i][e])), fabsf(x[i][e + 1]));
            float inv;
            const float f = sv_scale(__reduce_max_sync(0xffffffffu, __float_as_uint(top)), inv); // (and all lanes have read)
            uint8_t *to = group + sub * 16 + quad * 128;
            const int lo_at = is_v ? C::V_LO : C::K_LO;
#pragma unroll
            for (int i = 0; i < ITS; i++) {
                uint4 hi, lo;
                sv_cut(x[i][0] * f, x[i][1] * f, hi.x, lo.x);
                sv_cut(x[i][2] * f, x[i][3] * f, hi.y, lo.y);
                sv_cut(x[i][4] * f, x[i][5] * f, hi.z, lo.z);
                sv_cut(x[i][6] * f, x[i][7] * f, hi.w, lo.w);
                uint8_t *p = to + (is_v ? (i >> 1) * 8 * C::V_ROW + (i & 1) * 512 : i * 512);
                *reinterpret_cast<uint4 *>(p) = hi;
                if (C::F32) *reinterpret_cast<uint4 *>(p + lo_at) = lo;
            }
            if (lane == 0) (is_v ? s_vinv : s_kinv)[t & 7][w] = inv; // (who reads tile t - 8's is done: the ring's stages span three tiles, and what comes after MMAs two more)
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) ps_mbar_arrive(&ready[is_v][st]);
            // (what is asked for now has a tile's time to come)
            if (t && t + stages - 1 < tiles && !ps_tc_wait_warp(&unused[is_v][(t - 1) % stages], ((t - 1) / stages) & 1)) { *a.err = 11; break; }
            bring(t + stages - 1);
        }
        asm volatile("cp.async.wait_all;" ::: "memory"); // (what is in flight ends before the CTA does, even when a wait gave up)
    } else if (warp < 8) {
        // ===== soft-max: thread = row, warps 0-3 take a tile's first 32 slots, 4-7 the others
        const int r = (warp & 3) * 32 + lane, row = r0 + r, tok = row / a.R, rp = sv_rp(all_rows), half = warp >> 2;
        const bool mine = r < rows, any = (warp & 3) * 32 < rows; // (any: of the warp)
        const uint32_t lane_at = (uint32_t)((warp & 3) * 32) << 16;
        bool ok = true;
        for (int t = 0; t < tiles; t++) {
            const int b = t & 1, j = j0 + t * SV_TILE + 32 * half;
            uint32_t see = (uint32_t)(live_of(t) >> (32 * half));
            if (j + 32 > past && mine) // of the step's own slots those that this token sees
                for (int c = max(0, past - j); c < min(32, j_end - j); c++)
                    if (!sv_sees(s, tok, j + c - past)) see &= ~(1u << c);
            const bool whole = __all_sync(0xffffffffu, see == ~0u);
            sv_bar_wait(&s_full[b], (t >> 1) & 1, ok, a.err, 18);
            ps_tc_fence_after();
            __syncwarp();
            uint32_t v[32];
            float mx = SV_NONE;
            if (any && ok) {
                uint32_t (&va)[16] = *reinterpret_cast<uint32_t (*)[16]>(v), (&vb)[16] = *reinterpret_cast<uint32_t (*)[16]>(v + 16);
                sv_tm_ld16(va, tm_s + b * SV_TILE + 32 * half + lane_at);
                sv_tm_ld16(vb, tm_s + b * SV_TILE + 32 * half + 16 + lane_at);
                const float4 ki = *reinterpret_cast<const float4 *>(&s_kinv[t & 7][4 * half]);
                // (never zero: -inf times it is -inf)
                const float f[4] = {fmaxf(qinv * ki.x, 0x1p-126f), fmaxf(qinv * ki.y, 0x1p-126f), fmaxf(qinv * ki.z, 0x1p-126f), fmaxf(qinv * ki.w, 0x1p-126f)};
                ps_tc_ld_wait();
#pragma unroll
                for (int c = 0; c < 32; c++) v[c] = __float_as_uint(__uint_as_float(v[c]) * f[c / 8]);
                if (!whole) {
#pragma unroll
                    for (int c = 0; c < 32; c++)
                        if (!(see >> c & 1)) v[c] = __float_as_uint(SV_NONE);
                }
                float t0 = SV_NONE, t1 = SV_NONE;
#pragma unroll
                for (int c = 0; c < 16; c += 2) {
                    t0 = fmaxf(fmaxf(t0, __uint_as_float(v[c])), __uint_as_float(v[c + 1]));
                    t1 = fmaxf(fmaxf(t1, __uint_as_float(v[c + 16])), __uint_as_float(v[c + 17]));
                }
                mx = fmaxf(t0, t1);
            }
            s_half[b][half][r] = mx;
            ps_tc_fence_before();
            __syncwarp();
            if (lane == 0) ps_mbar_arrive(&s_free[b]); // the scores are in registers: those of tile t + 2 may come
            if (t >= 2) sv_bar_wait(&o_empty[b], ((t >> 1) - 1) & 1, ok, a.err, 19); // (tile t - 2's weights are used up, and its maximum and sum)
            ok = ps_bar_all(1 + (warp & 3), 64, ok); // the two warps of the same rows go on together, or give up together
            if (!ok) break;
            if (any) {
                if (s.scores && mine) {
                    float4 *to = reinterpret_cast<float4 *>(s.scores) + ((int64_t)g * sv_quads(s.n_kv) + j / 4) * rp + row;
#pragma unroll
                    for (int c = 0; c < 32; c += 4) to[(int64_t)(c / 4) * rp] = make_float4(__uint_as_float(v[c]), __uint_as_float(v[c + 1]), __uint_as_float(v[c + 2]), __uint_as_float(v[c + 3]));
                }
                mx = fmaxf(mx, s_half[b][half ^ 1][r]);
                // the weights are 2^15 p, and so is their sum
                const float shift = mx == SV_NONE ? 15.f : 15.f - mx;
                float sum = 0.f, sum1 = 0.f;
#pragma unroll
                for (int c = 0; c < 32; c += 16) {
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float p0 = sv_ex2(__uint_as_float(v[c + 2 * e]) + shift), p1 = sv_ex2(__uint_as_float(v[c + 2 * e + 1]) + shift);
                        sum += p0;
                        sum1 += p1;
                        sv_cut(p0, p1, hi[e], lo[e]);
                    }
                    sv_tm_st8(tm_p + b * SV_TILE + 16 * half + c / 2 + lane_at, hi);
                    sv_tm_st8(tm_p + b * SV_TILE + SV_TILE / 2 + 16 * half + c / 2 + lane_at, lo);
                }
                s_top[b][r] = mx; // (both warps write the same)
                s_sum[b][half][r] = sum + sum1;
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            }
            ps_tc_fence_before();
            __syncwarp();
            if (lane == 0) ps_mbar_arrive(&p_full[b]);
        }
    } else {
        // ===== output: thread = row, half of the channels; the row's maximum and sum so far
        sv_regs_more<88>();
        const int half = (warp - 8) >> 2, r = (warp & 3) * 32 + lane, row = r0 + r;
        const bool any = (warp & 3) * 32 < rows;
        const uint32_t lane_at = (uint32_t)((warp & 3) * 32) << 16;
        float acc[D / 2], m = SV_NONE, l = 0.f;
        bool ok = true;
#pragma unroll
        for (int c = 0; c < D / 2; c++) acc[c] = 0.f;
        for (int t = 0; t < tiles; t++) {
            const int b = t & 1;
            sv_bar_wait(&o_full[b], (t >> 1) & 1, ok, a.err, 22);
            if (!ok) break;
            ps_tc_fence_after();
            if (any) {
                const float top = s_top[b][r], mn = fmaxf(m, top), ref = mn == SV_NONE ? 0.f : mn, fo = sv_ex2(m - ref), fn = sv_ex2(top - ref);
                const float4 vi = *reinterpret_cast<const float4 *>(&s_vinv[t & 7][4 * half]);
                const float f[4] = {fn * vi.x, fn * vi.y, fn * vi.z, fn * vi.w};
                l = fmaf(l, fo, (s_sum[b][0][r] + s_sum[b][1][r]) * fn);
                m = mn;
                if (__any_sync(0xffffffffu, fo != 1.f)) {
#pragma unroll
                    for (int c = 0; c < D / 2; c++) acc[c] *= fo;
                }
#pragma unroll
                for (int c = 0; c < D / 2; c += 16) {
                    uint32_t v[16];
                    sv_tm_ld16(v, tm_o + (D == 64 ? b * D : 0) + half * (D / 2) + c + lane_at);
                    ps_tc_ld_wait();
#pragma unroll
                    for (int e = 0; e < 16; e++) acc[c + e] = fmaf(__uint_as_float(v[e]), f[(c + e) / (D / 8)], acc[c + e]);
                }
            }
            ps_tc_fence_before();
            __syncwarp();
            if (lane == 0) ps_mbar_arrive(&o_empty[b]);
        }
        if (r < rows) {
            if (half == 0) reinterpret_cast<float2 *>(s.part + (int64_t)s.splits * a.G * all_rows * D)[((int64_t)split * a.G + g) * all_rows + row] = make_float2(m, l * (1.f / 32768.f));
            const float f = s.splits == 1 ? (l > 0.f ? 1.f / l : 0.f) : 1.f / 32768.f;
            float *to = s.splits == 1 ? a.out + ((int64_t)(s.tok0 + row / a.R) * a.n_heads + g * a.R + row % a.R) * D : s.part + (((int64_t)split * a.G + g) * all_rows + row) * D;
            to += half * (D / 2);
            if (a.out_vec || s.splits > 1) {
#pragma unroll
                for (int c = 0; c < D / 2; c += 4) *reinterpret_cast<float4 *>(to + c) = make_float4(acc[c] * f, acc[c + 1] * f, acc[c + 2] * f, acc[c + 3] * f);
            } else {
#pragma unroll
                for (int c = 0; c < D / 2; c++) to[c] = acc[c] * f;
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
