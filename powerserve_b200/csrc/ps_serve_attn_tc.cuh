// ps_serve_attn_tc.cuh - ps_serve_attn.cuh's attention for head sizes 64 and 128, on the fifth-generation tensor cores, to float32's precision.
//
// Operands.  A number x is cut into two fp16 parts, hi = fp16(x 2^e) and lo = fp16(x 2^e - hi), with 2^e from the largest of its group so that the
// group fits fp16's range from the top: what is lost is below 2^-22 of x, or 2^-39 of the group's largest.  Three MMAs (lo hi, hi lo, hi hi) replace the
// 32-bit products; the missing lo lo is below 2^-22 of the product.  bfloat16 caches have no lo part: two MMAs.  Groups: a query row; 16 slots' K rows;
// hs / 4 channels of a tile of V.  The weights p of the soft-max, at most 1, are cut after a factor 2^15.
// A tile's output leaves the tensor memory after every tile and is added up in registers, with rounding: the accumulator, which truncates, sees the
// twelve MMAs of one tile, and groups' and rows' factors may differ from tile to tile.
//
// A CTA takes up to 128 query rows (the MMAs' M side: one row, one lane of tensor memory, one thread of the soft-max) of one kv head over one split.
// Roles: warps 0-3 soft-max; 4-11 output (a row's channels in two halves); 12-15 load K rows, 16-19 V columns: from memory to registers a tile ahead,
// into parts, to shared memory in the K-major no-swizzle layout; 20 issues MMAs.  Tensor memory: two tiles of scores, of weights (both parts), of outputs.
// Bound by memory: a tile of 64 slots at head size 128 is 64 KB, some 2 850 cycles of an SM's share of the bandwidth; its MMAs take some 1 500.
#pragma once
#include "ps_serve_attn.cuh"

#include <cuda_fp16.h>

#define SV_TC_THREADS 672
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
PS_D void sv_cut(float a, float b, uint32_t &hi, uint32_t &lo) {
    hi = sv_pack(a, b);
    const float2 h = __half22float2(*reinterpret_cast<__half2 *>(&hi));
    lo = sv_pack(a - h.x, b - h.y);
}
PS_D float sv_ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// eight elements of a cache as they lie in memory
struct SvRaw32 { float v[8]; };
struct SvRaw16 { uint4 v; };
PS_D void sv_get(SvRaw32 &r, const float *p, int mode, uint32_t live) { // mode 2: 32 bytes at once, 1: twice 16, 0: one by one, the live ones
    if (mode == 2) {
        asm volatile("ld.global.nc.L1::no_allocate.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=f"(r.v[0]), "=f"(r.v[1]), "=f"(r.v[2]), "=f"(r.v[3]), "=f"(r.v[4]), "=f"(r.v[5]), "=f"(r.v[6]), "=f"(r.v[7]) : "l"(p));
    } else if (mode == 1) {
        const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
        r.v[0] = a.x; r.v[1] = a.y; r.v[2] = a.z; r.v[3] = a.w; r.v[4] = b.x; r.v[5] = b.y; r.v[6] = b.z; r.v[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) r.v[i] = live >> i & 1 ? __ldg(p + i) : 0.f;
    }
}
PS_D void sv_get(SvRaw16 &r, const __nv_bfloat16 *p, int mode, uint32_t live) {
    if (mode) r.v = __ldg(reinterpret_cast<const uint4 *>(p));
    else {
        uint32_t w[4] = {};
        const uint16_t *u = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (live >> i & 1) w[i / 2] |= (uint32_t)__ldg(u + i) << (16 * (i & 1));
        r.v = make_uint4(w[0], w[1], w[2], w[3]);
    }
}
PS_D void sv_zero(SvRaw32 &r) {
#pragma unroll
    for (int i = 0; i < 8; i++) r.v[i] = 0.f;
}
PS_D void sv_zero(SvRaw16 &r) { r.v = make_uint4(0, 0, 0, 0); }
PS_D float sv_at(const SvRaw32 &r, int i) { return r.v[i]; }
PS_D float sv_at(const SvRaw16 &r, int i) {
    const uint32_t w = i < 2 ? r.v.x : i < 4 ? r.v.y : i < 6 ? r.v.z : r.v.w;
    return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
}
template <typename R> PS_D void sv_keep(R &r, uint32_t live);
template <> PS_D void sv_keep<SvRaw32>(SvRaw32 &r, uint32_t live) {
#pragma unroll
    for (int i = 0; i < 8; i++) r.v[i] = live >> i & 1 ? r.v[i] : 0.f;
}
template <> PS_D void sv_keep<SvRaw16>(SvRaw16 &r, uint32_t live) {
    uint32_t *w = &r.v.x;
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (!(live >> i & 1)) w[i / 2] &= i & 1 ? 0x0000ffffu : 0xffff0000u;
}

template <typename T, int D> struct SvTc {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int PARTS = F32 ? 2 : 1;
    static constexpr int KPART = SV_TILE * D * 2;                     // bytes of one part of a tile of K or of V
    static constexpr int STAGE = PARTS * KPART;
    static constexpr int Q = 2 * SV_TC_ROWS * D * 2;                  // both parts of the queries
    static constexpr int SMEM = Q + 4 * STAGE + 1024;
    static constexpr int ITS = D / 16;                                // eights that a loading thread holds
    using Raw = typename std::conditional<F32, SvRaw32, SvRaw16>::type;
};

template <typename T, int D>
__global__ void __launch_bounds__(SV_TC_THREADS, 1) sv_k_attn_tc(const __grid_constant__ SvAttn a) {
    using C = SvTc<T, D>;
    using Raw = typename C::Raw;
    extern __shared__ __align__(1024) uint8_t sv_tc_raw[];
    __shared__ __align__(8) uint64_t full_k[2], full_v[2], s_full[2], s_empty[2], p_full[2], o_full[2], o_empty[2], done;
    __shared__ uint32_t tmem_smem;
    __shared__ float s_alpha[2][SV_TC_ROWS], s_kinv[2][4], s_vinv[2][4], s_qinv[SV_TC_ROWS], s_sum[SV_TC_ROWS];
    __shared__ uint64_t s_live[SV_TC_TILES];
    uint8_t *smem = reinterpret_cast<uint8_t *>(((uintptr_t)sv_tc_raw + 1023) & ~(uintptr_t)1023);
    uint8_t *sm_q = smem, *sm_k = smem + C::Q, *sm_v = sm_k + 2 * C::STAGE;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int si = sv_find(a, blockIdx.x), split = blockIdx.x - a.seq[si].unit0, g = blockIdx.y;
    const SvSeq &s = a.seq[si];
    const int all_rows = s.n_tok * a.R, r0 = blockIdx.z * SV_TC_ROWS, rows = min(all_rows - r0, SV_TC_ROWS);
    if (rows <= 0) return;
    const int j0 = split * a.tps * SV_TILE, j_end = min(s.n_kv, j0 + a.tps * SV_TILE), tiles = (j_end - j0 + SV_TILE - 1) / SV_TILE, past = s.n_kv - s.n_tok;

    if (tid == 0) {
        for (int b = 0; b < 2; b++) {
            ps_mbar_init(&full_k[b], 4); ps_mbar_init(&full_v[b], 4); ps_mbar_init(&s_full[b], 1); ps_mbar_init(&s_empty[b], 4);
            ps_mbar_init(&p_full[b], 4); ps_mbar_init(&o_full[b], 1); ps_mbar_init(&o_empty[b], 8);
        }
        ps_mbar_init(&done, 1);
        ps_fence_barrier_init();
    }
    if (warp == 20) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(ps_smem_u32(&tmem_smem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // live slots of a tile: in the split and not hidden
    auto in_split = [&](int t) -> uint64_t {
        const int n = j_end - j0 - t * SV_TILE;
        return n >= SV_TILE ? ~0ull : (1ull << n) - 1;
    };
    if (s.hidden)
        for (int t = warp; t < tiles; t += SV_TC_THREADS / 32) {
            const int j = j0 + t * SV_TILE + lane;
            const uint32_t lo = __ballot_sync(0xffffffffu, j < j_end && !s.hidden[min(j, j_end - 1)]), hi = __ballot_sync(0xffffffffu, j + 32 < j_end && !s.hidden[min(j + 32, j_end - 1)]);
            if (lane == 0) s_live[t] = (uint64_t)hi << 32 | lo;
        }
    auto live_of = [&](int t) -> uint64_t { return s.hidden ? s_live[t] : in_split(t); };
    // queries: a half-warp (quarter-warp for head size 64) per row
    for (int i = tid; i < rows * (D / 8); i += SV_TC_THREADS) { // (rows * D / 8 is a multiple of D / 8: the lanes of a row are there together)
        const int r = i / (D / 8), c = i % (D / 8), row = r0 + r;
        const float *q = a.q + ((int64_t)(s.tok0 + row / a.R) * a.n_heads + g * a.R + row % a.R) * D + c * 8;
        const unsigned mates = (D == 128 ? 0xffffu : 0xffu) << (lane & (D == 128 ? 16 : 24));
        float x[8], inv;
        uint32_t mx = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            x[e] = q[e] * a.scale;
            mx = max(mx, __float_as_uint(x[e]) & 0x7fffffffu);
        }
#pragma unroll
        for (int o = D / 16; o; o >>= 1) mx = max(mx, __shfl_xor_sync(mates, mx, o));
        const float f = sv_scale(mx, inv);
        uint4 hi, lo;
        sv_cut(x[0] * f, x[1] * f, hi.x, lo.x);
        sv_cut(x[2] * f, x[3] * f, hi.y, lo.y);
        sv_cut(x[4] * f, x[5] * f, hi.z, lo.z);
        sv_cut(x[6] * f, x[7] * f, hi.w, lo.w);
        *reinterpret_cast<uint4 *>(sm_q + c * (SV_TC_ROWS * 16) + r * 16) = hi;
        *reinterpret_cast<uint4 *>(sm_q + C::Q / 2 + c * (SV_TC_ROWS * 16) + r * 16) = lo;
        if (c == 0) s_qinv[r] = inv;
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    ps_tc_fence_before();
    __syncthreads();
    ps_tc_fence_after();
    const uint32_t tm = tmem_smem, tm_s = tm, tm_p = tm + 2 * SV_TILE, tm_o = tm + 4 * SV_TILE; // columns: scores 2 x 64, weights 2 x (32 + 32), outputs 2 x D
    bool ok = true;

    if (warp >= 12 && warp < 20) {
        // ===== loaders: K by warps 12-15 (16 slots each), V by warps 16-19 (D / 4 channels each).  A thread's eights: lane % 8 picks one of eight rows (slots of
        // K, channels of V), lane / 8 one of four neighbouring eights of the row: a warp's load is 8 rows x 128 bytes, its store eight times 128 bytes
        const bool is_v = warp >= 16;
        const int w = warp & 3, sub = lane & 7, quad = lane >> 3;
        const int64_t ld = is_v ? s.n_ctx : (int64_t)a.G * D;
        const T *base = static_cast<const T *>(is_v ? s.v : s.k) + (is_v ? ((int64_t)g * D + w * (D / 4) + sub) * ld : (int64_t)g * D);
        const int mode = is_v ? s.v_mode : s.k_mode;
        uint8_t *sm = is_v ? sm_v : sm_k;
        uint64_t *full = is_v ? full_v : full_k, *empty = is_v ? o_empty : s_empty;
        Raw raw[C::ITS];
        auto load = [&](int t) {
            const uint64_t live = live_of(t);
            const int j = j0 + t * SV_TILE;
#pragma unroll
            for (int i = 0; i < C::ITS; i++) {
                if (is_v) { // i: channel group (of eight), half of the tile
                    const int chunk = quad + 4 * (i & 1);
                    const uint32_t m = (uint32_t)(live >> (8 * chunk)) & 0xffu;
                    if (m) sv_get(raw[i], base + (int64_t)(i >> 1) * 8 * ld + j + 8 * chunk, mode, m);
                    else sv_zero(raw[i]);
                } else {    // i: slot group (of eight), four eights of the row
                    const int slot = w * 16 + (i / (D / 32)) * 8 + sub;
                    if (live >> slot & 1) sv_get(raw[i], base + (int64_t)(j + slot) * ld + ((i % (D / 32)) * 4 + quad) * 8, mode, 0xffu);
                    else sv_zero(raw[i]);
                }
            }
        };
        load(0);
        for (int t = 0; t < tiles && ok; t++) {
            const int b = t & 1;
            if (is_v) {
                const uint64_t live = live_of(t);
                if (live != ~0ull) {
#pragma unroll
                    for (int i = 0; i < C::ITS; i++) sv_keep(raw[i], (uint32_t)(live >> (8 * (quad + 4 * (i & 1)))) & 0xffu);
                }
            }
            uint32_t mx = 0;
#pragma unroll
            for (int i = 0; i < C::ITS; i++)
#pragma unroll
                for (int e = 0; e < 8; e++) mx = max(mx, __float_as_uint(sv_at(raw[i], e)) & 0x7fffffffu);
            mx = __reduce_max_sync(0xffffffffu, mx);
            float inv;
            const float f = sv_scale(mx, inv);
            if (t >= 2) sv_bar_wait(&empty[b], ((t >> 1) - 1) & 1, ok, a.err, 11);
            if (!ok) break;
            uint8_t *to = sm + b * C::STAGE;
#pragma unroll
            for (int i = 0; i < C::ITS; i++) {
                uint4 hi, lo;
                sv_cut(sv_at(raw[i], 0) * f, sv_at(raw[i], 1) * f, hi.x, lo.x);
                sv_cut(sv_at(raw[i], 2) * f, sv_at(raw[i], 3) * f, hi.y, lo.y);
                sv_cut(sv_at(raw[i], 4) * f, sv_at(raw[i], 5) * f, hi.z, lo.z);
                sv_cut(sv_at(raw[i], 6) * f, sv_at(raw[i], 7) * f, hi.w, lo.w);
                const int at = is_v ? (quad + 4 * (i & 1)) * (D * 16) + (w * (D / 4) + (i >> 1) * 8 + sub) * 16
                                    : ((i % (D / 32)) * 4 + quad) * (SV_TILE * 16) + (w * 16 + (i / (D / 32)) * 8 + sub) * 16;
                *reinterpret_cast<uint4 *>(to + at) = hi;
                if (C::F32) *reinterpret_cast<uint4 *>(to + C::KPART + at) = lo;
            }
            if (lane == 0) (is_v ? s_vinv : s_kinv)[b][w] = inv;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) ps_mbar_arrive(&full[b]);
            if (t + 1 < tiles) load(t + 1);
        }
    } else if (warp == 20) {
        // ===== MMAs.  Small products first, while the truncating accumulator is small
        const uint32_t idesc_s = (1u << 4) | ((uint32_t)(SV_TILE >> 3) << 17) | ((uint32_t)(SV_TC_ROWS >> 4) << 24);
        const uint32_t idesc_o = (1u << 4) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(SV_TC_ROWS >> 4) << 24);
        const uint64_t dq = ps_tc_smem_desc(ps_smem_u32(sm_q), SV_TC_ROWS * 16, 128), dk = ps_tc_smem_desc(ps_smem_u32(sm_k), SV_TILE * 16, 128), dv = ps_tc_smem_desc(ps_smem_u32(sm_v), D * 16, 128);
        auto scores = [&](int t) {
            const int b = t & 1;
            sv_bar_wait(&full_k[b], (t >> 1) & 1, ok, a.err, 12);
            if (t >= 2) sv_bar_wait(&s_empty[b], ((t >> 1) - 1) & 1, ok, a.err, 13);
            if (!ok) return;
            ps_tc_fence_after();
            if (ps_elect_one()) {
                const uint64_t kb = dk + (uint64_t)(b * (C::STAGE >> 4));
                const uint32_t to = tm_s + b * SV_TILE;
#pragma unroll
                for (int p = 0; p < C::PARTS + 1; p++) // lo hi, hi lo, hi hi (bfloat16 caches: lo hi, hi hi)
#pragma unroll
                    for (int j = 0; j < D / 16; j++)
                        ps_tc_mma_f16(to, dq + (p == 0 ? (C::Q / 2) >> 4 : 0) + j * ((2 * SV_TC_ROWS * 16) >> 4), kb + (C::F32 && p == 1 ? C::KPART >> 4 : 0) + j * ((2 * SV_TILE * 16) >> 4), idesc_s, (p | j) != 0);
                ps_tc_commit(&s_full[b]);
            }
            __syncwarp();
        };
        if (tiles > 0) scores(0);
        for (int t = 0; t < tiles && ok; t++) {
            const int b = t & 1;
            if (t + 1 < tiles) scores(t + 1);
            sv_bar_wait(&full_v[b], (t >> 1) & 1, ok, a.err, 14);
            sv_bar_wait(&p_full[b], (t >> 1) & 1, ok, a.err, 15); // (the soft-max has waited for the output of tile t - 2)
            if (!ok) break;
            ps_tc_fence_after();
            if (ps_elect_one()) {
                const uint64_t vb = dv + (uint64_t)(b * (C::STAGE >> 4));
                const uint32_t to = tm_o + b * D, pa = tm_p + b * SV_TILE;
#pragma unroll
                for (int p = 0; p < C::PARTS + 1; p++)
#pragma unroll
                    for (int j = 0; j < SV_TILE / 16; j++)
                        ps_tc_mma_f16_ta(to, pa + (p == 0 ? SV_TILE / 2 : 0) + j * 8, vb + (C::F32 && p == 1 ? C::KPART >> 4 : 0) + j * ((2 * D * 16) >> 4), idesc_o, (p | j) != 0);
                ps_tc_commit(&o_full[b]);
            }
            __syncwarp();
        }
        if (ps_elect_one()) ps_tc_commit(&done); // MMAs in flight end before the tensor memory is given back
        __syncwarp();
        if (!ps_tc_wait_warp(&done, 0)) *a.err = 16;
    } else if (warp < 4) {
        // ===== soft-max: thread = row
        const int r = warp * 32 + lane, row = r0 + r;
        const bool mine = r < rows, any = warp * 32 < rows; // (any: of the warp)
        const uint32_t lane_at = (uint32_t)(warp * 32) << 16;
        const float qinv = mine ? s_qinv[r] : 0.f;
        const int tok = row / a.R;
        const int rp = sv_rp(all_rows);
        float m = SV_NONE, l = 0.f;
        for (int t = 0; t < tiles && ok; t++) {
            const int b = t & 1, j = j0 + t * SV_TILE;
            uint64_t see = live_of(t);
            if (j + SV_TILE > past && any) { // of the step's own slots those that this token sees
                for (int c = max(0, past - j); c < min(SV_TILE, j_end - j); c++)
                    if (mine && !sv_sees(s, tok, j + c - past)) see &= ~(1ull << c);
            }
            sv_bar_wait(&full_k[b], (t >> 1) & 1, ok, a.err, 17); // (the groups' factors)
            sv_bar_wait(&s_full[b], (t >> 1) & 1, ok, a.err, 18);
            if (!ok) break;
            ps_tc_fence_after();
            __syncwarp();
            uint32_t v[SV_TILE];
            if (any) {
#pragma unroll
                for (int c = 0; c < SV_TILE; c += 32)
                    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                                 : "=r"(v[c]), "=r"(v[c + 1]), "=r"(v[c + 2]), "=r"(v[c + 3]), "=r"(v[c + 4]), "=r"(v[c + 5]), "=r"(v[c + 6]), "=r"(v[c + 7]), "=r"(v[c + 8]), "=r"(v[c + 9]),
                                   "=r"(v[c + 10]), "=r"(v[c + 11]), "=r"(v[c + 12]), "=r"(v[c + 13]), "=r"(v[c + 14]), "=r"(v[c + 15]), "=r"(v[c + 16]), "=r"(v[c + 17]), "=r"(v[c + 18]),
                                   "=r"(v[c + 19]), "=r"(v[c + 20]), "=r"(v[c + 21]), "=r"(v[c + 22]), "=r"(v[c + 23]), "=r"(v[c + 24]), "=r"(v[c + 25]), "=r"(v[c + 26]), "=r"(v[c + 27]),
                                   "=r"(v[c + 28]), "=r"(v[c + 29]), "=r"(v[c + 30]), "=r"(v[c + 31])
                                 : "r"(tm_s + b * SV_TILE + c + lane_at)
                                 : "memory");
                ps_tc_ld_wait();
            }
            float f[4];
#pragma unroll
            for (int k = 0; k < 4; k++) f[k] = qinv * s_kinv[b][k];
            ps_tc_fence_before();
            __syncwarp();
            if (lane == 0) ps_mbar_arrive(&s_empty[b]);
            float mx = SV_NONE;
            if (any) {
                const bool whole = __all_sync(0xffffffffu, see == ~0ull);
#pragma unroll
                for (int c = 0; c < SV_TILE; c++) {
                    float z = __uint_as_float(v[c]) * f[c / 16];
                    if (!whole) z = see >> c & 1 ? z : SV_NONE;
                    v[c] = __float_as_uint(z);
                    mx = fmaxf(mx, z);
                }
                if (s.scores && mine) {
                    float *to = s.scores + ((int64_t)g * s.n_kv + j) * rp + row;
                    const int n = min(SV_TILE, j_end - j);
#pragma unroll
                    for (int c = 0; c < SV_TILE; c++)
                        if (c < n) to[(int64_t)c * rp] = __uint_as_float(v[c]);
                }
            }
            const float mn = fmaxf(m, mx), ref = mn == SV_NONE ? 0.f : mn, alpha = sv_ex2(m - ref);
            m = mn;
            if (t >= 2) sv_bar_wait(&o_empty[b], ((t >> 1) - 1) & 1, ok, a.err, 19); // (its weights are used up, and its factors)
            if (!ok) break;
            s_alpha[b][r] = alpha;
            __syncwarp();
            if (any) {
                float sum = 0.f;
#pragma unroll
                for (int c = 0; c < SV_TILE; c += 16) {
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float p0 = sv_ex2(__uint_as_float(v[c + 2 * e]) - ref), p1 = sv_ex2(__uint_as_float(v[c + 2 * e + 1]) - ref);
                        sum += p0 + p1;
                        sv_cut(p0 * 32768.f, p1 * 32768.f, hi[e], lo[e]);
                    }
                    const uint32_t to = tm_p + b * SV_TILE + c / 2 + lane_at;
                    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(to), "r"(hi[0]), "r"(hi[1]), "r"(hi[2]), "r"(hi[3]), "r"(hi[4]), "r"(hi[5]), "r"(hi[6]),
                                 "r"(hi[7]) : "memory");
                    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(to + SV_TILE / 2), "r"(lo[0]), "r"(lo[1]), "r"(lo[2]), "r"(lo[3]), "r"(lo[4]), "r"(lo[5]),
                                 "r"(lo[6]), "r"(lo[7]) : "memory");
                }
                l = fmaf(l, alpha, sum);
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            }
            ps_tc_fence_before();
            __syncwarp();
            if (lane == 0) ps_mbar_arrive(&p_full[b]);
        }
        if (mine) {
            s_sum[r] = l;
            reinterpret_cast<float2 *>(s.part + (int64_t)s.splits * a.G * all_rows * D)[((int64_t)split * a.G + g) * all_rows + row] = make_float2(m, l);
        }
    }
    float acc[D / 2];
    if (warp >= 4 && warp < 12) {
        // ===== output: thread = row, half of the channels
        const int half = (warp - 4) >> 2, r = (warp & 3) * 32 + lane;
        const bool any = (warp & 3) * 32 < rows;
        const uint32_t lane_at = (uint32_t)((warp & 3) * 32) << 16;
#pragma unroll
        for (int c = 0; c < D / 2; c++) acc[c] = 0.f;
        for (int t = 0; t < tiles && ok; t++) {
            const int b = t & 1;
            sv_bar_wait(&full_v[b], (t >> 1) & 1, ok, a.err, 20);
            sv_bar_wait(&p_full[b], (t >> 1) & 1, ok, a.err, 21);
            sv_bar_wait(&o_full[b], (t >> 1) & 1, ok, a.err, 22);
            if (!ok) break;
            ps_tc_fence_after();
            if (any) {
                const float alpha = s_alpha[b][r];
                const float f[2] = {s_vinv[b][half * 2], s_vinv[b][half * 2 + 1]};
#pragma unroll
                for (int c = 0; c < D / 2; c += 16) {
                    uint32_t v[16];
                    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
                                   "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                                 : "r"(tm_o + b * D + half * (D / 2) + c + lane_at)
                                 : "memory");
                    ps_tc_ld_wait();
#pragma unroll
                    for (int e = 0; e < 16; e++) acc[c + e] = fmaf(acc[c + e], alpha, __uint_as_float(v[e]) * f[(c + e) / (D / 4)]);
                }
            }
            ps_tc_fence_before();
            __syncwarp();
            if (lane == 0) ps_mbar_arrive(&o_empty[b]);
        }
    }
    ps_tc_fence_before();
    __syncthreads();
    if (warp == 20) {
        ps_tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tm) : "memory");
    }
    if (warp >= 4 && warp < 12) {
        const int half = (warp - 4) >> 2, r = (warp & 3) * 32 + lane, row = r0 + r;
        if (r < rows) {
            const float l = s_sum[r], f = (s.splits == 1 ? (l > 0.f ? 1.f / l : 0.f) : 1.f) * (1.f / 32768.f);
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
}
