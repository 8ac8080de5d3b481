// ps_page_rows.cuh - rows of K and V into blocks of 8-bit codes, and back.
//
//   scale' = max(scale, where earlier slots lie in the block; max |x| / 127),   code = rint(x / scale'),   earlier codes rint(code * (scale / scale'))
//
// store: a CTA takes a block of sixteen slots of one head's K or V, a thread sixteen of its numbers, which are read once: a slot's sixteen channels (K), a channel's sixteen slots (V), so that sixteen bytes a lane go to
// memory lane after lane.  Bound by instructions (the SMs issue 47 % of the time) and latency for prompts: 6 385 tokens of 8 heads of 128 in bfloat16 33 us, 1.2 TB/s;
// by latency (a chain of table, numbers, the CTA's largest) for single tokens.  (A warp a block, 64 numbers a lane: 55 us, for few warps an SM.  At 64 registers, which heads of 256 need for four CTAs an SM, 72 bytes a thread
// of numbers whose codes are asked again lie in local memory.)
// load: a warp a block.
#pragma once
#include "ps_page.cuh"

#define PG_ROW_WARPS 4

struct PgRowSeq {
    const int32_t *table;
    int n_kv, n_tok, tok0, block0;  // block0: number of its first block among all of the launch
};
struct PgRows {
    PgRowSeq seq[PG_SEQS];
    PgPool pool;
    void *k, *v;
    int n_seqs, blocks, k_vec, v_vec;       // vec: rows begin at 16-byte boundaries
};

struct PgRowTask { // a warp's block
    int kv, g, lo, hi;      // slots lo .. hi of the block are the call's
    int64_t at, row;        // number of the page's head; the call's row of the block's slot 0 (may be before the first)
    int block;              // of the page
    bool there;
};
PS_D PgRowTask pg_row_task(const PgRows &a, uint32_t task) {
    const int heads = 2 * a.pool.G;
    PgRowTask t;
    const int u = (int)(task / (uint32_t)heads), h = (int)(task % (uint32_t)heads);
    t.there = u < a.blocks;
    if (!t.there) return t;
    t.kv = h & 1; t.g = h >> 1;
    int lo = 0, hi = a.n_seqs - 1; // the last sequence that begins at or before block u
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (a.seq[mid].block0 <= u) lo = mid;
        else hi = mid - 1;
    }
    const PgRowSeq &s = a.seq[lo];
    const int first = s.n_kv - s.n_tok, b = first / PG_BLOCK + (u - s.block0), j0 = b * PG_BLOCK;
    t.lo = max(first - j0, 0);
    t.hi = min(s.n_kv - j0, PG_BLOCK);
    t.row = (int64_t)s.tok0 + j0 - first;
    const int page = s.table[j0 >> a.pool.shift];
    t.there = a.pool.has(page);
    t.at = t.there ? a.pool.at(page, t.g, t.kv) : 0;
    t.block = (j0 & (a.pool.P - 1)) / PG_BLOCK;
    return t;
}
template <typename T> PS_D void pg_get16(float (&x)[16], const T *p, bool vec) {
    if (vec) {
        constexpr int N = sizeof(T); // 16-byte words
        uint4 raw[N];
#pragma unroll
        for (int i = 0; i < N; i++) raw[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
        const T *r = reinterpret_cast<const T *>(raw);
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = pg_num(r[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = pg_num(p[i]);
    }
}
PS_D uint32_t pg_bytes_from(int n) { return n <= 0 ? ~0u : n >= 4 ? 0u : ~0u << (8 * n); } // a word's bytes n, n + 1, ...
// bytes below lo from `below`, below hi from x, the others from `above`
PS_D uint4 pg_three(const uint4 &below, const uint4 &x, const uint4 &above, int lo, int hi) {
    auto one = [&](uint32_t a, uint32_t b, uint32_t c, int at) {
        const uint32_t from_lo = pg_bytes_from(lo - at), from_hi = pg_bytes_from(hi - at);
        return (a & ~from_lo) | (b & from_lo & ~from_hi) | (c & from_hi);
    };
    return make_uint4(one(below.x, x.x, above.x, 0), one(below.y, x.y, above.y, 4), one(below.z, x.z, above.z, 8), one(below.w, x.w, above.w, 12));
}

// as many threads as a head has channels
template <typename T>
__global__ void __launch_bounds__(256, 4) pg_k_store(const __grid_constant__ PgRows a) {
    __shared__ float s_top[8];
    const int i = threadIdx.x, hs = blockDim.x, ld = a.pool.G * hs;
    const PgRowTask t = pg_row_task(a, blockIdx.x);
    if (!t.there) return; // (the whole CTA)
    const T *x = static_cast<const T *>(t.kv ? a.v : a.k) + (int64_t)t.g * hs;
    uint4 *codes = reinterpret_cast<uint4 *>(a.pool.codes + t.at * a.pool.page_codes() + (int64_t)t.block * PG_BLOCK * hs) + i;
    float *scale = a.pool.scales + t.at * (a.pool.P / PG_BLOCK) + t.block;
    const int second = i >= hs / 2, slot = second * 8 + (i & 7), c = (i - second * (hs / 2)) >> 3; // K's
    const bool part = t.lo > 0 || t.hi < 16;
    const float was = t.lo ? *scale : 0.f;
    uint4 old = make_uint4(0, 0, 0, 0);
    if (part) old = *codes;
    float n[16], top = 0.f;
    if (t.kv) {
        const T *x0 = x + t.row * ld + i;
#pragma unroll
        for (int s = 0; s < 16; s++) n[s] = s >= t.lo && s < t.hi ? pg_num(x0[s * ld]) : 0.f;
    } else if (slot >= t.lo && slot < t.hi) pg_get16(n, x + (t.row + slot) * ld + c * 16, a.k_vec);
    else {
#pragma unroll
        for (int s = 0; s < 16; s++) n[s] = 0.f;
    }
#pragma unroll
    for (int s = 0; s < 16; s++) top = fmaxf(top, fabsf(n[s])); // (fmaxf passes over what is no number)
    top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
    if ((i & 31) == 0) s_top[i >> 5] = top;
    __syncthreads();
    for (int w = 0; w < hs / 32; w++) top = fmaxf(top, s_top[w]);
    const float now = fmaxf(was, __fdiv_rn(top, 127.f));
    const uint4 codes_now = PgDivide(now)(n);
    if (!part) *codes = codes_now;
    else {
        uint4 r = old;
        if (t.lo > 0 && now != was) { // codes that stay get another scale
            const float f = pg_follow(was, now);
            r = make_uint4(pg_recode4(old.x, f), pg_recode4(old.y, f), pg_recode4(old.z, f), pg_recode4(old.w, f));
        }
        if (t.kv) *codes = pg_three(r, codes_now, old, t.lo, t.hi);
        else if (slot < t.hi) *codes = slot < t.lo ? r : codes_now;
    }
    if (i == 0) *scale = now;
}

template <typename T>
__global__ void __launch_bounds__(32 * PG_ROW_WARPS) pg_k_load(const __grid_constant__ PgRows a) {
    const int lane = threadIdx.x & 31, hs = a.pool.hs, ld = a.pool.G * hs;
    const PgRowTask t = pg_row_task(a, blockIdx.x * PG_ROW_WARPS + (threadIdx.x >> 5));
    T *x = static_cast<T *>(t.there ? (t.kv ? a.v : a.k) : nullptr);
    if (!x) return;
    x += (int64_t)t.g * hs;
    const uint4 *codes = reinterpret_cast<const uint4 *>(a.pool.codes + t.at * a.pool.page_codes() + (int64_t)t.block * PG_BLOCK * hs);
    const float scale = a.pool.scales[t.at * (a.pool.P / PG_BLOCK) + t.block];
    for (int i = lane; i < hs; i += 32) {
        const uint4 c = codes[i];
        if (t.kv) {
#pragma unroll
            for (int s = 0; s < 16; s++)
                if (s >= t.lo && s < t.hi) (x + t.row * ld + i)[s * ld] = pg_to<T>((float)pg_byte(c, s) * scale);
        } else {
            const int second = i >= hs / 2, slot = second * 8 + (i & 7), ch = (i - second * (hs / 2)) >> 3;
            if (slot < t.lo || slot >= t.hi) continue;
            T *to = x + (t.row + slot) * ld + ch * 16;
            alignas(16) T n[16];
#pragma unroll
            for (int s = 0; s < 16; s++) n[s] = pg_to<T>((float)pg_byte(c, s) * scale);
            if (a.k_vec) {
#pragma unroll
                for (int s = 0; s < (int)sizeof(T); s++) reinterpret_cast<uint4 *>(to)[s] = reinterpret_cast<const uint4 *>(n)[s];
            } else {
#pragma unroll
                for (int s = 0; s < 16; s++) to[s] = n[s];
            }
        }
    }
}
