// ps_page_rows.cuh - rows of K and V into blocks of 8-bit codes, and back.
//
//   scale' = max(scale, where earlier slots lie in the block; max |x| / 127),   code = rint(x / scale'),   earlier codes rint(code * (scale / scale'))
//
// A warp takes a block of sixteen slots of one head's K or V: it holds the block's numbers, so that they are read once, finds their largest by shuffles, and writes sixteen bytes a lane, lane after
// lane.  K: a lane's item is a slot's sixteen channels; V: a channel's sixteen slots.  Bound by memory for prompts, by latency (a chain of table, scale, numbers) for single tokens.
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
PS_D PgRowTask pg_row_task(const PgRows &a) {
    const int heads = 2 * a.pool.G;
    const int64_t task = (int64_t)blockIdx.x * PG_ROW_WARPS + (threadIdx.x >> 5);
    PgRowTask t;
    t.there = task < (int64_t)a.blocks * heads;
    if (!t.there) return t;
    const int u = (int)(task / heads), h = (int)(task % heads);
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
PS_D uint4 pg_pack(const int (&c)[16]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = (uint32_t)(c[4 * i] & 255) | (uint32_t)(c[4 * i + 1] & 255) << 8 | (uint32_t)(c[4 * i + 2] & 255) << 16 | (uint32_t)c[4 * i + 3] << 24;
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// ITEMS: head size / 32
template <typename T, int ITEMS>
__global__ void __launch_bounds__(32 * PG_ROW_WARPS) pg_k_store(const __grid_constant__ PgRows a) {
    const int lane = threadIdx.x & 31, hs = 32 * ITEMS, ld = a.pool.G * hs;
    const PgRowTask t = pg_row_task(a);
    if (!t.there) return;
    const T *x = static_cast<const T *>(t.kv ? a.v : a.k) + (int64_t)t.g * hs;
    uint4 *codes = reinterpret_cast<uint4 *>(a.pool.codes + t.at * a.pool.page_codes() + (int64_t)t.block * PG_BLOCK * hs);
    float *scale = a.pool.scales + t.at * (a.pool.P / PG_BLOCK) + t.block;
    const float was = t.lo ? *scale : 0.f;
    float n[ITEMS][16], top = 0.f;
#pragma unroll
    for (int e = 0; e < ITEMS; e++) {
        const int i = e * 32 + lane;
        if (t.kv) {         // channel i of every slot
#pragma unroll
            for (int s = 0; s < 16; s++) n[e][s] = s >= t.lo && s < t.hi ? pg_num(x[(t.row + s) * ld + i]) : 0.f;
        } else {            // slot, sixteen channels
            const int slot = i / (hs / 2) * 8 + i % 8, c = i % (hs / 2) / 8;
            if (slot >= t.lo && slot < t.hi) pg_get16(n[e], x + (t.row + slot) * ld + c * 16, a.k_vec);
            else {
#pragma unroll
                for (int s = 0; s < 16; s++) n[e][s] = 0.f;
            }
        }
#pragma unroll
        for (int s = 0; s < 16; s++) top = fmaxf(top, fabsf(n[e][s])); // (fmaxf passes over what is no number)
    }
    const float now = fmaxf(was, __fdiv_rn(pg_warp_max(top), 127.f)), f = pg_follow(was, now);
    const bool move = t.lo > 0 && now != was; // codes that stay get another scale
#pragma unroll
    for (int e = 0; e < ITEMS; e++) {
        const int i = e * 32 + lane;
        int c[16];
#pragma unroll
        for (int s = 0; s < 16; s++) c[s] = pg_code(n[e][s], now);
        if (t.kv) {
            if (t.lo > 0 || t.hi < 16) {
                const uint4 old = codes[i];
#pragma unroll
                for (int s = 0; s < 16; s++) {
                    const int o = pg_byte(old, s);
                    if (s < t.lo) c[s] = move ? pg_recode(o, f) : o;
                    else if (s >= t.hi) c[s] = o;
                }
            }
            codes[i] = pg_pack(c);
        } else {
            const int slot = i / (hs / 2) * 8 + i % 8;
            if (slot >= t.lo && slot < t.hi) codes[i] = pg_pack(c);
            else if (slot < t.lo && move) {
                const uint4 old = codes[i];
#pragma unroll
                for (int s = 0; s < 16; s++) c[s] = pg_recode(pg_byte(old, s), f);
                codes[i] = pg_pack(c);
            }
        }
    }
    if (lane == 0) *scale = now;
}

template <typename T>
__global__ void __launch_bounds__(32 * PG_ROW_WARPS) pg_k_load(const __grid_constant__ PgRows a) {
    const int lane = threadIdx.x & 31, hs = a.pool.hs, ld = a.pool.G * hs;
    const PgRowTask t = pg_row_task(a);
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
                if (s >= t.lo && s < t.hi) x[(t.row + s) * ld + i] = pg_to<T>((float)pg_byte(c, s) * scale);
        } else {
            const int slot = i / (hs / 2) * 8 + i % 8, ch = i % (hs / 2) / 8;
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
