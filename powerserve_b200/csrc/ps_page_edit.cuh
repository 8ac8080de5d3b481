// ps_page_edit.cuh - pages taken, shared, given back and copied; slots that move together.
//
// A page is free where no table holds it (refs = 0), and growth takes the free pages of the lowest numbers: so what is handed out depends on the tables alone, not on the order in which threads come.
// Counts are changed by whole-number atomics, whose order does not matter, in three phases that the CTA passes together: shares, releases, growth.
#pragma once
#include "ps_page.cuh"

#define PG_EDIT_THREADS 1024

struct PgEditOp {
    int32_t *table;
    const int32_t *from;
    int32_t n_old, n_new;
};
struct PgEdits {
    PgEditOp op[PS_CUDA_EDITS];
    int32_t *refs, *held;
    int4 *copies;           // [n]: source, destination (-1: none), blocks; or null, where none can be
    int32_t *free;          // room for the numbers of all pages that the edits can ask for
    int n, n_pages, shift;
    int *err;
};
struct PgCopies {
    PgPool pool;
    const int4 *copies;
    int64_t layer_codes, layer_scales;
};

PS_D int pg_scan(int v, int *warp_sum, int &all) { // sum of the threads before this one, and of all
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
    }
    __syncthreads();
    if (lane == 31) warp_sum[warp] = inc;
    __syncthreads();
    const int w = lane < (int)blockDim.x / 32 ? warp_sum[lane] : 0;
    int before = warp > lane ? w : 0, total = w;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        before += __shfl_xor_sync(0xffffffffu, before, o);
        total += __shfl_xor_sync(0xffffffffu, total, o);
    }
    all = total;
    return before + inc - v;
}

// One CTA: bound by latency, a few dependent rounds of loads and atomics; the search for free pages reads 16 KB of counts at a time and ends when it has found enough
__global__ void __launch_bounds__(PG_EDIT_THREADS) pg_k_edit(const __grid_constant__ PgEdits a) {
    int32_t *pg_free = a.free; // numbers of free pages, rising
    __shared__ int s_last[PS_CUDA_EDITS], s_first[PS_CUDA_EDITS], s_need[PS_CUDA_EDITS], s_warp[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, P = 1 << a.shift, warps = PG_EDIT_THREADS / 32;
    auto pages = [&](int n) { return (n + P - 1) >> a.shift; };
    auto good = [&](int page) {
        const bool ok = (unsigned)page < (unsigned)a.n_pages;
        if (!ok) *a.err = PS_ERR_PAGE;
        return ok;
    };
    for (int e = warp; e < a.n; e += warps) {
        const PgEditOp &op = a.op[e];
        if (!op.from) continue;
        for (int i = lane; i < pages(op.n_old); i += 32) {
            const int page = op.from[i];
            op.table[i] = page;
            if (good(page)) atomicAdd(a.refs + page, 1);
        }
    }
    __syncthreads();
    for (int e = warp; e < a.n; e += warps) {
        const PgEditOp &op = a.op[e];
        for (int i = pages(op.n_new) + lane; i < pages(op.n_old); i += 32) {
            const int page = op.table[i];
            if (good(page) && atomicSub(a.refs + page, 1) <= 0) { // (nobody held it: it stays free)
                atomicAdd(a.refs + page, 1);
                *a.err = PS_ERR_PAGE;
            }
        }
    }
    __syncthreads();
    // growth: thread = edit
    const bool mine = tid < a.n;
    const int n_old = mine ? a.op[tid].n_old : 0, n_new = mine ? a.op[tid].n_new : 0;
    const bool grows = n_new > n_old, part = grows && (n_old & (P - 1));
    const int had = pages(n_old);
    int last = -1;
    if (part) {
        last = a.op[tid].table[had - 1];
        if (!good(last)) last = -1;
    }
    if (mine) s_last[tid] = last;
    __syncthreads();
    int rank = 0; // of those that grow from the same page
    if (last >= 0)
        for (int e = 0; e < tid; e++) rank += s_last[e] == last;
    const bool copy = last >= 0 && *static_cast<volatile int32_t *>(a.refs + last) - rank > 1;
    int need = grows ? (int)copy + pages(n_new) - had : 0, want;
    const int before = pg_scan(need, s_warp, want);
    int found = 0;
    if (want > 0) { // (all threads agree)
        const bool vec = (reinterpret_cast<uintptr_t>(a.refs) & 15) == 0;
        for (int p0 = 0; p0 < a.n_pages && found < want; p0 += 4 * PG_EDIT_THREADS) {
            const int p = p0 + 4 * tid;
            int r[4];
            if (vec && p + 4 <= a.n_pages) {
                const int4 v = __ldcg(reinterpret_cast<const int4 *>(a.refs + p));
                r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w;
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) r[i] = p + i < a.n_pages ? __ldcg(a.refs + p + i) : 1;
            }
            int all, at = found + pg_scan((r[0] == 0) + (r[1] == 0) + (r[2] == 0) + (r[3] == 0), s_warp, all);
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (r[i] == 0) {
                    if (at < want) pg_free[at] = p + i;
                    at++;
                }
            found += all;
        }
    }
    // the first edit that finds too few ends the handing out, for those behind it too, but for who needs no page and shares none with one before
    const bool fits = before + need <= found || (need == 0 && rank == 0);
    if (!fits) need = 0;
    __syncthreads();
    if (mine) {
        s_need[tid] = need;
        s_first[tid] = before;
        if (a.held) a.held[tid] = grows && !fits ? n_old : n_new;
        const bool copies = copy && fits;
        if (a.copies) a.copies[tid] = make_int4(last, copies ? pg_free[before] : -1, ((n_old & (P - 1)) + PG_BLOCK - 1) / PG_BLOCK, 0);
        if (copies) {
            atomicSub(a.refs + last, 1);
            s_last[tid] = had - 1; // where its pages begin in its table
        } else s_last[tid] = had;
    }
    __syncthreads();
    for (int e = warp; e < a.n; e += warps)
        for (int i = lane; i < s_need[e]; i += 32) {
            const int page = pg_free[s_first[e] + i];
            a.op[e].table[s_last[e] + i] = page;
            a.refs[page] = 1;
        }
}

// x: edit, y: layer, z: a share of its heads. The filled blocks of a page are one run of bytes a head's K or V
__global__ void __launch_bounds__(256) pg_k_copy(const __grid_constant__ PgCopies a) {
    ps_grid_dep_wait();
    const int4 c = a.copies[blockIdx.x];
    if (c.y < 0) return;
    const int hs = a.pool.hs, words = c.z * hs, n = 2 * a.pool.G, B = a.pool.P / PG_BLOCK; // 16-byte words, scales of a head's K or V
    const int64_t code0 = (int64_t)blockIdx.y * a.layer_codes, scale0 = (int64_t)blockIdx.y * a.layer_scales;
    for (int h = blockIdx.z; h < n; h += gridDim.z) {
        const int64_t from = a.pool.at(c.x, 0, 0) + h, to = a.pool.at(c.y, 0, 0) + h;
        const uint4 *src = reinterpret_cast<const uint4 *>(a.pool.codes + code0 + from * a.pool.page_codes());
        uint4 *dst = reinterpret_cast<uint4 *>(a.pool.codes + code0 + to * a.pool.page_codes());
        for (int i = threadIdx.x; i < words; i += 4 * 256) {
            uint4 v[4];
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (i + 256 * e < words) v[e] = __ldcs(src + i + 256 * e);
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (i + 256 * e < words) __stcs(dst + i + 256 * e, v[e]);
        }
        if ((int)threadIdx.x < c.z) a.pool.scales[scale0 + to * B + threadIdx.x] = a.pool.scales[scale0 + from * B + threadIdx.x];
    }
}

// ---------------------------------------------------------------------------------------------------- slots that move together
struct PgMoveOp {
    const int32_t *table, *keep, *n_dev;
    int first, n_kv, n_keep;
};
struct PgMoves {
    PgMoveOp op[PG_SEQS];
    PgPool pool;
    int64_t layer_codes, layer_scales;
};

// x: a layer's head's K or V, y: move.  A warp takes a block; the CTA's eight blocks are read before one of them is written, and what a later block reads lies behind it, as the list rises: so they may
// move in place.  ITEMS: head size / 32
template <int ITEMS>
__global__ void __launch_bounds__(256) pg_k_compact(const __grid_constant__ PgMoves a) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hs = 32 * ITEMS, B = a.pool.P / PG_BLOCK;
    const PgMoveOp &op = a.op[blockIdx.y];
    const int heads = 2 * a.pool.G, layer = blockIdx.x / heads, h = blockIdx.x % heads, kv = h & 1;
    int8_t *codes = a.pool.codes + (int64_t)layer * a.layer_codes + (int64_t)h * a.pool.page_codes();
    float *scales = a.pool.scales + (int64_t)layer * a.layer_scales + (int64_t)h * B;
    const int64_t page_codes = (int64_t)heads * a.pool.page_codes(), page_scales = (int64_t)heads * B;
    const int n_keep = op.n_dev ? min(*op.n_dev, op.n_keep) : op.n_keep;
    if (n_keep <= 0) return;
    const int b0 = op.first / PG_BLOCK, b1 = (op.first + n_keep - 1) / PG_BLOCK;
    bool bad = false;
    for (int b = b0; b <= b1; b += 8) {
        const int j = (b + warp) * PG_BLOCK + (lane & 15), i = j - op.first; // lane: a slot of the block
        const bool mine = b + warp <= b1 && lane < 16;
        // where the slot comes from: before `first`, itself
        int src = -1;
        if (mine && i < n_keep && !bad) {
            const int k = i < 0 ? 0 : op.keep[i], ahead = i <= 0 ? -1 : op.keep[i - 1];
            if (i < 0) src = j;
            else if (k >= i && k > ahead && k < op.n_kv - op.first) src = op.first + k;
        }
        bad = __syncthreads_or(bad || (mine && i < n_keep && src < 0)) != 0; // (the list ends here: these eight blocks stay as they are)
        if (bad) {
            if (threadIdx.x == 0) *a.pool.err = PS_ERR_PAGE;
            break;
        }
        int page = -1, to = -1;
        if (src >= 0) {
            page = op.table[src >> a.pool.shift];
            to = op.table[j >> a.pool.shift];
            if (!a.pool.has(page) || !a.pool.has(to)) page = to = -1;
        }
        const bool lost = __syncthreads_or(src >= 0 && page < 0) != 0;
        if (lost) break;
        const float was = page >= 0 ? scales[page * page_scales + (src & (a.pool.P - 1)) / PG_BLOCK] : 0.f;
        const float now = pg_warp_max(was), f = pg_follow(was, now);
        const unsigned live = __ballot_sync(0xffffffffu, page >= 0), moves = __ballot_sync(0xffffffffu, page >= 0 && (src != j || was != now));
        to = __shfl_sync(0xffffffffu, to, live ? __ffs(live) - 1 : 0); // (a block's slots are one page's)
        uint4 out[ITEMS];
        const int off = src & (a.pool.P - 1); // slot of the page
        int8_t *dst = codes + to * page_codes + (int64_t)((b + warp) * PG_BLOCK & (a.pool.P - 1)) * hs;
        if (moves) {
            if (kv) {       // a channel's sixteen slots, byte by byte
#pragma unroll
                for (int e = 0; e < ITEMS; e++) {
                    const int ch = e * 32 + lane;
                    out[e] = reinterpret_cast<const uint4 *>(dst)[ch]; // (slots behind the last one stay)
                }
                const int64_t base = page * page_codes + (int64_t)(off & ~15) * hs;
#pragma unroll
                for (int s = 0; s < 16; s++) {
                    if (!(live >> s & 1)) continue;
                    const int8_t *from = codes + __shfl_sync(0xffffffffu, base, s) + __shfl_sync(0xffffffffu, off & 15, s);
                    const float fs = __shfl_sync(0xffffffffu, f, s);
#pragma unroll
                    for (int e = 0; e < ITEMS; e++) {
                        const uint32_t c = (uint32_t)pg_recode(from[(e * 32 + lane) * 16], fs) & 255u;
                        uint32_t &w = s < 8 ? (s < 4 ? out[e].x : out[e].y) : (s < 12 ? out[e].z : out[e].w);
                        w = (w & ~(255u << (8 * (s & 3)))) | c << (8 * (s & 3));
                    }
                }
            } else {        // a slot's sixteen channels
                const int64_t base = page * page_codes + (int64_t)(off / 8) * 8 * hs + (off % 8) * 16;
#pragma unroll
                for (int e = 0; e < ITEMS; e++) {
                    const int it = e * 32 + lane, s = it / (hs / 2) * 8 + it % 8, c = it % (hs / 2) / 8;
                    const int64_t from = __shfl_sync(0xffffffffu, base, s);
                    const float fs = __shfl_sync(0xffffffffu, f, s);
                    if (!(live >> s & 1)) continue;
                    const uint4 v = *reinterpret_cast<const uint4 *>(codes + from + c * 128);
                    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        uint32_t r = 0;
#pragma unroll
                        for (int k = 0; k < 4; k++) r |= ((uint32_t)pg_recode((int8_t)(w[q] >> (8 * k)), fs) & 255u) << (8 * k);
                        w[q] = r;
                    }
                    out[e] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
        __syncthreads();
        if (moves) {
#pragma unroll
            for (int e = 0; e < ITEMS; e++) {
                const int it = e * 32 + lane;
                if (kv || (live >> (it / (hs / 2) * 8 + it % 8) & 1)) reinterpret_cast<uint4 *>(dst)[it] = out[e];
            }
            if (lane == 0) scales[to * page_scales + ((b + warp) * PG_BLOCK & (a.pool.P - 1)) / PG_BLOCK] = now;
        }
    }
}
