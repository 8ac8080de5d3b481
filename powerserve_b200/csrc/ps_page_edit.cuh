// ps_page_edit.cuh - pages taken, shared, given back and copied; slots that move together.
//
// A page is free where no table holds it (refs = 0), and growth takes the free pages of the lowest numbers: so what is handed out depends on the tables alone, not on the order in which threads come.
// Counts are changed by whole-number atomics, whose order does not matter, in three phases that the CTA passes together: shares, releases, growth.
// Latency bounds the edits (64 sequences: 6 us that grow, 3 that shrink), memory the copies (64 pages of 32 layers: 56 us, 7.4 TB/s with what L2 holds).
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
    int heads;              // K and V of all layers' heads
};
#define PG_MOVE_WARPS(wide) ((wide) ? 32 : 16) // of a CTA
#define PG_MOVE_FEW 4       // blocks

// A block of sixteen slots is a warp's: lane: a slot's source, then a channel (V) or a slot's sixteen channels (K).  WIDE: x a layer's head's K or V, the CTA's blocks are all read before one of them is written; else
// a warp a head, which reads a block and writes it before the next.  What a later block reads lies behind what is written, as the list rises: so slots may move in place.  ITEMS: head size / 32.
// Bound by latency: a chain of five loads (count, list, table, scale, codes) for a block, or a round of blocks; the next round's list, table and scales are asked for before this one is written
template <int ITEMS, bool WIDE>
__global__ void __launch_bounds__(32 * PG_MOVE_WARPS(WIDE)) pg_k_compact(const __grid_constant__ PgMoves a) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hs = 32 * ITEMS, B = a.pool.P / PG_BLOCK, step = WIDE ? PG_MOVE_WARPS(true) : 1;
    const PgMoveOp &op = a.op[blockIdx.y];
    const int head = WIDE ? blockIdx.x : blockIdx.x * PG_MOVE_WARPS(false) + warp, heads = 2 * a.pool.G, layer = head / heads, h = head % heads, kv = h & 1;
    if (!WIDE && head >= a.heads) return;
    int8_t *codes = a.pool.codes + (int64_t)layer * a.layer_codes + (int64_t)h * a.pool.page_codes();
    float *scales = a.pool.scales + (int64_t)layer * a.layer_scales + (int64_t)h * B;
    const int64_t page_codes = (int64_t)heads * a.pool.page_codes(), page_scales = (int64_t)heads * B;
    const int n_keep = op.n_dev ? min(*op.n_dev, op.n_keep) : op.n_keep;
    if (n_keep <= 0) return;
    const int b0 = op.first / PG_BLOCK, b1 = (op.first + n_keep - 1) / PG_BLOCK;
    struct Slot { int src, page, to; float was; bool bad; };
    auto look = [&](int b) { // where the slots of a block come from: before `first`, from themselves
        Slot o{-1, -1, -1, 0.f, false};
        const int j = b * PG_BLOCK + (lane & 15), i = j - op.first;
        if (b > b1 || lane >= 16 || i >= n_keep) return o;
        if (i < 0) o.src = j;
        else {
            const int k = op.keep[i], ahead = i ? op.keep[i - 1] : -1;
            if (k >= i && k > ahead && k < op.n_kv - op.first) o.src = op.first + k;
        }
        if (o.src >= 0) {
            o.page = op.table[o.src >> a.pool.shift];
            o.to = op.table[j >> a.pool.shift];
            if (!a.pool.has(o.page) || !a.pool.has(o.to)) o.src = -1;
        }
        if (o.src < 0) { o.bad = true; return o; }
        o.was = scales[o.page * page_scales + (o.src & (a.pool.P - 1)) / PG_BLOCK];
        return o;
    };
    Slot now_at = look(b0 + (WIDE ? warp : 0));
    for (int b = b0; b <= b1; b += step) {
        const int mine = b + (WIDE ? warp : 0);
        const Slot at = now_at;
        // (the list ends where it goes wrong: this block, or these 32, and all behind them stay as they are)
        if (WIDE ? __syncthreads_or(at.bad) : __any_sync(0xffffffffu, at.bad)) {
            if ((WIDE ? threadIdx.x : lane) == 0) *a.pool.err = PS_ERR_PAGE;
            break;
        }
        const int j = mine * PG_BLOCK + (lane & 15);
        const float now = pg_warp_max(at.was), f = pg_follow(at.was, now);
        const unsigned live = __ballot_sync(0xffffffffu, at.src >= 0), moves = __ballot_sync(0xffffffffu, at.src >= 0 && (at.src != j || at.was != now));
        const int to = __shfl_sync(0xffffffffu, at.to, 0); // (a block's slots are one page's; the first one is there if any is)
        uint4 out[ITEMS];
        const int off = at.src & (a.pool.P - 1); // slot of the page
        int8_t *dst = codes + to * page_codes + (int64_t)(mine * PG_BLOCK & (a.pool.P - 1)) * hs;
        if (moves) {
            if (kv) {       // a channel's sixteen slots, byte by byte
#pragma unroll
                for (int e = 0; e < ITEMS; e++) out[e] = reinterpret_cast<const uint4 *>(dst)[e * 32 + lane]; // (slots behind the last one stay)
                const int64_t base = at.page * page_codes + (int64_t)(off & ~15) * hs + (off & 15);
#pragma unroll
                for (int s = 0; s < 16; s++) {
                    if (!(live >> s & 1)) continue;
                    const uint8_t *from = reinterpret_cast<const uint8_t *>(codes) + __shfl_sync(0xffffffffu, base, s);
                    const float fs = __shfl_sync(0xffffffffu, f, s);
#pragma unroll
                    for (int e = 0; e < ITEMS; e++) {
                        uint32_t &w = s < 8 ? (s < 4 ? out[e].x : out[e].y) : (s < 12 ? out[e].z : out[e].w);
                        w = __byte_perm(w, pg_recode(from[(e * 32 + lane) * 16], 0, fs), (s & 3) == 0 ? 0x3214 : (s & 3) == 1 ? 0x3240 : (s & 3) == 2 ? 0x3410 : 0x4210);
                    }
                }
            } else {        // a slot's sixteen channels
                const int64_t base = at.page * page_codes + (int64_t)(off / 8) * 8 * hs + (off % 8) * 16;
#pragma unroll
                for (int e = 0; e < ITEMS; e++) {
                    const int it = e * 32 + lane, s = it / (hs / 2) * 8 + it % 8, c = it % (hs / 2) / 8;
                    const int64_t from = __shfl_sync(0xffffffffu, base, s);
                    const float fs = __shfl_sync(0xffffffffu, f, s);
                    if (!(live >> s & 1)) continue;
                    const uint4 v = *reinterpret_cast<const uint4 *>(codes + from + c * 128);
                    out[e] = make_uint4(pg_recode4(v.x, fs), pg_recode4(v.y, fs), pg_recode4(v.z, fs), pg_recode4(v.w, fs));
                }
            }
        }
        now_at = look(mine + step);
        if (WIDE) __syncthreads();
        else __syncwarp();
        if (moves) {
#pragma unroll
            for (int e = 0; e < ITEMS; e++) {
                const int it = e * 32 + lane;
                if (kv || (live >> (it / (hs / 2) * 8 + it % 8) & 1)) reinterpret_cast<uint4 *>(dst)[it] = out[e];
            }
            if (lane == 0) scales[to * page_scales + (mine * PG_BLOCK & (a.pool.P - 1)) / PG_BLOCK] = now;
        }
        if (!WIDE) __syncwarp();
    }
}
