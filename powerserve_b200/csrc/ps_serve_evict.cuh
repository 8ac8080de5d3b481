// ps_serve_evict.cuh - eviction from caches by the weight that their slots have gathered.
//
// Per cache and kv head: the slots in the order (safe, weight, lower slot), safe = a position below n_sink or among the n_recent latest; the first
// n_keep of them are kept.  Attention does not mind the order of slots, so no more moves than must: the i-th kept slot at n_keep or behind goes
// into the i-th freed slot before n_keep.  Sources and destinations are apart, so the moves need no order among themselves.
#pragma once
#include "ps_ptx.cuh"

#define SV_SETS 64
#define SV_SEL_THREADS 1024

struct SvSet {
    void *k, *v;
    const float *weight;
    float *weight_to;
    const int32_t *pos;
    int32_t *pos_to;
    int32_t *list;      // [kv head][1 + 2 moves]: number of moves, then pairs (from, to)
    int n_ctx, n_kv, n_keep, moves; // moves: the most that there can be
};
struct SvEvict {
    SvSet set[SV_SETS];
    int G, hs, n_sink, n_recent;
};

// larger weight, larger number; no number at all comes last, both zeros are one
PS_D uint32_t sv_order(float w) {
    if (!(w == w)) return 0;
    const uint32_t b = __float_as_uint(w + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// sums of `v` over the block's threads before this one, and over all
PS_D uint32_t sv_scan(uint32_t v, uint32_t *ws, uint32_t &all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockDim.x >> 5;
    uint32_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
    }
    __syncthreads();
    if (lane == 31) ws[warp] = inc;
    __syncthreads();
    uint32_t w = lane < n ? ws[lane] : 0, winc = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, winc, o);
        if (lane >= o) winc += u;
    }
    all = __shfl_sync(0xffffffffu, winc, 31);
    return inc - v + __shfl_sync(0xffffffffu, winc - w, warp);
}

__global__ void __launch_bounds__(SV_SEL_THREADS) sv_k_select(const __grid_constant__ SvEvict a) {
    __shared__ uint32_t hist[2048], ws[32];
    __shared__ int s_new;
    __shared__ uint32_t s_bin, s_above;
    const SvSet &s = a.set[blockIdx.y];
    const int g = blockIdx.x, tid = threadIdx.x, n = s.n_kv, keep = s.n_keep;
    const float *w = s.weight + (int64_t)g * s.n_ctx;
    const int32_t *pos = s.pos ? s.pos + (int64_t)g * s.n_ctx : nullptr;
    float *w_to = s.weight_to + (int64_t)g * s.n_ctx;
    int32_t *pos_to = s.pos_to ? s.pos_to + (int64_t)g * s.n_ctx : nullptr;
    int32_t *list = s.list + (int64_t)g * (1 + 2 * (int64_t)s.moves);
    if (tid == 0) s_new = INT32_MIN;
    __syncthreads();
    int newest = INT32_MIN;
    if (pos)
        for (int j = tid; j < n; j += SV_SEL_THREADS) newest = max(newest, pos[j]);
    newest = __reduce_max_sync(0xffffffffu, newest);
    if ((tid & 31) == 0) atomicMax(&s_new, newest);
    __syncthreads();
    newest = s_new;
    auto safe = [&](int j) { return pos && (pos[j] < a.n_sink || (int64_t)pos[j] > (int64_t)newest - a.n_recent); };
    uint32_t n_safe, c = 0;
    for (int j = tid; j < n; j += SV_SEL_THREADS) c += safe(j);
    sv_scan(c, ws, n_safe);
    // the class that the border lies in, and how many of it are kept
    const bool in_safe = n_safe >= (uint32_t)keep;
    const uint32_t need = in_safe ? keep : keep - n_safe;
    uint32_t above = 0, key = 0, mask = 0;   // members with a larger key; the border's key as far as it is known
    for (int pass = 0; pass < 3; pass++) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t bins = pass == 2 ? 1024 : 2048;
        for (int i = tid; i < 2048; i += SV_SEL_THREADS) hist[i] = 0;
        __syncthreads();
        for (int j = tid; j < n; j += SV_SEL_THREADS) {
            const uint32_t k = sv_order(w[j]);
            if (safe(j) == in_safe && (k & mask) == key) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1u);
        }
        __syncthreads();
        const uint32_t h0 = hist[2047 - 2 * tid], h1 = hist[2046 - 2 * tid];    // from the largest bin down
        uint32_t all, before = sv_scan(h0 + h1, ws, all) + above;
        if (need > before && need <= before + h0) { s_bin = 2047 - 2 * tid; s_above = before; }
        if (need > before + h0 && need <= before + h0 + h1) { s_bin = 2046 - 2 * tid; s_above = before + h0; }
        __syncthreads();
        if (need) {
            key |= s_bin << shift;
            mask |= (bins - 1) << shift;
            above = s_above;
        }
    }
    const uint32_t ties = need - above;      // of the slots with the border's key: the lowest ones
    // a thread takes a run of slots, so that ranks are sums over the threads before it
    const int run = (n + SV_SEL_THREADS - 1) / SV_SEL_THREADS, j0 = min(tid * run, n), j1 = min(j0 + run, n);
    c = 0;
    for (int j = j0; j < j1; j++) c += need && safe(j) == in_safe && sv_order(w[j]) == key;
    uint32_t all, tie = sv_scan(c, ws, all);
    const uint32_t tie0 = tie;
    auto kept = [&](int j) {
        if (safe(j) != in_safe) return !in_safe;     // (a safe slot while the border lies among the others)
        const uint32_t k = sv_order(w[j]);
        if (!need || k < key) return false;
        return k > key || tie++ < ties;
    };
    uint32_t holes = 0, movers = 0, n_holes, n_movers;
    for (int j = j0; j < j1; j++) {
        const bool yes = kept(j);
        holes += !yes && j < keep;
        movers += yes && j >= keep;
    }
    holes = sv_scan(holes, ws, n_holes);
    movers = sv_scan(movers, ws, n_movers);
    tie = tie0;
    for (int j = j0; j < j1; j++) {
        const bool yes = kept(j);
        if (!yes && j < keep) list[2 + 2 * holes++] = j;
        if (yes && j >= keep) list[1 + 2 * movers++] = j;
    }
    if (tid == 0) list[0] = n_movers;
    __syncthreads();
    // the new arrays: what stays, then what moved (with the same arrays in and out nothing that is still to be read is written)
    if (w_to != w)
        for (int j = tid; j < keep; j += SV_SEL_THREADS) w_to[j] = w[j];
    if (pos && pos_to != pos)
        for (int j = tid; j < keep; j += SV_SEL_THREADS) pos_to[j] = pos[j];
    __syncthreads();
    for (uint32_t i = tid; i < n_movers; i += SV_SEL_THREADS) {
        const int from = list[1 + 2 * i], to = list[2 + 2 * i];
        w_to[to] = w[from];
        if (pos) pos_to[to] = pos[from];
    }
}

// x: groups of 32 moves of kv head y of set z: a warp copies K rows, then channels of V
template <typename T>
__global__ void __launch_bounds__(256) sv_k_move(const __grid_constant__ SvEvict a) {
    const SvSet &s = a.set[blockIdx.z];
    const int g = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hs = a.hs;
    const int32_t *list = s.list + (int64_t)g * (1 + 2 * (int64_t)s.moves);
    const int n = list[0], i0 = blockIdx.x * 32;
    if (i0 >= n) return;
    T *k = static_cast<T *>(s.k) + (int64_t)g * hs, *v = static_cast<T *>(s.v) + (int64_t)g * hs * s.n_ctx;
    const int64_t kvd = (int64_t)a.G * hs;
    for (int i = i0 + warp; i < min(i0 + 32, n); i += 8) {
        const int64_t from = list[1 + 2 * i], to = list[2 + 2 * i];
        for (int d = lane; d < hs; d += 32) k[to * kvd + d] = k[from * kvd + d];
    }
    const int i = i0 + lane;
    if (i >= n) return;
    const int from = list[1 + 2 * i], to = list[2 + 2 * i];
    for (int d = warp; d < hs; d += 8) v[(int64_t)d * s.n_ctx + to] = v[(int64_t)d * s.n_ctx + from];
}
