// ps_serve_evict.cuh - eviction from caches by the weight that their slots have gathered.
//
// Per cache and kv head: the slots in the order (safe, weight, lower slot), safe = a position below n_sink or among the n_recent latest; the first
// n_keep of them are kept.  Attention does not mind the order of slots, so no more moves than must: the i-th kept slot at n_keep or behind goes
// into the i-th freed slot before n_keep.  Sources and destinations are apart, so the moves need no order among themselves.
#pragma once
#include "ps_ptx.cuh"

#define SV_SETS 64
#define SV_SEL_THREADS 1024
#define SV_KEYS 49152       // slots whose keys fit shared memory
#define SV_FEW 8            // evictions of a head that sv_k_evict_few finds one by one

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

// Larger weight, larger number (both zeros are one); no number at all: 1, after all others; safe: above all
PS_D uint32_t sv_order(float w) {
    if (!(w == w)) return 1;
    const uint32_t b = __float_as_uint(w + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
#define SV_SAFE 0xffffffffu
// a head's arrays
struct SvHead {
    const float *w;
    const int32_t *pos;
    float *w_to;
    int32_t *pos_to;
    int n, keep;
    int64_t first, after;   // safe: positions below first, positions above after
    PS_D SvHead(const SvEvict &a, const SvSet &s, int g) : n(s.n_kv), keep(s.n_keep), first(a.n_sink), after(INT64_MAX) {
        const int64_t at = (int64_t)g * s.n_ctx;
        w = s.weight + at; w_to = s.weight_to + at;
        pos = s.pos ? s.pos + at : nullptr; pos_to = s.pos ? s.pos_to + at : nullptr;
    }
    PS_D bool safe(int j) const { return pos && (pos[j] < first || pos[j] > after); }
};

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

// the block's largest value
PS_D int sv_block_max(int v, int *ws) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockDim.x >> 5;
    v = __reduce_max_sync(0xffffffffu, v);
    __syncthreads();
    if (lane == 0) ws[warp] = v;
    __syncthreads();
    return __reduce_max_sync(0xffffffffu, lane < n ? ws[lane] : INT32_MIN);
}
// positions above this are among the latest
PS_D int64_t sv_after(const SvEvict &a, const SvHead &h, int *ws) {
    int newest = INT32_MIN;
    if (!h.pos) return INT64_MAX;
    for (int j = threadIdx.x; j < h.n; j += blockDim.x) newest = max(newest, h.pos[j]);
    return (int64_t)sv_block_max(newest, ws) - a.n_recent;
}

// Few evictions (one for every token that comes, once a cache is at its budget): the slots that go are found one by one, each the least of (key, higher slot
// first), and the same CTA moves what has to move.  One launch; a CTA a head, so 256 for every layer of a model of 32.  Bound by latency: one pass over the weights
// and positions, a reduction, a row to copy; 256 heads of 1 025 slots, one each: 6 us (in a captured graph; calls from the host come every 9 to 14).
template <typename T>
__global__ void __launch_bounds__(256) sv_k_evict_few(const __grid_constant__ SvEvict a) {
    __shared__ int ws[32];
    __shared__ unsigned long long gone_ws[8];
    const SvSet &s = a.set[blockIdx.y];
    const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, hs = a.hs;
    SvHead h(a, s, g);
    const int go = h.n - h.keep;        // at most SV_FEW
    h.after = sv_after(a, h, ws);
    int gone[SV_FEW];
#pragma unroll
    for (int e = 0; e < SV_FEW; e++) {
        gone[e] = -1;
        if (e >= go) continue;
        unsigned long long least = ~0ull;
        for (int j = tid; j < h.n; j += 256) {
            bool out = false;
#pragma unroll
            for (int o = 0; o < e; o++) out |= gone[o] == j;
            // (safe slots go last, among themselves in the same order)
            const unsigned long long k = (unsigned long long)h.safe(j) << 63 | (unsigned long long)sv_order(h.w[j]) << 31 | (uint32_t)(INT32_MAX - j);
            if (!out) least = min(least, k);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
        __syncthreads();
        if (lane == 0) gone_ws[warp] = least;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; w++) least = min(least, gone_ws[w]);
        gone[e] = INT32_MAX - (int)(least & 0x7fffffffu);
    }
    // the i-th slot at keep or behind that stays goes to the i-th lowest slot before it that goes
    int from[SV_FEW], to[SV_FEW], moves = 0;
#pragma unroll
    for (int e = 0; e < SV_FEW; e++) from[e] = to[e] = -1;
#pragma unroll
    for (int e = 0; e < SV_FEW; e++) { // (rank by counting)
        int below = 0;
#pragma unroll
        for (int o = 0; o < SV_FEW; o++) below += gone[o] >= 0 && gone[o] < gone[e];
        if (gone[e] >= 0 && gone[e] < h.keep) {
#pragma unroll
            for (int i = 0; i < SV_FEW; i++)
                if (i == below) to[i] = gone[e];
            moves++;
        }
    }
    int at = 0;
#pragma unroll
    for (int j = 0; j < SV_FEW; j++) {
        bool stays = j < go;
#pragma unroll
        for (int o = 0; o < SV_FEW; o++) stays &= gone[o] != h.keep + j;
        if (stays) {
#pragma unroll
            for (int i = 0; i < SV_FEW; i++)
                if (i == at) from[i] = h.keep + j;
            at++;
        }
    }
    if (h.w_to != h.w || (h.pos && h.pos_to != h.pos)) {
        for (int j = tid; j < h.keep; j += 256) {
            h.w_to[j] = h.w[j];
            if (h.pos) h.pos_to[j] = h.pos[j];
        }
        __syncthreads();
    }
    T *k = static_cast<T *>(s.k) + (int64_t)g * hs, *v = static_cast<T *>(s.v) + (int64_t)g * hs * s.n_ctx;
    const int64_t kvd = (int64_t)a.G * hs;
#pragma unroll
    for (int i = 0; i < SV_FEW; i++) {
        if (i >= moves) break;
        if (tid < hs) k[to[i] * kvd + tid] = k[from[i] * kvd + tid];
        if (tid < hs) v[(int64_t)tid * s.n_ctx + to[i]] = v[(int64_t)tid * s.n_ctx + from[i]];
        if (tid == 0) {
            h.w_to[to[i]] = h.w[from[i]];
            if (h.pos) h.pos_to[to[i]] = h.pos[from[i]];
        }
    }
}

// (a thread that walks a run of slots meets other banks than its neighbours)
PS_HD int sv_key_at(int j) { return j + (j >> 5); }

// Many evictions: a CTA a head finds the border's key by three passes of a radix select and lists the moves; sv_k_move makes them. Bound by latency: seven passes over a head's keys, most with a scan
// over the block; 32 heads of 8 190 slots 20 us alone (28 with three readings of weights and positions and
// runs of keys in one bank), 96 of 5 001 18.
__global__ void __launch_bounds__(SV_SEL_THREADS) sv_k_select(const __grid_constant__ SvEvict a, int keys) {
    extern __shared__ uint32_t sv_keys[];   // of `keys` slots: as many as the longest cache has, or none
    __shared__ uint32_t hist[2048], ws[32];
    __shared__ uint32_t s_bin, s_above;
    const SvSet &s = a.set[blockIdx.y];
    const int g = blockIdx.x, tid = threadIdx.x;
    SvHead h(a, s, g);
    const int n = h.n, keep = h.keep;
    int32_t *list = s.list + (int64_t)g * (1 + 2 * (int64_t)s.moves);
    int newest = INT32_MIN;
#pragma unroll 4
    for (int j = tid; j < n; j += SV_SEL_THREADS) {
        if (keys) sv_keys[sv_key_at(j)] = sv_order(h.w[j]);
        if (h.pos) newest = max(newest, h.pos[j]);
    }
    newest = sv_block_max(newest, reinterpret_cast<int *>(ws));
    if (h.pos) h.after = (int64_t)newest - a.n_recent;
    uint32_t n_safe, c = 0, safe_bits = 0; // (of the thread's first 32 slots)
    if (h.pos)
#pragma unroll 4
        for (int j = tid, i = 0; j < n; j += SV_SEL_THREADS, i++) {
            const bool safe = h.safe(j);
            c += safe;
            if (i < 32) safe_bits |= (uint32_t)safe << i;
        }
    sv_scan(c, ws, n_safe);
    // where the safe slots alone are more than are kept, the others are out (0) and the border lies among the safe; else the safe are above all
    const bool in_safe = n_safe >= (uint32_t)keep && keep > 0;
    auto make = [&](int j) {
        const bool safe = h.safe(j);
        return safe == in_safe ? sv_order(h.w[j]) : in_safe ? 0u : SV_SAFE;
    };
    if (keys && h.pos) {
        for (int j = tid, i = 0; j < n; j += SV_SEL_THREADS, i++)
            if ((i < 32 ? (safe_bits >> i & 1) != 0 : h.safe(j)) != in_safe) sv_keys[sv_key_at(j)] = in_safe ? 0u : SV_SAFE;
        __syncthreads();
    }
    auto key_of = [&](int j) { return keys ? sv_keys[sv_key_at(j)] : make(j); };
    uint32_t above = 0, key = 0, mask = 0;   // slots with a larger key; the border's key as far as it is known
    for (int pass = 0; pass < 3; pass++) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t bins = pass == 2 ? 1024 : 2048;
        for (int i = tid; i < 2048; i += SV_SEL_THREADS) hist[i] = 0;
        __syncthreads();
        for (int j = tid; j < n; j += SV_SEL_THREADS) {
            const uint32_t k = key_of(j);
            if ((k & mask) == key) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1u);
        }
        __syncthreads();
        const uint32_t h0 = hist[2047 - 2 * tid], h1 = hist[2046 - 2 * tid];    // from the largest bin down
        uint32_t all, before = sv_scan(h0 + h1, ws, all) + above;
        const uint32_t need = (uint32_t)keep;
        if (need > before && need <= before + h0) { s_bin = 2047 - 2 * tid; s_above = before; }
        if (need > before + h0 && need <= before + h0 + h1) { s_bin = 2046 - 2 * tid; s_above = before + h0; }
        __syncthreads();
        if (keep) {
            key |= s_bin << shift;
            mask |= (bins - 1) << shift;
            above = s_above;
        }
    }
    const uint32_t ties = keep - above;      // of the slots with the border's key: the lowest ones
    // a thread takes a run of slots, so that ranks are sums over the threads before it
    const int run = (n + SV_SEL_THREADS - 1) / SV_SEL_THREADS, j0 = min(tid * run, n), j1 = min(j0 + run, n);
    c = 0;
    for (int j = j0; j < j1; j++) c += key_of(j) == key;
    uint32_t all, tie = sv_scan(c, ws, all);
    const uint32_t tie0 = tie;
    auto kept = [&](int j) {
        const uint32_t k = key_of(j);
        return keep && k >= key && (k > key || tie++ < ties);
    };
    uint32_t holes = 0, movers = 0, n_movers, n_holes;
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
    ps_grid_dep_launch();
    // the new arrays: what stays, then what moved (with the same arrays in and out nothing that is still to be read is written)
    if (h.w_to != h.w)
        for (int j = tid; j < keep; j += SV_SEL_THREADS) h.w_to[j] = h.w[j];
    if (h.pos && h.pos_to != h.pos)
        for (int j = tid; j < keep; j += SV_SEL_THREADS) h.pos_to[j] = h.pos[j];
    __syncthreads();
    for (uint32_t i = tid; i < n_movers; i += SV_SEL_THREADS) {
        const int from = list[1 + 2 * i], to = list[2 + 2 * i];
        h.w_to[to] = h.w[from];
        if (h.pos) h.pos_to[to] = h.pos[from];
    }
}

// x: groups of 128 moves, of each a CTA for K (a warp a row, four rows under way) and SV_V_PARTS for V's channels (a thread a move and every other channel of the part,
// eight under way); y: kv head; z: set.  The lists are in order, so that a warp's 32 columns of a channel lie side by side as nearly as they can.  Bound by latency,
// then by the 32-byte pieces that V's columns are read and written in: the kept quarter of 8 190 slots reads four bytes of V for one that it moves:
// 32 heads 35 us, 179 MB = 5.1 TB/s.
#define SV_MOVES 128
#define SV_V_PARTS 4
template <typename T, int VEC>
__global__ void __launch_bounds__(256) sv_k_move(const __grid_constant__ SvEvict a) {
    const SvSet &s = a.set[blockIdx.z];
    const int g = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, hs = a.hs;
    const int part = blockIdx.x % (1 + SV_V_PARTS), i0 = blockIdx.x / (1 + SV_V_PARTS) * SV_MOVES;
    const int32_t *list = s.list + (int64_t)g * (1 + 2 * (int64_t)s.moves);
    ps_grid_dep_wait();
    if (i0 >= s.moves) return;
    const int n = list[0];
    if (i0 >= n) return;
    if (part == 0) {
        T *k = static_cast<T *>(s.k) + (int64_t)g * hs;
        const int64_t kvd = (int64_t)a.G * hs;
        struct alignas(sizeof(T) * VEC) Piece { T x[VEC]; };
        for (int i = i0 + 4 * warp; i < min(i0 + SV_MOVES, n); i += 32)
            for (int d = lane * VEC; d < hs; d += 32 * VEC) {
                Piece p[4];
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (i + e < n) p[e] = *reinterpret_cast<const Piece *>(k + list[1 + 2 * (i + e)] * kvd + d);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (i + e < n) *reinterpret_cast<Piece *>(k + list[2 + 2 * (i + e)] * kvd + d) = p[e];
            }
        return;
    }
    const int i = i0 + (tid & (SV_MOVES - 1)), d0 = (part - 1) * hs / SV_V_PARTS, d1 = part * hs / SV_V_PARTS; // (head sizes are multiples of 32: parts of 8 channels or more)
    if (i >= n) return;
    const int64_t from = list[1 + 2 * i], to = list[2 + 2 * i];
    T *v = static_cast<T *>(s.v) + (int64_t)g * hs * s.n_ctx;
    for (int d = d0 + tid / SV_MOVES; d < d1; d += 16) {
        T x[8];
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (d + 2 * e < d1) x[e] = v[(int64_t)(d + 2 * e) * s.n_ctx + from];
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (d + 2 * e < d1) v[(int64_t)(d + 2 * e) * s.n_ctx + to] = x[e];
    }
}
