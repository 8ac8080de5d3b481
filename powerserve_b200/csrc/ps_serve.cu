// ps_serve.cu - host side of the serving operators (ps_serve.h): what they accept, how they are cut into launches, and what they work in.
#include "ps_serve.h"

#include "ps_serve_attn.cuh"
#include "ps_serve_attn_tc.cuh"
#include "ps_serve_attn_few.cuh"
#include "ps_serve_evict.cuh"
#include "ps_serve_sample.cuh"
#include "ps_serve_verify.cuh"

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <type_traits>
#include <vector>

namespace {

int fail(PsServeCall *c, int code, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(c->msg, sizeof c->msg, fmt, ap);
    va_end(ap);
    return code;
}

#define SV_CK(call)                                                                                                    \
    do {                                                                                                               \
        const cudaError_t e_ = (call);                                                                                 \
        if (e_ != cudaSuccess) return fail(c, PS_CUDA_ERR_CUDA, "%s failed: %s", #call, cudaGetErrorString(e_));       \
    } while (0)
#define SV_LAUNCHED(what)                                                                                              \
    do {                                                                                                               \
        const cudaError_t e_ = cudaGetLastError();                                                                     \
        if (e_ != cudaSuccess) return fail(c, PS_CUDA_ERR_CUDA, what ": launch failed: %s", cudaGetErrorString(e_));   \
        c->launches++;                                                                                                 \
    } while (0)

bool aligned(const void *p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
size_t up(size_t v) { return (v + 255) & ~(size_t)255; }

int check_caches(PsServeCall *c, const char *what, const ps_cuda_cache *caches, int n, int cache_type, int head_size, int n_kv_heads) {
    if (n < 0 || (n > 0 && !caches)) return fail(c, PS_CUDA_ERR_INVALID, "%s: no caches", what);
    if (cache_type != PS_TYPE_F32 && cache_type != PS_TYPE_BF16) return fail(c, PS_CUDA_ERR_UNSUPPORTED, "%s: cache type %d (float32 and bfloat16 are there)", what, cache_type);
    if (head_size <= 0 || head_size % 32 || head_size > 256) return fail(c, PS_CUDA_ERR_UNSUPPORTED, "%s: head size %d (multiples of 32 up to 256)", what, head_size);
    if (n_kv_heads <= 0 || n_kv_heads > 1024) return fail(c, PS_CUDA_ERR_INVALID, "%s: %d kv heads", what, n_kv_heads);
    const size_t es = cache_type == PS_TYPE_F32 ? 4 : 2;
    for (int i = 0; i < n; i++) {
        const ps_cuda_cache &s = caches[i];
        if (s.n_ctx <= 0 || s.n_kv < 0 || s.n_kv > s.n_ctx) return fail(c, PS_CUDA_ERR_INVALID, "%s: cache %d holds %d of %d slots", what, i, s.n_kv, s.n_ctx);
        if (s.n_ctx > 1 << 30) return fail(c, PS_CUDA_ERR_UNSUPPORTED, "%s: cache %d has %d slots (at most 2^30)", what, i, s.n_ctx);
        if (s.n_kv && (!s.k || !s.v)) return fail(c, PS_CUDA_ERR_INVALID, "%s: cache %d has no rows", what, i);
        if (!aligned(s.k, es) || !aligned(s.v, es) || !aligned(s.weight, 4) || !aligned(s.weight_to, 4) || !aligned(s.pos, 4) || !aligned(s.pos_to, 4))
            return fail(c, PS_CUDA_ERR_INVALID, "%s: cache %d: an array that is not aligned to its elements", what, i);
    }
    return 0;
}

// Whether two of the arrays are the same
bool twice(std::vector<const void *> &p) {
    std::sort(p.begin(), p.end());
    return std::adjacent_find(p.begin(), p.end()) != p.end();
}

// Tiles of a split: the fewest with which the launch has no more CTAs than the GPU takes at once
int split_tiles(const ps_cuda_cache *caches, int n, int per_split, int target) {
    int64_t lo = 1, hi = 1;
    for (int i = 0; i < n; i++)
        if (caches[i].n_tok > 0) hi = std::max<int64_t>(hi, (caches[i].n_kv + SV_TILE - 1) / SV_TILE); // (a split a sequence)
    while (lo < hi) {
        const int64_t tps = (lo + hi) / 2;
        int64_t ctas = 0;
        for (int i = 0; i < n; i++)
            if (caches[i].n_tok > 0) ctas += ((caches[i].n_kv + SV_TILE - 1) / SV_TILE + tps - 1) / tps;
        if (ctas * per_split <= target) hi = tps;
        else lo = tps + 1;
    }
    return (int)lo;
}

// Tiles of a split for the kernel of few rows, of which `slots` CTAs run at once: the least of an estimate in tiles' time.  A CTA costs its tiles and one more to begin and end;
// CTAs that do not all run at once end half a CTA apart; joining splits costs one and a half.  64 sequences, 8 kv heads, head size 128, us with four / eight / sixteen
// CTAs an SM asked for: lengths 256 to 2 041 145 / 124 / 126, all 2 041 294 / 254 / 237; head size 64, all at once without splits, 104 / 117 / 122
int split_few(const ps_cuda_cache *caches, int n, int heads, int slots) {
    int most = 1, best = 1;
    for (int i = 0; i < n; i++)
        if (caches[i].n_tok > 0) most = std::max(most, (caches[i].n_kv + SV_TILE - 1) / SV_TILE);
    double least = 1e30;
    for (int tps = 2, last = 0; !last; tps = std::max(tps + 1, tps * 5 / 4)) {
        if (tps >= most) { tps = most; last = 1; }
        double ctas = 0, tiles = 0;
        for (int i = 0; i < n; i++)
            if (caches[i].n_tok > 0) {
                const int t = (caches[i].n_kv + SV_TILE - 1) / SV_TILE;
                ctas += (double)heads * ((t + tps - 1) / tps);
                tiles += (double)heads * t;
            }
        const double longest = std::min(tps, most) + 1.0;
        const double cost = (ctas <= slots ? longest : (tiles + ctas) / slots + 0.5 * longest) + (tps < most ? 1.5 : 0.0);
        if (cost < least) { least = cost; best = tps; }
    }
    return best;
}

} // namespace

int ps_serve_attn_tree(PsServeCall *c, float *out, const float *q, const ps_cuda_cache *caches, int n_seqs, int cache_type, int head_size, int n_heads, int n_kv_heads,
                       const uint8_t *tree_mask, float scale) {
    if (int rc = check_caches(c, "attn_tree", caches, n_seqs, cache_type, head_size, n_kv_heads)) return rc;
    if (n_heads <= 0 || n_heads % n_kv_heads || n_heads / n_kv_heads > 32) return fail(c, PS_CUDA_ERR_UNSUPPORTED, "attn_tree: %d heads over %d kv heads", n_heads, n_kv_heads);
    const int R = n_heads / n_kv_heads, hs = head_size;
    int64_t tokens = 0;
    std::vector<const void *> gather;
    for (int i = 0; i < n_seqs; i++) {
        const ps_cuda_cache &s = caches[i];
        if (s.n_tok < 0 || s.n_tok > s.n_kv) return fail(c, PS_CUDA_ERR_INVALID, "attn_tree: sequence %d brings %d tokens, its cache holds %d", i, s.n_tok, s.n_kv);
        if (s.weight && s.n_tok) gather.push_back(s.weight);
        if (s.n_tok > PS_CUDA_TREE_TOKENS) return fail(c, PS_CUDA_ERR_UNSUPPORTED, "attn_tree: sequence %d brings %d tokens (at most %d)", i, s.n_tok, PS_CUDA_TREE_TOKENS);
        tokens += s.n_tok;
    }
    if (tokens == 0) return 0;
    if (twice(gather)) return fail(c, PS_CUDA_ERR_INVALID, "attn_tree: two sequences gather their weights in the same array");
    if (tokens > INT32_MAX / 1024) return fail(c, PS_CUDA_ERR_UNSUPPORTED, "attn_tree: %lld tokens in one call", (long long)tokens);
    if (!out || !q) return fail(c, PS_CUDA_ERR_INVALID, "attn_tree: null argument");
    if (!aligned(out, 4) || !aligned(q, 4)) return fail(c, PS_CUDA_ERR_INVALID, "attn_tree: an array that is not aligned to its elements");

    int tok0 = 0;
    for (int first = 0; first < n_seqs;) {
        // sequences of a launch: as many as the table takes, and as their scores leave the workspace at a size
        int n = 0;
        size_t scores = 0;
        int most_tok = 0, most_kv = 0;
        bool weights = false;
        while (first + n < n_seqs && n < SV_SEQS) {
            const ps_cuda_cache &s = caches[first + n];
            const size_t more = s.weight && s.n_tok ? up(16 * (size_t)n_kv_heads * sv_quads(s.n_kv) * sv_rp(s.n_tok * R)) : 0;
            if (n && scores + more > ((size_t)1 << 30)) break;
            scores += more;
            weights |= more != 0;
            most_tok = std::max(most_tok, s.n_tok);
            most_kv = std::max(most_kv, s.n_kv);
            n++;
        }
        SvAttn a{};
        a.q = q; a.out = out; a.hs = hs; a.n_heads = n_heads; a.G = n_kv_heads; a.R = R; a.scale = scale * SV_LOG2E; a.err = c->err_dev; a.n_seqs = n;
        const bool own = hs == 64 || hs == 128, few = own && most_tok * R <= SV_FEW_ROWS, tc = own && !few;
        const int tile_rows = tc ? SV_TC_ROWS : 16, row_tiles = (most_tok * R + tile_rows - 1) / tile_rows;
        a.out_vec = aligned(out, 16);
        a.q_vec = aligned(q, 16);
        if (most_tok) {
            a.tps = few ? split_few(caches + first, n, n_kv_heads, c->n_sm * (hs == 128 && cache_type == PS_TYPE_F32 ? 3 : 4)) : split_tiles(caches + first, n, n_kv_heads * row_tiles, tc ? c->n_sm : c->n_sm * 4);
            // (one tile a split: more to join than it saves, but for the shortest; 12 tokens, 32 / 8 heads of 128 over 315 slots 18.5 us and 20.5 with two tiles, over 1 015 22.5 and
            // 20.5, heads of 64 18.5 and 14.9)
            if (tc && most_kv > 8 * SV_TILE) a.tps = std::max(a.tps, 2);
            if (tc) a.tps = std::min(a.tps, SV_TC_TILES);
            // Few rows, few splits, and no more CTAs than two an SM: a sequence's splits are a cluster, which joins them itself. 32 / 8 heads of 128 over 1 000 slots, one sequence
            // 18.5 us (20.5 with a launch to join), four 24.0 (26.6); eight, whose 512 CTAs are more than that, 42.8 (29.4)
            auto splits_at = [&](int tps, int &active) {
                int most = 1;
                active = 0;
                for (int i = 0; i < n; i++)
                    if (caches[first + i].n_tok) active++, most = std::max(most, ((caches[first + i].n_kv + SV_TILE - 1) / SV_TILE + tps - 1) / tps);
                return most;
            };
            int active, splits = splits_at(a.tps, active);
            if (few && splits > 8 && splits <= 16) { // (one sequence of 2 000 slots, two kv heads of 64: 14.4 us for eight splits in a cluster, 16.5 for sixteen to join)
                const int wider = ((most_kv + SV_TILE - 1) / SV_TILE + 7) / 8;
                if ((int64_t)active * 8 * n_kv_heads <= c->n_sm * 2) a.tps = wider, splits = splits_at(wider, active);
            }
            a.cluster = few && splits <= 8 && (int64_t)active * splits * n_kv_heads <= c->n_sm * 2 ? splits : 1;
            // (one split, or a cluster's: nothing is left for another kernel)
            auto parts = [&](const SvSeq &d) { return d.splits > 1 && a.cluster == 1 ? up(4 * (size_t)d.splits * n_kv_heads * d.n_tok * R * (hs + 2)) : 0; };
            size_t bytes = scores;
            int units = 0;
            bool joined = false;
            for (int i = 0; i < n; i++) {
                const ps_cuda_cache &s = caches[first + i];
                SvSeq &d = a.seq[i];
                d.k = s.k; d.v = s.v; d.weight = s.n_tok ? s.weight : nullptr; d.hidden = s.hidden; d.n_ctx = s.n_ctx; d.n_kv = s.n_kv; d.n_tok = s.n_tok; d.tok0 = tok0;
                d.mask = tree_mask;
                if (tree_mask) tree_mask += (size_t)s.n_tok * s.n_tok;
                tok0 += s.n_tok;
                const int tiles = s.n_tok ? (s.n_kv + SV_TILE - 1) / SV_TILE : 0;
                d.splits = a.cluster > 1 && s.n_tok ? a.cluster : (tiles + a.tps - 1) / a.tps;
                d.unit0 = units;
                const bool f32 = cache_type == PS_TYPE_F32;
                d.k_mode = aligned(s.k, 16);
                d.v_mode = aligned(s.v, 16) && s.n_ctx % (f32 ? 4 : 8) == 0;
                units += d.splits;
                joined |= d.splits > 1 && a.cluster == 1;
                if (d.weight) bytes += up(4 * (size_t)n_kv_heads * s.n_tok * R);
                bytes += parts(d);
            }
            void *mem = nullptr;
            if (int rc = c->workspace(c->user, bytes, &mem)) return rc;
            char *at = static_cast<char *>(mem);
            for (int i = 0; i < n; i++) {
                SvSeq &d = a.seq[i];
                if (d.weight) {
                    d.scores = reinterpret_cast<float *>(at);
                    at += up(16 * (size_t)n_kv_heads * sv_quads(d.n_kv) * sv_rp(d.n_tok * R));
                    d.lse = reinterpret_cast<float *>(at);
                    at += up(4 * (size_t)n_kv_heads * d.n_tok * R);
                }
                d.part = reinterpret_cast<float *>(at);
                at += parts(d);
            }
            const dim3 grid(units, n_kv_heads, row_tiles);
            if (few) {
                const bool f32 = cache_type == PS_TYPE_F32;
                auto pick = [&](auto cl) {
                    constexpr bool CL = decltype(cl)::value;
                    return hs == 64 ? (f32 ? sv_k_attn_few<float, 64, CL> : sv_k_attn_few<__nv_bfloat16, 64, CL>) : (f32 ? sv_k_attn_few<float, 128, CL> : sv_k_attn_few<__nv_bfloat16, 128, CL>);
                };
                auto kern = a.cluster > 1 ? pick(std::true_type{}) : pick(std::false_type{});
                cudaLaunchConfig_t cfg{};
                cudaLaunchAttribute attr[1];
                attr[0].id = cudaLaunchAttributeClusterDimension;
                attr[0].val.clusterDim.x = a.cluster; attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
                cfg.gridDim = grid; cfg.blockDim = dim3(128); cfg.stream = c->stream; cfg.attrs = attr; cfg.numAttrs = a.cluster > 1;
                SV_CK(cudaLaunchKernelEx(&cfg, kern, a));
            } else if (tc) {
                auto launch = [&](auto kern, int smem) -> int {
                    SV_CK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
                    kern<<<grid, SV_TC_THREADS, smem, c->stream>>>(a);
                    return 0;
                };
                auto pick = [&](auto w) -> int { // (with weights the soft-max needs more registers)
                    constexpr bool W = decltype(w)::value;
                    if (cache_type == PS_TYPE_F32) return hs == 64 ? launch(sv_k_attn_tc<float, 64, W>, SvTc<float, 64>::SMEM) : launch(sv_k_attn_tc<float, 128, W>, SvTc<float, 128>::SMEM);
                    return hs == 64 ? launch(sv_k_attn_tc<__nv_bfloat16, 64, W>, SvTc<__nv_bfloat16, 64>::SMEM) : launch(sv_k_attn_tc<__nv_bfloat16, 128, W>, SvTc<__nv_bfloat16, 128>::SMEM);
                };
                const int rc = weights ? pick(std::true_type{}) : pick(std::false_type{});
                if (rc) return rc;
            } else if (cache_type == PS_TYPE_F32) {
                const size_t smem = sv_attn_smem(hs);
                SV_CK(cudaFuncSetAttribute(sv_k_attn<float>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
                sv_k_attn<float><<<grid, 128, smem, c->stream>>>(a);
            } else {
                const size_t smem = sv_attn_smem(hs);
                SV_CK(cudaFuncSetAttribute(sv_k_attn<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
                sv_k_attn<__nv_bfloat16><<<grid, 128, smem, c->stream>>>(a);
            }
            SV_LAUNCHED("attn_tree");
            auto after = [&](auto kern, dim3 g, size_t smem) -> int { // (its start overlaps the end of the kernel before)
                cudaLaunchConfig_t cfg{};
                cudaLaunchAttribute attr[1];
                attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
                attr[0].val.programmaticStreamSerializationAllowed = 1;
                cfg.gridDim = g; cfg.blockDim = dim3(256); cfg.dynamicSmemBytes = smem; cfg.stream = c->stream; cfg.attrs = attr; cfg.numAttrs = 1;
                SV_CK(cudaLaunchKernelEx(&cfg, kern, a));
                SV_LAUNCHED("attn_tree");
                return 0;
            };
            if (joined)
                if (int rc = after(sv_k_join, dim3((most_tok * R + 7) / 8, n_kv_heads, n), 0)) return rc;
            if (weights)
                if (int rc = after(sv_k_weights, dim3((most_kv + SV_FIN_SLOTS - 1) / SV_FIN_SLOTS, n_kv_heads, n), 4 * (size_t)most_tok * R)) return rc;
        }
        first += n;
    }
    return 0;
}

int ps_serve_kv_evict(PsServeCall *c, const ps_cuda_cache *caches, int n_sets, int cache_type, int head_size, int n_kv_heads, int n_sink, int n_recent) {
    if (int rc = check_caches(c, "kv_evict", caches, n_sets, cache_type, head_size, n_kv_heads)) return rc;
    std::vector<const void *> written, read;
    if (n_sink < 0 || n_recent < 0) return fail(c, PS_CUDA_ERR_INVALID, "kv_evict: %d first and %d latest positions", n_sink, n_recent);
    for (int i = 0; i < n_sets; i++) {
        const ps_cuda_cache &s = caches[i];
        if (s.n_keep < 0 || s.n_keep > s.n_kv) return fail(c, PS_CUDA_ERR_INVALID, "kv_evict: cache %d keeps %d of %d slots", i, s.n_keep, s.n_kv);
        if (s.n_kv && (!s.weight || !s.weight_to)) return fail(c, PS_CUDA_ERR_INVALID, "kv_evict: cache %d has no gathered weights", i);
        if ((s.pos != nullptr) != (s.pos_to != nullptr)) return fail(c, PS_CUDA_ERR_INVALID, "kv_evict: cache %d: pos and pos_to go together", i);
        if (!s.pos && (n_sink || n_recent)) return fail(c, PS_CUDA_ERR_INVALID, "kv_evict: cache %d has no positions to keep the first or latest of", i);
        if (s.n_kv) { // (what a cache writes, no other one may touch)
            const void *own[4] = {s.k, s.v, s.weight_to, s.pos ? s.pos_to : s.k};
            for (int e = 0; e < 4; e++)
                if (std::find(own, own + e, own[e]) == own + e) written.push_back(own[e]);
            if (s.weight != s.weight_to) read.push_back(s.weight);
            if (s.pos && s.pos != s.pos_to) read.push_back(s.pos);
        }
        if (s.hidden) return fail(c, PS_CUDA_ERR_UNSUPPORTED, "kv_evict: cache %d has hidden slots (every kv head moves its own)", i);
    }
    if (twice(written)) return fail(c, PS_CUDA_ERR_INVALID, "kv_evict: two caches share an array that is written");
    for (const void *p : read) // (what is only read may be shared)
        if (std::binary_search(written.begin(), written.end(), p)) return fail(c, PS_CUDA_ERR_INVALID, "kv_evict: two caches share an array that is written");
    for (int first = 0; first < n_sets; first += SV_SETS) {
        const int n = std::min(n_sets - first, SV_SETS);
        SvEvict a{};
        a.G = n_kv_heads; a.hs = head_size; a.n_sink = n_sink; a.n_recent = n_recent;
        size_t bytes = 0;
        int most = 0, most_kv = 0, most_gone = 0;
        bool vec = true;
        const size_t es = cache_type == PS_TYPE_F32 ? 4 : 2;
        for (int i = 0; i < n; i++) {
            const ps_cuda_cache &s = caches[first + i];
            SvSet &d = a.set[i];
            d.k = s.k; d.v = s.v; d.weight = s.weight; d.weight_to = s.weight_to; d.pos = s.pos; d.pos_to = s.pos_to; d.n_ctx = s.n_ctx; d.n_kv = s.n_kv; d.n_keep = s.n_keep;
            d.moves = std::min(s.n_keep, s.n_kv - s.n_keep);
            most = std::max(most, d.moves);
            most_kv = std::max(most_kv, s.n_kv);
            most_gone = std::max(most_gone, s.n_kv - s.n_keep);
            vec &= aligned(s.k, 16);
            bytes += up(4 * (size_t)n_kv_heads * (1 + 2 * (size_t)d.moves));
        }
        const dim3 heads(n_kv_heads, n);
        // One by one costs a pass over the weights each. 256 heads of 1 025 slots, us one by one / by the select and its moves, arrays apart from the old ones: one 6.1 / 18.9, four 11.2 / 19.8, eight
        // 18.5 / 20.0; of 4 097 slots 11.5 / 25, 23.6 / 26.2, and eight 39 / 27: there four would be the border
        if (most_gone <= SV_FEW) {
            if (es == 4) sv_k_evict_few<uint32_t><<<heads, 256, 0, c->stream>>>(a);
            else sv_k_evict_few<uint16_t><<<heads, 256, 0, c->stream>>>(a);
            SV_LAUNCHED("kv_evict");
            continue;
        }
        void *mem = nullptr;
        if (int rc = c->workspace(c->user, bytes, &mem)) return rc;
        char *at = static_cast<char *>(mem);
        for (int i = 0; i < n; i++) {
            a.set[i].list = reinterpret_cast<int32_t *>(at);
            at += up(4 * (size_t)n_kv_heads * (1 + 2 * (size_t)a.set[i].moves));
        }
        // (with keys in shared memory / read again in every pass, us with the moves: 32 heads of 2 000 slots 16.8 / 17.8, 8 190 33 / 43, 20 000 80 / 103, 49 152 175 / 337; above there is no room: 131 072 842)
        const int keys = most_kv <= SV_KEYS ? most_kv : 0;
        SV_CK(cudaFuncSetAttribute(sv_k_select, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * sv_key_at(SV_KEYS)));
        sv_k_select<<<heads, SV_SEL_THREADS, 4 * (size_t)sv_key_at(keys), c->stream>>>(a, keys);
        SV_LAUNCHED("kv_evict");
        if (most) {
            cudaLaunchConfig_t cfg{};
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr[0].val.programmaticStreamSerializationAllowed = 1;
            cfg.gridDim = dim3((most + SV_MOVES - 1) / SV_MOVES * (1 + SV_V_PARTS), n_kv_heads, n); cfg.blockDim = dim3(256); cfg.stream = c->stream; cfg.attrs = attr; cfg.numAttrs = 1;
            // (rows of head sizes that are multiples of 32 begin at 16-byte boundaries where the cache does)
            SV_CK(es == 4 ? vec ? cudaLaunchKernelEx(&cfg, sv_k_move<uint32_t, 4>, a) : cudaLaunchKernelEx(&cfg, sv_k_move<uint32_t, 1>, a)
                          : vec ? cudaLaunchKernelEx(&cfg, sv_k_move<uint16_t, 8>, a) : cudaLaunchKernelEx(&cfg, sv_k_move<uint16_t, 1>, a));
            SV_LAUNCHED("kv_evict");
        }
    }
    return 0;
}

int ps_serve_sample(PsServeCall *c, int32_t *ids, float *probs, const float *logits, int64_t row_stride, int64_t vocab, int64_t rows, const ps_cuda_sampler *samplers, const float *u) {
    if (rows < 0 || vocab <= 0 || vocab > 1 << 18 || row_stride < vocab)
        return fail(c, PS_CUDA_ERR_INVALID, "sample: %lld rows of %lld tokens (1 to 262144), %lld apart", (long long)rows, (long long)vocab, (long long)row_stride);
    if (rows == 0) return 0;
    if (!ids || !logits || !samplers || !u) return fail(c, PS_CUDA_ERR_INVALID, "sample: null argument");
    if (!aligned(ids, 4) || !aligned(probs, 4) || !aligned(logits, 4) || !aligned(samplers, 4) || !aligned(u, 4)) return fail(c, PS_CUDA_ERR_INVALID, "sample: an array that is not aligned to its elements");
    SvSample a{};
    a.logits = logits; a.samplers = samplers; a.u = u; a.ids = ids; a.probs = probs; a.row_stride = row_stride; a.vocab = (int)vocab;
    // Few rows: as many CTAs a row as a cluster can have, so that the GPU is at work; many: eight.  Rows of 151 936, us for eight / sixteen CTAs: one, no filter 11.3 / 10.3, top-p 36 / 31, top-p with
    // min-p 11.1 / 9.8, top-k with top-p 15.8 / 16.3, largest logit 5.7 / 5.6; four 18.3 / 11.1, 69 / 35, 11.2 / 10.0, 16.0 / 16.5, 5.9 / 5.7; nine 17.7 / 15.0, 42 / 43, 11.2 / 13.7, 17.2 / 20.9, 6.0 / 7.0;
    // sixteen 20.4 / 18.4, 63 / 60, 18.2 / 19.4, 20.6 / 23.7, 7.6 / 10.8; 32: 24.4 / 30.3, 72 / 96, 16.1 / 29.7, 21.1 / 33.7, 7.8 / 16.9
    const int C = rows * 16 <= c->n_sm ? 16 : 8;
    a.chunk = (int)((vocab + C - 1) / C + 31) & ~31;
    a.vec = aligned(logits, 16) && row_stride % 4 == 0;
    const size_t smem = sizeof(SvSmpShared) + 4 * (size_t)a.chunk;
    for (int64_t r0 = 0; r0 < rows; r0 += 1 << 20) {
        const int n = (int)std::min<int64_t>(rows - r0, 1 << 20);
        cudaLaunchConfig_t cfg{};
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = C; at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.gridDim = dim3(n * C); cfg.blockDim = dim3(SV_SMP_THREADS); cfg.dynamicSmemBytes = smem; cfg.stream = c->stream; cfg.attrs = at; cfg.numAttrs = 1;
        SV_CK(cudaFuncSetAttribute(sv_k_sample, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        SV_CK(cudaFuncSetAttribute(sv_k_sample, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        SV_CK(cudaLaunchKernelEx(&cfg, sv_k_sample, a));
        SV_LAUNCHED("sample");
        a.logits += (int64_t)n * row_stride; a.samplers += n; a.u += n; a.ids += n;
        if (a.probs) a.probs += n;
    }
    return 0;
}

int ps_serve_verify(PsServeCall *c, int32_t *ids, int32_t *path, int32_t *n_path, const int32_t *n_nodes, int n_seqs, const int32_t *parents, const int32_t *tokens, const float *logits, int64_t row_stride, int64_t vocab,
                    const ps_cuda_sampler *samplers, const float *u, const float *draft_logits, const ps_cuda_sampler *draft_samplers) {
    if (n_seqs < 0 || (n_seqs > 0 && !n_nodes)) return fail(c, PS_CUDA_ERR_INVALID, "verify: no sequences");
    if (vocab <= 0 || vocab > 1 << 18 || row_stride < vocab) return fail(c, PS_CUDA_ERR_INVALID, "verify: rows of %lld tokens (1 to 262144), %lld apart", (long long)vocab, (long long)row_stride);
    int64_t rows = 0;
    for (int i = 0; i < n_seqs; i++) {
        if (n_nodes[i] < 1) return fail(c, PS_CUDA_ERR_INVALID, "verify: sequence %d has %d nodes", i, n_nodes[i]);
        if (n_nodes[i] > PS_CUDA_TREE_TOKENS) return fail(c, PS_CUDA_ERR_UNSUPPORTED, "verify: sequence %d has %d nodes (at most %d)", i, n_nodes[i], PS_CUDA_TREE_TOKENS);
        rows += n_nodes[i];
    }
    if (rows == 0) return 0;
    if (rows > 1 << 20) return fail(c, PS_CUDA_ERR_UNSUPPORTED, "verify: %lld nodes in one call", (long long)rows);
    if (!ids || !path || !n_path || !parents || !tokens || !logits || !samplers || !u) return fail(c, PS_CUDA_ERR_INVALID, "verify: null argument");
    if ((draft_logits != nullptr) != (draft_samplers != nullptr)) return fail(c, PS_CUDA_ERR_INVALID, "verify: the draft's rows and their settings go together");
    for (const void *p : {(const void *)ids, (const void *)path, (const void *)n_path, (const void *)parents, (const void *)tokens, (const void *)logits, (const void *)samplers, (const void *)u, (const void *)draft_logits, (const void *)draft_samplers})
        if (!aligned(p, 4)) return fail(c, PS_CUDA_ERR_INVALID, "verify: an array that is not aligned to its elements");
    for (int s0 = 0; s0 < n_seqs;) {
        SvVerify v{};
        int n = 0;
        v.first[0] = 0;
        for (; s0 + n < n_seqs && n < SV_VERIFY_SEQS; n++) v.first[n + 1] = v.first[n] + n_nodes[s0 + n];
        const int nodes = v.first[n];
        void *mem = nullptr;
        if (int rc = c->workspace(c->user, 2 * (sizeof(SvRowStats) + 1) * (size_t)nodes, &mem)) return rc;
        SvRowStats *stats[2] = {static_cast<SvRowStats *>(mem), static_cast<SvRowStats *>(mem) + nodes};
        v.target = stats[0]; v.draft = stats[1];
        v.ids = ids; v.path = path; v.n_path = n_path; v.parents = parents; v.tokens = tokens; v.logits = logits; v.draft_logits = draft_logits; v.samplers = samplers; v.draft_samplers = draft_samplers;
        v.u = u; v.row_stride = row_stride; v.vocab = (int)vocab;
        cudaLaunchConfig_t cfg{};
        cudaLaunchAttribute at[2];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.blockDim = dim3(SV_SMP_THREADS); cfg.stream = c->stream; cfg.attrs = at; cfg.numAttrs = 1;
        auto chunk_of = [&](int C) { return (int)((vocab + C - 1) / C + 31) & ~31; };
        const int all = nodes * (draft_logits ? 2 : 1);
        SvStats a{};
        a.logits[0] = logits; a.logits[1] = draft_logits; a.samplers[0] = samplers; a.samplers[1] = draft_samplers; a.stats[0] = stats[0]; a.stats[1] = stats[1]; a.parents = parents; a.row_stride = row_stride;
        a.vocab = (int)vocab; a.n_seqs = n;
        for (int d = 0; d < 2; d++) a.vec[d] = aligned(a.logits[d], 16) && row_stride % 4 == 0;
        std::copy(v.first, v.first + n + 1, a.first);
        if (all > 2 * c->n_sm / 8) { // (more rows than clusters run at once)
            a.todo = reinterpret_cast<uint8_t *>(stats[1] + nodes);
            sv_k_rows<<<all, SV_SMP_THREADS, 0, c->stream>>>(a);
            SV_LAUNCHED("verify");
        }
        {
            const int C = all * 16 <= c->n_sm ? 16 : 8; // (as in ps_serve_sample)
            a.chunk = chunk_of(C);
            const size_t smem = sizeof(SvSmpShared) + 4 * (size_t)a.chunk;
            at[0].val.clusterDim.x = C;
            at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            at[1].val.programmaticStreamSerializationAllowed = 1;
            cfg.numAttrs = a.todo ? 2 : 1;
            cfg.gridDim = dim3(all * C); cfg.dynamicSmemBytes = smem;
            SV_CK(cudaFuncSetAttribute(sv_k_stats, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
            SV_CK(cudaFuncSetAttribute(sv_k_stats, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
            SV_CK(cudaLaunchKernelEx(&cfg, sv_k_stats, a));
            SV_LAUNCHED("verify");
        }
        const int C = n * 16 <= c->n_sm * 2 ? 16 : 8;
        v.chunk = chunk_of(C);
        at[0].val.clusterDim.x = C;
        cfg.gridDim = dim3(n * C); cfg.dynamicSmemBytes = 0; cfg.numAttrs = 1;
        SV_CK(cudaFuncSetAttribute(sv_k_verify, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        SV_CK(cudaLaunchKernelEx(&cfg, sv_k_verify, v));
        SV_LAUNCHED("verify");
        ids += n; n_path += n; path += nodes; parents += nodes; tokens += nodes; u += nodes; samplers += nodes; logits += (int64_t)nodes * row_stride;
        if (draft_logits) { draft_logits += (int64_t)nodes * row_stride; draft_samplers += nodes; }
        s0 += n;
    }
    return 0;
}
