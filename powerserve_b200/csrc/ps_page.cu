// ps_page.cu - host side of the caches in 8 bits and in pages (ps_serve.h): what the calls accept, and their launches.
#include "ps_page_attn.cuh"
#include "ps_page_edit.cuh"
#include "ps_page_rows.cuh"

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <vector>

namespace {

int fail(PsServeCall *c, int code, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(c->msg, sizeof c->msg, fmt, ap);
    va_end(ap);
    return code;
}

#define PG_CK(call)                                                                                                    \
    do {                                                                                                               \
        const cudaError_t e_ = (call);                                                                                 \
        if (e_ != cudaSuccess) return fail(c, PS_CUDA_ERR_CUDA, "%s failed: %s", #call, cudaGetErrorString(e_));       \
    } while (0)
#define PG_LAUNCHED(what)                                                                                              \
    do {                                                                                                               \
        const cudaError_t e_ = cudaGetLastError();                                                                     \
        if (e_ != cudaSuccess) return fail(c, PS_CUDA_ERR_CUDA, "%s: launch failed: %s", what, cudaGetErrorString(e_)); \
        c->launches++;                                                                                                 \
    } while (0)

bool aligned(const void *p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
size_t up(size_t v) { return (v + 255) & ~(size_t)255; }

int check_pages(PsServeCall *c, const char *what, const ps_cuda_pages *p, bool data) {
    if (!p) return fail(c, PS_CUDA_ERR_INVALID, "%s: no cache", what);
    if (p->page_tokens != 16 && p->page_tokens != 32 && p->page_tokens != 64 && p->page_tokens != 128)
        return fail(c, PS_CUDA_ERR_UNSUPPORTED, "%s: pages of %d tokens (16, 32, 64 and 128 are there)", what, p->page_tokens);
    if (p->head_size <= 0 || p->head_size % 32 || p->head_size > 256) return fail(c, PS_CUDA_ERR_UNSUPPORTED, "%s: head size %d (multiples of 32 up to 256)", what, p->head_size);
    if (p->n_kv_heads <= 0 || p->n_kv_heads > 1024) return fail(c, PS_CUDA_ERR_INVALID, "%s: %d kv heads", what, p->n_kv_heads);
    if (p->n_layers <= 0 || p->n_layers > 4096 || p->n_pages <= 0 || p->n_pages > 1 << 26) return fail(c, PS_CUDA_ERR_INVALID, "%s: %d layers of %d pages", what, p->n_layers, p->n_pages);
    if (data) {
        if (!p->codes || !p->scales) return fail(c, PS_CUDA_ERR_INVALID, "%s: a cache without codes or scales", what);
        if (!aligned(p->codes, 16) || !aligned(p->scales, 4)) return fail(c, PS_CUDA_ERR_INVALID, "%s: codes that are not aligned to 16 bytes, or scales to 4", what);
    }
    return 0;
}
int64_t layer_codes(const ps_cuda_pages *p) { return (int64_t)p->n_pages * p->n_kv_heads * 2 * p->page_tokens * p->head_size; }
int64_t layer_scales(const ps_cuda_pages *p) { return (int64_t)p->n_pages * p->n_kv_heads * 2 * (p->page_tokens / PG_BLOCK); }
PgPool pool_of(PsServeCall *c, const ps_cuda_pages *p, int layer) {
    PgPool q{};
    q.codes = p->codes ? p->codes + layer * layer_codes(p) : nullptr;
    q.scales = p->scales ? p->scales + layer * layer_scales(p) : nullptr;
    q.n_pages = p->n_pages; q.P = p->page_tokens; q.G = p->n_kv_heads; q.hs = p->head_size; q.err = c->err_dev;
    for (q.shift = 0; 1 << q.shift < q.P;) q.shift++;
    return q;
}
int64_t pages_of(int64_t n, int P) { return (n + P - 1) / P; }

int check_seqs(PsServeCall *c, const char *what, const ps_cuda_pages *p, int layer, const ps_cuda_paged_seq *seqs, int n, int io_type, int64_t &tokens) {
    if (int rc = check_pages(c, what, p, true)) return rc;
    if (layer < 0 || layer >= p->n_layers) return fail(c, PS_CUDA_ERR_INVALID, "%s: layer %d of %d", what, layer, p->n_layers);
    if (io_type != PS_TYPE_F32 && io_type != PS_TYPE_BF16) return fail(c, PS_CUDA_ERR_UNSUPPORTED, "%s: type %d (float32 and bfloat16 are there)", what, io_type);
    if (n < 0 || (n > 0 && !seqs)) return fail(c, PS_CUDA_ERR_INVALID, "%s: no sequences", what);
    tokens = 0;
    for (int i = 0; i < n; i++) {
        const ps_cuda_paged_seq &s = seqs[i];
        if (s.n_kv < 0 || s.n_kv > 1 << 30) return fail(c, PS_CUDA_ERR_INVALID, "%s: sequence %d holds %d slots (at most 2^30)", what, i, s.n_kv);
        if (s.n_tok < 0 || s.n_tok > s.n_kv) return fail(c, PS_CUDA_ERR_INVALID, "%s: sequence %d has %d tokens of its %d slots", what, i, s.n_tok, s.n_kv);
        if (!s.n_tok) continue;
        if (!s.table || !aligned(s.table, 4)) return fail(c, PS_CUDA_ERR_INVALID, "%s: sequence %d has no table, or one that is not aligned to its elements", what, i);
        if (s.n_table < pages_of(s.n_kv, p->page_tokens)) return fail(c, PS_CUDA_ERR_INVALID, "%s: sequence %d holds %d slots, its table has %d pages", what, i, s.n_kv, s.n_table);
        tokens += s.n_tok;
    }
    if (tokens > INT32_MAX / 2048) return fail(c, PS_CUDA_ERR_UNSUPPORTED, "%s: %lld tokens in one call", what, (long long)tokens);
    return 0;
}

// f(a std::integral_constant of head size / 32)
template <typename F> auto by_items(int hs, F f) {
    switch (hs / 32) {
    case 1: return f(std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 2>{});
    case 3: return f(std::integral_constant<int, 3>{});
    case 4: return f(std::integral_constant<int, 4>{});
    case 5: return f(std::integral_constant<int, 5>{});
    case 6: return f(std::integral_constant<int, 6>{});
    case 7: return f(std::integral_constant<int, 7>{});
    default: return f(std::integral_constant<int, 8>{});
    }
}

} // namespace

int ps_serve_paged_rows(PsServeCall *c, bool store, const ps_cuda_pages *pages, int layer, void *k, void *v, int io_type, const ps_cuda_paged_seq *seqs, int n_seqs) {
    const char *what = store ? "paged_store" : "paged_load";
    int64_t tokens;
    if (int rc = check_seqs(c, what, pages, layer, seqs, n_seqs, io_type, tokens)) return rc;
    if (!tokens) return 0;
    const int es = io_type == PS_TYPE_F32 ? 4 : 2;
    if (store ? !k || !v : !k && !v) return fail(c, PS_CUDA_ERR_INVALID, "%s: null argument", what);
    if (!aligned(k, es) || !aligned(v, es)) return fail(c, PS_CUDA_ERR_INVALID, "%s: an array that is not aligned to its elements", what);
    PgRows a{};
    a.pool = pool_of(c, pages, layer);
    a.k = k; a.v = v; a.k_vec = aligned(k, 16); a.v_vec = aligned(v, 16);
    for (int i = 0, tok0 = 0; i < n_seqs;) {
        int64_t blocks = 0;
        a.n_seqs = 0;
        for (; i < n_seqs && a.n_seqs < PG_SEQS; i++) {
            const ps_cuda_paged_seq &s = seqs[i];
            if (!s.n_tok) continue;
            a.seq[a.n_seqs++] = PgRowSeq{s.table, s.n_kv, s.n_tok, tok0, (int)blocks};
            blocks += (s.n_kv - 1) / PG_BLOCK - (s.n_kv - s.n_tok) / PG_BLOCK + 1;
            tok0 += s.n_tok;
        }
        if (!a.n_seqs) break;
        a.blocks = (int)blocks; // (tokens fit an int's 2 048th part, so all that follows fits 32 bits)
        const int64_t tasks = blocks * 2 * pages->n_kv_heads;
        const unsigned grid = (unsigned)((tasks + PG_ROW_WARPS - 1) / PG_ROW_WARPS);
        if (store) {
            if (es == 4) pg_k_store<float><<<(unsigned)tasks, pages->head_size, 0, c->stream>>>(a);
            else pg_k_store<__nv_bfloat16><<<(unsigned)tasks, pages->head_size, 0, c->stream>>>(a);
        }
        else if (es == 4) pg_k_load<float><<<grid, 32 * PG_ROW_WARPS, 0, c->stream>>>(a);
        else pg_k_load<__nv_bfloat16><<<grid, 32 * PG_ROW_WARPS, 0, c->stream>>>(a);
        PG_LAUNCHED(what);
    }
    return 0;
}

int ps_serve_paged_attn(PsServeCall *c, const ps_cuda_pages *pages, int layer, void *out, const void *q, int io_type, const ps_cuda_paged_seq *seqs, int n_seqs, int n_heads, const uint8_t *tree_mask,
                        float scale) {
    int64_t tokens;
    if (int rc = check_seqs(c, "paged_attn", pages, layer, seqs, n_seqs, io_type, tokens)) return rc;
    const int G = pages->n_kv_heads;
    if (n_heads <= 0 || n_heads % G || n_heads / G > 32) return fail(c, PS_CUDA_ERR_UNSUPPORTED, "paged_attn: %d heads over %d kv heads", n_heads, G);
    for (int i = 0; i < n_seqs; i++)
        if (seqs[i].n_tok > PS_CUDA_TREE_TOKENS) return fail(c, PS_CUDA_ERR_UNSUPPORTED, "paged_attn: sequence %d brings %d tokens (at most %d)", i, seqs[i].n_tok, PS_CUDA_TREE_TOKENS);
    if (!tokens) return 0;
    const int es = io_type == PS_TYPE_F32 ? 4 : 2;
    if (!out || !q) return fail(c, PS_CUDA_ERR_INVALID, "paged_attn: null argument");
    if (!aligned(out, es) || !aligned(q, es)) return fail(c, PS_CUDA_ERR_INVALID, "paged_attn: an array that is not aligned to its elements");
    const int hs = pages->head_size, R = n_heads / G;
    PgAttn a{};
    a.pool = pool_of(c, pages, layer);
    a.q = q; a.out = out; a.n_heads = n_heads; a.R = R; a.scale = scale * 1.4426950408889634f; a.bf16 = es == 2; a.q_vec = aligned(q, 4 * es);
    for (int i = 0, tok0 = 0; i < n_seqs;) {
        PgAttnSeq all[PG_SEQS];
        int most = 0, n = 0; // most: query rows of a kv head
        int64_t tiles = 0;
        for (; i < n_seqs && n < PG_SEQS; i++) {
            const ps_cuda_paged_seq &s = seqs[i];
            if (!s.n_tok) continue;
            const int t = (s.n_kv + PG_TILE - 1) / PG_TILE;
            if (n && tiles + (int64_t)t * G > INT32_MAX / 2) break;
            tiles += (int64_t)t * G;
            all[n++] = PgAttnSeq{s.table, s.hidden, tree_mask, s.n_kv, s.n_tok, tok0, t};
            tok0 += s.n_tok;
            if (tree_mask) tree_mask += (size_t)s.n_tok * s.n_tok;
            most = std::max(most, s.n_tok * R);
        }
        if (!n) break;
        if (tiles > INT32_MAX / 2) return fail(c, PS_CUDA_ERR_UNSUPPORTED, "paged_attn: %lld tiles of one sequence", (long long)tiles);
        auto launch = [&](auto cfg) -> int {
            using C = decltype(cfg);
            constexpr int RT = C::RT;
            auto kern = pg_k_attn<C::RT, C::MT, C::SG, C::OG>;
            // those with more row tiles first: a run of row tiles is that of the first so many
            auto row_tiles = [&](const PgAttnSeq &s) { return (s.n_tok * R + RT - 1) / RT; };
            std::stable_sort(all, all + n, [&](const PgAttnSeq &x, const PgAttnSeq &y) { return row_tiles(x) > row_tiles(y); });
            a.n_seqs = n;
            a.tile0[0] = 0;
            for (int k = 0; k < n; k++) { a.seq[k] = all[k]; a.tile0[k + 1] = a.tile0[k] + all[k].tiles * G; }
            a.n_lanes = row_tiles(all[0]);
            int64_t total = 0;
            for (int z = 0, k = n; z < a.n_lanes; z++) {
                while (row_tiles(all[k - 1]) <= z) k--;
                a.lane_tiles[z] = a.tile0[k];
                total += a.lane_tiles[z];
            }
            // CTAs of an SM, and the stages that their shares of its shared memory hold: two at least
            static const int fixed = [&] { cudaFuncAttributes f{}; return cudaFuncGetAttributes(&f, kern) == cudaSuccess ? (int)f.sharedSizeBytes : 1 << 20; }();
            const int stage = PG_TILE * hs;
            int per_sm = C::CTAS, room;
            while ((room = 233472 / per_sm - 1024 - fixed - 128 - C::tail(hs)) < 4 * stage && per_sm > 1) per_sm--;
            room = std::min(room, 232448 - fixed - 128 - C::tail(hs)); // (what one CTA can have)
            a.stages = std::min(PG_STAGES, room / (2 * stage));
            if (a.stages < 2) return fail(c, PS_CUDA_ERR_CUDA, "paged_attn: no room for two stages in %d bytes of shared memory", room);
            const int slots = c->n_sm * per_sm;
            // Nothing to join where no sequence has many more tiles than a fair share: the kernel that joins takes as long as four tiles
            int64_t units = 0;
            int longest = 0;
            for (int k = 0; k < n; k++) { units += (int64_t)G * row_tiles(all[k]); longest = std::max(longest, all[k].tiles); }
            a.whole = units <= slots && longest <= total / slots + 4;
            a.n_ctas = 0;
            for (int z = 0, k = n; z < a.n_lanes; z++) {
                a.lane_cta0[z] = a.n_ctas;
                while (row_tiles(all[k - 1]) <= z) k--;
                a.n_ctas += a.whole ? k * G : (int)std::max<int64_t>(1, std::min<int64_t>(a.lane_tiles[z], (int64_t)slots * a.lane_tiles[z] / total));
            }
            a.lane_cta0[a.n_lanes] = a.n_ctas;
            const size_t smem = 128 + (size_t)a.stages * 2 * stage + C::tail(hs);
            // whether runs begin where rows' tiles do: nothing is left to join, and no memory asked for
            bool split = false;
            for (int z = 0; z < a.n_lanes && !split && !a.whole; z++) {
                const int m = a.lane_cta0[z + 1] - a.lane_cta0[z];
                for (int k = 1, s = 0; k < m && !split; k++) {
                    const int x = pg_run(a.lane_tiles[z], m, k);
                    while (a.tile0[s + 1] <= x) s++;
                    split = (x - a.tile0[s]) % all[s].tiles != 0;
                }
            }
            if (split) {
                void *mem = nullptr;
                if (int rc = c->workspace(c->user, up(4 * (size_t)a.n_ctas * 2 * RT * (hs + 2)), &mem)) return rc;
                a.part = static_cast<float *>(mem);
            }
            PG_CK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
            kern<<<a.n_ctas, C::THREADS, smem, c->stream>>>(a);
            PG_LAUNCHED("paged_attn");
            if (split) {
                cudaLaunchConfig_t cfg2{};
                cudaLaunchAttribute attr[1];
                attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
                attr[0].val.programmaticStreamSerializationAllowed = 1;
                cfg2.gridDim = dim3(a.n_ctas, (RT + 7) / 8); cfg2.blockDim = dim3(256); cfg2.stream = c->stream; cfg2.attrs = attr; cfg2.numAttrs = 1;
                PG_CK(cudaLaunchKernelEx(&cfg2, pg_k_join<RT>, a));
                PG_LAUNCHED("paged_attn");
            }
            return 0;
        };
        int rc;
        if (hs <= 128) rc = most <= 5 ? launch(PgCfg<5, 1, 1, 1>{}) : most <= 8 ? launch(PgCfg<8, 1, 1, 1>{}) : most <= 16 ? launch(PgCfg<16, 1, 1, 1>{}) : launch(PgCfg<32, 1, 3, 2>{});
        else rc = most <= 5 ? launch(PgCfg<5, 2, 1, 1>{}) : launch(PgCfg<16, 2, 1, 1>{});
        if (rc) return rc;
    }
    return 0;
}

int ps_serve_paged_edit(PsServeCall *c, const ps_cuda_pages *pages, const ps_cuda_page_edit *edits, int n, int32_t *held) {
    if (int rc = check_pages(c, "paged_edit", pages, true)) return rc;
    if (!pages->refs || !aligned(pages->refs, 4)) return fail(c, PS_CUDA_ERR_INVALID, "paged_edit: a cache without refs, or with ones that are not aligned to their elements");
    if (n < 0 || (n > 0 && !edits)) return fail(c, PS_CUDA_ERR_INVALID, "paged_edit: no edits");
    if (n > PS_CUDA_EDITS) return fail(c, PS_CUDA_ERR_UNSUPPORTED, "paged_edit: %d edits (at most %d)", n, PS_CUDA_EDITS);
    if (!aligned(held, 4)) return fail(c, PS_CUDA_ERR_INVALID, "paged_edit: an array that is not aligned to its elements");
    if (n == 0) return 0;
    PgEdits a{};
    const int P = pages->page_tokens;
    int64_t most = 0;
    int copies = 0;
    std::vector<const void *> tables, begun; // begun: those that share from now on
    for (int i = 0; i < n; i++) {
        const ps_cuda_page_edit &e = edits[i];
        if (e.n_old < 0 || e.n_new < 0 || e.n_old > 1 << 30 || e.n_new > 1 << 30) return fail(c, PS_CUDA_ERR_INVALID, "paged_edit: edit %d: from %d to %d tokens", i, e.n_old, e.n_new);
        if (e.from && e.n_new < e.n_old) return fail(c, PS_CUDA_ERR_INVALID, "paged_edit: edit %d shares %d tokens and shall hold %d", i, e.n_old, e.n_new);
        const int64_t need = pages_of(std::max(e.n_old, e.n_new), P);
        if (need > e.n_table) return fail(c, PS_CUDA_ERR_INVALID, "paged_edit: edit %d: %d tokens, its table has %d pages", i, std::max(e.n_old, e.n_new), e.n_table);
        if (e.from && e.from == e.table) return fail(c, PS_CUDA_ERR_INVALID, "paged_edit: edit %d: a table that begins as itself", i);
        if ((need && !e.table) || !aligned(e.table, 4) || !aligned(e.from, 4)) return fail(c, PS_CUDA_ERR_INVALID, "paged_edit: edit %d has no table, or one that is not aligned to its elements", i);
        if (e.table) tables.push_back(e.table);
        if (e.from && e.table) begun.push_back(e.table);
        a.op[i] = PgEditOp{e.table, e.from, e.n_old, e.n_new};
        if (e.n_new > e.n_old) {
            const bool part = e.n_old % P != 0;
            most += pages_of(e.n_new, P) - pages_of(e.n_old, P) + part;
            copies = part ? i + 1 : copies;
        }
    }
    std::sort(tables.begin(), tables.end());
    if (std::adjacent_find(tables.begin(), tables.end()) != tables.end()) return fail(c, PS_CUDA_ERR_INVALID, "paged_edit: two edits of one table");
    std::sort(begun.begin(), begun.end());
    for (int i = 0; i < n && !begun.empty(); i++) // (all `from` are read while those tables are written)
        if (edits[i].from && std::binary_search(begun.begin(), begun.end(), static_cast<const void *>(edits[i].from)))
            return fail(c, PS_CUDA_ERR_INVALID, "paged_edit: edit %d begins as a table that begins anew in the same call", i);
    if (most > INT32_MAX / 8) return fail(c, PS_CUDA_ERR_UNSUPPORTED, "paged_edit: %lld pages in one call", (long long)most);
    void *mem = nullptr;
    const size_t list = up(sizeof(int4) * (size_t)n);
    if (most)
        if (int rc = c->workspace(c->user, list + up(4 * (size_t)most), &mem)) return rc;
    a.copies = copies ? static_cast<int4 *>(mem) : nullptr;
    a.free = reinterpret_cast<int32_t *>(static_cast<char *>(mem) + list);
    a.refs = pages->refs; a.held = held; a.n = n; a.n_pages = pages->n_pages; a.err = c->err_dev;
    const PgPool pool = pool_of(c, pages, 0);
    a.shift = pool.shift;
    pg_k_edit<<<1, PG_EDIT_THREADS, 0, c->stream>>>(a);
    PG_LAUNCHED("paged_edit");
    if (copies) {
        PgCopies b{pool, a.copies, layer_codes(pages), layer_scales(pages)};
        cudaLaunchConfig_t cfg{};
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.gridDim = dim3(copies, pages->n_layers, 1); cfg.blockDim = dim3(256); cfg.stream = c->stream; cfg.attrs = attr; cfg.numAttrs = 1;
        PG_CK(cudaLaunchKernelEx(&cfg, pg_k_copy, b));
        PG_LAUNCHED("paged_edit");
    }
    return 0;
}

int ps_serve_paged_compact(PsServeCall *c, const ps_cuda_pages *pages, const ps_cuda_page_move *moves, int n) {
    if (int rc = check_pages(c, "paged_compact", pages, true)) return rc;
    if (n < 0 || (n > 0 && !moves)) return fail(c, PS_CUDA_ERR_INVALID, "paged_compact: no moves");
    PgMoves a{};
    a.pool = pool_of(c, pages, 0);
    a.layer_codes = layer_codes(pages); a.layer_scales = layer_scales(pages);
    for (int i = 0; i < n; i++) {
        const ps_cuda_page_move &m = moves[i];
        if (m.first < 0 || m.n_kv < m.first || m.n_kv > 1 << 30) return fail(c, PS_CUDA_ERR_INVALID, "paged_compact: move %d: from slot %d of %d", i, m.first, m.n_kv);
        if (m.n_keep < 0 || m.n_keep > m.n_kv - m.first) return fail(c, PS_CUDA_ERR_INVALID, "paged_compact: move %d keeps %d of %d slots", i, m.n_keep, m.n_kv - m.first);
        if (!m.n_keep) continue;
        if (!m.table || !m.keep || !aligned(m.table, 4) || !aligned(m.keep, 4) || !aligned(m.n_keep_dev, 4))
            return fail(c, PS_CUDA_ERR_INVALID, "paged_compact: move %d has no table or list, or one that is not aligned to its elements", i);
        if (m.n_table < pages_of(m.n_kv, pages->page_tokens)) return fail(c, PS_CUDA_ERR_INVALID, "paged_compact: move %d: %d slots, its table has %d pages", i, m.n_kv, m.n_table);
    }
    const int heads = 2 * pages->n_kv_heads * pages->n_layers;
    for (int i = 0; i < n;) {
        int k = 0, most = 0;
        for (; i < n && k < PG_SEQS; i++) {
            const ps_cuda_page_move &m = moves[i];
            if (!m.n_keep) continue;
            a.op[k++] = PgMoveOp{m.table, m.keep, m.n_keep_dev, m.first, m.n_kv, m.n_keep};
            most = std::max(most, (m.first + m.n_keep - 1) / PG_BLOCK - m.first / PG_BLOCK + 1);
        }
        if (!k) break;
        // few blocks: a warp a head, one block after the other; many: a CTA a head, a block a warp
        const bool few = most <= PG_MOVE_FEW;
        a.heads = heads;
        by_items(pages->head_size, [&](auto items) {
            constexpr int I = decltype(items)::value;
            if (few) pg_k_compact<I, false><<<dim3((heads + PG_MOVE_WARPS(false) - 1) / PG_MOVE_WARPS(false), k), 32 * PG_MOVE_WARPS(false), 0, c->stream>>>(a);
            else pg_k_compact<I, true><<<dim3(heads, k), 32 * PG_MOVE_WARPS(true), 0, c->stream>>>(a);
        });
        PG_LAUNCHED("paged_compact");
    }
    return 0;
}
