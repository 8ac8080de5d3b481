// ps_serve.h - internal interface between the context (ps_cuda.cu) and the serving operators (ps_serve.cu): attention of a step's tokens over
// several caches, eviction from caches, sampling.  The context owns the stream, the error text and the memory that the operators work in.
#pragma once
#include "../../include/ps_cuda.h"

#include <cuda_runtime.h>

struct PsServeCall {
    cudaStream_t stream;
    int n_sm;
    int *err_dev;    // [0] of the context's error flags: a pipeline that lost step
    int64_t launches; // kernels enqueued by the call
    char msg[256];
    // device memory of at least `bytes` that stays the context's (and keeps its contents while the call's kernels run); 0 or a ps_cuda_status
    int (*workspace)(void *user, size_t bytes, void **p);
    void *user;
};

int ps_serve_attn_tree(PsServeCall *c, float *out, const float *q, const ps_cuda_cache *caches, int n_seqs, int cache_type, int head_size, int n_heads, int n_kv_heads,
                       const uint8_t *tree_mask, float scale);
int ps_serve_kv_evict(PsServeCall *c, const ps_cuda_cache *caches, int n_sets, int cache_type, int head_size, int n_kv_heads, int n_sink, int n_recent);
// a flag's value beside those of the pipelines' waits: a table or a list that names what is not there
#define PS_ERR_PAGE 64

int ps_serve_paged_rows(PsServeCall *c, bool store, const ps_cuda_pages *pages, int layer, void *k, void *v, int io_type, const ps_cuda_paged_seq *seqs, int n_seqs);
int ps_serve_paged_attn(PsServeCall *c, const ps_cuda_pages *pages, int layer, void *out, const void *q, int io_type, const ps_cuda_paged_seq *seqs, int n_seqs, int n_heads, const uint8_t *tree_mask, float scale);
int ps_serve_paged_edit(PsServeCall *c, const ps_cuda_pages *pages, const ps_cuda_page_edit *edits, int n, int32_t *held);
int ps_serve_paged_compact(PsServeCall *c, const ps_cuda_pages *pages, const ps_cuda_page_move *moves, int n);
int ps_serve_verify(PsServeCall *c, int32_t *ids, int32_t *path, int32_t *n_path, const int32_t *n_nodes, int n_seqs, const int32_t *parents, const int32_t *tokens, const float *logits, int64_t row_stride, int64_t vocab,
                    const ps_cuda_sampler *samplers, const float *u, const float *draft_logits, const ps_cuda_sampler *draft_samplers);
int ps_serve_sample(PsServeCall *c, int32_t *ids, float *probs, const float *logits, int64_t row_stride, int64_t vocab, int64_t rows, const ps_cuda_sampler *samplers, const float *u);
