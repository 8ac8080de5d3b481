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
int ps_serve_sample(PsServeCall *c, int32_t *ids, float *probs, const float *logits, int64_t row_stride, int64_t vocab, int64_t rows, const ps_cuda_sampler *samplers, const float *u);
