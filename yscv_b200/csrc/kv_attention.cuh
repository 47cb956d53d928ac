// A call of attention over a paged 8-bit cache, as its kernels take it (kv_block_attention.cu: a few rows a sequence,
// kv_block_prompt.cu: prompts).
#pragma once

#include "kv_pool.cuh"

namespace yscv {

struct KvAttention {
    KvLayer l;
    const float *q;
    float *out;
    size_t q_stride, out_stride;
    const int32_t *offsets, *start;
    int n_q, group, causal, wide;             // wide: rows of queries and results begin at 16 bytes (2: results at 32)
    int window;                               // 0: none
    float scale;                              // times log2(e)
    long long *plan;                          // [0] steps, [1] steps of a warp, [2 ..] steps in front of a sequence
    float *records;
    int *status;
};

// kv_block_prompt.cu: heads of 64 or 128, at most 128 query heads per KV head. `takes` says whether it is the kernel for a call.
bool kv_prompt_takes(size_t d_head, size_t n_seq, size_t group, size_t most_rows);
size_t kv_prompt_bytes(const yscv_cuda_ctx *ctx, size_t d_head, size_t n_seq);
int kv_prompt(yscv_cuda_ctx *ctx, KvAttention a, void *workspace, size_t rows);

}  // namespace yscv
