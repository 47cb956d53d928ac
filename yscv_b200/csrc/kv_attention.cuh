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
    int rows, room;                           // rows of q and out; positions that a table has room for
    float scale;                              // times log2(e)
    void *plan;                               // what the first kernel of a call lays down for the second
    float *records;
    int *status;
};

// The rows of a sequence: none if it takes no part or its offsets lie outside the call's rows. `ok`: it can be served as it is.
struct KvSeqRows {
    int start, rows, row0;
    bool ok;
};
__device__ __forceinline__ KvSeqRows kv_rows(const KvAttention &a, int seq) {
    KvSeqRows r;
    const int end = a.offsets[seq + 1];
    r.row0 = a.offsets[seq];
    r.start = a.start[seq];
    const bool inside = r.row0 >= 0 && r.row0 <= end && end <= a.rows;
    r.rows = inside && r.start >= 0 ? end - r.row0 : 0;
    r.ok = inside && (r.rows == 0 || r.start <= a.room - r.rows);
    r.start = min(r.start, a.room);
    return r;
}
// (by one thread)
__device__ __forceinline__ void kv_rows_status(const KvAttention &a, const KvSeqRows &r) {
    if (!r.ok) atomicExch(a.status, r.rows > 0 ? YSCV_DEV_POS_OVERFLOW : YSCV_DEV_BAD_NUMBER);
}

// kv_block_prompt.cu: heads of 64 or 128, at most 128 query heads per KV head. `takes` says whether it is the kernel for a call.
bool kv_prompt_takes(const yscv_cuda_kv_pool *pool, size_t group, size_t rows, size_t most_rows);
size_t kv_prompt_bytes(const yscv_cuda_ctx *ctx, size_t d_head);
int kv_prompt(yscv_cuda_ctx *ctx, KvAttention a, void *workspace);

}  // namespace yscv
