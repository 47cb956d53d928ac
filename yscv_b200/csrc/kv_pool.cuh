// What the kernels over a paged 8-bit cache know of a yscv_cuda_kv_pool (include/yscv_cuda.h): one layer of it, and the
// checks that every entry point makes.
//
// A page is a block of `page` consecutive tokens of one sequence. Tokens lie in groups of 16, 16 * d bytes a group, in the
// order the tensor cores take them: keys [d / 16][16 tokens][16 d], eight tokens' 16 bytes being one 128-byte operand block
// of scores = Q K^T, values [d][16 tokens], eight rows being one of out = P V. So a run of tokens goes from memory into an
// operand by one bulk copy, bytes as they are, without a swizzle, a transposition or a conversion.
#pragma once

#include <initializer_list>

#include "common.cuh"
#include "kernels.cuh"

namespace yscv {

constexpr int KV_GROUP = 16;          // tokens of a group
constexpr float KV_LEAST = 7.8886091e-31f;   // 2^-100, the smallest magnitude a block is scaled to

struct KvLayer {
    int8_t *k, *v;
    float *ks, *vs;
    const int32_t *table;             // [n_seq][max_pages]
    int n_pages, n_kv, d, page, page_shift, n_seq, max_pages;
};

// Whether f32 or i32 operands lie where they can be read
inline bool kv_aligned(std::initializer_list<const void *> operands) {
    for (const void *p : operands)
        if (reinterpret_cast<uintptr_t>(p) & 3) return false;
    return true;
}
// Everything about a pool that does not depend on the call: sizes, alignment, null pointers
int kv_check_pool(const yscv_cuda_kv_pool *p);
// One layer of a checked pool
int kv_layer_of(const yscv_cuda_kv_pool *p, size_t layer, KvLayer *out);

#ifdef __CUDACC__
// The first byte of a group of 16 tokens of a page and head
__device__ __forceinline__ size_t kv_group_at(const KvLayer &l, int page_id, int head, int group) {
    return (((size_t)page_id * l.n_kv + head) * (l.page / KV_GROUP) + group) * (size_t)(KV_GROUP * l.d);
}
#endif

}  // namespace yscv
