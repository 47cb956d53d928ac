// Keys and values of ragged rows into the pages of a paged 8-bit cache, and back.
//
// A block of the cache is a page's tokens of one KV head, keys or values; its scale s = fp32(m / 127), m its largest magnitude,
// its values rne(x / s) of the real quotient. The quotient is taken as x * (1 / s) in fp32, which is within 2^-15 of it (three
// roundings of 2^-24 on at most 127.5); where that lies within 2^-13 of a border between two whole numbers the fp64
// quotient decides. That one is exact enough: x and s have 24 bits, so x / s is a border or 2^-26 of its size away from it.
//
// Append: one CTA per (page that a sequence's rows touch, head, keys or values), so nobody else writes the block or its scale.
// Bound: bytes (4 in, 1 out per value), a decode step: latency, three dependent loads deep. Values leave as whole 16-byte
// rows of 16 tokens, turned in shared memory; the first and last group, which may hold other tokens, byte by byte.
#include <cfloat>

#include "kv_pool.cuh"

namespace yscv {

struct KvRows {
    const int32_t *offsets, *start;
    size_t stride;                 // floats between rows
};

// Whole number nearest to x / s. NaN: 0, infinities: +-127.
__device__ __forceinline__ int kv_quantise(float x, float s, float inv) {
    const float v = x * inv;
    float r = rintf(v);
    if (fabsf(fabsf(v - r) - 0.5f) < 1.220703125e-4f) r = (float)rint((double)x / (double)s);
    r = fminf(fmaxf(r, -127.0f), 127.0f);
    return x == x ? (int)r : 0;
}
__device__ __forceinline__ float kv_magnitude(float x) {
    const float a = fabsf(x);
    return a <= FLT_MAX ? a : 0.0f;
}
__device__ __forceinline__ float4 kv_load4(const float *p, bool wide) {
    if (wide) return *reinterpret_cast<const float4 *>(p);
    return make_float4(p[0], p[1], p[2], p[3]);
}
// the first `count` of four numbers, the others as they are
__device__ __forceinline__ uint32_t kv_requantise(uint32_t w, int count, float ratio, float s_old, float s_new) {
    uint32_t out = w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (i >= count) break;
        const int q = (int)(int8_t)(w >> (8 * i));
        const float v = (float)q * ratio;
        float r = rintf(v);
        if (fabsf(fabsf(v - r) - 0.5f) < 1.220703125e-4f) r = (float)rint((double)q * (double)s_old / (double)s_new);
        out = (out & ~(255u << (8 * i))) | (uint32_t)((int)r & 255) << (8 * i);
    }
    return out;
}

// Pages of the rows of sequence `seq`: the first and how many
struct KvSpan {
    int row0, rows, p0;            // first row, rows, position of the first
    bool live;
};
__device__ __forceinline__ KvSpan kv_span(const KvRows &r, int seq) {
    KvSpan s;
    s.row0 = r.offsets[seq];
    s.rows = r.offsets[seq + 1] - s.row0;
    s.p0 = r.start[seq];
    s.live = s.rows > 0 && s.p0 >= 0;
    return s;
}

constexpr int KVB_KEEP = 8;        // float4 a thread keeps in registers between the maximum and the quantising

template <int T>
__global__ void __launch_bounds__(T) kv_append_kernel(const KvLayer l, const float *__restrict__ k, const float *__restrict__ v, const KvRows rows,
                                                      int per_seq, int wide, int *__restrict__ status) {
    extern __shared__ __align__(16) unsigned char stage[];   // values: [tokens][d + 4]
    __shared__ float red[T / 32];
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, seq = blockIdx.x / per_seq, head = blockIdx.y;
    const bool values = blockIdx.z != 0;
    const KvSpan sp = kv_span(rows, seq);
    if (!sp.live) return;
    const long long end = (long long)sp.p0 + sp.rows;
    const int d4 = l.d >> 2;
    const float *src = (values ? v : k) + (size_t)sp.row0 * rows.stride + (size_t)head * l.d;
    for (long long pg = (sp.p0 >> l.page_shift) + blockIdx.x % per_seq; (pg << l.page_shift) < end; pg += per_seq) {
        if (pg >= l.max_pages) {
            if (tid == 0) atomicExch(status, YSCV_DEV_POS_OVERFLOW);
            return;
        }
        const int id = l.table[(size_t)seq * l.max_pages + pg];
        if (id < 0 || id >= l.n_pages) {
            if (tid == 0) atomicExch(status, YSCV_DEV_BAD_NUMBER);
            continue;
        }
        const long long base = pg << l.page_shift;
        const int t0 = (int)max(0ll, (long long)sp.p0 - base), t1 = (int)min((long long)l.page, end - base);   // new tokens of the page
        const int row = (int)(base + t0 - sp.p0), items = (t1 - t0) * d4;
        float *scale = (values ? l.vs : l.ks) + (size_t)id * l.n_kv + head;
        const float s_old = t0 > 0 ? *scale : 0.0f;
        // largest magnitude of the new tokens
        float4 x[KVB_KEEP];
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < KVB_KEEP; ++i) {
            const int at = tid + T * i;
            if (at < items) {
                const int t = at / d4, c = at - t * d4;
                x[i] = kv_load4(src + (size_t)(row + t) * rows.stride + 4 * c, wide);
                m = fmaxf(m, fmaxf(fmaxf(kv_magnitude(x[i].x), kv_magnitude(x[i].y)), fmaxf(kv_magnitude(x[i].z), kv_magnitude(x[i].w))));
            }
        }
        for (int at = tid + T * KVB_KEEP; at < items; at += T) {
            const int t = at / d4, c = at - t * d4;
            const float4 y = kv_load4(src + (size_t)(row + t) * rows.stride + 4 * c, wide);
            m = fmaxf(m, fmaxf(fmaxf(kv_magnitude(y.x), kv_magnitude(y.y)), fmaxf(kv_magnitude(y.z), kv_magnitude(y.w))));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if ((tid & 31) == 0) red[tid >> 5] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < T / 32; ++i) m = fmaxf(m, red[i]);
        float s = __fdiv_rn(fmaxf(m, KV_LEAST), 127.0f);
        const bool grows = t0 > 0 && s > s_old;
        if (t0 > 0 && !grows) s = s_old;
        const float inv = __fdiv_rn(1.0f, s);
        int8_t *page = (values ? l.v : l.k) + kv_group_at(l, id, head, 0);
        if (grows) {
            // what the page holds, once more: rows of 16 bytes, one token's keys or 16 tokens' values
            const float ratio = __fdiv_rn(s_old, s);
            const int groups = (t0 + KV_GROUP - 1) / KV_GROUP;
            for (int i = tid; i < groups * l.d; i += T) {
                const int in = i % l.d, token = (i / l.d) * KV_GROUP + (values ? 0 : in % KV_GROUP);
                if (token >= t0) continue;
                uint4 *p = reinterpret_cast<uint4 *>(page) + i;
                uint4 w = *p;
                const int count = values ? t0 - token : KV_GROUP;
                w.x = kv_requantise(w.x, count, ratio, s_old, s);
                w.y = kv_requantise(w.y, count - 4, ratio, s_old, s);
                w.z = kv_requantise(w.z, count - 8, ratio, s_old, s);
                w.w = kv_requantise(w.w, count - 12, ratio, s_old, s);
                *p = w;
            }
            if (values) __syncthreads();   // (the last row's bytes of new tokens follow below)
        }
        if (tid == 0 && (t0 == 0 || grows)) *scale = s;
        auto put = [&](int at, const float4 &y) {
            const int t = at / d4, c = at - t * d4;
            const uint32_t w = (uint32_t)(kv_quantise(y.x, s, inv) & 255) | (uint32_t)(kv_quantise(y.y, s, inv) & 255) << 8 |
                               (uint32_t)(kv_quantise(y.z, s, inv) & 255) << 16 | (uint32_t)(kv_quantise(y.w, s, inv) & 255) << 24;
            if (values) {
                *reinterpret_cast<uint32_t *>(stage + t * (l.d + 4) + 4 * c) = w;
            } else {
                const int token = t0 + t;
                *reinterpret_cast<uint32_t *>(page + (token / KV_GROUP) * (KV_GROUP * l.d) + (c >> 2) * 256 + (token % KV_GROUP) * 16 + (c & 3) * 4) = w;
            }
        };
#pragma unroll
        for (int i = 0; i < KVB_KEEP; ++i)
            if (tid + T * i < items) put(tid + T * i, x[i]);
        for (int at = tid + T * KVB_KEEP; at < items; at += T) {
            const int t = at / d4, c = at - t * d4;
            put(at, kv_load4(src + (size_t)(row + t) * rows.stride + 4 * c, wide));
        }
        if (values) {
            __syncthreads();
            const int g0 = t0 / KV_GROUP, g1 = (t1 + KV_GROUP - 1) / KV_GROUP;
            for (int i = tid; i < (g1 - g0) * l.d; i += T) {
                const int g = g0 + i / l.d, c = i % l.d, a = g * KV_GROUP - t0;
                int8_t *p = page + ((size_t)g * l.d + c) * KV_GROUP;
                if (a >= 0 && g * KV_GROUP + KV_GROUP <= t1) {
                    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                    for (int j = 0; j < KV_GROUP; ++j) w[j >> 2] |= (uint32_t)stage[(a + j) * (l.d + 4) + c] << (8 * (j & 3));
                    *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
                } else {
                    for (int j = max(0, -a); j < min(KV_GROUP, t1 - g * KV_GROUP); ++j) p[j] = (int8_t)stage[(a + j) * (l.d + 4) + c];
                }
            }
        }
        __syncthreads();   // red and stage are used again
    }
}

// Cached rows as f32: a CTA per (page, head, keys or values). A thread takes 16 bytes, 16 values of a token's keys or one value
// of 16 tokens.
__global__ void __launch_bounds__(128) kv_read_kernel(const KvLayer l, const KvRows rows, int per_seq, float *__restrict__ k_out, float *__restrict__ v_out,
                                                      int *__restrict__ status) {
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, seq = blockIdx.x / per_seq, head = blockIdx.y;
    const bool values = blockIdx.z != 0;
    const KvSpan sp = kv_span(rows, seq);
    if (!sp.live) return;
    const long long end = (long long)sp.p0 + sp.rows;
    float *dst = (values ? v_out : k_out) + (size_t)sp.row0 * rows.stride + (size_t)head * l.d;
    for (long long pg = (sp.p0 >> l.page_shift) + blockIdx.x % per_seq; (pg << l.page_shift) < end; pg += per_seq) {
        if (pg >= l.max_pages) {
            if (tid == 0) atomicExch(status, YSCV_DEV_POS_OVERFLOW);
            return;
        }
        const int id = l.table[(size_t)seq * l.max_pages + pg];
        if (id < 0 || id >= l.n_pages) {
            if (tid == 0) atomicExch(status, YSCV_DEV_BAD_NUMBER);
            continue;
        }
        const long long base = pg << l.page_shift;
        const int t0 = (int)max(0ll, (long long)sp.p0 - base), t1 = (int)min((long long)l.page, end - base);
        const float s = (values ? l.vs : l.ks)[(size_t)id * l.n_kv + head];
        const int g0 = t0 / KV_GROUP, g1 = (t1 + KV_GROUP - 1) / KV_GROUP;
        const uint4 *page = reinterpret_cast<const uint4 *>((values ? l.v : l.k) + kv_group_at(l, id, head, 0));
        float *out = dst + (base - sp.p0) * (long long)rows.stride;    // the row of the page's first token
        for (int i = g0 * l.d + tid; i < g1 * l.d; i += 128) {
            const int g = i / l.d, in = i - g * l.d;
            const uint4 w = page[i];
            const uint32_t word[4] = {w.x, w.y, w.z, w.w};
            if (values) {
#pragma unroll
                for (int j = 0; j < KV_GROUP; ++j) {
                    const int t = g * KV_GROUP + j;
                    if (t >= t0 && t < t1) out[(size_t)t * rows.stride + in] = (float)(int8_t)(word[j >> 2] >> (8 * (j & 3))) * s;
                }
            } else {
                const int t = g * KV_GROUP + in % KV_GROUP;
                if (t < t0 || t >= t1) continue;
                float *o = out + (size_t)t * rows.stride + (in / KV_GROUP) * 16;
#pragma unroll
                for (int j = 0; j < 16; ++j) o[j] = (float)(int8_t)(word[j >> 2] >> (8 * (j & 3))) * s;
            }
        }
    }
}

// CTAs that a sequence's pages take at most_rows rows, wherever they begin
static int pages_per_seq(const KvLayer &l, size_t most_rows) {
    const size_t n = (most_rows + l.page - 2) / l.page + 1;
    return (int)(n < (size_t)l.max_pages ? n : (size_t)l.max_pages);
}
static int check_rows(yscv_cuda_ctx *ctx, const yscv_cuda_kv_pool *pool, size_t layer, const int32_t *d_offsets, const int32_t *d_start, size_t stride,
                      size_t most_rows, KvLayer *l) {
    if (!ctx) return fail(YSCV_CUDA_ERR_BAD_ARG, "ctx is null");
    if (const int rc = kv_check_pool(pool)) return rc;
    if (const int rc = kv_layer_of(pool, layer, l)) return rc;
    if (!d_offsets || !d_start) return fail(YSCV_CUDA_ERR_BAD_ARG, "null operand");
    if (stride < pool->n_kv * pool->d_head) return fail(YSCV_CUDA_ERR_BAD_ARG, "row stride %zu is shorter than n_kv * d_head", stride);
    if (most_rows >= (1u << 31)) return fail(YSCV_CUDA_ERR_BAD_ARG, "most_rows is too large");
    if (pool->n_seq * (size_t)pages_per_seq(*l, most_rows ? most_rows : 1) >= (1u << 31)) return fail(YSCV_CUDA_ERR_UNSUPPORTED, "too many pages for one call");
    return YSCV_CUDA_OK;
}

}  // namespace yscv

using namespace yscv;

extern "C" {

int yscv_cuda_kv_block_append_dev(yscv_cuda_ctx *ctx, const yscv_cuda_kv_pool *pool, size_t layer, const float *d_k, const float *d_v,
                                  size_t row_stride, const int32_t *d_offsets, const int32_t *d_start, size_t most_rows) {
    KvLayer l;
    if (const int rc = check_rows(ctx, pool, layer, d_offsets, d_start, row_stride, most_rows, &l)) return rc;
    if (!d_k || !d_v) return fail(YSCV_CUDA_ERR_BAD_ARG, "null operand");
    YSCV_CUDA_TRY(cudaSetDevice(ctx->device));
    const int per = pages_per_seq(l, most_rows);
    const bool wide = ((reinterpret_cast<uintptr_t>(d_k) | reinterpret_cast<uintptr_t>(d_v)) & 15) == 0 && row_stride % 4 == 0;
    // two warps where a page gets a token or a few, eight for prompts
    const bool small = most_rows * (size_t)l.d <= 2 * 64 * 4;
    const dim3 grid((unsigned)(l.n_seq * per), (unsigned)l.n_kv, 2);
    const KvRows rows = {d_offsets, d_start, row_stride};
    // (room for a whole page: a sequence may have more rows than were expected)
    const size_t smem = (size_t)l.page * (l.d + 4);
    auto kern = small ? kv_append_kernel<64> : kv_append_kernel<256>;
    YSCV_CUDA_TRY(launch_pdl(kern, grid, dim3(small ? 64 : 256), smem, ctx->stream, l, d_k, d_v, rows, per, (int)wide, ctx->d_status));
    YSCV_CUDA_TRY(cudaGetLastError());
    ctx->launches++;
    ctx->last_kernel = "kv_block_append";
    return YSCV_CUDA_OK;
}

int yscv_cuda_kv_block_read_dev(yscv_cuda_ctx *ctx, const yscv_cuda_kv_pool *pool, size_t layer, const int32_t *d_offsets,
                                const int32_t *d_start, size_t most_rows, float *d_k_out, float *d_v_out, size_t row_stride) {
    KvLayer l;
    if (const int rc = check_rows(ctx, pool, layer, d_offsets, d_start, row_stride, most_rows, &l)) return rc;
    if (!d_k_out || !d_v_out) return fail(YSCV_CUDA_ERR_BAD_ARG, "null operand");
    YSCV_CUDA_TRY(cudaSetDevice(ctx->device));
    const int per = pages_per_seq(l, most_rows);
    const KvRows rows = {d_offsets, d_start, row_stride};
    YSCV_CUDA_TRY(launch_pdl(kv_read_kernel, dim3((unsigned)(l.n_seq * per), (unsigned)l.n_kv, 2), dim3(128), 0, ctx->stream, l, rows, per, d_k_out,
                             d_v_out, ctx->d_status));
    YSCV_CUDA_TRY(cudaGetLastError());
    ctx->launches++;
    ctx->last_kernel = "kv_block_read";
    return YSCV_CUDA_OK;
}

}  // extern "C"
