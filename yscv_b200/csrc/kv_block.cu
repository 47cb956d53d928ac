// Keys and values of ragged rows into the pages of a paged 8-bit cache, and back.
//
// A block of the cache is a page's tokens of one KV head, keys or values; its scale s = fp32(m / 127), m its largest magnitude,
// its values rne(x / s) of the real quotient. The quotient is taken as x * (1 / s) in fp32, which is within 2^-15 of it (three
// roundings of 2^-24 on at most 127.5); where that lies within 2^-13 of a border b between two whole numbers, x - b s decides, whose
// sign one fused multiply-add has exactly.
//
// Append: one CTA per (page that a sequence's rows touch, head, keys or values), so nobody else writes the block or its scale.
// Bound: bytes (4 in, 1 out per value), a decode step: latency, three dependent loads deep. Numbers go through shared memory
// and leave as the cache has them, lanes side by side: 16 bytes of a token's keys, 16 tokens of a value row (a group that other tokens
// share: byte by byte). 3700 rows of 8 heads of 128, pages of 32: 33.9 us with keys stored 4 bytes and value rows gathered a
// byte at a time and an index division per access, 18.5 us, 16.5 with four numbers rounded at once (kv_round4).
#include <cfloat>
#include <type_traits>

#include "attention_tc.cuh"
#include "kv_pool.cuh"

namespace yscv {

struct KvRows {
    const int32_t *offsets, *start;
    size_t stride;                 // floats between rows
    int room;                      // rows of the operands, -1: as many as the last offset says
};

// The whole number next to the border b on the side that the sign of `off` says, the even one on the border itself
__device__ __forceinline__ float kv_side(float b, float off) {
    const float below = b - 0.5f;
    return off > 0.0f || (off == 0.0f && ((int)below & 1)) ? below + 1.0f : below;
}
__device__ __forceinline__ bool kv_near_border(float v, float r) { return fabsf(fabsf(v - r) - 0.5f) < 1.220703125e-4f; }

// Whole number nearest to x / s. NaN: 0, infinities: +-127.
__device__ __noinline__ int kv_quantise(float x, float s, float inv) {
    const float v = x * inv;
    float r = rintf(v);
    if (kv_near_border(v, r)) {
        const float b = floorf(v) + 0.5f;
        r = kv_side(b, fmaf(-b, s, x));
    }
    r = fminf(fmaxf(r, -127.0f), 127.0f);
    return x == x ? (int)r : 0;
}
// Four quotients' whole numbers, where none is near a border or no number: v + 1.5 * 2^23 rounds v to the nearest one and has it in its
// low bits (10 instructions for two numbers; rounding and converting instructions and a test of each took 40)
constexpr float KVB_MAGIC = 12582912.0f;
__device__ __forceinline__ bool kv_round4(uint64_t v01, uint64_t v23, uint32_t &out) {
    const uint64_t magic = f2(KVB_MAGIC, KVB_MAGIC), back = f2(-KVB_MAGIC, -KVB_MAGIC), minus = f2(-1.0f, -1.0f);
    const uint64_t t01 = f2_add(v01, magic), t23 = f2_add(v23, magic);
    float a, b, c, d, t0, t1, t2, t3;
    f2_get(f2_fma(f2_add(t01, back), minus, v01), a, b);
    f2_get(f2_fma(f2_add(t23, back), minus, v23), c, d);
    f2_get(t01, t0, t1);
    f2_get(t23, t2, t3);
    out = __byte_perm(__byte_perm(__float_as_uint(t0), __float_as_uint(t1), 0x0040), __byte_perm(__float_as_uint(t2), __float_as_uint(t3), 0x0040), 0x5410);
    const float sure = 0.5f - 1.220703125e-4f;
    return fabsf(a) < sure && fabsf(b) < sure && fabsf(c) < sure && fabsf(d) < sure;
}
__device__ __forceinline__ uint32_t kv_quantise4(const float4 &x, float s, float inv) {
    uint32_t out;
    if (kv_round4(f2_mul(f2(x.x, x.y), f2(inv, inv)), f2_mul(f2(x.z, x.w), f2(inv, inv)), out)) return out;
    return (uint32_t)(kv_quantise(x.x, s, inv) & 255) | (uint32_t)(kv_quantise(x.y, s, inv) & 255) << 8 | (uint32_t)(kv_quantise(x.z, s, inv) & 255) << 16 |
           (uint32_t)(kv_quantise(x.w, s, inv) & 255) << 24;
}
// the largest magnitude but for infinities (and NaN, which a maximum passes over)
__device__ __forceinline__ float kv_most(const float4 &x) {
    const float m = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
    if (m <= FLT_MAX) return m;
    auto finite = [](float y) { return fabsf(y) <= FLT_MAX ? fabsf(y) : 0.0f; };
    return fmaxf(fmaxf(finite(x.x), finite(x.y)), fmaxf(finite(x.z), finite(x.w)));
}
__device__ __forceinline__ float4 kv_load4(const float *p, bool wide) {
    if (wide) return *reinterpret_cast<const float4 *>(p);
    return make_float4(p[0], p[1], p[2], p[3]);
}
// Whole number nearest to q s_old / s_new
__device__ __noinline__ int kv_requantise1(int q, float ratio, float s_old, float s_new) {
    const float v = (float)q * ratio;
    float r = rintf(v);
    if (kv_near_border(v, r)) {
        // q s_old - b s_new: the product's rounding apart, the difference of what is left is exact so near the border
        const float b = floorf(v) + 0.5f, p = (float)q * s_old;
        r = kv_side(b, fmaf(-b, s_new, p) + fmaf((float)q, s_old, -p));
    }
    return (int)r;
}
// the first `count` of four numbers, the others as they are
__device__ __forceinline__ uint32_t kv_requantise(uint32_t w, int count, float ratio, float s_old, float s_new) {
    if (count <= 0) return w;
    // 2^23 + q + 128, less that
    const uint32_t x = w ^ 0x80808080u, top = 0x4B000000u;
    const uint64_t off = f2(-8388736.0f, -8388736.0f), by = f2(ratio, ratio);
    auto number = [&](int sel) { return __uint_as_float(__byte_perm(x, top, sel)); };
    uint32_t out;
    if (!kv_round4(f2_mul(f2_add(f2(number(0x7440), number(0x7441)), off), by), f2_mul(f2_add(f2(number(0x7442), number(0x7443)), off), by), out)) {
        out = 0;
#pragma unroll 1
        for (int i = 0; i < 4; ++i) out |= (uint32_t)(kv_requantise1((int)(int8_t)(w >> (8 * i)), ratio, s_old, s_new) & 255) << (8 * i);
    }
    const uint32_t mask = count >= 4 ? 0xffffffffu : (1u << (8 * count)) - 1u;
    return (out & mask) | (w & ~mask);
}

// Pages of the rows of sequence `seq`: the first and how many
struct KvSpan {
    int row0, rows, p0;            // first row, rows, position of the first
    bool live, inside;             // takes part; has rows of the operands
};
__device__ __forceinline__ KvSpan kv_span(const KvRows &r, int seq, int n_seq) {
    KvSpan s;
    const int end = r.offsets[seq + 1], last = r.offsets[n_seq];
    s.row0 = r.offsets[seq];
    s.p0 = r.start[seq];
    // (as kv_rows() of kv_attention.cuh: offsets that fall, or lie outside the operands, are nobody's rows)
    s.inside = s.row0 >= 0 && s.row0 <= end && end <= (r.room >= 0 ? r.room : last);
    s.rows = end - s.row0;
    s.live = s.inside && s.rows > 0 && s.p0 >= 0;
    return s;
}
// What is said of a sequence that takes no part, once
__device__ __forceinline__ void kv_span_status(const KvSpan &s, int per_seq, int *status) {
    if (!s.inside && threadIdx.x == 0 && blockIdx.x % per_seq == 0 && blockIdx.y == 0 && blockIdx.z == 0) atomicExch(status, YSCV_DEV_BAD_NUMBER);
}

constexpr int KVB_KEEP = 8;        // float4 a thread keeps in registers between the maximum and the quantising
__host__ __device__ constexpr int kv_stage_pitch(int d) { return d + 16; }   // bytes of a staged token

// four tokens' words of four d -> four d's words of four tokens
__device__ __forceinline__ void kv_turn(const uint32_t (&w)[4], uint32_t (&out)[4]) {
    const uint32_t a = __byte_perm(w[0], w[1], 0x5140), b = __byte_perm(w[2], w[3], 0x5140);   // {0.0, 1.0, 0.1, 1.1}, ...
    const uint32_t c = __byte_perm(w[0], w[1], 0x7362), d = __byte_perm(w[2], w[3], 0x7362);   // {0.2, 1.2, 0.3, 1.3}, ...
    out[0] = __byte_perm(a, b, 0x5410);
    out[1] = __byte_perm(a, b, 0x7632);
    out[2] = __byte_perm(c, d, 0x5410);
    out[3] = __byte_perm(c, d, 0x7632);
}

// (D: the head size, 0 for any; a division by it is a shift where it is known)
template <int T, int D>
__global__ void __launch_bounds__(T, 1024 / T) kv_append_kernel(const KvLayer l, const float *k, const float *v, const KvRows rows,
                                                      int per_seq, int wide, int *__restrict__ status) {
    extern __shared__ __align__(16) unsigned char stage[];   // [tokens][kv_stage_pitch(d)]
    __shared__ float red[T / 32];
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, seq = blockIdx.x / per_seq, head = blockIdx.y;
    const bool values = blockIdx.z != 0;
    const KvSpan sp = kv_span(rows, seq, l.n_seq);
    if (!sp.live) {
        kv_span_status(sp, per_seq, status);
        return;
    }
    const long long end = (long long)sp.p0 + sp.rows;
    // a thread has four d of every `step`-th token
    const int d = D ? D : l.d, d4 = d >> 2, step = T / d4, c = tid % d4, first = tid / d4 < step ? tid / d4 : 1 << 30, pitch = kv_stage_pitch(d);
    const float *src = (values ? v : k) + (size_t)sp.row0 * rows.stride + (size_t)head * d + 4 * c;
    for (long long pg = (sp.p0 >> l.page_shift) + blockIdx.x % per_seq; (pg << l.page_shift) < end; pg += per_seq) {
        if (pg >= l.max_pages) {
            if (tid == 0) atomicExch(status, YSCV_DEV_POS_OVERFLOW);
            return;
        }
        const int id = l.table[(size_t)seq * l.max_pages + pg];
        const long long base = pg << l.page_shift;
        const int t0 = (int)max(0ll, (long long)sp.p0 - base), t1 = (int)min((long long)l.page, end - base);   // new tokens of the page
        const int n = t1 - t0;
        const float *row = src + (size_t)(base + t0 - sp.p0) * rows.stride;
        // largest magnitude of the new tokens
        float4 x[KVB_KEEP];
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < KVB_KEEP; ++i) {
            const int t = first + step * i;
            if (t < n) x[i] = kv_load4(row + (size_t)t * rows.stride, wide);
        }
        if (id < 0 || id >= l.n_pages) {
            if (tid == 0) atomicExch(status, YSCV_DEV_BAD_NUMBER);
            continue;
        }
        float *scale = (values ? l.vs : l.ks) + (size_t)id * l.n_kv + head;
        const float s_old = t0 > 0 ? *scale : 0.0f;
#pragma unroll
        for (int i = 0; i < KVB_KEEP; ++i)
            if (first + step * i < n)
                m = fmaxf(m, kv_most(x[i]));
        for (int t = first + step * KVB_KEEP; t < n; t += step) {
            m = fmaxf(m, kv_most(kv_load4(row + (size_t)t * rows.stride, wide)));
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
            for (int i = tid; i < groups * d; i += T) {
                const int in = i % d, token = (i / d) * KV_GROUP + (values ? 0 : in % KV_GROUP);
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
        }
        if (tid == 0 && (t0 == 0 || grows)) *scale = s;
        auto put = [&](int t, const float4 &y) {
            *reinterpret_cast<uint32_t *>(stage + t * pitch + 4 * c) = kv_quantise4(y, s, inv);
        };
#pragma unroll
        for (int i = 0; i < KVB_KEEP; ++i)
            if (first + step * i < n) put(first + step * i, x[i]);
        for (int t = first + step * KVB_KEEP; t < n; t += step) put(t, kv_load4(row + (size_t)t * rows.stride, wide));
        __syncthreads();   // (the last value row's bytes of new tokens follow those that were rounded again)
        if (!values) {
            const int i1 = ((t1 + KV_GROUP - 1) / KV_GROUP) * d;
            for (int i = t0 / KV_GROUP * d + tid; i < i1; i += T) {
                const int g = i / d, in = i - g * d, t = g * KV_GROUP + in % KV_GROUP - t0;
                if (t >= 0 && t < n) reinterpret_cast<uint4 *>(page)[i] = *reinterpret_cast<const uint4 *>(stage + t * pitch + (in / KV_GROUP) * 16);
            }
        } else {
            const int i1 = ((t1 + KV_GROUP - 1) / KV_GROUP) * d4;
            for (int i = t0 / KV_GROUP * d4 + tid; i < i1; i += T) {
                const int g = i / d4, at = i - g * d4, t = g * KV_GROUP - t0;     // four rows of the group's d
                int8_t *p = page + (size_t)i * (4 * KV_GROUP);
                const unsigned char *from = stage + t * pitch + 4 * at;
                if (t >= 0 && t + KV_GROUP <= n) {
                    uint32_t out[4][4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        uint32_t w[4], r[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const uint32_t *>(from + (4 * q + j) * pitch);
                        kv_turn(w, r);
#pragma unroll
                        for (int j = 0; j < 4; ++j) out[j][q] = r[j];
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) reinterpret_cast<uint4 *>(p)[j] = make_uint4(out[j][0], out[j][1], out[j][2], out[j][3]);
                } else {
                    for (int q = max(0, -t); q < min(KV_GROUP, n - t); ++q) {
                        const uint32_t w = *reinterpret_cast<const uint32_t *>(from + q * pitch);
#pragma unroll
                        for (int j = 0; j < 4; ++j) p[j * KV_GROUP + q] = (int8_t)(w >> (8 * j));
                    }
                }
            }
        }
        __syncthreads();   // red and stage are used again
    }
}

// four numbers times s: 2^23 + q + 128, less that (a conversion is a quarter of the rate)
__device__ __forceinline__ float4 kv_floats(uint32_t w, float s) {
    const uint32_t x = w ^ 0x80808080u, top = 0x4B000000u;
    auto number = [&](int sel) { return __uint_as_float(__byte_perm(x, top, sel)); };
    const uint64_t off = f2(-8388736.0f, -8388736.0f), by = f2(s, s);
    float4 y;
    f2_get(f2_mul(f2_add(f2(number(0x7440), number(0x7441)), off), by), y.x, y.y);
    f2_get(f2_mul(f2_add(f2(number(0x7442), number(0x7443)), off), by), y.z, y.w);
    return y;
}

// Cached rows as f32: a CTA per (page, head, keys or values), a warp per group of 16 tokens. A lane has four d, keys as they lie,
// values turned around, so that a row leaves in whole lines. 3700 rows of 8 heads of 128: 13.3 us with a d of 16 tokens per lane, 10.1 so.
__global__ void __launch_bounds__(128, 8) kv_read_kernel(const KvLayer l, const KvRows rows, int per_seq, float *__restrict__ k_out, float *__restrict__ v_out,
                                                      int wide, int *__restrict__ status) {
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, seq = blockIdx.x / per_seq, head = blockIdx.y;
    const bool values = blockIdx.z != 0;
    const KvSpan sp = kv_span(rows, seq, l.n_seq);
    if (!sp.live) {
        kv_span_status(sp, per_seq, status);
        return;
    }
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
        const int8_t *page = (values ? l.v : l.k) + kv_group_at(l, id, head, 0);
        float *out = dst + (base - sp.p0) * (long long)rows.stride;    // the row of the page's first token
        for (int g = t0 / KV_GROUP + (tid >> 5); g * KV_GROUP < t1; g += 4) {
            const int a = max(t0, g * KV_GROUP), b = min(t1, g * KV_GROUP + KV_GROUP);
            const int8_t *group = page + (size_t)g * (KV_GROUP * l.d);
            float *o = out + (size_t)a * rows.stride;
            auto put = [&](float *p, uint32_t w) {
                const float4 y = kv_floats(w, s);
                if (wide) {
                    *reinterpret_cast<float4 *>(p) = y;
                } else {
                    p[0] = y.x; p[1] = y.y; p[2] = y.z; p[3] = y.w;
                }
            };
            if (values) {
                for (int c = lane; c < l.d >> 2; c += 32) {
                    uint4 w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] = reinterpret_cast<const uint4 *>(group)[4 * c + j];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        auto word = [&](const uint4 &y) { return q == 0 ? y.x : q == 1 ? y.y : q == 2 ? y.z : y.w; };
                        const uint32_t in[4] = {word(w[0]), word(w[1]), word(w[2]), word(w[3])};
                        uint32_t out[4];
                        kv_turn(in, out);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int t = g * KV_GROUP + 4 * q + j;
                            if (t >= a && t < b) put(o + (size_t)(t - a) * rows.stride + 4 * c, out[j]);
                        }
                    }
                }
            } else {
                for (int c = lane; c < l.d >> 2; c += 32) {
                    const int8_t *from = group + (c >> 2) * 256 + (c & 3) * 4 + (a - g * KV_GROUP) * 16;
#pragma unroll 8
                    for (int t = 0; t < b - a; ++t) {
                        put(o + (size_t)t * rows.stride + 4 * c, *reinterpret_cast<const uint32_t *>(from + t * 16));
                    }
                }
            }
        }
    }
}

// CTAs that a sequence's pages take at most_rows rows, wherever they begin
static int pages_per_seq(const KvLayer &l, size_t most_rows) {
    const size_t n = (most_rows + l.page - 2) / l.page + 1;
    return (int)(n < (size_t)l.max_pages ? n : (size_t)l.max_pages);
}
constexpr size_t KVB_ROWS_UNKNOWN = ~(size_t)0;
static int room_of(size_t rows) { return rows == KVB_ROWS_UNKNOWN ? -1 : (int)rows; }
static int check_rows(yscv_cuda_ctx *ctx, const yscv_cuda_kv_pool *pool, size_t layer, const int32_t *d_offsets, const int32_t *d_start, size_t stride,
                      size_t rows, size_t most_rows, KvLayer *l) {
    if (!ctx) return fail(YSCV_CUDA_ERR_BAD_ARG, "ctx is null");
    if (const int rc = kv_check_pool(pool)) return rc;
    if (const int rc = kv_layer_of(pool, layer, l)) return rc;
    if (!d_offsets || !d_start) return fail(YSCV_CUDA_ERR_BAD_ARG, "null operand");
    if (!kv_aligned({d_offsets, d_start})) return fail(YSCV_CUDA_ERR_UNSUPPORTED, "operands must be 4-byte aligned");
    if (stride < pool->n_kv * pool->d_head) return fail(YSCV_CUDA_ERR_BAD_ARG, "row stride %zu is shorter than n_kv * d_head", stride);
    if (most_rows >= (1u << 31)) return fail(YSCV_CUDA_ERR_BAD_ARG, "most_rows is too large");
    if (rows != KVB_ROWS_UNKNOWN && rows >= (1u << 31)) return fail(YSCV_CUDA_ERR_UNSUPPORTED, "too many rows");
    if (pool->n_seq * (size_t)pages_per_seq(*l, most_rows ? most_rows : 1) >= (1u << 31)) return fail(YSCV_CUDA_ERR_UNSUPPORTED, "too many pages for one call");
    return YSCV_CUDA_OK;
}

static int kv_append(yscv_cuda_ctx *ctx, const yscv_cuda_kv_pool *pool, size_t layer, const float *d_k, const float *d_v, size_t row_stride,
                     const int32_t *d_offsets, const int32_t *d_start, size_t n_rows, size_t most_rows) {
    KvLayer l;
    if (const int rc = check_rows(ctx, pool, layer, d_offsets, d_start, row_stride, n_rows, most_rows, &l)) return rc;
    if (!d_k || !d_v) return fail(YSCV_CUDA_ERR_BAD_ARG, "null operand");
    if (!kv_aligned({d_k, d_v})) return fail(YSCV_CUDA_ERR_UNSUPPORTED, "operands must be 4-byte aligned");
    YSCV_CUDA_TRY(cudaSetDevice(ctx->device));
    const int per = pages_per_seq(l, most_rows);
    const bool wide = ((reinterpret_cast<uintptr_t>(d_k) | reinterpret_cast<uintptr_t>(d_v)) & 15) == 0 && row_stride % 4 == 0;
    // threads by what a page gets, so that KVB_KEEP loads a thread hold it: two warps for a token or a few, up to 16
    const size_t most = (most_rows < pool->page ? most_rows : pool->page) * pool->d_head;
    const int threads = most <= 2 * 64 * 4 ? 64 : most <= 128 * 4 * KVB_KEEP ? 128 : most <= 256 * 4 * KVB_KEEP ? 256 : 512;
    const dim3 grid((unsigned)(l.n_seq * per), (unsigned)l.n_kv, 2);
    const KvRows rows = {d_offsets, d_start, row_stride, room_of(n_rows)};
    // (room for a whole page: a sequence may have more rows than were expected)
    const size_t smem = (size_t)l.page * kv_stage_pitch(l.d);
    auto of = [&](auto size) {
        constexpr int D = decltype(size)::value;
        return threads == 64 ? kv_append_kernel<64, D> : threads == 128 ? kv_append_kernel<128, D> : threads == 256 ? kv_append_kernel<256, D> : kv_append_kernel<512, D>;
    };
    auto kern = l.d == 64    ? of(std::integral_constant<int, 64>())
                : l.d == 128 ? of(std::integral_constant<int, 128>())
                : l.d == 256 ? of(std::integral_constant<int, 256>())
                             : of(std::integral_constant<int, 0>());
    YSCV_CUDA_TRY(launch_pdl(kern, grid, dim3((unsigned)threads), smem, ctx->stream, l, d_k, d_v, rows, per, (int)wide, ctx->d_status));
    YSCV_CUDA_TRY(cudaGetLastError());
    ctx->launches++;
    ctx->last_kernel = "kv_block_append";
    return YSCV_CUDA_OK;
}

static int kv_read(yscv_cuda_ctx *ctx, const yscv_cuda_kv_pool *pool, size_t layer, const int32_t *d_offsets, const int32_t *d_start, size_t n_rows,
                   size_t most_rows, float *d_k_out, float *d_v_out, size_t row_stride) {
    KvLayer l;
    if (const int rc = check_rows(ctx, pool, layer, d_offsets, d_start, row_stride, n_rows, most_rows, &l)) return rc;
    if (!d_k_out || !d_v_out) return fail(YSCV_CUDA_ERR_BAD_ARG, "null operand");
    if (!kv_aligned({d_k_out, d_v_out})) return fail(YSCV_CUDA_ERR_UNSUPPORTED, "operands must be 4-byte aligned");
    YSCV_CUDA_TRY(cudaSetDevice(ctx->device));
    const int per = pages_per_seq(l, most_rows);
    const KvRows rows = {d_offsets, d_start, row_stride, room_of(n_rows)};
    YSCV_CUDA_TRY(launch_pdl(kv_read_kernel, dim3((unsigned)(l.n_seq * per), (unsigned)l.n_kv, 2), dim3(128), 0, ctx->stream, l, rows, per, d_k_out,
                             d_v_out, (int)(((reinterpret_cast<uintptr_t>(d_k_out) | reinterpret_cast<uintptr_t>(d_v_out)) & 15) == 0 && row_stride % 4 == 0),
                             ctx->d_status));
    YSCV_CUDA_TRY(cudaGetLastError());
    ctx->launches++;
    ctx->last_kernel = "kv_block_read";
    return YSCV_CUDA_OK;
}

}  // namespace yscv

using namespace yscv;

extern "C" {

int yscv_cuda_kv_block_append_dev(yscv_cuda_ctx *ctx, const yscv_cuda_kv_pool *pool, size_t layer, const float *d_k, const float *d_v,
                                  size_t row_stride, const int32_t *d_offsets, const int32_t *d_start, size_t most_rows) {
    return kv_append(ctx, pool, layer, d_k, d_v, row_stride, d_offsets, d_start, KVB_ROWS_UNKNOWN, most_rows);
}
int yscv_cuda_kv_block_append_rows_dev(yscv_cuda_ctx *ctx, const yscv_cuda_kv_pool *pool, size_t layer, const float *d_k, const float *d_v,
                                       size_t row_stride, const int32_t *d_offsets, const int32_t *d_start, size_t rows, size_t most_rows) {
    if (rows == KVB_ROWS_UNKNOWN) return fail(YSCV_CUDA_ERR_UNSUPPORTED, "too many rows");
    return kv_append(ctx, pool, layer, d_k, d_v, row_stride, d_offsets, d_start, rows, most_rows);
}

int yscv_cuda_kv_block_read_dev(yscv_cuda_ctx *ctx, const yscv_cuda_kv_pool *pool, size_t layer, const int32_t *d_offsets,
                                const int32_t *d_start, size_t most_rows, float *d_k_out, float *d_v_out, size_t row_stride) {
    return kv_read(ctx, pool, layer, d_offsets, d_start, KVB_ROWS_UNKNOWN, most_rows, d_k_out, d_v_out, row_stride);
}
int yscv_cuda_kv_block_read_rows_dev(yscv_cuda_ctx *ctx, const yscv_cuda_kv_pool *pool, size_t layer, const int32_t *d_offsets,
                                     const int32_t *d_start, size_t rows, size_t most_rows, float *d_k_out, float *d_v_out, size_t row_stride) {
    if (rows == KVB_ROWS_UNKNOWN) return fail(YSCV_CUDA_ERR_UNSUPPORTED, "too many rows");
    return kv_read(ctx, pool, layer, d_offsets, d_start, rows, most_rows, d_k_out, d_v_out, row_stride);
}

}  // extern "C"
