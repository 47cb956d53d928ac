// Rotary positions of ragged rows: every row has a position of its own, pairs lie half a head apart or side by side, the first
// `rotary_dim` values of a head turn and the rest pass through, frequencies are stretched for contexts longer than the model's.
//
//   (a, b) -> f (a cos(p w_i) - b sin(p w_i), b cos(p w_i) + a sin(p w_i)),   w_i = theta^(-2 i / rotary_dim), stretched
//
// The one product that needs more than fp32 is p w_i: at position 10^6 an fp32 angle is off by 0.06 radians. It is formed in
// fp64 as quarter turns and reduced there to [-1/2, 1/2] of one, so what is left for fp32 is exact to 2^-25 of a quarter.
// The frequencies come from the host in fp64, as an argument.
//
// Bound: bytes, 8 per value; a few rows: latency. A block takes a row, or as many heads of it as leave every SM a block; its
// first threads work the factors out once for all heads, while the block's first values are on their way. A thread keeps its
// place in the head and walks the heads, so its four factors stay in registers.
#include <cmath>

#include "common.cuh"
#include "kv_pool.cuh"

namespace yscv {

constexpr int ROPE_DEV_THREADS = 256, ROPE_MOST_PAIRS = 256;

struct RopeCall {
    const float *x;
    float *out;
    const int32_t *pos;
    size_t x_stride, out_stride;
    int heads, d, rot, interleaved, in_place;
    float factor;                          // on cosine and sine
    double turns[ROPE_MOST_PAIRS];         // quarter turns per position
};

// cosine and sine of `q` quarter turns, times f
__device__ __forceinline__ float2 rope_factors(double q, float f) {
    const double k = rint(q);
    const int quadrant = (int)(long long)k & 3;
    float s, c;
    sincospif(0.5f * (float)(q - k), &s, &c);
    const float cq = quadrant & 1 ? s : c, sq = quadrant & 1 ? c : s;
    return make_float2(quadrant == 1 || quadrant == 2 ? -cq * f : cq * f, quadrant & 2 ? -sq * f : sq * f);
}

// Eight values of a head: the pairs 4 u .. 4 u + 3, or eight that pass through
__device__ __forceinline__ void rope_load8(const float *h, int u, const RopeCall &a, float4 &lo, float4 &hi) {
    const int turning = a.rot >> 3;
    const bool halves = u < turning && !a.interleaved;
    const float *p = h + (halves ? 4 * u : 8 * u);
    lo = *reinterpret_cast<const float4 *>(p);
    hi = *reinterpret_cast<const float4 *>(halves ? p + a.rot / 2 : p + 4);
}

// d and rot multiples of 8, rows 16-byte aligned
__global__ void __launch_bounds__(ROPE_DEV_THREADS) rope_rows_kernel(const __grid_constant__ RopeCall a) {
    __shared__ float2 cs[ROPE_MOST_PAIRS];
    pdl_wait();
    pdl_trigger();
    const int p = a.pos[blockIdx.x];
    if (p < 0) return;                     // a row that belongs to nobody
    const int units = a.d >> 3, per = ROPE_DEV_THREADS / units;
    const int u = threadIdx.x % units, turning = a.rot >> 3;
    const int step = per * gridDim.y;
    int head = blockIdx.y * per + threadIdx.x / units;
    if ((int)threadIdx.x / units >= per) head = a.heads;
    const float *x = a.x + blockIdx.x * a.x_stride;
    float *out = a.out + blockIdx.x * a.out_stride;
    float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
    if (head < a.heads) rope_load8(x + (size_t)head * a.d, u, a, lo, hi);
    for (int i = threadIdx.x; i < a.rot / 2; i += ROPE_DEV_THREADS) cs[i] = rope_factors((double)p * a.turns[i], a.factor);
    __syncthreads();
    float c[4], s[4];
    if (u < turning) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { c[i] = cs[4 * u + i].x; s[i] = cs[4 * u + i].y; }
    } else if (a.in_place) {
        return;
    }
    while (head < a.heads) {
        const int next = head + step;
        float4 nlo = lo, nhi = hi;
        if (next < a.heads) rope_load8(x + (size_t)next * a.d, u, a, nlo, nhi);
        float *o = out + (size_t)head * a.d;
        if (u >= turning) {
            *reinterpret_cast<float4 *>(o + 8 * u) = lo;
            *reinterpret_cast<float4 *>(o + 8 * u + 4) = hi;
        } else if (a.interleaved) {
            *reinterpret_cast<float4 *>(o + 8 * u) = make_float4(lo.x * c[0] - lo.y * s[0], lo.y * c[0] + lo.x * s[0],
                                                                 lo.z * c[1] - lo.w * s[1], lo.w * c[1] + lo.z * s[1]);
            *reinterpret_cast<float4 *>(o + 8 * u + 4) = make_float4(hi.x * c[2] - hi.y * s[2], hi.y * c[2] + hi.x * s[2],
                                                                     hi.z * c[3] - hi.w * s[3], hi.w * c[3] + hi.z * s[3]);
        } else {
            *reinterpret_cast<float4 *>(o + 4 * u) = make_float4(lo.x * c[0] - hi.x * s[0], lo.y * c[1] - hi.y * s[1],
                                                                 lo.z * c[2] - hi.z * s[2], lo.w * c[3] - hi.w * s[3]);
            *reinterpret_cast<float4 *>(o + a.rot / 2 + 4 * u) = make_float4(hi.x * c[0] + lo.x * s[0], hi.y * c[1] + lo.y * s[1],
                                                                             hi.z * c[2] + lo.z * s[2], hi.w * c[3] + lo.w * s[3]);
        }
        head = next;
        lo = nlo;
        hi = nhi;
    }
}

// Any sizes and alignment: a thread per pair or value that passes through
__global__ void __launch_bounds__(ROPE_DEV_THREADS) rope_rows_any_kernel(const __grid_constant__ RopeCall a) {
    __shared__ float2 cs[ROPE_MOST_PAIRS];
    pdl_wait();
    pdl_trigger();
    const int p = a.pos[blockIdx.x];
    if (p < 0) return;
    const int pairs = a.rot / 2, units = a.d - pairs;
    for (int i = threadIdx.x; i < pairs; i += ROPE_DEV_THREADS) cs[i] = rope_factors((double)p * a.turns[i], a.factor);
    __syncthreads();
    const float *x = a.x + blockIdx.x * a.x_stride;
    float *out = a.out + blockIdx.x * a.out_stride;
    const int items = a.heads * units, step = ROPE_DEV_THREADS * gridDim.y;
    for (int i = blockIdx.y * ROPE_DEV_THREADS + threadIdx.x; i < items; i += step) {
        const int head = i / units, u = i - head * units;
        const float *h = x + (size_t)head * a.d;
        float *o = out + (size_t)head * a.d;
        if (u < pairs) {
            const int i0 = a.interleaved ? 2 * u : u, i1 = a.interleaved ? 2 * u + 1 : u + pairs;
            const float v0 = h[i0], v1 = h[i1];
            o[i0] = v0 * cs[u].x - v1 * cs[u].y;
            o[i1] = v1 * cs[u].x + v0 * cs[u].y;
        } else if (!a.in_place) {
            o[u + pairs] = h[u + pairs];
        }
    }
}

// Radians per position of every pair, in fp64, and the factor on cosine and sine
static int rope_frequencies(const yscv_cuda_rope *r, RopeCall &a) {
    const int pairs = (int)r->rotary_dim / 2;
    const double pi = 3.14159265358979323846, rot = (double)r->rotary_dim;
    if (!(r->theta > 1.0) || !std::isfinite(r->theta)) return fail(YSCV_CUDA_ERR_BAD_ARG, "theta must be above 1");
    const bool stretched = r->scaling != YSCV_CUDA_ROPE_NONE;
    if (r->scaling < YSCV_CUDA_ROPE_NONE || r->scaling > YSCV_CUDA_ROPE_YARN) return fail(YSCV_CUDA_ERR_BAD_ARG, "scaling %d is not one of yscv_cuda_rope's", r->scaling);
    if (stretched && (!(r->factor >= 1.0) || !std::isfinite(r->factor))) return fail(YSCV_CUDA_ERR_BAD_ARG, "factor must be at least 1");
    if (r->scaling >= YSCV_CUDA_ROPE_BANDED && !(r->original_positions > 0.0)) return fail(YSCV_CUDA_ERR_BAD_ARG, "original_positions must be positive");
    if (r->scaling == YSCV_CUDA_ROPE_BANDED && !(r->low_band > 0.0 && r->high_band > r->low_band))
        return fail(YSCV_CUDA_ERR_BAD_ARG, "high_band must be above low_band, and both positive");
    if (r->scaling == YSCV_CUDA_ROPE_YARN && !(r->beta_slow > 0.0 && r->beta_fast > r->beta_slow))
        return fail(YSCV_CUDA_ERR_BAD_ARG, "beta_fast must be above beta_slow, and both positive");
    if (!(r->attention_factor >= 0.0) || !std::isfinite(r->attention_factor)) return fail(YSCV_CUDA_ERR_BAD_ARG, "attention_factor must be 0 (the default) or positive");
    double low = 0.0, high = 0.0;
    if (r->scaling == YSCV_CUDA_ROPE_YARN) {
        auto pair_of = [&](double beta) { return rot * std::log(r->original_positions / (2.0 * pi * beta)) / (2.0 * std::log(r->theta)); };
        low = std::max(std::floor(pair_of(r->beta_fast)), 0.0);
        high = std::min(std::ceil(pair_of(r->beta_slow)), rot - 1.0);
    }
    // (a product each in the place of a power: 0.2 us a call for 64 pairs, not 3; off by i 2^-53 of w_i, which falls faster)
    const double ratio = std::pow(r->theta, -2.0 / rot);
    double natural = 1.0;
    for (int i = 0; i < pairs; ++i, natural *= ratio) {
        double w = natural;
        double kept = stretched ? 0.0 : 1.0;           // the part of the frequency that is not stretched
        if (r->scaling == YSCV_CUDA_ROPE_BANDED) {
            const double turns = r->original_positions * w / (2.0 * pi);
            kept = std::min(1.0, std::max(0.0, (turns - r->low_band) / (r->high_band - r->low_band)));
        } else if (r->scaling == YSCV_CUDA_ROPE_YARN) {
            kept = 1.0 - std::min(1.0, std::max(0.0, (i - low) / std::max(high - low, 0.001)));
        }
        if (stretched) w *= kept + (1.0 - kept) / r->factor;
        a.turns[i] = w * (2.0 / pi);
    }
    a.factor = r->attention_factor > 0.0 ? (float)r->attention_factor
               : r->scaling == YSCV_CUDA_ROPE_YARN ? (float)(0.1 * std::log(r->factor) + 1.0) : 1.0f;
    return YSCV_CUDA_OK;
}

}  // namespace yscv

using namespace yscv;

extern "C" int yscv_cuda_rope_dev(yscv_cuda_ctx *ctx, const float *d_x, size_t x_stride, size_t rows, size_t n_heads, size_t d_head,
                                  const int32_t *d_pos, const yscv_cuda_rope *rope, float *d_out, size_t out_stride) {
    if (!ctx) return fail(YSCV_CUDA_ERR_BAD_ARG, "ctx is null");
    if (!rope) return fail(YSCV_CUDA_ERR_BAD_ARG, "rope is null");
    if (n_heads == 0 || d_head == 0 || n_heads > (1u << 20) || d_head > (1u << 16) || n_heads * d_head >= (1u << 30))
        return fail(YSCV_CUDA_ERR_BAD_ARG, "n_heads=%zu and d_head=%zu must be positive and of a row's size", n_heads, d_head);
    if (rope->rotary_dim == 0 || rope->rotary_dim % 2 != 0 || rope->rotary_dim > d_head)
        return fail(YSCV_CUDA_ERR_BAD_ARG, "rotary_dim=%zu must be even, positive and at most d_head", rope->rotary_dim);
    if (rope->rotary_dim > 2 * ROPE_MOST_PAIRS) return fail(YSCV_CUDA_ERR_UNSUPPORTED, "rotary_dim is at most %d", 2 * ROPE_MOST_PAIRS);
    if (x_stride < n_heads * d_head || out_stride < n_heads * d_head)
        return fail(YSCV_CUDA_ERR_BAD_ARG, "a row stride is shorter than n_heads * d_head");
    if (d_x == d_out && x_stride != out_stride) return fail(YSCV_CUDA_ERR_BAD_ARG, "in place the two row strides are one");
    if (rows >= (1u << 31)) return fail(YSCV_CUDA_ERR_UNSUPPORTED, "too many rows");
    RopeCall a;
    int rc = rope_frequencies(rope, a);
    if (rc || rows == 0) return rc;
    if (!d_x || !d_pos || !d_out) return fail(YSCV_CUDA_ERR_BAD_ARG, "null operand");
    if (!kv_aligned({d_x, d_pos, d_out})) return fail(YSCV_CUDA_ERR_UNSUPPORTED, "operands must be 4-byte aligned");
    YSCV_CUDA_TRY(cudaSetDevice(ctx->device));
    a.x = d_x; a.out = d_out; a.pos = d_pos; a.x_stride = x_stride; a.out_stride = out_stride;
    a.heads = (int)n_heads; a.d = (int)d_head; a.rot = (int)rope->rotary_dim; a.interleaved = rope->interleaved != 0;
    a.in_place = d_x == d_out;
    const uintptr_t at = reinterpret_cast<uintptr_t>(d_x) | reinterpret_cast<uintptr_t>(d_out);
    const bool wide = d_head % 8 == 0 && a.rot % 8 == 0 && x_stride % 4 == 0 && out_stride % 4 == 0 && (at & 15) == 0 &&
                      d_head <= 8 * ROPE_DEV_THREADS;
    const size_t items = wide ? (n_heads + ROPE_DEV_THREADS / (d_head / 8) - 1) / (ROPE_DEV_THREADS / (d_head / 8))
                              : (n_heads * (d_head - a.rot / 2) + ROPE_DEV_THREADS - 1) / ROPE_DEV_THREADS;
    // blocks per row: what it takes to give every SM four blocks, as far as a row has work for them
    size_t pieces = (4 * (size_t)ctx->sm_count + rows - 1) / rows;
    if (pieces > items) pieces = items;
    if (pieces > 65535) pieces = 65535;
    YSCV_CUDA_TRY(launch_pdl(wide ? rope_rows_kernel : rope_rows_any_kernel, dim3((unsigned)rows, (unsigned)pieces), dim3(ROPE_DEV_THREADS), 0,
                             ctx->stream, a));
    YSCV_CUDA_TRY(cudaGetLastError());
    ctx->launches++;
    ctx->last_kernel = wide ? "rope(rows)" : "rope(rows,any)";
    return YSCV_CUDA_OK;
}
