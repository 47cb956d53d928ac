// Attention of ragged rows over a paged 8-bit cache, for the single tokens and short drafts of a decode step.
//
// With q = a_q n_q (n_q whole numbers of 24 bits, a row's largest at 8355711), k = s_k n_k and v = s_v n_v as the cache holds them,
//   scores   q k = a_q s_k sum n_q n_k          n_q = 65536 q2 + 256 q1 + q0, digits in [-128, 127]
//   output   p v = (2^T / 2^23) sum n_p n_v     n_p = p s_v 2^-T 2^23 of the softmax weights p of a step, bytes p2 p1 p0
// so both contractions are integer tensor-core products (mma.sync m16n8k32, int32 sums, exact) on the cache's bytes as they lie:
// nothing is converted or transposed. Against two fp16 terms per operand, which the framework's other int8 cache takes, that is
// three or two products for two and no conversion of the cache, which there is most of what the kernel issues. What is rounded: the
// query to 2^-23 of its row's largest, a weight to 2^-23 of its row's and step's largest weight times scale, and fp32 sums over steps.
// T is a row's own: with one for a step's largest scale a row that sees, or weighs, only pages whose values are 2^12 times smaller kept 12
// bits.
//
// Work: a step is 64 keys of a (sequence, KV head, block of R (position, head) pairs). All steps of a call are laid end to
// end, sequence after sequence, and every warp of the GPU takes an equal run of them, so that neither one long conversation nor
// many short ones leave SMs idle, whatever the lengths, which only the device knows. A warp is alone: it fetches its own keys and
// values (bulk copies: the next step's keys under this one's softmax and values, its values under its scores), keeps its own running
// maximum, sum and output, and writes a segment's result, or, where the segment goes on in another warp, a record that
// kv_attention_merge_kernel adds to the others. No barrier joins warps.
//
// A step is a chain of some 1100 instructions, so what counts is how many warps an SM has, and their buffers: with two stages of both
// operands and six warps at D = 128 the chain's latencies showed (64 sequences of 1000 to 8000 keys, 64 / 8 heads of 128: 133 us, IPC
// 0.3 per scheduler); one place each for keys and values gives twelve: 114 us, 118 with the joining kernel. With both products taken out
// the kernel took 106: what bounds it is the fetching of 8 KB pieces from all over the pool, 5.6 TB/s with its beginning and end.
//
// R = 8: the 16 rows of a product hold two digits of eight pairs, two products per tile instead of three.
// Bound: the cache's bytes from HBM (594 MB there, 92 us at the copy rate).
#include <cfloat>

#include "attention_tc.cuh"
#include "kv_attention.cuh"
#include "tma.cuh"

namespace yscv {

constexpr int KA_STEP = 64;                   // keys of a step
constexpr float KA_Q = 8355711.0f;            // 127 * (65536 + 256 + 1)
constexpr float KA_P = 8387584.0f;            // 2^23 - 1024: T goes by a logarithm that is good to 2^-15
constexpr int KA_OCTAVES = 90;                // a step's scales count as powers of two down to 2^-90 of its largest, smaller ones by fewer bits
constexpr float KA_MAGIC = 12582912.0f;       // 1.5 * 2^23: a sum that starts at its bits is the float MAGIC + sum (|sum| < 2^22)
constexpr int KA_MAGIC_BITS = 0x4B400000;

template <int D, int R> struct KaGeom {
    // as many as registers (two rows a thread take about 200) and shared memory hold
    static constexpr int WARPS = D == 256 ? 6 : D == 128 ? (R == 8 ? 12 : 8) : R == 8 ? 16 : 12;
    static constexpr int TILE = KA_STEP * D;                          // keys, or values, of a step
    static constexpr int WARP_BYTES = 2 * TILE + 16;                  // and two barriers
    static constexpr int RECORD_ROW = D + 2;
};

// A sequence's part of a call
struct KaSeq {
    int start, rows, lo, steps, blocks;       // lo: first key that any row sees, at a step's border
};
__device__ __forceinline__ KaSeq ka_seq(const KvAttention &a, int start, int rows, int R) {
    KaSeq s;
    s.start = start;
    s.rows = rows;
    s.lo = a.window > 0 ? max(0, start + 1 - a.window) & ~(KA_STEP - 1) : 0;
    // (positions behind the table's end have no keys; a segment has a step at least)
    s.steps = s.rows > 0 ? max((min(start, a.room - s.rows) + s.rows - s.lo + KA_STEP - 1) / KA_STEP, 1) : 0;
    s.blocks = (int)(((long long)s.rows * a.group + R - 1) / R);
    return s;
}

// D = A B + C: C the sums so far, or, for the first product, MAGIC's bits
#define KA_MMA(name, type)                                                                                                              \
    __device__ __forceinline__ void name(int (&d)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1, bool first) {                   \
        if (first)                                                                                                                      \
            asm("mma.sync.aligned.m16n8k32.row.col.s32." type ".s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"    \
                : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])                                                                        \
                : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b0), "r"(b1), "r"(KA_MAGIC_BITS));                                    \
        else                                                                                                                            \
            asm("mma.sync.aligned.m16n8k32.row.col.s32." type ".s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"        \
                : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])                                                                        \
                : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b0), "r"(b1));                                                        \
    }
KA_MMA(ka_mma_s8, "s8")
KA_MMA(ka_mma_u8, "u8")
#undef KA_MMA
__device__ __forceinline__ void ka_ldmatrix(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// e of x = f 2^e, f in [1/2, 1) (zero and subnormal numbers: -126)
__device__ __forceinline__ int ka_exponent(float x) { return min((__float_as_int(x) >> 23) - 126, 126); }
__device__ __forceinline__ float ka_log2(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
// two sums that began at MAGIC's bits
__device__ __forceinline__ uint64_t ka_sum2(int a, int b) { return f2_add(f2(__int_as_float(a), __int_as_float(b)), f2(-KA_MAGIC, -KA_MAGIC)); }

// Steps in front of every sequence, into shared memory, by all threads; returns the steps of the call
__device__ __forceinline__ long long ka_plan(const KvAttention &a, int R, long long *cum, int2 *info, long long *sums, int threads) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.l.n_seq;
    const int per = (n + threads - 1) / threads, i0 = min(tid * per, n), i1 = min(i0 + per, n);
    long long mine = 0;
    for (int i = i0; i < i1; ++i) {
        const KvSeqRows v = kv_rows(a, i);
        if (blockIdx.x == 0) kv_rows_status(a, v);
        const KaSeq s = ka_seq(a, v.start, v.rows, R);
        info[i] = make_int2(v.start, v.rows);
        cum[i] = mine;
        mine += (long long)s.steps * s.blocks * a.l.n_kv;
    }
    long long x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) sums[warp] = x;
    __syncthreads();
    long long before = x - mine, total = 0;
    for (int w = 0; w < threads / 32; ++w) {
        if (w < warp) before += sums[w];
        total += sums[w];
    }
    for (int i = i0; i < i1; ++i) cum[i] += before;
    if (tid == 0) cum[n] = total;
    __syncthreads();
    return total;
}

// Where a warp is in the steps of the call
struct KaWalk {
    int seq, head, block, step;
    KaSeq s;
    __device__ void load(const KvAttention &a, const int2 *info, int R) { s = ka_seq(a, info[seq].x, info[seq].y, R); }
    __device__ void seek(const KvAttention &a, const long long *cum, const int2 *info, int R, long long u) {
        int lo = 0, hi = a.l.n_seq;
        while (hi - lo > 1) {
            const int m = (lo + hi) >> 1;
            if (cum[m] <= u) lo = m;
            else hi = m;
        }
        seq = lo;
        load(a, info, R);
        const long long r = u - cum[seq], segment = r / s.steps;
        step = (int)(r - segment * s.steps);
        head = (int)(segment / s.blocks);
        block = (int)(segment - (long long)head * s.blocks);
    }
    // the next step of the call (there is one)
    __device__ void next(const KvAttention &a, const int2 *info, int R) {
        if (++step < s.steps) return;
        step = 0;
        if (++block < s.blocks) return;
        block = 0;
        if (++head < a.l.n_kv) return;
        head = 0;
        do {
            ++seq;
            load(a, info, R);
        } while (s.rows == 0);
    }
};

template <int D, int R>
__global__ void __launch_bounds__(KaGeom<D, R>::WARPS * 32, 1) kv_attention_kernel(const __grid_constant__ KvAttention a) {
    using G = KaGeom<D, R>;
    constexpr int NR = R / 8, KS = D / 32, NT = D / 8, THREADS = G::WARPS * 32;
    constexpr int TERMS = R == 8 ? 2 : 3;     // products per tile and 32 of the contraction
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ long long sums[G::WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const uint32_t ks_at = smem_u32(smem) + warp * (2 * G::TILE), vs_at = ks_at + G::TILE;
    const uint32_t k_bar = smem_u32(smem) + G::WARPS * (2 * G::TILE) + warp * 16, v_bar = k_bar + 8;
    long long *cum = reinterpret_cast<long long *>(smem + G::WARPS * G::WARP_BYTES);
    int2 *info = reinterpret_cast<int2 *>(cum + a.l.n_seq + 1);
    if (lane == 0) {
        mbar_init(k_bar, 1);
        mbar_init(v_bar, 1);
        mbar_fence_init();
    }
    __syncwarp();
    pdl_wait();
    pdl_trigger();
    const long long total = ka_plan(a, R, cum, info, sums, THREADS);
    // consecutive runs lie on different SMs
    const long long w = (long long)warp * gridDim.x + blockIdx.x, warps = (long long)gridDim.x * G::WARPS;
    const long long share = (total + warps - 1) / warps;
    if (blockIdx.x == 0) {
        long long *plan = static_cast<long long *>(a.plan);      // [0] steps, [1] steps of a warp, [2 ..] steps in front of a sequence
        for (int i = tid; i <= a.l.n_seq; i += THREADS) plan[2 + i] = cum[i];
        if (tid == 0) { plan[0] = total; plan[1] = share; }
    }
    const long long u0 = w * share, u1 = min(total, u0 + share);
    if (u0 >= u1) return;
    const int n = (int)(u1 - u0);

    // ---- fetching: lane i < 4 looks after the step's i-th group of 16 keys ----
    KaWalk f;
    f.seek(a, cum, info, R, u0);
    int next_id = -1, ahead = 0;              // the page of this lane's group in the step that is fetched next; steps fetched
    auto groups_of = [&](const KaWalk &x) { return min(4, (x.s.start + x.s.rows - (x.s.lo + x.step * KA_STEP) + KV_GROUP - 1) / KV_GROUP); };
    auto page = [&]() {
        next_id = -1;
        if (lane < groups_of(f)) {
            const int at = (f.s.lo + f.step * KA_STEP + KV_GROUP * lane) >> a.l.page_shift;
            if (at < a.l.max_pages) next_id = a.l.table[(size_t)f.seq * a.l.max_pages + at];
            if (at >= a.l.max_pages) atomicExch(a.status, YSCV_DEV_POS_OVERFLOW);
            else if (next_id < 0 || next_id >= a.l.n_pages) { next_id = -1; atomicExch(a.status, YSCV_DEV_BAD_NUMBER); }
        }
    };
    const int piece = min(a.l.page, KA_STEP) / KV_GROUP;   // groups that lie together
    size_t from = 0;                          // the lane's bytes in the pool, keys and values alike, and how many it copies
    int bytes = 0, all_bytes = 0;
    float next_ks = 0.0f, next_vs = -1.0f;    // scales of the lane's group; values' -1: no such keys
    auto copy = [&](const int8_t *pool, uint32_t to, uint32_t bar) {
        if (lane == 0) mbar_expect_tx(bar, all_bytes);
        __syncwarp();
        if (bytes > 0) bulk_load(to + lane * (KV_GROUP * D), pool + from, bytes, bar);
    };
    auto fetch_keys = [&]() {
        const bool there = next_id >= 0;
        all_bytes = __popc(__ballot_sync(0xffffffffu, there)) * (KV_GROUP * D);
        bytes = 0;
        next_ks = 0.0f;
        next_vs = -1.0f;
        if (there) {
            const size_t s_at = (size_t)next_id * a.l.n_kv + f.head;
            next_ks = a.l.ks[s_at];
            next_vs = a.l.vs[s_at];
            from = kv_group_at(a.l, next_id, f.head, ((f.s.lo + f.step * KA_STEP + KV_GROUP * lane) & (a.l.page - 1)) / KV_GROUP);
            if (lane % piece == 0) bytes = min(piece, groups_of(f) - lane) * (KV_GROUP * D);
        }
        copy(a.l.k, ks_at, k_bar);
        if (++ahead < n) {
            f.next(a, info, R);
            page();
        }
    };
    page();
    fetch_keys();
    copy(a.l.v, vs_at, v_bar);

    KaWalk c;
    c.seek(a, cum, info, R, u0);
    uint32_t qa[KS][NR == 1 ? 6 : 12];        // the query's digits as operands
    float qs[NR], m[NR], l[NR];
    uint64_t o[NT][NR];                       // two columns each
    int lim[NR], low[NR];
    const int first = t < 2 ? 0 : 2;          // of its four tokens of a group, which two a thread has in the first tile
    const uint32_t sel0 = t < 2 ? 0x5410u : 0x1054u, sel1 = t < 2 ? 0x7632u : 0x3276u;
    // rows of ldmatrix: tokens 0,1,4,5,10,11,14,15 and 2,3,6,7,8,9,12,13 of a group: a thread then has tokens 4 t .. 4 t + 3, and the
    // eight rows of a tile touch all banks
    const int r8 = lane & 7, half = lane >> 4, tq = r8 >> 1;
    const int token = 4 * tq + ((tq >> 1) ^ half) * 2 + (r8 & 1);
    const uint32_t k_lane = ((lane >> 3) & 1) * 256 + token * 16;
    const uint32_t v_lane = ((lane >> 3) & 1) * (KV_GROUP * D) + ((lane >> 4) * 8 + r8) * 16;

    bool begin = true, alive = true;
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        const int key0 = c.s.lo + c.step * KA_STEP;
        if (begin) {
            begin = false;
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                const int pair = c.block * R + 8 * r + g, s = pair / a.group;
                const bool live = pair < c.s.rows * a.group;
                lim[r] = !live ? 0 : a.causal ? c.s.start + s + 1 : c.s.start + c.s.rows;
                low[r] = a.window > 0 ? c.s.start + s + 1 - a.window : 0;
                const float *src = a.q + (size_t)(a.offsets[c.seq] + (live ? s : 0)) * a.q_stride + (size_t)(c.head * a.group + (live ? pair - s * a.group : 0)) * D;
                // (read twice, from L1 the second time: kept in registers between the two it would be spilled)
                auto load = [&](int k, int h) {
                    const float *p = src + 32 * k + 16 * h + 4 * t;
                    if (!live) return make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    return a.wide ? *reinterpret_cast<const float4 *>(p) : make_float4(p[0], p[1], p[2], p[3]);
                };
                float most = 0.0f, bad = 0.0f;
#pragma unroll 4
                for (int k = 0; k < 2 * KS; ++k) {
                    const float4 y = load(k >> 1, k & 1);
                    most = fmaxf(fmaxf(most, fmaxf(fabsf(y.x), fabsf(y.y))), fmaxf(fabsf(y.z), fabsf(y.w)));
                    bad = fmaf(y.x, 0.0f, fmaf(y.y, 0.0f, fmaf(y.z, 0.0f, fmaf(y.w, 0.0f, bad))));
                }
#pragma unroll
                for (int d = 1; d < 4; d <<= 1) {
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
                    bad += __shfl_xor_sync(0xffffffffu, bad, d);
                }
                most = fminf(fmaxf(most, KV_LEAST), FLT_MAX);
                const float up = __fdiv_rn(KA_Q, most);
                qs[r] = __fdiv_rn(most, KA_Q) * a.scale + bad;   // (bad: 0, or NaN)
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    uint32_t dig[3][2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float4 y = load(k, h);
                        const float x[4] = {y.x, y.y, y.z, y.w};
                        dig[0][h] = dig[1][h] = dig[2][h] = 0u;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int v = __float2int_rn(fminf(fmaxf(x[j] * up, -KA_Q), KA_Q));
                            const int d0 = (int)(int8_t)v, v1 = (v - d0) >> 8, d1 = (int)(int8_t)v1, d2 = (v1 - d1) >> 8;
                            dig[0][h] |= (uint32_t)(d0 & 255) << (8 * j);
                            dig[1][h] |= (uint32_t)(d1 & 255) << (8 * j);
                            dig[2][h] |= (uint32_t)(d2 & 255) << (8 * j);
                        }
                    }
                    if constexpr (NR == 1) {   // {q2, q1} in one operand, {q0, 0} in the other
                        qa[k][0] = dig[2][0]; qa[k][1] = dig[1][0]; qa[k][2] = dig[2][1]; qa[k][3] = dig[1][1];
                        qa[k][4] = dig[0][0]; qa[k][5] = dig[0][1];
                    } else {
#pragma unroll
                        for (int d = 0; d < 3; ++d) { qa[k][4 * d + r] = dig[2 - d][0]; qa[k][4 * d + 2 + r] = dig[2 - d][1]; }
                    }
                }
                m[r] = -INFINITY;
                l[r] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int r = 0; r < NR; ++r) o[j][r] = 0ull;
        }
        float kscale[4], vscale[4];
#pragma unroll
        for (int grp = 0; grp < 4; ++grp) {
            kscale[grp] = __shfl_sync(0xffffffffu, next_ks, grp);
            vscale[grp] = __shfl_sync(0xffffffffu, next_vs, grp);
        }
        alive = __all_sync(0xffffffffu, mbar_wait(k_bar, (uint32_t)i & 1u, a.status));
        if (!alive) break;
        // ---- scores ----
        float s[NR][16];                       // [row][4 group + token of the thread], tile order
#pragma unroll
        for (int grp = 0; grp < 4; ++grp) {
            int acc[2][TERMS][4];
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t b[4];
                ka_ldmatrix(b, ks_at + grp * (KV_GROUP * D) + k * 512 + k_lane);
#pragma unroll
                for (int tile = 0; tile < 2; ++tile) {
                    if constexpr (NR == 1) {
                        const uint32_t x1[4] = {qa[k][0], qa[k][1], qa[k][2], qa[k][3]}, x0[4] = {qa[k][4], 0u, qa[k][5], 0u};
                        ka_mma_s8(acc[tile][0], x1, b[2 * tile], b[2 * tile + 1], k == 0);
                        ka_mma_s8(acc[tile][1], x0, b[2 * tile], b[2 * tile + 1], k == 0);
                    } else {
#pragma unroll
                        for (int d = 0; d < 3; ++d) {
                            const uint32_t x[4] = {qa[k][4 * d], qa[k][4 * d + 1], qa[k][4 * d + 2], qa[k][4 * d + 3]};
                            ka_mma_s8(acc[tile][d], x, b[2 * tile], b[2 * tile + 1], k == 0);
                        }
                    }
                }
            }
#pragma unroll
            for (int tile = 0; tile < 2; ++tile)
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    const int *m1 = NR == 1 ? acc[tile][0] + 2 : acc[tile][1] + 2 * r, *m0 = acc[tile][TERMS - 1] + 2 * r, *m2 = acc[tile][0] + 2 * r;
                    const float f = qs[r] * kscale[grp];
                    const uint64_t x = f2_fma(ka_sum2(m2[0], m2[1]), f2(65536.0f, 65536.0f), f2_fma(ka_sum2(m1[0], m1[1]), f2(256.0f, 256.0f), ka_sum2(m0[0], m0[1])));
                    f2_get(f2_mul(x, f2(f, f)), s[r][4 * grp + 2 * tile], s[r][4 * grp + 2 * tile + 1]);
                }
        }
        __syncwarp();                          // every lane is done with the keys
        if (i + 1 < n) fetch_keys();
        bool edge = vscale[0] < 0.0f || vscale[1] < 0.0f || vscale[2] < 0.0f || vscale[3] < 0.0f;
#pragma unroll
        for (int r = 0; r < NR; ++r) edge |= key0 + KA_STEP > lim[r] || key0 < low[r];
        if (__any_sync(0xffffffffu, edge)) {
#pragma unroll
            for (int grp = 0; grp < 4; ++grp)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int key = key0 + 16 * grp + 4 * t + ((j & 2) ^ first) + (j & 1);
#pragma unroll
                    for (int r = 0; r < NR; ++r)
                        if (key >= lim[r] || key < low[r] || vscale[grp] < 0.0f) s[r][4 * grp + j] = -INFINITY;
                }
        }
        // ---- weights, relative to the step's own maximum ----
        // A value scale is f 2^e: a weight takes both, the sum takes e back. f is in [1/2, 1), or smaller where KA_OCTAVES holds e up
        float ve[4], vc[4], vl[4], back[4];
        const float vmost = fmaxf(fmaxf(vscale[0], vscale[1]), fmaxf(vscale[2], vscale[3]));
        const int e_least = max(ka_exponent(fmaxf(vmost, 0.0f)) - KA_OCTAVES, -126);
#pragma unroll
        for (int grp = 0; grp < 4; ++grp) {
            const float vs = fmaxf(vscale[grp], 0.0f);
            const int e = max(ka_exponent(vs), e_least);
            back[grp] = __int_as_float((127 - e) << 23);
            ve[grp] = (float)e;
            vc[grp] = fminf(vs * back[grp], 1.0f) * KA_P;
            vl[grp] = fmaxf(ka_log2(vs), ve[grp] - 1.0f);
        }
        uint32_t pa[4][NR][3];                 // [group][row][digit, the highest first]
        float w0[NR], alpha[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            float most[4];
#pragma unroll
            for (int grp = 0; grp < 4; ++grp) most[grp] = fmaxf(fmaxf(s[r][4 * grp], s[r][4 * grp + 1]), fmaxf(s[r][4 * grp + 2], s[r][4 * grp + 3]));
            float mx = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float ref = mx == -INFINITY ? 0.0f : mx, m_new = fmaxf(m[r], mx);
            // 2^T: the row's largest weight times scale, or up to twice that
            float T = fmaxf(fmaxf(most[0] - ref + vl[0], most[1] - ref + vl[1]), fmaxf(most[2] - ref + vl[2], most[3] - ref + vl[3]));
            T = fmaxf(T, __shfl_xor_sync(0xffffffffu, T, 1));
            T = fmaxf(T, __shfl_xor_sync(0xffffffffu, T, 2));
            T = fminf(fmaxf(ceilf(T), -126.0f), 126.0f);
            const float two_T = __int_as_float(((int)T + 127) << 23);
            float sum = 0.0f;
#pragma unroll
            for (int grp = 0; grp < 4; ++grp) {
                const uint64_t by_e = f2(ve[grp] - T, ve[grp] - T), by_ref = f2(-ref, -ref);
                uint32_t x[4];
                float p[4];
#pragma unroll
                for (int j = 0; j < 4; j += 2) {
                    // (the difference of the scores first: it is exact where it counts, whatever their size)
                    f2_get(f2_add(f2_add(f2(s[r][4 * grp + j], s[r][4 * grp + j + 1]), by_ref), by_e), p[j], p[j + 1]);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    p[j] = at_exp2(p[j]);
                    x[j] = __float_as_uint(fmaf(p[j], vc[grp], 8388608.0f));   // 2^23 + n_p: the low bytes are the digits
                }
                sum = fmaf((p[0] + p[1]) + (p[2] + p[3]), two_T * back[grp], sum);
                const uint32_t y = __byte_perm(x[0], x[1], 0x5140), z = __byte_perm(x[2], x[3], 0x5140);
                pa[grp][r][2] = __byte_perm(y, z, sel0);
                pa[grp][r][1] = __byte_perm(y, z, sel1);
                pa[grp][r][0] = __byte_perm(__byte_perm(x[0], x[1], 0x0062), __byte_perm(x[2], x[3], 0x0062), sel0);
            }
            alpha[r] = m_new == -INFINITY ? 1.0f : at_exp2(m[r] - m_new);
            const float beta = m_new == -INFINITY ? 0.0f : at_exp2(mx - m_new);
            l[r] = fmaf(l[r], alpha[r], beta * sum);
            m[r] = m_new;
            w0[r] = beta * two_T * (1.0f / KA_P);
        }
        // ---- weighted values ----
        alive = __all_sync(0xffffffffu, mbar_wait(v_bar, (uint32_t)i & 1u, a.status));
        if (!alive) break;
#pragma unroll
        for (int j = 0; j < NT; j += 2) {
            int acc[2][TERMS][4];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                uint32_t b[4];
                ka_ldmatrix(b, vs_at + k * (2 * KV_GROUP * D) + j * 128 + v_lane);
#pragma unroll
                for (int tile = 0; tile < 2; ++tile) {
                    if constexpr (NR == 1) {
                        const uint32_t x1[4] = {pa[2 * k][0][0], pa[2 * k][0][1], pa[2 * k + 1][0][0], pa[2 * k + 1][0][1]};
                        const uint32_t x0[4] = {pa[2 * k][0][2], 0u, pa[2 * k + 1][0][2], 0u};
                        ka_mma_u8(acc[tile][0], x1, b[2 * tile], b[2 * tile + 1], k == 0);
                        ka_mma_u8(acc[tile][1], x0, b[2 * tile], b[2 * tile + 1], k == 0);
                    } else {
#pragma unroll
                        for (int d = 0; d < 3; ++d) {
                            const uint32_t x[4] = {pa[2 * k][0][d], pa[2 * k][NR - 1][d], pa[2 * k + 1][0][d], pa[2 * k + 1][NR - 1][d]};
                            ka_mma_u8(acc[tile][d], x, b[2 * tile], b[2 * tile + 1], k == 0);
                        }
                    }
                }
            }
#pragma unroll
            for (int tile = 0; tile < 2; ++tile)
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    const int *m1 = NR == 1 ? acc[tile][0] + 2 : acc[tile][1] + 2 * r, *m0 = acc[tile][TERMS - 1] + 2 * r, *m2 = acc[tile][0] + 2 * r;
                    uint64_t &x = o[j + tile][r];
                    x = f2_fma(ka_sum2(m2[0], m2[1]), f2(w0[r] * 65536.0f, w0[r] * 65536.0f),
                               f2_fma(ka_sum2(m1[0], m1[1]), f2(w0[r] * 256.0f, w0[r] * 256.0f),
                                      f2_fma(ka_sum2(m0[0], m0[1]), f2(w0[r], w0[r]), f2_mul(x, f2(alpha[r], alpha[r])))));
                }
        }
        __syncwarp();
        if (i + 1 < n) copy(a.l.v, vs_at, v_bar);
        // ---- the end of a segment, or of this warp's part of it ----
        const bool last = c.step + 1 == c.s.steps;
        if (last || i + 1 == n) {
            const bool whole = last && i >= c.step;   // began here too
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
                l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
                const int pair = c.block * R + 8 * r + g, sq = pair / a.group;
                if (whole) {
                    if (pair < c.s.rows * a.group) {
                        const float inv = l[r] == 0.0f ? 0.0f : 1.0f / l[r];
                        float *dst = a.out + (size_t)(a.offsets[c.seq] + sq) * a.out_stride + (size_t)(c.head * a.group + pair - sq * a.group) * D + 2 * t;
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            float2 y;
                            f2_get(f2_mul(o[j][r], f2(inv, inv)), y.x, y.y);
                            if (a.wide) {
                                *reinterpret_cast<float2 *>(dst + 8 * j) = y;
                            } else {
                                dst[8 * j] = y.x;
                                dst[8 * j + 1] = y.y;
                            }
                        }
                    }
                } else {
                    // slot 2 w: the segment began in an earlier warp, 2 w + 1: here
                    float *rec = a.records + ((size_t)(2 * w + (i >= c.step)) * R + 8 * r + g) * G::RECORD_ROW;
#pragma unroll
                    for (int j = 0; j < NT; ++j) *reinterpret_cast<uint64_t *>(rec + 8 * j + 2 * t) = o[j][r];
                    if (t == 0) *reinterpret_cast<float2 *>(rec + D) = make_float2(m[r], l[r]);
                }
            }
            begin = true;
        }
        if (i + 1 < n) c.next(a, info, R);
    }
    if (!alive) {   // no copy may be in flight when the CTA leaves (bounded)
        mbar_wait(k_bar, (uint32_t)(ahead - 1) & 1u, nullptr);
        mbar_wait(v_bar, (uint32_t)(ahead - 1) & 1u, nullptr);
        mbar_wait(v_bar, (uint32_t)ahead & 1u, nullptr);
    }
}

// Adds the records of a segment that several warps shared: for each (sequence, KV head) W warps a pair, P pairs a CTA. Either one warp a
// pair, or, where there are fewer (sequence, head, pair)s than four an SM, sixteen, a share of the records each (one sequence of
// 131000 keys, 64 / 8 heads: 8 warps 69.7 us for both kernels, 16 65.9, 32 64.5, but 10.1 us for one of 200 keys where 16 take 9.6).
// 64 sequences, four warps a pair for all: 122 us, one warp 117.5. A table of 2048 positions has 33 records at most, which a warp adds by
// itself (one sequence of 200 keys: 9.3 us, 9.5 with sixteen).
template <int D, int R, int W, int P>
__global__ void __launch_bounds__(32 * W * P) kv_attention_merge_kernel(const __grid_constant__ KvAttention a) {
    static_assert(W == 1 || P == 1, "the shares of a pair are added by its whole CTA");
    pdl_wait();
    pdl_trigger();
    constexpr int ROW = D + 2, C = D / 64, FIRST = 4;   // pairs of columns of a lane: 2 lane + 64 e
    __shared__ __align__(8) float part[W][D];
    __shared__ float red[W][2];
    const int tid = threadIdx.x, lane = tid & 31, warp = W == 1 ? 0 : tid >> 5, seq = blockIdx.x, head = blockIdx.y;
    const long long share = static_cast<const long long *>(a.plan)[1], base = static_cast<const long long *>(a.plan)[2 + seq];
    const KvSeqRows v = kv_rows(a, seq);
    const int row0 = v.row0;
    const KaSeq s = ka_seq(a, v.start, v.rows, R);
    if (s.steps == 0) return;
    for (int pair = blockIdx.z * P + (W == 1 ? tid >> 5 : 0); pair < s.rows * a.group; pair += gridDim.z * P) {
        const int block = pair / R, r = pair - block * R;
        const long long from = base + ((long long)head * s.blocks + block) * s.steps, to = from + s.steps;
        const long long wa = from / share, wb = (to - 1) / share;
        if (wa == wb) continue;                  // one warp had it all and wrote it
        const int parts = (int)(wb - wa) + 1;
        auto record = [&](int p) { return a.records + ((size_t)(2 * (wa + p) + (p == 0)) * R + r) * ROW; };
        // every warp its records, 32 at a time, by its own maximum; the first ones are fetched beside their maxima and sums
        float m = -INFINITY, l = 0.0f;
        uint64_t acc[C] = {}, x[FIRST][C];
        for (int p0 = warp; p0 < parts; p0 += 32 * W) {
            const int mine = p0 + W * lane, np = min(32, (parts - p0 + W - 1) / W);
            float2 ml = make_float2(-INFINITY, 0.0f);
            if (mine < parts) ml = *reinterpret_cast<const float2 *>(record(mine) + D);
            auto fetch = [&](int p, uint64_t (&y)[C]) {
                const float *rec = record(p0 + W * min(p, np - 1)) + 2 * lane;
#pragma unroll
                for (int e = 0; e < C; ++e) y[e] = *reinterpret_cast<const uint64_t *>(rec + 64 * e);
            };
#pragma unroll
            for (int p = 0; p < FIRST; ++p) fetch(p, x[p]);
            float mx = ml.x;
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            const float m_new = fmaxf(m, mx), ref = m_new == -INFINITY ? 0.0f : m_new;
            const float old = at_exp2(m - ref), w = at_exp2(ml.x - ref);   // (0 for a lane without a record)
            m = m_new;
            l = fmaf(l, old, w * ml.y);          // (of the lane's records)
#pragma unroll
            for (int e = 0; e < C; ++e) acc[e] = f2_mul(acc[e], f2(old, old));
            for (int p = 0; p < np; p += FIRST) {
#pragma unroll
                for (int q = 0; q < FIRST; ++q) {
                    const float y = __shfl_sync(0xffffffffu, w, min(p + q, 31));
                    if (p + q < np)
#pragma unroll
                        for (int e = 0; e < C; ++e) acc[e] = f2_fma(f2(y, y), x[q][e], acc[e]);
                }
                if (p + FIRST < np)
#pragma unroll
                    for (int q = 0; q < FIRST; ++q) fetch(p + FIRST + q, x[q]);
            }
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
        const int sq = pair / a.group;
        float *dst = a.out + (size_t)(row0 + sq) * a.out_stride + (size_t)(head * a.group + pair - sq * a.group) * D;
        if (W == 1) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
            for (int e = 0; e < C; ++e) {
                float2 y;
                f2_get(f2_mul(acc[e], f2(inv, inv)), y.x, y.y);
                dst[2 * lane + 64 * e] = y.x;
                dst[2 * lane + 64 * e + 1] = y.y;
            }
            continue;
        }
#pragma unroll
        for (int e = 0; e < C; ++e) *reinterpret_cast<uint64_t *>(&part[warp][2 * lane + 64 * e]) = acc[e];
        if (lane == 0) { red[warp][0] = m; red[warp][1] = l; }
        __syncthreads();
        float all = red[0][0];
#pragma unroll
        for (int i = 1; i < W; ++i) all = fmaxf(all, red[i][0]);
        const float ref = all == -INFINITY ? 0.0f : all;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < W; ++i) sum = fmaf(at_exp2(red[i][0] - ref), red[i][1], sum);
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        for (int c = tid; c < D; c += 32 * W) {
            float y = 0.0f;
#pragma unroll
            for (int i = 0; i < W; ++i) y = fmaf(at_exp2(red[i][0] - ref), part[i][c], y);
            dst[c] = y * inv;
        }
        __syncthreads();
    }
}

// ---- host -----------------------------------------------------------------------------------------
static int ka_rows(size_t d, size_t pairs) { return d == 256 || pairs <= 8 ? 8 : 16; }

// warps of a CTA, and bytes of one's buffers
static void ka_geometry(size_t d, int R, size_t &warps, size_t &bytes) {
    auto of = [&](auto g) { warps = decltype(g)::WARPS; bytes = decltype(g)::WARP_BYTES; };
    if (d == 64) R == 8 ? of(KaGeom<64, 8>()) : of(KaGeom<64, 16>());
    else if (d == 128) R == 8 ? of(KaGeom<128, 8>()) : of(KaGeom<128, 16>());
    else of(KaGeom<256, 8>());
}
static size_t ka_smem(size_t d, int R, size_t n_seq) {
    size_t warps, bytes;
    ka_geometry(d, R, warps, bytes);
    return warps * bytes + (n_seq + 1) * sizeof(long long) + n_seq * sizeof(int2);
}
static size_t ka_plan_bytes(size_t n_seq) { return (2 + n_seq + 1) * sizeof(long long) + 15 & ~(size_t)15; }
static size_t ka_bytes(const yscv_cuda_ctx *ctx, size_t d, size_t n_seq, int R) {
    size_t warps, bytes;
    ka_geometry(d, R, warps, bytes);
    warps *= ctx->sm_count;
    return ka_plan_bytes(n_seq) + 2 * warps * R * (d + 2) * sizeof(float);
}

template <int D, int R> static int ka_launch(yscv_cuda_ctx *ctx, const KvAttention &a, size_t pairs) {
    auto kern = kv_attention_kernel<D, R>;
    if (const int rc = ensure_dynamic_smem(reinterpret_cast<const void *>(kern), ctx->device, 226 * 1024)) return rc;
    YSCV_CUDA_TRY(launch_pdl(kern, dim3((unsigned)ctx->sm_count), dim3(KaGeom<D, R>::WARPS * 32), ka_smem(D, R, a.l.n_seq), ctx->stream, a));
    ctx->launches++;
    const size_t z = pairs < 1024 ? pairs : 1024;
    const bool few = (size_t)a.l.n_seq * a.l.n_kv * z < (size_t)4 * ctx->sm_count && a.room > 32 * KA_STEP;
    YSCV_CUDA_TRY(launch_pdl(few ? kv_attention_merge_kernel<D, R, 16, 1> : kv_attention_merge_kernel<D, R, 1, 8>,
                             dim3((unsigned)a.l.n_seq, (unsigned)a.l.n_kv, (unsigned)(few ? z : (z + 7) / 8)), dim3(few ? 512 : 256), 0, ctx->stream, a));
    ctx->launches++;
    YSCV_CUDA_TRY(cudaGetLastError());
    ctx->last_kernel = "kv_block_attention(steps,imma)";
    return YSCV_CUDA_OK;
}

// What any kernel needs that a call of so many rows, or of fewer, can run: who has sized a workspace for prompts decodes with it
static size_t attention_bytes(const yscv_cuda_ctx *ctx, const yscv_cuda_kv_pool *pool, size_t group, size_t most_rows) {
    size_t bytes = std::max(ka_bytes(ctx, pool->d_head, pool->n_seq, 8), ka_bytes(ctx, pool->d_head, pool->n_seq, ka_rows(pool->d_head, most_rows * group)));
    if (kv_prompt_takes(pool, group, 0, most_rows)) bytes = std::max(bytes, kv_prompt_bytes(ctx, pool->d_head));
    return bytes;
}

// A guess of no rows may be wrong: what a call launches and what it needs both go by one row at least
static size_t ka_guess(size_t most_rows) { return most_rows > 0 ? most_rows : 1; }

static int ka_check(yscv_cuda_ctx *ctx, const yscv_cuda_kv_pool *pool, size_t n_q, size_t rows, size_t most_rows) {
    if (!ctx) return fail(YSCV_CUDA_ERR_BAD_ARG, "ctx is null");
    if (const int rc = kv_check_pool(pool)) return rc;
    if (pool->d_head != 64 && pool->d_head != 128 && pool->d_head != 256)
        return fail(YSCV_CUDA_ERR_UNSUPPORTED, "attention takes heads of 64, 128 or 256, got %zu", pool->d_head);
    if (n_q == 0 || n_q % pool->n_kv != 0) return fail(YSCV_CUDA_ERR_BAD_ARG, "n_q=%zu must be a positive multiple of n_kv=%zu", n_q, pool->n_kv);
    if (n_q > 65535 || rows * n_q >= (1u << 31) || most_rows * n_q >= (1u << 31)) return fail(YSCV_CUDA_ERR_UNSUPPORTED, "too many rows or heads");
    if (ka_smem(pool->d_head, 8, pool->n_seq) > 226 * 1024 || ka_smem(pool->d_head, 16, pool->n_seq) > 226 * 1024)
        return fail(YSCV_CUDA_ERR_UNSUPPORTED, "attention takes pools of up to %zu sequences at this head size",
                    (226 * 1024 - std::max(ka_smem(pool->d_head, 8, 0), ka_smem(pool->d_head, 16, 0))) / (sizeof(long long) + sizeof(int2)));
    return YSCV_CUDA_OK;
}

}  // namespace yscv

using namespace yscv;

extern "C" {

int yscv_cuda_kv_block_attention_workspace(yscv_cuda_ctx *ctx, const yscv_cuda_kv_pool *pool, size_t n_q, size_t rows, size_t most_rows,
                                           size_t *bytes) {
    if (const int rc = ka_check(ctx, pool, n_q, rows, most_rows)) return rc;
    if (!bytes) return fail(YSCV_CUDA_ERR_BAD_ARG, "bytes is null");
    *bytes = attention_bytes(ctx, pool, n_q / pool->n_kv, ka_guess(most_rows));
    return YSCV_CUDA_OK;
}

int yscv_cuda_kv_block_attention_dev(yscv_cuda_ctx *ctx, const yscv_cuda_kv_pool *pool, size_t layer, const float *d_q, size_t q_stride,
                                     size_t n_q, const int32_t *d_offsets, const int32_t *d_start, size_t rows, size_t most_rows, int causal,
                                     size_t window, float scale, float *d_out, size_t out_stride, void *d_workspace, size_t workspace_bytes) {
    if (const int rc = ka_check(ctx, pool, n_q, rows, most_rows)) return rc;
    KvAttention a = {};
    if (const int rc = kv_layer_of(pool, layer, &a.l)) return rc;
    if (!d_q || !d_offsets || !d_start || !d_out || !d_workspace) return fail(YSCV_CUDA_ERR_BAD_ARG, "null operand");
    if (!kv_aligned({d_q, d_offsets, d_start, d_out})) return fail(YSCV_CUDA_ERR_UNSUPPORTED, "operands must be 4-byte aligned");
    if (q_stride < n_q * pool->d_head || out_stride < n_q * pool->d_head)
        return fail(YSCV_CUDA_ERR_BAD_ARG, "a row stride is shorter than n_q * d_head");
    if (d_q == d_out) return fail(YSCV_CUDA_ERR_BAD_ARG, "d_out is d_q");
    if (!(scale >= 0.0f && scale <= FLT_MAX)) return fail(YSCV_CUDA_ERR_BAD_ARG, "scale must be 0 (the default) or positive");
    if (reinterpret_cast<uintptr_t>(d_workspace) & 15) return fail(YSCV_CUDA_ERR_UNSUPPORTED, "the workspace must be 16-byte aligned");
    most_rows = ka_guess(most_rows);
    const size_t group = n_q / pool->n_kv, pairs = most_rows * group;
    const int R = ka_rows(pool->d_head, pairs);
    const size_t need = attention_bytes(ctx, pool, group, most_rows);
    if (workspace_bytes < need) return fail(YSCV_CUDA_ERR_BAD_ARG, "workspace of %zu bytes, %zu are needed", workspace_bytes, need);
    if (rows == 0) return YSCV_CUDA_OK;
    YSCV_CUDA_TRY(cudaSetDevice(ctx->device));
    a.q = d_q;
    a.out = d_out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.offsets = d_offsets;
    a.start = d_start;
    a.n_q = (int)n_q;
    a.group = (int)group;
    a.causal = causal != 0;
    a.window = (int)(window < (1u << 31) ? window : 0);   // (no position is farther than that)
    a.wide = ((reinterpret_cast<uintptr_t>(d_q) | reinterpret_cast<uintptr_t>(d_out)) & 15) == 0 && q_stride % 4 == 0 && out_stride % 4 == 0;
    a.scale = (scale > 0.0f ? scale : 1.0f / sqrtf((float)pool->d_head)) * 1.4426950408889634f;
    a.rows = (int)rows;
    a.room = (int)(pool->max_pages * pool->page);
    a.plan = d_workspace;
    a.records = reinterpret_cast<float *>(static_cast<unsigned char *>(d_workspace) + ka_plan_bytes(pool->n_seq));
    a.status = ctx->d_status;
    if (kv_prompt_takes(pool, group, rows, most_rows)) return kv_prompt(ctx, a, d_workspace);
    switch (pool->d_head) {
        case 64: return R == 8 ? ka_launch<64, 8>(ctx, a, pairs) : ka_launch<64, 16>(ctx, a, pairs);
        case 128: return R == 8 ? ka_launch<128, 8>(ctx, a, pairs) : ka_launch<128, 16>(ctx, a, pairs);
        default: return ka_launch<256, 8>(ctx, a, pairs);
    }
}

}  // extern "C"
