// Attention of prompts, or of pieces of them, over a paged 8-bit cache on the 5th-generation tensor cores.
//
// An int8 number is exact in fp16, so the cache enters both products as one fp16 operand; queries (scaled by a power of two per
// row) and softmax weights (times 2^10) are two fp16 terms each, 22 bits: two products per contraction, where fp32 caches take
// three (gqa_prefill_tc.cu). Pages' scales are applied in fp32: the keys' to the scores as they are read, the values' as an offset in
// the weights' exponent. The tensor core adds into its accumulator by truncation, so no accumulator outlives 128 keys.
//
// A CTA works on tiles of 128 (position, query head) pairs of one KV head and 128 keys:
//   warp 0       TMEM; the products S = Q K^T and O = P V, both with the A operand in TMEM (from shared memory a product of 128 x 128
//                reads two operands and takes 125 cycles, with A in TMEM 70): S of the next tile runs under the softmax of this one
//   warp 1       queries of the next segment into shared memory, by bulk copies
//   warps 2, 3   keys and values of the tiles as they are cached, by bulk copies a tile ahead, and what the others have to know
//   warps 4-7    the tile's bytes as fp16 operands
//   warps 8-15   softmax, two threads a row: the queries' two terms to TMEM for a segment's first tile; scores from TMEM, the tile's own
//                maximum and sum, weights back to where the scores were. They keep nothing from tile to tile
//   warps 16-19  the output in registers, a thread per row: o = o 2^(M - M') + O 2^(m - M'), and results
// With the output in the softmax threads' registers those have too few left to keep several exponentials in flight: 2048 x 2048
// keys, 64 / 8 heads of 128, 507 us, a tile of 128 rows 6300 cycles.
// Registers are moved between the warpgroups: 640 threads x 96 = 128 x (56 + 72 + 96 + 96 + 160).
//
// Work: the tiles of all (sequence, pairs, KV head) segments are laid end to end, with room for KP_BEGIN tiles in front of each
// segment, about what its beginning and end take, and every SM takes an equal run; a segment that several SMs share leaves records, which
// kv_prompt_merge_kernel adds. So a short piece over a long cache fills the machine too, and causal prompts, whose first
// segments have one tile, need no order of CTAs (2047 tokens, 64 / 8 heads of 128: 456 us with tiles alone, 210 so; 276 with one, 212 with four).
// Bound: the tensor pipe, 2 x (128 D + 128 D) x 128 MACs a tile, 2048 cycles at the nominal rate for D = 128.
#include <cfloat>

#include "attention_tc.cuh"
#include "kv_attention.cuh"
#include "tma.cuh"

namespace yscv {

constexpr int KP_KEYS = 128, KP_ROWS = 128, KP_THREADS = 640, KP_NOTES = 8, KP_BEGIN = 2;

template <int D> struct KpGeom {
    static constexpr int OPERAND = KP_KEYS * D * 2, RAW = KP_KEYS * D;   // keys, or values, of a tile, in fp16 and as cached
    static constexpr int K_AT = 0, V_AT = 2 * OPERAND;         // two stages of keys, one of values
    static constexpr int RAW_K = 3 * OPERAND, RAW_V = RAW_K + RAW;
    static constexpr int Q_AT = RAW_V + RAW;                   // the next segment's queries, f32
    static constexpr int Q_PITCH = D * 4 + 16;
    static constexpr int OUT_AT = Q_AT + KP_ROWS * Q_PITCH;    // 4 KB a warp of the output
    static constexpr int STATS = OUT_AT + 16384;               // [2][2][128] {maximum, sum} of a tile's rows over 64 keys each
    static constexpr int NOTES = STATS + 4096;
    static constexpr int BARS = NOTES + KP_NOTES * 128;
    static constexpr int PLAN = BARS + 256;
    static constexpr int RECORD_ROW = D + 2;
};

__device__ __forceinline__ void kp_ld16(uint32_t taddr, float (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]),
          "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void kp_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};\n" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
        "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
// (what was loaded hangs on the wait)
__device__ __forceinline__ void kp_wait_ld16(float (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;\n"
                 : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]), "+f"(r[8]), "+f"(r[9]), "+f"(r[10]),
                   "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15])::"memory");
}

// Bounded waits without a status word (a role that gives up says so once, at the end): the kernel's loops have to fit the SM's
// instruction cache together
__device__ __forceinline__ bool kp_wait(uint32_t bar, uint32_t parity) {
#pragma unroll 1
    for (uint32_t i = 0; i < (1u << 22); ++i)
        if (mbar_try_wait(bar, parity)) return true;
    return false;
}
__device__ __forceinline__ bool kp_wait3(uint32_t b0, uint32_t p0, uint32_t b1, uint32_t p1, uint32_t b2, uint32_t p2) {
#pragma unroll 1
    for (uint32_t i = 0; i < (1u << 22); ++i) {
        const bool r0 = mbar_try_wait(b0, p0), r1 = mbar_try_wait(b1, p1), r2 = mbar_try_wait(b2, p2);
        if (r0 & r1 & r2) return true;
    }
    return false;
}

// at_desc() of a place in shared memory `bytes` behind the one of `low`, the lower half of its descriptor
__device__ __forceinline__ uint64_t kp_desc(uint32_t low, int bytes) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "r"(low + (uint32_t)(bytes >> 4)), "r"((1024u >> 4) | 1u << 14 | 2u << 29));
    return r;
}

// 16 int8 -> 16 fp16, exact: 0x6400 | (q ^ 0x80) is 1024 + q + 128
__device__ __forceinline__ void kp_convert(const uint4 &w, uint4 &lo, uint4 &hi) {
    const uint32_t in[4] = {w.x, w.y, w.z, w.w};
    uint32_t out[8];
    const __half2 bias = __floats2half2_rn(1152.0f, 1152.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t x = in[i] ^ 0x80808080u;
        uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
        const __half2 ha = __hsub2(*reinterpret_cast<__half2 *>(&a), bias), hb = __hsub2(*reinterpret_cast<__half2 *>(&b), bias);
        out[2 * i] = *reinterpret_cast<const uint32_t *>(&ha);
        out[2 * i + 1] = *reinterpret_cast<const uint32_t *>(&hb);
    }
    lo = make_uint4(out[0], out[1], out[2], out[3]);
    hi = make_uint4(out[4], out[5], out[6], out[7]);
}

// ---- where a call's tiles are -----------------------------------------------------------------------
// Pairs tile q of a sequence: positions q * QB .. ; the keys that any of them sees, from a group's border on
struct KpTile {
    int lo, hi, steps;
};
__device__ __forceinline__ KpTile kp_tile(const KvAttention &a, int start, int rows, int QB, int q) {
    const int s0 = q * QB, s1 = min(rows, s0 + QB);
    KpTile t;
    t.lo = a.window > 0 ? max(0, start + s0 + 1 - a.window) & ~(KV_GROUP - 1) : 0;
    t.hi = a.causal ? start + s1 : start + rows;
    t.steps = (t.hi - t.lo + KP_KEYS - 1) / KP_KEYS;
    return t;
}
__device__ __forceinline__ int kp_tiles(int start, int rows, int QB) { return start < 0 || rows <= 0 ? 0 : (rows + QB - 1) / QB; }
// Tiles of a sequence for one KV head, a warp together
__device__ __forceinline__ long long kp_steps(const KvAttention &a, int start, int rows, int QB) {
    long long n = 0;
    for (int q = threadIdx.x & 31; q < kp_tiles(start, rows, QB); q += 32) n += kp_tile(a, start, rows, QB, q).steps;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    return n;
}

struct KpWalk {
    int seq, q, head, step, start, rows, row0;
    KpTile t;
    __device__ void load(const KvAttention &a) {
        start = a.start[seq];
        row0 = a.offsets[seq];
        rows = a.offsets[seq + 1] - row0;
    }
    // The first tile at place u or behind it (u below the last place), a warp together. `at` [n_seq]: places in front of a sequence.
    // Returns the tiles of the sequence in front of it; `gap`: places between u and it.
    __device__ long long seek(const KvAttention &a, const long long *at, int QB, long long u, int &gap) {
        int lo = 0, hi = a.l.n_seq;
        while (hi - lo > 1) {
            const int m = (lo + hi) >> 1;
            if (at[m] <= u) lo = m;
            else hi = m;
        }
        seq = lo;
        load(a);
        long long left = u - at[seq], tiles = 0;
        const int lane = threadIdx.x & 31;
        for (int q0 = 0;; q0 += 32) {
            const int steps = q0 + lane < kp_tiles(start, rows, QB) ? kp_tile(a, start, rows, QB, q0 + lane).steps : 0;
            const int n = steps > 0 ? (steps + KP_BEGIN) * a.l.n_kv : 0;
            long long upto = n, tiles_upto = (long long)steps * a.l.n_kv;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long y = __shfl_up_sync(0xffffffffu, upto, o), z = __shfl_up_sync(0xffffffffu, tiles_upto, o);
                if (lane >= o) { upto += y; tiles_upto += z; }
            }
            const unsigned past = __ballot_sync(0xffffffffu, upto > left);
            if (past) {
                const int f = __ffs(past) - 1;
                left -= __shfl_sync(0xffffffffu, upto - n, f);
                tiles += __shfl_sync(0xffffffffu, tiles_upto - (long long)steps * a.l.n_kv, f);
                q = q0 + f;
                break;
            }
            left -= __shfl_sync(0xffffffffu, upto, 31);
            tiles += __shfl_sync(0xffffffffu, tiles_upto, 31);
        }
        t = kp_tile(a, start, rows, QB, q);
        head = (int)(left / (t.steps + KP_BEGIN));
        const int in = (int)(left - (long long)head * (t.steps + KP_BEGIN));
        gap = max(0, KP_BEGIN - in);
        step = max(0, in - KP_BEGIN);
        return tiles + (long long)head * t.steps + step;
    }
    // the first step of the next segment (there is one)
    __device__ void next_segment(const KvAttention &a, int QB) {
        step = 0;
        if (++head < a.l.n_kv) return;
        head = 0;
        if (++q >= kp_tiles(start, rows, QB)) {
            q = 0;
            do {
                ++seq;
                load(a);
            } while (kp_tiles(start, rows, QB) == 0);
        }
        t = kp_tile(a, start, rows, QB, q);
    }
    __device__ void next(const KvAttention &a, int QB) {
        if (++step == t.steps) next_segment(a, QB);
    }
};

// What warp 2 writes down about a tile for the others
struct KpNote {
    float ks[8], lv[8], iv[8];     // of its groups: keys' scale; values' scale over the largest one of the tile, log2 and inverse
    float vmost;                   // (a group that is not there: 1, -inf, 0)
    int key0, last, begins;        // first key; the segment's last tile (1), or only the run's (2); the first of either
    int start, rows, row0, first;  // the sequence: position of its first row, rows, number of the first; first row of the pairs tile
};
static_assert(sizeof(KpNote) == 128, "KP_NOTES of them lie in shared memory");

template <int D>
__global__ void __launch_bounds__(KP_THREADS, 1) kv_prompt_kernel(const __grid_constant__ KvAttention a) {
    using G = KpGeom<D>;
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ longlong2 sums[KP_THREADS / 32];
    __shared__ int run_tiles;
    __shared__ uint32_t tmem_slot;
    __shared__ int heads[KP_NOTES], begun[KP_NOTES];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t base = smem_u32(smem), bars = base + G::BARS;
    // [2] by tile & 1, each used again two tiles later; nfull [KP_NOTES]; from vfull on one phase a tile; from qstaged on one a segment
    const uint32_t kfull = bars, sfull = bars + 32, pfull = bars + 48, ofull = bars + 64, ofree = bars + 80;
    const uint32_t nfull = bars + 96, vfull = bars + 160, raw_k = bars + 176, raw_v = bars + 184, raw_k_free = bars + 192;
    const uint32_t raw_v_free = bars + 200, qstaged = bars + 208, qtaken = bars + 216, qfull = bars + 224, maxima = bars + 232;   // [2] by tile & 1
    float2 *stats = reinterpret_cast<float2 *>(smem + G::STATS);
    KpNote *notes = reinterpret_cast<KpNote *>(smem + G::NOTES);
    longlong2 *before = reinterpret_cast<longlong2 *>(smem + G::PLAN);     // [n_seq + 1] places, tiles
    long long *cum = reinterpret_cast<long long *>(before + a.l.n_seq + 1); // [n_seq + 1] places
    const int group = a.group, QB = KP_ROWS / group;

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(kfull + i * 8, 4);
            mbar_init(sfull + i * 8, 1);
            mbar_init(pfull + i * 8, 8);
            mbar_init(maxima + i * 8, 8);
            mbar_init(ofull + i * 8, 1);
            mbar_init(ofree + i * 8, 4);
        }
        for (int i = 0; i < KP_NOTES; ++i) mbar_init(nfull + i * 8, 1);
        mbar_init(vfull, 4);
        mbar_init(raw_k, 1);
        mbar_init(raw_v, 1);
        mbar_init(raw_k_free, 4);
        mbar_init(raw_v_free, 4);
        mbar_init(qstaged, 1);
        mbar_init(qtaken, 8);
        mbar_init(qfull, 8);
        mbar_fence_init();
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&tmem_slot)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
    }
    pdl_wait();
    pdl_trigger();
    // ---- places and tiles in front of every sequence, and which are this CTA's ----
    for (int i = warp; i < a.l.n_seq; i += KP_THREADS / 32) {
        const int row0 = a.offsets[i], rows = a.offsets[i + 1] - row0, start = a.start[i];
        const long long n = kp_steps(a, start, rows, QB);
        if (lane == 0) {
            before[i].y = n * a.l.n_kv;
            before[i].x = (n + (long long)KP_BEGIN * kp_tiles(start, rows, QB)) * a.l.n_kv;
        }
    }
    __syncthreads();
    {
        const int n = a.l.n_seq, per = (n + KP_THREADS - 1) / KP_THREADS, i0 = min(tid * per, n), i1 = min(i0 + per, n);
        longlong2 mine = make_longlong2(0, 0);
        for (int i = i0; i < i1; ++i) { mine.x += before[i].x; mine.y += before[i].y; }
        longlong2 x = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x.x, o), z = __shfl_up_sync(0xffffffffu, x.y, o);
            if (lane >= o) { x.x += y; x.y += z; }
        }
        if (lane == 31) sums[warp] = x;
        __syncthreads();
        longlong2 at = make_longlong2(x.x - mine.x, x.y - mine.y);
        for (int w = 0; w < warp; ++w) { at.x += sums[w].x; at.y += sums[w].y; }
        for (int i = i0; i < i1; ++i) {
            const longlong2 c = before[i];
            cum[i] = at.x;
            before[i] = at;
            at.x += c.x;
            at.y += c.y;
        }
        if (tid == KP_THREADS - 1) { cum[n] = at.x; before[n] = at; }
    }
    at_fence_before();
    __syncthreads();
    at_fence_after();
    const uint32_t tmem = tmem_slot;
    const long long total = before[a.l.n_seq].x, share = (total + gridDim.x - 1) / gridDim.x;
    if (blockIdx.x == 0) {
        for (int i = tid; i <= a.l.n_seq; i += KP_THREADS) a.plan[2 + i] = cum[i];
        if (tid == 0) { a.plan[0] = total; a.plan[1] = share; }
    }
    const long long u0 = min(total, blockIdx.x * share), u1 = min(total, u0 + share);
    if (warp == 0 && u0 < u1) {
        KpWalk w;
        int gap;
        const long long t0 = w.seek(a, cum, QB, u0, gap) + before[w.seq].y;
        const long long t1 = u1 < total ? w.seek(a, cum, QB, u1, gap) + before[w.seq].y : before[a.l.n_seq].y;
        if (lane == 0) run_tiles = (int)(t1 - t0);
    }
    if (tid == 0 && u0 >= u1) run_tiles = 0;
    __syncthreads();
    const int n = run_tiles;
    // TMEM columns: queries (both terms), scores and then weights [2] x 128, weighted values
    const uint32_t t_q = tmem, t_s = tmem + 128, t_o = tmem + 384;
    auto par = [](int i) { return (uint32_t)(i >> 1) & 1u; };
    bool alive = true;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;\n");
        if (warp == 0) {
            // ---- products, a thread: what it waits for is asked for at once, since a barrier that is ready takes 100 cycles to say so ----
            if (lane == 0 && n > 0) {
                const uint32_t id_s = (1u << 4) | ((uint32_t)(KP_KEYS >> 3) << 17) | ((uint32_t)(KP_ROWS >> 4) << 24);
                const uint32_t id_o = (1u << 4) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(KP_ROWS >> 4) << 24);
                const uint32_t at = (base >> 4) | 1u << 16;
                uint32_t segments = 0;
                auto scores = [&](int i, bool begins) {
                    const int st = i & 1;
                    if (begins && !kp_wait(qfull, segments++ & 1u)) return false;
                    // the weights of tile i - 2, which lie where these scores go, have been multiplied
                    if (i > 1 && !kp_wait(ofull + st * 8, par(i - 2))) return false;
                    at_fence_after();
                    const uint32_t k_at = at + (uint32_t)((G::K_AT + st * G::OPERAND) >> 4);
#pragma unroll 4
                    for (int e = 0; e < D / 8; ++e) {           // remainders first
                        const int kk = e & (D / 16 - 1), term = e < D / 16;
                        at_mma_ts(t_s + st * 128, t_q + (kk >> 1) * 32 + term * 16 + (kk & 1) * 8, kp_desc(k_at, (kk >> 2) * (KP_KEYS * 128) + (kk & 3) * 32),
                                  id_s, e > 0);
                    }
                    at_commit(sfull + st * 8);
                    return true;
                };
                auto values = [&](int i) {
                    const int st = i & 1;
                    if (!kp_wait3(vfull, (uint32_t)i & 1u, pfull + st * 8, par(i), i > 0 ? ofree + (st ^ 1) * 8 : vfull,
                                  i > 0 ? par(i - 1) : (uint32_t)i & 1u)) return false;
                    at_fence_after();
#pragma unroll 4
                    for (int e = 0; e < KP_KEYS / 8; ++e) {
                        const int kk = e & (KP_KEYS / 16 - 1), term = e < KP_KEYS / 16;
                        at_mma_ts(t_o, t_s + st * 128 + kk * 16 + term * 8, kp_desc(at, G::V_AT + (kk >> 2) * (D * 128) + (kk & 3) * 32), id_o, e > 0);
                    }
                    at_commit(ofull + st * 8);
                    return true;
                };
                alive = kp_wait(kfull, 0u) && scores(0, true);
#pragma unroll 1
                for (int i = 0; i < n && alive; ++i) {
                    // the next tile's scores first, unless its queries still have to take the place of this segment's
                    bool later = false;
                    if (i + 1 < n) {
                        alive = kp_wait(kfull + ((i + 1) & 1) * 8, par(i + 1));
                        if (!alive) break;
                        later = begun[(i + 1) % KP_NOTES] != 0;
                        if (!later) alive = scores(i + 1, false);
                    }
                    alive = alive && values(i);
                    if (later) alive = alive && scores(i + 1, true);
                }
            }
            __syncwarp();
        } else if (warp == 1 && n > 0) {
            // ---- queries of the next segment, as they are: a copy a row, 16 bytes apart so that threads can read a row each ----
            KpWalk w;
            int gap;
            w.seek(a, cum, QB, u0, gap);
            int i = 0, loaded = 1;
            for (int segment = 0;; ++segment) {
                if (segment > 0) alive = __all_sync(0xffffffffu, kp_wait(qtaken, (uint32_t)(segment - 1) & 1u));
                if (!alive) break;
                const int s0 = w.q * QB, live = min(QB, w.rows - s0) * group;
                const float *src = a.q + (size_t)(w.row0 + s0) * a.q_stride + (size_t)w.head * group * D;
                if (a.wide) {
                    if (lane == 0) mbar_expect_tx(qstaged, live * D * 4);
                    __syncwarp();
                    for (int r = lane; r < live; r += 32)
                        bulk_load(base + G::Q_AT + r * G::Q_PITCH, src + (size_t)(r / group) * a.q_stride + (size_t)(r % group) * D, D * 4, qstaged);
                } else {
                    for (int r = 0; r < live; ++r) {
                        const float *from = src + (size_t)(r / group) * a.q_stride + (size_t)(r % group) * D;
                        float *to = reinterpret_cast<float *>(smem + G::Q_AT + r * G::Q_PITCH);
#pragma unroll
                        for (int c = 0; c < D; c += 32) to[c + lane] = __ldg(from + c + lane);
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(qstaged);
                }
                i += w.t.steps - w.step;
                if (i >= n) break;
                w.next_segment(a, QB);
                loaded = segment + 2;
            }
            // no copy may be in flight when the CTA leaves (bounded)
            if (!alive) kp_wait(qstaged, (uint32_t)(loaded - 1) & 1u);
        } else if (warp > 1 && n > 0) {
            // ---- keys (warp 2) and values (warp 3) as they are cached, by bulk copies; what the others have to know about a tile.
            // Lane g < 8 looks after group g: its page, a tile ahead, and its scales ----
            const bool values = warp == 3;
            const int8_t *pool = values ? a.l.v : a.l.k;
            const uint32_t full = values ? raw_v : raw_k, free = values ? raw_v_free : raw_k_free;
            const uint32_t to = base + (values ? G::RAW_V : G::RAW_K) + lane * (KV_GROUP * D);
            KpWalk w;
            int gap;
            w.seek(a, cum, QB, u0, gap);
            const int piece = min(a.l.page / KV_GROUP, 8);        // groups that lie together, from a page's border on
            int id = -1;
            auto page = [&]() {
                const int key = w.t.lo + w.step * KP_KEYS + KV_GROUP * lane, at = key >> a.l.page_shift;
                id = -1;
                if (lane < 8 && key < w.t.hi) {
                    if (at < a.l.max_pages) id = __ldg(a.l.table + (size_t)w.seq * a.l.max_pages + at);
                    else atomicExch(a.status, YSCV_DEV_POS_OVERFLOW);
                }
            };
            bool begins = true;
            int copied = 0;                                       // tiles on their way or there
            page();
#pragma unroll 1
            for (int i = 0; i < n; ++i) {
                const int key0 = w.t.lo + w.step * KP_KEYS, key = key0 + KV_GROUP * lane;
                const bool wanted = lane < 8 && key < w.t.hi, there = wanted && id >= 0 && id < a.l.n_pages;
                if (wanted && !there && (key >> a.l.page_shift) < a.l.max_pages) atomicExch(a.status, YSCV_DEV_BAD_NUMBER);
                float ks = 1.0f, vs = -1.0f;
                if (!values && there) {
                    ks = __ldg(a.l.ks + (size_t)id * a.l.n_kv + w.head);
                    vs = __ldg(a.l.vs + (size_t)id * a.l.n_kv + w.head);
                }
                const int group_in = (key & (a.l.page - 1)) / KV_GROUP;
                const unsigned groups = __ballot_sync(0xffffffffu, there);
                if (i > 0) alive = __all_sync(0xffffffffu, kp_wait(free, (uint32_t)(i - 1) & 1u));
                if (!alive) break;
                if (lane == 0) {
                    if (!values) begun[i % KP_NOTES] = begins;    // (seen by whoever sees the keys)
                    mbar_expect_tx(full, __popc(groups) * (KV_GROUP * D));
                }
                __syncwarp();
                // the lane of a page's first group of the tile copies what the page has of it
                if (there && (lane == 0 || group_in == 0))
                    bulk_load(to, pool + kv_group_at(a.l, id, w.head, group_in), min(piece - group_in, __popc(groups >> lane)) * (KV_GROUP * D), full);
                copied = i + 1;
                if (!values) {
                    // (a row of notes is used again KP_NOTES tiles later, when every role has long been through)
                    KpNote &o = notes[i % KP_NOTES];
                    float vmost = vs;
#pragma unroll
                    for (int d = 4; d > 0; d >>= 1) vmost = fmaxf(vmost, __shfl_xor_sync(0xffffffffu, vmost, d));
                    if (lane < 8) {
                        o.ks[lane] = ks;
                        o.lv[lane] = there ? (vs == vmost ? 0.0f : log2f(__fdiv_rn(vs, vmost))) : -INFINITY;
                        o.iv[lane] = there ? __fdiv_rn(vmost, vs) : 0.0f;
                    }
                    if (lane == 0) {
                        o.vmost = vmost;
                        o.key0 = key0;
                        o.last = w.step + 1 == w.t.steps ? 1 : i + 1 == n ? 2 : 0;
                        o.begins = begins ? 1 + w.step : 0;
                        o.start = w.start; o.rows = w.rows; o.row0 = w.row0; o.first = w.q * QB;
                        heads[i % KP_NOTES] = w.head;
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(nfull + i % KP_NOTES * 8);
                }
                begins = w.step + 1 == w.t.steps;
                if (i + 1 < n) {
                    w.next(a, QB);
                    page();
                }
            }
            if (!alive && copied > 0) kp_wait(full, (uint32_t)(copied - 1) & 1u);
        }
    } else if (warp < 8) {
        // ---- the tile's bytes as fp16 operands ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;\n");
        // a group of 16 tokens is D pieces of 16 bytes, keys and values alike; PER groups for 128 threads at once
        constexpr int ITEMS = KP_KEYS * D / 16 / 128, PER = D == 64 ? 2 : 1;
        const int t = tid - 128, in = t % D, g0 = t / D;
        // (no load from memory may be on its way here: the fence in front of the tensor core would wait for it)
        // keys a tile ahead of the values, whose place is free only when the product in front has read it: K 0, K 1, V 0, K 2, V 1, ...
#pragma unroll 1
        for (int j = 0; j < 2 * n + 2; ++j) {
            const bool values = j & 1;
            const int i = (j >> 1) - values, st = i & 1;
            if (i < 0 || i >= n) continue;
            alive = kp_wait(values ? raw_v : raw_k, (uint32_t)i & 1u);
            // (keys: the scores of tile i - 2 are there; values: the weighted values of tile i - 1)
            if (i > 1 - values) alive = alive && kp_wait(values ? ofull + (st ^ 1) * 8 : sfull + st * 8, values ? par(i - 1) : par(i - 2));
            alive = __all_sync(0xffffffffu, alive);
            if (!alive) break;
            // keys: 16 d of a token are pieces 2 c and 2 c + 1 of its 128-byte row of the 64-d sub-tile. Values: 16 tokens of a row
            // are pieces 2 (g & 3) and the next of row d of the 64-key half
            const unsigned char *from = smem + (values ? G::RAW_V : G::RAW_K) + t * 16;
            unsigned char *to = smem + (values ? G::V_AT + in * 128
                                               : G::K_AT + st * G::OPERAND + (in >> 6) * (KP_KEYS * 128) + (g0 * KV_GROUP + (in & 15)) * 128);
#pragma unroll 2
            for (int e = 0; e < ITEMS; ++e) {
                const int g = e * PER + g0, piece = values ? g & 3 : (in >> 4) & 3;
                const int at0 = (values ? (g >> 2) * (D * 128) : e * (PER * KV_GROUP * 128)) + (((2 * piece) ^ (in & 7)) << 4);
                uint4 lo, hi;
                kp_convert(*reinterpret_cast<const uint4 *>(from + e * 2048), lo, hi);
                *reinterpret_cast<uint4 *>(to + at0) = lo;
                *reinterpret_cast<uint4 *>(to + (at0 ^ 16)) = hi;
            }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(values ? vfull : kfull + st * 8);
                mbar_arrive(values ? raw_v_free : raw_k_free);
            }
        }
    } else if (warp < 16) {
        // ---- softmax: a thread has 64 keys of a row, warps 8-11 the first of the tile, warps 12-15 the others ----
        const int half = warp >= 12, row = (warp & 3) * 32 + lane, in_tile = row / group;
        const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
        uint32_t segment = 0;
        float to_log2 = 0.0f;
        int lim = 0, low = 0;
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
            const int st = i & 1;
            const uint32_t s_at = t_s + st * 128 + half * 64 + lane_off;
            alive = __all_sync(0xffffffffu, kp_wait(nfull + i % KP_NOTES * 8, (uint32_t)(i / KP_NOTES) & 1u));
            if (!alive) break;
            const KpNote &note = notes[i % KP_NOTES];
            if (note.begins) {
                // the staged queries take the place of the last segment's, whose scores are done: half the columns each
                alive = __all_sync(0xffffffffu, kp_wait(qstaged, segment++ & 1u));
                if (!alive) break;
                at_fence_after();
                const int s_pos = note.first + in_tile;
                const bool there = row < QB * group && s_pos < note.rows;
                const float4 *q = reinterpret_cast<const float4 *>(smem + G::Q_AT + row * G::Q_PITCH);
                float most = 0.0f;
#pragma unroll 4
                for (int j = 0; j < D / 4; ++j) {
                    const float4 y = q[j];
                    most = fmaxf(fmaxf(most, fmaxf(fabsf(y.x), fabsf(y.y))), fmaxf(fabsf(y.z), fabsf(y.w)));
                }
                float up, down;
                at_scale(there ? most : 0.0f, up, down);
#pragma unroll 1
                for (int j0 = half * (D / 2); j0 < (half + 1) * (D / 2); j0 += 32) {
                    uint32_t x[32];               // 16 columns of leading terms, 16 of remainders
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        float4 y = q[j0 / 4 + j];
                        if (!there) y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        at_split(y.x * up, y.y * up, x[2 * j], x[16 + 2 * j]);
                        at_split(y.z * up, y.w * up, x[2 * j + 1], x[16 + 2 * j + 1]);
                    }
                    at_st32(t_q + lane_off + j0, x);
                }
                asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
                at_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(qfull);
                    mbar_arrive(qtaken);
                }
                to_log2 = down * a.scale;
                lim = !there ? 0 : a.causal ? note.start + s_pos + 1 : note.start + note.rows;
                low = a.window > 0 ? note.start + s_pos + 1 - a.window : 0;
            }
            const int key0 = note.key0 + half * 64, from = low - key0, to = lim - key0;     // the keys of its 64 that this row sees
            const float *ks = note.ks + half * 4, *lv = note.lv + half * 4, *iv = note.iv + half * 4;
            const float4 iv4 = *reinterpret_cast<const float4 *>(iv);
            const bool edge = __any_sync(0xffffffffu, to < 64 || from > 0 || iv4.x == 0.0f || iv4.y == 0.0f || iv4.z == 0.0f || iv4.w == 0.0f);
            alive = __all_sync(0xffffffffu, kp_wait(sfull + st * 8, par(i)));
            if (!alive) break;
            at_fence_after();
            // The loops are kept small: with every role's code laid out flat most of the time went to fetching instructions
            if (edge) {                        // keys that a row does not see
#pragma unroll 1
                for (int g = 0; g < 4; ++g) {
                    float v[16];
                    kp_ld16(s_at + 16 * g, v);
                    kp_wait_ld16(v);
                    const bool gone = iv[g] == 0.0f;
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (gone || 16 * g + e >= to || 16 * g + e < from) v[e] = -INFINITY;
                    kp_st16(s_at + 16 * g, reinterpret_cast<const uint32_t(&)[16]>(v));
                }
                asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
            }
            float mx = -INFINITY;
#pragma unroll 1
            for (int g = 0; g < 4; g += 2) {
                float v[16], u[16];
                kp_ld16(s_at + 16 * g, v);
                kp_ld16(s_at + 16 * g + 16, u);
                kp_wait_ld16(v);
                kp_wait_ld16(u);
                float x = fmaxf(v[0], v[1]), y = fmaxf(u[0], u[1]);
#pragma unroll
                for (int e = 2; e < 16; e += 2) {
                    x = fmaxf(x, fmaxf(v[e], v[e + 1]));
                    y = fmaxf(y, fmaxf(u[e], u[e + 1]));
                }
                mx = fmaxf(mx, fmaxf(x * (to_log2 * ks[g]), y * (to_log2 * ks[g + 1])));
            }
            // the row's maximum over both halves of the tile; what the output's warps were told last there they have read
            float2 *mine = stats + (st * 2 + half) * KP_ROWS + row, *other = stats + (st * 2 + (half ^ 1)) * KP_ROWS + row;
            if (i > 1) alive = __all_sync(0xffffffffu, kp_wait(ofree + st * 8, par(i - 2)));
            if (!alive) break;
            mine->x = mx;
            __syncwarp();
            if (lane == 0) mbar_arrive(maxima + st * 8);
            alive = __all_sync(0xffffffffu, kp_wait(maxima + st * 8, par(i)));
            if (!alive) break;
            mx = fmaxf(mx, other->x);
            const float off = mx == -INFINITY ? 0.0f : 10.0f - mx;
            float sum = 0.0f;
#pragma unroll 1
            for (int g = 0; g < 4; ++g) {
                float v[16];
                kp_ld16(s_at + 16 * g, v);
                const float c = to_log2 * ks[g], og = off + lv[g], inv = iv[g];
                const uint64_t c2 = f2(c, c), og2 = f2(og, og), minus = f2(-1.0f, -1.0f);
                kp_wait_ld16(v);
                uint32_t p[16];               // leading terms of 16 weights, remainders
                uint64_t s2 = 0ull;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float x, y;
                    f2_get(f2_fma(f2(v[2 * e], v[2 * e + 1]), c2, og2), x, y);
                    x = at_exp2(x);
                    y = at_exp2(y);
                    const uint64_t w2 = f2(x, y);
                    s2 = f2_add(s2, w2);
                    const __half2 hh = __floats2half2_rn(x, y);
                    const float2 back = __half22float2(hh);
                    f2_get(f2_fma(f2(back.x, back.y), minus, w2), x, y);
                    const __half2 ll = __floats2half2_rn(x, y);
                    p[e] = *reinterpret_cast<const uint32_t *>(&hh);
                    p[8 + e] = *reinterpret_cast<const uint32_t *>(&ll);
                }
                kp_st16(s_at + 16 * g, p);
                float x, y;
                f2_get(s2, x, y);
                sum = fmaf(x + y, inv, sum);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
            mine->y = sum;
            at_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(pfull + st * 8);
        }
    } else {
        // ---- output ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 160;\n");
        const int row = (warp & 3) * 32 + lane;
        const uint32_t o_at = t_o + ((uint32_t)((warp & 3) * 32) << 16);
        unsigned char *stage = smem + G::OUT_AT + (warp & 3) * 4096;
        uint64_t o[D / 2];
        float m = -INFINITY, l = 0.0f;
        bool here = false;                             // here: the segment began in this run
        for (int i = 0; i < n; ++i) {
            const int st = i & 1;
            alive = __all_sync(0xffffffffu, kp_wait(nfull + i % KP_NOTES * 8, (uint32_t)(i / KP_NOTES) & 1u) &&
                                                kp_wait(pfull + st * 8, par(i)));
            if (!alive) break;
            const KpNote &note = notes[i % KP_NOTES];
            const float2 ms0 = stats[st * 2 * KP_ROWS + row], ms1 = stats[(st * 2 + 1) * KP_ROWS + row];
            const float2 ms = make_float2(fmaxf(ms0.x, ms1.x), ms0.y + ms1.y);
            if (note.begins) {
                here = note.begins == 1;
                m = -INFINITY;
                l = 0.0f;
#pragma unroll
                for (int j = 0; j < D / 2; ++j) o[j] = 0ull;
            }
            const float m_new = fmaxf(m, ms.x);
            const float alpha = m_new == -INFINITY ? 1.0f : at_exp2(m - m_new), beta = m_new == -INFINITY ? 0.0f : at_exp2(ms.x - m_new);
            l = fmaf(l, alpha, beta * ms.y);
            m = m_new;
            const float b = beta * fmaxf(note.vmost, 0.0f);
            const uint64_t al2 = f2(alpha, alpha), b2 = f2(b, b);
            alive = __all_sync(0xffffffffu, kp_wait(ofull + st * 8, par(i)));
            if (!alive) break;
            at_fence_after();
            // (read as fast as it goes: the next product with weights waits for it)
            float t0[16], t1[16];
            kp_ld16(o_at, t0);
#pragma unroll
            for (int j0 = 0; j0 < D; j0 += 32) {
                kp_wait_ld16(t0);
                kp_ld16(o_at + j0 + 16, t1);
#pragma unroll
                for (int e = 0; e < 8; ++e) o[j0 / 2 + e] = f2_fma(o[j0 / 2 + e], al2, f2_mul(f2(t0[2 * e], t0[2 * e + 1]), b2));
                kp_wait_ld16(t1);
                if (j0 + 32 < D) kp_ld16(o_at + j0 + 32, t0);
#pragma unroll
                for (int e = 0; e < 8; ++e) o[j0 / 2 + 8 + e] = f2_fma(o[j0 / 2 + 8 + e], al2, f2_mul(f2(t1[2 * e], t1[2 * e + 1]), b2));
            }
            at_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(ofree + st * 8);
            if (note.last) {
                // ---- the end of a segment, or of this run's part of it, 32 columns at a time through shared memory, so that it
                // leaves in whole lines ----
                const bool whole = here && note.last == 1;
                const float f = !whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
                const uint64_t f_2 = f2(f, f);
                const int head = heads[i % KP_NOTES];
                float *rec = a.records + ((size_t)(2 * blockIdx.x + here) * KP_ROWS + (warp & 3) * 32) * G::RECORD_ROW;
                // (a row of the tile is position rr / group: rr * inverse >> 16, exact for rr below 128)
                const uint32_t inverse = 65536u / (uint32_t)group + 1u;
                float *out = a.out + (size_t)(note.row0 + note.first) * a.out_stride + (size_t)head * group * D;
                const int live = min(QB, note.rows - note.first) * group - (warp & 3) * 32;     // of this warp's rows
#pragma unroll
                for (int j0 = 0; j0 < D / 32; ++j0) {
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        ulonglong2 y;
                        y.x = f2_mul(o[16 * j0 + 2 * j], f_2);
                        y.y = f2_mul(o[16 * j0 + 2 * j + 1], f_2);
                        *reinterpret_cast<ulonglong2 *>(stage + lane * 128 + ((j ^ (lane & 7)) << 4)) = y;
                    }
                    __syncwarp();
#pragma unroll 1
                    for (int r = lane >> 3; r < min(live, 32); r += 4) {
                        const float4 y = *reinterpret_cast<const float4 *>(stage + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
                        const int rr = (warp & 3) * 32 + r, at = (int)((uint32_t)rr * inverse >> 16);
                        float *p = whole ? out + (size_t)at * a.out_stride + (size_t)(rr - at * group) * D : rec + r * G::RECORD_ROW;
                        p += 32 * j0 + 4 * (lane & 7);
                        if (whole && a.wide) {
                            *reinterpret_cast<float4 *>(p) = y;
                        } else {
                            p[0] = y.x; p[1] = y.y; p[2] = y.z; p[3] = y.w;
                        }
                    }
                }
                if (!whole) *reinterpret_cast<float2 *>(rec + lane * G::RECORD_ROW + D) = make_float2(m, l);
            }
        }
    }
    if (!alive) atomicExch(a.status, YSCV_DEV_MBARRIER_TIMEOUT);
    at_fence_before();
    __syncthreads();
    if (warp == 0) {
        at_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512));
    }
}

// Adds the records of segments that several SMs shared: CTAs (border between two runs, eight rows), a warp per row. A segment is
// merged by its first border.
template <int D>
__global__ void __launch_bounds__(256) kv_prompt_merge_kernel(const __grid_constant__ KvAttention a) {
    pdl_wait();
    pdl_trigger();
    constexpr int ROW = KpGeom<D>::RECORD_ROW, N = D / 32;
    const int lane = threadIdx.x & 31, r = blockIdx.y * 8 + (threadIdx.x >> 5), group = a.group, QB = KP_ROWS / group;
    const long long total = a.plan[0], share = a.plan[1], border = (blockIdx.x + 1) * share;
    if (border >= total) return;
    KpWalk w;
    int gap;
    w.seek(a, a.plan + 2, QB, border, gap);
    // places of the segment's first tile and of the end of its last
    const long long from = border + gap - w.step, to = from + w.t.steps;
    if (w.step == 0 || from < border - share) return;      // no segment is cut here, or it was cut before
    const int s = w.q * QB + r / group;
    if (r >= QB * group || s >= w.rows) return;
    const int first = blockIdx.x, parts = (int)((to - 1) / share) - first + 1;
    auto record = [&](int p) { return a.records + ((size_t)(2 * (first + p) + (p == 0)) * KP_ROWS + r) * ROW; };
    float mx = -INFINITY;
    for (int p = lane; p < parts; p += 32) mx = fmaxf(mx, record(p)[D]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    const float ref = mx == -INFINITY ? 0.0f : mx;
    float sum = 0.0f, acc[N] = {};
    for (int p0 = 0; p0 < parts; p0 += 32) {
        float x = 0.0f;
        if (p0 + lane < parts) {
            const float2 ml = *reinterpret_cast<const float2 *>(record(p0 + lane) + D);
            x = at_exp2(ml.x - ref);
            sum = fmaf(x, ml.y, sum);
        }
        const int np = min(32, parts - p0);
#pragma unroll 8
        for (int p = 0; p < np; ++p) {
            const float y = __shfl_sync(0xffffffffu, x, p);
            const float *rec = record(p0 + p);
#pragma unroll
            for (int e = 0; e < N; ++e) acc[e] = fmaf(y, rec[lane + 32 * e], acc[e]);
        }
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    float *dst = a.out + (size_t)(w.row0 + s) * a.out_stride + (size_t)(w.head * group + r % group) * D;
#pragma unroll
    for (int e = 0; e < N; ++e) dst[lane + 32 * e] = acc[e] * inv;
}

// ---- host -----------------------------------------------------------------------------------------
static size_t kp_smem(size_t d, size_t n_seq) { return (d == 64 ? KpGeom<64>::PLAN : KpGeom<128>::PLAN) + (n_seq + 1) * (sizeof(longlong2) + sizeof(long long)); }
static size_t kp_plan_bytes(size_t n_seq) { return ((2 + n_seq + 1) * sizeof(long long) + 15) & ~(size_t)15; }

size_t kv_prompt_bytes(const yscv_cuda_ctx *ctx, size_t d_head, size_t n_seq) {
    return kp_plan_bytes(n_seq) + (size_t)2 * ctx->sm_count * KP_ROWS * (d_head + 2) * sizeof(float);
}
bool kv_prompt_takes(size_t d_head, size_t n_seq, size_t group, size_t most_rows) {
    return (d_head == 64 || d_head == 128) && group <= KP_ROWS && most_rows * group > 64 && kp_smem(d_head, n_seq) <= 226 * 1024;
}

template <int D> static int kp_launch(yscv_cuda_ctx *ctx, const KvAttention &a) {
    auto kern = kv_prompt_kernel<D>;
    if (const int rc = ensure_dynamic_smem(reinterpret_cast<const void *>(kern), ctx->device, 226 * 1024)) return rc;
    YSCV_CUDA_TRY(launch_pdl(kern, dim3((unsigned)ctx->sm_count), dim3(KP_THREADS), kp_smem(D, a.l.n_seq), ctx->stream, a));
    ctx->launches++;
    YSCV_CUDA_TRY(launch_pdl(kv_prompt_merge_kernel<D>, dim3((unsigned)ctx->sm_count - 1, KP_ROWS / 8), dim3(256), 0, ctx->stream, a));
    ctx->launches++;
    YSCV_CUDA_TRY(cudaGetLastError());
    ctx->last_kernel = "kv_block_attention(prompt tiles,tcgen05)";
    return YSCV_CUDA_OK;
}

int kv_prompt(yscv_cuda_ctx *ctx, KvAttention a, void *workspace) {
    a.plan = static_cast<long long *>(workspace);
    a.records = reinterpret_cast<float *>(static_cast<unsigned char *>(workspace) + kp_plan_bytes(a.l.n_seq));
    return a.l.d == 64 ? kp_launch<64>(ctx, a) : kp_launch<128>(ctx, a);
}

}  // namespace yscv
