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
//   warp 1       queries of the next segment into shared memory, by tensor copies
//   warps 2, 3   keys and values of the tiles as they are cached, by bulk copies a tile ahead, and what the others have to know
//   warps 4-7    the tile's bytes as fp16 operands
//   warps 8-15   softmax, a thread a row, two tiles at a time: the queries' two terms to TMEM for a segment's first tile; scores from
//                TMEM, the tile's own maximum (of weight times value scale) and sum, weights back to where the scores were. They keep
//                nothing from tile to tile
//   warps 16-19  the output in registers, a thread per row: o = o + O 2^(m - M), M at most 2^8 below the running maximum, and results
// With the output in the softmax threads' registers those have too few left to keep several exponentials in flight: 2048 x 2048
// keys, 64 / 8 heads of 128, 507 us, a tile of 128 rows 6300 cycles. With all eight softmax warps on one tile, which then hand its
// maxima to each other, a tile takes 3950 cycles, with four warps on each of two tiles 3600.
// Registers are moved between the warpgroups: 640 threads x 96 = 128 x (56 + 72 + 96 + 96 + 160).
//
// Work: the tiles of all (sequence, pairs, KV head) segments are laid end to end, KP_TILE places each, with KP_BEGIN places in front of
// each segment, about what its beginning and end take, and every SM takes an equal run; a segment that several SMs share leaves records, which
// kv_prompt_merge_kernel adds. So a short piece over a long cache fills the machine too, and causal prompts, whose first
// segments have one tile, need no order of CTAs (2047 tokens, 64 / 8 heads of 128, in runs of a few calls: 151 us where it took 162
// with four places in front of a segment, 154 with five. A call among many takes 164, at a lower clock).
// Bound: the tensor pipe, 2 x (128 D + 128 D) x 128 MACs a tile, 2048 cycles at the nominal rate for D = 128; what holds a tile for 3600
// is the chain of its two products and its softmax, with as many tiles on their way as TMEM has room for (two), and the issue slots,
// of which a tile takes 2100 of each scheduler.
#include <cfloat>
#include <climits>

#include "attention_tc.cuh"
#include "kv_attention.cuh"
#include "tma.cuh"

namespace yscv {

constexpr int KP_KEYS = 128, KP_ROWS = 128, KP_THREADS = 640, KP_NOTES = 8;
constexpr int KP_TILE = 4, KP_BEGIN = 6;   // places that a tile takes, and the beginning and end of a segment

template <int D> struct KpGeom {
    static constexpr int OPERAND = KP_KEYS * D * 2, RAW = KP_KEYS * D;   // keys, or values, of a tile, in fp16 and as cached
    static constexpr int K_AT = 0, V_AT = OPERAND;             // one stage of keys, two of values
    static constexpr int RAW_K = 3 * OPERAND, RAW_V = RAW_K + RAW;
    static constexpr int Q_AT = RAW_V + RAW;                   // the next segment's queries, f32: 32 columns of all rows, the next 32, ...
    static constexpr int Q_PART = KP_ROWS * 128;
    static constexpr int STATS = Q_AT + D / 32 * Q_PART;               // [4][128] {maximum, sum} of a tile's rows
    static constexpr int NOTES = STATS + 4096;
    static constexpr int SCALES = NOTES + KP_NOTES * 128;      // [4][128] powers of two of a segment's queries, read until its last tile
    static constexpr int BARS = SCALES + 4 * KP_ROWS * 4;
    static constexpr int PLAN = BARS + 256;
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
// instruction cache together. A probe may sleep for 2 us, or fifteen waiting warps take issue slots from the others.
__device__ __forceinline__ bool kp_wait(uint32_t bar, uint32_t parity) {
#pragma unroll 1
    for (uint32_t i = 0; i < (1u << 22); ++i) {
        uint32_t ok;
        asm volatile(
            "{\n.reg .pred p;\n"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
            "selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(ok)
            : "r"(bar), "r"(parity), "r"(2000u)
            : "memory");
        if (ok) return true;
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
// Pairs tile q of a sequence: positions q * QB .. ; the keys that any of them sees, from a group's border on. (Positions behind the
// table's end have no keys; a tile of pairs has a tile of keys at least.)
struct KpTile {
    int lo, hi, steps;
};
__device__ __forceinline__ KpTile kp_tile(const KvAttention &a, int start, int rows, int QB, int q) {
    const int s0 = q * QB, s1 = min(rows, s0 + QB);
    KpTile t;
    t.lo = a.window > 0 ? max(0, start + s0 + 1 - a.window) & ~(KV_GROUP - 1) : 0;
    t.hi = min(a.causal ? start + s1 : start + rows, a.room);
    t.steps = max((t.hi - t.lo + KP_KEYS - 1) / KP_KEYS, 1);
    return t;
}
__device__ __forceinline__ int kp_tiles(int rows, int QB) { return (rows + QB - 1) / QB; }
// Tiles of a sequence for one KV head, a warp together
__device__ __forceinline__ int kp_steps(const KvAttention &a, int start, int rows, int QB) {
    int n = 0;
    for (int q = threadIdx.x & 31; q < kp_tiles(rows, QB); q += 32) n += kp_tile(a, start, rows, QB, q).steps;
    return __reduce_add_sync(0xffffffffu, n);
}

struct KpWalk {
    int seq, q, head, step, start, rows, row0;
    KpTile t;
    __device__ void load(const KvAttention &a) {
        const KvSeqRows r = kv_rows(a, seq);
        start = r.start;
        rows = r.rows;
        row0 = r.row0;
    }
    // The tile that place `left` of sequence `seq` is within, or whose beginning it is in front of, a warp together. Returns the tiles of
    // the sequence in front of it; `in`: places of its segment in front of that place.
    __device__ int seek(const KvAttention &a, int QB, int left, int &in) {
        load(a);
        int tiles = 0;
        const int lane = threadIdx.x & 31;
        for (int q0 = 0;; q0 += 32) {
            const int steps = q0 + lane < kp_tiles(rows, QB) ? kp_tile(a, start, rows, QB, q0 + lane).steps : 0;
            const int n = steps > 0 ? (KP_TILE * steps + KP_BEGIN) * a.l.n_kv : 0;
            int upto = n, tiles_upto = steps * a.l.n_kv;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, upto, o), z = __shfl_up_sync(0xffffffffu, tiles_upto, o);
                if (lane >= o) { upto += y; tiles_upto += z; }
            }
            const unsigned past = __ballot_sync(0xffffffffu, upto > left);
            if (past) {
                const int f = __ffs(past) - 1;
                left -= __shfl_sync(0xffffffffu, upto - n, f);
                tiles += __shfl_sync(0xffffffffu, tiles_upto - steps * a.l.n_kv, f);
                q = q0 + f;
                break;
            }
            left -= __shfl_sync(0xffffffffu, upto, 31);
            tiles += __shfl_sync(0xffffffffu, tiles_upto, 31);
        }
        t = kp_tile(a, start, rows, QB, q);
        const int places = KP_TILE * t.steps + KP_BEGIN;
        head = left / places;
        in = left - head * places;
        step = max(0, in - KP_BEGIN) / KP_TILE;
        return tiles + head * t.steps + step;
    }
    // the first step of the next segment (there is one)
    __device__ void next_segment(const KvAttention &a, int QB) {
        step = 0;
        if (++head < a.l.n_kv) return;
        head = 0;
        if (++q >= kp_tiles(rows, QB)) {
            q = 0;
            do {
                ++seq;
                load(a);
            } while (rows == 0);
        }
        t = kp_tile(a, start, rows, QB, q);
    }
    __device__ void next(const KvAttention &a, int QB) {
        if (++step == t.steps) next_segment(a, QB);
    }
};

// What a CTA writes down for kv_prompt_merge_kernel about the segment that its run begins within
struct KpCut {
    int parts;                     // runs that have a part of it, 0: there is none, or an earlier run says so
    int row, live, head;           // its first row of the output, its pairs, its KV head
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
__global__ void __launch_bounds__(KP_THREADS, 1) kv_prompt_kernel(const __grid_constant__ KvAttention a, const __grid_constant__ CUtensorMap q_map) {
    using G = KpGeom<D>;
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ KpWalk run;                  // the CTA's first tile
    __shared__ int run_ends[2];
    __shared__ uint32_t tmem_slot;
    __shared__ int heads[KP_NOTES], begun[KP_NOTES], segments[KP_NOTES];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t base = smem_u32(smem), bars = base + G::BARS;
    // [2] by tile & 1, each used again two tiles later (pfull: another two for the tile's second 64 keys); nfull [KP_NOTES]; from kfull on
    // one phase a tile; from qstaged on one a segment
    const uint32_t vfull = bars, sfull = bars + 16, pfull = bars + 32, ofull = bars + 64, ofree = bars + 80;
    const uint32_t nfull = bars + 96, kfull = bars + 160, raw_k = bars + 176, raw_v = bars + 184, raw_k_free = bars + 192;
    const uint32_t raw_v_free = bars + 200, qstaged = bars + 216, qtaken = bars + 224, qfull = bars + 232;
    float2 *stats = reinterpret_cast<float2 *>(smem + G::STATS);
    float *scales = reinterpret_cast<float *>(smem + G::SCALES);
    KpNote *notes = reinterpret_cast<KpNote *>(smem + G::NOTES);
    int2 *counted = reinterpret_cast<int2 *>(smem + G::PLAN);               // [n_seq] places and tiles
    const int group = a.group, QB = KP_ROWS / group;

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(vfull + i * 8, 4);
            mbar_init(sfull + i * 8, 1);
            mbar_init(pfull + i * 8, 4);
            mbar_init(pfull + 16 + i * 8, 4);
            mbar_init(ofull + i * 8, 1);
            mbar_init(ofree + i * 8, 4);
        }
        for (int i = 0; i < KP_NOTES; ++i) mbar_init(nfull + i * 8, 1);
        mbar_init(kfull, 4);
        mbar_init(raw_k, 1);
        mbar_init(raw_v, 1);
        mbar_init(raw_k_free, 4);
        mbar_init(raw_v_free, 4);
        mbar_init(qstaged, 1);
        mbar_init(qtaken, 4);
        mbar_init(qfull, 4);
        mbar_fence_init();
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&tmem_slot)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
    }
    pdl_wait();
    pdl_trigger();
    // ---- places and tiles of every sequence, and which are this CTA's ----
    for (int i = warp; i < a.l.n_seq; i += KP_THREADS / 32) {
        const KvSeqRows r = kv_rows(a, i);
        const int n = kp_steps(a, r.start, r.rows, QB);
        if (lane == 0) {
            counted[i] = make_int2((KP_TILE * n + KP_BEGIN * kp_tiles(r.rows, QB)) * a.l.n_kv, n * a.l.n_kv);
            if (blockIdx.x == 0) kv_rows_status(a, r);
        }
    }
    at_fence_before();
    __syncthreads();
    at_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
    if (warp < 2) {                         // where this run begins, and where the next does
        const int n_seq = a.l.n_seq;
        auto counts = [&](int i0) { return i0 + lane < n_seq ? counted[i0 + lane] : make_int2(0, 0); };
        long long places = 0;               // of the call
        int t = 0;                          // tiles in front of place u
        for (int i0 = 0; i0 < n_seq; i0 += 32) {
            const int2 c = counts(i0);
            places += ((long long)__reduce_add_sync(0xffffffffu, c.x >> 16) << 16) + __reduce_add_sync(0xffffffffu, c.x & 0xffff);
            t += __reduce_add_sync(0xffffffffu, c.y);
        }
        // (more than 32 bits hold: only of sequences that overlap. Then nobody takes part.)
        const int total = places <= INT_MAX ? (int)places : 0;
        if (places > INT_MAX) {
            t = 0;
            if (blockIdx.x == 0 && tid == 0) atomicExch(a.status, YSCV_DEV_BAD_NUMBER);
        }
        // (no run in the middle of a segment is without a tile)
        const int share = max((int)(((unsigned)total + gridDim.x - 1) / gridDim.x), KP_TILE), u0 = (int)min((long long)total, (long long)blockIdx.x * share);
        const int u = warp == 0 ? u0 : (int)min((long long)total, (long long)u0 + share);
        KpWalk w;
        int in = 0;
        if (u < total) {
            int i0 = 0, front = 0;
            t = 0;
            int2 c = counts(0);
            for (int x; (x = __reduce_add_sync(0xffffffffu, c.x)) <= u - front; c = counts(i0 += 32)) {
                front += x;
                t += __reduce_add_sync(0xffffffffu, c.y);
            }
            int2 x = c;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x.x, o), z = __shfl_up_sync(0xffffffffu, x.y, o);
                if (lane >= o) { x.x += y; x.y += z; }
            }
            const int f = __ffs(__ballot_sync(0xffffffffu, x.x > u - front)) - 1;
            front += __shfl_sync(0xffffffffu, x.x - c.x, f);
            t += __shfl_sync(0xffffffffu, x.y - c.y, f);
            w.seq = i0 + f;
            t += w.seek(a, QB, u - front, in);
        }
        if (lane == 0) {
            run_ends[warp] = t;
            if (warp == 0) {
                KpCut cut = {};
                if (u < total) {
                    run = w;
                    // a tile is in the run of its last place; is the segment cut for the first time?
                    const int first = u - in + KP_BEGIN + KP_TILE - 1, last = first + KP_TILE * (w.t.steps - 1), s0 = w.q * QB;
                    if (w.step > 0 && first / share == (int)blockIdx.x - 1)
                        cut = {last / share - (int)blockIdx.x + 2, w.row0 + s0, min(QB, w.rows - s0) * group, w.head};
                }
                static_cast<KpCut *>(a.plan)[blockIdx.x] = cut;
            }
        }
    }
    __syncthreads();
    const int n = run_ends[1] - run_ends[0];
    // TMEM columns: queries (both terms), scores and then weights [2] x 128, weighted values
    const uint32_t t_q = tmem, t_s = tmem + 128, t_o = tmem + 384;
    auto par = [](int i) { return (uint32_t)(i >> 1) & 1u; };
    bool alive = true;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;\n");
        if (warp == 0) {
            // ---- products: what comes last is waited for last, since a barrier that is ready takes 100 cycles to say so ----
            if (n > 0) {
                const uint32_t id_s = (1u << 4) | ((uint32_t)(KP_KEYS >> 3) << 17) | ((uint32_t)(KP_ROWS >> 4) << 24);
                const uint32_t id_o = (1u << 4) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(KP_ROWS >> 4) << 24);
                const uint32_t at = (base >> 4) | 1u << 16;
                uint32_t segments = 0;
                auto scores = [&](int i, bool begins) {
                    const int st = i & 1;
                    if (begins && !__all_sync(0xffffffffu, kp_wait(qfull, segments++ & 1u))) return false;
                    at_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int e = 0; e < D / 8; ++e) {           // remainders first
                            const int kk = e & (D / 16 - 1), term = e < D / 16;
                            at_mma_ts(t_s + st * 128, t_q + (kk >> 1) * 32 + term * 16 + (kk & 1) * 8,
                                      kp_desc(at, G::K_AT + (kk >> 2) * (KP_KEYS * 128) + (kk & 3) * 32), id_s, e > 0);
                        }
                        at_commit(sfull + st * 8);
                    }
                    __syncwarp();
                    return true;
                };
                auto values = [&](int i) {
                    const int st = i & 1;
                    if (!__all_sync(0xffffffffu, (i == 0 || kp_wait(ofree + (st ^ 1) * 8, par(i - 1))) && kp_wait(vfull + st * 8, par(i)))) return false;
                    // as soon as the weights of 64 keys are there: theirs, under the exponentials of the others
#pragma unroll 1
                    for (int h = 0; h < 2; ++h) {
                        if (!__all_sync(0xffffffffu, kp_wait(pfull + h * 16 + st * 8, par(i)))) return false;
                        at_fence_after();
                        if (elect_one()) {
                            const uint32_t v_at = at + (uint32_t)((G::V_AT + st * G::OPERAND + h * (D * 128)) >> 4), p_at = t_s + st * 128 + h * 64;
#pragma unroll
                            for (int e = 0; e < KP_KEYS / 16; ++e) {
                                const int kk = e & 3, term = e < 4;
                                at_mma_ts(t_o, p_at + kk * 16 + term * 8, kp_desc(v_at, kk * 32), id_o, e + h > 0);
                            }
                            if (h) at_commit(ofull + st * 8);
                        }
                        __syncwarp();
                    }
                    return true;
                };
                alive = __all_sync(0xffffffffu, kp_wait(kfull, 0u)) && scores(0, true);
#pragma unroll 1
                for (int i = 0; i < n && alive; ++i) {
                    // the next tile's scores first. The weights of tile i - 1, which lie where these scores go, have been multiplied by then
                    if (i + 1 < n) {
                        const int st = (i + 1) & 1;
                        alive = __all_sync(0xffffffffu, kp_wait(kfull, (uint32_t)(i + 1) & 1u) && (i == 0 || kp_wait(ofull + st * 8, par(i - 1))));
                        if (!alive) break;
                        alive = scores(i + 1, begun[(i + 1) % KP_NOTES] != 0);
                    }
                    alive = alive && values(i);
                }
            }
        } else if (warp == 1 && n > 0) {
            // ---- queries of the next segment, as they are: one tensor copy per 32 columns of its positions and heads, with the 128-byte
            // swizzle, so that threads can read a row each (a copy a row took 11,000 cycles, stores of this warp more). Rows behind the
            // sequence come along and are not looked at ----
            KpWalk w = run;
            int i = 0, loaded = 0;
            for (int segment = 0;; ++segment) {
                if (segment > 0) alive = __all_sync(0xffffffffu, kp_wait(qtaken, (uint32_t)(segment - 1) & 1u));
                if (!alive) break;
                const int s0 = w.q * QB;
                if (a.wide) {
                    if (lane == 0) mbar_expect_tx(qstaged, QB * group * D * 4);
                    __syncwarp();
                    if (lane < D / 32)
                        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(
                                         base + G::Q_AT + lane * G::Q_PART),
                                     "l"(&q_map), "r"(32 * lane), "r"(w.head * group), "r"(w.row0 + s0), "r"(qstaged)
                                     : "memory");
                } else {
                    const int live = min(QB, w.rows - s0) * group;
                    for (int r = 0; r < live; ++r) {
                        const float *from = a.q + (size_t)(w.row0 + s0 + r / group) * a.q_stride + (size_t)(w.head * group + r % group) * D;
                        unsigned char *to = smem + G::Q_AT + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4;
#pragma unroll
                        for (int c = 0; c < D / 32; ++c) *reinterpret_cast<float *>(to + c * G::Q_PART) = from[32 * c + lane];
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(qstaged);
                }
                loaded = segment + 1;
                i += w.t.steps - w.step;
                if (i >= n) break;
                w.next_segment(a, QB);
            }
            // no copy may be in flight when the CTA leaves (bounded)
            if (!alive && loaded > 0) kp_wait(qstaged, (uint32_t)(loaded - 1) & 1u);
        } else if (warp > 1 && n > 0) {
            // ---- keys (warp 2) and values (warp 3) as they are cached, by bulk copies; what the others have to know about a tile.
            // Lane g < 8 looks after group g: its page, a tile ahead, and its scales ----
            const bool values = warp == 3;
            const int8_t *pool = values ? a.l.v : a.l.k;
            const uint32_t full = values ? raw_v : raw_k, free = values ? raw_v_free : raw_k_free;
            const uint32_t to = base + (values ? G::RAW_V : G::RAW_K) + lane * (KV_GROUP * D);
            KpWalk w = run;
            const int piece = min(a.l.page / KV_GROUP, 8);        // groups that lie together, from a page's border on
            int id = -1;
            auto page = [&]() {
                const int key = w.t.lo + w.step * KP_KEYS + KV_GROUP * lane, at = key >> a.l.page_shift;
                id = -1;
                if (lane < 8 && key < w.t.hi) {
                    if (at < a.l.max_pages) id = a.l.table[(size_t)w.seq * a.l.max_pages + at];
                    else atomicExch(a.status, YSCV_DEV_POS_OVERFLOW);
                }
            };
            bool begins = true;
            int segment = 0, copied = 0;                                       // tiles on their way or there
            page();
#pragma unroll 1
            for (int i = 0; i < n; ++i) {
                const int key0 = w.t.lo + w.step * KP_KEYS, key = key0 + KV_GROUP * lane;
                const bool wanted = lane < 8 && key < w.t.hi, there = wanted && id >= 0 && id < a.l.n_pages;
                if (wanted && !there && (key >> a.l.page_shift) < a.l.max_pages) atomicExch(a.status, YSCV_DEV_BAD_NUMBER);
                float ks = 1.0f, vs = -1.0f;
                if (!values && there) {
                    ks = a.l.ks[(size_t)id * a.l.n_kv + w.head];
                    vs = a.l.vs[(size_t)id * a.l.n_kv + w.head];
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
                        // (at least 2^-80: a group whose values are 0 counts in the sum all the same, and the inverse stays far below
                        // what sums over a sequence can hold)
                        const float ratio = fmaxf(__fdiv_rn(vs, fmaxf(vmost, 7.5e-37f)), 8.2718061e-25f);
                        o.ks[lane] = ks;
                        o.lv[lane] = there ? log2f(ratio) : -INFINITY;
                        o.iv[lane] = there ? __fdiv_rn(1.0f, ratio) : 0.0f;
                    }
                    if (lane == 0) {
                        o.vmost = vmost;
                        o.key0 = key0;
                        o.last = w.step + 1 == w.t.steps ? 1 : i + 1 == n ? 2 : 0;
                        o.begins = begins ? 1 + w.step : 0;
                        o.start = w.start; o.rows = w.rows; o.row0 = w.row0; o.first = w.q * QB;
                        heads[i % KP_NOTES] = w.head;
                        segments[i % KP_NOTES] = segment;
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(nfull + i % KP_NOTES * 8);
                }
                begins = w.step + 1 == w.t.steps;
                segment += begins;
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
        // (values have two places: in one their conversion, which takes as long as a product, would stand between any two of them)
#pragma unroll 1
        for (int j = 0; j < 2 * n; ++j) {
            const bool values = j & 1;
            const int i = j >> 1, st = i & 1;
            alive = kp_wait(values ? raw_v : raw_k, (uint32_t)i & 1u);
            // (keys: the scores of tile i - 1 are there; values: the weighted values of tile i - 2)
            if (i > values) alive = alive && kp_wait(values ? ofull + st * 8 : sfull + (st ^ 1) * 8, values ? par(i - 2) : par(i - 1));
            alive = __all_sync(0xffffffffu, alive);
            if (!alive) break;
            const unsigned char *from = smem + (values ? G::RAW_V : G::RAW_K) + t * 16;
            if (values) {   // 16 tokens of a row are pieces 2 (g & 3) and the next of row d of the 64-key half
                unsigned char *to = smem + G::V_AT + st * G::OPERAND + in * 128;
                const int swizzle = ((2 * g0) ^ (in & 7)) << 4;
#pragma unroll
                for (int e = 0; e < ITEMS; ++e) {
                    uint4 lo, hi;
                    kp_convert(*reinterpret_cast<const uint4 *>(from + e * 2048), lo, hi);
                    const int at0 = (e * PER >> 2) * (D * 128) + (swizzle ^ ((e * PER & 3) << 5));
                    *reinterpret_cast<uint4 *>(to + at0) = lo;
                    *reinterpret_cast<uint4 *>(to + (at0 ^ 16)) = hi;
                }
            } else {        // 16 d of a token are pieces 2 c and 2 c + 1 of its 128-byte row of the 64-d sub-tile
                unsigned char *to = smem + G::K_AT + (in >> 6) * (KP_KEYS * 128) + (g0 * KV_GROUP + (in & 15)) * 128;
                const int at0 = ((2 * ((in >> 4) & 3)) ^ (in & 7)) << 4;
                unsigned char *to0 = to + at0, *to1 = to + (at0 ^ 16);
#pragma unroll
                for (int e = 0; e < ITEMS; ++e) {
                    uint4 lo, hi;
                    kp_convert(*reinterpret_cast<const uint4 *>(from + e * 2048), lo, hi);
                    *reinterpret_cast<uint4 *>(to0 + e * (PER * KV_GROUP * 128)) = lo;
                    *reinterpret_cast<uint4 *>(to1 + e * (PER * KV_GROUP * 128)) = hi;
                }
            }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(values ? vfull + st * 8 : kfull);
                mbar_arrive(values ? raw_v_free : raw_k_free);
            }
        }
    } else if (warp < 16) {
        // ---- softmax, a thread a row: warps 8-11 the even tiles, warps 12-15 the odd ones, so that one tile's exponentials run while
        // the other's products are waited for ----
        const int row = (warp & 3) * 32 + lane, in_tile = row / group;
        const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
#pragma unroll 1
        for (int i = warp >= 12; i < n; i += 2) {
            const int st = i & 1;
            const uint32_t s_at = t_s + st * 128 + lane_off;
            alive = __all_sync(0xffffffffu, kp_wait(nfull + i % KP_NOTES * 8, (uint32_t)(i / KP_NOTES) & 1u));
            if (!alive) break;
            const KpNote &note = notes[i % KP_NOTES];
            const int segment = segments[i % KP_NOTES], s_pos = note.first + in_tile;
            const bool there = row < QB * group && s_pos < note.rows;
            volatile float *scale_at = scales + (segment & 3) * KP_ROWS + row;
            if (note.begins) {
                // its queries take the place of the last segment's, once those scores are done
                if (i > 0) alive = kp_wait(sfull + (st ^ 1) * 8, par(i - 1));
                alive = __all_sync(0xffffffffu, alive && kp_wait(qstaged, (uint32_t)segment & 1u));
                if (!alive) break;
                at_fence_after();
                const unsigned char *q = smem + G::Q_AT + row * 128;
                const int swizzle = (row & 7) << 4;
                float most = 0.0f;
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float4 y = *reinterpret_cast<const float4 *>(q + c * G::Q_PART + ((16 * j) ^ swizzle));
                        most = fmaxf(fmaxf(most, fmaxf(fabsf(y.x), fabsf(y.y))), fmaxf(fabsf(y.z), fabsf(y.w)));
                    }
                }
                float up, down;
                at_scale(most, up, down);
                *scale_at = up;
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t x[32];               // 16 columns of leading terms, 16 of remainders
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        float4 y = *reinterpret_cast<const float4 *>(q + c * G::Q_PART + ((16 * j) ^ swizzle));
                        if (!there) y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        at_split(y.x * up, y.y * up, x[2 * j], x[16 + 2 * j]);
                        at_split(y.z * up, y.w * up, x[2 * j + 1], x[16 + 2 * j + 1]);
                    }
                    at_st32(t_q + lane_off + 32 * c, x);
                }
                asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
                at_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(qfull);
                    mbar_arrive(qtaken);
                }
            }
            // the keys of the tile that this row sees (one that is not there sees all, which nobody reads: masks cost time)
            const int to = !there ? KP_KEYS : (a.causal ? note.start + s_pos + 1 : note.start + note.rows) - note.key0;
            const int from = a.window > 0 && there ? note.start + s_pos + 1 - a.window - note.key0 : 0;
            const float *ks = note.ks, *lv = note.lv, *iv = note.iv;
            // (groups up to the last one that is there, in pairs)
            const int groups = (32 - __clz(__ballot_sync(0xffffffffu, lane < 8 && iv[lane & 7] != 0.0f)) + 1) & ~1;
            const bool edge = __any_sync(0xffffffffu, to < KP_KEYS || from > 0 || iv[lane & 7] == 0.0f);
            alive = __all_sync(0xffffffffu, kp_wait(sfull + st * 8, par(i)));
            if (!alive) break;
            at_fence_after();
            // (the power of two's inverse)
            const float to_log2 = there ? a.scale * __uint_as_float((254u << 23) - __float_as_uint(*scale_at)) : 0.0f;
            // The loops are kept small: with every role's code laid out flat most of the time went to fetching instructions
            if (edge) {                        // keys that a row does not see
#pragma unroll 1
                for (int g = 0; g < groups; ++g) {
                    const bool gone = iv[g] == 0.0f;
                    if (!__any_sync(0xffffffffu, gone || 16 * g + 16 > to || 16 * g < from)) continue;
                    float v[16];
                    kp_ld16(s_at + 16 * g, v);
                    kp_wait_ld16(v);
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (gone || 16 * g + e >= to || 16 * g + e < from) v[e] = -INFINITY;
                    kp_st16(s_at + 16 * g, reinterpret_cast<const uint32_t(&)[16]>(v));
                }
                asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
            }
            // (never 0, where pages have no scale or products leave fp32's range: a hidden key's -inf has to stay one. What a seen key's
            // score, at most 2^29 here, becomes by it is 2^-97 at most, a weight's exponent of nothing)
            auto times = [&](float k) { return fmaxf(to_log2 * k, FLT_MIN); };
            // The largest weight times value scale, not the largest weight: what a row sees has its 22 bits whatever lies beside it
            float mx = -INFINITY, v[16], u[16];
            kp_ld16(s_at, v);
#pragma unroll 1
            for (int g = 0; g < groups; g += 2) {
                const float2 k2 = *reinterpret_cast<const float2 *>(ks + g), l2 = *reinterpret_cast<const float2 *>(lv + g);
                auto most = [&](const float (&z)[16], float k, float lv) {
                    float x = fmaxf(z[0], z[1]), y = fmaxf(z[2], z[3]);
#pragma unroll
                    for (int e = 4; e < 16; e += 4) {
                        x = fmaxf(x, fmaxf(z[e], z[e + 1]));
                        y = fmaxf(y, fmaxf(z[e + 2], z[e + 3]));
                    }
                    mx = fmaxf(mx, fmaf(fmaxf(x, y), times(k), lv));
                };
                kp_wait_ld16(v);
                kp_ld16(s_at + 16 * g + 16, u);
                most(v, k2.x, l2.x);
                kp_wait_ld16(u);
                kp_ld16(s_at + (g + 2 < groups ? 16 * g + 32 : 0), v);     // (at the end the first ones again)
                most(u, k2.y, l2.y);
            }
            const float off = mx == -INFINITY ? 0.0f : 10.0f - mx;
            float sum = 0.0f;
            auto half_done = [&]() {
                asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
                at_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(pfull + st * 8);
            };
            auto weights = [&](int g, const float (&v)[16], float k, float lv, float inv) {
                const float c = times(k), og = off + lv;
                const uint64_t c2 = f2(c, c), og2 = f2(og, og), minus = f2(-1.0f, -1.0f);
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
            };
#pragma unroll 1
            for (int g = 0; g < groups; g += 2) {
                if (g == 4) half_done();
                const float2 k2 = *reinterpret_cast<const float2 *>(ks + g), l2 = *reinterpret_cast<const float2 *>(lv + g), i2 = *reinterpret_cast<const float2 *>(iv + g);
                kp_wait_ld16(v);
                kp_ld16(s_at + 16 * g + 16, u);
                weights(g, v, k2.x, l2.x, i2.x);
                kp_wait_ld16(u);
                if (g + 2 < groups) kp_ld16(s_at + 16 * g + 32, v);
                weights(g + 1, u, k2.y, l2.y, i2.y);
            }
            if (groups == 0) kp_wait_ld16(v);
#pragma unroll 1
            for (int g = groups; g < 8; g += 2) {
                if (g == 4) half_done();
                const uint32_t none[16] = {};
                kp_st16(s_at + 16 * g, none);
                kp_st16(s_at + 16 * g + 16, none);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
            stats[(i & 3) * KP_ROWS + row] = make_float2(mx, sum);
            at_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(pfull + 16 + st * 8);
        }
    } else {
        // ---- output ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 160;\n");
        const int row = (warp & 3) * 32 + lane;
        const uint32_t o_at = t_o + ((uint32_t)((warp & 3) * 32) << 16);
        uint64_t o[D / 2];
        float m = -INFINITY, l = 0.0f;
        bool here = false;                             // here: the segment began in this run
        for (int i = 0; i < n; ++i) {
            const int st = i & 1;
            // (the note and the rows' statistics were there before. Weights may be a tile ahead by now, so theirs is no barrier to wait on)
            alive = __all_sync(0xffffffffu, kp_wait(ofull + st * 8, par(i)));
            if (!alive) break;
            at_fence_after();
            const KpNote &note = notes[i % KP_NOTES];
            const float2 ms = stats[(i & 3) * KP_ROWS + row];
            if (note.begins) {
                here = note.begins == 1;
                m = -INFINITY;
                l = 0.0f;
#pragma unroll
                for (int j = 0; j < D / 2; ++j) o[j] = 0ull;
            }
            // What the output is relative to follows the maximum only where that is 2^8 above it, which after a segment's first tiles is
            // rare (pieces of three prompts, in runs of a few calls: 88 us, 91 with a factor on the output for every tile)
            if (__any_sync(0xffffffffu, ms.x > m + 8.0f)) {
                const float m_new = fmaxf(m, ms.x), alpha = m_new == -INFINITY ? 1.0f : at_exp2(m - m_new);
                const uint64_t al2 = f2(alpha, alpha);
                l *= alpha;
                m = m_new;
#pragma unroll
                for (int j = 0; j < D / 2; ++j) o[j] = f2_mul(o[j], al2);
            }
            float t0[16], t1[16];
            kp_ld16(o_at, t0);
            const float beta = m == -INFINITY ? 0.0f : at_exp2(ms.x - m);
            l = fmaf(beta, ms.y, l);
            const float b = beta * fmaxf(note.vmost, 0.0f);
            const uint64_t b2 = f2(b, b);
            // (read as fast as it goes: the next product with weights waits for it)
#pragma unroll
            for (int j0 = 0; j0 < D; j0 += 32) {
                kp_wait_ld16(t0);
                kp_ld16(o_at + j0 + 16, t1);
#pragma unroll
                for (int e = 0; e < 8; ++e) o[j0 / 2 + e] = f2_fma(f2(t0[2 * e], t0[2 * e + 1]), b2, o[j0 / 2 + e]);
                kp_wait_ld16(t1);
                if (j0 + 32 < D) kp_ld16(o_at + j0 + 32, t0);
#pragma unroll
                for (int e = 0; e < 8; ++e) o[j0 / 2 + 8 + e] = f2_fma(f2(t1[2 * e], t1[2 * e + 1]), b2, o[j0 / 2 + 8 + e]);
            }
            at_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(ofree + st * 8);
            if (note.last) {
                // ---- the end of a segment, or of this run's part of it: each thread its row, 32 bytes at a time ----
                const bool whole = here && note.last == 1;
                const float f = !whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
                const uint64_t f_2 = f2(f, f);
                const int in_tile = row / group;
                const size_t slot = (size_t)(2 * blockIdx.x + here) * KP_ROWS + row;
                float *dst = !whole ? a.records + slot * D
                                    : a.out + (size_t)(note.row0 + note.first + in_tile) * a.out_stride + (size_t)(heads[i % KP_NOTES] * group + row - in_tile * group) * D;
                if (!whole) reinterpret_cast<float2 *>(a.records + (size_t)2 * gridDim.x * KP_ROWS * D)[slot] = make_float2(m, l);
                if (row < min(QB, note.rows - note.first) * group) {
#pragma unroll
                    for (int j = 0; j < D / 8; ++j) {
                        float y[8];
#pragma unroll
                        for (int e = 0; e < 4; ++e) f2_get(f2_mul(o[4 * j + e], f_2), y[2 * e], y[2 * e + 1]);
                        if (!whole || a.wide > 1) {
                            asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(dst + 8 * j), "f"(y[0]), "f"(y[1]), "f"(y[2]),
                                         "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7])
                                         : "memory");
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e) dst[8 * j + e] = y[e];
                        }
                    }
                }
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
// merged by its first border, whose run has written down what it is.
template <int D>
__global__ void __launch_bounds__(256) kv_prompt_merge_kernel(const __grid_constant__ KvAttention a) {
    pdl_wait();
    pdl_trigger();
    constexpr int N = D / 32;
    const int lane = threadIdx.x & 31, r = blockIdx.y * 8 + (threadIdx.x >> 5), group = a.group, first = blockIdx.x;
    const KpCut cut = static_cast<const KpCut *>(a.plan)[first + 1];
    const int parts = cut.parts;
    if (parts == 0 || r >= cut.live) return;
    auto slot = [&](int p) { return (size_t)(2 * (first + p) + (p == 0)) * KP_ROWS + r; };
    const float2 *stats = reinterpret_cast<const float2 *>(a.records + (size_t)2 * (gridDim.x + 1) * KP_ROWS * D);   // (a CTA a border)
    float mx = -INFINITY;
    for (int p = lane; p < parts; p += 32) mx = fmaxf(mx, stats[slot(p)].x);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    const float ref = mx == -INFINITY ? 0.0f : mx;
    float sum = 0.0f, acc[N] = {};
    for (int p0 = 0; p0 < parts; p0 += 32) {
        float x = 0.0f;
        if (p0 + lane < parts) {
            const float2 ml = stats[slot(p0 + lane)];
            x = at_exp2(ml.x - ref);
            sum = fmaf(x, ml.y, sum);
        }
        const int np = min(32, parts - p0);
#pragma unroll 8
        for (int p = 0; p < np; ++p) {
            const float y = __shfl_sync(0xffffffffu, x, p);
            const float *rec = a.records + slot(p0 + p) * D;
#pragma unroll
            for (int e = 0; e < N; ++e) acc[e] = fmaf(y, rec[lane + 32 * e], acc[e]);
        }
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    float *dst = a.out + (size_t)(cut.row + r / group) * a.out_stride + (size_t)(cut.head * group + r % group) * D;
#pragma unroll
    for (int e = 0; e < N; ++e) dst[lane + 32 * e] = acc[e] * inv;
}

// ---- host -----------------------------------------------------------------------------------------
static size_t kp_smem(size_t d, size_t n_seq) { return (d == 64 ? KpGeom<64>::PLAN : KpGeom<128>::PLAN) + n_seq * sizeof(int2); }
static size_t kp_plan_bytes(const yscv_cuda_ctx *ctx) { return (ctx->sm_count * sizeof(KpCut) + 31) & ~(size_t)31; }

size_t kv_prompt_bytes(const yscv_cuda_ctx *ctx, size_t d_head) {
    return 32 + kp_plan_bytes(ctx) + (size_t)2 * ctx->sm_count * KP_ROWS * (d_head * sizeof(float) + sizeof(float2));
}
// Above 32 pairs a KV head, which the other kernel takes as two blocks of 16 that read the cache once each (us here, by steps):
//                                                   heads of 128, group 4                  heads of 64, group 8
//   pairs                                           16          32          64             32          64
//   8 sequences of 300 keys, 32 query heads         18.6, 20.8  19.0, 19.8  19.8, 28.3     15.2, 15.8  15.3, 16.5
//   8 of 4000                                       43.4, 39.4  44.0, 47.1  45.2, 76.7     26.8, 27.8  26.5, 36.1
//   64 of 2000                                      128, 89     131, 147    136, 265       61, 55      63, 89
//   one of 8000                                     26.4, 21.6  26.8, 24.2  27.6, 37.7     19.2, 16.4  19.6, 18.4
bool kv_prompt_takes(const yscv_cuda_kv_pool *pool, size_t group, size_t rows, size_t most_rows) {
    if ((pool->d_head != 64 && pool->d_head != 128) || group > KP_ROWS || kp_smem(pool->d_head, pool->n_seq) > 226 * 1024) return false;
    // (places are counted in 32 bits)
    const size_t tiles = rows / (KP_ROWS / group) + pool->n_seq, steps = KP_TILE * (pool->max_pages * pool->page / KP_KEYS + 2) + KP_BEGIN;
    if (tiles >= (1u << 31) / pool->n_kv / steps) return false;
    return most_rows * group > 32;
}

template <int D> static int kp_launch(yscv_cuda_ctx *ctx, const KvAttention &a) {
    auto kern = kv_prompt_kernel<D>;
    if (const int rc = ensure_dynamic_smem(reinterpret_cast<const void *>(kern), ctx->device, 226 * 1024)) return rc;
    CUtensorMap q_map = {};
    if (a.wide) {
        const EncodeTiledFn encode = tensor_map_encoder();
        if (!encode) return fail(YSCV_CUDA_ERR_UNSUPPORTED, "no tensor-map encoder in this driver");
        const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)a.n_q, (cuuint64_t)a.rows}, strides[2] = {(cuuint64_t)D * 4, (cuuint64_t)a.q_stride * 4};
        const cuuint32_t box[3] = {32, (cuuint32_t)a.group, (cuuint32_t)(KP_ROWS / a.group)}, ones[3] = {1, 1, 1};
        const CUresult r = encode(&q_map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<float *>(a.q), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS) return fail(YSCV_CUDA_ERR_CUDA, "cuTensorMapEncodeTiled failed: %d", (int)r);
    }
    YSCV_CUDA_TRY(launch_pdl(kern, dim3((unsigned)ctx->sm_count), dim3(KP_THREADS), kp_smem(D, a.l.n_seq), ctx->stream, a, q_map));
    ctx->launches++;
    YSCV_CUDA_TRY(launch_pdl(kv_prompt_merge_kernel<D>, dim3((unsigned)ctx->sm_count - 1, KP_ROWS / 8), dim3(256), 0, ctx->stream, a));
    ctx->launches++;
    YSCV_CUDA_TRY(cudaGetLastError());
    ctx->last_kernel = "kv_block_attention(prompt tiles,tcgen05)";
    return YSCV_CUDA_OK;
}

int kv_prompt(yscv_cuda_ctx *ctx, KvAttention a, void *workspace) {
    a.plan = workspace;
    // (32 bytes at a time: the output's stores)
    a.records = reinterpret_cast<float *>((reinterpret_cast<uintptr_t>(workspace) + kp_plan_bytes(ctx) + 31) & ~(uintptr_t)31);
    if (a.wide && reinterpret_cast<uintptr_t>(a.out) % 32 == 0 && a.out_stride % 8 == 0) a.wide = 2;
    return a.l.d == 64 ? kp_launch<64>(ctx, a) : kp_launch<128>(ctx, a);
}

}  // namespace yscv
