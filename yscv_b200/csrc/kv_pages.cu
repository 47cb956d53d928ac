// Pages of a paged KV cache: which sequence has which (extend, trim, fork, compact), and the copies that follow.
//
// What is decided (who needs pages, which ones are free, what moves) is a few thousand integers and prefix sums in the order
// of the sequences and of the pages: one block, so that no two launches have to agree on a count, bound by the latency of what hangs on
// one another (a load from memory costs as much as all the arithmetic): which pages are used is read once, into a bit each in
// shared memory, and what a sequence needs stays with its thread. What is moved (shared last pages, pages that close gaps) is bound by bytes, twice a page's in every layer:
// kv_apply_kernel, behind it, reads how much there is from the workspace. Nothing comes back to the host.
#include "kv_pool.cuh"

namespace yscv {

int kv_check_pool(const yscv_cuda_kv_pool *p) {
    if (!p) return fail(YSCV_CUDA_ERR_BAD_ARG, "pool is null");
    if (!p->d_k || !p->d_v || !p->d_kscale || !p->d_vscale || !p->d_refs || !p->d_table || !p->d_length)
        return fail(YSCV_CUDA_ERR_BAD_ARG, "null array in the pool");
    if (p->layers == 0 || p->n_pages == 0 || p->n_kv == 0 || p->d_head == 0 || p->n_seq == 0 || p->max_pages == 0)
        return fail(YSCV_CUDA_ERR_BAD_ARG, "a size of the pool is zero");
    if (p->page != 16 && p->page != 32 && p->page != 64 && p->page != 128)
        return fail(YSCV_CUDA_ERR_UNSUPPORTED, "pages hold 16, 32, 64 or 128 tokens, got %zu", p->page);
    if (p->d_head % 16 != 0 || p->d_head > 256)
        return fail(YSCV_CUDA_ERR_UNSUPPORTED, "d_head %zu is not a multiple of 16 up to 256", p->d_head);
    if (p->n_kv > 65535 || p->layers > 65535 || p->n_pages >= (1u << 30) || p->n_seq >= (1u << 20) || p->max_pages >= (1u << 24) ||
        p->n_seq * p->max_pages >= (1u << 31) || p->max_pages * p->page >= (1u << 31))
        return fail(YSCV_CUDA_ERR_UNSUPPORTED, "a size of the pool is too large");
    if ((reinterpret_cast<uintptr_t>(p->d_k) | reinterpret_cast<uintptr_t>(p->d_v)) & 15)
        return fail(YSCV_CUDA_ERR_UNSUPPORTED, "d_k and d_v must be 16-byte aligned");
    if (!kv_aligned({p->d_kscale, p->d_vscale, p->d_refs, p->d_table, p->d_length}))
        return fail(YSCV_CUDA_ERR_UNSUPPORTED, "the pool's scales and numbers must be 4-byte aligned");
    return YSCV_CUDA_OK;
}

int kv_layer_of(const yscv_cuda_kv_pool *p, size_t layer, KvLayer *out) {
    if (layer >= p->layers) return fail(YSCV_CUDA_ERR_BAD_ARG, "layer %zu of a pool with %zu", layer, p->layers);
    const size_t heads = layer * p->n_pages * p->n_kv, bytes = heads * p->page * p->d_head;
    out->k = p->d_k + bytes;
    out->v = p->d_v + bytes;
    out->ks = p->d_kscale + heads;
    out->vs = p->d_vscale + heads;
    out->table = p->d_table;
    out->n_pages = (int)p->n_pages;
    out->n_kv = (int)p->n_kv;
    out->d = (int)p->d_head;
    out->page = (int)p->page;
    out->page_shift = p->page == 16 ? 4 : p->page == 32 ? 5 : p->page == 64 ? 6 : 7;
    out->n_seq = (int)p->n_seq;
    out->max_pages = (int)p->max_pages;
    return YSCV_CUDA_OK;
}

constexpr int KVP_THREADS = 1024, KVP_WARPS = KVP_THREADS / 32;

struct KvPages {
    int32_t *refs, *table, *length;
    int n_pages, n_seq, max_pages, page_shift;
};

// Workspace: how many copies, pages in use, pieces that copying blocks have taken, whether offsets are wrong; the copies' sources and
// destinations, the free pages that are given out, where a page went, the shared last page of a sequence
struct KvWork {
    int32_t *copies, *src, *dst, *free, *moved, *last;
};
static size_t kv_work_bytes(const yscv_cuda_kv_pool *p) {
    const size_t list = p->n_seq > p->n_pages ? p->n_seq : p->n_pages;
    return (16 + 2 * list + 2 * p->n_pages + p->n_seq) * sizeof(int32_t);
}
static KvWork kv_work_of(const yscv_cuda_kv_pool *p, void *ws) {
    const size_t list = p->n_seq > p->n_pages ? p->n_seq : p->n_pages;
    KvWork w;
    w.copies = static_cast<int32_t *>(ws);
    w.src = w.copies + 16;
    w.dst = w.src + list;
    w.free = w.dst + list;
    w.moved = w.free + p->n_pages;
    w.last = w.moved + p->n_pages;
    return w;
}

// Exclusive prefix sum over the block's threads, and the sum of all (32 bits hold the pages of all tables)
__device__ __forceinline__ long long block_prefix(long long v, uint32_t *shared, long long &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t x = (uint32_t)v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();   // (an earlier sum's readers are done)
    if (lane == 31) shared[warp] = x;
    __syncthreads();
    static_assert(KVP_WARPS == 32, "a lane a warp");
    const uint32_t w = shared[lane];
    total = __reduce_add_sync(0xffffffffu, w);
    return (long long)(__reduce_add_sync(0xffffffffu, lane < warp ? w : 0u) + x - (uint32_t)v);
}

// Which pages are used, a bit each: of the first KVP_SEEN pages in shared memory, of those behind them looked up again
constexpr int KVP_SEEN = 131072;
struct KvUsed {
    const int32_t *refs;
    uint32_t *seen;
    int n_pages;
    // word w: pages 32 w ..., a warp together
    __device__ __forceinline__ uint32_t look(int w) const {
        const int p = 32 * w + (threadIdx.x & 31);
        return __ballot_sync(0xffffffffu, p < n_pages && refs[p] > 0);
    }
    __device__ __forceinline__ uint32_t word(int w) const { return w < KVP_SEEN / 32 ? seen[w] : look(w); }
};
// A warp's run of words; how many of its pages are used
__device__ __forceinline__ void word_run(int n_pages, int &lo, int &hi) {
    const int warp = threadIdx.x >> 5, words = (n_pages + 31) / 32, per = (words + KVP_WARPS - 1) / KVP_WARPS;
    lo = min(warp * per, words);
    hi = min(lo + per, words);
}
__device__ __forceinline__ int look_at_pages(const KvUsed &u, int lo, int hi) {
    const int lane = threadIdx.x & 31;
    int n = 0;
#pragma unroll 8
    for (int w = lo; w < hi; ++w) {
        const uint32_t m = u.look(w);
        n += __popc(m);
        if (lane == 0 && w < KVP_SEEN / 32) u.seen[w] = m;
    }
    __syncwarp();
    return n;
}
// Pages of words [lo, hi) from page `from` on and below `to` in order, a warp: list(at, page) for those that are used (or free), while
// at < room
template <typename List>
__device__ __forceinline__ void list_pages(const KvUsed &u, int lo, int hi, int from, int to, bool used, long long at, long long room, const List &list) {
    const int lane = threadIdx.x & 31;
    for (int w = lo; w < hi && at < room; ++w) {
        const int p = 32 * w + lane;
        const uint32_t bits = u.word(w);
        const bool take = p >= from && p < to && ((bits >> lane) & 1u) == (used ? 1u : 0u);
        const unsigned m = __ballot_sync(0xffffffffu, take);
        const long long mine = at + __popc(m & ((1u << lane) - 1u));
        if (take && mine < room) list(mine, p);
        at += __popc(m);
    }
}
// used pages of words [lo, hi) below page `to`
__device__ __forceinline__ int used_below(const KvUsed &u, int lo, int hi, int to) {
    int n = 0;
    for (int w = lo; w < hi && 32 * w < to; ++w) n += __popc(u.word(w) & (to - 32 * w >= 32 ? 0xffffffffu : (1u << (to - 32 * w)) - 1u));
    return n;
}

// ---- extend ---------------------------------------------------------------------------------------
// Growth of a sequence but for its last page: tokens it has and gets, pages it has and will have
struct KvGrowth {
    int length, rows, held, wanted;
    bool fits, inside;             // the table has room; the offsets neither fall nor lie outside the call's rows
};
__device__ __forceinline__ KvGrowth growth_of(const KvPages &a, const int32_t *offsets, int rows, int i) {
    KvGrowth g;
    g.length = a.length[i];
    const int row0 = offsets[i], row1 = offsets[i + 1];
    g.inside = row0 >= 0 && row0 <= row1 && row1 <= rows;
    g.rows = g.inside ? row1 - row0 : 0;
    const int page = 1 << a.page_shift;
    const long long end = (long long)g.length + g.rows;
    g.fits = g.length >= 0 && end <= ((long long)a.max_pages << a.page_shift);
    g.held = g.fits ? (g.length + page - 1) >> a.page_shift : 0;
    g.wanted = g.fits ? (int)((end + page - 1) >> a.page_shift) : 0;
    return g;
}

constexpr int KVP_LISTED = 2048;   // free pages that are given out from shared memory

__global__ void __launch_bounds__(KVP_THREADS) kv_extend_kernel(const KvPages a, const int32_t *offsets, int rows,
                                                                int32_t *__restrict__ start, const KvWork w, int *__restrict__ status) {
    __shared__ uint32_t sums[KVP_WARPS];
    __shared__ uint32_t seen[KVP_SEEN / 32];
    __shared__ int listed[KVP_LISTED];
    __shared__ int copies;
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31;
    if (tid == 0) copies = 0;
    if (rows == 0) rows = offsets[a.n_seq];       // (no positions are asked for: the last offset is believed)
    // what the sequences need, in their order: a thread takes a run of them (its first one's growth and shared last page stay with it)
    const int per = (a.n_seq + KVP_THREADS - 1) / KVP_THREADS, i0 = min(tid * per, a.n_seq), i1 = min(i0 + per, a.n_seq);
    long long need = 0, wanted;
    KvGrowth first = {};
    int first_last = -1;
    bool wrong = false;
    if (i0 < i1) first = growth_of(a, offsets, rows, i0);
    const KvUsed u = {a.refs, seen, a.n_pages};
    int lo, hi;
    word_run(a.n_pages, lo, hi);
    const int used = look_at_pages(u, lo, hi);
    for (int i = i0; i < i1; ++i) {
        const KvGrowth g = i == i0 ? first : growth_of(a, offsets, rows, i);
        int last = -1;
        if (g.rows > 0 && g.fits && (g.length & ((1 << a.page_shift) - 1))) {
            const int p = a.table[(size_t)i * a.max_pages + g.held - 1];
            if (p >= 0 && p < a.n_pages && a.refs[p] > 1) last = p;
        }
        if (i == i0) first_last = last;
        else w.last[i] = last;
        if (g.rows > 0 && g.fits) need += g.wanted - g.held + (last >= 0);
        if (g.rows > 0 && !g.fits) atomicExch(status, YSCV_DEV_POS_OVERFLOW);
        if (!g.inside) {
            wrong = true;
            atomicExch(status, YSCV_DEV_BAD_NUMBER);
        }
    }
    const long long before = block_prefix(need, sums, wanted);
    // the free pages, as many as are wanted, in their order
    long long all_free;
    const int pages = max(0, min(32 * hi, a.n_pages) - 32 * lo);
    const long long free_before = block_prefix(lane == 0 ? pages - used : 0, sums, all_free);
    list_pages(u, lo, hi, 0, a.n_pages, false, __shfl_sync(0xffffffffu, free_before, 0), wanted < all_free ? wanted : all_free, [&](long long at, int p) {
        if (at < KVP_LISTED) listed[at] = p;
        else w.free[at] = p;
    });
    if (wanted > all_free && tid == 0) atomicExch(status, YSCV_DEV_NO_PAGE);
    __syncthreads();   // the list is there, and nobody reads refs as they were any more
    auto free_page = [&](long long at) { return at < KVP_LISTED ? listed[at] : w.free[at]; };
    long long upto = before;
    for (int i = i0; i < i1; ++i) {
        const KvGrowth g = i == i0 ? first : growth_of(a, offsets, rows, i);
        const int last = i == i0 ? first_last : w.last[i];
        long long at = upto;
        const int mine = g.rows > 0 && g.fits ? g.wanted - g.held + (last >= 0) : 0;
        upto += mine;
        const bool ok = g.rows > 0 && g.fits && (mine == 0 || upto <= all_free);
        start[i] = ok ? g.length : -1;
        if (!ok) continue;
        int32_t *row = a.table + (size_t)i * a.max_pages;
        if (last >= 0) {
            const int p = free_page(at++), k = atomicAdd(&copies, 1);
            w.src[k] = last;
            w.dst[k] = p;
            row[g.held - 1] = p;
            a.refs[p] = 1;
            atomicSub(a.refs + last, 1);
        }
        for (int c = g.held; c < g.wanted; ++c) {
            const int p = free_page(at++);
            row[c] = p;
            a.refs[p] = 1;
        }
        a.length[i] = g.length + g.rows;
    }
    wrong = __syncthreads_or(wrong);
    if (tid == 0) { w.copies[0] = copies; w.copies[2] = 0; w.copies[3] = wrong; }
}

// ---- compact --------------------------------------------------------------------------------------
__global__ void __launch_bounds__(KVP_THREADS) kv_compact_kernel(const KvPages a, const KvWork w) {
    __shared__ uint32_t sums[KVP_WARPS];
    __shared__ uint32_t seen[KVP_SEEN / 32];
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31;
    const KvUsed u = {a.refs, seen, a.n_pages};
    int lo, hi;
    word_run(a.n_pages, lo, hi);
    long long used, gaps, above;
    const int mine = look_at_pages(u, lo, hi);
    block_prefix(lane == 0 ? mine : 0, sums, used);
    // gaps below `used`, and as many used pages from there on
    const int mid = (int)used, below = max(0, min(32 * hi, mid) - 32 * lo), low_used = used_below(u, lo, hi, mid);
    const long long gap_at = block_prefix(lane == 0 ? below - low_used : 0, sums, gaps);
    const long long above_at = block_prefix(lane == 0 ? mine - low_used : 0, sums, above);
    list_pages(u, lo, hi, 0, mid, false, __shfl_sync(0xffffffffu, gap_at, 0), gaps, [&](long long at, int p) { w.dst[at] = p; });
    list_pages(u, lo, hi, mid, a.n_pages, true, __shfl_sync(0xffffffffu, above_at, 0), above, [&](long long at, int p) { w.src[at] = p; });
    __syncthreads();
    for (int k = tid; k < (int)gaps; k += KVP_THREADS) {
        const int s = w.src[k], d = w.dst[k];
        w.moved[s] = d;
        a.refs[d] = a.refs[s];
        a.refs[s] = 0;
    }
    if (tid == 0) { w.copies[0] = (int32_t)gaps; w.copies[1] = (int32_t)used; w.copies[2] = 0; }
}

// ---- trim and fork: a warp per list entry ---------------------------------------------------------
// The same sequence twice: an exchange gives a page to one of the two, the shorter length stays.
__global__ void __launch_bounds__(256) kv_trim_kernel(const KvPages a, const int32_t *seqs, const int32_t *keep, int count,
                                                      int *__restrict__ status) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    for (int j = blockIdx.x * 8 + (threadIdx.x >> 5); j < count; j += gridDim.x * 8) {
        const int i = seqs[j];
        if (i < 0 || i >= a.n_seq) {
            if (lane == 0) atomicExch(status, YSCV_DEV_BAD_NUMBER);
            continue;
        }
        // (the same sequence twice: each takes what lies behind the shorter of its own and what it finds)
        const int k = keep ? max(0, keep[j]) : 0, had = a.length[i], length = max(0, min(k, had)), page = 1 << a.page_shift;
        const int held = (int)(((long long)length + page - 1) >> a.page_shift);
        const int end = min(a.max_pages, (int)(((long long)max(had, 0) + page - 1) >> a.page_shift));
        if (lane == 0 && k < had) atomicMin(a.length + i, k);
        int32_t *row = a.table + (size_t)i * a.max_pages;
        for (int c = held + lane; c < end; c += 32) {
            const int p = atomicExch(row + c, -1);
            if (p >= 0 && p < a.n_pages) atomicSub(a.refs + p, 1);
        }
    }
}

// The lists are looked through for a second use of a number, so that what is left out does not depend on timing
__global__ void __launch_bounds__(256) kv_fork_kernel(const KvPages a, const int32_t *src, const int32_t *dst, int count,
                                                      int *__restrict__ status) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    for (int j = blockIdx.x * 8 + (threadIdx.x >> 5); j < count; j += gridDim.x * 8) {
        const int s = src[j], d = dst[j];
        bool bad = s < 0 || s >= a.n_seq || d < 0 || d >= a.n_seq;
        for (int o = lane; o < count; o += 32) bad |= dst[o] == s || (o < j && dst[o] == d);
        bad = __any_sync(0xffffffffu, bad);
        const int there = bad ? 0 : a.length[d], from_length = bad ? 0 : a.length[s];   // (only this warp writes to d)
        bad |= there != 0;
        if (bad) {
            if (lane == 0) atomicExch(status, YSCV_DEV_BAD_NUMBER);
            continue;
        }
        const int length = min(max(0, from_length), a.max_pages << a.page_shift);
        const int held = (int)(((long long)length + (1 << a.page_shift) - 1) >> a.page_shift);
        const int32_t *from = a.table + (size_t)s * a.max_pages;
        int32_t *to = a.table + (size_t)d * a.max_pages;
        for (int c = lane; c < held; c += 32) {
            const int p = from[c];
            to[c] = p;
            if (p >= 0 && p < a.n_pages) atomicAdd(a.refs + p, 1);
        }
        __syncwarp();
        if (lane == 0) a.length[d] = length;
    }
}

// ---- what follows: copies of pages, positions of rows, page numbers that changed -------------------
constexpr int KVP_PIECE = 16384;   // bytes a block copies at once: four loads of 16 in flight per thread

struct KvApply {
    unsigned char *k, *v;
    float *ks, *vs;
    size_t bytes;                  // of a page, keys or values
    int n_kv, layers, n_pages, n_seq;
    const int32_t *src, *dst;
    int32_t *copies;                     // null: `count` of them
    int count;
    const int32_t *offsets, *start;      // null, or the positions of `rows` rows
    int32_t *pos;
    long long rows;
    int32_t *table;                      // null, or the page numbers from copies[1] on become moved[]
    const int32_t *moved;
    long long entries;
};

// Piece t of the copies: (copy, layer, keys or values, 16 KB of the page)
__device__ __forceinline__ void copy_piece(const KvApply &a, long long t, int pieces, int *status) {
    const int tid = threadIdx.x, piece = (int)(t % pieces), which = (int)(t / pieces & 1);
    const long long cl = t / pieces >> 1;
    const int layer = (int)(cl % a.layers), c = (int)(cl / a.layers);
    const int s = a.src[c], d = a.dst[c];
    if (s < 0 || d < 0 || s == d) return;
    if (s >= a.n_pages || d >= a.n_pages) {
        if (tid == 0) atomicExch(status, YSCV_DEV_BAD_NUMBER);
        return;
    }
    unsigned char *base = (which ? a.v : a.k) + (size_t)layer * a.n_pages * a.bytes;
    const size_t at = (size_t)piece * KVP_PIECE, left = a.bytes - at;
    const uint4 *from = reinterpret_cast<const uint4 *>(base + (size_t)s * a.bytes + at);
    uint4 *to = reinterpret_cast<uint4 *>(base + (size_t)d * a.bytes + at);
    const int n = (int)((left < KVP_PIECE ? left : KVP_PIECE) / 16);
    uint4 x[KVP_PIECE / 4096];
#pragma unroll
    for (int i = 0; i < KVP_PIECE / 4096; ++i)
        if (tid + 256 * i < n) x[i] = from[tid + 256 * i];
#pragma unroll
    for (int i = 0; i < KVP_PIECE / 4096; ++i)
        if (tid + 256 * i < n) to[tid + 256 * i] = x[i];
    if (piece == 0) {
        float *scale = (which ? a.vs : a.ks) + (size_t)layer * a.n_pages * a.n_kv;
        for (int h = tid; h < a.n_kv; h += 256) scale[(size_t)d * a.n_kv + h] = scale[(size_t)s * a.n_kv + h];
    }
}

__global__ void __launch_bounds__(256) kv_apply_kernel(const KvApply a, int *__restrict__ status) {
    __shared__ long long taken[2];
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x;
    const int copies = a.copies ? a.copies[0] : a.count;
    const long long thread = (long long)blockIdx.x * 256 + tid, threads = (long long)gridDim.x * 256;
    if (a.pos) {
        const int last = a.offsets[a.n_seq];
        const bool wrong = a.copies[3] != 0;
        for (long long r = thread; r < a.rows; r += threads) {
            if (wrong) {                   // offsets in no order: the first sequence that has the row and takes part
                int i = 0;
                while (i < a.n_seq && (a.start[i] < 0 || r < a.offsets[i] || r >= a.offsets[i + 1])) ++i;
                a.pos[r] = i < a.n_seq ? a.start[i] + (int)(r - a.offsets[i]) : -1;
                continue;
            }
            int lo = 0, hi = a.n_seq;      // the last sequence whose rows begin at r or before
            while (hi - lo > 1) {
                const int m = (lo + hi) >> 1;
                if (a.offsets[m] <= r) lo = m;
                else hi = m;
            }
            const int p0 = r < last ? a.start[lo] : -1;
            a.pos[r] = p0 < 0 ? -1 : p0 + (int)(r - a.offsets[lo]);
        }
    }
    if (a.table) {
        const int used = a.copies[1];
        for (long long e = thread; copies > 0 && e < a.entries; e += threads) {
            const int p = a.table[e];
            if (p >= used && p < a.n_pages) a.table[e] = a.moved[p];
        }
    }
    const int pieces = (int)((a.bytes + KVP_PIECE - 1) / KVP_PIECE);
    const long long tasks = (long long)copies * a.layers * 2 * pieces;
    // Many pieces: a block takes another one when it is done, since SMs are not alike far from memory (1.2 GB to new places 430 us in
    // equal shares, 367 taken: the copy rate); the number of the next is asked for while this one is copied. Few: equal shares (3 a
    // block 8.9 us, 11.6 taken). A caller's own list has no counter.
    if (!a.copies || tasks < 8ll * gridDim.x) {
        for (long long t = blockIdx.x; t < tasks; t += gridDim.x) copy_piece(a, t, pieces, status);
        return;
    }
    int round = 0;
    for (long long t = blockIdx.x; t < tasks; round ^= 1) {
        if (tid == 0) taken[round] = (long long)gridDim.x + atomicAdd(a.copies + 2, 1);
        copy_piece(a, t, pieces, status);
        __syncthreads();   // (the other place of `taken` was read before the last of these)
        t = taken[round];
    }
}

static KvPages pages_of(const yscv_cuda_kv_pool *p) {
    KvPages a;
    a.refs = p->d_refs;
    a.table = p->d_table;
    a.length = p->d_length;
    a.n_pages = (int)p->n_pages;
    a.n_seq = (int)p->n_seq;
    a.max_pages = (int)p->max_pages;
    a.page_shift = p->page == 16 ? 4 : p->page == 32 ? 5 : p->page == 64 ? 6 : 7;
    return a;
}
static KvApply apply_of(const yscv_cuda_kv_pool *p) {
    KvApply a = {};
    a.k = reinterpret_cast<unsigned char *>(p->d_k);
    a.v = reinterpret_cast<unsigned char *>(p->d_v);
    a.ks = p->d_kscale;
    a.vs = p->d_vscale;
    a.bytes = p->n_kv * p->page * p->d_head;
    a.n_kv = (int)p->n_kv;
    a.layers = (int)p->layers;
    a.n_pages = (int)p->n_pages;
    a.n_seq = (int)p->n_seq;
    return a;
}
static int launch_apply(yscv_cuda_ctx *ctx, const KvApply &a, size_t most_copies) {
    const size_t pieces = (a.bytes + KVP_PIECE - 1) / KVP_PIECE, most = (size_t)8 * ctx->sm_count;
    size_t blocks = most_copies * a.layers * 2 * pieces, others = (size_t)(a.rows > a.entries ? a.rows : a.entries) / 256 + 1;
    if (blocks < others) blocks = others;
    if (blocks > most) blocks = most;
    YSCV_CUDA_TRY(launch_pdl(kv_apply_kernel, dim3((unsigned)blocks), dim3(256), 0, ctx->stream, a, ctx->d_status));
    YSCV_CUDA_TRY(cudaGetLastError());
    ctx->launches++;
    return YSCV_CUDA_OK;
}
static int check_work(const yscv_cuda_kv_pool *p, const void *ws, size_t bytes) {
    if (!ws) return fail(YSCV_CUDA_ERR_BAD_ARG, "workspace is null");
    if (bytes < kv_work_bytes(p)) return fail(YSCV_CUDA_ERR_BAD_ARG, "workspace of %zu bytes, %zu are needed", bytes, kv_work_bytes(p));
    if (reinterpret_cast<uintptr_t>(ws) & 3) return fail(YSCV_CUDA_ERR_UNSUPPORTED, "the workspace must be 4-byte aligned");
    return YSCV_CUDA_OK;
}

}  // namespace yscv

using namespace yscv;

#define KV_PROLOGUE(ctx, pool)                                     \
    if (!(ctx)) return fail(YSCV_CUDA_ERR_BAD_ARG, "ctx is null"); \
    if (const int rc_ = kv_check_pool(pool)) return rc_

extern "C" {

int yscv_cuda_kv_pages_workspace(yscv_cuda_ctx *ctx, const yscv_cuda_kv_pool *pool, size_t *bytes) {
    if (!ctx || !bytes) return fail(YSCV_CUDA_ERR_BAD_ARG, "null argument");
    if (const int rc = kv_check_pool(pool)) return rc;
    *bytes = kv_work_bytes(pool);
    return YSCV_CUDA_OK;
}

int yscv_cuda_kv_pages_extend_dev(yscv_cuda_ctx *ctx, const yscv_cuda_kv_pool *pool, const int32_t *d_offsets, size_t rows,
                                  int32_t *d_start, int32_t *d_pos, void *d_workspace, size_t workspace_bytes) {
    KV_PROLOGUE(ctx, pool);
    if (!d_offsets || !d_start || (rows > 0 && !d_pos)) return fail(YSCV_CUDA_ERR_BAD_ARG, "null operand");
    if (!kv_aligned({d_offsets, d_start, d_pos})) return fail(YSCV_CUDA_ERR_UNSUPPORTED, "operands must be 4-byte aligned");
    if (rows >= (1u << 31)) return fail(YSCV_CUDA_ERR_UNSUPPORTED, "too many rows");
    if (const int rc = check_work(pool, d_workspace, workspace_bytes)) return rc;
    YSCV_CUDA_TRY(cudaSetDevice(ctx->device));
    const KvWork w = kv_work_of(pool, d_workspace);
    YSCV_CUDA_TRY(launch_pdl(kv_extend_kernel, dim3(1), dim3(KVP_THREADS), 0, ctx->stream, pages_of(pool), d_offsets, (int)rows, d_start, w,
                             ctx->d_status));
    YSCV_CUDA_TRY(cudaGetLastError());
    ctx->launches++;
    KvApply a = apply_of(pool);
    a.src = w.src;
    a.dst = w.dst;
    a.copies = w.copies;
    a.offsets = d_offsets;
    a.start = d_start;
    a.pos = d_pos;
    a.rows = (long long)rows;
    ctx->last_kernel = "kv_pages_extend";
    return launch_apply(ctx, a, pool->n_seq);
}

int yscv_cuda_kv_pages_trim_dev(yscv_cuda_ctx *ctx, const yscv_cuda_kv_pool *pool, const int32_t *d_seqs, const int32_t *d_keep,
                                size_t count) {
    KV_PROLOGUE(ctx, pool);
    if (count == 0) return YSCV_CUDA_OK;
    if (!d_seqs) return fail(YSCV_CUDA_ERR_BAD_ARG, "null operand");
    if (!kv_aligned({d_seqs, d_keep})) return fail(YSCV_CUDA_ERR_UNSUPPORTED, "operands must be 4-byte aligned");
    if (count >= (1u << 30)) return fail(YSCV_CUDA_ERR_UNSUPPORTED, "list too long");
    YSCV_CUDA_TRY(cudaSetDevice(ctx->device));
    const unsigned blocks = (unsigned)((count + 7) / 8 < 4096 ? (count + 7) / 8 : 4096);
    YSCV_CUDA_TRY(launch_pdl(kv_trim_kernel, dim3(blocks), dim3(256), 0, ctx->stream, pages_of(pool), d_seqs, d_keep, (int)count, ctx->d_status));
    YSCV_CUDA_TRY(cudaGetLastError());
    ctx->launches++;
    ctx->last_kernel = "kv_pages_trim";
    return YSCV_CUDA_OK;
}

int yscv_cuda_kv_pages_fork_dev(yscv_cuda_ctx *ctx, const yscv_cuda_kv_pool *pool, const int32_t *d_src, const int32_t *d_dst,
                                size_t count) {
    KV_PROLOGUE(ctx, pool);
    if (count == 0) return YSCV_CUDA_OK;
    if (!d_src || !d_dst) return fail(YSCV_CUDA_ERR_BAD_ARG, "null operand");
    if (!kv_aligned({d_src, d_dst})) return fail(YSCV_CUDA_ERR_UNSUPPORTED, "operands must be 4-byte aligned");
    if (count >= (1u << 20)) return fail(YSCV_CUDA_ERR_UNSUPPORTED, "list too long");
    YSCV_CUDA_TRY(cudaSetDevice(ctx->device));
    const unsigned blocks = (unsigned)((count + 7) / 8 < 4096 ? (count + 7) / 8 : 4096);
    YSCV_CUDA_TRY(launch_pdl(kv_fork_kernel, dim3(blocks), dim3(256), 0, ctx->stream, pages_of(pool), d_src, d_dst, (int)count, ctx->d_status));
    YSCV_CUDA_TRY(cudaGetLastError());
    ctx->launches++;
    ctx->last_kernel = "kv_pages_fork";
    return YSCV_CUDA_OK;
}

int yscv_cuda_kv_pages_compact_dev(yscv_cuda_ctx *ctx, const yscv_cuda_kv_pool *pool, void *d_workspace, size_t workspace_bytes) {
    KV_PROLOGUE(ctx, pool);
    if (const int rc = check_work(pool, d_workspace, workspace_bytes)) return rc;
    YSCV_CUDA_TRY(cudaSetDevice(ctx->device));
    const KvWork w = kv_work_of(pool, d_workspace);
    YSCV_CUDA_TRY(launch_pdl(kv_compact_kernel, dim3(1), dim3(KVP_THREADS), 0, ctx->stream, pages_of(pool), w));
    YSCV_CUDA_TRY(cudaGetLastError());
    ctx->launches++;
    KvApply a = apply_of(pool);
    a.src = w.src;
    a.dst = w.dst;
    a.copies = w.copies;
    a.table = pool->d_table;
    a.moved = w.moved;
    a.entries = (long long)(pool->n_seq * pool->max_pages);
    ctx->last_kernel = "kv_pages_compact";
    return launch_apply(ctx, a, pool->n_pages);
}

int yscv_cuda_kv_pages_copy_dev(yscv_cuda_ctx *ctx, const yscv_cuda_kv_pool *pool, const int32_t *d_src, const int32_t *d_dst,
                                size_t count) {
    KV_PROLOGUE(ctx, pool);
    if (count == 0) return YSCV_CUDA_OK;
    if (!d_src || !d_dst) return fail(YSCV_CUDA_ERR_BAD_ARG, "null operand");
    if (!kv_aligned({d_src, d_dst})) return fail(YSCV_CUDA_ERR_UNSUPPORTED, "operands must be 4-byte aligned");
    if (count >= (1u << 30)) return fail(YSCV_CUDA_ERR_UNSUPPORTED, "list too long");
    YSCV_CUDA_TRY(cudaSetDevice(ctx->device));
    KvApply a = apply_of(pool);
    a.src = d_src;
    a.dst = d_dst;
    a.count = (int)count;
    ctx->last_kernel = "kv_pages_copy";
    return launch_apply(ctx, a, count);
}

}  // extern "C"
