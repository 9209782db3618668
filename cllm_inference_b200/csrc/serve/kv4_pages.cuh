// Sequences over shared pages (cllm_cuda_kv4_fork, cllm_cuda_kv4_compact).
//
// A page is in use when a sequence names it, so there is no reference count
// that could drift: each call derives what it needs from the tables.
//   mark     every page the new sequences continue: whole (shared), or the last,
//            unfinished one of a sequence, whose owner is the lowest sequence
//            that ends in it
//   plan     which sequences keep their last page, the pages each one needs,
//            their prefix sum, the free pages in order (prefix sum over the
//            bitmap), the list of copies.  The sum goes on past the pages there
//            are, so the first sequence without room and all after it get none
//   apply    the table rows, and the copies in every layer, 16 bytes a load
// The results depend on no order of execution: marks are bits and minima, and
// pages are handed out by prefix sums.
//
// What bounds the calls: the copies' bytes (read and written once) for large
// pools, launches and latency for small ones.  So where the tables fit, one
// launch does it all: every CTA derives the whole plan in shared memory, writes
// its share of the rows and copies its share of the pages, and no CTA waits for
// another.  Larger tables, and compact in place, take four launches through the
// workspace.  Forking 8 sequences of 1001 positions (8 layers) 11 us, 192 of 40 to
// 500 (4 layers) 16.7 us, where the plan and the launch are most of it; compacting
// 96 of 100 to 900 in 2048 pages of 4 layers 55 us, 5.0 TB/s read and written (78 %
// of a copy's rate).
#pragma once
#include "kv4_format.cuh"

namespace cllm {
namespace serve {

constexpr int kPlanThreads = 1024;
constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 8;  // 16-byte loads in flight per thread

struct PagesArgs {
    uint8_t* pages;
    int n_layers, n_pages, page_len, max_pages;
    int64_t page_bytes;
    const int *table, *seq_len, *source, *new_len;
    int n_old, n_new;
    int *table_out, *len_out, *n_live;
    // workspace; the first three start as all ones
    uint32_t* free_bits;   // [words] 1: no new sequence holds the page
    uint32_t* part_bits;   // [words] 1: no new sequence holds the whole page
    uint32_t* owner;       // [n_pages] lowest sequence that ends in the page
    int* ids;              // [n_pages] pages handed out / holes
    int* moved;            // [n_pages] compact: where a page goes
    int2* copies;          // [n_pages] (from, to)
    int* first;            // [n_new] first of ids that is the sequence's
    int* held;             // [n_new] pages it keeps of its source (-1: no room)
    int* count;            // copies
};

__device__ __forceinline__ int pages_of(int len, int page_len) {
    return len > 0 ? (int)(((int64_t)len + page_len - 1) / page_len) : 0;
}

// What new sequence s continues: `kept` positions of `src` and `want` in all.
__device__ __forceinline__ bool fork_request(const PagesArgs& a, int s, int* src, int* kept, int* want) {
    *src = a.source[s];
    *want = max(0, a.new_len[s]);
    *kept = 0;
    if (pages_of(*want, a.page_len) > a.max_pages) {
        *src = 0;
        return false;
    }
    if (*src < 0) {
        if (*src != -1) return false;
        *src = 0;
        return true;
    }
    if (*src >= a.n_old) {
        *src = 0;
        return false;
    }
    const int64_t most = (int64_t)a.max_pages * a.page_len;
    *kept = min(*want, (int)min(most, (int64_t)max(0, a.seq_len[*src])));
    return true;
}

// Entry of the table as a page of the pool; -1 (and the status) otherwise.
__device__ __forceinline__ int page_at(const PagesArgs& a, int s, int i) {
    const int id = a.table[(int64_t)s * a.max_pages + i];
    if ((unsigned)id < (unsigned)a.n_pages) return id;
    atomicOr(&g_serve_status, kServeBadPage);
    return -1;
}

// One launch: limits, and what a CTA holds.
constexpr int kSmallThreads = 1024, kSmallPages = 16384, kSmallSeqs = 1024, kSmallEntries = 65536, kSmallUnroll = 4;
struct SmallPlan {
    uint32_t free_bits[kSmallPages / 32], part_bits[kSmallPages / 32];
    union {
        uint32_t owner[kSmallPages];  // until the sequences know which last pages they keep
        uint16_t to[kSmallPages];     // compact: where a page goes
    };
    uint16_t ids[kSmallPages];        // free pages / holes
    int2 copies[kSmallSeqs];          // fork
    int src[kSmallSeqs], held[kSmallSeqs], want[kSmallSeqs], first[kSmallSeqs];
    int warp[32];
    int count;
};

__device__ __forceinline__ void clear_bit(uint32_t* bits, int i) {
    const uint32_t b = 1u << (i & 31);
    if (bits[i >> 5] & b) atomicAnd(bits + (i >> 5), ~b);
}

// grid (n_new, chunks of 1024 slots)
__global__ void __launch_bounds__(256) fork_mark_kernel(const PagesArgs a) {
    const int s = blockIdx.x;
    int src, kept, want;
    if (!fork_request(a, s, &src, &kept, &want)) return;
    const int whole = kept / a.page_len, n = whole + (kept % a.page_len > 0);
    for (int i = blockIdx.y * 1024 + threadIdx.x; i < min(n, ((int)blockIdx.y + 1) * 1024); i += 256) {
        const int id = page_at(a, src, i);
        if (id < 0) continue;
        clear_bit(a.free_bits, id);
        if (i < whole) clear_bit(a.part_bits, id);
        else atomicMin(a.owner + id, (uint32_t)s);
    }
}

// grid (n_seqs, chunks of 1024 slots)
__global__ void __launch_bounds__(256) compact_mark_kernel(const PagesArgs a) {
    const int s = blockIdx.x;
    const int n = min(a.max_pages, pages_of(a.seq_len[s], a.page_len));
    for (int i = blockIdx.y * 1024 + threadIdx.x; i < min(n, ((int)blockIdx.y + 1) * 1024); i += 256) {
        const int id = page_at(a, s, i);
        if (id >= 0) clear_bit(a.free_bits, id);
    }
}

// Exclusive prefix sum over the CTA; *total gets the sum.
__device__ __forceinline__ int block_scan(int v, int* s_warp, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xFFFFFFFFu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    int w = s_warp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xFFFFFFFFu, w, o);
        if (lane >= o) w += y;
    }
    *total = __shfl_sync(0xFFFFFFFFu, w, 31);
    const int before = __shfl_sync(0xFFFFFFFFu, w, max(0, warp - 1));
    return x - v + (warp ? before : 0);
}

__device__ __forceinline__ uint32_t word_mask(int n_pages, int w) {  // the bits of word w that are pages
    const int left = n_pages - 32 * w;
    return left >= 32 ? 0xFFFFFFFFu : left > 0 ? (1u << left) - 1u : 0u;
}

__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(const PagesArgs a) {
    __shared__ int s_warp[32];
    const int words = (a.n_pages + 31) / 32;
    // free pages, in order
    int room = 0;
    for (int base = 0; base < words; base += kPlanThreads) {
        const int w = base + threadIdx.x;
        uint32_t bits = w < words ? a.free_bits[w] & word_mask(a.n_pages, w) : 0u;
        int total;
        int at = room + block_scan(__popc(bits), s_warp, &total);
        for (; bits; bits &= bits - 1) a.ids[at++] = 32 * w + __ffs(bits) - 1;
        room += total;
    }
    __syncthreads();
    // pages each sequence needs, and its copy
    int given = 0, copies = 0;
    for (int base = 0; base < a.n_new; base += kPlanThreads) {
        const int s = base + threadIdx.x;
        int need = 0, held = -1, goal = 0, last = -1;
        bool fine = false, copy = false;
        if (s < a.n_new) {
            int src, kept, want;
            fine = fork_request(a, s, &src, &kept, &want);
            goal = fine ? pages_of(want, a.page_len) : 0;
            held = kept / a.page_len;
            if (kept % a.page_len) {
                last = page_at(a, src, held);
                // an id outside the pool stays in the table, where every reader finds it
                const bool keeps = last < 0 || ((a.part_bits[last >> 5] >> (last & 31) & 1u) && a.owner[last] == (uint32_t)s);
                held += keeps;
                copy = !keeps;
            }
            need = goal - held;
        }
        int total;
        const int at = given + block_scan(need, s_warp, &total);
        given += total;
        fine = fine && (int64_t)at + need <= room;
        int n;
        const int c = copies + block_scan(fine && copy, s_warp, &n);
        copies += n;
        if (fine && copy) a.copies[c] = make_int2(last, a.ids[at]);
        if (s < a.n_new) {
            a.first[s] = at;
            a.held[s] = fine ? held : -1;
        }
    }
    if (threadIdx.x == 0) *a.count = copies;
}

__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const PagesArgs a) {
    __shared__ int s_warp[32];
    const int words = (a.n_pages + 31) / 32;
    int live = 0;
    for (int base = 0; base < words; base += kPlanThreads) {
        const int w = base + threadIdx.x;
        int total;
        block_scan(w < words ? __popc(~a.free_bits[w] & word_mask(a.n_pages, w)) : 0, s_warp, &total);
        live += total;
    }
    // holes below `live`, then the pages that move into them
    int holes = 0, moves = 0;
    for (int base = 0; base < words; base += kPlanThreads) {
        const int w = base + threadIdx.x;
        const uint32_t low = w < words ? word_mask(min(live, a.n_pages), w) : 0u;
        uint32_t bits = w < words ? a.free_bits[w] & low : 0u;
        int total;
        int at = holes + block_scan(__popc(bits), s_warp, &total);
        for (; bits; bits &= bits - 1) a.ids[at++] = 32 * w + __ffs(bits) - 1;
        holes += total;
    }
    __syncthreads();
    for (int base = 0; base < words; base += kPlanThreads) {
        const int w = base + threadIdx.x;
        const uint32_t high = w < words ? word_mask(a.n_pages, w) & ~word_mask(min(live, a.n_pages), w) : 0u;
        uint32_t bits = w < words ? ~a.free_bits[w] & high : 0u;
        int total;
        int at = moves + block_scan(__popc(bits), s_warp, &total);
        for (; bits; bits &= bits - 1, ++at) {
            const int from = 32 * w + __ffs(bits) - 1, to = a.ids[at];
            a.copies[at] = make_int2(from, to);
            a.moved[from] = to;
        }
        moves += total;
    }
    if (threadIdx.x == 0) {
        *a.count = moves;
        *a.n_live = live;
    }
}

// The copies of `count` pages in every layer, CTA `cta` of `ctas`' share.
template <int THREADS, int UNROLL>
__device__ __forceinline__ void copy_pages(const PagesArgs& a, const int2* copies, int count, int cta, int ctas) {
    constexpr int kPiece = THREADS * UNROLL;  // 16-byte units of a piece
    const int64_t vecs = a.page_bytes / 16;
    const int64_t pieces = (vecs + kPiece - 1) / kPiece, all = pieces * a.n_layers * (int64_t)count;
    for (int64_t i = cta; i < all; i += ctas) {
        const int64_t page = i / pieces, at = (i - page * pieces) * kPiece + threadIdx.x;
        const int layer = (int)(page % a.n_layers);
        const int2 c = copies[page / a.n_layers];
        const uint4* from = reinterpret_cast<const uint4*>(a.pages + ((int64_t)layer * a.n_pages + c.x) * a.page_bytes);
        uint4* to = reinterpret_cast<uint4*>(a.pages + ((int64_t)layer * a.n_pages + c.y) * a.page_bytes);
        uint4 v[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (at + u * THREADS < vecs) v[u] = __ldcs(from + at + u * THREADS);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (at + u * THREADS < vecs) __stcs(to + at + u * THREADS, v[u]);
    }
}

// CTAs below n_new write a table row each, the others copy.
__global__ void __launch_bounds__(kCopyThreads) fork_apply_kernel(const PagesArgs a) {
    if ((int)blockIdx.x >= a.n_new) {
        copy_pages<kCopyThreads, kCopyUnroll>(a, a.copies, *a.count, blockIdx.x - a.n_new, gridDim.x - a.n_new);
        return;
    }
    const int s = blockIdx.x;
    int src, kept, want;
    fork_request(a, s, &src, &kept, &want);
    const int held = a.held[s], goal = held < 0 ? 0 : pages_of(want, a.page_len);
    if (threadIdx.x == 0) a.len_out[s] = held < 0 ? -1 : want;
    for (int i = threadIdx.x; i < a.max_pages; i += kCopyThreads) {
        int id = -1;
        if (i < held) id = a.table[(int64_t)src * a.max_pages + i];
        else if (i < goal) id = a.ids[a.first[s] + i - held];
        a.table_out[(int64_t)s * a.max_pages + i] = id;
    }
}

__global__ void __launch_bounds__(kCopyThreads) compact_apply_kernel(const PagesArgs a) {
    if ((int)blockIdx.x >= a.n_new) {
        copy_pages<kCopyThreads, kCopyUnroll>(a, a.copies, *a.count, blockIdx.x - a.n_new, gridDim.x - a.n_new);
        return;
    }
    const int s = blockIdx.x, n = min(a.max_pages, pages_of(a.seq_len[s], a.page_len)), live = *a.n_live;
    for (int i = threadIdx.x; i < a.max_pages; i += kCopyThreads) {
        const int64_t at = (int64_t)s * a.max_pages + i;
        int id = -1;
        if (i < n) {
            id = a.table[at];
            if (id >= live && id < a.n_pages) id = a.moved[id];
        }
        a.table_out[at] = id;
    }
}

// Exclusive prefix sum over the free (or, `used`, the used) pages of the bitmap
// from page `from` on; each(id, rank) for every one.  Returns their number.
template <class F>
__device__ __forceinline__ int each_page(const uint32_t* bits, bool used, int from, int n_pages, int* s_warp, F each) {
    int total;
    const int w = threadIdx.x;  // at most kSmallPages / 32 words
    uint32_t b = 0;
    if (32 * w < n_pages) {
        b = (used ? ~bits[w] : bits[w]) & word_mask(n_pages, w);
        b &= ~word_mask(from, w);
    }
    int at = block_scan(__popc(b), s_warp, &total);
    for (; b; b &= b - 1) each(32 * w + __ffs(b) - 1, at++);
    return total;
}

__global__ void __launch_bounds__(kSmallThreads, 1) fork_small_kernel(const PagesArgs a) {
    extern __shared__ __align__(128) uint8_t smem_raw[];
    SmallPlan& sm = *reinterpret_cast<SmallPlan*>(smem_raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int i = tid; i < kSmallPages / 32; i += kSmallThreads) sm.free_bits[i] = sm.part_bits[i] = ~0u;
    for (int i = tid; i < a.n_pages; i += kSmallThreads) sm.owner[i] = ~0u;
    bool fine = false;
    int src = 0, kept = 0, want = 0;
    if (tid < a.n_new) {
        fine = fork_request(a, tid, &src, &kept, &want);
        sm.src[tid] = src;
        sm.held[tid] = fine ? kept : 0;
        sm.want[tid] = want;
    }
    if (tid == 0) sm.count = 0;
    __syncthreads();
    for (int s = warp; s < a.n_new; s += kSmallThreads / 32) {
        const int k = sm.held[s], whole = k / a.page_len, n = whole + (k % a.page_len > 0);
        for (int i = lane; i < n; i += 32) {
            const int id = page_at(a, sm.src[s], i);
            if (id < 0) continue;
            clear_bit(sm.free_bits, id);
            if (i < whole) clear_bit(sm.part_bits, id);
            else atomicMin(sm.owner + id, (uint32_t)s);
        }
    }
    __syncthreads();
    const int room = each_page(sm.free_bits, false, 0, a.n_pages, sm.warp, [&](int id, int rank) { sm.ids[rank] = (uint16_t)id; });
    int need = 0, held = 0, last = -1;
    bool copy = false;
    if (tid < a.n_new) {
        held = kept / a.page_len;
        if (kept % a.page_len) {
            last = page_at(a, src, held);
            const bool keeps = last < 0 || ((sm.part_bits[last >> 5] >> (last & 31) & 1u) && sm.owner[last] == (uint32_t)tid);
            held += keeps;
            copy = !keeps;
        }
        need = (fine ? pages_of(want, a.page_len) : 0) - held;
        if (!fine) need = 0;
    }
    int total;
    const int at = block_scan(need, sm.warp, &total);
    fine = fine && (int64_t)at + need <= room;
    const int c = block_scan(fine && copy, sm.warp, &total);
    if (tid < a.n_new) {
        if (fine && copy) sm.copies[c] = make_int2(last, sm.ids[at]);
        sm.first[tid] = at;
        sm.held[tid] = fine ? held : -1;
    }
    __syncthreads();
    for (int s = blockIdx.x * (kSmallThreads / 32) + warp; s < a.n_new; s += gridDim.x * (kSmallThreads / 32)) {
        const int h = sm.held[s], goal = h < 0 ? 0 : pages_of(sm.want[s], a.page_len);
        if (lane == 0) a.len_out[s] = h < 0 ? -1 : sm.want[s];
        for (int i = lane; i < a.max_pages; i += 32) {
            int id = -1;
            if (i < h) id = a.table[(int64_t)sm.src[s] * a.max_pages + i];
            else if (i < goal) id = sm.ids[sm.first[s] + i - h];
            a.table_out[(int64_t)s * a.max_pages + i] = id;
        }
    }
    copy_pages<kSmallThreads, kSmallUnroll>(a, sm.copies, total, blockIdx.x, gridDim.x);
}

__global__ void __launch_bounds__(kSmallThreads, 1) compact_small_kernel(const PagesArgs a) {
    extern __shared__ __align__(128) uint8_t smem_raw[];
    SmallPlan& sm = *reinterpret_cast<SmallPlan*>(smem_raw);
    int2* moves = reinterpret_cast<int2*>(sm.copies);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int i = tid; i < kSmallPages / 32; i += kSmallThreads) sm.free_bits[i] = ~0u;
    if (tid < a.n_new) sm.held[tid] = min(a.max_pages, pages_of(a.seq_len[tid], a.page_len));
    __syncthreads();
    for (int s = warp; s < a.n_new; s += kSmallThreads / 32)
        for (int i = lane; i < sm.held[s]; i += 32) {
            const int id = page_at(a, s, i);
            if (id >= 0) clear_bit(sm.free_bits, id);
        }
    __syncthreads();
    const int live = each_page(sm.free_bits, true, 0, a.n_pages, sm.warp, [](int, int) {});
    each_page(sm.free_bits, false, 0, min(live, a.n_pages), sm.warp, [&](int id, int rank) { sm.ids[rank] = (uint16_t)id; });
    __syncthreads();
    const int count = each_page(sm.free_bits, true, live, a.n_pages, sm.warp, [&](int id, int rank) { sm.to[id] = sm.ids[rank]; });
    __syncthreads();
    if (tid == 0 && blockIdx.x == 0) *a.n_live = live;
    for (int s = blockIdx.x * (kSmallThreads / 32) + warp; s < a.n_new; s += gridDim.x * (kSmallThreads / 32))
        for (int i = lane; i < a.max_pages; i += 32) {
            int id = -1;
            if (i < sm.held[s]) {
                id = a.table[(int64_t)s * a.max_pages + i];
                if (id >= live && id < a.n_pages) id = sm.to[id];
            }
            a.table_out[(int64_t)s * a.max_pages + i] = id;
        }
    // the moves, as many at a time as the list holds
    for (int base = 0; base < count; base += kSmallSeqs) {
        __syncthreads();
        each_page(sm.free_bits, true, live, a.n_pages, sm.warp, [&](int id, int rank) {
            if (rank >= base && rank < base + kSmallSeqs) moves[rank - base] = make_int2(id, sm.ids[rank]);
        });
        __syncthreads();
        copy_pages<kSmallThreads, kSmallUnroll>(a, moves, min(kSmallSeqs, count - base), blockIdx.x, gridDim.x);
    }
}

}  // namespace serve
}  // namespace cllm
