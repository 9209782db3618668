// Attention of many rows per sequence over the 4-bit cache
// (cllm_cuda_kv4_attention; prompts): a CTA takes 128 rows (tokens x heads of one
// KV head) over all the positions they see, 64 at a time, on tcgen05 tensor cores.
//
// The bits of fp32 from fp16 operands: q, k, p and v enter as hi + lo (22 bits
// together), and a product is lo*hi + hi*lo + hi*hi, in that order, the small
// terms first because the tensor cores cut off as they add.  lo*lo is left out:
// up to 2^-21 of a product, with a sign of its own since q and p are split to the
// nearest.  For the same reason
// a tile's p v is not accumulated in TMEM over the whole sequence but added to
// fp32 registers, rounded to nearest, tile by tile; that also does the rescaling.
// k and v of a tile are scaled by a power of two that brings its largest value to
// [2^10, 2^11), so that lo stays above fp16's subnormals.  S takes the keys' out.
// The values' stays in the fp32 sums, of weights as of weighted values, and a
// tile's rescaling brings them to its power: p is not touched by it, and the largest
// weight is 2^10 to 2^14 whatever the values are, so a weight keeps its 22 bits down to
// 2^-12 of it and is no further off than 2^-35 of it below that.  One position 17.5
// nats above 8000 others, of small value: off by 8e-7 of the output's largest value
// (fp32 arithmetic 6e-7).
//
// What bounds it: three products a term, 6 * 128 * 64 * HD multiply-adds a tile
// for 128 x 64 scores: 1536 cycles of the tensor cores (HD 128), beside which the
// CTA's four schedulers issue 2100 instructions each (numbers to fp16, softmax,
// sums), and shared memory moves 96 KB of operands to the tensor cores and 64 KB
// from the numbers: q and p come from TMEM, or the operands alone would take all
// of its bandwidth.  A tile takes 3600 cycles, in which the schedulers issue 59 %
// of what they could and the tensor cores work 44 %: 1024 tokens of 32 heads over
// 8 on 8000 positions 417 to 428 us, 294 to 301 TFLOP/s counted once, three times
// that in products (53 % of a plain bf16 GEMM's rate).  Each role is busy some 70 %
// of the time and waits for the others in turn.  Most instructions turn keys and
// values into operands, which every CTA does for its own 128 rows: here 32 CTAs do
// the same ones.
//
// Work: tiles of (sequence, KV head, 128 rows), numbered through by
// prompt_plan_kernel and cut into equal runs, one per SM; a run that ends inside an
// item leaves a partial result, and the CTA whose part of an item comes last adds
// them up in order (9 sequences of 5 to 2500 positions, two of them prompts of 65
// and 99 rows, while these were this kernel's: 36 us with that, 46 with a kernel of
// its own).
//
// Warps (5 warpgroups; registers moved to where they are needed):
//   0       raw tiles of the pages into a ring (bulk copies)
//   1       TMEM, and the one thread that issues the products
//   4..7    a row each: softmax with a running reference (kv4_decode.cuh), p to TMEM
//   8..11   a row each: the fp32 sums of p v, and the output
//   12..15  the keys' numbers and scales to fp16 operands in the 128-byte swizzle
//   16..19  the values'
// All waits are bounded; one that expires sets the status, and the CTA runs to its
// end without waiting.
#pragma once
#include <type_traits>

#include "../tc_ptx.cuh"
#include "kv4_decode.cuh"

namespace cllm {
namespace serve {

constexpr int kPromptThreads = 640;
// An item costs as much again as kPromptUnits tiles: 256 rows of 32 heads over 8 on
// 4096 positions at 1, 3, 6: 61, 59, 57 us, 512 rows 74, 72, 68.  A run has
// kPromptMinRun units or more; 16 instead: 70 and 72 us for 59 and 72 (at 3 units).
constexpr int kPromptUnits = 6;
constexpr int kPromptMinRun = 6;
constexpr int kPromptRows = 128, kPromptCols = 64;
constexpr int kRawStages = 3;
constexpr int kStats = 8;  // the operands' warps are at most 7 tiles ahead of the softmax (raw ring, then theirs)

template <int HD>
struct PromptSmem {
    static constexpr uint32_t kOperand = kPromptCols * HD * 2;  // bytes of a tile's k (or v), hi or lo
    uint8_t k[2][2][kOperand];  // [stage][hi, lo]: [64 values][position][128 bytes]
    uint8_t v[2][2][kOperand];  // [stage][hi, lo]: [value][128 bytes of positions]
    uint8_t raw[kRawStages][4 * Tile<HD>::kBytes];
    float2 k_scale[4][Tile<HD>::G][kTile];    // [raw tile][group][position] (d, m), scaled
    float v_scale[4][Tile<HD>::G][2][kTile];  // [raw tile][group][d, m][position]
    float alpha[4][kPromptRows];  // what a tile's new reference leaves of the sums
    float sum[2][kPromptRows], ref[2][kPromptRows];  // of an item: its rows' sums of weights and references
    float down[2];                                   // and what takes the values' power out of its sums
    uint32_t bad[2][kPromptRows];                    // groups that a NaN of the values reaches
    struct Stat {
        float k_down, v_up;  // 2^-(the keys' power), 2^(the values' power)
        int v_power;
        uint32_t bad;        // 1: a value has a NaN
    } stat[kStats];
    uint32_t top[2][kStats][4];  // [keys, values][tile][warp]: largest exponent
    uint32_t warp_bad[kStats][4];
    uint8_t nan[kStats][kPromptCols];  // groups of a position that are NaN
    uint64_t raw_full[kRawStages], raw_empty[kRawStages];
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2], o_empty[2];
    uint64_t alpha_full[4], stat_full[kStats], q_full, done;
    uint32_t tmem;
    int abort;
    int join[2];
};

// One lane of the warp.  The compiler knows that a branch on this has one thread
// and passes the products' operands straight to uniform registers; behind a
// comparison of the lane number it loops over lanes for each of them (1024 tokens
// on 8000 positions: 886 us instead of 669).
__device__ __forceinline__ bool elect_one() {
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xFFFFFFFF;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok));
    return ok != 0;
}
// One product step, A in TMEM, B the shared-memory operand at byte `at` (128-byte
// swizzle; the descriptor's upper half is a constant, its lower the address / 16).
// Few instructions: one thread issues 36 of these per tile.
__device__ __forceinline__ void tc_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t at, uint32_t idesc, bool accumulate) {
    constexpr uint32_t kHigh = (uint32_t)(1024 >> 4) | (1u << 14) | (2u << 29);
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 b;\n mov.b64 b, {%2, %5};\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n}\n" ::"r"(d_tmem),
        "r"(a_tmem), "r"((at >> 4) | (1u << 16)), "r"(idesc), "r"((uint32_t)accumulate), "r"(kHigh)
        : "memory");
}
__device__ __forceinline__ void tmem_st16u(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void sts128u(uint32_t a, const uint32_t (&v)[4]) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}

// Wait as one thread; false once a wait of the CTA has expired.
__device__ __forceinline__ bool wait_or_abort(uint32_t bar, uint32_t parity, volatile int* abort) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = global_timer_ns();
    for (uint32_t it = 1;; ++it) {
        if (mbar_try_wait_long(bar, parity)) return true;
        if ((it & 15u) == 0) {
            if (*abort) return false;
            if (global_timer_ns() - t0 > kWaitLimitNs) {
                atomicOr(&g_serve_status, kServeTimeout);
                *abort = 1;
                return false;
            }
        }
    }
}
__device__ __forceinline__ void warp_wait(uint32_t bar, uint32_t parity, volatile int* abort) {
    if ((threadIdx.x & 31) == 0) wait_or_abort(bar, parity, abort);
    __syncwarp();
}
// Wait as a warpgroup: its first warp polls, the others sleep in hardware barrier
// ID (four polling warps took a third of the SM's issue slots and fetches).
template <int ID>
__device__ __forceinline__ void group_wait(uint32_t bar, uint32_t parity, volatile int* abort) {
    if (((threadIdx.x >> 5) & 3) == 0) warp_wait(bar, parity, abort);
    asm volatile("bar.sync %0, 128;" ::"n"(ID) : "memory");
}
__device__ __forceinline__ void warp_arrive(uint32_t bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// Two values as an fp16 pair and what is left of them as another: hi is the value
// cut to 11 bits, so lo holds the next 11.  For keys and values, whose tile's largest
// is 2^10 or more: what lies below fp16's normal range, where hi's conversion is not
// exact, is 2^-24 of it.  Queries and weights are split to the nearest (split2).
__device__ __forceinline__ void split_pair(float2 x, uint32_t& hi, uint32_t& lo) {
    const float2 h = make_float2(__uint_as_float(__float_as_uint(x.x) & 0xFFFFE000u), __uint_as_float(__float_as_uint(x.y) & 0xFFFFE000u));
    const float2 l = add2(x, make_float2(-h.x, -h.y));
    hi = h2bits(__floats2half2_rn(h.x, h.y));
    lo = h2bits(__floats2half2_rn(l.x, l.y));
}

// 128 rows of a sequence, for every KV head: its tiles per head, and where its units begin.
struct PromptItem {
    int seq, block, tiles, pad;
    int64_t unit;  // units (tiles + kPromptUnits, times KV heads) of the items before it
};
struct PromptArgs {
    AttnArgs a;
    int most;            // room for items
    PromptItem* items;   // [most + 1]; the last one's unit is the total
    int* seq_items;      // [n_seqs] scratch
    int* count;          // items
    int ctas;
    unsigned* arrived;   // [ctas] parts of the item that begins in CTA c that are there; the plan clears it
    float* part_ml;      // [2 * ctas][128][2]
    uint32_t* part_bad;  // [2 * ctas][128]
    float* part_o;       // [2 * ctas][HD / 4][128][4]
};

__device__ __forceinline__ int prompt_tiles(int len, int n, int rep, int block) {
    const int last = (int)(min((int64_t)(block + 1) * kPromptRows, (int64_t)n * rep) - 1) / rep;  // token of the last row
    return (max(0, len - (n - 1 - last)) + kPromptCols - 1) / kPromptCols;
}

// The list of items, one CTA: items per sequence, their prefix sum, then the
// tiles of each and theirs.
constexpr int kPromptPlanThreads = 1024;
__global__ void __launch_bounds__(kPromptPlanThreads) prompt_plan_kernel(const PromptArgs p) {
    __shared__ int64_t s_warp[32];
    const AttnArgs& a = p.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto scan = [&](int64_t v, int64_t* total) -> int64_t {  // exclusive
        int64_t x = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xFFFFFFFFu, x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 31) s_warp[warp] = x;
        __syncthreads();
        int64_t w = s_warp[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xFFFFFFFFu, w, o);
            if (lane >= o) w += y;
        }
        *total = __shfl_sync(0xFFFFFFFFu, w, 31);
        const int64_t before = __shfl_sync(0xFFFFFFFFu, w, max(0, warp - 1));
        return x - v + (warp ? before : 0);
    };
    for (int i = threadIdx.x; i < p.ctas; i += kPromptPlanThreads) p.arrived[i] = 0;
    int64_t count = 0, steps = 0;
    for (int s = threadIdx.x; s < a.c.n_seqs; s += kPromptPlanThreads) steps += seq_steps(a, s);
    scan(steps, &steps);
    const int limit = rows_limit(a, steps);
    for (int base = 0; base < a.c.n_seqs; base += kPromptPlanThreads) {
        const int s = base + threadIdx.x;
        int64_t blocks = 0, total;
        if (s < a.c.n_seqs) {
            int begin, n;
            seq_rows(a, s, &begin, &n);
            const int64_t rows = (int64_t)n * a.rep;
            if (rows > limit) blocks = (rows + kPromptRows - 1) / kPromptRows;
        }
        const int64_t at = count + scan(blocks, &total);
        if (s < a.c.n_seqs) p.seq_items[s] = (int)min(at, (int64_t)p.most);
        count += total;
    }
    count = min(count, (int64_t)p.most);
    __syncthreads();
    int64_t units = 0;
    for (int64_t base = 0; base < count; base += kPromptPlanThreads) {
        const int i = (int)base + threadIdx.x;
        PromptItem it{};
        int64_t mine = 0, total;
        if (i < count) {
            int lo = 0, hi = a.c.n_seqs - 1;  // the last sequence whose first item is at most i
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (p.seq_items[mid] <= i) lo = mid;
                else hi = mid - 1;
            }
            int begin, n;
            seq_rows(a, lo, &begin, &n);
            it.seq = lo;
            it.block = i - p.seq_items[lo];
            it.tiles = prompt_tiles(a.c.length(lo), n, a.rep, it.block);
            mine = (int64_t)(it.tiles + kPromptUnits) * a.c.n_kv;
        }
        it.unit = units + scan(mine, &total);
        if (i < count) p.items[i] = it;
        units += total;
    }
    if (threadIdx.x == 0) {
        p.items[count].unit = units;
        *p.count = (int)count;
    }
}

// A place in the numbered units.
struct PromptCursor {
    int item, kvh, unit, tiles;
    int64_t left;
    // Step over what the run has of this item; its tiles are [*from, *to).
    __device__ __forceinline__ void range(int* from, int* to) const {
        *from = max(0, unit - kPromptUnits);
        *to = max(0, (int)min((int64_t)unit + left, (int64_t)tiles + kPromptUnits) - kPromptUnits);
    }
    __device__ __forceinline__ void next(const PromptArgs& p) {
        left -= tiles + kPromptUnits - unit;
        unit = 0;
        if (left > 0 && ++kvh == p.a.c.n_kv) {
            kvh = 0;
            tiles = p.items[++item].tiles;
        }
    }
    // Whether the run has something of this item to do: a tile of it, or an item without any.
    __device__ __forceinline__ bool here(int from, int to) const { return from < to || (tiles == 0 && unit == 0); }
};

// The parts of an item, added in their order whichever CTA does it: thread =
// row, 64 values at a time, so that 16 loads are in flight.  Other CTAs wrote
// them during this kernel: read past L1.
template <int HD>
__device__ __forceinline__ void prompt_join(const PromptArgs& p, int c0, int parts, const PromptItem& item, int begin, int n,
                                            int kvh, int row) {
    const AttnArgs& a = p.a;
    auto ml = [&](int i) {
        return __ldcg(reinterpret_cast<const float2*>(p.part_ml) + (int64_t)part_slot(c0, i) * kPromptRows + row);
    };
    float m = -3.0e38f, sum = 0.f;
    uint32_t bad = 0;
#pragma unroll 4
    for (int i = 0; i < parts; ++i) m = fmaxf(m, ml(i).x);
    const int j = item.block * kPromptRows + row;
    const bool live = j < n * a.rep;
    const int64_t at = (int64_t)(begin + j / a.rep) * a.n_head + kvh * a.rep + j % a.rep;
#pragma unroll 1
    for (int h = 0; h < HD; h += 64) {
        float4 x[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = make_float4(0.f, 0.f, 0.f, 0.f);
        sum = 0.f;
#pragma unroll 1
        for (int i = 0; i < parts; ++i) {
            const float4* from = reinterpret_cast<const float4*>(p.part_o) +
                                 ((int64_t)part_slot(c0, i) * (HD / 4) + h / 4) * kPromptRows + row;
            float4 y[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) y[e] = __ldcg(from + e * kPromptRows);
            const float2 z = ml(i);
            bad |= __ldcg(p.part_bad + (int64_t)part_slot(c0, i) * kPromptRows + row);
            const float k = exp2_fast(z.x - m);
            sum = fmaf(k, z.y, sum);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                x[e].x = fmaf(k, y[e].x, x[e].x); x[e].y = fmaf(k, y[e].y, x[e].y);
                x[e].z = fmaf(k, y[e].z, x[e].z); x[e].w = fmaf(k, y[e].w, x[e].w);
            }
        }
        if (!live) continue;
        const float inv = sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float by = bad >> (h / 32 + e / 8) & 1 ? NAN : inv;
            *reinterpret_cast<float4*>(a.out + at * HD + h + 4 * e) =
                sum == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(x[e].x * by, x[e].y * by, x[e].z * by, x[e].w * by);
        }
    }
    if (live && a.lse) a.lse[at] = sum == 0.f ? -INFINITY : 0.69314718055994530942f * (m + log2f(sum));
}

template <int HD>
__global__ void __launch_bounds__(kPromptThreads, 1) kv4_prompt_kernel(const PromptArgs p) {
    constexpr int G = Tile<HD>::G;
    constexpr uint32_t kIdescS = (1u << 4) | ((uint32_t)(kPromptCols >> 3) << 17) | ((uint32_t)(kPromptRows >> 4) << 24);
    constexpr uint32_t kIdescO = (1u << 4) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(kPromptRows >> 4) << 24);
    constexpr uint32_t kColQ = 0, kColS = 128, kColO = 256;  // TMEM: q hi | lo; two S, 16 scores overwritten by p hi | lo; two O
    extern __shared__ __align__(128) uint8_t smem_raw[];
    PromptSmem<HD>& sm = *reinterpret_cast<PromptSmem<HD>*>(smem_raw + (-smem_addr(smem_raw) & 1023u));
    const AttnArgs& a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* abort = &sm.abort;
    auto bar = [](uint64_t& b) { return smem_addr(&b); };

    // this CTA's run of the units
    const int count = *p.count;
    const int64_t all = count ? p.items[count].unit : 0;
    const int ctas = (int)min((int64_t)gridDim.x, (all + kPromptMinRun - 1) / kPromptMinRun);
    if ((int)blockIdx.x >= ctas) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    const int64_t run0 = blockIdx.x * all / ctas, run1 = (blockIdx.x + 1) * all / ctas;
    PromptCursor cur;
    {
        int lo = 0, hi = count - 1;  // the last item that begins at or before run0
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (p.items[mid].unit <= run0) lo = mid;
            else hi = mid - 1;
        }
        cur.item = lo;
        cur.tiles = p.items[lo].tiles;
        const int64_t at = run0 - p.items[lo].unit;
        cur.kvh = (int)(at / (cur.tiles + kPromptUnits));
        cur.unit = (int)(at - (int64_t)cur.kvh * (cur.tiles + kPromptUnits));
        cur.left = run1 - run0;
    }

    if (threadIdx.x == 0) {
        for (int i = 0; i < kRawStages; ++i) {
            mbar_init(bar(sm.raw_full[i]), 1);
            mbar_init(bar(sm.raw_empty[i]), 8);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(sm.k_full[i]), 4);
            mbar_init(bar(sm.k_empty[i]), 1);
            mbar_init(bar(sm.v_full[i]), 4);
            mbar_init(bar(sm.v_empty[i]), 1);
            mbar_init(bar(sm.s_full[i]), 1);
            mbar_init(bar(sm.p_full[i]), 4);
            mbar_init(bar(sm.o_full[i]), 1);
            mbar_init(bar(sm.o_empty[i]), 4);
        }
        for (int i = 0; i < 4; ++i) mbar_init(bar(sm.alpha_full[i]), 4);
        for (int i = 0; i < kStats; ++i) mbar_init(bar(sm.stat_full[i]), 2);
        mbar_init(bar(sm.q_full), 4);
        mbar_init(bar(sm.done), 1);
        sm.abort = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&sm.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&sm.tmem);

    // Every role walks the same run; `it` counts its tiles, and barrier phases go by it.
    int it = 0, from, to;
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 0) {
            // ---- raw tiles
            for (; cur.left > 0; cur.next(p)) {
                cur.range(&from, &to);
                if (from >= to) continue;
                const int seq = p.items[cur.item].seq, len = a.c.length(seq);
                for (int i = from; i < to && !*abort; ++i) {
                    const int st = it % kRawStages, tile = 4 * i + lane;
                    const bool there = lane < 4 && tile * kTile < len;
                    const uint8_t* src = a.nan_tile;
                    if (there) {
                        const int slot = a.page_of(tile);
                        const int id = a.c.page(seq, slot);
                        if (id >= 0)
                            src = a.c.pages + (((int64_t)id * a.c.n_kv + cur.kvh) * a.page_tiles + (tile - slot * a.page_tiles)) * Tile<HD>::kBytes;
                    }
                    if (it >= kRawStages) warp_wait(bar(sm.raw_empty[st]), (uint32_t)(it / kRawStages - 1) & 1u, abort);
                    const uint32_t n = __popc(__ballot_sync(0xFFFFFFFFu, there));
                    const int dead = __shfl_sync(0xFFFFFFFFu, *abort, 0);
                    if (dead) break;
                    if (lane == 0) mbar_arrive_expect_tx(bar(sm.raw_full[st]), n * Tile<HD>::kBytes);
                    __syncwarp();
                    if (there) bulk_g2s(smem_addr(sm.raw[st]) + lane * Tile<HD>::kBytes, src, Tile<HD>::kBytes, bar(sm.raw_full[st]));
                    ++it;
                }
            }
            if (*abort)  // let the copies in flight land
                for (int i = max(0, it - kRawStages); i < it; ++i) wait_full(bar(sm.raw_full[i % kRawStages]), (uint32_t)(i / kRawStages) & 1u);
        } else if (warp == 1 && elect_one()) {
            // ---- products: S of a tile, then O of the one before it
            using Smem = PromptSmem<HD>;
            const uint32_t k0 = smem_addr(sm.k), v0 = smem_addr(sm.v);
            auto values = [&](int j) {
                const int st = j & 1;
                wait_or_abort(bar(sm.p_full[st]), (uint32_t)(j >> 1) & 1u, abort);
                wait_or_abort(bar(sm.v_full[st]), (uint32_t)(j >> 1) & 1u, abort);
                if (j >= 2) wait_or_abort(bar(sm.o_empty[st]), (uint32_t)((j >> 1) - 1) & 1u, abort);
                tc_fence_after();
                const uint32_t d = tmem + kColO + 128 * st;
                const uint32_t w = tmem + kColS + 64 * st, v = v0 + st * (2 * Smem::kOperand);
#pragma unroll 1
                for (int term = 0; term < 3; ++term)  // lo hi, hi lo, hi hi
#pragma unroll
                    for (int s = 0; s < kPromptCols / 16; ++s)
                        tc_mma_ts(d, w + (term == 0 ? 8 : 0) + 16 * s, v + (term == 1 ? Smem::kOperand : 0) + s * 32, kIdescO, term | s);
                tc_commit(bar(sm.o_full[st]));
                tc_commit(bar(sm.v_empty[st]));
            };
            for (int items = 0; cur.left > 0; cur.next(p)) {
                cur.range(&from, &to);
                if (!cur.here(from, to)) continue;
                wait_or_abort(bar(sm.q_full), (uint32_t)(items++) & 1u, abort);
                tc_fence_after();
                for (int i = from; i < to; ++i, ++it) {
                    // S goes into the buffer that the products of p two tiles ago, issued before, have read
                    const int st = it & 1;
                    wait_or_abort(bar(sm.k_full[st]), (uint32_t)(it >> 1) & 1u, abort);
                    tc_fence_after();
                    const uint32_t d = tmem + kColS + 64 * st;
                    const uint32_t q = tmem + kColQ, k = k0 + st * (2 * Smem::kOperand);
#pragma unroll 1
                    for (int term = 0; term < 3; ++term)
#pragma unroll
                        for (int s = 0; s < HD / 16; ++s)
                            tc_mma_ts(d, q + (term == 0 ? HD / 2 : 0) + 8 * s,
                                      k + (term == 1 ? Smem::kOperand : 0) + (s / 4) * (kPromptCols * 128) + (s % 4) * 32, kIdescS,
                                      term | s);
                    tc_commit(bar(sm.s_full[st]));
                    tc_commit(bar(sm.k_empty[st]));
                    if (i > from) values(it - 1);
                }
                if (from < to) values(it - 1);
            }
            tc_commit(bar(sm.done));
            wait_full(bar(sm.done), 0);
        }
    } else if (warp < 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
        // ---- softmax: thread = row
        const int row = 32 * (warp - 4) + lane;
        const uint32_t lanes = (uint32_t)(32 * (warp - 4)) << 16;
        const bool vec = ((reinterpret_cast<uintptr_t>(a.q) | (a.ldq * 4)) & 15) == 0;
        for (int items = 0; cur.left > 0; cur.next(p)) {
            cur.range(&from, &to);
            if (!cur.here(from, to)) continue;
            const int seq = p.items[cur.item].seq, j = p.items[cur.item].block * kPromptRows + row, len = a.c.length(seq);
            int begin, n;
            seq_rows(a, seq, &begin, &n);
            const bool on = j < n * a.rep;
            const int sees = on ? max(0, len - (n - 1 - j / a.rep)) : 0;
            const float* src = a.q + (int64_t)(begin + j / a.rep) * a.ldq + (cur.kvh * a.rep + j % a.rep) * HD;
            float f_log2;
            {
                float top = 0.f;
                if (on) {
                    if (vec) {
                        for (int i = 0; i < HD; i += 4) {
                            const float4 x = *reinterpret_cast<const float4*>(src + i);
                            top = fmaxf(fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(x.z), fabsf(x.w)));
                        }
                    } else {
                        for (int i = 0; i < HD; ++i) top = fmaxf(top, fabsf(src[i]));
                    }
                }
                const int e = min(max((int)(__float_as_uint(top) >> 23), 30), 230);
                // the row's largest value to [2^9, 2^10), with the sign of the scale, so that f_log2 is not negative
                const float up = copysignf(__uint_as_float((uint32_t)(263 - e) << 23), a.scale);
                f_log2 = fabsf(a.scale) * 1.44269504088896340736f * __uint_as_float((uint32_t)(e - 9) << 23);
#pragma unroll 1
                for (int i = 0; i < HD; i += 32) {
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int k = 0; k < 32; k += 4) {
                        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (on) {
                            if (vec) x = *reinterpret_cast<const float4*>(src + i + k);
                            else x = make_float4(src[i + k], src[i + k + 1], src[i + k + 2], src[i + k + 3]);
                        }
                        split2(x.x * up, x.y * up, &hi[k / 2], &lo[k / 2]);
                        split2(x.z * up, x.w * up, &hi[k / 2 + 1], &lo[k / 2 + 1]);
                    }
                    tmem_st16u(tmem + lanes + kColQ + i / 2, hi);
                    tmem_st16u(tmem + lanes + kColQ + HD / 2 + i / 2, lo);
                }
                tmem_st_wait();
                tc_fence_before();
                warp_arrive(bar(sm.q_full));
            }
            float ref = -3.0e38f, l = 0.f;
            int power = 0;  // of the values in the sums
            uint32_t bad = 0;
            // EDGE: some row of the warp does not see all of the tile (a copy of its own, or every tile pays the selects)
            auto tile = [&](auto edge, int i) {
                constexpr bool EDGE = decltype(edge)::value;
                const int st = it & 1, r4 = it & 3, rs = it % kStats;
                if (warp == 4) warp_wait(bar(sm.stat_full[rs]), (uint32_t)(it / kStats) & 1u, abort);
                group_wait<4>(bar(sm.s_full[st]), (uint32_t)(it >> 1) & 1u, abort);
                tc_fence_after();
                const float f = f_log2 * sm.stat[rs].k_down, v_up = sm.stat[rs].v_up;
                const int change = sm.stat[rs].v_power - power;
                power += change;
                const uint32_t col = tmem + lanes + kColS + 64 * st;
                const int limit = sees - i * kPromptCols;  // columns that the row sees
                if (sm.stat[rs].bad)
                    for (int c = 0; c < min(limit, kPromptCols); ++c) bad |= sm.nan[rs][c];
                float top = -INFINITY;
#pragma unroll 1
                for (int c = 0; c < kPromptCols; c += 16) {
                    uint32_t x[16];
                    tmem_ld16_issue(col + c, x);
                    tmem_ld_wait(x);
                    float m = -INFINITY;
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        if (!EDGE || c + k < limit) m = fmaxf(m, __uint_as_float(x[k]));
                    }
                    top = fmaxf(top, m);
                }
                top *= f;
                float alpha = __uint_as_float((uint32_t)(127 + change) << 23);
                if (top > ref + 14.f) {
                    const float now = top - 10.f;
                    alpha *= exp2_fast(ref - now);
                    ref = now;
                }
                sm.alpha[r4][row] = alpha;
                const float off = -ref;
                const float2 f2 = make_float2(f, f), off2 = make_float2(off, off);
                float2 sum = make_float2(0.f, 0.f);
#pragma unroll 1
                for (int c = 0; c < kPromptCols; c += 16) {  // 16 weights, hi in 8 columns and lo in 8, in place of their scores
                    uint32_t x[16], w[16];
                    tmem_ld16_issue(col + c, x);
                    tmem_ld_wait(x);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float2 e = __ffma2_rn(make_float2(__uint_as_float(x[2 * k]), __uint_as_float(x[2 * k + 1])), f2, off2);
                        float2 y = make_float2(exp2_fast(e.x), exp2_fast(e.y));
                        if (EDGE && c + 2 * k >= limit) y.x = 0.f;
                        if (EDGE && c + 2 * k + 1 >= limit) y.y = 0.f;
                        sum = add2(sum, y);
                        split2(y.x, y.y, &w[k], &w[8 + k]);
                    }
                    tmem_st16u(col + c, w);
                }
                l = fmaf(sum.x + sum.y, v_up, l * alpha);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(bar(sm.alpha_full[r4]));
                    mbar_arrive(bar(sm.p_full[st]));
                }
            };
            const int plain = min(to, __reduce_min_sync(0xFFFFFFFFu, on ? sees : INT_MAX) / kPromptCols);  // no rows past the end
#pragma unroll 1
            for (int i = from; i < plain; ++i, ++it) tile(std::false_type{}, i);
#pragma unroll 1
            for (int i = max(from, plain); i < to; ++i, ++it) tile(std::true_type{}, i);
            const int slot = items++ & 1;
            sm.sum[slot][row] = l;
            sm.ref[slot][row] = ref;
            if (row == 0) sm.down[slot] = __uint_as_float((uint32_t)(127 - power) << 23);
            sm.bad[slot][row] = bad;
            asm volatile("bar.sync 2, 256;" ::: "memory");
        }
    } else if (warp < 12) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
        // ---- sums: thread = row
        const int row = 32 * (warp - 8) + lane;
        const uint32_t lanes = (uint32_t)(32 * (warp - 8)) << 16;
        for (int items = 0; cur.left > 0; cur.next(p)) {
            cur.range(&from, &to);
            if (!cur.here(from, to)) continue;
            float2 acc[HD / 2];
#pragma unroll
            for (int i = 0; i < HD / 2; ++i) acc[i] = make_float2(0.f, 0.f);
#pragma unroll 1
            for (int i = from; i < to; ++i, ++it) {
                const int st = it & 1, r4 = it & 3;
                if (warp == 8) warp_wait(bar(sm.alpha_full[r4]), (uint32_t)(it >> 2) & 1u, abort);
                group_wait<5>(bar(sm.o_full[st]), (uint32_t)(it >> 1) & 1u, abort);
                tc_fence_after();
                const float alpha = sm.alpha[r4][row];
                const uint32_t col = tmem + lanes + kColO + 128 * st;
                const float2 keep = make_float2(alpha, alpha);
                uint32_t x[2][16];
                tmem_ld16_issue(col, x[0]);
#pragma unroll
                for (int c = 0; c < HD / 16; ++c) {
                    tmem_ld_wait(x[c & 1]);
                    if (c + 1 < HD / 16) tmem_ld16_issue(col + 16 * (c + 1), x[(c + 1) & 1]);
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        acc[8 * c + k] = __ffma2_rn(acc[8 * c + k], keep,
                                                    make_float2(__uint_as_float(x[c & 1][2 * k]), __uint_as_float(x[c & 1][2 * k + 1])));
                }
                tc_fence_before();
                warp_arrive(bar(sm.o_empty[st]));
            }
            asm volatile("bar.sync 2, 256;" ::: "memory");
            const PromptItem item = p.items[cur.item];
            int begin, n;
            seq_rows(a, item.seq, &begin, &n);
            const int j = item.block * kPromptRows + row;
            const float sum = sm.sum[items & 1][row], ref = sm.ref[items & 1][row], down = sm.down[items & 1];
            const uint32_t bad = sm.bad[items & 1][row];
            if (to - from == item.tiles) {
                if (j < n * a.rep) {
                    const int64_t at = (int64_t)(begin + j / a.rep) * a.n_head + cur.kvh * a.rep + j % a.rep;
                    const float inv = sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);
                    float* out = a.out + at * HD;
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const float by = bad >> g & 1 ? NAN : inv;
#pragma unroll
                        for (int i = 16 * g; i < 16 * g + 16; i += 2)
                            *reinterpret_cast<float4*>(out + 2 * i) =
                                sum == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                                           : make_float4(acc[i].x * by, acc[i].y * by, acc[i + 1].x * by, acc[i + 1].y * by);
                    }
                    if (a.lse) a.lse[at] = sum == 0.f ? -INFINITY : 0.69314718055994530942f * (ref + log2f(sum * down));
                }
            } else {
                const int slot = 2 * blockIdx.x + (from == 0 ? 1 : 0);
                float4* out = reinterpret_cast<float4*>(p.part_o) + (int64_t)slot * (kPromptRows * HD / 4) + row;
#pragma unroll
                for (int i = 0; i < HD / 2; i += 2)
                    out[i / 2 * kPromptRows] = make_float4(acc[i].x * down, acc[i].y * down, acc[i + 1].x * down, acc[i + 1].y * down);
                *reinterpret_cast<float2*>(p.part_ml + 2 * (slot * kPromptRows + row)) = make_float2(ref, sum * down);
                p.part_bad[slot * kPromptRows + row] = bad;
                // the CTA whose part is the last to come joins them
                asm volatile("bar.sync 5, 128;" ::: "memory");
                if (row == 0) {
                    const int64_t unit0 = item.unit + (int64_t)cur.kvh * (item.tiles + kPromptUnits);
                    const int c0 = run_of(unit0 + kPromptUnits, ctas, all);
                    const int c1 = run_of(unit0 + kPromptUnits + item.tiles - 1, ctas, all);
                    __threadfence();
                    const bool last = atomicAdd(&p.arrived[c0], 1u) == (unsigned)(c1 - c0);
                    __threadfence();
                    sm.join[0] = last ? c1 - c0 + 1 : 0;
                    sm.join[1] = c0;
                }
                asm volatile("bar.sync 5, 128;" ::: "memory");
                if (sm.join[0]) prompt_join<HD>(p, sm.join[1], sm.join[0], item, begin, n, cur.kvh, row);
            }
            ++items;
        }
    } else if (warp < 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        // ---- keys to operands: warp w has the 16 positions of raw tile w
        const int w = warp - 12, tid = threadIdx.x - 384;
        for (; cur.left > 0; cur.next(p)) {
            cur.range(&from, &to);
            if (from >= to) continue;
            const int len = a.c.length(p.items[cur.item].seq);
#pragma unroll 1
            for (int i = from; i < to; ++i, ++it) {
                const int rs = it % kRawStages, st = it & 1, si = it % kStats;
                group_wait<1>(bar(sm.raw_full[rs]), (uint32_t)(it / kRawStages) & 1u, abort);
                const uint32_t raw = smem_addr(sm.raw[rs]), tile = raw + w * Tile<HD>::kBytes;
                // the largest exponent: a value is below 2^(e - 14) for e = max(exponent of m, exponent of d + 4)
                uint32_t sc[G], e = 0;
                const int pos = lane & 15;
                const bool live = i * kPromptCols + w * kTile + pos < len;
                lds_words<G>(tile + Tile<HD>::kScaleK + pos * (HD / 8), sc);
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    if (!live) sc[g] = 0u;
                    const uint32_t d = sc[g] >> 10 & 31, m = sc[g] >> 26 & 31;
                    if (max(d, m) < 31) e = max(e, max(m, d + 4));
                }
                e = __reduce_max_sync(0xFFFFFFFFu, e);
                if (lane == 0) sm.top[0][si][w] = e;
                asm volatile("bar.sync 1, 128;" ::: "memory");
                e = max(max(sm.top[0][si][0], sm.top[0][si][1]), max(sm.top[0][si][2], sm.top[0][si][3]));
                const int power = min(14, 25 - (int)e);  // the largest value to [2^10, 2^11)
                if (tid == 0) {
                    sm.stat[si].k_down = __uint_as_float((uint32_t)(127 - power) << 23);
                    mbar_arrive(bar(sm.stat_full[si]));
                }
                // a NaN stays one (its scores are NaN)
                if (lane < 16)
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const float up = __uint_as_float((uint32_t)(127 + power) << 23);
                        const float2 dm = __half22float2(bits_h2(sc[g]));
                        sm.k_scale[w][g][pos] = make_float2(dm.x * up, dm.y * up);
                    }
                __syncwarp();
                if (it >= 2) group_wait<1>(bar(sm.k_empty[st]), (uint32_t)((it >> 1) - 1) & 1u, abort);
                const int row = w * kTile + pos;
                const uint32_t hi_at = smem_addr(sm.k[st][0]) + row * 128, lo_at = smem_addr(sm.k[st][1]) + row * 128;
#pragma unroll 2
                for (int c = 0; c < 2 * G; ++c) {  // a word of eight numbers is a 16-byte chunk of the operand's row
                    const int t = 2 * (lane >> 4) + c / G, g = c % G;
                    const uint32_t word = lds32(tile + pos * (HD / 2) + t * (HD / 8) + 4 * g);
                    const float2 dm = sm.k_scale[w][g][pos], d = make_float2(dm.x, dm.x), m = make_float2(dm.y, dm.y);
                    float2 n[4];  // numbers j and j + 4
#pragma unroll
                    for (int j = 0; j < 4; ++j) n[j] = __half22float2(bits_h2(numbers<false>(word >> (4 * j), 0.f)));
                    uint32_t hi[4], lo[4];
                    split_pair(__ffma2_rn(make_float2(n[0].x, n[1].x), d, m), hi[0], lo[0]);
                    split_pair(__ffma2_rn(make_float2(n[2].x, n[3].x), d, m), hi[1], lo[1]);
                    split_pair(__ffma2_rn(make_float2(n[0].y, n[1].y), d, m), hi[2], lo[2]);
                    split_pair(__ffma2_rn(make_float2(n[2].y, n[3].y), d, m), hi[3], lo[3]);
                    const uint32_t at = (g >> 1) * (kPromptCols * 128) + ((((g & 1) * 4 + t) ^ (row & 7)) << 4);
                    sts128u(hi_at + at, hi);
                    sts128u(lo_at + at, lo);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(bar(sm.k_full[st]));
                    mbar_arrive(bar(sm.raw_empty[rs]));
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        // ---- values to operands: a lane has a column r of 8 positions and half of the groups
        constexpr int NG = G / 2;
        const int w = warp - 16, tid = threadIdx.x - 512, r = lane & 7, q = lane >> 3 & 1, h = lane >> 4;
        for (; cur.left > 0; cur.next(p)) {
            cur.range(&from, &to);
            if (from >= to) continue;
            const int len = a.c.length(p.items[cur.item].seq);
#pragma unroll 1
            for (int i = from; i < to; ++i, ++it) {
                const int rs = it % kRawStages, st = it & 1, si = it % kStats;
                group_wait<3>(bar(sm.raw_full[rs]), (uint32_t)(it / kRawStages) & 1u, abort);
                const uint32_t raw = smem_addr(sm.raw[rs]), tile = raw + w * Tile<HD>::kBytes;
                const int here = len - i * kPromptCols - w * kTile;  // positions of this tile that are stored
                const int pos = lane & 15;
                uint32_t sc[G];
                {
                    uint32_t e = 0, nan = 0;
                    lds_words<G>(tile + Tile<HD>::kScaleV + pos * (HD / 8), sc);
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const uint32_t d = sc[g] >> 10 & 31, m = sc[g] >> 26 & 31;
                        if (pos >= here) {
                            sc[g] = 0u;
                        } else if (max(d, m) < 31) {
                            e = max(e, max(m, d + 4));
                        } else {  // must not reach the sums of the rows that do not see it
                            nan |= 1u << g;
                            sc[g] = 0u;
                        }
                    }
                    e = __reduce_max_sync(0xFFFFFFFFu, e);
                    const bool any = __any_sync(0xFFFFFFFFu, nan != 0);
                    if (lane < 16) sm.nan[si][w * kTile + pos] = (uint8_t)nan;
                    if (lane == 0) {
                        sm.top[1][si][w] = e;
                        sm.warp_bad[si][w] = any;
                    }
                }
                asm volatile("bar.sync 3, 128;" ::: "memory");
                const uint32_t e = max(max(sm.top[1][si][0], sm.top[1][si][1]), max(sm.top[1][si][2], sm.top[1][si][3]));
                const int power = 25 - (int)e;
                if (tid == 0) {
                    sm.stat[si].v_up = __uint_as_float((uint32_t)(127 + power) << 23);
                    sm.stat[si].v_power = power;
                    sm.stat[si].bad = sm.warp_bad[si][0] | sm.warp_bad[si][1] | sm.warp_bad[si][2] | sm.warp_bad[si][3];
                    mbar_arrive(bar(sm.stat_full[si]));
                }
                if (lane < 16)
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const float up = __uint_as_float((uint32_t)(127 + power) << 23);
                        const float2 dm = __half22float2(bits_h2(sc[g]));
                        sm.v_scale[w][g][0][pos] = dm.x * up;
                        sm.v_scale[w][g][1][pos] = dm.y * up;
                    }
                __syncwarp();
                if (it >= 2) group_wait<3>(bar(sm.v_empty[st]), (uint32_t)((it >> 1) - 1) & 1u, abort);
                uint32_t num[8];
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    const uint32_t at = tile + Tile<HD>::kV + ((x % 4) / 2) * (4 * HD) + (r * 4 + 2 * q + x / 4) * (HD / 8) +
                                        (x & 1) * (HD / 16) + h * (HD / 32);
                    num[x] = HD == 128 ? lds32(at) : lds16(at);
                }
#pragma unroll 1
                for (int g = 0; g < NG; ++g) {
                    float2 d[4], m[4];
                    uint32_t pair[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        d[x] = *reinterpret_cast<const float2*>(&sm.v_scale[w][h * NG + g][0][8 * q + 2 * x]);
                        m[x] = *reinterpret_cast<const float2*>(&sm.v_scale[w][h * NG + g][1][8 * q + 2 * x]);
                    }
                    const uint32_t sel = g ? 0x7632u : 0x5410u;
#pragma unroll
                    for (int x = 0; x < 4; ++x) pair[x] = __byte_perm(num[2 * x], num[2 * x + 1], sel);
#pragma unroll 2
                    for (int c = 0; c < 4; ++c) {  // eight positions of one value are a 16-byte chunk
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const float2 n = __half22float2(bits_h2(numbers<false>(pair[x] >> (4 * c), 0.f)));
                            split_pair(__ffma2_rn(n, d[x], m[x]), hi[x], lo[x]);
                        }
                        const uint32_t at = (32 * (h * NG + g) + 8 * c + r) * 128 + (((2 * w + q) ^ r) << 4);
                        sts128u(smem_addr(sm.v[st][0]) + at, hi);
                        sts128u(smem_addr(sm.v[st][1]) + at, lo);
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(bar(sm.v_full[st]));
                    mbar_arrive(bar(sm.raw_empty[rs]));
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    // This kernel may have begun before kv4_rows_kernel, of which it needs nothing, was done; what follows both waits
    // for this one.
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

}  // namespace serve
}  // namespace cllm
