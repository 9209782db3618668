// Attention of a few rows per sequence over the 4-bit cache
// (cllm_cuda_kv4_attention; generated tokens).
//
// What bounds it: every stored byte is read once and serves rep query heads
// with 4 * rep * head_dim operations a position: the HBM stream, were it not for
// the instructions.  At 6.4 TB/s an SM gets a tile of 16 positions every 110
// cycles (head_dim 128), in which its four schedulers issue 440 instructions: the
// numbers must reach the tensor cores with very few of them.  This takes 520 a
// tile (8 rows), and the schedulers issue in half of the cycles: each warp is one
// chain of loads, conversions, products and weights, and the registers that it
// holds allow three warps a scheduler.  64 sequences of 150 to 8190 positions, 64
// heads over 8, 67.8 us, 2.5 TB/s; one of 131071, 32 over 8, 67.7 us, 2.5 TB/s
// (38 % of a copy's rate).
//
// * Numbers become fp16 two at a time: (w & 0x000F000F) | 0x64006400 is the pair
//   (1024 + n, 1024 + n'), and one fused operation takes the 1024 off (and the 16
//   of a number that sits in the next four bits): two instructions a pair.
//   Subnormals (the bare four bits) would save one of them, but the tensor cores
//   align products by the exponents of the operands' encodings and cut off what
//   lies 24 bits below: 37 positions were off by 7e-6, 131071 by 4e-4.
// * Scales outside.  q.k = sum over groups of d_g (q . n)_g + m_g sum(q)_g: one
//   accumulator per group, multiplied by d_g in fp32, and one more product whose
//   operand is the scale words themselves (k index 2g is d_g, met by a zero, 2g + 1
//   is m_g, met by sum(q)_g).  sum p v = (p d) . (n - 8) + p . (m + 8 d): around the
//   middle of the numbers, because p d n alone adds up to many times the result
//   and every instruction cuts off towards zero; m + 8 d is an exact fp16 pair.
// * The bits of fp32.  The query rows (and p, p d) enter as fp16 hi + lo in the two
//   halves of the instruction's 16 rows, 22 bits together, rounded to the nearest:
//   with at most 8 rows of one KV head the second half would be empty anyway.  hi
//   and lo of p d come from three fp16 operations: hi = p_hi d, lo = fma(p_lo, d,
//   fma(p_hi, d, -hi)).  Of the last digits of small ones see below.
// * The tensor cores add up the 32 positions of a step only; their sums are added
//   to the result in fp32, rounded to nearest.
// * No number changes lanes.  The tile's order gives each lane its operands of a
//   16 x head_dim tile in two 16-byte loads, for keys and for values, and the
//   score a lane computes is the p that the same lane needs as an operand.
// * The running reference (in place of the maximum) of a row moves only when a
//   score exceeds it by 2^14, so the accumulators are hardly ever rescaled.
// * The values' scales get a power of two, which the accumulators carry, that brings
//   the largest one so far below 2 and to 2^-3 or more: a p of at most 2^14 then keeps
//   p d inside fp16.  fp16's last digit is 2^-24, so beside a largest weight of 2^10 or
//   more a p is off by 2^-35 of it at most, beyond its 22 bits, and a p d by that much of
//   a scale of 1: small weights count beside a dominating one however small the values
//   are.  Scales of 2^-3 to 2 need no power and take no time.  One position 17.5 nats
//   above 8000 others, of small value: off by 9e-7 of the output's largest value (fp32
//   arithmetic 6e-7), and by 3e-6 where the values are of 0.0004.
// * Work: steps of 128 positions of (sequence, KV head, 8 rows), numbered through
//   (and some for the item itself) and cut into equal runs, one per CTA,
//   whatever the lengths are.  A CTA's four
//   warps take two tiles each, from a ring of their own that one lane fills with
//   bulk copies across the runs' borders.  Three stages of the ring leave room for
//   two CTAs an SM only, which is slower (below).
// * A run that ends inside an item leaves a partial result; the CTA whose part of
//   an item comes last adds them up in order (64 sequences: 6 us less than a second
//   kernel's launch and its chain of loads).
#pragma once
#include "kv4_format.cuh"

namespace cllm {
namespace serve {

constexpr int kRowWarps = 4;
constexpr int kRowThreads = 32 * kRowWarps;
constexpr int kRowStages = 2;               // pairs of tiles in a warp's ring
constexpr int kRowTile = 8;                 // query rows of an item
constexpr int kPairLen = 2 * kTile;         // positions of a warp's step
constexpr int kStepLen = kPairLen * kRowWarps;
constexpr int kRowCtasPerSm = 3;            // of 168 registers a thread: 64 sequences 67.6 us, 2 of 255 registers 73.3
constexpr int kMaxRowCtas = 640;

struct AttnArgs {
    const float* q;
    int64_t ldq;
    const int* q_begin;  // nullptr: row s belongs to sequence s
    int n_tok, n_head, rep;
    int rows_max;        // sequences with more rows * rep are the prompt kernel's,
    int all_steps;       // but not in a call of at most so many steps in all
    float scale;
    float *out, *lse;
    Cache c;
    const uint8_t* nan_tile;  // g_nan_tile
    int page_tiles;        // tiles of a page and head
    uint32_t page_magic;   // ceil(2^32 / page_tiles), 0 where that is 2^32
    // Slot of the page that holds a tile (< 2^27): the product is at most one too large.
    __device__ __forceinline__ int page_of(int tile) const {
        if (page_magic == 0) return tile;
        const int s = (int)__umulhi((uint32_t)tile, page_magic);
        return s * page_tiles > tile ? s - 1 : s;
    }
};

// An item that lies in several CTAs' runs has a part in each.  CTA c keeps the
// part that the item begins with in slot 2c + 1, another's continuation in 2c.
struct RowsArgs {
    AttnArgs a;
    int set;         // of g_rows_arrived, that this call counts in
    float* part_ml;  // [2 * ctas][kRowTile][2] reference (log2) and sum
    float* part_o;   // [2 * ctas][kRowTile][HD]
};
// Parts of the item that begins in CTA c that are there.  The last one to come
// sets it back to 0.  Calls take the two sets in turn, and each clears the other
// one: a wrong count (of calls that overlapped, which their caller must not let
// happen) does not reach later calls.  A captured call has the same set in every
// replay; in a graph with one such call a wrong count stays until a call outside of it.
__device__ unsigned g_rows_arrived[2][kMaxRowCtas];

// CTA whose run has unit u: runs begin at floor(c * all / ctas).
__device__ __forceinline__ int run_of(int64_t u, int ctas, int64_t all) { return (int)(((u + 1) * ctas - 1) / all); }
__device__ __forceinline__ int part_slot(int c0, int i) { return i ? 2 * (c0 + i) : 2 * c0 + 1; }  // part i of c0's item

// ---- rows of a sequence -------------------------------------------------------

__device__ __forceinline__ void seq_rows(const AttnArgs& a, int s, int* begin, int* n) {
    if (!a.q_begin) {
        *begin = s;
        *n = 1;
        return;
    }
    const int b = min(max(a.q_begin[s], 0), a.n_tok), e = min(max(a.q_begin[s + 1], 0), a.n_tok);
    *begin = b;
    *n = max(0, e - b);
}

// What a sequence asks of this kernel: items (0: nothing) of `steps` steps
// each.  An item costs as much again as kItemUnits steps (its queries, the
// warps' results put together), so it counts steps + kItemUnits units (64
// sequences of 150 to 8190 positions: 1 70.6 us, 2 67.6, 4 71.7).
constexpr int kItemUnits = 2;
struct SeqWork {
    int begin, n, len, items, steps;
    __device__ __forceinline__ int units() const { return steps + kItemUnits; }
    __device__ __forceinline__ int step(int unit) const { return max(0, unit - kItemUnits); }
};
__device__ __forceinline__ SeqWork seq_work(const AttnArgs& a, int s, int limit) {
    SeqWork w;
    seq_rows(a, s, &w.begin, &w.n);
    w.items = 0;
    w.steps = 1;
    w.len = 0;
    const int64_t rows = (int64_t)w.n * a.rep;
    if (rows == 0 || rows > limit) return w;
    w.len = a.c.length(s);
    w.items = a.c.n_kv * (int)((rows + kRowTile - 1) / kRowTile);
    w.steps = max(1, (w.len + kStepLen - 1) / kStepLen);  // one even for no positions: its rows are zeros
    return w;
}

// Steps of a sequence if this kernel took it, at most all_steps + 1.  The rows
// up to which it takes sequences follow from their sum.
__device__ __forceinline__ int64_t seq_steps(const AttnArgs& a, int s) {
    int begin, n;
    seq_rows(a, s, &begin, &n);
    const int64_t groups = ((int64_t)n * a.rep + kRowTile - 1) / kRowTile, most = (int64_t)a.all_steps + 1;
    if (groups >= most) return most;
    return min(most, groups * a.c.n_kv * max(1, (a.c.length(s) + kStepLen - 1) / kStepLen));
}
__device__ __forceinline__ int rows_limit(const AttnArgs& a, int64_t steps) { return steps <= a.all_steps ? INT_MAX : a.rows_max; }

// A place in the numbered units.
struct Cursor {
    int s, item, unit, left;  // left: units up to the end of this CTA's run
    SeqWork w;
    __device__ __forceinline__ void next(const AttnArgs& a, int units, const volatile int* limit) {  // over `units` units inside the item
        left -= units;
        unit += units;
        if (unit < w.units()) return;
        unit = 0;
        if (++item < w.items) return;
        item = 0;
        while (left > 0 && s + 1 < a.c.n_seqs) {
            w = seq_work(a, ++s, limit ? *limit : INT_MAX);
            if (w.items) return;
        }
    }
};

__device__ __forceinline__ int64_t cta_scan(int64_t v, int64_t* s_warp, int64_t* total) {  // exclusive, kRowThreads threads
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xFFFFFFFFu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    int64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
        before += w < warp ? s_warp[w] : 0;
        all += s_warp[w];
    }
    __syncthreads();
    *total = all;
    return before + x - v;
}

// ---- instructions ---------------------------------------------------------------

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The product alone (accumulator 0).
__device__ __forceinline__ void mma16816_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t h2bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t b) { return *reinterpret_cast<__half2*>(&b); }
// (x, y) = hi + lo, each an fp16 pair, to 22 bits
__device__ __forceinline__ void split2(float x, float y, uint32_t* hi, uint32_t* lo) {
    const uint32_t h = h2bits(__floats2half2_rn(x, y));
    const uint32_t minus = h ^ 0x80008000u;
    float ex, ey;  // x - hi, exact
    asm("add.rn.f32.f16 %0, %1, %2;" : "=f"(ex) : "h"((unsigned short)minus), "f"(x));
    asm("add.rn.f32.f16 %0, %1, %2;" : "=f"(ey) : "h"((unsigned short)(minus >> 16)), "f"(y));
    *hi = h;
    *lo = h2bits(__floats2half2_rn(ex, ey));
}
// The numbers in bits 0-3 (UP: 4-7) of both halves of w, plus `off`, as an fp16 pair.
template <bool UP>
__device__ __forceinline__ uint32_t numbers(uint32_t w, float off) {
    uint32_t x;
    if constexpr (UP) {
        asm("lop3.b32 %0, %1, 0x00F000F0, 0x64006400, 0xEA;" : "=r"(x) : "r"(w));
        return h2bits(__hfma2(bits_h2(x), __float2half2_rn(0.0625f), __float2half2_rn(off - 64.f)));
    }
    asm("lop3.b32 %0, %1, 0x000F000F, 0x64006400, 0xEA;" : "=r"(x) : "r"(w));
    return h2bits(__hadd2(bits_h2(x), __float2half2_rn(off - 1024.f)));
}
// The exact sum of two fp16 pairs as a pair of fp16 pairs.
__device__ __forceinline__ void sum2(__half2 a, __half2 b, uint32_t* hi, uint32_t* lo) {
    const __half2 s = __hadd2(a, b), x = __hsub2(s, a);
    *hi = h2bits(s);
    *lo = h2bits(__hadd2(__hsub2(a, __hsub2(s, x)), __hsub2(b, x)));
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}
template <int W>
__device__ __forceinline__ void lds_words(uint32_t a, uint32_t (&w)[W]) {
    if constexpr (W == 4) {
        const uint4 v = lds128(a);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else {
        const uint2 v = lds64(a);
        w[0] = v.x; w[1] = v.y;
    }
}
// mbarrier.try_wait that suspends the thread for up to about 2 us: a warp that
// polls takes issue slots and instruction fetches from the ones it waits for.
__device__ __forceinline__ bool mbar_try_wait_long(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(2000u)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool wait_full(uint32_t bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = global_timer_ns();
    for (uint32_t it = 1;; ++it) {
        if (mbar_try_wait_long(bar, parity)) return true;
        if ((it & 15u) == 0 && global_timer_ns() - t0 > kWaitLimitNs) {
            atomicOr(&g_serve_status, kServeTimeout);
            return false;
        }
    }
}

template <int HD>
struct RowsSmem {
    static constexpr int kLd = HD + 8;  // row stride of the merge buffer: no two rows of a half warp in one bank
    uint8_t ring[kRowWarps][kRowStages][2 * Tile<HD>::kBytes];
    uint4 qa[HD / 16][32];  // the query rows as operands: a k step of 16, a lane
    uint32_t qs[2][32];     // and their groups' sums
    float o[kRowWarps][kRowTile][kLd];
    float ml[kRowWarps][kRowTile][2];
    uint64_t full[kRowWarps][kRowStages];
    int64_t scan[kRowWarps];
    int start[3], limit;
};

// A place in a warp's ring.
struct Stage {
    uint32_t i = 0, parity = 0;
    __device__ __forceinline__ void next() {
        if (++i == kRowStages) {
            i = 0;
            parity ^= 1u;
        }
    }
};
// A lane's offset into a tile, computed once: without this it is computed again for every tile.
__device__ __forceinline__ uint32_t keep(uint32_t x) {
    asm volatile("" : "+r"(x));
    return x;
}

// Column r of a score tile i (and row of a values' operand) is this position of the tile: lane t of
// a row group then holds the positions 4t .. 4t+3, whose scale rows lie in different banks for all t.
__device__ __forceinline__ int tile_pos(int i, int r) { return 4 * (r >> 1) + 2 * i + ((r & 1) ^ (r >> 2)); }

// ---- the parts of an item ------------------------------------------------------------

// Added in their order, whichever CTA does it.  A lane has four values of a row.
// Other CTAs wrote them during this kernel: read past L1.
template <int HD>
__device__ __forceinline__ void rows_join(const RowsArgs& ra, int c0, int parts, const SeqWork& w, int kvh, int row0) {
    constexpr int kLanes = HD / 4, kPass = kRowWarps * (32 / kLanes), kPasses = kRowTile / kPass;
    const AttnArgs& a = ra.a;
    const int d = threadIdx.x % kLanes, r0 = threadIdx.x / kLanes;
    float m[kPasses], sum[kPasses];
    float4 x[kPasses];
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        m[p] = -3.0e38f;
        sum[p] = 0.f;
        x[p] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    auto ml = [&](int i, int p) {
        return __ldcg(reinterpret_cast<const float2*>(ra.part_ml) + (int64_t)part_slot(c0, i) * kRowTile + r0 + p * kPass);
    };
#pragma unroll 1
    for (int i = d; i < parts; i += kLanes)
#pragma unroll
        for (int p = 0; p < kPasses; ++p) m[p] = fmaxf(m[p], ml(i, p).x);
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1)
#pragma unroll
        for (int p = 0; p < kPasses; ++p) m[p] = fmaxf(m[p], __shfl_xor_sync(0xFFFFFFFFu, m[p], o));
#pragma unroll 1
    for (int base = 0; base < parts; base += kLanes) {
        float k[kPasses];  // the weight of part base + d
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
            const float2 z = base + d < parts ? ml(base + d, p) : make_float2(-INFINITY, 0.f);
            k[p] = exp2_fast(z.x - m[p]);
            sum[p] = fmaf(k[p], z.y, sum[p]);
        }
        const int n = min(kLanes, parts - base);
#pragma unroll 8
        for (int i = 0; i < n; ++i)
#pragma unroll
            for (int p = 0; p < kPasses; ++p) {
                const float4 y = __ldcg(reinterpret_cast<const float4*>(
                    ra.part_o + ((int64_t)part_slot(c0, base + i) * kRowTile + r0 + p * kPass) * HD + 4 * d));
                const float by = __shfl_sync(0xFFFFFFFFu, k[p], i, kLanes);
                x[p].x = fmaf(by, y.x, x[p].x); x[p].y = fmaf(by, y.y, x[p].y);
                x[p].z = fmaf(by, y.z, x[p].z); x[p].w = fmaf(by, y.w, x[p].w);
            }
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1)
#pragma unroll
        for (int p = 0; p < kPasses; ++p) sum[p] += __shfl_xor_sync(0xFFFFFFFFu, sum[p], o);
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        const int row = row0 + r0 + p * kPass;
        if (row >= w.n * a.rep) break;
        const int64_t at = (int64_t)(w.begin + row / a.rep) * a.n_head + kvh * a.rep + row % a.rep;
        const float inv = sum[p] == 0.f ? 0.f : __fdiv_rn(1.f, sum[p]);
        *reinterpret_cast<float4*>(a.out + at * HD + 4 * d) =
            sum[p] == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(x[p].x * inv, x[p].y * inv, x[p].z * inv, x[p].w * inv);
        if (a.lse && d == 0) a.lse[at] = sum[p] == 0.f ? -INFINITY : 0.69314718055994530942f * (m[p] + log2f(sum[p]));
    }
}

// ---- the kernel --------------------------------------------------------------------

// ALL: every sequence is this kernel's (no limit to look up: 64 sequences 67.6 us
// instead of 69.0).
template <int HD, bool ALL>
__global__ void __launch_bounds__(kRowThreads, kRowCtasPerSm) kv4_rows_kernel(const RowsArgs ra) {
    constexpr int G = Tile<HD>::G;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    RowsSmem<HD>& sm = *reinterpret_cast<RowsSmem<HD>*>(smem_raw);
    const AttnArgs& a = ra.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the prompt kernel needs nothing of this one
    const uint32_t full = smem_addr(sm.full[warp]), ring = smem_addr(sm.ring[warp]);
    if (lane == 0) {
        for (int i = 0; i < kRowStages; ++i) mbar_init(full + 8 * i, 1);
        fence_mbar_init();
    }
    // rows of no sequence
    if (a.q_begin) {
        const int b = min(max(a.q_begin[0], 0), a.n_tok), e = max(b, min(a.q_begin[a.c.n_seqs], a.n_tok));
        for (int i = blockIdx.x; i < b + a.n_tok - e; i += gridDim.x) {
            const int64_t row = i < b ? i : e + i - b;
            for (int j = threadIdx.x; j < a.n_head * HD; j += kRowThreads) a.out[row * a.n_head * HD + j] = 0.f;
            if (a.lse)
                for (int j = threadIdx.x; j < a.n_head; j += kRowThreads) a.lse[row * a.n_head + j] = -INFINITY;
        }
    }
    // all units, and this CTA's run of them
    const int per = (a.c.n_seqs + kRowThreads - 1) / kRowThreads;
    const int s0 = min(a.c.n_seqs, (int)threadIdx.x * per), s1 = min(a.c.n_seqs, s0 + per);
    int64_t mine = 0, all;
    int limit = INT_MAX;
    const volatile int* limit_at = ALL ? nullptr : &sm.limit;
    if (!ALL) {
        for (int s = s0; s < s1; ++s) mine += seq_steps(a, s);
        cta_scan(mine, sm.scan, &all);
        limit = rows_limit(a, all);
        mine = 0;
        if (threadIdx.x == 0) sm.limit = limit;
    }
    for (int s = s0; s < s1; ++s) {
        const SeqWork w = seq_work(a, s, limit);
        mine += (int64_t)w.items * w.units();
    }
    const int64_t before = cta_scan(mine, sm.scan, &all);
    const int ctas = (int)min((int64_t)gridDim.x, all);
    if (threadIdx.x == 0) g_rows_arrived[ra.set ^ 1][blockIdx.x] = 0;
    if ((int)blockIdx.x >= ctas) return;
    const int64_t run0 = blockIdx.x * all / ctas, run1 = (blockIdx.x + 1) * all / ctas;
    if (mine && before <= run0 && run0 < before + mine) {
        int64_t at = before;
        for (int s = s0; s < s1; ++s) {
            const SeqWork w = seq_work(a, s, limit);
            const int64_t next = at + (int64_t)w.items * w.units();
            if (run0 < next) {
                sm.start[0] = s;
                sm.start[1] = (int)((run0 - at) / w.units());
                sm.start[2] = (int)((run0 - at) % w.units());
                break;
            }
            at = next;
        }
    }
    __syncthreads();
    Cursor cur;
    cur.s = sm.start[0];
    cur.item = sm.start[1];
    cur.unit = sm.start[2];
    cur.left = (int)(run1 - run0);
    cur.w = seq_work(a, cur.s, limit);

    // The producer runs ahead of the warp's own tiles.  Lane i holds the places
    // of the i-th of up to 32 pairs of one item and copies them itself.
    Cursor pro = cur;
    const uint8_t *pro_a = nullptr, *pro_b = nullptr;  // no second tile: nullptr
    int pro_i = 0, pro_n = 0;
    Stage put, get;
    bool alive = true;  // no wait has expired
    auto place = [&](int tile) -> const uint8_t* {
        const int slot = a.page_of(tile);
        const int id = a.c.page(pro.s, slot);
        const uint32_t at = ((uint32_t)id * a.c.n_kv + pro.item / (pro.w.items / a.c.n_kv)) * a.page_tiles + (tile - slot * a.page_tiles);
        return id < 0 ? a.nan_tile : a.c.pages + (uint64_t)at * Tile<HD>::kBytes;
    };
    auto refill = [&]() {
        pro_i = pro_n = 0;
        while (pro.left > 0 && pro_n == 0) {
            const int units = min(32, min(pro.left, pro.w.units() - pro.unit));
            const int step = pro.unit + lane - kItemUnits, tile = 2 * (step * kRowWarps + warp);
            const bool there = lane < units && step >= 0 && tile * kTile < pro.w.len;
            if (there) {
                pro_a = place(tile);
                pro_b = (tile + 1) * kTile < pro.w.len ? place(tile + 1) : nullptr;
            }
            const uint32_t lanes = __ballot_sync(0xFFFFFFFFu, there);  // consecutive
            if (lanes) {
                pro_i = __ffs(lanes) - 1;
                pro_n = pro_i + __popc(lanes);
            }
            pro.next(a, units, limit_at);
        }
    };
    auto produce = [&]() {
        if (pro_i == pro_n) {
            refill();
            if (pro_n == 0) return;
        }
        if (lane == pro_i && alive) {
            const uint32_t bar = full + 8 * put.i, to = ring + put.i * (2 * Tile<HD>::kBytes);
            const bool two = pro_b != nullptr;
            mbar_arrive_expect_tx(bar, two ? 2 * Tile<HD>::kBytes : Tile<HD>::kBytes);
            bulk_g2s(to, pro_a, Tile<HD>::kBytes, bar);
            if (two) bulk_g2s(to + Tile<HD>::kBytes, pro_b, Tile<HD>::kBytes, bar);
        }
        ++pro_i;
        put.next();
    };
#pragma unroll 1
    for (int i = 0; i < kRowStages; ++i) produce();

    const uint32_t at_k = keep(tile_pos(0, r) * (HD / 2) + t * (HD / 8));                             // keys' numbers
    const uint32_t at_m = keep(Tile<HD>::kScaleK + tile_pos(0, r) * (HD / 8) + t * 4);                // word (d, m) t
    const uint32_t at_d0 = keep(Tile<HD>::kScaleK + (4 * t + (t >> 1)) * (HD / 8));                   // scale rows of
    const uint32_t at_d1 = keep(Tile<HD>::kScaleK + (4 * t + 1 - (t >> 1)) * (HD / 8));               // two columns
    const uint32_t at_v = keep(Tile<HD>::kV + lane * (HD / 8));                                       // values' numbers
    const uint32_t low = keep(t < 2 ? 0x5410u : 0x1054u), high = keep(t < 2 ? 0x7632u : 0x3276u);
    constexpr uint32_t kToV = Tile<HD>::kScaleV - Tile<HD>::kScaleK, kTwo = 2 * (HD / 8);             // two rows on
    while (cur.left > 0) {
        // ---- one item (or the part of it inside the run)
        const int units = min(cur.left, cur.w.units() - cur.unit), groups = cur.w.items / a.c.n_kv;
        const int step0 = cur.w.step(cur.unit), step1 = cur.w.step(cur.unit + units);
        if (step0 == step1) {  // the run ends before the item's first step
            cur.next(a, units, limit_at);
            continue;
        }
        const int kvh = cur.item / groups, row0 = (cur.item - kvh * groups) * kRowTile;
        const int rows = min(kRowTile, cur.w.n * a.rep - row0);
        const int tok = (row0 + r) / a.rep;  // row r of the tile: token and head
        const int sees = r < rows ? cur.w.len - (cur.w.n - 1 - tok) : 0;
        const int sees_all = cur.w.len - (cur.w.n - 1 - row0 / a.rep);  // positions that every row sees
        // the query rows as operands: q * 2^k, the row's largest value in [2^9, 2^10); a group per warp
        float f_log2;  // score (log2) over what the products give
        {
            float q[G][8];
            float top = 0.f;
            const float* src = a.q + (int64_t)(cur.w.begin + tok) * a.ldq + (kvh * a.rep + (row0 + r) % a.rep) * HD + 8 * t;
            const bool vec = ((reinterpret_cast<uintptr_t>(a.q) | (a.ldq * 4)) & 15) == 0;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                if (r < rows && vec) {
                    const float4 x = *reinterpret_cast<const float4*>(src + 32 * g);
                    const float4 y = *reinterpret_cast<const float4*>(src + 32 * g + 4);
                    q[g][0] = x.x; q[g][1] = x.y; q[g][2] = x.z; q[g][3] = x.w;
                    q[g][4] = y.x; q[g][5] = y.y; q[g][6] = y.z; q[g][7] = y.w;
                } else {
#pragma unroll
                    for (int n = 0; n < 8; ++n) q[g][n] = r < rows ? src[32 * g + n] : 0.f;
                }
            }
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int n = 0; n < 8; ++n) top = fmaxf(top, fabsf(q[g][n]));
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            const int e = min(max((int)(__float_as_uint(top) >> 23), 30), 230);
            const float up = __uint_as_float((uint32_t)(127 + 136 - e) << 23), down = __uint_as_float((uint32_t)(e - 9) << 23);
            f_log2 = a.scale * 1.44269504088896340736f * down;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                if (g != warp) continue;
                float sum = 0.f;
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    q[g][n] *= up;
                    sum += q[g][n];
                }
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
                if (t == g) split2(0.f, sum, &sm.qs[0][lane], &sm.qs[1][lane]);
                if (G == 2 && t == g + 2) sm.qs[0][lane] = sm.qs[1][lane] = 0u;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    uint4 x;
                    split2(q[g][2 * k], q[g][2 * k + 4], &x.x, &x.y);
                    split2(q[g][2 * k + 1], q[g][2 * k + 5], &x.z, &x.w);
                    sm.qa[2 * g + k][lane] = x;
                }
            }
        }
        __syncthreads();
        const uint32_t qa = smem_addr(sm.qa) + 16 * lane, qs_hi = sm.qs[0][lane], qs_lo = sm.qs[1][lane];
        float2 o[G][4];  // values' numbers less 8: [group][c], times 2^k
        constexpr uint32_t kFirst = 0x78007800u, kOne = 0x3C003C00u;
        uint32_t d_up = kFirst;  // 2^k as an fp16 pair; k = 15 before the first scale
        float om = 0.f;  // and their middles, of group t
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[g][c] = make_float2(0.f, 0.f);
        float ref = -3.0e38f, l = 0.f;

#pragma unroll 1
        for (int i = step0; i < step1; ++i) {
            const int p0 = (i * kRowWarps + warp) * kPairLen;
            if (p0 >= cur.w.len) break;  // and so are the warp's further tiles
            if (alive && !wait_full(full + 8 * get.i, get.parity)) {
                // no copies from here on; those in flight have to land before the CTA ends
                for (Stage s = get; s.i != put.i || s.parity != put.parity; s.next()) wait_full(full + 8 * s.i, s.parity);
                alive = false;
            }
            const uint32_t pair = ring + get.i * (2 * Tile<HD>::kBytes);
            get.next();
            // ---- scores of positions 4t .. 4t+3 of both tiles for row r
            float s[2][4];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint32_t tile = pair + u * Tile<HD>::kBytes;
                uint32_t kw[2][G], kd[4][G];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    lds_words<G>(tile + at_k + h * HD, kw[h]);
                    lds_words<G>(tile + at_d0 + h * kTwo, kd[2 * h]);
                    lds_words<G>(tile + at_d1 + h * kTwo, kd[2 * h + 1]);
                }
                float2 acc[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float cm[4];
                    mma16816_zero(cm, qs_hi, qs_lo, 0u, 0u, G == 4 || t < G ? lds32(tile + at_m + h * kTwo) : 0u, 0u);
                    acc[h] = add2(make_float2(cm[0], cm[1]), make_float2(cm[2], cm[3]));
                }
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const uint4 q0 = lds128(qa + 1024 * g), q1 = lds128(qa + 1024 * g + 512);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float c[4];
                        const uint32_t w = kw[h][g], w8 = w >> 8;
                        mma16816_zero(c, q0.x, q0.y, q0.z, q0.w, numbers<false>(w, 0.f), numbers<true>(w, 0.f));
                        mma16816(c, q1.x, q1.y, q1.z, q1.w, numbers<false>(w8, 0.f), numbers<true>(w8, 0.f));
                        acc[h] = __ffma2_rn(add2(make_float2(c[0], c[1]), make_float2(c[2], c[3])),
                                            make_float2(h2f(kd[2 * h][g]), h2f(kd[2 * h + 1][g])), acc[h]);
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    s[u][2 * h] = acc[h].x * f_log2;
                    s[u][2 * h + 1] = acc[h].y * f_log2;
                }
            }
            // ---- the values' scales of the lane's positions as pairs, times 2^k
            __half2 d[2][2][G];
            const bool edge = p0 + kPairLen > sees_all;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    uint32_t w0[G], w1[G];
                    lds_words<G>(pair + u * Tile<HD>::kBytes + at_d0 + kToV + k * kTwo, w0);
                    lds_words<G>(pair + u * Tile<HD>::kBytes + at_d1 + kToV + k * kTwo, w1);
#pragma unroll
                    for (int g = 0; g < G; ++g) d[u][k][g] = bits_h2(__byte_perm(w0[g], w1[g], 0x5410));
                }
            if (edge) {  // positions that the row does not see: whatever is stored there must not touch it
                __syncwarp();
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (p0 + u * kTile + 4 * t + (j ^ (t >> 1)) >= sees) {
                            s[u][j] = -INFINITY;
#pragma unroll
                            for (int g = 0; g < G; ++g)
                                d[u][j >> 1][g] = bits_h2(h2bits(d[u][j >> 1][g]) & (j & 1 ? 0x0000FFFFu : 0xFFFF0000u));
                        }
            }
            uint32_t big = 0;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int g = 0; g < G; ++g) big |= h2bits(d[u][k][g]);
            if (__any_sync(0xFFFFFFFFu, d_up != kOne || (big & 0x40004000u) != 0)) {  // k is not 0, or a scale is 2 or more
                // a first scale of 2^-3 or more (or of 2^-7 with some a sixteenth of it) needs no k
                const bool plain = d_up == kFirst && !__any_sync(0xFFFFFFFFu, (big & 0x40004000u) != 0) &&
                                   __any_sync(0xFFFFFFFFu, (big & big << 1 & 0x20002000u) != 0);
                if (plain) {
                    d_up = kOne;
                } else {
                    __half2 some[4];  // NaNs do not count
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        some[i] = __hmax2(__habs2(d[i / 2][i % 2][0]), __habs2(d[i / 2][i % 2][1]));
                        if constexpr (G == 4) some[i] = __hmax2(some[i], __hmax2(__habs2(d[i / 2][i % 2][2]), __habs2(d[i / 2][i % 2][3])));
                    }
                    const __half2 most = __hmax2(__hmax2(some[0], some[1]), __hmax2(some[2], some[3]));
                    const uint32_t lo = h2bits(most) & 0xFFFFu, hi = h2bits(most) >> 16;
                    const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, max(lo > 0x7C00u ? 0u : lo, hi > 0x7C00u ? 0u : hi));
                    const int e = (int)(top >> 10) - 15, k0 = (int)(d_up >> 26) - 15;
                    const int k = min(k0, e >= 1 ? max(-14, -e) : e >= -3 ? 0 : -e);
                    if (k != k0) {
                        const float by = __uint_as_float((uint32_t)(127 + k - k0) << 23);
                        const float2 b2 = make_float2(by, by);
#pragma unroll
                        for (int g = 0; g < G; ++g)
#pragma unroll
                            for (int c = 0; c < 4; ++c) o[g][c] = __fmul2_rn(o[g][c], b2);
                        d_up = (uint32_t)(15 + k) * 0x04000400u;
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int k = 0; k < 2; ++k)
#pragma unroll
                            for (int g = 0; g < G; ++g) d[u][k][g] = __hmul2(d[u][k][g], bits_h2(d_up));
                }
            }
            // ---- weights
            const float smax = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                                     fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
            if (__any_sync(0xFFFFFFFFu, smax > ref + 14.f)) {
                float m = fmaxf(smax, __shfl_xor_sync(0xFFFFFFFFu, smax, 1));
                m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
                const float to = m > ref + 14.f ? m - 10.f : ref;
                const float keep = exp2_fast(ref - to);
                ref = to;
                l *= keep;
                const float2 k2 = make_float2(keep, keep);
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int c = 0; c < 4; ++c) o[g][c] = __fmul2_rn(o[g][c], k2);
                om *= keep;
            }
            uint32_t ph[2][2], pl[2][2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float p[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) p[j] = exp2_fast(s[u][j] - ref);
                l += (p[0] + p[1]) + (p[2] + p[3]);
                split2(p[0], p[1], &ph[u][0], &pl[u][0]);
                split2(p[2], p[3], &ph[u][1], &pl[u][1]);
                if (edge) {  // p . (m / 2 + 4 d) row by row, so that a NaN stays with the rows that see it
                    __syncwarp();
#pragma unroll 1
                    for (int g = 0; g < G; ++g) {
                        float x = 0.f;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint32_t w = lds32(pair + u * Tile<HD>::kBytes + (j & 1 ? at_d1 : at_d0) + kToV + (j >> 1) * kTwo + 4 * g);
                            if (p0 + u * kTile + 4 * t + (j ^ (t >> 1)) < sees) x = fmaf(p[j], fmaf(4.f, h2f(w), 0.5f * h2f(w >> 16)), x);
                        }
                        x += __shfl_xor_sync(0xFFFFFFFFu, x, 1);
                        x += __shfl_xor_sync(0xFFFFFFFFu, x, 2);
                        if (t == g) om += x;
                    }
                }
            }
            // ---- p . (m / 2 + 4 d): column 2g of the product, lanes of an even r
            if (!edge) {
                // twice of it where k >= 0 (d is below 2, so m + 8 d rounds to a finite number): m may be subnormal, and
                // half of one is not exact
                const uint32_t twice = d_up >= kOne ? 0x04000400u : 0u;
                const __half2 by_d = bits_h2(0x44004400u + twice), by_m = bits_h2(0x38003800u + twice);  // 4 and 1/2
                float chi[4], clo[4];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    uint32_t hi[2], lo[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {  // (d, m) of group r / 2 at the positions of the lane's operand
                        const uint32_t row = pair + u * Tile<HD>::kBytes + kToV + k * kTwo + (r >> 1) * 4;
                        const uint32_t w0 = G == 4 || r < 4 ? lds32(row + at_d0) : 0u, w1 = G == 4 || r < 4 ? lds32(row + at_d1) : 0u;
                        sum2(__hmul2(bits_h2(__byte_perm(w0, w1, 0x5410)), by_d),
                             __hmul2(bits_h2(__byte_perm(w0, w1, 0x7632)), by_m), &hi[k], &lo[k]);
                    }
                    if (u == 0) {
                        mma16816_zero(chi, ph[u][0], pl[u][0], ph[u][1], pl[u][1], hi[0], hi[1]);
                        mma16816_zero(clo, ph[u][0], pl[u][0], ph[u][1], pl[u][1], lo[0], lo[1]);
                    } else {
                        mma16816(chi, ph[u][0], pl[u][0], ph[u][1], pl[u][1], hi[0], hi[1]);
                        mma16816(clo, ph[u][0], pl[u][0], ph[u][1], pl[u][1], lo[0], lo[1]);
                    }
                }
                om = fmaf(twice ? 0.5f : 1.f, (chi[0] + chi[2]) + (clo[0] + clo[2]), om);
            }
            // ---- (p d) . (n - 8)
            uint32_t v[2][2][G];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    lds_words<G>(pair + u * Tile<HD>::kBytes + at_v + k * (4 * HD), v[u][k]);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float c[4][4];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    uint32_t hi[2], lo[2], x[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const __half2 h = __hmul2(bits_h2(ph[u][k]), d[u][k][g]);
                        hi[k] = h2bits(h);
                        lo[k] = h2bits(__hfma2(bits_h2(pl[u][k]), d[u][k][g], __hfma2(bits_h2(ph[u][k]), d[u][k][g], __hneg2(h))));
                        x[k] = __byte_perm(v[u][k][g / 2], v[u][k][G / 2 + g / 2], g & 1 ? high : low);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t x0 = j < 2 ? x[0] : x[0] >> 8, x1 = j < 2 ? x[1] : x[1] >> 8;
                        const uint32_t b0 = j & 1 ? numbers<true>(x0, -8.f) : numbers<false>(x0, -8.f);
                        const uint32_t b1 = j & 1 ? numbers<true>(x1, -8.f) : numbers<false>(x1, -8.f);
                        if (u == 0) mma16816_zero(c[j], hi[0], lo[0], hi[1], lo[1], b0, b1);
                        else mma16816(c[j], hi[0], lo[0], hi[1], lo[1], b0, b1);
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    o[g][j] = add2(o[g][j], add2(make_float2(c[j][0], c[j][1]), make_float2(c[j][2], c[j][3])));
            }
            __syncwarp();
            produce();
        }

        // ---- the four warps' results together
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
        {
            // sums of p (m / 2 + 4 d): column 2g, i.e. lane t = g, element 0
            const float down = __uint_as_float((127 + 15 - (d_up >> 26)) << 23);  // 2^-k
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const float mid = 2.f * __shfl_sync(0xFFFFFFFFu, om, (lane & ~3) + g);
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    *reinterpret_cast<float2*>(&sm.o[warp][r][32 * g + 8 * c + 2 * t]) =
                        make_float2(fmaf(o[g][c].x, down, mid), fmaf(o[g][c].y, down, mid));
            }
            if (t == 0) {
                sm.ml[warp][r][0] = ref;
                sm.ml[warp][r][1] = l;
            }
        }
        __syncthreads();
        const bool whole = step1 - step0 == cur.w.steps;
        const int slot = 2 * blockIdx.x + (step0 == 0 ? 1 : 0);
        for (int i = threadIdx.x; i < kRowTile * HD / 4; i += kRowThreads) {
            const int rr = i / (HD / 4), d = 4 * (i % (HD / 4));
            float m = sm.ml[0][rr][0];
#pragma unroll
            for (int w = 1; w < kRowWarps; ++w) m = fmaxf(m, sm.ml[w][rr][0]);
            float sum = 0.f;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kRowWarps; ++w) {
                const float k = exp2_fast(sm.ml[w][rr][0] - m);
                const float4 y = *reinterpret_cast<const float4*>(&sm.o[w][rr][d]);
                sum = fmaf(k, sm.ml[w][rr][1], sum);
                x.x = fmaf(k, y.x, x.x); x.y = fmaf(k, y.y, x.y); x.z = fmaf(k, y.z, x.z); x.w = fmaf(k, y.w, x.w);
            }
            if (whole) {
                if (rr < rows) {
                    const int64_t at = (int64_t)(cur.w.begin + (row0 + rr) / a.rep) * a.n_head + kvh * a.rep + (row0 + rr) % a.rep;
                    const float inv = sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);
                    if (sum == 0.f) x = make_float4(0.f, 0.f, 0.f, 0.f);
                    *reinterpret_cast<float4*>(a.out + at * HD + d) = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
                    if (a.lse && d == 0) a.lse[at] = sum == 0.f ? -INFINITY : 0.69314718055994530942f * (m + log2f(sum));
                }
            } else {
                *reinterpret_cast<float4*>(ra.part_o + ((int64_t)slot * kRowTile + rr) * HD + d) = x;
                if (d == 0) *reinterpret_cast<float2*>(ra.part_ml + (slot * kRowTile + rr) * 2) = make_float2(m, sum);
            }
        }
        if (!whole) {  // the CTA whose part is the last to come joins them
            __syncthreads();
            if (threadIdx.x == 0) {
                const int64_t unit0 = run1 - cur.left - cur.unit;  // number of the item's first unit
                const int c0 = run_of(unit0 + kItemUnits, ctas, all), c1 = run_of(unit0 + cur.w.units() - 1, ctas, all);
                __threadfence();
                const bool last = atomicAdd(&g_rows_arrived[ra.set][c0], 1u) == (unsigned)(c1 - c0);
                if (last) g_rows_arrived[ra.set][c0] = 0;
                __threadfence();
                sm.start[0] = last ? c1 - c0 + 1 : 0;
                sm.start[1] = c0;
            }
            __syncthreads();
            if (sm.start[0]) rows_join<HD>(ra, sm.start[1], sm.start[0], cur.w, kvh, row0);
        }
        __syncthreads();
        cur.next(a, units, limit_at);
    }
}

}  // namespace serve
}  // namespace cllm
