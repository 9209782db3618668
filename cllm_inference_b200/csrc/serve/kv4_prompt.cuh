// Attention of many rows per sequence over the 4-bit cache
// (cllm_cuda_kv4_attention; prompts): a CTA takes 128 rows (tokens x heads of one
// KV head) over all the positions they see, 64 at a time, on tcgen05 tensor cores.
//
// fp32 accuracy from fp16 operands: q, k, p and v enter as hi + lo (22 bits
// together), and a product is lo*hi + hi*lo + hi*hi, in that order, the small
// terms first because the tensor cores cut off as they add.  For the same reason
// a tile's p v is not accumulated in TMEM over the whole sequence but added to
// fp32 registers, rounded to nearest, tile by tile; that also does the rescaling.
// k and v of a tile are scaled by a power of two that brings its largest value to
// [2^10, 2^11), so that lo stays above fp16's subnormals; S and p take it out.
//
// What bounds it: three products a term, 6 * 128 * 64 * HD multiply-adds a tile
// for 128 x 64 scores: 1536 cycles of the tensor cores (HD 128), beside which the
// CTA's four schedulers issue some 500 (softmax) + 600 (numbers to fp16) + 130
// (sums) instructions each, and shared memory moves 96 KB of operands to the
// tensor cores and 64 KB from the numbers: q and p come from TMEM, or the
// operands alone would take all of its bandwidth.
//
// Warps (4 warpgroups; registers moved to where they are needed):
//   0       raw tiles of the pages into a ring (bulk copies)
//   1       TMEM, and the one thread that issues the products
//   4..7    a row each: softmax with a running reference (kv4_decode.cuh), p to TMEM
//   8..11   a row each: the fp32 sums of p v, and the output
//   12..15  numbers and scales to fp16 operands in the 128-byte swizzle
// All waits are bounded; one that expires sets the status, and the CTA runs to its
// end without waiting.
#pragma once
#include "../tc_ptx.cuh"
#include "kv4_decode.cuh"

namespace cllm {
namespace serve {

constexpr int kPromptThreads = 512;
constexpr int kPromptRows = 128, kPromptCols = 64;
constexpr int kRawStages = 3;

template <int HD>
struct PromptSmem {
    static constexpr uint32_t kOperand = kPromptCols * HD * 2;  // bytes of a tile's k (or v), hi or lo
    uint8_t k[2][2][kOperand];  // [stage][hi, lo]: [64 values][position][128 bytes]
    uint8_t v[2][2][kOperand];  // [stage][hi, lo]: [value][128 bytes of positions]
    uint8_t raw[kRawStages][4 * Tile<HD>::kBytes];
    float alpha[4][kPromptRows];  // what a tile's new reference leaves of the sums
    float sum[kPromptRows];
    uint32_t bad[kPromptRows];    // groups that a NaN of the values reaches
    struct Stat {
        float k_down, v_up;  // 2^-(the keys' power), 2^(the values' power)
        int v_power;
        uint32_t bad;        // 1: a value has a NaN
    } stat[4];
    uint32_t top[4][4][2];        // [tile][warp]: largest exponents of keys and values
    uint32_t warp_bad[4][4];
    uint8_t nan[4][kPromptCols];  // groups of a position that are NaN
    uint64_t raw_full[kRawStages], raw_empty[kRawStages];
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2], o_empty[2];
    uint64_t alpha_full[4], stat_full[4], q_full, done;
    uint32_t tmem;
    int abort;
    int item[4];
};

__device__ __forceinline__ void tc_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
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
        if (mbar_try_wait(bar, parity)) return true;
        if ((it & 63u) == 0) {
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
__device__ __forceinline__ void warp_arrive(uint32_t bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// Two values as an fp16 pair and what is left of them as another.
__device__ __forceinline__ void split_pair(float x, float y, uint32_t& hi, uint32_t& lo) { split2(x, y, &hi, &lo); }

// The item of CTA blockIdx.x: sequence, KV head, tile of 128 rows (the last, longest, first).
__device__ __forceinline__ bool prompt_item(const AttnArgs& a, int* out) {
    int left = blockIdx.x;
    for (int s = 0; s < a.c.n_seqs; ++s) {
        int begin, n;
        seq_rows(a, s, &begin, &n);
        const int64_t rows = (int64_t)n * a.rep;
        if (rows <= a.rows_max) continue;
        const int tiles = (int)((rows + kPromptRows - 1) / kPromptRows);
        if (left < tiles * a.c.n_kv) {
            out[0] = s;
            out[1] = left % a.c.n_kv;
            out[2] = tiles - 1 - left / a.c.n_kv;
            return true;
        }
        left -= tiles * a.c.n_kv;
    }
    return false;
}

template <int HD>
__global__ void __launch_bounds__(kPromptThreads, 1) kv4_prompt_kernel(const AttnArgs a) {
    constexpr int G = Tile<HD>::G;
    constexpr uint32_t kIdescS = (1u << 4) | ((uint32_t)(kPromptCols >> 3) << 17) | ((uint32_t)(kPromptRows >> 4) << 24);
    constexpr uint32_t kIdescO = (1u << 4) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(kPromptRows >> 4) << 24);
    constexpr uint32_t kColQ = 0, kColS = 128, kColO = 256;  // TMEM: q hi | lo; two S, each overwritten by p hi | lo; two O
    extern __shared__ uint8_t smem_raw[];
    PromptSmem<HD>& sm =
        *reinterpret_cast<PromptSmem<HD>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* abort = &sm.abort;
    auto bar = [](uint64_t& b) { return smem_addr(&b); };

    if (threadIdx.x == 0) {
        sm.item[3] = prompt_item(a, sm.item);
        for (int i = 0; i < kRawStages; ++i) {
            mbar_init(bar(sm.raw_full[i]), 1);
            mbar_init(bar(sm.raw_empty[i]), 4);
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
        for (int i = 0; i < 4; ++i) {
            mbar_init(bar(sm.alpha_full[i]), 4);
            mbar_init(bar(sm.stat_full[i]), 1);
        }
        mbar_init(bar(sm.q_full), 4);
        mbar_init(bar(sm.done), 1);
        sm.abort = 0;
        fence_mbar_init();
    }
    __syncthreads();
    if (!sm.item[3]) return;  // fewer items than CTAs
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&sm.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&sm.tmem);

    const int seq = sm.item[0], kvh = sm.item[1], row0 = sm.item[2] * kPromptRows;
    int begin, n;
    seq_rows(a, seq, &begin, &n);
    const int len = a.c.length(seq);
    const int last = (int)(min((int64_t)row0 + kPromptRows, (int64_t)n * a.rep) - 1) / a.rep;  // token of the last row
    const int tiles = (max(0, len - (n - 1 - last)) + kPromptCols - 1) / kPromptCols;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 0) {
            // ---- raw tiles
            int issued = 0;
            for (int i = 0; i < tiles && !*abort; ++i) {
                const int st = i % kRawStages, tile = 4 * i + lane;
                if (i >= kRawStages) warp_wait(bar(sm.raw_empty[st]), (uint32_t)(i / kRawStages - 1) & 1u, abort);
                const bool there = lane < 4 && tile * kTile < len;
                const uint32_t count = __popc(__ballot_sync(0xFFFFFFFFu, there));
                if (*abort) break;
                if (lane == 0) mbar_arrive_expect_tx(bar(sm.raw_full[st]), count * Tile<HD>::kBytes);
                __syncwarp();
                if (there) {
                    const int slot = a.page_of(tile);
                    const int id = max(0, a.c.page(seq, slot));  // a bad one is flagged; the copy stays inside the pool
                    bulk_g2s(smem_addr(sm.raw[st]) + lane * Tile<HD>::kBytes,
                             a.c.pages + (((int64_t)id * a.c.n_kv + kvh) * a.page_tiles + (tile - slot * a.page_tiles)) * Tile<HD>::kBytes,
                             Tile<HD>::kBytes, bar(sm.raw_full[st]));
                }
                issued = i + 1;
            }
            if (*abort)  // let the copies in flight land
                for (int i = max(0, issued - kRawStages); i < issued; ++i) wait_full(bar(sm.raw_full[i % kRawStages]), (uint32_t)(i / kRawStages) & 1u);
        } else if (warp == 1 && lane == 0) {
            // ---- products
            wait_or_abort(bar(sm.q_full), 0, abort);
            tc_fence_after();
            for (int i = 0; i <= tiles; ++i) {
                if (i < tiles) {  // S = q k, into the buffer that the products of p(i - 2), issued before, have read
                    const int st = i & 1;
                    wait_or_abort(bar(sm.k_full[st]), (uint32_t)(i >> 1) & 1u, abort);
                    tc_fence_after();
                    const uint32_t d = tmem + kColS + 64 * st;
                    for (int term = 0; term < 3; ++term) {  // lo hi, hi lo, hi hi
                        const uint32_t q = tmem + kColQ + (term == 0 ? HD / 2 : 0), k = smem_addr(sm.k[st][term == 1]);
                        for (int s = 0; s < HD / 16; ++s)
                            tc_mma_ts(d, q + 8 * s, umma_desc_sw128(k + (s / 4) * (kPromptCols * 128) + (s % 4) * 32), kIdescS, term | s);
                    }
                    tc_commit(bar(sm.s_full[st]));
                    tc_commit(bar(sm.k_empty[st]));
                }
                if (i > 0) {  // O = p v of the tile before
                    const int j = i - 1, st = j & 1;
                    wait_or_abort(bar(sm.p_full[st]), (uint32_t)(j >> 1) & 1u, abort);
                    wait_or_abort(bar(sm.v_full[st]), (uint32_t)(j >> 1) & 1u, abort);
                    if (j >= 2) wait_or_abort(bar(sm.o_empty[st]), (uint32_t)((j >> 1) - 1) & 1u, abort);
                    tc_fence_after();
                    const uint32_t d = tmem + kColO + 128 * st;
                    for (int term = 0; term < 3; ++term) {
                        const uint32_t p = tmem + kColS + 64 * st + (term == 0 ? 32 : 0), v = smem_addr(sm.v[st][term == 1]);
                        for (int s = 0; s < kPromptCols / 16; ++s) tc_mma_ts(d, p + 8 * s, umma_desc_sw128(v + s * 32), kIdescO, term | s);
                    }
                    tc_commit(bar(sm.o_full[st]));
                    tc_commit(bar(sm.v_empty[st]));
                }
            }
            tc_commit(bar(sm.done));
            wait_full(bar(sm.done), 0);
        }
    } else if (warp < 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 120;");
        // ---- softmax: thread = row
        const int row = 32 * (warp - 4) + lane, j = row0 + row;
        const uint32_t lanes = (uint32_t)(32 * (warp - 4)) << 16;
        const bool on = j < n * a.rep;
        const int tok = j / a.rep, head = kvh * a.rep + j % a.rep;
        const int sees = on ? max(0, len - (n - 1 - tok)) : 0;
        const float* src = a.q + (int64_t)(begin + tok) * a.ldq + head * HD;
        const bool vec = ((reinterpret_cast<uintptr_t>(a.q) | (a.ldq * 4)) & 15) == 0;
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
            const float up = __uint_as_float((uint32_t)(263 - e) << 23);  // the row's largest value to [2^9, 2^10)
            f_log2 = a.scale * 1.44269504088896340736f * __uint_as_float((uint32_t)(e - 9) << 23);
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
                    split_pair(x.x * up, x.y * up, hi[k / 2], lo[k / 2]);
                    split_pair(x.z * up, x.w * up, hi[k / 2 + 1], lo[k / 2 + 1]);
                }
                tmem_st16u(tmem + lanes + kColQ + i / 2, hi);
                tmem_st16u(tmem + lanes + kColQ + HD / 2 + i / 2, lo);
            }
            tmem_st_wait();
            tc_fence_before();
            warp_arrive(bar(sm.q_full));
        }
        float ref = -3.0e38f, l = 0.f;
        uint32_t bad = 0;
#pragma unroll 1
        for (int i = 0; i < tiles; ++i) {
            const int st = i & 1, r4 = i & 3;
            warp_wait(bar(sm.stat_full[r4]), (uint32_t)(i >> 2) & 1u, abort);
            warp_wait(bar(sm.s_full[st]), (uint32_t)(i >> 1) & 1u, abort);
            tc_fence_after();
            const float f = f_log2 * sm.stat[r4].k_down, v_up = sm.stat[r4].v_up;
            const int v_power = sm.stat[r4].v_power;
            const uint32_t col = tmem + lanes + kColS + 64 * st;
            uint32_t x[4][16];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld16_issue(col + 16 * c, x[c]);
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld_wait(x[c]);
            const int limit = sees - i * kPromptCols;  // columns that the row sees
            if (__any_sync(0xFFFFFFFFu, limit < kPromptCols)) {
                const uint32_t none = __float_as_uint(f < 0.f ? INFINITY : -INFINITY);
#pragma unroll
                for (int c = 0; c < kPromptCols; ++c)
                    if (c >= limit) x[c / 16][c % 16] = none;
            }
            if (sm.stat[r4].bad)
                for (int c = 0; c < min(limit, kPromptCols); ++c) bad |= sm.nan[r4][c];
            float m[4];
            if (f >= 0.f) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    m[c] = __uint_as_float(x[c][0]);
#pragma unroll
                    for (int k = 1; k < 16; ++k) m[c] = fmaxf(m[c], __uint_as_float(x[c][k]));
                }
                m[0] = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    m[c] = __uint_as_float(x[c][0]);
#pragma unroll
                    for (int k = 1; k < 16; ++k) m[c] = fminf(m[c], __uint_as_float(x[c][k]));
                }
                m[0] = fminf(fminf(m[0], m[1]), fminf(m[2], m[3]));
            }
            const float top = m[0] * f, room = 14.f + (float)min(0, v_power);
            float alpha = 1.f;
            if (top > ref + room) {
                const float to = top - (room - 4.f);
                alpha = exp2_fast(ref - to);
                ref = to;
            }
            sm.alpha[r4][row] = alpha;
            const float off = -ref - (float)v_power;
            const float2 f2 = make_float2(f, f), off2 = make_float2(off, off);
            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float2 e = __ffma2_rn(make_float2(__uint_as_float(x[c][2 * k]), __uint_as_float(x[c][2 * k + 1])), f2, off2);
                    const float2 p = make_float2(exp2_fast(e.x), exp2_fast(e.y));
                    sum = add2(sum, p);
                    split_pair(p.x, p.y, hi[k], lo[k]);
                }
                // columns 8c.. of hi and of lo take the place of the scores just read
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    x[c][k] = hi[k];
                    x[c][8 + k] = lo[k];
                }
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    hi[k] = x[2 * c][k];
                    hi[8 + k] = x[2 * c + 1][k];
                    lo[k] = x[2 * c][8 + k];
                    lo[8 + k] = x[2 * c + 1][8 + k];
                }
                tmem_st16u(col + 16 * c, hi);
                tmem_st16u(col + 32 + 16 * c, lo);
            }
            l = fmaf(sum.x + sum.y, v_up, l * alpha);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(bar(sm.alpha_full[r4]));
                mbar_arrive(bar(sm.p_full[st]));
            }
        }
        sm.sum[row] = l;
        sm.bad[row] = bad;
        if (on && a.lse)
            a.lse[(int64_t)(begin + tok) * a.n_head + head] = l == 0.f ? -INFINITY : 0.69314718055994530942f * (ref + log2f(l));
        asm volatile("bar.sync 2, 256;" ::: "memory");
    } else if (warp < 12) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        // ---- sums: thread = row
        const int row = 32 * (warp - 8) + lane, j = row0 + row;
        const uint32_t lanes = (uint32_t)(32 * (warp - 8)) << 16;
        float2 acc[HD / 2];
#pragma unroll
        for (int i = 0; i < HD / 2; ++i) acc[i] = make_float2(0.f, 0.f);
#pragma unroll 1
        for (int i = 0; i < tiles; ++i) {
            const int st = i & 1, r4 = i & 3;
            warp_wait(bar(sm.alpha_full[r4]), (uint32_t)(i >> 2) & 1u, abort);
            const float alpha = sm.alpha[r4][row];
            warp_wait(bar(sm.o_full[st]), (uint32_t)(i >> 1) & 1u, abort);
            tc_fence_after();
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
        if (j < n * a.rep) {
            const float sum = sm.sum[row], inv = sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);
            const uint32_t bad = sm.bad[row];
            float* out = a.out + ((int64_t)(begin + j / a.rep) * a.n_head + kvh * a.rep + j % a.rep) * HD;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const float by = bad >> g & 1 ? NAN : inv;
#pragma unroll
                for (int i = 16 * g; i < 16 * g + 16; i += 2)
                    *reinterpret_cast<float4*>(out + 2 * i) =
                        sum == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                                   : make_float4(acc[i].x * by, acc[i].y * by, acc[i + 1].x * by, acc[i + 1].y * by);
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 112;");
        // ---- numbers to operands: warp w has the 16 positions of raw tile w
        const int w = warp - 12, tid = threadIdx.x - 384;
#pragma unroll 1
        for (int i = 0; i < tiles; ++i) {
            const int rs = i % kRawStages, st = i & 1, r4 = i & 3;
            warp_wait(bar(sm.raw_full[rs]), (uint32_t)(i / kRawStages) & 1u, abort);
            const uint32_t raw = smem_addr(sm.raw[rs]);
            // the largest exponents: a value is below 2^(e - 14) for e = max(exponent of m, exponent of d + 4)
            {
                const int p = tid >> 1, half = tid & 1;  // position, half of its groups
                uint32_t ek = 0, ev = 0, nan = 0;
                if (i * kPromptCols + p < len) {
                    const uint32_t tile = raw + (p / kTile) * Tile<HD>::kBytes + (p % kTile) * (HD / 8) + half * (HD / 16);
#pragma unroll
                    for (int g = 0; g < G / 2; ++g) {
                        const uint32_t k = lds32(tile + Tile<HD>::kScaleK + 4 * g), v = lds32(tile + Tile<HD>::kScaleV + 4 * g);
                        const uint32_t kd = k >> 10 & 31, km = k >> 26 & 31, vd = v >> 10 & 31, vm = v >> 26 & 31;
                        if (max(kd, km) < 31) ek = max(ek, max(km, kd + 4));
                        if (max(vd, vm) < 31) ev = max(ev, max(vm, vd + 4));
                        else nan |= 1u << (half * (G / 2) + g);
                    }
                }
                ek = __reduce_max_sync(0xFFFFFFFFu, ek);
                ev = __reduce_max_sync(0xFFFFFFFFu, ev);
                const bool any = __any_sync(0xFFFFFFFFu, nan != 0);
                nan |= __shfl_xor_sync(0xFFFFFFFFu, nan, 1);
                if (half == 0) sm.nan[r4][p] = (uint8_t)nan;
                if (lane == 0) {
                    sm.top[r4][w][0] = ek;
                    sm.top[r4][w][1] = ev;
                    sm.warp_bad[r4][w] = any;
                }
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            const int ek = (int)max(max(sm.top[r4][0][0], sm.top[r4][1][0]), max(sm.top[r4][2][0], sm.top[r4][3][0]));
            const int ev = (int)max(max(sm.top[r4][0][1], sm.top[r4][1][1]), max(sm.top[r4][2][1], sm.top[r4][3][1]));
            const int kp = min(14, 25 - ek), vp = min(12, 25 - ev);  // powers of two: the largest value to [2^10, 2^11)
            if (tid == 0) {
                sm.stat[r4].k_down = __uint_as_float((uint32_t)(127 - kp) << 23);
                sm.stat[r4].v_up = __uint_as_float((uint32_t)(127 + vp) << 23);
                sm.stat[r4].v_power = vp;
                sm.stat[r4].bad = sm.warp_bad[r4][0] | sm.warp_bad[r4][1] | sm.warp_bad[r4][2] | sm.warp_bad[r4][3];
                mbar_arrive(bar(sm.stat_full[r4]));
            }
            const float k_up = __uint_as_float((uint32_t)(127 + kp) << 23), v_up = __uint_as_float((uint32_t)(127 + vp) << 23);
            const uint32_t tile = raw + w * Tile<HD>::kBytes;
            const int here = len - i * kPromptCols - w * kTile;  // positions of this tile that are stored
            // keys: a word of eight numbers is a 16-byte chunk of the operand's row
            if (i >= 2) warp_wait(bar(sm.k_empty[st]), (uint32_t)((i >> 1) - 1) & 1u, abort);
            {
                const int p = lane & 15, row = w * kTile + p;
                uint32_t sc[G];
                lds_words<G>(tile + Tile<HD>::kScaleK + p * (HD / 8), sc);
                const bool live = p < here;
#pragma unroll
                for (int t2 = 0; t2 < 2; ++t2) {
                    const int t = 2 * (lane >> 4) + t2;
                    uint32_t kw[G];
                    lds_words<G>(tile + p * (HD / 2) + t * (HD / 8), kw);
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const float d = live ? h2f(sc[g]) * k_up : 0.f, m = live ? h2f(sc[g] >> 16) * k_up : 0.f;
                        const uint32_t word = kw[g], word8 = word >> 8;
                        const float2 n04 = __half22float2(bits_h2(numbers<false>(word, 0.f))), n15 = __half22float2(bits_h2(numbers<true>(word, 0.f)));
                        const float2 n26 = __half22float2(bits_h2(numbers<false>(word8, 0.f))), n37 = __half22float2(bits_h2(numbers<true>(word8, 0.f)));
                        uint32_t hi[4], lo[4];
                        split_pair(fmaf(n04.x, d, m), fmaf(n15.x, d, m), hi[0], lo[0]);
                        split_pair(fmaf(n26.x, d, m), fmaf(n37.x, d, m), hi[1], lo[1]);
                        split_pair(fmaf(n04.y, d, m), fmaf(n15.y, d, m), hi[2], lo[2]);
                        split_pair(fmaf(n26.y, d, m), fmaf(n37.y, d, m), hi[3], lo[3]);
                        const uint32_t at = (g >> 1) * (kPromptCols * 128) + row * 128 + ((((g & 1) * 4 + t) ^ (row & 7)) << 4);
                        sts128u(smem_addr(sm.k[st][0]) + at, hi);
                        sts128u(smem_addr(sm.k[st][1]) + at, lo);
                    }
                }
                fence_proxy_async_smem();
                warp_arrive(bar(sm.k_full[st]));
            }
            // values: eight positions of one value are a 16-byte chunk
            if (i >= 2) warp_wait(bar(sm.v_empty[st]), (uint32_t)((i >> 1) - 1) & 1u, abort);
            {
                const int r = lane & 7, q = lane >> 3 & 1, h = lane >> 4;
                constexpr int NG = G / 2;  // groups of a lane
                float d[NG][8], m[NG][8];
                uint32_t num[8];
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    const int t = 2 * q + x / 4;
                    const uint32_t at = tile + Tile<HD>::kV + ((x % 4) / 2) * (4 * HD) + (r * 4 + t) * (HD / 8) + (x & 1) * (HD / 16) + h * (HD / 32);
                    num[x] = HD == 128 ? lds32(at) : lds16(at);
                    const bool live = 8 * q + x < here;
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        const uint32_t sc = lds32(tile + Tile<HD>::kScaleV + (8 * q + x) * (HD / 8) + (h * NG + g) * 4);
                        const bool fine = live && (sc >> 10 & 31) < 31 && (sc >> 26 & 31) < 31;
                        d[g][x] = fine ? h2f(sc) * v_up : 0.f;
                        m[g][x] = fine ? h2f(sc >> 16) * v_up : 0.f;
                    }
                }
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    uint32_t pair[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) pair[x] = __byte_perm(num[2 * x], num[2 * x + 1], g ? 0x7632 : 0x5410);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const uint32_t y = c < 2 ? pair[x] : pair[x] >> 8;
                            const float2 f = __half22float2(bits_h2(c & 1 ? numbers<true>(y, 0.f) : numbers<false>(y, 0.f)));
                            split_pair(fmaf(f.x, d[g][2 * x], m[g][2 * x]), fmaf(f.y, d[g][2 * x + 1], m[g][2 * x + 1]), hi[x], lo[x]);
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
}

}  // namespace serve
}  // namespace cllm
