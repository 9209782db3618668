// RoPE on q and k, K and V quantised to 4 bits into their pages
// (cllm_cuda_kv4_append).
//
// A head's vector is HD/4 lanes of four consecutive values: the rotation's
// partner (i + HD/2) is HD/8 lanes away and a group of 32 values is eight
// lanes, so the rotation is one shuffle per value and min and max are three
// shuffle steps each.  Every operation is a single rounded fp32 operation in
// the order of the header's formula, so the stored numbers do not depend on
// how the work is spread.
//
// What bounds it: HBM for many tokens (q, k and v read, q and the numbers
// written), latency for few.  A warp takes `span` vectors of one token, so the
// token's page, position and rotation are looked up once for them and the next
// vector is on its way while one is worked on; with few tokens span is 1.
#pragma once
#include "kv4_format.cuh"

namespace cllm {
namespace serve {

constexpr int kAppendThreads = 128;

struct AppendArgs {
    const float *q, *k, *v, *rope;
    float *q_out, *k_out, *v_out;
    int64_t ldq, ldkv;
    const int *token_seq, *token_pos;
    int n_tok, n_head, n_pos;
    int vec;   // rows 16-byte aligned: float4 accesses
    int rope_vec;  // and the rotation table
    int span;      // steps (of 128 / HD vectors) of a warp
    Cache c;
};

__device__ __forceinline__ float4 load4(const float* p, bool vec) {
    if (vec) return *reinterpret_cast<const float4*>(p);
    return make_float4(p[0], p[1], p[2], p[3]);
}
__device__ __forceinline__ void store4(float* p, const float4& x, bool vec) {
    if (vec) {
        *reinterpret_cast<float4*>(p) = x;
    } else {
        p[0] = x.x; p[1] = x.y; p[2] = x.z; p[3] = x.w;
    }
}

// Vectors of a token: q heads first, then the key heads, then the value heads.
template <int HD>
__global__ void __launch_bounds__(kAppendThreads) kv4_append_kernel(const AppendArgs a) {
    constexpr int LANES = HD / 4, G = Tile<HD>::G, VECS = 32 / LANES;  // lanes of a vector, vectors of a step
    __shared__ __align__(16) uint8_t s_num[kAppendThreads / 32][128];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int sub = lane & (LANES - 1), part = lane / LANES;  // lane of the vector, vector of the step
    const int units = a.n_head + 2 * a.c.n_kv, steps = (units + VECS - 1) / VECS, parts = (steps + a.span - 1) / a.span;
    const int64_t at = (int64_t)blockIdx.x * (kAppendThreads / 32) + warp;
    const int t = (int)(at / parts), step0 = (int)(at - (int64_t)t * parts) * a.span, step1 = min(steps, step0 + a.span);
    if (t >= a.n_tok) return;

    const int seq = a.token_seq[t], pos = a.token_pos[t];
    bool live = seq >= 0;
    int id = -1;
    if (live && (seq >= a.c.n_seqs || pos < 0 || pos >= (int64_t)a.c.max_pages * a.c.page_len || (a.rope && pos >= a.n_pos))) {
        atomicOr(&g_serve_status, kServeBadPage);
        live = false;
    }
    if (live) id = a.c.page(seq, pos / a.c.page_len);
    const int p = live ? pos % kTile : 0, in_page = live ? pos % a.c.page_len : 0;
    auto source = [&](int u) -> const float* {  // the lane's four values of vector u
        const float* row = u < a.n_head ? a.q + (int64_t)t * a.ldq + u * HD
                                        : (u < a.n_head + a.c.n_kv ? a.k + (int64_t)t * a.ldkv + (u - a.n_head) * HD
                                                                   : a.v + (int64_t)t * a.ldkv + (u - a.n_head - a.c.n_kv) * HD);
        return row + 4 * sub;
    };
    auto has = [&](int u) { return live && u < units && (u < a.n_head || id >= 0); };
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    int u = step0 * VECS + part;
    float4 next = has(u) ? load4(source(u), a.vec) : zero;
    float c[8];  // cos, sin of the lane's four pairs
    if (a.rope && live) {
        const float4* cs = reinterpret_cast<const float4*>(a.rope + ((int64_t)pos * (HD / 2) + 4 * (sub & (LANES / 2 - 1))) * 2);
        const float4 x = a.rope_vec ? cs[0] : load4(reinterpret_cast<const float*>(cs), false);
        const float4 y = a.rope_vec ? cs[1] : load4(reinterpret_cast<const float*>(cs) + 4, false);
        c[0] = x.x; c[1] = x.y; c[2] = x.z; c[3] = x.w; c[4] = y.x; c[5] = y.y; c[6] = y.z; c[7] = y.w;
    }
#pragma unroll 1
    for (int step = step0; step < step1; ++step, u += VECS) {
        float4 x = next;
        next = step + 1 < step1 && has(u + VECS) ? load4(source(u + VECS), a.vec) : zero;
        const bool on = u < units, is_q = u < a.n_head, is_k = !is_q && u < a.n_head + a.c.n_kv, stored = on && !is_q && live && id >= 0;
        const int h = is_q ? u : is_k ? u - a.n_head : u - a.n_head - a.c.n_kv;
        if (a.rope) {  // the same branch for the whole grid; values pass through
            float4 o;
            o.x = __shfl_xor_sync(0xFFFFFFFFu, x.x, LANES / 2);
            o.y = __shfl_xor_sync(0xFFFFFFFFu, x.y, LANES / 2);
            o.z = __shfl_xor_sync(0xFFFFFFFFu, x.z, LANES / 2);
            o.w = __shfl_xor_sync(0xFFFFFFFFu, x.w, LANES / 2);
            if (live && (is_q || is_k)) {
                const bool hi = sub >= LANES / 2;
                auto turn = [&](float own, float other, int i) {
                    // low half: x0 cos - x1 sin; high half: x0 sin + x1 cos
                    return hi ? __fadd_rn(__fmul_rn(other, c[2 * i + 1]), __fmul_rn(own, c[2 * i]))
                              : __fsub_rn(__fmul_rn(own, c[2 * i]), __fmul_rn(other, c[2 * i + 1]));
                };
                x = make_float4(turn(x.x, o.x, 0), turn(x.y, o.y, 1), turn(x.z, o.z, 2), turn(x.w, o.w, 3));
            }
        }
        if (on && is_q) store4(a.q_out + (int64_t)t * a.n_head * HD + h * HD + 4 * sub, x, a.vec);
        if (!__any_sync(0xFFFFFFFFu, on && !is_q)) continue;

        // min and max of the group (eight lanes)
        float lo = fminf(fminf(x.x, x.y), fminf(x.z, x.w)), hi = fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w));
        bool nan = x.x != x.x || x.y != x.y || x.z != x.z || x.w != x.w;
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
        }
        nan = ((__ballot_sync(0xFFFFFFFFu, nan) >> (lane & ~7)) & 0xFFu) != 0;
        __half d16 = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f)), m16 = __float2half_rn(lo);
        const bool bad = nan || !(fabsf(__half2float(d16)) <= 65504.f) || !(fabsf(__half2float(m16)) <= 65504.f);
        if (bad) d16 = m16 = __ushort_as_half(0x7E00);
        const float d = __half2float(d16), m = __half2float(m16);
        auto number = [&](float v) -> uint32_t {
            if (!(d > 0.f)) return 0u;
            return (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(v, m), d)), 0.f), 15.f);
        };
        const uint32_t n0 = number(x.x), n1 = number(x.y), n2 = number(x.z), n3 = number(x.w);
        if (on && !is_q) {
            float* out = is_k ? a.k_out : a.v_out;
            if (out) {
                auto value = [&](uint32_t n) { return stored ? __fadd_rn(__fmul_rn((float)n, d), m) : 0.f; };
                store4(out + (int64_t)t * a.c.n_kv * HD + h * HD + 4 * sub,
                       make_float4(value(n0), value(n1), value(n2), value(n3)), a.vec);
            }
        }
        // the values' numbers change places: lane (r, group) writes numbers c = 0..3
        // (value 32 group + 8 c + r) as one 16-bit store
        __syncwarp();
        *reinterpret_cast<uint32_t*>(&s_num[warp][4 * lane]) = n0 | (n1 << 8) | (n2 << 16) | (n3 << 24);
        __syncwarp();
        if (stored) {
            uint8_t* tile = a.c.tile<HD>(id, h, in_page);
            const int g = sub >> 3, j = sub & 7;
            if (is_k) {  // four consecutive values are one 16-bit store
                *reinterpret_cast<uint16_t*>(tile + ((p * 4 + (j >> 1)) * G + g) * 4 + (j & 1) * 2) =
                    (uint16_t)(n0 | (n1 << 4) | (n2 << 8) | (n3 << 12));
            } else {
                const int r = sub / G, gv = sub % G;
                const uint8_t* n = &s_num[warp][part * HD + 32 * gv + r];
                *reinterpret_cast<uint16_t*>(tile + Tile<HD>::kV + ((((p & 3) >> 1) * 8 + r) * 4 + (p >> 2)) * (4 * G) +
                                             (p & 1) * (2 * G) + gv * 2) =
                    (uint16_t)(n[0] | (n[8] << 4) | (n[16] << 8) | (n[24] << 12));
            }
            if (j == 0)
                *reinterpret_cast<uint32_t*>(tile + (is_k ? Tile<HD>::kScaleK : Tile<HD>::kScaleV) + (p * G + g) * 4) =
                    (uint32_t)__half_as_ushort(d16) | ((uint32_t)__half_as_ushort(m16) << 16);
        }
    }
}

}  // namespace serve
}  // namespace cllm
