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
// written) together with the instructions (60 a query vector, 130 a key or value),
// latency for few.  A warp takes `span` vectors of one token, so the token's
// page, position and rotation are looked up once for them, and four vectors'
// loads are issued together; with few tokens span is 1.  2048 tokens of 32 query
// and 8 + 8 key and value vectors of 128, all written out: 28.7 us, 3.6 TB/s (56 %
// of a copy's rate).  The warps wait for loads: the vectors', whose addresses are
// known from the start, are issued only once the token's sequence and position, and for
// keys and values its page, are there to say whether they are wanted.  One token: 5 us
// on the GPU.
#pragma once
#include <type_traits>

#include "kv4_format.cuh"

namespace cllm {
namespace serve {

constexpr int kAppendThreads = 128;
constexpr int kAppendTogether = 4;  // steps whose loads are issued together

struct AppendArgs {
    const float *q, *k, *v, *rope;
    float *q_out, *k_out, *v_out;
    int64_t ldq, ldkv;
    const int *token_seq, *token_pos;
    int n_tok, n_head, n_pos;
    int vec;   // rows 16-byte aligned: float4 accesses
    int rope_vec;  // and the rotation table
    int span;      // vectors of a warp
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

// rint(t / d), the quotient rounded to nearest first.  1 / d is off by an ulp, the
// product by another; only beside a half can that choose another number, and
// there the division itself decides.
__device__ __forceinline__ float quotient_number(float t, float d, float by) {
    const float r = __fmul_rn(t, by), n = rintf(r);
    if (fabsf(fabsf(r - n) - 0.5f) > 1e-4f) return n;  // |r| is below 16.1 where it matters
    return rintf(__fdiv_rn(t, d));
}

// Vectors of a token: q heads first, then the key heads, then the value heads.
template <int HD>
__global__ void __launch_bounds__(kAppendThreads) kv4_append_kernel(const AppendArgs a) {
    constexpr int LANES = HD / 4, G = Tile<HD>::G, VECS = 32 / LANES;  // lanes of a vector, vectors of a step
    __shared__ __align__(16) uint8_t s_num[kAppendThreads / 32][128];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int sub = lane & (LANES - 1), part = lane / LANES;  // lane of the vector, vector of the step
    const int n_kv = a.c.n_kv, units = a.n_head + 2 * n_kv, parts = (units + a.span - 1) / a.span;
    const int64_t at = (int64_t)blockIdx.x * (kAppendThreads / 32) + warp;
    const int t = (int)(at / parts), u0 = (int)(at - (int64_t)t * parts) * a.span, u1 = min(units, u0 + a.span);
    if (t >= a.n_tok) return;

    const int seq = a.token_seq[t], pos = a.token_pos[t];
    bool live = seq >= 0;
    int id = -1;
    if (live && (seq >= a.c.n_seqs || pos < 0 || pos >= (int64_t)a.c.max_pages * a.c.page_len || (a.rope && pos >= a.n_pos))) {
        atomicOr(&g_serve_status, kServeBadPage);
        live = false;
    }
    if (live && u1 > a.n_head) id = a.c.page(seq, pos / a.c.page_len);
    const bool turns = live && a.rope;
    float c[8];  // cos, sin of the lane's four pairs
    if (turns) {
        const float* cs = a.rope + ((int64_t)pos * (HD / 2) + 4 * (sub & (LANES / 2 - 1))) * 2;
        const float4 x = load4(cs, a.rope_vec), y = load4(cs + 4, a.rope_vec);
        c[0] = x.x; c[1] = x.y; c[2] = x.z; c[3] = x.w; c[4] = y.x; c[5] = y.y; c[6] = y.z; c[7] = y.w;
        if (sub < LANES / 2) c[1] = -c[1], c[3] = -c[3], c[5] = -c[5], c[7] = -c[7];
    }
    auto rotate = [&](float4 x) -> float4 {  // warp-uniform: token and table are
        if (!turns) return x;
        float4 o;
        o.x = __shfl_xor_sync(0xFFFFFFFFu, x.x, LANES / 2);
        o.y = __shfl_xor_sync(0xFFFFFFFFu, x.y, LANES / 2);
        o.z = __shfl_xor_sync(0xFFFFFFFFu, x.z, LANES / 2);
        o.w = __shfl_xor_sync(0xFFFFFFFFu, x.w, LANES / 2);
        // low half: x0 cos - x1 sin; high half: x1 cos + x0 sin
        return make_float4(__fadd_rn(__fmul_rn(x.x, c[0]), __fmul_rn(o.x, c[1])), __fadd_rn(__fmul_rn(x.y, c[2]), __fmul_rn(o.y, c[3])),
                           __fadd_rn(__fmul_rn(x.z, c[4]), __fmul_rn(o.z, c[5])), __fadd_rn(__fmul_rn(x.w, c[6]), __fmul_rn(o.w, c[7])));
    };
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);

    // queries
    {
        const int h0 = u0, h1 = min(u1, a.n_head);
        const float* src = a.q + (int64_t)t * a.ldq + 4 * sub;
        float* out = a.q_out + (int64_t)t * a.n_head * HD + 4 * sub;
        for (int i = h0; i < h1; i += VECS * kAppendTogether) {
            float4 x[kAppendTogether];
#pragma unroll
            for (int k = 0; k < kAppendTogether; ++k) {
                const int h = i + k * VECS + part;
                x[k] = live && h < h1 ? load4(src + h * HD, a.vec) : zero;
            }
#pragma unroll
            for (int k = 0; k < kAppendTogether; ++k) {
                const int h = i + k * VECS + part;
                if (i + k * VECS >= h1) break;
                const float4 y = rotate(x[k]);
                if (h < h1) store4(out + h * HD, y, a.vec);
            }
        }
    }
    // keys, then values
    const int p = live ? pos % kTile : 0, in_page = live ? pos % a.c.page_len : 0;
    const bool stored = live && id >= 0;
    auto store = [&](auto keys, const float* src, float* out, int h0, int h1) {
        constexpr bool KEYS = decltype(keys)::value;
        src += 4 * sub;
        for (int i = h0; i < h1; i += VECS * kAppendTogether) {
            float4 ahead[kAppendTogether];
#pragma unroll
            for (int k = 0; k < kAppendTogether; ++k) {
                const int h = i + k * VECS + part;
                ahead[k] = stored && h < h1 ? load4(src + h * HD, a.vec) : zero;
            }
#pragma unroll 1
            for (int k = 0; k < kAppendTogether && i + k * VECS < h1; ++k) {
                const int h = i + k * VECS + part;
                float4 x = ahead[0];
#pragma unroll
                for (int m = 0; m + 1 < kAppendTogether; ++m) ahead[m] = ahead[m + 1];
                if (KEYS) x = rotate(x);
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
                const float d = __half2float(d16), m = __half2float(m16), by = __frcp_rn(d);
                auto number = [&](float v) -> uint32_t {
                    if (!(d > 0.f)) return 0u;
                    return (uint32_t)fminf(fmaxf(quotient_number(__fsub_rn(v, m), d, by), 0.f), 15.f);
                };
                const uint32_t n0 = number(x.x), n1 = number(x.y), n2 = number(x.z), n3 = number(x.w);
                if (out && h < h1) {
                    auto value = [&](uint32_t n) { return stored ? __fadd_rn(__fmul_rn((float)n, d), m) : 0.f; };
                    store4(out + h * HD + 4 * sub, make_float4(value(n0), value(n1), value(n2), value(n3)), a.vec);
                }
                const int g = sub >> 3, j = sub & 7;
                uint8_t* tile = a.c.tile<HD>(max(id, 0), min(h, n_kv - 1), in_page);
                if constexpr (KEYS) {  // four consecutive values are one 16-bit store
                    if (stored && h < h1)
                        *reinterpret_cast<uint16_t*>(tile + ((p * 4 + (j >> 1)) * G + g) * 4 + (j & 1) * 2) =
                            (uint16_t)(n0 | (n1 << 4) | (n2 << 8) | (n3 << 12));
                } else {
                    // the numbers change places: lane (r, group) writes numbers c = 0..3 (value
                    // 32 group + 8 c + r) as one 16-bit store
                    __syncwarp();
                    *reinterpret_cast<uint32_t*>(&s_num[warp][4 * lane]) = n0 | (n1 << 8) | (n2 << 16) | (n3 << 24);
                    __syncwarp();
                    const int r = sub / G, gv = sub % G;
                    const uint8_t* n = &s_num[warp][part * HD + 32 * gv + r];
                    if (stored && h < h1)
                        *reinterpret_cast<uint16_t*>(tile + Tile<HD>::kV + ((((p & 3) >> 1) * 8 + r) * 4 + (p >> 2)) * (4 * G) +
                                                     (p & 1) * (2 * G) + gv * 2) =
                            (uint16_t)(n[0] | (n[8] << 4) | (n[16] << 8) | (n[24] << 12));
                }
                if (j == 0 && stored && h < h1)
                    *reinterpret_cast<uint32_t*>(tile + (KEYS ? Tile<HD>::kScaleK : Tile<HD>::kScaleV) + (p * G + g) * 4) =
                        (uint32_t)__half_as_ushort(d16) | ((uint32_t)__half_as_ushort(m16) << 16);
            }
        }
    };
    const int64_t row = (int64_t)t * n_kv * HD;
    store(std::true_type{}, a.k + (int64_t)t * a.ldkv, a.k_out ? a.k_out + row : nullptr, max(0, u0 - a.n_head),
          min(n_kv, u1 - a.n_head));
    store(std::false_type{}, a.v + (int64_t)t * a.ldkv, a.v_out ? a.v_out + row : nullptr, max(0, u0 - a.n_head - n_kv),
          min(n_kv, u1 - a.n_head - n_kv));
}

}  // namespace serve
}  // namespace cllm
