// Attention of many rows per sequence: one warp per query
// row and head, lane = head_dim/32 values, positions one after the other with
// the running maximum and sum of the softmax.
#pragma once
#include "kv4_decode.cuh"

namespace cllm {
namespace serve {

// Sequence of row t and the positions it sees (0 for a row of no sequence, -1
// for one that kv4_rows_kernel has).
__device__ __forceinline__ int row_sees(const AttnArgs& a, int t, int* seq) {
    int s = t, i = 0, n = 1;
    if (a.q_begin) {
        int lo = 0, hi = a.c.n_seqs;  // the last s with q_begin[s] <= t
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (a.q_begin[mid + 1] <= t) lo = mid + 1;
            else hi = mid;
        }
        s = lo;
        if (s >= a.c.n_seqs || t < a.q_begin[s]) return -1;
        i = t - a.q_begin[s];
        n = a.q_begin[s + 1] - a.q_begin[s];
    }
    *seq = s;
    if ((int64_t)n * a.rep <= a.rows_max) return -1;
    return max(0, a.c.length(s) - (n - 1 - i));
}

template <int HD>
__global__ void __launch_bounds__(128) kv4_attention_kernel(const AttnArgs a) {
    constexpr int D = HD / 32, G = Tile<HD>::G;
    const int lane = threadIdx.x & 31, h = blockIdx.y * 4 + (threadIdx.x >> 5), t = blockIdx.x;
    if (h >= a.n_head) return;
    const int kvh = h / (a.n_head / a.c.n_kv);
    int seq = 0;
    const int sees = row_sees(a, t, &seq);
    if (sees < 0) return;
    float q[D], acc[D];
#pragma unroll
    for (int e = 0; e < D; ++e) {
        q[e] = a.q[(int64_t)t * a.ldq + h * HD + lane * D + e];
        acc[e] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int p = 0; p < sees; ++p) {
        const int id = a.c.page(seq, p / a.c.page_len);
        if (id < 0) continue;
        const uint8_t* tile = a.c.tile<HD>(id, kvh, p % a.c.page_len);
        const int pt = p % kTile;
        float s = 0.f, v[D];
#pragma unroll
        for (int e = 0; e < D; ++e) {
            const int i = lane * D + e, g = i / 32, j = i % 32;
            const int kn = ((pt * 4 + j / 8) * G + g) * 8 + j % 8;
            const int vn = ((((pt % 4 / 2) * 8 + j % 8) * 4 + pt / 4) * 2 + pt % 2) * (4 * G) + g * 4 + j / 8;
            const uint32_t ks = *reinterpret_cast<const uint32_t*>(tile + Tile<HD>::kScaleK + (pt * G + g) * 4);
            const uint32_t vs = *reinterpret_cast<const uint32_t*>(tile + Tile<HD>::kScaleV + (pt * G + g) * 4);
            const float kf = (float)((tile[kn / 2] >> (4 * (kn & 1))) & 15);
            const float vf = (float)((tile[Tile<HD>::kV + vn / 2] >> (4 * (vn & 1))) & 15);
            s = fmaf(q[e], fmaf(kf, h2f(ks), h2f(ks >> 16)), s);
            v[e] = fmaf(vf, h2f(vs), h2f(vs >> 16));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
        s *= a.scale;
        const float mn = fmaxf(m, s), keep = expf(m - mn), w = expf(s - mn);
        l = fmaf(l, keep, w);
#pragma unroll
        for (int e = 0; e < D; ++e) acc[e] = fmaf(acc[e], keep, w * v[e]);
        m = mn;
    }
#pragma unroll
    for (int e = 0; e < D; ++e)
        a.out[((int64_t)t * a.n_head + h) * HD + lane * D + e] = l == 0.f ? 0.f : acc[e] / l;
    if (a.lse && lane == 0) a.lse[(int64_t)t * a.n_head + h] = l == 0.f ? -INFINITY : m + logf(l);
}

}  // namespace serve
}  // namespace cllm
