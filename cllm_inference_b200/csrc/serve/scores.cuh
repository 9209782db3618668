// What a sampler reports of a row of logits (cllm_cuda_token_scores): one CTA
// per row, one pass for maximum, sum and rank, one for the entropy's sum, and
// one search per entry of the top list.
#pragma once
#include "kv4_format.cuh"

namespace cllm {
namespace serve {

constexpr int kScoreThreads = 1024;

struct ScoreArgs {
    const float* x;
    int64_t ld;
    int rows, vocab, top_k;
    const int* tokens;
    float *logprob, *entropy;
    int *rank, *top_ids;
    float* top_logprobs;
};

// A logit and its index as one number: larger is earlier in the order (value
// descending, index ascending); NaN counts as -inf.
__device__ __forceinline__ uint64_t order_key(float v, int i) {
    if (v != v) v = -INFINITY;
    const uint32_t b = __float_as_uint(v == 0.f ? 0.f : v);  // -0 and 0 are equal
    const uint32_t k = b & 0x80000000u ? ~b : b | 0x80000000u;
    return ((uint64_t)k << 32) | (uint32_t)~i;
}

__device__ __forceinline__ double block_add(double v, double* s) {
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    double t = 0;
    for (int i = 0; i < kScoreThreads / 32; ++i) t += s[i];
    return t;
}
__device__ __forceinline__ uint64_t block_max(uint64_t v, uint64_t* s) {
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    uint64_t t = 0;
    for (int i = 0; i < kScoreThreads / 32; ++i) t = max(t, s[i]);
    return t;
}

__global__ void __launch_bounds__(kScoreThreads) token_scores_kernel(const ScoreArgs a) {
    __shared__ double s_d[32];
    __shared__ uint64_t s_k[32];
    const float* x = a.x + (int64_t)blockIdx.x * a.ld;
    const int token = a.tokens ? a.tokens[blockIdx.x] : -1;
    const bool known = token >= 0 && token < a.vocab;
    const uint64_t mine = known ? order_key(x[token], token) : ~0ull;
    uint64_t best = 0;
    double nan = 0, before = 0;
    for (int i = threadIdx.x; i < a.vocab; i += kScoreThreads) {
        const uint64_t k = order_key(x[i], i);
        best = max(best, k);
        before += k > mine;
        nan += x[i] != x[i];
    }
    best = block_max(best, s_k);
    before = block_add(before, s_d);
    nan = block_add(nan, s_d);
    const float m = nan > 0 ? NAN : x[(uint32_t)~best];
    double l = 0, lc = 0;
    for (int i = threadIdx.x; i < a.vocab; i += kScoreThreads) {
        const float c = x[i] - m, e = expf(c);
        l += e;
        if (e > 0) lc += (double)e * c;
    }
    l = block_add(l, s_d);
    lc = block_add(lc, s_d);
    const bool none = !(m > -INFINITY && m < INFINITY);  // no distribution
    const float log_l = none ? NAN : (float)log(l);
    if (threadIdx.x == 0) {
        if (a.logprob) a.logprob[blockIdx.x] = known ? (x[token] - m) - log_l : NAN;
        if (a.rank) a.rank[blockIdx.x] = known ? (int)before : -1;
        if (a.entropy) a.entropy[blockIdx.x] = none ? NAN : (float)(log(l) - lc / l);
    }
    uint64_t last = ~0ull;
    for (int j = 0; j < a.top_k; ++j) {
        uint64_t k = 0;
        for (int i = threadIdx.x; i < a.vocab; i += kScoreThreads) {
            const uint64_t c = order_key(x[i], i);
            if (c < last) k = max(k, c);
        }
        last = block_max(k, s_k);
        if (threadIdx.x == 0) {
            const int i = (int)(uint32_t)~last;
            a.top_ids[(int64_t)blockIdx.x * a.top_k + j] = i;
            a.top_logprobs[(int64_t)blockIdx.x * a.top_k + j] = (x[i] - m) - log_l;
        }
    }
}

}  // namespace serve
}  // namespace cllm
