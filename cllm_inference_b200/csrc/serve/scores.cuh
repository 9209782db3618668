// What a sampler reports of a row of logits (cllm_cuda_token_scores): log
// probability and rank of a token, entropy, the top_k entries.
//
// One pass over the row, which bounds it: 4 bytes a logit from HBM, so an SM has
// 22 issue slots per 32 logits, and this takes 22 (top 20), issued in two cycles of
// three: 512 rows of 128256 69 us, 3.8 TB/s (59 % of a copy's rate).  One row takes
// 9 us on the GPU: the launch, its eight CTAs' reading and the join of their lists.
//   * softmax: each thread keeps a reference instead of the maximum; it moves only
//     when a logit exceeds it by 14, so the sums are hardly ever rescaled.  With c
//     = x - reference (exact or nearly so): l += exp(c), lc += exp(c) * c, fp32.
//   * top_k: an entry can be among the first k only if it is not behind a bound
//     that k entries are known to reach: the k-th of the best lanes (a lane's best
//     so far) of each warp, renewed after 2, 8 and 32 periods.  What
//     reaches it (some hundreds of 128256) goes to a list; at the end the list is pruned once more and each entry counts the
//     entries before it.  A list that overflows (logits in ascending order) is
//     replaced by k searches of the row.
//   * rank: a compare and an add per logit; what equals the token's logit counts
//     before the token only, i.e. the threshold behind it is the next number up.
// Order is a 64-bit key (value, then lower index), so no result depends on the
// order in which threads append.  Few rows: a cluster of up to 8 CTAs shares a row
// and rank 0 joins the parts through distributed shared memory.
#pragma once
#include <cooperative_groups.h>

#include <cfloat>

#include "kv4_format.cuh"

namespace cllm {
namespace serve {

constexpr int kScoreThreads = 256, kScoreWarps = kScoreThreads / 32;
constexpr int kScoreList = 4096;   // entries of a CTA's list
constexpr int kScoreGroups = 4;    // groups of four logits a thread has in flight
constexpr int kMaxTop = 32;
constexpr int kBestLanes = 1 + kMaxTop / kScoreWarps;  // of a warp, at most, that a bound is taken from

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
// descending, index ascending); NaN counts as -inf, -0 as 0.
__device__ __forceinline__ uint64_t order_key(float v, int i) {
    if (v != v) v = -INFINITY;
    const uint32_t b = __float_as_uint(v == 0.f ? 0.f : v);
    const uint32_t k = b & 0x80000000u ? ~b : b | 0x80000000u;
    return ((uint64_t)k << 32) | (uint32_t)~i;
}
// The value of a key; -inf for 0, which every key reaches.
__device__ __forceinline__ float key_value(uint64_t key) {
    if (key == 0) return -INFINITY;
    const uint32_t k = (uint32_t)(key >> 32);
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
__device__ __forceinline__ float exp2_score(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint64_t warp_max(uint64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max(v, (uint64_t)__shfl_xor_sync(0xFFFFFFFFu, (unsigned long long)v, o));
    return v;
}

// Sums around `from` to sums around `to`; nothing is left where they are more than fp32 apart.
__device__ __forceinline__ void moved(float from, float to, float* l, float* lc) {
    const float by = fmaxf(from - to, -1e30f), k = exp2_score(by * 1.44269504088896340736f);
    *lc = *l == 0.f ? 0.f : k * fmaf(*l, by, *lc);
    *l *= k;
}

struct ScorePart {  // what a CTA knows of its part of the row
    float ref, l, lc;
    int before;
    uint64_t top[kMaxTop];
};
struct ScoreSmem {
    alignas(16) uint64_t list[kScoreList];  // while reading: logit (low word) and index; then keys
    uint64_t warp_key[kScoreWarps];
    uint64_t best[kScoreWarps * kBestLanes];
    uint64_t bound;
    float ref[kScoreWarps], l[kScoreWarps], lc[kScoreWarps];
    int before[kScoreWarps];
    int count;
    uint64_t top[kMaxTop];  // of the list, of the joined lists
    ScorePart part;
};

// A key that k keys reach: the k-th of the best lanes of each warp (`best`: a
// lane's key, 0 for none).  0 where there are fewer than k.  Whole CTA.
__device__ __noinline__ uint64_t reach_bound(uint64_t best, int k, ScoreSmem& sm) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, lanes = 1 + (k + kScoreWarps - 1) / kScoreWarps;
    uint32_t value = (uint32_t)(best >> 32), index = (uint32_t)best;
    __syncthreads();
    for (int i = 0; i < lanes; ++i) {
        const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, value);
        const int from = __ffs(__ballot_sync(0xFFFFFFFFu, value == top)) - 1;
        const uint32_t at = __shfl_sync(0xFFFFFFFFu, index, from);
        if (lane == from) {
            sm.best[warp * lanes + i] = top ? ((uint64_t)top << 32) | at : 0;
            value = 0;
        }
    }
    if (threadIdx.x == 0) sm.bound = 0;
    __syncthreads();
    const int n = kScoreWarps * lanes;
    if ((int)threadIdx.x < n) {
        const uint64_t mine = sm.best[threadIdx.x];
        int before = 0;
#pragma unroll 8
        for (int i = 0; i < n; ++i) before += sm.best[i] > mine;
        if (mine && before == k - 1) sm.bound = mine;
    }
    __syncthreads();
    return sm.bound;
}

// The first k of n keys (all different) of `list` into out, in order; entries there are too few of stay 0.
__device__ __noinline__ void first_of(const uint64_t* list, int n, int k, uint64_t* out) {
    if ((int)threadIdx.x < k) out[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kScoreThreads) {
        const uint64_t key = list[i];
        int before = 0;
        const ulonglong2* two = reinterpret_cast<const ulonglong2*>(list);
#pragma unroll 8
        for (int m = 0; m < n / 2; ++m) {
            const ulonglong2 y = two[m];
            before += (y.x > key) + (y.y > key);
        }
        if (n & 1) before += list[n - 1] > key;
        if (before < k) out[before] = key;
    }
    __syncthreads();
}

__global__ void __launch_bounds__(kScoreThreads, 4) token_scores_kernel(const ScoreArgs a) {
    namespace cg = cooperative_groups;
    __shared__ ScoreSmem sm;
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = cluster.num_blocks(), part = cluster.block_rank(), row = blockIdx.x / parts;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float* x = a.x + (int64_t)row * a.ld;
    // groups of four at 16-byte boundaries; up to three logits before and after them
    const int head = min(a.vocab, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / 4);
    const int groups = (a.vocab - head) / 4, tail = head + 4 * groups;
    const int g0 = (int)((int64_t)groups * part / parts), g1 = (int)((int64_t)groups * (part + 1) / parts);

    // two periods in registers: one on its way, one worked on
    float4 next[kScoreGroups];
    auto load = [&](int base) {
#pragma unroll
        for (int u = 0; u < kScoreGroups; ++u) {
            const int g = base + u * kScoreThreads + tid;
            if (g < g1) next[u] = __ldcs(reinterpret_cast<const float4*>(x + head) + g);
        }
    };
    load(g0);
    const int token = a.tokens ? a.tokens[row] : -1;
    const bool known = token >= 0 && token < a.vocab;
    float xt = known ? x[token] : INFINITY;
    if (xt != xt) xt = -INFINITY;
    const bool odd = known && !(fabsf(xt) < INFINITY);  // an infinite logit: count by the order itself
    const float above = nextafterf(xt, INFINITY);
    float ref = -FLT_MAX, l = 0.f, lc = 0.f;
    float2 l2 = make_float2(0.f, 0.f), lc2 = make_float2(0.f, 0.f);  // of the groups: even and odd logits
    int before = 0;
    uint64_t bound = 0;
    float best_value = -INFINITY;  // of the logits considered
    int best_index = -1;
    // the bound's value, the next number up for logits behind the bound's index, and that index
    float reach = a.top_k ? -INFINITY : INFINITY, reach_up = reach;
    int reach_to = INT_MAX;
    auto set_bound = [&](uint64_t to) {
        bound = to;
        reach = key_value(to);
        reach_up = to ? nextafterf(reach, INFINITY) : reach;
        reach_to = to ? (int)(uint32_t)~to : INT_MAX;
    };
    if (tid == 0) sm.count = 0;
    __syncthreads();

    auto consider = [&](float v, int i) {  // for the list
        if (v > best_value || best_index < 0) {
            best_value = v;
            best_index = i;
        }
        const int at = atomicAdd(&sm.count, 1);
        if (at < kScoreList) sm.list[at] = ((uint64_t)i << 32) | __float_as_uint(v);
    };
    auto best = [&]() -> uint64_t { return best_index < 0 ? 0 : order_key(best_value, best_index); };  // this lane's
    auto count = [&](float v, int i) {  // for the rank
        if (v != v) v = -INFINITY;
        before += v > xt || (v == xt && i < token);
    };
    auto weigh = [&](float v) {
        const float c = v - ref, e = exp2_score(c * 1.44269504088896340736f);
        l += e;
        lc = fmaf(e, fmaxf(c, -1e30f), lc);  // -inf: 0 * a number
    };
    auto weigh2 = [&](float v, float w) {
        const float2 c = __fadd2_rn(make_float2(v, w), make_float2(-ref, -ref));
        const float2 t = __fmul2_rn(c, make_float2(1.44269504088896340736f, 1.44269504088896340736f));
        const float2 e = make_float2(exp2_score(t.x), exp2_score(t.y));
        l2 = __fadd2_rn(l2, e);
        lc2 = __ffma2_rn(e, make_float2(fmaxf(c.x, -1e30f), fmaxf(c.y, -1e30f)), lc2);
    };
    auto raise = [&](float top) {
        if (top > ref + 14.f) {
            moved(ref, top, &l, &lc);
            moved(ref, top, &l2.x, &lc2.x);
            moved(ref, top, &l2.y, &lc2.y);
            ref = top;
        }
    };
    auto one = [&](int i) {  // a logit outside the groups
        const float v = x[i];
        raise(v);
        weigh(v);
        if (known) count(v, i);
        if (a.top_k) consider(v, i);
    };
    if (part == 0 && tid < head) one(tid);
    if (part == parts - 1 && tid < a.vocab - tail) one(tail + tid);

    constexpr int kPeriod = kScoreGroups * kScoreThreads;
    int period = 0;
    auto four = [&](const float4& v, int i) {
        const float top = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)), least = i > reach_to ? reach_up : reach;
        if (!(top < fminf(least, ref + 14.f))) {
            raise(top);
            if (!(v.x < least)) consider(v.x, i);
            if (!(v.y < least)) consider(v.y, i + 1);
            if (!(v.z < least)) consider(v.z, i + 2);
            if (!(v.w < least)) consider(v.w, i + 3);
        }
        if (odd || (unsigned)(token - i) < 4u) {
            count(v.x, i); count(v.y, i + 1); count(v.z, i + 2); count(v.w, i + 3);
        } else {
            const float at = i < token ? xt : above;
            before += (v.x >= at) + (v.y >= at) + (v.z >= at) + (v.w >= at);
        }
        weigh2(v.x, v.y);
        weigh2(v.z, v.w);
    };
    for (int base = g0; base < g1; base += kPeriod) {
        float4 v[kScoreGroups];
#pragma unroll
        for (int u = 0; u < kScoreGroups; ++u) v[u] = next[u];
        load(base + kPeriod);
        const int g = base + tid;
        if (base == g0 && a.top_k) {  // a first bound, from the first period
            float most = -INFINITY;
            int at = g < g1 ? head + 4 * g : -1;
            auto look = [&](float y, int i) {
                if (y > most) {
                    most = y;
                    at = i;
                }
            };
#pragma unroll
            for (int u = 0; u < kScoreGroups; ++u) {
                const int i = head + 4 * (g + u * kScoreThreads);
                if (g + u * kScoreThreads < g1) {
                    look(v[u].x, i); look(v[u].y, i + 1); look(v[u].z, i + 2); look(v[u].w, i + 3);
                }
            }
            set_bound(reach_bound(max(best(), at < 0 ? 0 : order_key(most, at)), a.top_k, sm));
        }
        if (base + kPeriod <= g1) {
#pragma unroll
            for (int u = 0; u < kScoreGroups; ++u) four(v[u], head + 4 * (g + u * kScoreThreads));
        } else {
#pragma unroll 1
            for (int u = 0; u < kScoreGroups; ++u) {
                if (g + u * kScoreThreads < g1) four(v[0], head + 4 * (g + u * kScoreThreads));
#pragma unroll
                for (int w = 0; w + 1 < kScoreGroups; ++w) v[w] = v[w + 1];
            }
        }
        ++period;
        if (a.top_k && (period == 2 || period == 8 || period == 32) && base + kPeriod < g1) {
            const uint64_t now = reach_bound(best(), a.top_k, sm);
            if (now > bound) set_bound(now);
        }
    }

    // the CTA's sums
    l += l2.x + l2.y;
    lc += lc2.x + lc2.y;
    float m = ref;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    if (lane == 0) sm.ref[warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kScoreWarps; ++w) m = fmaxf(m, sm.ref[w]);
    moved(ref, m, &l, &lc);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
        lc += __shfl_xor_sync(0xFFFFFFFFu, lc, o);
        before += __shfl_xor_sync(0xFFFFFFFFu, before, o);
    }
    if (lane == 0) {
        sm.l[warp] = l;
        sm.lc[warp] = lc;
        sm.before[warp] = before;
    }
    __syncthreads();
    if (tid == 0) {
        float sl = 0.f, slc = 0.f;
        int sb = 0;
        for (int w = 0; w < kScoreWarps; ++w) {
            sl += sm.l[w];
            slc += sm.lc[w];
            sb += sm.before[w];
        }
        sm.part.ref = m;
        sm.part.l = sl;
        sm.part.lc = slc;
        sm.part.before = sb;
    }
    // the CTA's first top_k
    if (a.top_k) {
        int n = sm.count;
        if (n > kScoreList) {  // it overflowed: search the part once for each entry
            uint64_t last = ~0ull;
            for (int k = 0; k < a.top_k; ++k) {
                uint64_t key = 0;
                auto look = [&](int i) {
                    const uint64_t c = order_key(x[i], i);
                    if (c < last) key = max(key, c);
                };
                if (part == 0 && tid < head) look(tid);
                if (part == parts - 1 && tid < a.vocab - tail) look(tail + tid);
                for (int i = head + 4 * g0 + tid; i < head + 4 * g1; i += kScoreThreads) look(i);
                key = warp_max(key);
                __syncthreads();
                if (lane == 0) sm.warp_key[warp] = key;
                __syncthreads();
                last = 0;
                for (int w = 0; w < kScoreWarps; ++w) last = max(last, sm.warp_key[w]);
                if (tid == 0) sm.part.top[k] = last;
            }
        } else {
            uint64_t mine[kScoreList / kScoreThreads], top = 0;
            for (int i = 0; i * kScoreThreads < n; ++i) {
                const int at = i * kScoreThreads + tid;
                if (at < n) top = max(top, sm.list[at] = order_key(__uint_as_float((uint32_t)sm.list[at]), (int)(sm.list[at] >> 32)));
            }
            if (n > kScoreThreads) {  // keep what reaches the bound now
                const uint64_t now = reach_bound(top, a.top_k, sm);
                bound = max(bound, now);
#pragma unroll
                for (int i = 0; i < kScoreList / kScoreThreads; ++i) {
                    const int at = i * kScoreThreads + tid;
                    mine[i] = at < n ? sm.list[at] : 0;
                }
                __syncthreads();
                if (tid == 0) sm.count = 0;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < kScoreList / kScoreThreads; ++i)
                    if (mine[i] && mine[i] >= bound) sm.list[atomicAdd(&sm.count, 1)] = mine[i];
                __syncthreads();
                n = sm.count;
            }
            first_of(sm.list, n, a.top_k, sm.part.top);
        }
    }
    cluster.sync();
    if (part == 0) {
        m = sm.part.ref;
        for (int p = 1; p < parts; ++p) m = fmaxf(m, cluster.map_shared_rank(&sm.part, p)->ref);
        l = lc = 0.f;
        before = 0;
        for (int p = 0; p < parts; ++p) {
            const ScorePart* q = cluster.map_shared_rank(&sm.part, p);
            float pl = q->l, plc = q->lc;
            moved(q->ref, m, &pl, &plc);
            l += pl;
            lc += plc;
            before += q->before;
        }
        const float log_l = l == 0.f ? NAN : logf(l);  // nothing but -inf: no distribution
        if (tid == 0) {
            if (a.logprob) a.logprob[row] = known ? (x[token] - m) - log_l : NAN;
            if (a.rank) a.rank[row] = known ? before : -1;
            if (a.entropy) a.entropy[row] = log_l - lc / l;
        }
        if (a.top_k) {
            const uint64_t* top = sm.part.top;
            if (parts > 1) {
                for (int i = tid; i < parts * a.top_k; i += kScoreThreads)
                    sm.list[i] = cluster.map_shared_rank(&sm.part, i / a.top_k)->top[i % a.top_k];
                __syncthreads();
                first_of(sm.list, parts * a.top_k, a.top_k, sm.top);
                top = sm.top;
            }
            if (tid < a.top_k) {
                const int i = (int)(uint32_t)~top[tid];  // top_k <= vocab, so there is an entry
                a.top_ids[(int64_t)row * a.top_k + tid] = i;
                a.top_logprobs[(int64_t)row * a.top_k + tid] = (unsigned)i < (unsigned)a.vocab ? (x[i] - m) - log_l : NAN;
            }
        }
    }
    cluster.sync();  // the other parts' memory stays until it has been read
}

}  // namespace serve
}  // namespace cllm
