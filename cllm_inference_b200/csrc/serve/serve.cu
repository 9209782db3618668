// C ABI of the serving operators (include/cllm_cuda.h, "Serving many
// sequences"): argument checks, workspace layout and launches.  A translation
// unit of its own beside cllm_cuda.cu, whose host services it uses (host.h).
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "kv4_append.cuh"
#include "kv4_decode.cuh"
#include "kv4_format.cuh"
#include "kv4_pages.cuh"
#include "kv4_prompt.cuh"
#include "scores.cuh"

namespace cllm {

int serve_take_status(int* bits) {
    int zero = 0;
    CLLM_HOST_TRY(cudaMemcpyFromSymbol(bits, serve::g_serve_status, sizeof(int)));
    CLLM_HOST_TRY(cudaMemcpyToSymbol(serve::g_serve_status, &zero, sizeof(int)));
    return CLLM_OK;
}

namespace serve {
namespace {

size_t align256(size_t v) { return (v + 255) & ~size_t(255); }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_geometry(const char* who, int n_pages, int page_len, int n_head_kv, int head_dim) {
    if (head_dim != 64 && head_dim != 128)
        return host_fail(CLLM_ERR_INVALID_ARG, "%s: head_dim %d (64 or 128)", who, head_dim);
    if (page_len <= 0 || page_len % kTile || page_len > 4096)
        return host_fail(CLLM_ERR_INVALID_ARG, "%s: page_len %d (a multiple of 16, at most 4096)", who, page_len);
    if (n_head_kv <= 0 || n_head_kv > 65535 || n_pages <= 0)
        return host_fail(CLLM_ERR_INVALID_ARG, "%s: bad arguments (%d KV heads, %d pages)", who, n_head_kv, n_pages);
    return CLLM_OK;
}

// Rows (of all heads of a KV head) up to which a sequence is kv4_rows_kernel's.  Its time grows with every 8 rows, the
// prompt kernel's only with every 128.  8 KV heads of 128, us, rows kernel / prompt kernel at 16, 40, 48, 64 rows:
//   16 sequences of 1024 positions    33/64    55/65    63/67    76/67
//   64 of 1024                        78/167   160/171  187/173  244/179
//   16 of 8192                        119/239  260/241  309/245  402/245
//   64 of 4096                        219/452  506/462  602/462  796/468
constexpr int kRowsMax = 40;
// A call of no more steps (of 8 rows, 128 positions, a KV head) for each of its CTAs is the rows kernel's alone.  8 KV
// heads of 128 (64), us, rows kernel / prompt kernel, 444 CTAs:
//   128 rows on 2048 positions, 2048 steps               33/50 (26/38)
//   1024 on 500, 512 on 1024 or 128 on 4096, 4096 steps  51/46, 45/50, 43/54 (38/38, 33/38, 33/40)
//   4 sequences of 192 on 1024, 6144 steps               61/56 (43/42)
//   1024 on 1024 or 256 on 4096, 8192 steps              78/54, 68/56 (53/42, 47/42)
// Where the sizes alone show it, the launches that look for prompts are left out.
constexpr int kRowsAllSteps = 10;

// Launch `kern` so that it may start before the kernel before it is done (programmatic
// dependent launch); it waits with griddepcontrol.wait where it needs to.
template <class... KArgs>
int launch_early(void (*kern)(KArgs...), int ctas, int threads, size_t smem, cudaStream_t st, const std::common_type_t<KArgs>&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute pdl[1];
    pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = pdl;
    cfg.numAttrs = 1;
    CLLM_HOST_TRY(cudaLaunchKernelEx(&cfg, kern, args...));
    return CLLM_OK;
}

int g_set[64];  // of g_rows_arrived, the last call's; host_workspace's lock guards it

template <int HD>
int launch_attention(AttnArgs a, int dev, int sms, cudaStream_t st) {
    static std::once_flag once[64];
    static void* nan_tile[64];
    static cudaError_t ready[64];
    std::call_once(once[dev], [dev] {
        cudaError_t& attr = ready[dev];
        attr = cudaGetSymbolAddress(&nan_tile[dev], g_nan_tile);
        if (attr == cudaSuccess)
            attr = cudaFuncSetAttribute(kv4_rows_kernel<HD, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(RowsSmem<HD>));
        if (attr == cudaSuccess)
            attr = cudaFuncSetAttribute(kv4_rows_kernel<HD, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        sizeof(RowsSmem<HD>));
        if (attr == cudaSuccess)
            attr = cudaFuncSetAttribute(kv4_prompt_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        sizeof(PromptSmem<HD>) + 1024);
    });
    CLLM_HOST_TRY(ready[dev]);
    a.nan_tile = static_cast<const uint8_t*>(nan_tile[dev]);
    const int ctas = std::min(kMaxRowCtas, kRowCtasPerSm * sms);
    const int64_t rows = (int64_t)a.n_tok * a.rep, groups = rows / kRowTile + a.c.n_seqs;  // at most
    const int64_t steps = ((int64_t)a.c.max_pages * a.c.page_len + kStepLen - 1) / kStepLen;
    a.all_steps = kRowsAllSteps * ctas;
    const bool prompts = a.q_begin && rows > a.rows_max && (groups > a.all_steps || groups * a.c.n_kv * steps > a.all_steps);
    // blocks of rows of sequences with more rows than rows_max: at most
    const int64_t most = prompts ? rows / kPromptRows + std::min<int64_t>(a.c.n_seqs, rows / (a.rows_max + 1)) : 0;
    if (most > INT_MAX / 2) return host_fail(CLLM_ERR_TOO_LARGE, "kv4_attention: too many rows in one call");

    size_t bytes = 0;
    auto part = [&](size_t n) {
        const size_t at = bytes;
        bytes += align256(n);
        return at;
    };
    const size_t r_ml = part((size_t)2 * ctas * kRowTile * 2 * 4);
    const size_t r_o = part((size_t)2 * ctas * kRowTile * HD * 4);
    const size_t p_items = part(prompts ? sizeof(PromptItem) * (most + 1) : 0), p_seq = part(prompts ? 4 * (size_t)a.c.n_seqs : 0);
    const size_t p_count = part(256), p_arrived = part(4 * (size_t)sms);
    const size_t p_ml = part(prompts ? (size_t)2 * sms * kPromptRows * 2 * 4 : 0), p_bad = part(prompts ? (size_t)2 * sms * kPromptRows * 4 : 0);
    const size_t p_o = part(prompts ? (size_t)2 * sms * kPromptRows * HD * 4 : 0);
    uint8_t* ws;
    std::unique_lock<std::mutex> lk;
    if (int rc = host_workspace(dev, bytes, st, &ws, lk)) return rc;

    RowsArgs ra{a, g_set[dev] ^= 1, reinterpret_cast<float*>(ws + r_ml), reinterpret_cast<float*>(ws + r_o)};
    PromptArgs pa{};
    if (prompts) {
        pa.a = a;
        pa.most = (int)most;
        pa.items = reinterpret_cast<PromptItem*>(ws + p_items);
        pa.seq_items = reinterpret_cast<int*>(ws + p_seq);
        pa.count = reinterpret_cast<int*>(ws + p_count);
        pa.ctas = sms;
        pa.arrived = reinterpret_cast<unsigned*>(ws + p_arrived);
        pa.part_ml = reinterpret_cast<float*>(ws + p_ml);
        pa.part_bad = reinterpret_cast<uint32_t*>(ws + p_bad);
        pa.part_o = reinterpret_cast<float*>(ws + p_o);
        prompt_plan_kernel<<<1, kPromptPlanThreads, 0, st>>>(pa);
        kv4_rows_kernel<HD, false><<<ctas, kRowThreads, sizeof(RowsSmem<HD>), st>>>(ra);
    } else {
        kv4_rows_kernel<HD, true><<<ctas, kRowThreads, sizeof(RowsSmem<HD>), st>>>(ra);
    }
    CLLM_HOST_TRY(cudaGetLastError());
    if (prompts)
        if (int rc = launch_early(kv4_prompt_kernel<HD>, sms, kPromptThreads, sizeof(PromptSmem<HD>) + 1024, st, pa)) return rc;
    return CLLM_OK;
}

}  // namespace
}  // namespace serve
}  // namespace cllm

using namespace cllm;
using namespace cllm::serve;

extern "C" {

int64_t cllm_cuda_kv4_page_bytes(int page_len, int n_head_kv, int head_dim) {
    if ((head_dim != 64 && head_dim != 128) || page_len <= 0 || page_len % kTile || page_len > 4096 || n_head_kv <= 0)
        return 0;
    return (int64_t)page_len / kTile * n_head_kv * (20 * head_dim);
}

int cllm_cuda_kv4_append(const float* q, int64_t ldq, float* q_out, const float* k, const float* v, int64_t ldkv,
                         int n_tok, int n_head, const float* rope_table, int n_pos, const int* token_seq,
                         const int* token_pos, void* pages, int n_pages, int page_len, int n_head_kv, int head_dim,
                         const int* page_table, int n_seqs, int max_pages, float* k_out, float* v_out, void* stream) {
    if (int rc = check_geometry("kv4_append", n_pages, page_len, n_head_kv, head_dim)) return rc;
    if (n_tok < 0 || n_head < 0 || n_seqs < (n_tok > 0) || max_pages <= 0 || (rope_table && n_pos <= 0))
        return host_fail(CLLM_ERR_INVALID_ARG, "kv4_append: bad sizes");
    if (n_tok == 0) return CLLM_OK;
    if (!k || !v || !token_seq || !token_pos || !pages || !page_table || (n_head > 0 && (!q || !q_out)))
        return host_fail(CLLM_ERR_INVALID_ARG, "kv4_append: null argument");
    if (!aligned16(pages)) return host_fail(CLLM_ERR_INVALID_ARG, "kv4_append: pages must be 16-byte aligned");
    if (ldkv < (int64_t)n_head_kv * head_dim || (n_head > 0 && ldq < (int64_t)n_head * head_dim))
        return host_fail(CLLM_ERR_INVALID_ARG, "kv4_append: a row is shorter than its heads");
    if (n_head > 0 && q_out == q && ldq != (int64_t)n_head * head_dim)
        return host_fail(CLLM_ERR_INVALID_ARG, "kv4_append: q in place needs dense rows");
    int dev, sms;
    if (int rc = host_device(&dev, &sms)) return rc;
    AppendArgs a{};
    a.q = q; a.k = k; a.v = v; a.rope = rope_table;
    a.q_out = q_out; a.k_out = k_out; a.v_out = v_out;
    a.ldq = ldq; a.ldkv = ldkv;
    a.token_seq = token_seq; a.token_pos = token_pos;
    a.n_tok = n_tok; a.n_head = n_head; a.n_pos = n_pos;
    a.vec = aligned16(q) && aligned16(q_out) && aligned16(k) && aligned16(v) && aligned16(k_out) && aligned16(v_out) &&
            ldkv % 4 == 0 && (n_head == 0 || ldq % 4 == 0);
    a.c = Cache{static_cast<uint8_t*>(pages), page_table, nullptr, n_pages, page_len, n_head_kv, n_seqs, max_pages};
    a.rope_vec = aligned16(rope_table);
    // Vectors of a warp: as many as leave 32 warps for every SM, up to 12 steps' worth, in whole rounds of loads.
    // 32 query and 16 other vectors of 128 a token, us at 1 step a warp / 12 / by the rule: 64 tokens 10/14/8, 512
    // 20/16/14, 1024 35/18/18, 2048 61/31/31.
    const int vecs = 128 / head_dim, warps = kAppendThreads / 32;
    const int64_t units = n_head + 2 * n_head_kv, steps = (units + vecs - 1) / vecs;
    const int64_t share = std::min<int64_t>(12, n_tok * steps / (32 * (int64_t)sms));
    a.span = vecs * (int)(share <= 1 ? 1 : (share + kAppendTogether - 1) / kAppendTogether * kAppendTogether);
    const int64_t ctas = (n_tok * ((units + a.span - 1) / a.span) + warps - 1) / warps;
    if (ctas > INT_MAX) return host_fail(CLLM_ERR_TOO_LARGE, "kv4_append: too many tokens in one call");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (head_dim == 128) kv4_append_kernel<128><<<(unsigned)ctas, kAppendThreads, 0, st>>>(a);
    else kv4_append_kernel<64><<<(unsigned)ctas, kAppendThreads, 0, st>>>(a);
    CLLM_HOST_TRY(cudaGetLastError());
    return CLLM_OK;
}

int cllm_cuda_kv4_attention(const float* q, int64_t ldq, const int* q_begin, int n_tok, int n_head, const void* pages,
                            int n_pages, int page_len, int n_head_kv, int head_dim, const int* page_table,
                            const int* seq_len, int n_seqs, int max_pages, float scale, float* out, float* lse,
                            void* stream) {
    if (int rc = check_geometry("kv4_attention", n_pages, page_len, n_head_kv, head_dim)) return rc;
    if (n_tok < 0 || n_head <= 0 || n_head % n_head_kv || n_seqs < (n_tok > 0) || max_pages <= 0 ||
        (int64_t)max_pages * page_len > INT_MAX || !(std::fabs(scale) <= 3e38f))
        return host_fail(CLLM_ERR_INVALID_ARG, "kv4_attention: bad sizes (%d heads over %d KV heads)", n_head, n_head_kv);
    if (!q_begin && n_tok != n_seqs)
        return host_fail(CLLM_ERR_INVALID_ARG, "kv4_attention: %d rows for %d sequences need q_begin", n_tok, n_seqs);
    if (n_tok == 0) return CLLM_OK;
    if (!q || !pages || !page_table || !seq_len || !out)
        return host_fail(CLLM_ERR_INVALID_ARG, "kv4_attention: null argument");
    if (!aligned16(pages) || !aligned16(out))
        return host_fail(CLLM_ERR_INVALID_ARG, "kv4_attention: pages and out must be 16-byte aligned");
    if (ldq < (int64_t)n_head * head_dim)
        return host_fail(CLLM_ERR_INVALID_ARG, "kv4_attention: a row is shorter than its heads");
    if ((int64_t)n_pages * n_head_kv > (int64_t)0xFFFFFFFE / (page_len / kTile))
        return host_fail(CLLM_ERR_TOO_LARGE, "kv4_attention: a layer of more than 2^32 tiles");
    int dev, sms;
    if (int rc = host_device(&dev, &sms)) return rc;
    AttnArgs a{};
    a.q = q; a.ldq = ldq; a.q_begin = q_begin; a.n_tok = n_tok; a.n_head = n_head; a.rep = n_head / n_head_kv;
    a.rows_max = std::max(kRowsMax, a.rep);
    a.scale = scale == 0.f ? 1.f / std::sqrt((float)head_dim) : scale;
    a.out = out; a.lse = lse;
    a.c = Cache{const_cast<uint8_t*>(static_cast<const uint8_t*>(pages)), page_table, seq_len, n_pages, page_len,
                n_head_kv, n_seqs, max_pages};
    a.page_tiles = page_len / kTile;
    a.page_magic = (uint32_t)(((uint64_t(1) << 32) + a.page_tiles - 1) / a.page_tiles);
    return head_dim == 128 ? launch_attention<128>(a, dev, sms, static_cast<cudaStream_t>(stream))
                           : launch_attention<64>(a, dev, sms, static_cast<cudaStream_t>(stream));
}

static int pages_call(const char* who, PagesArgs a, void* pages, int64_t page_bytes, bool fork, void* stream) {
    if (a.n_layers <= 0 || a.n_pages <= 0 || a.page_len <= 0 || a.page_len % kTile || a.max_pages <= 0 ||
        page_bytes <= 0 || page_bytes % 16 || page_bytes > (int64_t(1) << 34) || (int64_t)a.max_pages * a.page_len > INT_MAX)
        return host_fail(CLLM_ERR_INVALID_ARG, "%s: bad sizes", who);
    if (!aligned16(pages)) return host_fail(CLLM_ERR_INVALID_ARG, "%s: pages must be 16-byte aligned", who);
    int dev, sms;
    if (int rc = host_device(&dev, &sms)) return rc;
    a.pages = static_cast<uint8_t*>(pages);
    a.page_bytes = page_bytes;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // Tables that a CTA can hold: one launch instead of four.  8 sequences of 17 pages 11.3 us instead of 16.9, 192 of 8
    // 16.5 instead of 21.3, compact of 96 of 14 in a pool of 2048 55.3 instead of 60.6.
    if (a.n_pages <= kSmallPages && a.n_new <= kSmallSeqs && (int64_t)a.n_new * a.max_pages <= kSmallEntries &&
        a.table_out != a.table) {
        static std::once_flag once[64];
        cudaError_t attr = cudaSuccess;
        std::call_once(once[dev], [&] {
            attr = cudaFuncSetAttribute(fork_small_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(SmallPlan));
            if (attr == cudaSuccess)
                attr = cudaFuncSetAttribute(compact_small_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(SmallPlan));
        });
        CLLM_HOST_TRY(attr);
        if (fork) fork_small_kernel<<<sms, kSmallThreads, sizeof(SmallPlan), st>>>(a);
        else compact_small_kernel<<<sms, kSmallThreads, sizeof(SmallPlan), st>>>(a);
        CLLM_HOST_TRY(cudaGetLastError());
        return CLLM_OK;
    }
    const size_t words = ((size_t)a.n_pages + 31) / 32, n = (size_t)a.n_pages;
    const size_t bits = align256(4 * words), list = align256(4 * n), pairs = align256(8 * n);
    const size_t seqs = align256(4 * (size_t)a.n_new);
    uint8_t* ws;
    std::unique_lock<std::mutex> lk;
    if (int rc = host_workspace(dev, 2 * bits + 3 * list + pairs + 2 * seqs + 256, st, &ws, lk)) return rc;
    auto take = [&](size_t bytes) {
        uint8_t* p = ws;
        ws += bytes;
        return p;
    };
    uint8_t* ones = ws;
    a.free_bits = reinterpret_cast<uint32_t*>(take(bits));
    a.part_bits = reinterpret_cast<uint32_t*>(take(bits));
    a.owner = reinterpret_cast<uint32_t*>(take(list));
    a.ids = reinterpret_cast<int*>(take(list));
    a.moved = reinterpret_cast<int*>(take(list));
    a.copies = reinterpret_cast<int2*>(take(pairs));
    a.first = reinterpret_cast<int*>(take(seqs));
    a.held = reinterpret_cast<int*>(take(seqs));
    a.count = reinterpret_cast<int*>(take(256));
    CLLM_HOST_TRY(cudaMemsetAsync(ones, 0xFF, 2 * bits + list, st));
    const dim3 mark(a.n_new, (a.max_pages + 1023) / 1024);
    if (mark.y > 65535) return host_fail(CLLM_ERR_TOO_LARGE, "%s: %d pages per sequence", who, a.max_pages);
    const unsigned apply = (unsigned)a.n_new + 8u * (unsigned)sms;
    if (fork) {
        fork_mark_kernel<<<mark, 256, 0, st>>>(a);
        fork_plan_kernel<<<1, kPlanThreads, 0, st>>>(a);
        fork_apply_kernel<<<apply, kCopyThreads, 0, st>>>(a);
    } else {
        compact_mark_kernel<<<mark, 256, 0, st>>>(a);
        compact_plan_kernel<<<1, kPlanThreads, 0, st>>>(a);
        compact_apply_kernel<<<apply, kCopyThreads, 0, st>>>(a);
    }
    CLLM_HOST_TRY(cudaGetLastError());
    return CLLM_OK;
}

int cllm_cuda_kv4_fork(void* pages, int n_layers, int n_pages, int64_t page_bytes, int page_len,
                       const int* page_table, const int* seq_len, int n_old, const int* source, const int* new_len,
                       int n_new, int max_pages, int* table_out, int* len_out, void* stream) {
    if (n_old < (n_new > 0) || n_new < 0) return host_fail(CLLM_ERR_INVALID_ARG, "kv4_fork: bad sizes");
    if (n_new == 0) return CLLM_OK;
    if (!pages || !page_table || !seq_len || !source || !new_len || !table_out || !len_out)
        return host_fail(CLLM_ERR_INVALID_ARG, "kv4_fork: null argument");
    if (table_out == page_table || len_out == seq_len || len_out == source || len_out == new_len)
        return host_fail(CLLM_ERR_INVALID_ARG, "kv4_fork: the new table and lengths need buffers of their own");
    PagesArgs a{};
    a.n_layers = n_layers; a.n_pages = n_pages; a.page_len = page_len; a.max_pages = max_pages;
    a.table = page_table; a.seq_len = seq_len; a.source = source; a.new_len = new_len;
    a.n_old = n_old; a.n_new = n_new; a.table_out = table_out; a.len_out = len_out;
    return pages_call("kv4_fork", a, pages, page_bytes, true, stream);
}

int cllm_cuda_kv4_compact(void* pages, int n_layers, int n_pages, int64_t page_bytes, int page_len,
                          const int* page_table, const int* seq_len, int n_seqs, int max_pages, int* table_out,
                          int* n_live, void* stream) {
    if (n_seqs <= 0) return host_fail(CLLM_ERR_INVALID_ARG, "kv4_compact: bad sizes");
    if (!pages || !page_table || !seq_len || !table_out || !n_live)
        return host_fail(CLLM_ERR_INVALID_ARG, "kv4_compact: null argument");
    PagesArgs a{};
    a.n_layers = n_layers; a.n_pages = n_pages; a.page_len = page_len; a.max_pages = max_pages;
    a.table = page_table; a.seq_len = seq_len; a.n_old = a.n_new = n_seqs; a.table_out = table_out; a.n_live = n_live;
    return pages_call("kv4_compact", a, pages, page_bytes, false, stream);
}

int cllm_cuda_token_scores(const float* logits, int64_t ld, int rows, int vocab, const int* tokens, int top_k,
                           float* logprob, float* entropy, int* rank, int* top_ids, float* top_logprobs,
                           void* stream) {
    if (rows < 0 || vocab <= 0 || (ld < vocab && ld != 0)) return host_fail(CLLM_ERR_INVALID_ARG, "token_scores: bad sizes");
    if (top_k < 0 || top_k > CLLM_MAX_TOP_K || top_k > vocab)
        return host_fail(CLLM_ERR_INVALID_ARG, "token_scores: top_k %d (0 to %d, at most the vocabulary)", top_k,
                         CLLM_MAX_TOP_K);
    if (rows == 0) return CLLM_OK;
    if (!logits || (top_k > 0 && (!top_ids || !top_logprobs)) || ((logprob || rank) && !tokens))
        return host_fail(CLLM_ERR_INVALID_ARG, "token_scores: null argument");
    int dev, sms;
    if (int rc = host_device(&dev, &sms)) return rc;
    ScoreArgs a{logits, ld, rows, vocab, top_k, tokens, logprob, entropy, rank, top_ids, top_logprobs};
    // CTAs per row (a cluster): what makes the slowest SM's share shortest.  Measured, in cycles: 15000 for what a
    // CTA does besides reading (bounds, list, join), then 0.19 a logit for each of the up to four CTAs that share an
    // SM's bandwidth, 0.25 at least.  512 rows of 128256: 1 CTA a row 68 us, 2 (two waves) 77.
    int parts = 1;
    double best = 0;
    for (int p = 1; p <= 8 && (p == 1 || vocab / p >= 4096); p *= 2) {
        const double ctas = (double)rows * p, waves = std::ceil(ctas / (4.0 * sms)), share = std::min(4.0, std::ceil(ctas / sms));
        const double cycles = waves * (15000 + std::max(0.25, 0.19 * share) * vocab / p);
        if (p == 1 || cycles < best) {
            best = cycles;
            parts = p;
        }
    }
    if ((int64_t)rows * parts > INT_MAX) return host_fail(CLLM_ERR_TOO_LARGE, "token_scores: too many rows");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * parts));
    cfg.blockDim = dim3(kScoreThreads);
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    CLLM_HOST_TRY(cudaLaunchKernelEx(&cfg, token_scores_kernel, a));
    return CLLM_OK;
}

}  // extern "C"
