// The 4-bit cache's tile (include/cllm_cuda.h, "Serving many sequences") and
// what the kernels that read or write it share.
//
// The order of the numbers inside a tile is the order in which the tensor-core
// instructions of attention want them: a lane's operand words are one 16-byte
// (head_dim 64: 8-byte) shared-memory load, and no number has to change place
// in a register.  See kv4_decode.cuh.
#pragma once
#include "../common.cuh"
#include "../host.h"

namespace cllm {
namespace serve {

constexpr int kTile = 16;  // positions of a tile

// Bits of kServe*, set by kernels, read and cleared by serve_take_status.
__device__ int g_serve_status;

template <int HD>
struct Tile {
    static constexpr int G = HD / 32;              // groups of a vector
    static constexpr uint32_t kNibbles = 8 * HD;   // bytes of the keys' (or the values') numbers
    static constexpr uint32_t kV = kNibbles;
    static constexpr uint32_t kScaleK = 2 * kNibbles;
    static constexpr uint32_t kScaleV = kScaleK + 2 * HD;
    static constexpr uint32_t kBytes = 20 * HD;
};

// What attention reads for a page that does not exist: a tile whose scales are
// all NaN, so the rows that see it are NaN.  All bits set, for either head_dim.
struct NanTile {
    uint64_t bits[Tile<128>::kBytes / 8];
    constexpr NanTile() : bits() {
        for (uint64_t& b : bits) b = ~0ull;
    }
};
__device__ const NanTile g_nan_tile alignas(128);

// One layer's pool and the sequences in it.
struct Cache {
    uint8_t* pages;
    const int* table;    // [n_seqs][max_pages]
    const int* seq_len;  // [n_seqs] (nullptr: append)
    int n_pages, page_len, n_kv, n_seqs, max_pages;

    __device__ __forceinline__ int length(int s) const {
        const int n = max(0, seq_len[s]);
        const int64_t most = (int64_t)max_pages * page_len;
        if (n > most) {
            atomicOr(&g_serve_status, kServeBadPage);
            return (int)most;
        }
        return n;
    }
    // Page of slot i of sequence s; -1 (and the status) for an id outside the pool.
    __device__ __forceinline__ int page(int s, int i) const {
        const int id = table[(int64_t)s * max_pages + i];
        if ((unsigned)id < (unsigned)n_pages) return id;
        atomicOr(&g_serve_status, kServeBadPage);
        return -1;
    }
    // First byte of the tile that holds slot-local position `at` of head h in page `id`.
    template <int HD>
    __device__ __forceinline__ uint8_t* tile(int id, int h, int at) const {
        return pages + ((int64_t)id * n_kv + h) * (page_len / kTile) * (int64_t)Tile<HD>::kBytes +
               (at / kTile) * (int64_t)Tile<HD>::kBytes;
    }
};

}  // namespace serve
}  // namespace cllm
