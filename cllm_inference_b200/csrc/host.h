// Host-side services of cllm_cuda.cu for the library's other translation
// units: the calling thread's error message, the device check and the
// per-device workspace (one workspace and one lock for the whole library).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <mutex>

#include "../../include/cllm_cuda.h"

namespace cllm {

// Record the message of the calling thread's failure; returns `code`.
int host_fail(int code, const char* fmt, ...);

// The current device, checked for sm_100, and its SM count.
int host_device(int* dev, int* sms);

// The device's workspace of at least `bytes` for kernels on `st`; keep `lk`
// until every one that uses it is enqueued.
int host_workspace(int dev, size_t bytes, cudaStream_t st, uint8_t** out, std::unique_lock<std::mutex>& lk);

// Device status bits of the serving operators' translation unit.
constexpr int kServeTimeout = 1;   // a bounded wait expired
constexpr int kServeBadPage = 2;   // a page id or a position outside the cache

// Read and clear those bits on the current device (which must be idle).
int serve_take_status(int* bits);

#define CLLM_HOST_TRY(expr)                                                                              \
    do {                                                                                                 \
        cudaError_t e_ = (expr);                                                                         \
        if (e_ != cudaSuccess)                                                                           \
            return ::cllm::host_fail(CLLM_ERR_CUDA, "%s failed: %s", #expr, cudaGetErrorString(e_));     \
    } while (0)

}  // namespace cllm
