// Host-side helpers of the translation units that implement the C ABI: status macros, the device
// scope, and device buffers whose allocations the failure injection of the tests can reach.
#pragma once

#include <cuda_runtime.h>

#include "common.h"

namespace stt {

#define CUDA_TRY(expr)                                                                              \
    do {                                                                                            \
        cudaError_t e_ = (expr);                                                                    \
        if (e_ != cudaSuccess)                                                                      \
            return set_error(STT_E_CUDA, "%s failed: %s (%s:%d)", #expr, cudaGetErrorString(e_),    \
                             __FILE__, __LINE__);                                                   \
    } while (0)

#define TRY(expr)                  \
    do {                           \
        int rc_ = (expr);          \
        if (rc_ != STT_OK) return rc_; \
    } while (0)

// cudaMalloc and cudaHostAlloc behind the allocation-failure injection (stt_debug_fail_allocation).
cudaError_t dev_alloc(void** p, size_t bytes);
cudaError_t host_alloc(void** p, size_t bytes);

// An allocation: out of memory is STT_E_OOM, any other failure STT_E_CUDA.
#define ALLOC_TRY(expr)                                                                             \
    do {                                                                                            \
        cudaError_t e_ = (expr);                                                                    \
        if (e_ != cudaSuccess) {                                                                    \
            (void)cudaGetLastError();                                                               \
            return set_error(e_ == cudaErrorMemoryAllocation ? STT_E_OOM : STT_E_CUDA,              \
                             "%s failed: %s (%s:%d)", #expr, cudaGetErrorString(e_), __FILE__,      \
                             __LINE__);                                                             \
        }                                                                                           \
    } while (0)

// Makes `dev` the calling thread's current device and restores the one before on scope exit.
struct DeviceScope {
    int prev = 0;
    bool ok = false, moved = false;
    explicit DeviceScope(int dev) {
        if (cudaGetDevice(&prev) != cudaSuccess) return;
        // (a thread that has made no call yet has device 0 as current, without a context: set it)
        thread_local bool set = false;
        if (prev == dev && set) {
            ok = true;
            return;
        }
        ok = set = moved = cudaSetDevice(dev) == cudaSuccess;
    }
    ~DeviceScope() {
        if (moved && cudaSetDevice(prev) != cudaSuccess) (void)cudaGetLastError();
    }
};

// Device buffer that grows on demand.
struct DevBuf {
    void* p = nullptr;
    size_t cap = 0;
    void release() {
        if (p) cudaFree(p);
        p = nullptr;
        cap = 0;
    }
    int ensure(size_t bytes) {
        if (bytes <= cap) return STT_OK;
        if (p) cudaFree(p);
        p = nullptr;
        cap = 0;
        ALLOC_TRY(dev_alloc(&p, bytes));
        cap = bytes;
        return STT_OK;
    }
    ~DevBuf() {
        if (p) cudaFree(p);
    }
};

}  // namespace stt
