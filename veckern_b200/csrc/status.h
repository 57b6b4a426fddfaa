// The error convention of the C ABI (int status + the thread's message for vk_last_error) and the device-memory
// helpers that its implementation files share.
#pragma once
#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <string>

#include <cuda_runtime.h>

#include "../../include/vk_abi.h"

namespace vk_status {

inline thread_local std::string g_error;

inline int fail(int code, const char* fmt, ...) {
    char buf[1024];
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    g_error = buf;
    return code;
}

#define VK_TRY_CUDA(call)                                                                                  \
    do {                                                                                                   \
        const cudaError_t e_ = (call);                                                                     \
        if (e_ != cudaSuccess) return fail(e_ == cudaErrorMemoryAllocation ? VK_ERR_NOMEM : VK_ERR_CUDA, \
                                           "%s failed: %s", #call, cudaGetErrorString(e_));                \
    } while (0)

#define VK_TRY(call)                    \
    do {                                \
        const int r_ = (call);          \
        if (r_ != VK_OK) return r_;     \
    } while (0)

// Restores the caller's current device on scope exit.
struct DeviceGuard {
    int prev = -1;
    cudaError_t err = cudaSuccess;
    explicit DeviceGuard(int dev) {
        cudaGetDevice(&prev);
        if (prev != dev) err = cudaSetDevice(dev);
    }
    ~DeviceGuard() {
        int cur = -1;
        cudaGetDevice(&cur);
        if (prev >= 0 && cur != prev) cudaSetDevice(prev);
    }
};

template <typename T>
struct DevBuf {
    T* ptr = nullptr;
    size_t cap = 0;  // elements
    ~DevBuf() { release(); }
    void release() {
        if (ptr) cudaFree(ptr);
        ptr = nullptr;
        cap = 0;
    }
    // Grows (never shrinks), like the reference's DeviceBuffer::ensure (src/cuda/searcher.cu:31-37).
    int ensure(size_t count) {
        if (count <= cap) return VK_OK;
        release();
        const cudaError_t e = cudaMalloc(&ptr, std::max<size_t>(count, 1) * sizeof(T));
        if (e != cudaSuccess) {
            ptr = nullptr;
            return fail(VK_ERR_NOMEM, "cudaMalloc of %zu bytes failed: %s", count * sizeof(T), cudaGetErrorString(e));
        }
        cap = count;
        return VK_OK;
    }
};

}  // namespace vk_status

using vk_status::DevBuf;
using vk_status::DeviceGuard;
using vk_status::fail;
