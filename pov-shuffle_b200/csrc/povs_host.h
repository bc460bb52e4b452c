// Host helpers shared by the C ABI's source files: the calling thread's error message and the
// guard that makes a device current for the length of a call.
#pragma once

#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdio>

#include "../../include/povs.h"

namespace povs_host {

inline thread_local char g_err[512] = "";

inline int fail(int code, const char* fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
    return code;
}

inline int cuda_fail(cudaError_t e, const char* what)
{
    return fail(POVS_ERR_CUDA, "%s: %s (%s)", what, cudaGetErrorName(e), cudaGetErrorString(e));
}

#define POVS_CUDA_TRY(expr)                                \
    do {                                                   \
        cudaError_t e_ = (expr);                           \
        if (e_ != cudaSuccess) return cuda_fail(e_, #expr); \
    } while (0)

constexpr int MAX_DEVICES = 64;

struct DeviceGuard {
    int prev = -1;
    bool changed = false;
    int enter(int dev)
    {
        cudaError_t e = cudaGetDevice(&prev);
        if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
        if (prev != dev) {
            e = cudaSetDevice(dev);
            if (e != cudaSuccess) return cuda_fail(e, "cudaSetDevice");
            changed = true;
        }
        return POVS_OK;
    }
    ~DeviceGuard()
    {
        if (changed) cudaSetDevice(prev);
    }
};

} // namespace povs_host
