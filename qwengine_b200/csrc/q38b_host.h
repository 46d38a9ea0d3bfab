// q38b_host.h -- host-side helpers of the entry points that take a context's device as their own.
#pragma once
#include <cuda_runtime.h>

#include "q38b_internal.h"

// Makes the context's device current while an entry point launches, and the caller's device again when it returns, so that
// a call works whatever device the calling thread has current.
struct DeviceGuard {
    int before = -1;
    explicit DeviceGuard(const q38b_ctx* ctx) {
        int now = 0;
        if (cudaGetDevice(&now) == cudaSuccess && now != ctx->device && cudaSetDevice(ctx->device) == cudaSuccess) before = now;
    }
    ~DeviceGuard() { if (before >= 0) cudaSetDevice(before); }
};

// the status of the launch just made
inline int launch_status(q38b_ctx* ctx, cudaError_t e) {
    if (e == cudaSuccess) e = cudaGetLastError();
    else (void)cudaGetLastError();
    if (e == cudaSuccess) return 0;
    ctx->last_cuda = (int)e;
    return -4;   // Q38B_ERR_CUDA
}
