// Host-side helpers shared by the translation units of the library: error
// reporting (kvx_last_error), device selection and the SM count.
#pragma once

#include <cuda_runtime.h>

#include "kvx.h"

namespace kvx {

constexpr int kMaxDevices = 64;

int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t e, const char* what);
int sm_count(int dev, int* out);

#define KVX_CUDA(call, what)                         \
    do {                                             \
        cudaError_t e_ = (call);                     \
        if (e_ != cudaSuccess) return cuda_fail(e_, what); \
    } while (0)

struct DeviceGuard {
    int prev = -1;
    bool changed = false;
    cudaError_t err = cudaSuccess;
    explicit DeviceGuard(int dev) {
        err = cudaGetDevice(&prev);
        if (err == cudaSuccess && prev != dev) {
            err = cudaSetDevice(dev);
            changed = (err == cudaSuccess);
        }
    }
    ~DeviceGuard() {
        if (changed) cudaSetDevice(prev);
    }
};

#define KVX_DEVICE_GUARD(dev)                                            \
    DeviceGuard guard_(dev);                                             \
    if (guard_.err != cudaSuccess) return cuda_fail(guard_.err, "select device")

}  // namespace kvx
