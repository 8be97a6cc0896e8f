// Host-side helpers shared by the translation units of the library: error
// reporting (kvx_last_error), device selection and the SM count.
#pragma once

#include <cuda_runtime.h>

#include <cmath>

#include "kvx.h"

namespace kvx {

constexpr int kMaxDevices = 64;

int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t e, const char* what);
int sm_count(int dev, int* out);

// Whether x is a power of two in [2^-64, 2^63].
inline bool power_of_two(float x) {
    int e;
    return std::isfinite(x) && x > 0.f && std::frexp(x, &e) == 0.5f && e >= -63 && e <= 64;
}

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
