// Host-side checks shared by the translation units of librgb200.so.
#pragma once
#include <cuda_runtime.h>

namespace rgb200 {

// cudaSuccess on the architecture this library carries code for, "not supported" elsewhere.
inline cudaError_t check_b200() {
    int dev, major = 0, minor = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev);
    if (e != cudaSuccess) return e;
    return major == 10 && minor == 0 ? cudaSuccess : cudaErrorNotSupported;
}

}  // namespace rgb200
