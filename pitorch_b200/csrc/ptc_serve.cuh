// ptc_serve.cuh -- shared by the serving operators (include/ptc_serve.h):
// refusals, the device of a call, and 16-byte vectors of the element types.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/ptc_serve.h"
#include "ptc_common.cuh"

// A refused call: message and -1 (these entry points never abort).
#define SERVE_REFUSE(...)                                    \
    do {                                                     \
        fprintf(stderr, "pitorch_b200: %s: ", __func__);     \
        fprintf(stderr, __VA_ARGS__);                        \
        fputc('\n', stderr);                                 \
        return -1;                                           \
    } while (0)

// The runtime also remembers a call's error for whoever asks for the last one:
// it is taken back, as it is this call's and told by its return value.
#define SERVE_CUDA(call)                                              \
    do {                                                              \
        cudaError_t e_ = (call);                                      \
        if (e_ != cudaSuccess) {                                      \
            cudaGetLastError();                                       \
            SERVE_REFUSE("%s: %s", #call, cudaGetErrorString(e_));    \
        }                                                             \
    } while (0)

namespace ptc {

// Makes the device that holds `mem` current for a call, and puts the caller's
// back. Allowed while a stream is captured (asking a stream for its device is
// not).
class MemoryDevice {
public:
    explicit MemoryDevice(const void *mem) {
        cudaPointerAttributes at;
        err_ = cudaGetDevice(&prev_);
        dev_ = prev_;
        if (err_ == cudaSuccess) err_ = cudaPointerGetAttributes(&at, mem);
        if (err_ == cudaSuccess && at.type == cudaMemoryTypeUnregistered) err_ = cudaErrorInvalidDevicePointer;
        if (err_ == cudaSuccess && at.type != cudaMemoryTypeHost) dev_ = at.device;
        if (err_ == cudaSuccess && dev_ != prev_) err_ = cudaSetDevice(dev_);
    }
    ~MemoryDevice() {
        if (err_ == cudaSuccess && dev_ != prev_) cudaSetDevice(prev_);
    }
    cudaError_t error() const { return err_; }
    int device() const { return dev_; }

private:
    int prev_ = 0, dev_ = 0;
    cudaError_t err_;
};

// Lets `kernel` have `most` bytes of dynamic shared memory on the current
// device. The limit belongs to the function, not to a call: `most` is what
// the largest call of the kernel takes, the same in every call, as a
// smaller one from another host thread would refuse a launch in between.
template <typename Kernel>
cudaError_t allow_smem(Kernel *kernel, int most) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
}

// A launch that answers for itself: the last error, which <<<>>> leaves to ask
// for, may be an older one of the calling thread, and the call would be
// refused although its kernel runs.
template <typename... P, typename... A>
cudaError_t launch_kernel(void (*kernel)(P...), unsigned grid, unsigned threads, size_t smem, cudaStream_t s, const A &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }
inline int dtype_bytes(int dtype) { return dtype == PTC_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == PTC_F32 || dtype == PTC_F16 || dtype == PTC_BF16; }

// What is wrong with a cache descriptor, or NULL.
const char *check_cache(const ptc_paged_cache &c);

template <typename T>
struct Elem;
template <>
struct Elem<float> {
    static constexpr int TYPE = PTC_F32;
    static __device__ __forceinline__ float up(float v) { return v; }
    static __device__ __forceinline__ float down(float v) { return v; }
};
template <>
struct Elem<__half> {
    static constexpr int TYPE = PTC_F16;
    static __device__ __forceinline__ float up(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half down(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<__nv_bfloat16> {
    static constexpr int TYPE = PTC_BF16;
    static __device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 down(float v) { return __float2bfloat16_rn(v); }
};

// 16 bytes of elements.
template <typename T>
struct alignas(16) Vec16 {
    static constexpr int N = 16 / sizeof(T);
    T e[N];
};

__device__ __forceinline__ void serve_err(int *err, int bits) {
    if (err) atomicOr(err, bits);
}

}  // namespace ptc
