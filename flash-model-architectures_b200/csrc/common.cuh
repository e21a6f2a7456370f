// Shared device/host helpers for libxma_b200 (sm_100a only).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "xma_b200.h"

namespace xma {

constexpr int kDtypeBF16 = 0;
constexpr int kDtypeF16 = 1;
constexpr int kDtypeF32 = 2;
constexpr int kDtypeU8 = 3;  // tensor maps over bytes; no entry point takes it

constexpr int kMaxExperts = 1024;

inline int dtype_size(int dtype) { return dtype == kDtypeF32 ? 4 : 2; }

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Number of SMs of the current device, cached per device.
int sm_count();

// Launch-error check used after every kernel launch.
inline int launch_status() { return cudaGetLastError() == cudaSuccess ? XMA_OK : XMA_ERR_LAUNCH; }

// Lets a kernel use `bytes` of dynamic shared memory; asked of the runtime once per kernel and device.
template <auto kKernel>
bool allow_smem(uint32_t bytes) {
    constexpr int kMaxDevices = 64;
    static std::atomic<bool> set[kMaxDevices];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return false;
    if (set[dev].load(std::memory_order_relaxed)) return true;
    if (cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)) != cudaSuccess) {
        cudaGetLastError();
        return false;
    }
    set[dev].store(true, std::memory_order_relaxed);
    return true;
}

template <typename T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elem<__half> {
    static __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<float> {
    static __device__ __forceinline__ float to_float(float v) { return v; }
    static __device__ __forceinline__ float from_float(float v) { return v; }
};

// Two elements in one 32-bit word, the first in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
    return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
    return __half22float2(*reinterpret_cast<__half2*>(&v));
}

// 16 bytes of elements of type T.
template <typename T>
struct alignas(16) Vec16 {
    static constexpr int kCount = 16 / sizeof(T);
    T v[kCount];
};

template <typename T>
__device__ __forceinline__ Vec16<T> load16(const T* p) {
    Vec16<T> r;
    *reinterpret_cast<uint4*>(&r) = __ldg(reinterpret_cast<const uint4*>(p));
    return r;
}

template <typename T>
__device__ __forceinline__ void store16(T* p, const Vec16<T>& r) {
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&r);
}

}  // namespace xma
