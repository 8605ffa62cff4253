// ela_expert.cuh -- shared by the expert-layer kernels: element types, 16-byte
// accesses and the reading of offsets.
#pragma once

#include <cuda_runtime.h>
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <stdint.h>

#include "ela_expert.h"

namespace ela_expert {

// Element type of a row: conversion to and from fp32, W elements in 16 bytes.
template <typename T> struct El;
template <> struct El<float> {
    static constexpr int W = 4;
    static __device__ __forceinline__ float to(float v) { return v; }
    static __device__ __forceinline__ float from(float v) { return v; }
};
template <> struct El<__half> {
    static constexpr int W = 8;
    static constexpr bool BF16 = false;
    static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};
template <> struct El<__nv_bfloat16> {
    static constexpr int W = 8;
    static constexpr bool BF16 = true;
    static __device__ __forceinline__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};

// W consecutive elements: 16 bytes when VEC, else one element at a time (rows
// that are not 16-byte aligned).
template <typename T> struct alignas(16) Pack { T v[El<T>::W]; };

__host__ inline int dtype_bytes(int dtype) {
    return dtype == ELA_DTYPE_F32 ? 4 : (dtype == ELA_DTYPE_F16 || dtype == ELA_DTYPE_BF16) ? 2 : 0;
}
__host__ inline bool aligned16(const void* p, int64_t ld_bytes = 0) {
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld_bytes % 16 == 0;
}
__host__ inline int launch_status() { return cudaGetLastError() == cudaSuccess ? ELA_OK : ELA_ERR_CUDA; }

// Rows of expert e, kept inside [0, R] whatever the offsets hold.
__device__ __forceinline__ int clampi(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }
__device__ __forceinline__ void expert_rows(const int32_t* offsets, int e, int R, int& r0, int& r1) {
    r0 = offsets ? clampi(__ldg(offsets + e), 0, R) : 0;
    r1 = offsets ? clampi(__ldg(offsets + e + 1), r0, R) : R;
}

// Activation and its derivative, fp32.
template <int ACT> __device__ __forceinline__ float act_value(float z) {
    if (ACT == ELA_ACT_RELU) return z < 0.f ? 0.f : z;  // NaN stays NaN
    if (ACT == ELA_ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    if (ACT == ELA_ACT_SILU) return z / (1.f + __expf(-z));
    return z;
}
template <int ACT> __device__ __forceinline__ float act_slope(float z) {
    if (ACT == ELA_ACT_RELU) return z > 0.f ? 1.f : 0.f;
    if (ACT == ELA_ACT_GELU)  // Phi(z) + z * phi(z)
        return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * __expf(-0.5f * z * z) * 0.39894228040143268f;
    if (ACT == ELA_ACT_SILU) {
        const float q = 1.f / (1.f + __expf(-z));
        return q * (1.f + z * (1.f - q));
    }
    return 1.f;
}

}  // namespace ela_expert
