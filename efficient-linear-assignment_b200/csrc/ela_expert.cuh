// ela_expert.cuh -- shared by the expert-layer kernels: element types, 16-byte
// accesses and the reading of offsets.
#pragma once

#include <cuda_runtime.h>
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <stdint.h>

#include <atomic>

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

// W consecutive elements, 16 bytes.
template <typename T> struct alignas(16) Pack { T v[El<T>::W]; };

__host__ inline int dtype_bytes(int dtype) {
    return dtype == ELA_DTYPE_F32 ? 4 : (dtype == ELA_DTYPE_F16 || dtype == ELA_DTYPE_BF16) ? 2 : 0;
}
__host__ inline bool aligned16(const void* p, int64_t ld_bytes = 0) {
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld_bytes % 16 == 0;
}

// Pointers that the kernels may read and write elements of this size through (NULL is one).
template <typename... P> __host__ inline bool on_elements(int size, P... p) {
    return ((reinterpret_cast<uintptr_t>(p) | ...) & (uintptr_t)(size - 1)) == 0;
}

inline int sm_count() {
    static std::atomic<int> counts[64];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    if ((n = counts[dev].load(std::memory_order_relaxed)) != 0) return n;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    counts[dev].store(n, std::memory_order_relaxed);
    return n;
}

// Lets a kernel use this much dynamic shared memory; asked of the driver once per kernel and device.
template <auto KERNEL> __host__ inline bool allow_smem(int bytes) {
    static std::atomic<bool> done[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    if (done[dev].load(std::memory_order_relaxed)) return true;
    if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
    done[dev].store(true, std::memory_order_relaxed);
    return true;
}

// Lets a kernel run in clusters of 16 (8 is what every device of the architecture has).
template <auto KERNEL> __host__ inline bool allow_wide_cluster() {
    static std::atomic<bool> done[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    if (done[dev].load(std::memory_order_relaxed)) return true;
    if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return false;
    done[dev].store(true, std::memory_order_relaxed);
    return true;
}

// Every kernel here is launched so that it may start while the one before it in the stream
// ends (programmatic stream serialization): its prologue, and its CTAs' places on SMs that
// are done, overlap that kernel's tail.  In return every kernel calls previous_done() before
// it touches memory, which waits until the kernels before it are complete and visible, and
// reads with ordinary loads: the non-coherent path is for data that does not change while the
// kernel lives, which begins before the wait, and its loads may be moved above it.
template <typename... P, typename... A>
__host__ inline int launch(void (*kern)(P...), unsigned grid, unsigned block, size_t smem, cudaStream_t st, A... args) {
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...) == cudaSuccess) return ELA_OK;
    cudaGetLastError();
    return ELA_ERR_CUDA;
}
__device__ __forceinline__ void next_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void previous_done() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Rows of expert e, kept inside [0, R] whatever the offsets hold.
__device__ __forceinline__ int clampi(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }
__device__ __forceinline__ void expert_rows(const int32_t* offsets, int e, int R, int& r0, int& r1) {
    r0 = offsets ? clampi(offsets[e], 0, R) : 0;
    r1 = offsets ? clampi(offsets[e + 1], r0, R) : R;
}

// Complementary error function of x / sqrt(2) for x >= 0: Abramowitz and Stegun
// 7.1.26, a polynomial in t = 1 / (1 + 0.3275911 x / sqrt(2)) times exp(-x^2 / 2)
// (absolute error of erf below 1.5e-7); gauss receives the exponential.  Two special
// function calls and no branch, where erff takes a divergent one and 1 + erf cancels
// in the negative tail.
__device__ __forceinline__ float erfc_sqrt2(float x, float& gauss) {
    const float t = __fdividef(1.f, fmaf(0.3275911f * 0.70710678f, x, 1.f));
    gauss = __expf(-0.5f * x * x);
    float q = fmaf(1.061405429f, t, -1.453152027f);
    q = fmaf(q, t, 1.421413741f);
    q = fmaf(q, t, -0.284496736f);
    q = fmaf(q, t, 0.254829592f);
    return q * t * gauss;
}

// Activation and its derivative, fp32.
template <int ACT> __device__ __forceinline__ float act_value(float z) {
    if (ACT == ELA_ACT_RELU) return z < 0.f ? 0.f : z;  // NaN stays NaN
    if (ACT == ELA_ACT_GELU) {
        float g;
        const float tail = 0.5f * erfc_sqrt2(fabsf(z), g);  // 1 - Phi(|z|)
        return z * (z < 0.f ? tail : 1.f - tail);
    }
    if (ACT == ELA_ACT_SILU) return __fdividef(z, 1.f + __expf(-z));
    return z;
}
template <int ACT> __device__ __forceinline__ float act_slope(float z) {
    if (ACT == ELA_ACT_RELU) return z > 0.f ? 1.f : 0.f;
    if (ACT == ELA_ACT_GELU) {  // Phi(z) + z * phi(z)
        float g;
        const float tail = 0.5f * erfc_sqrt2(fabsf(z), g);
        return fmaf(z * 0.39894228040143268f, g, z < 0.f ? tail : 1.f - tail);
    }
    if (ACT == ELA_ACT_SILU) {
        const float q = __fdividef(1.f, 1.f + __expf(-z));
        return q * fmaf(z, 1.f - q, 1.f);
    }
    return 1.f;
}

// ReLU's slope jumps at 0, and a sum on the tensor cores, which drop low bits at every step,
// can come out on the other side of it: about one in eight million at K = 1024, each of which
// moves a row of the weight gradient.  Where z is kept for the gradient, those within the
// sums' error of 0 are summed again to twice the digits, which settles the sign; each of them
// is, so nothing depends on the order in which warps run.  The error, against the largest sum of the same row by 32 features, was at most
// 0.94 * (K + 64) * 2^-28 for K of 16 to 16384 (normal values, rows whose halves cancel, columns
// of sizes 2^-6 to 2^6, both types); the band is 1.5 times (K + 64) * 2^-28.  (Sums that are all far smaller than their partial
// sums, which leave no sum beside them to tell, keep the fp32 sum's sign.)
__device__ __forceinline__ float sign_band(float largest, int K) { return largest * ((float)K + 64.f) * 5.587935447692871e-9f; }

// The type that z is kept in for the gradient: fp32 for GELU and SiLU, whose slope moves with
// z's rounding and is NaN at the infinity that a finite z past fp16's range would become; 16
// bits for ReLU, whose slope is z's sign.  Training 16384 rows through 8 experts of 8192 x 2048
// took 1667 us with 16 bits for GELU, too, and takes 1728; its outputs were off by 0.0024 and
// are by 0.0023, the rest of it dz's own rounding.
template <typename T, int ACT> struct Kept { typedef T Type; };
template <typename T> struct Kept<T, ELA_ACT_GELU> { typedef float Type; };
template <typename T> struct Kept<T, ELA_ACT_SILU> { typedef float Type; };

// z as it is kept for ReLU's gradient, which needs its sign alone: what rounds to 0 in fp16
// (below 2^-25) is kept as the smallest number there is, so a positive z stays positive.
template <typename T> __device__ __forceinline__ float sign_kept(float z) {
    if constexpr (!El<T>::BF16) return z > 0.f ? fmaxf(z, 5.9604644775390625e-8f) : z;
    return z;  // (bf16 has fp32's range)
}

// A sum in two floats: the rounding error of each addition, which is itself a float (Knuth's
// two-sum), is added up beside it.  Products of 16-bit values are exact in fp32.
struct TwoFloats {
    float s, c;
    __device__ __forceinline__ void add_product(float a, float b) {
        const float p = __fmul_rn(a, b), t = __fadd_rn(s, p), q = __fsub_rn(t, s);
        c = __fadd_rn(c, __fadd_rn(__fsub_rn(s, __fsub_rn(t, q)), __fsub_rn(p, q)));
        s = t;
    }
    __device__ __forceinline__ double value() const { return (double)s + (double)c; }
};

// <x, w> to some 2^-45 of its terms, by a whole warp, in a fixed order.  In two floats: on
// doubles throughout, whose conversions and products are far slower, the forward pass of 16384
// rows by 8192 x 8192 took 1900 us instead of 1610.
template <typename T> __device__ __noinline__ double exact_sum(const T* x, const T* w, int K) {
    constexpr int STEP = 4;  // 16-byte loads of each a lane has in flight
    const int lane = threadIdx.x & 31;
    TwoFloats part[2] = {};
    int done = 0;
    if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15) == 0) {
        done = K & ~7;
        for (int k = lane * 8; k < done; k += 256 * STEP) {
            Pack<T> a[STEP], b[STEP];
#pragma unroll
            for (int s = 0; s < STEP; ++s)
                if (s == 0 || k + 256 * s < done) {
                    a[s] = *reinterpret_cast<const Pack<T>*>(x + k + 256 * s);
                    b[s] = *reinterpret_cast<const Pack<T>*>(w + k + 256 * s);
                }
#pragma unroll
            for (int s = 0; s < STEP; ++s)
                if (s == 0 || k + 256 * s < done)
#pragma unroll
                    for (int i = 0; i < 8; ++i) part[i & 1].add_product(El<T>::to(a[s].v[i]), El<T>::to(b[s].v[i]));
        }
    }
    for (int k = done + lane; k < K; k += 32) part[0].add_product(El<T>::to(x[k]), El<T>::to(w[k]));
    double sum = part[0].value() + part[1].value();
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    return sum;
}

}  // namespace ela_expert
