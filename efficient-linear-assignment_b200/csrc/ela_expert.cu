// ela_expert.cu -- tokens sorted by expert and back (include/ela_expert.h): the
// plan (a stable counting sort), the dispatch of token rows into expert order
// and the weighted combine with its gradient.

#include "ela_expert.cuh"

namespace ela_expert {

// ------------------------------------------------------------------- plan
// A stable counting sort in one CTA.  Every warp owns a contiguous range of
// slots; count[w][b] = slots of bucket b in warp w's range; the exclusive sum
// over (bucket, warp) is each warp's first row in each bucket; the warp then
// walks its range 32 slots at a time, and the lanes of one bucket
// (__match_any_sync) take consecutive rows in lane order.
#define ELA_PLAN_THREADS 1024

template <typename Id>
__global__ void __launch_bounds__(ELA_PLAN_THREADS) plan_kernel(const Id* expert, int slots, int E, int nwarps,
                                                                int32_t* offsets, int32_t* position,
                                                                int32_t* source) {
    extern __shared__ int count[];  // [nwarps][E + 1]
    __shared__ int warp_sum[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = E + 1;
    for (int i = tid; i < nwarps * B; i += blockDim.x) count[i] = 0;
    __syncthreads();
    const int per = (int)((((int64_t)slots + nwarps - 1) / nwarps + 31) / 32 * 32);
    const int64_t first = (int64_t)warp * per;
    const int s0 = warp < nwarps && first < slots ? (int)first : slots;
    const int s1 = (int64_t)s0 + per < slots ? s0 + per : slots;
    int* mine = count + (warp < nwarps ? warp : 0) * B;
    for (int s = s0 + lane; s < s1; s += 32) {
        const Id e = expert[s];
        atomicAdd(&mine[e >= 0 && e < (Id)E ? (int)e : E], 1);
    }
    __syncthreads();
    // exclusive sum in (bucket, warp) order: each thread sums a run of buckets
    const int run = (B + blockDim.x - 1) / blockDim.x;
    const int b0 = min(tid * run, B), b1 = min(b0 + run, B);
    int total = 0;
    for (int b = b0; b < b1; ++b)
        for (int w = 0; w < nwarps; ++w) total += count[w * B + b];
    int incl = total;
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(~0u, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    int base = incl - total;
    for (int w = 0; w < warp; ++w) base += warp_sum[w];
    for (int b = b0; b < b1; ++b) {
        offsets[b] = base;
        for (int w = 0; w < nwarps; ++w) {
            const int c = count[w * B + b];
            count[w * B + b] = base;
            base += c;
        }
    }
    __syncthreads();
    for (int s = s0; s < s1; s += 32) {
        const bool in = s + lane < s1;
        int b = -1;
        if (in) {
            const Id e = expert[s + lane];
            b = e >= 0 && e < (Id)E ? (int)e : E;
        }
        const unsigned same = __match_any_sync(~0u, b);
        const int ahead = __popc(same & ((1u << lane) - 1));
        int row = 0;
        if (in) row = mine[b] + ahead;
        __syncwarp();
        if (in && ahead == 0) mine[b] += __popc(same);
        __syncwarp();
        if (in) {
            position[s + lane] = row;
            source[row] = s + lane;
        }
    }
}

// --------------------------------------------------------- dispatch, combine
// One CTA per token: every row is read once and written once.

template <typename T, bool VEC> __device__ __forceinline__ void load_piece(const T* row, int64_t i, int64_t H, float* f) {
    constexpr int W = El<T>::W;
    if (VEC) {
        const Pack<T> p = *reinterpret_cast<const Pack<T>*>(row + i);
#pragma unroll
        for (int c = 0; c < W; ++c) f[c] = El<T>::to(p.v[c]);
    } else {
        f[0] = El<T>::to(row[i]);
    }
}
template <typename T, bool VEC> __device__ __forceinline__ void store_piece(T* row, int64_t i, const float* f) {
    constexpr int W = El<T>::W;
    if (VEC) {
        Pack<T> p;
#pragma unroll
        for (int c = 0; c < W; ++c) p.v[c] = El<T>::from(f[c]);
        *reinterpret_cast<Pack<T>*>(row + i) = p;
    } else {
        row[i] = El<T>::from(f[0]);
    }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dispatch_kernel(const T* x, int k, int64_t H, int64_t ldx,
                                                       const int32_t* position, const int32_t* offsets, int E,
                                                       int rows, T* out) {
    constexpr int W = VEC ? El<T>::W : 1;
    const int64_t t = blockIdx.x;
    const int valid = offsets[E];
    for (int64_t i = (int64_t)threadIdx.x * W; i < H; i += (int64_t)blockDim.x * W) {
        float f[El<T>::W], zero[El<T>::W] = {};
        load_piece<T, VEC>(x + t * ldx, i, H, f);
        for (int j = 0; j < k; ++j) {
            const int p = position[t * k + j];
            if (p < 0 || p >= rows) continue;
            store_piece<T, VEC>(out + (int64_t)p * H, i, p < valid ? f : zero);
        }
    }
}

template <typename T, typename Wt, bool VEC>
__global__ void __launch_bounds__(256) combine_kernel(const T* y, int k, int64_t H, int64_t ldy,
                                                      const int32_t* position, const int32_t* offsets, int E,
                                                      int rows, const Wt* weights, T* out) {
    constexpr int W = VEC ? El<T>::W : 1;
    const int64_t t = blockIdx.x;
    const int valid = min(offsets[E], rows);
    for (int64_t i = (int64_t)threadIdx.x * W; i < H; i += (int64_t)blockDim.x * W) {
        float acc[El<T>::W] = {};
        for (int j = 0; j < k; ++j) {
            const int p = position[t * k + j];
            if (p < 0 || p >= valid) continue;
            const float w = weights ? El<Wt>::to(weights[t * k + j]) : 1.f;
            float f[El<T>::W];
            load_piece<T, VEC>(y + (int64_t)p * ldy, i, H, f);
#pragma unroll
            for (int c = 0; c < W; ++c) acc[c] = fmaf(w, f[c], acc[c]);
        }
        store_piece<T, VEC>(out + t * H, i, acc);
    }
}

template <typename T, typename Wt, bool VEC>
__global__ void __launch_bounds__(256) combine_grad_kernel(const T* dout, const T* y, int k, int64_t H, int64_t lddo,
                                                           int64_t ldy, const int32_t* position,
                                                           const int32_t* offsets, int E, int rows,
                                                           const Wt* weights, T* dy, Wt* dweights) {
    constexpr int W = VEC ? El<T>::W : 1;
    __shared__ float part[8];
    const int64_t t = blockIdx.x;
    const int valid = min(offsets[E], rows);
    for (int j = 0; j < k; ++j) {
        const int p = position[t * k + j];
        const bool in = p >= 0 && p < rows, has = in && p < valid;
        const float w = has ? (weights ? El<Wt>::to(weights[t * k + j]) : 1.f) : 0.f;
        float dot = 0.f;
        for (int64_t i = (int64_t)threadIdx.x * W; i < H; i += (int64_t)blockDim.x * W) {
            float d[El<T>::W], f[El<T>::W];
            load_piece<T, VEC>(dout + t * lddo, i, H, d);
            if (dweights && has) {
                load_piece<T, VEC>(y + (int64_t)p * ldy, i, H, f);
#pragma unroll
                for (int c = 0; c < W; ++c) dot = fmaf(d[c], f[c], dot);
            }
            if (dy && in) {
#pragma unroll
                for (int c = 0; c < W; ++c) d[c] = has ? w * d[c] : 0.f;
                store_piece<T, VEC>(dy + (int64_t)p * H, i, d);
            }
        }
        if (dweights) {
            for (int o = 16; o; o >>= 1) dot += __shfl_xor_sync(~0u, dot, o);
            if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = dot;
            __syncthreads();
            if (threadIdx.x == 0) {
                float sum = 0.f;
                for (int w8 = 0; w8 < (int)(blockDim.x >> 5); ++w8) sum += part[w8];
                dweights[t * k + j] = El<Wt>::from(has ? sum : 0.f);
            }
            __syncthreads();
        }
    }
}

inline bool sizes_ok(int dtype, int64_t T, int64_t k, int64_t H, int64_t E) {
    return dtype_bytes(dtype) != 0 && T >= 0 && k >= 0 && H >= 0 && E >= 1 && E <= ELA_EXPERT_MAX &&
           (k == 0 || T <= INT32_MAX / k) && T <= INT32_MAX;
}

#define ELA_BY_DTYPE(dtype, ...)                              \
    switch (dtype) {                                           \
    case ELA_DTYPE_F32: { typedef float T_; __VA_ARGS__; break; }     \
    case ELA_DTYPE_F16: { typedef __half T_; __VA_ARGS__; break; }    \
    default: { typedef __nv_bfloat16 T_; __VA_ARGS__; break; }        \
    }

}  // namespace ela_expert

using namespace ela_expert;

extern "C" {

size_t ela_expert_plan_workspace_bytes(int64_t, int64_t) { return 0; }

int ela_expert_plan(const void* expert, int id_bytes, int64_t slots, int64_t num_experts, int32_t* offsets,
                    int32_t* position, int32_t* source, void*, size_t, void* stream) {
    if ((id_bytes != 4 && id_bytes != 8) || slots < 0 || slots > INT32_MAX || num_experts < 1 ||
        num_experts > ELA_EXPERT_MAX || !offsets || (slots > 0 && (!expert || !position || !source)))
        return ELA_ERR_ARGUMENT;
    const int E = (int)num_experts;
    const int fit = 200 * 1024 / (4 * (E + 1));
    const int nwarps = fit < 32 ? fit : 32;
    const size_t smem = (size_t)nwarps * (E + 1) * 4;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (id_bytes == 4) {
        if (cudaFuncSetAttribute(plan_kernel<int32_t>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
            return ELA_ERR_CUDA;
        plan_kernel<int32_t><<<1, ELA_PLAN_THREADS, smem, st>>>((const int32_t*)expert, (int)slots, E, nwarps, offsets, position, source);
    } else {
        if (cudaFuncSetAttribute(plan_kernel<int64_t>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
            return ELA_ERR_CUDA;
        plan_kernel<int64_t><<<1, ELA_PLAN_THREADS, smem, st>>>((const int64_t*)expert, (int)slots, E, nwarps, offsets, position, source);
    }
    return launch_status();
}

int ela_expert_dispatch(const void* x, int dtype, int64_t T, int64_t k, int64_t H, int64_t ldx,
                        const int32_t* position, const int32_t* offsets, int64_t num_experts, void* rows,
                        void* stream) {
    if (!sizes_ok(dtype, T, k, H, num_experts) || ldx < 0) return ELA_ERR_ARGUMENT;
    if (T == 0 || k == 0 || H == 0) return ELA_OK;
    if (!x || !position || !offsets || !rows) return ELA_ERR_ARGUMENT;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const int es = dtype_bytes(dtype);
    const bool vec = aligned16(x, ldx * es) && aligned16(rows, H * es);
    ELA_BY_DTYPE(dtype, {
        auto kern = vec ? dispatch_kernel<T_, true> : dispatch_kernel<T_, false>;
        kern<<<(unsigned)T, 256, 0, st>>>((const T_*)x, (int)k, H, ldx, position, offsets, (int)num_experts, (int)(T * k), (T_*)rows);
    })
    return launch_status();
}

int ela_expert_combine(const void* y, int dtype, int64_t T, int64_t k, int64_t H, int64_t ldy,
                       const int32_t* position, const int32_t* offsets, int64_t num_experts, const void* weights,
                       int weights_dtype, void* out, void* stream) {
    if (!sizes_ok(dtype, T, k, H, num_experts) || ldy < 0) return ELA_ERR_ARGUMENT;
    if (weights && weights_dtype != ELA_DTYPE_F32 && weights_dtype != dtype) return ELA_ERR_ARGUMENT;
    if (T == 0 || H == 0) return ELA_OK;
    if (!out || !offsets || (k > 0 && (!y || !position))) return ELA_ERR_ARGUMENT;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const int es = dtype_bytes(dtype);
    const bool vec = aligned16(y, ldy * es) && aligned16(out, H * es);
    const bool w32 = !weights || weights_dtype == ELA_DTYPE_F32;
    ELA_BY_DTYPE(dtype, {
        if (w32) {
            auto kern = vec ? combine_kernel<T_, float, true> : combine_kernel<T_, float, false>;
            kern<<<(unsigned)T, 256, 0, st>>>((const T_*)y, (int)k, H, ldy, position, offsets, (int)num_experts, (int)(T * k), (const float*)weights, (T_*)out);
        } else {
            auto kern = vec ? combine_kernel<T_, T_, true> : combine_kernel<T_, T_, false>;
            kern<<<(unsigned)T, 256, 0, st>>>((const T_*)y, (int)k, H, ldy, position, offsets, (int)num_experts, (int)(T * k), (const T_*)weights, (T_*)out);
        }
    })
    return launch_status();
}

int ela_expert_combine_grad(const void* dout, const void* y, int dtype, int64_t T, int64_t k, int64_t H,
                            int64_t lddo, int64_t ldy, const int32_t* position, const int32_t* offsets,
                            int64_t num_experts, const void* weights, int weights_dtype, void* dy, void* dweights,
                            void* stream) {
    if (!sizes_ok(dtype, T, k, H, num_experts) || lddo < 0 || ldy < 0) return ELA_ERR_ARGUMENT;
    if ((weights || dweights) && weights_dtype != ELA_DTYPE_F32 && weights_dtype != dtype) return ELA_ERR_ARGUMENT;
    if (T == 0 || k == 0 || (!dy && !dweights)) return ELA_OK;
    if (!offsets || !position || (H > 0 && (!dout || (dweights && !y)))) return ELA_ERR_ARGUMENT;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const int es = dtype_bytes(dtype);
    const bool vec = aligned16(dout, lddo * es) && (!dy || aligned16(dy, H * es)) && (!dweights || aligned16(y, ldy * es)) &&
                     H * es % 16 == 0;
    const bool w32 = (!weights && !dweights) || weights_dtype == ELA_DTYPE_F32;
    ELA_BY_DTYPE(dtype, {
        if (w32) {
            auto kern = vec ? combine_grad_kernel<T_, float, true> : combine_grad_kernel<T_, float, false>;
            kern<<<(unsigned)T, 256, 0, st>>>((const T_*)dout, (const T_*)y, (int)k, H, lddo, ldy, position, offsets, (int)num_experts, (int)(T * k), (const float*)weights, (T_*)dy, (float*)dweights);
        } else {
            auto kern = vec ? combine_grad_kernel<T_, T_, true> : combine_grad_kernel<T_, T_, false>;
            kern<<<(unsigned)T, 256, 0, st>>>((const T_*)dout, (const T_*)y, (int)k, H, lddo, ldy, position, offsets, (int)num_experts, (int)(T * k), (const T_*)weights, (T_*)dy, (T_*)dweights);
        }
    })
    return launch_status();
}

}  // extern "C"
