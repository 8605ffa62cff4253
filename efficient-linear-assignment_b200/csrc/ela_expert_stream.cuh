// ela_expert_stream.cuh -- the forward product for a few rows per expert (included by
// ela_expert_linear.cu).
//
// With a few rows every weight is used a few times and the time is that of reading the
// weights once, which takes about 130 KB in flight on every SM all the time.  The
// persistent tiles of ela_expert_mma.cuh reach 5.6 TB/s and leave SMs idle in their last
// round (256 tiles on 74 pairs); here an item is 32 (or 16) features of an expert over
// the whole contraction, and two CTAs per SM walk the items with plain 32-byte loads
// that go straight to registers.  A batch of loads is issued as soon as the products of
// the batch before have taken its registers' contents, so the loads of the next item run
// during the reduction and the stores of the last.
//
// The 8 warps of a CTA share the contraction, a batch of k each in turn.  A lane
// (g = lane / 4, t = lane % 4) loads 16 consecutive k (one 32-byte sector) of rows g,
// g+8, ... of the weights and of token row g: as operands of four m16n8k16 products these
// 16 values are the lane's columns (2t, 2t+1, 2t+8, 2t+9) of four k steps.  The sum does not mind in which
// order k is taken as long as both operands agree, so no value changes lanes.  The
// warps' sums meet in shared memory and are added in the order of the warps.
#pragma once

#include "ela_expert.cuh"

namespace ela_expert {

constexpr int STREAM_WARPS = 8;

struct StreamParams {
    const void* x;
    const void* w;
    const void* bias;
    const void* residual;
    const int32_t* offsets;
    int R, E, K, N;
    int f_tiles;  // items per expert
    int64_t ldx, stride_e, ldw, ldr;
    void* y;
    void* z;
};

// 16 consecutive elements from k on as eight words of two; zeros past the row's end.
// VB: bytes every row is aligned to; K is a multiple of that many bytes.
struct Sixteen { uint32_t w[8]; };
template <int VB, bool ONCE> __device__ __forceinline__ Sixteen load16(const uint16_t* row, int k, int K, bool in) {
    Sixteen v = {};
    if constexpr (VB == 32) {
        if (in && k < K) {
            if (ONCE)  // the weights: not kept in L1, fetched into the L2 256 bytes at a time
                asm volatile("ld.global.L1::no_allocate.L2::256B.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                    : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]), "=r"(v.w[7]) : "l"(row + k) : "memory");
            else
                asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                    : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]), "=r"(v.w[7]) : "l"(row + k) : "memory");
        }
    } else if constexpr (VB == 16) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (in && k + 8 * h < K) {
                const uint4 q = *reinterpret_cast<const uint4*>(row + k + 8 * h);
                v.w[4 * h] = q.x; v.w[4 * h + 1] = q.y; v.w[4 * h + 2] = q.z; v.w[4 * h + 3] = q.w;
            }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (VB == 4) {
                if (in && k + 2 * i < K) v.w[i] = *reinterpret_cast<const uint32_t*>(row + k + 2 * i);
            } else {
                if (in && k + 2 * i < K) v.w[i] = row[k + 2 * i];
                if (in && k + 2 * i + 1 < K) v.w[i] |= (uint32_t)row[k + 2 * i + 1] << 16;
            }
        }
    }
    return v;
}

template <typename T> __device__ __forceinline__ void mma16816(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (El<T>::BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// RG: groups of 8 rows whose products are formed from one read of the weights.  MT: 16
// features each in an item.  LOADS: 32-byte loads of the weights a lane has in flight;
// two CTAs an SM leave 128 registers, which 8 loads fill for 8 rows and spill for 16.
// 16 experts of 4096 x 1024, 134 MB: 25 us (5.4 TB/s with the launch) for a row each with
// 8 loads, 28 with 4; 30 against 32 us the other way round for 8 rows each; 33 us by the
// tiles of ela_expert_mma.cuh.  16-byte loads: 27 us.
template <typename T, int ACT, int RG, int MT, int VB>
__global__ void __launch_bounds__(STREAM_WARPS * 32, 2) stream_kernel(const StreamParams p) {
    next_may_start();
    previous_done();
    constexpr int F = 16 * MT, LOADS = RG == 1 ? 8 : 4, SUB = LOADS / (2 * MT), KB = 64 * SUB;  // features, steps of 64 k, k of a batch
    __shared__ float part[STREAM_WARPS][RG * 8][F + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    T* y = reinterpret_cast<T*>(p.y);
    const T* residual = reinterpret_cast<const T*>(p.residual);
    if (p.offsets) {  // rows of no expert: the residual, or 0
        const int lo = clampi(p.offsets[0], 0, p.R), hi = clampi(p.offsets[p.E], 0, p.R);
        for (int r = blockIdx.x; r < p.R; r += gridDim.x)
            if (r < lo || r >= hi)
                for (int f = threadIdx.x; f < p.N; f += STREAM_WARPS * 32)
                    y[(int64_t)r * p.N + f] = residual ? residual[r * p.ldr + f] : El<T>::from(0.f);
    }
    const unsigned items = (unsigned)p.E * p.f_tiles;  // (below 2^31: the step past the last does not wrap)
    const int rounds = (p.K + STREAM_WARPS * KB - 1) / (STREAM_WARPS * KB);

    // the place of the next batch: item (expert e, features f0), rows rb.., round it
    unsigned item = blockIdx.x - gridDim.x;
    int e = 0, f0 = 0, rb = 0, r1 = 0, it = 0;
    const uint16_t *wrow[2 * MT] = {}, *xrow[RG] = {};
    bool win[2 * MT] = {}, xin[RG] = {};
    auto rows = [&]() {
#pragma unroll
        for (int q = 0; q < RG; ++q) {
            xin[q] = rb + 8 * q + g < r1;
            xrow[q] = reinterpret_cast<const uint16_t*>(p.x) + (int64_t)(xin[q] ? rb + 8 * q + g : 0) * p.ldx;
        }
    };
    auto next_item = [&]() {  // false: none left
        do {
            item += gridDim.x;
            if (item >= items) return false;
            e = (int)(item / (unsigned)p.f_tiles);
            expert_rows(p.offsets, e, p.R, rb, r1);
        } while (rb >= r1);
        f0 = (int)(item - (unsigned)e * p.f_tiles) * F;
#pragma unroll
        for (int h = 0; h < 2 * MT; ++h) {
            win[h] = f0 + g + 8 * h < p.N;
            wrow[h] = reinterpret_cast<const uint16_t*>(p.w) + (int64_t)e * p.stride_e + (int64_t)(win[h] ? f0 + g + 8 * h : 0) * p.ldw;
        }
        it = 0;
        rows();
        return true;
    };
    Sixteen a[SUB][2 * MT], b[SUB][RG];
    auto load = [&]() {
        const int k0 = (it * STREAM_WARPS + warp) * KB + 16 * t;
#pragma unroll
        for (int s = 0; s < SUB; ++s)
#pragma unroll
            for (int h = 0; h < 2 * MT; ++h) a[s][h] = load16<VB, true>(wrow[h], k0 + 64 * s, p.K, win[h]);
#pragma unroll
        for (int s = 0; s < SUB; ++s)
#pragma unroll
            for (int q = 0; q < RG; ++q) b[s][q] = load16<VB, false>(xrow[q], k0 + 64 * s, p.K, xin[q]);
    };
    bool more = next_item();
    if (more) load();
    float acc[MT][RG][4] = {};
    while (more) {
#pragma unroll
        for (int s = 0; s < SUB; ++s)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int q = 0; q < RG; ++q)
#pragma unroll
                    for (int j = 0; j < 8; j += 2)
                        mma16816<T>(acc[m][q], a[s][2 * m].w[j], a[s][2 * m + 1].w[j], a[s][2 * m].w[j + 1], a[s][2 * m + 1].w[j + 1],
                                    b[s][q].w[j], b[s][q].w[j + 1]);
        // the next batch's loads, then what this one completes
        const int done_e = e, done_f = f0, done_rb = rb, done_r1 = r1;
        const bool complete = ++it == rounds;
        if (complete) {
            rb += 8 * RG;
            if (rb < r1) { it = 0; rows(); } else more = next_item();
        }
        if (more) load();
        if (!complete) continue;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int q = 0; q < RG; ++q)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    part[warp][q * 8 + 2 * t + (i & 1)][16 * m + g + 8 * (i >> 1)] = acc[m][q][i];
                    acc[m][q][i] = 0.f;
                }
        __syncthreads();
        for (int i = threadIdx.x; i < RG * 8 * F; i += STREAM_WARPS * 32) {
            const int c = i / F, r = done_rb + c, f = done_f + i % F;
            if (r < done_r1 && f < p.N) {
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < STREAM_WARPS; ++w) v += part[w][c][i % F];
                if (p.bias) v += El<T>::to(reinterpret_cast<const T*>(p.bias)[(int64_t)done_e * p.N + f]);
                const int64_t at = (int64_t)r * p.N + f;
                typedef typename Kept<T, ACT>::Type Kt;
                if (p.z) reinterpret_cast<Kt*>(p.z)[at] = El<Kt>::from(ACT == ELA_ACT_RELU ? sign_kept<T>(v) : v);
                v = act_value<ACT>(v);
                if (residual) v += El<T>::to(residual[r * p.ldr + f]);
                y[at] = El<T>::from(v);
            }
        }
        __syncthreads();
    }
}

// ReLU's z next to 0, summed again where z is kept (sign_band): a pass of its own over z, which
// is small here, since the call of exact_sum cost the kernel above the registers of its loads
// (16 rows of 16 experts of 4096 x 1024: 23 -> 45 us inside it, 27 as a pass; 16 rows each
// 29 -> 57, 36).  A warp takes 256 features of a row, whose largest z is the scale.  Where every sum of them is 0, by
// a row of zeros, z is taken as it is, and so it is where a feature's sums are 0 in eight rows,
// by weights of zeros (a quarter of the features so: 38 us, 232 with all of them summed; other
// warps may be writing those rows, but no such z before or after).
constexpr int SETTLE_GROUPS = 8;  // of 32 features
template <typename T>
__global__ void __launch_bounds__(256) settle_kernel(const StreamParams p) {
    next_may_start();
    previous_done();
    const int lane = threadIdx.x & 31, segments = (p.N + 32 * SETTLE_GROUPS - 1) / (32 * SETTLE_GROUPS);
    const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (unit >= (int64_t)p.R * segments) return;
    const int r = (int)(unit / segments), f0 = (int)(unit - (int64_t)r * segments) * 32 * SETTLE_GROUPS;
    int e = 0, r0, r1;
    for (int end = p.E; p.offsets && end - e > 1;) {  // the last expert that starts at or before r
        const int mid = (e + end) >> 1;
        if (clampi(p.offsets[mid], 0, p.R) <= r) e = mid; else end = mid;
    }
    expert_rows(p.offsets, e, p.R, r0, r1);
    if (r < r0 || r >= r1) return;
    T* zrow = reinterpret_cast<T*>(p.z) + (int64_t)r * p.N;
    const T* bias = p.bias ? reinterpret_cast<const T*>(p.bias) + (int64_t)e * p.N : nullptr;
    float z[SETTLE_GROUPS], b[SETTLE_GROUPS], largest = 0.f;
    unsigned zeros = 0;  // a bit a group: the sum is 0 (or the bias hides it), or there is no feature
#pragma unroll
    for (int i = 0; i < SETTLE_GROUPS; ++i) {
        const int f = f0 + 32 * i + lane;
        z[i] = f < p.N ? El<T>::to(zrow[f]) : INFINITY;
        b[i] = f < p.N && bias ? El<T>::to(bias[f]) : 0.f;
        zeros |= (unsigned)(f >= p.N || z[i] == b[i]) << i;
    }
#pragma unroll
    for (int i = 0; i < SETTLE_GROUPS; ++i)
        if ((z[i] = fabsf(z[i])) < INFINITY) largest = fmaxf(largest, z[i] + (fabsf(b[i]) < INFINITY ? fabsf(b[i]) : 0.f));
    // (numbers from 0 on compare as their bits do; 1.01: z is rounded)
    const float band = 1.01f * sign_band(__uint_as_float(__reduce_max_sync(~0u, __float_as_uint(largest))), p.K);
    if (!(band > 0.f) || (p.N - f0 >= 8 && __all_sync(~0u, zeros == (1u << SETTLE_GROUPS) - 1))) return;
    const T* x = reinterpret_cast<const T*>(p.x) + (int64_t)r * p.ldx;
    const T* w = reinterpret_cast<const T*>(p.w) + (int64_t)e * p.stride_e;
    unsigned near = 0;  // a bit a group
#pragma unroll
    for (int i = 0; i < SETTLE_GROUPS; ++i) near |= (unsigned)(z[i] <= band) << i;
    if (r1 - r0 >= 8 && (near & zeros))
#pragma unroll
        for (int i = 0; i < SETTLE_GROUPS; ++i)
            if ((near & zeros) >> i & 1) {
                const T* column = reinterpret_cast<const T*>(p.z) + (int64_t)r0 * p.N + f0 + 32 * i + lane;
                bool always = true;
#pragma unroll
                for (int q = 0; q < 8; ++q) always &= El<T>::to(column[(int64_t)q * p.N]) == b[i];
                if (always) near &= ~(1u << i);
            }
    __syncwarp();
    for (unsigned any = __reduce_or_sync(~0u, near); any; any &= any - 1) {
        const int i = __ffs(any) - 1;
        for (unsigned todo = __ballot_sync(~0u, near >> i & 1); todo; todo &= todo - 1) {
            const int f = f0 + 32 * i + __ffs(todo) - 1;
            const double sum = exact_sum<T>(x, w + (int64_t)f * p.ldw, p.K);
            if (lane == 0) zrow[f] = El<T>::from(sign_kept<T>((float)(sum + (bias ? (double)El<T>::to(bias[f]) : 0.0))));
        }
    }
}
template <typename T> int settle_launch(const StreamParams& p, cudaStream_t st) {
    const int64_t units = (int64_t)p.R * ((p.N + 32 * SETTLE_GROUPS - 1) / (32 * SETTLE_GROUPS)), blocks = (units + 7) / 8;
    if (blocks > INT32_MAX) return ELA_ERR_UNSUPPORTED;
    return launch(settle_kernel<T>, (unsigned)blocks, 256, 0, st, p);
}

// Rows per expert up to which the weights' read is what the product costs: 16 rows for
// each of 16 experts take 31 us here and 33 us by tiles, 32 rows 45 and 34.  Where tiles
// of 256 features leave half of the pairs idle, which then read at 44 GB/s an SM, up to 64.
// The loads, which only the device knows, are taken to be equal, as an assignment makes them:
// experts of 2048 x 1024 with half of all rows on one of them take, here and by tiles, 30 and
// 18 us for 256 rows of 16 (equal loads: 14 and 14), 20 and 15 for 128 of 16 (13 and 15), 108
// and 79 for 512 of 128 (80 and 86), 231 and 102 for 2048 of 128 (98 and 89).
inline bool few_rows(int64_t R, int64_t E, int64_t N) {
    return R <= 16 * E || (R <= 64 * E && E * ((N + 255) / 256) <= sm_count() / 4);
}

template <typename T, int ACT, int RG, int MT>
int stream_launch_vb(StreamParams p, int vb, cudaStream_t st) {
    p.f_tiles = (p.N + 16 * MT - 1) / (16 * MT);
    const int64_t items = (int64_t)p.E * p.f_tiles, most = 2 * (int64_t)sm_count();
    const unsigned grid = (unsigned)(items < most ? items : most);
    auto kern = vb == 32 ? stream_kernel<T, ACT, RG, MT, 32> : vb == 16 ? stream_kernel<T, ACT, RG, MT, 16>
              : vb == 4 ? stream_kernel<T, ACT, RG, MT, 4> : stream_kernel<T, ACT, RG, MT, 2>;
    return launch(kern, grid, STREAM_WARPS * 32, 0, st, p);
}
// Items of 16 features where 32 would leave CTAs without one.
template <typename T, int ACT, int RG>
int stream_launch(const StreamParams& p, int vb, cudaStream_t st) {
    const int64_t experts = p.E < p.R ? p.E : p.R;
    return experts * ((p.N + 31) / 32) < 2 * sm_count() ? stream_launch_vb<T, ACT, RG, 1>(p, vb, st) : stream_launch_vb<T, ACT, RG, 2>(p, vb, st);
}

}  // namespace ela_expert
