// ela_expert_4bit.cuh -- the forward product with 4-bit weights for a few rows per expert
// (included by ela_expert_4bit.cu).
#pragma once

#include "ela_expert.cuh"
#include "ela_expert_stream.cuh"

namespace ela_expert {

struct Stream4Params {
    const void* x;
    const uint32_t* packed;
    const void* scales;
    const void* bias;
    const void* residual;
    const int32_t* offsets;
    int R, E, K, N;
    int words, parts, shift;  // of a packed row; groups of a row; log2(group)
    int f_tiles, act;
    int wide_scales;          // a lane's scales may be read at once
    int64_t ldx, ldr;
    void* y;
};

__device__ __forceinline__ float act_any(int act, float z) {
    return act == ELA_ACT_RELU ? act_value<ELA_ACT_RELU>(z) : act == ELA_ACT_GELU ? act_value<ELA_ACT_GELU>(z)
         : act == ELA_ACT_SILU ? act_value<ELA_ACT_SILU>(z) : z;
}

// Eight consecutive inputs of a row from k on as four pairs; zeros past the row's end.
template <int VB> __device__ __forceinline__ uint4 load8(const uint16_t* row, int k, int K, bool in) {
    uint4 v = {};
    if (VB == 16) {
        if (in && k < K) v = *reinterpret_cast<const uint4*>(row + k);
    } else {
        uint32_t w[4] = {};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (in && k + i < K) w[i / 2] |= (uint32_t)row[k + i] << (16 * (i & 1));
        v = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return v;
}

// As stream_kernel: items of 16 * MT features over the whole contraction, which the CTA's 8
// warps share; a batch of loads is issued when the one before it has been taken.  A lane
// (g = lane / 4, t = lane % 4) loads 32 consecutive inputs (16 bytes) of each of 2 * MT rows,
// SUB times; a row's place among the MMA's 16 is free, so they are neighbouring features
// (whose scales are neighbours too).  A group has at least 32 inputs: one scale for each load.
// The token's inputs come from L1 when they are needed.
template <typename T, int RG, int MT, int SUB, int VB>
__global__ void __launch_bounds__(STREAM_WARPS * 32, 2) stream4_kernel(const Stream4Params p) {
    next_may_start();
    previous_done();
    constexpr int F = 16 * MT, H = 2 * MT, KB = 128 * SUB;
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
    const int rounds = (p.words * 8 + STREAM_WARPS * KB - 1) / (STREAM_WARPS * KB);

    unsigned item = blockIdx.x - gridDim.x;
    int e = 0, f0 = 0, rb = 0, r1 = 0, it = 0;
    const uint32_t* wrow = nullptr;  // of the lane's first feature
    const T* srow = nullptr;
    const uint16_t* xrow[RG] = {};
    bool xin[RG] = {};
    int fin = 0;  // the lane's features that exist
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
        const int f = f0 + H * g;
        fin = clampi(p.N - f, 0, H);
        wrow = p.packed + ((int64_t)e * p.N + (fin ? f : 0)) * p.words;
        srow = reinterpret_cast<const T*>(p.scales) + (int64_t)e * p.parts * p.N + (fin ? f : 0);
        it = 0;
        return true;
    };
    uint4 a[SUB][H];
    uint32_t sc[SUB][MT];  // two features' scales each
    int k_now = 0;
    auto load = [&]() {
        k_now = (it * STREAM_WARPS + warp) * KB + 32 * t;
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
            const int k = k_now + 128 * s;
            const bool in = k < p.words * 8;
#pragma unroll
            for (int h = 0; h < H; ++h) {
                a[s][h] = make_uint4(Q_ZERO, Q_ZERO, Q_ZERO, Q_ZERO);
                if (in && h < fin)
                    asm volatile("ld.global.L1::no_allocate.L2::256B.v4.b32 {%0,%1,%2,%3}, [%4];"
                        : "=r"(a[s][h].x), "=r"(a[s][h].y), "=r"(a[s][h].z), "=r"(a[s][h].w) : "l"(wrow + (int64_t)h * p.words + k / 8) : "memory");
            }
            const int part_at = min(k >> p.shift, p.parts - 1);
            const T* from = srow + (int64_t)part_at * p.N;
#pragma unroll
            for (int m = 0; m < MT; ++m) sc[s][m] = 0;
            if (in && p.wide_scales && fin) {
                if constexpr (MT == 1) sc[s][0] = *reinterpret_cast<const uint32_t*>(from);
                if constexpr (MT == 2) { const uint2 v = *reinterpret_cast<const uint2*>(from); sc[s][0] = v.x; sc[s][1] = v.y; }
                if constexpr (MT == 4) {
                    const uint4 v = *reinterpret_cast<const uint4*>(from);
                    sc[s][0] = v.x; sc[s][1] = v.y; sc[s][2] = v.z; sc[s][3] = v.w;
                }
            } else if (in) {
#pragma unroll
                for (int h = 0; h < H; ++h)
                    if (h < fin) sc[s][h / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(from)[h] << (16 * (h & 1));
            }
        }
    };
    bool more = next_item();
    if (more) { rows(); load(); }
    float acc[MT][RG][4] = {};
    while (more) {
#pragma unroll
        for (int s = 0; s < SUB; ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint4 b[RG];
#pragma unroll
                for (int q = 0; q < RG; ++q) b[q] = load8<VB>(xrow[q], k_now + 128 * s + 8 * j, p.K, xin[q]);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    uint32_t lo[4], hi[4];
                    const uint4 &u = a[s][2 * m], &v = a[s][2 * m + 1];
                    unpack<T>(j == 0 ? u.x : j == 1 ? u.y : j == 2 ? u.z : u.w, __byte_perm(sc[s][m], 0, 0x1010), lo);
                    unpack<T>(j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w, __byte_perm(sc[s][m], 0, 0x3232), hi);
#pragma unroll
                    for (int q = 0; q < RG; ++q) {
                        mma16816<T>(acc[m][q], lo[0], hi[0], lo[1], hi[1], b[q].x, b[q].y);
                        mma16816<T>(acc[m][q], lo[2], hi[2], lo[3], hi[3], b[q].z, b[q].w);
                    }
                }
            }
        // the next batch's loads, then what this one completes
        const int done_e = e, done_f = f0, done_rb = rb, done_r1 = r1;
        const bool complete = ++it == rounds;
        if (complete) {
            rb += 8 * RG;
            if (rb < r1) it = 0; else more = next_item();
            if (more) rows();
        }
        if (more) load();
        if (!complete) continue;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int q = 0; q < RG; ++q)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    part[warp][q * 8 + 2 * t + (i & 1)][H * g + 2 * m + (i >> 1)] = acc[m][q][i];
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
                v = act_any(p.act, v);
                if (residual) v += El<T>::to(residual[r * p.ldr + f]);
                y[(int64_t)r * p.N + f] = El<T>::from(v);
            }
        }
        __syncthreads();
    }
}

template <typename T, int RG, int MT, int SUB> int stream4_launch(Stream4Params p, bool vec, cudaStream_t st) {
    p.f_tiles = (p.N + 16 * MT - 1) / (16 * MT);
    p.wide_scales = p.N % (2 * MT) == 0 && (reinterpret_cast<uintptr_t>(p.scales) & (4 * MT - 1)) == 0;
    const int64_t items = (int64_t)p.E * p.f_tiles, most = 2 * (int64_t)sm_count();
    if (items > INT32_MAX) return ELA_ERR_UNSUPPORTED;
    return launch(vec ? stream4_kernel<T, RG, MT, SUB, 16> : stream4_kernel<T, RG, MT, SUB, 2>, (unsigned)(items < most ? items : most),
                  STREAM_WARPS * 32, 0, st, p);
}

// Rows per expert up to which the weights are streamed.
inline bool few_rows_4bit(int64_t R, int64_t E, int64_t N) { return R <= 16 * E || (R <= 64 * E && E * ((N + 255) / 256) <= sm_count() / 4); }

}  // namespace ela_expert
