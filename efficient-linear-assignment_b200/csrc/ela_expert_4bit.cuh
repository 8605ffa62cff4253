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
    int k_warps, f_tiles;     // warps that share a contraction; items per expert
    int act, wide_scales;     // a lane's scales may be read at once
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

// As stream_kernel, plain loads straight to registers: an item is a few features of an expert over
// the whole contraction, which k_warps of the CTA's 8 warps share; the others take further
// features, 16 * MT a warp.  A lane (g = lane / 4, t = lane % 4) loads 32 consecutive inputs (16
// bytes) of each of 2 * MT rows, SUB times; a row's place among the MMA's 16 is free, so they are
// neighbouring features (whose scales are neighbours too).  A group has at least 32 inputs: one
// scale for each load.  For 8 tokens two loads are one of 32 bytes, so that a row's four lanes
// read a whole line (16 experts of 4096 x 1024, a token each: 13.7 -> 12.0 us; the second token's
// group would need the registers that hold the inputs of both halves).  The token's inputs come from L1 when they are needed, where a load that
// nobody waits for has brought them a batch ahead; what an item's end reads is loaded ahead, too.
//
// Two rows' words are loaded again, for the lane's next batch (of the next item, after the
// last), as soon as they have been multiplied, so that seven of the eight loads that a lane
// has registers for are in flight all the time.
template <typename T, int RG, int MT, int SUB, int VB>
__global__ void __launch_bounds__(STREAM_WARPS * 32, 2) stream4_kernel(const Stream4Params p) {
    next_may_start();
    previous_done();
    constexpr int WF = 16 * MT, H = 2 * MT, KB = 128 * SUB;  // features of a warp, rows of a lane, inputs of a batch
    constexpr int PAIR = RG == 1 ? 2 : 1;                    // 16-byte pieces of a load
    auto input_of = [](int s) { return s % PAIR * 32 + s / PAIR * 128 * PAIR; };  // piece s of a lane, from its first input
    __shared__ float parts[2][STREAM_WARPS][RG * 8][WF + 1];  // of this item and the one before: one barrier an item
    int turn = 0;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int kw = warp % p.k_warps, fw = warp / p.k_warps, F = STREAM_WARPS / p.k_warps * WF;
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
    const int rounds = (p.words * 8 + p.k_warps * KB - 1) / (p.k_warps * KB);

    // the place of a batch: item (expert e, features from f0 on), its rows rb.. of up to r1, round `it`
    struct At { int e, f0, rb, r1, it; } next = {}, now;
    unsigned item = blockIdx.x - gridDim.x;
    auto next_item = [&]() {  // false: none left
        do {
            item += gridDim.x;
            if (item >= items) return false;
            next.e = (int)(item / (unsigned)p.f_tiles);
            expert_rows(p.offsets, next.e, p.R, next.rb, next.r1);
        } while (next.rb >= next.r1);
        next.f0 = (int)(item - (unsigned)next.e * p.f_tiles) * F;
        next.it = 0;
        return true;
    };
    // where the lane reads the next batch
    const uint32_t* words = nullptr;
    const T* scales = nullptr;
    int fin = 0, k_next = 0;  // the lane's features that exist; its first input
    auto aim = [&]() {
        const int f = next.f0 + WF * fw + H * g;
        fin = clampi(p.N - f, 0, H);
        k_next = (next.it * p.k_warps + kw) * KB + 32 * PAIR * t;
        words = p.packed + ((int64_t)next.e * p.N + (fin ? f : 0)) * p.words + k_next / 8;
        scales = reinterpret_cast<const T*>(p.scales) + (int64_t)next.e * p.parts * p.N + (fin ? f : 0);
        // the batch's inputs of 8 tokens, a line of 64 a lane, into L1
#pragma unroll
        for (int q = 0; q < RG * KB / 256; ++q) {
            const int r = next.rb + 8 * (q % RG) + g, k = (next.it * p.k_warps + kw) * KB + 64 * t + 256 * (q / RG);
            if (r < next.r1 && k < p.K) {
                uint16_t touched;
                asm volatile("ld.global.b16 %0, [%1];" : "=h"(touched) : "l"(reinterpret_cast<const uint16_t*>(p.x) + (int64_t)r * p.ldx + k) : "memory");
            }
        }
    };
    uint4 a[SUB][H];
    uint32_t sc[SUB][MT];  // two features' scales each
    auto load_words = [&](int s, int h) {  // PAIR pieces from s on
#pragma unroll
        for (int i = 0; i < PAIR; ++i) a[s + i][h] = make_uint4(Q_ZERO, Q_ZERO, Q_ZERO, Q_ZERO);
        if (k_next + input_of(s) >= p.words * 8 || h >= fin) return;  // (rows are whole blocks of 64 inputs)
        const uint32_t* from = words + (int64_t)h * p.words + input_of(s) / 8;
        if constexpr (PAIR == 2)
            asm volatile("ld.global.L1::no_allocate.L2::256B.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                : "=r"(a[s][h].x), "=r"(a[s][h].y), "=r"(a[s][h].z), "=r"(a[s][h].w),
                  "=r"(a[s + 1][h].x), "=r"(a[s + 1][h].y), "=r"(a[s + 1][h].z), "=r"(a[s + 1][h].w) : "l"(from) : "memory");
        else
            asm volatile("ld.global.L1::no_allocate.L2::256B.v4.b32 {%0,%1,%2,%3}, [%4];"
                : "=r"(a[s][h].x), "=r"(a[s][h].y), "=r"(a[s][h].z), "=r"(a[s][h].w) : "l"(from) : "memory");
    };
    auto load_scales = [&](int s) {
        const int k = k_next + input_of(s);
        const T* from = scales + (int64_t)min(k >> p.shift, p.parts - 1) * p.N;
#pragma unroll
        for (int m = 0; m < MT; ++m) sc[s][m] = 0;
        if (k >= p.words * 8) return;
        if (p.wide_scales) {
            if constexpr (MT == 1) { if (fin) sc[s][0] = *reinterpret_cast<const uint32_t*>(from); }
            if constexpr (MT == 2) { if (fin) { const uint2 v = *reinterpret_cast<const uint2*>(from); sc[s][0] = v.x; sc[s][1] = v.y; } }
        } else {
#pragma unroll
            for (int h = 0; h < H; ++h)
                if (h < fin) sc[s][h / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(from)[h] << (16 * (h & 1));
        }
    };
    bool more = next_item();
    if (more) {
        aim();
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
            load_scales(s);
            if (s % PAIR == 0)
#pragma unroll
                for (int h = 0; h < H; ++h) load_words(s, h);
        }
    }
    float acc[MT][RG][4] = {};
    while (more) {
        now = next;
        const int k_now = k_next;
        if (++next.it == rounds) {
            next.it = 0;
            next.rb += 8 * RG;
            if (next.rb >= next.r1) more = next_item();
        }
        if (more) aim();
        const bool complete = now.it + 1 == rounds;
        const int rows = min(RG * 8, now.r1 - now.rb);
        float first = 0.f, first_res = 0.f;  // bias and residual of the thread's first value
        if (complete && threadIdx.x < rows * F) {
            const int c = threadIdx.x / F, f = now.f0 + threadIdx.x - c * F;
            if (f < p.N) {
                if (p.bias) first = El<T>::to(reinterpret_cast<const T*>(p.bias)[(int64_t)now.e * p.N + f]);
                if (residual) first_res = El<T>::to(residual[(now.rb + c) * p.ldr + f]);
            }
        }
#pragma unroll
        for (int s0 = 0; s0 < SUB; s0 += PAIR) {
            uint4 b[PAIR][4][RG];
#pragma unroll
            for (int q = 0; q < RG; ++q) {
                const int r = now.rb + 8 * q + g;
                const uint16_t* xrow = reinterpret_cast<const uint16_t*>(p.x) + (int64_t)(r < now.r1 ? r : 0) * p.ldx;
#pragma unroll
                for (int i = 0; i < PAIR; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) b[i][j][q] = load8<VB>(xrow, k_now + input_of(s0 + i) + 8 * j, p.K, r < now.r1);
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
#pragma unroll
                for (int i = 0; i < PAIR; ++i) {
                    const uint32_t even = __byte_perm(sc[s0 + i][m], 0, 0x1010), odd = __byte_perm(sc[s0 + i][m], 0, 0x3232);
                    const uint4 u = a[s0 + i][2 * m], v = a[s0 + i][2 * m + 1];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t lo[4], hi[4];
                        unpack<T>(j == 0 ? u.x : j == 1 ? u.y : j == 2 ? u.z : u.w, even, lo);
                        unpack<T>(j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w, odd, hi);
#pragma unroll
                        for (int q = 0; q < RG; ++q) {
                            mma16816<T>(acc[m][q], lo[0], hi[0], lo[1], hi[1], b[i][j][q].x, b[i][j][q].y);
                            mma16816<T>(acc[m][q], lo[2], hi[2], lo[3], hi[3], b[i][j][q].z, b[i][j][q].w);
                        }
                    }
                }
                if (more) {
                    load_words(s0, 2 * m);
                    load_words(s0, 2 * m + 1);
                }
            }
            if (more)
#pragma unroll
                for (int i = 0; i < PAIR; ++i) load_scales(s0 + i);
        }
        if (!complete) continue;
        auto& part = parts[turn];
        turn ^= 1;
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
        for (int i = threadIdx.x; i < rows * F; i += STREAM_WARPS * 32) {
            const int c = i / F, of = i - c * F, r = now.rb + c, f = now.f0 + of;
            if (f < p.N) {
                float v = 0.f;
                for (int w = 0; w < p.k_warps; ++w) v += part[of / WF * p.k_warps + w][c][of % WF];
                if (i >= STREAM_WARPS * 32) {
                    first = p.bias ? El<T>::to(reinterpret_cast<const T*>(p.bias)[(int64_t)now.e * p.N + f]) : 0.f;
                    first_res = residual ? El<T>::to(residual[r * p.ldr + f]) : 0.f;
                }
                y[(int64_t)r * p.N + f] = El<T>::from(act_any(p.act, v + first) + first_res);
            }
        }
    }
}

// As few warps share a contraction as leave no CTA without an item, since an item's end costs a
// barrier: 16 experts of 4096 x 1024, a token each, take 12.0 us with one (256 items of 256
// features), 14.0 with four; 4096 x 4096 alone 6.8 with eight, 24 with one.
template <typename T, int RG, int MT, int SUB> int stream4_launch(Stream4Params p, bool vec, cudaStream_t st) {
    const int64_t experts = p.E < p.R ? p.E : p.R;
    const auto tiles = [&](int k_warps) { return (p.N + STREAM_WARPS / k_warps * 16 * MT - 1) / (STREAM_WARPS / k_warps * 16 * MT); };
    p.k_warps = STREAM_WARPS;
    while (p.k_warps > 1 && experts * tiles(p.k_warps / 2) >= 3 * sm_count() / 2) p.k_warps /= 2;
    while (p.k_warps > 1 && p.k_warps / 2 * 128 * SUB >= p.words * 8) p.k_warps /= 2;  // (no batch for more)
    p.f_tiles = tiles(p.k_warps);
    p.wide_scales = p.N % (2 * MT) == 0 && (reinterpret_cast<uintptr_t>(p.scales) & (4 * MT - 1)) == 0;
    const int64_t items = (int64_t)p.E * p.f_tiles, most = 2 * (int64_t)sm_count();
    if (items > INT32_MAX) return ELA_ERR_UNSUPPORTED;
    return launch(vec ? stream4_kernel<T, RG, MT, SUB, 16> : stream4_kernel<T, RG, MT, SUB, 2>, (unsigned)(items < most ? items : most),
                  STREAM_WARPS * 32, 0, st, p);
}

// Rows per expert up to which the weights are streamed (both ways in loops of 20): 8 rows for
// each of 16 experts of 4096 x 1024 take 19.1 us here and 22.9 by tiles, of 4096 x 2048 31.0 and
// 34.5; 12 rows 37.3 and 34.6, 16 rows 26.6 and 22.4, 40.5 and 34.0.  Where tiles of 256 features
// leave half of the pairs idle, up to 24: 4096 x 4096 alone with 16 rows 8.8 and 18.6, with 32 15.6
// and 18.8, with 48 22.4 and 19.8; two of 2048 x 2048 with 16 rows each 8.9 and 13.1, with 32 15.6
// and 13.3.  The loads, which only the device knows, are taken to be equal.  Others cost here what the
// busiest expert does, whose weights are read again for each 8 rows: 128 rows of 16 experts of 4096 x 1024 take 18.8
// us, 102 with half of them on one expert and 181 with all, 1024 rows of 128 of 1024 x 512 24, 511 and 1130; by
// tiles (136 and 1032 rows) 22.4, 22.5 and 13.8, and 24.5, 26.7 and 12.3.
inline bool few_rows_4bit(int64_t R, int64_t E, int64_t N) { return R <= 8 * E || (R <= 24 * E && E * ((N + 255) / 256) <= sm_count() / 4); }

// Eight tokens from one read of the weights, or sixteen.  Items of 16 features a warp where 32
// would leave half of the CTAs without one.
template <typename T> int stream4(const Stream4Params& p, bool vec, cudaStream_t st) {
    const int64_t experts = p.E < p.R ? p.E : p.R;
    const bool narrow = experts * ((p.N + 31) / 32) <= sm_count();
    if (p.R <= 8 * p.E) return narrow ? stream4_launch<T, 1, 1, 4>(p, vec, st) : stream4_launch<T, 1, 2, 2>(p, vec, st);
    return narrow ? stream4_launch<T, 2, 1, 4>(p, vec, st) : stream4_launch<T, 2, 2, 2>(p, vec, st);
}

}  // namespace ela_expert
