// ela_expert_4bit.cu -- experts' weights in 4 bits with a scale per group of inputs
// (include/ela_expert.h): made from 16-bit weights, turned back into them, and multiplied.

#include "ela_expert_4bit.cuh"
#include "ela_expert_mma.cuh"

namespace ela_expert {

// A block takes 32 rows by 256 inputs; a warp a row at a time, a lane 8 inputs, which are a
// 16-byte load and a word.  The lanes of a group share its largest magnitude (as bits: those of
// 16-bit floats without a sign compare as numbers, NaN above all).  A block's scales go through
// shared memory, so that they are stored 64 bytes at a time.
constexpr int PACK_ROWS = 32, PACK_K = 256, PACK_WARPS = 8;

template <typename T, bool VEC>
__global__ void __launch_bounds__(PACK_WARPS * 32) quantize_kernel(const T* weight, int K, int N, int64_t stride_e, int64_t ldw, int shift,
                                                                   int words, int parts, uint32_t* packed, T* scales) {
    next_may_start();
    previous_done();
    __shared__ T s_scale[PACK_K / 32][PACK_ROWS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int chunks = (words * 8 + PACK_K - 1) / PACK_K, strips = (N + PACK_ROWS - 1) / PACK_ROWS;
    const int chunk = blockIdx.x % chunks, strip = blockIdx.x / chunks % strips, e = blockIdx.x / chunks / strips;
    const int k = chunk * PACK_K + 8 * lane, n0 = strip * PACK_ROWS, group_lanes = 1 << (shift - 3);
    constexpr int STEPS = PACK_ROWS / PACK_WARPS;
    constexpr float LEAST = El<T>::BF16 ? 1.17549435e-38f : 6.103515625e-5f;  // the least scale of full precision
    uint32_t w[STEPS][4];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int n = n0 + warp + PACK_WARPS * i;
        const uint16_t* row = reinterpret_cast<const uint16_t*>(weight) + e * stride_e + (int64_t)(n < N ? n : 0) * ldw;
        const uint4 v = load8<VEC ? 16 : 2>(row, k, K, n < N);
        memcpy(w[i], &v, 16);
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int r = warp + PACK_WARPS * i, n = n0 + r;
        uint32_t most = 0;  // of both halves
#pragma unroll
        for (int j = 0; j < 4; ++j) most = __vmaxu2(most, w[i][j] & 0x7fff7fffu);
        for (int o = 1; o < group_lanes; o <<= 1) most = __vmaxu2(most, __shfl_xor_sync(~0u, most, o));
        const uint16_t bits = (uint16_t)max(most >> 16, most & 0xffffu);
        T largest;
        memcpy(&largest, &bits, 2);
        // (a seventh is never halfway between two scales: 7 times an odd number has more bits than a
        // weight; so the product with 1/7, off by 2^-23, is rounded as the quotient)
        const T scale = El<T>::from(El<T>::to(largest) * 0.142857142857142857f);
        const float s = El<T>::to(scale);
        uint32_t word = 0;
        if (s >= LEAST && s < INFINITY) {
            // w / s by the reciprocal, onto multiples of 2^-14 and then onto whole numbers.  The product is
            // off by 2^-20 at most; w / s is halfway between whole numbers or, both having 11 bits at most,
            // 2^-12 and more away from there, so the second rounding decides as if on w / s.  The whole
            // number plus 8 is left in the last bits of the float; what the float has above them adds up to
            // the constant.
            const float reciprocal = reciprocal_fast(s);
            constexpr float GRID = 768.f, WHOLE = 12582912.f + 8.f;  // 1.5 * 2^9, 1.5 * 2^23
            constexpr uint32_t ABOVE = 0x4b400000u;
            uint32_t above = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 v = unpack2<T>(w[i][j]);
                const float q0 = __fadd_rn(__fadd_rn(__fmaf_rn(v.x, reciprocal, GRID), -GRID), WHOLE);
                const float q1 = __fadd_rn(__fadd_rn(__fmaf_rn(v.y, reciprocal, GRID), -GRID), WHOLE);
                word += (__float_as_uint(q0) << (4 * j)) + (__float_as_uint(q1) << (4 * j + 16));
                above += (ABOVE << (4 * j)) + (ABOVE << (4 * j + 16));
            }
            word -= above;
        } else {  // the scale is 0, has fewer bits (and |q| may pass 7), or is no number
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float2 pair = unpack2<T>(w[i][j / 2]);
                const float v = j & 1 ? pair.y : pair.x, q = s > 0.f && s < INFINITY ? fminf(fmaxf(rintf(v / s), -8.f), 7.f) : 0.f;
                word |= (uint32_t)((int)q + 8) << (4 * (j / 2) + 16 * (j % 2));
            }
        }
        if (n < N && k < words * 8) packed[((int64_t)e * N + n) * words + k / 8] = word;
        if ((lane & (group_lanes - 1)) == 0) s_scale[8 * lane >> shift][r] = scale;
    }
    __syncthreads();
    const int groups = PACK_K >> shift;
    for (int i = threadIdx.x; i < groups * PACK_ROWS; i += PACK_WARPS * 32) {
        const int part = chunk * groups + i / PACK_ROWS, n = n0 + i % PACK_ROWS;
        if (part < parts && n < N) scales[((int64_t)e * parts + part) * N + n] = s_scale[i / PACK_ROWS][i % PACK_ROWS];
    }
}

// Rows off their 16 bytes go through shared memory and are stored 4 bytes a lane, 128 in a row (1027 x 2051: 17 us
// with eight 2-byte stores a lane).
template <typename T, bool VEC>
__global__ void __launch_bounds__(PACK_WARPS * 32) dequantize_kernel(const uint32_t* packed, const T* scales, int K, int N, int shift, int words,
                                                                     int parts, T* weight) {
    next_may_start();
    previous_done();
    __shared__ __align__(16) uint16_t s_row[VEC ? 1 : PACK_WARPS][VEC ? 8 : PACK_K];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int chunks = (words * 8 + PACK_K - 1) / PACK_K, strips = (N + PACK_ROWS - 1) / PACK_ROWS;
    const int chunk = blockIdx.x % chunks, strip = blockIdx.x / chunks % strips, e = blockIdx.x / chunks / strips;
    const int k0 = chunk * PACK_K, k = k0 + 8 * lane, count = min(K - k0, PACK_K);
    if (count <= 0) return;
    constexpr int STEPS = PACK_ROWS / PACK_WARPS;
    uint32_t w[STEPS];
    T s[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int n = strip * PACK_ROWS + warp + PACK_WARPS * i;
        if (n < N && k < K) {
            w[i] = packed[((int64_t)e * N + n) * words + k / 8];
            s[i] = scales[((int64_t)e * parts + (k >> shift)) * N + n];
        }
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int n = strip * PACK_ROWS + warp + PACK_WARPS * i;
        if (n >= N) break;
        uint16_t* out = reinterpret_cast<uint16_t*>(weight) + ((int64_t)e * N + n) * K + k0;
        uint32_t v[4] = {};
        if (k < K) unpack<T>(w[i], scale_pair(s[i]), v);
        if constexpr (VEC) {
            if (k < K) *reinterpret_cast<uint4*>(out + 8 * lane) = make_uint4(v[0], v[1], v[2], v[3]);
        } else {
            *reinterpret_cast<uint4*>(&s_row[warp][8 * lane]) = make_uint4(v[0], v[1], v[2], v[3]);
            __syncwarp();
            const int odd = reinterpret_cast<uintptr_t>(out) >> 1 & 1;  // words start at the element before
            for (int j = 2 * lane - odd; j < count; j += 64) {
                if (j >= 0 && j + 1 < count) *reinterpret_cast<uint32_t*>(out + j) = s_row[warp][j] | (uint32_t)s_row[warp][j + 1] << 16;
                else if (j >= 0) out[j] = s_row[warp][j];
                else out[0] = s_row[warp][0];
            }
            __syncwarp();
        }
    }
}

inline int group_shift(int64_t group) { return group == 32 ? 5 : group == 64 ? 6 : group == 128 ? 7 : 0; }
inline bool sizes_4bit_ok(int dtype, int64_t E, int64_t K, int64_t N, int64_t group) {
    return (dtype == ELA_DTYPE_F16 || dtype == ELA_DTYPE_BF16) && E >= 1 && E <= ELA_EXPERT_MAX && K >= 1 && K <= (1ll << 30) &&
           N >= 1 && N <= (1ll << 30) && group_shift(group) != 0;
}
inline int64_t pack_blocks(int64_t E, int64_t K, int64_t N) {
    return (q_words(K) * 8 + PACK_K - 1) / PACK_K * ((N + PACK_ROWS - 1) / PACK_ROWS) * E;
}

// Error of the tiles' waits on the current device, read and cleared (for ela_expert_status).
int status_4bit(int* status) {
    const int zero = ELA_OK;
    if (cudaMemcpyFromSymbol(status, g_expert_error, sizeof(int)) != cudaSuccess) return ELA_ERR_CUDA;
    if (*status != ELA_OK && cudaMemcpyToSymbol(g_expert_error, &zero, sizeof(int)) != cudaSuccess) return ELA_ERR_CUDA;
    return ELA_OK;
}

}  // namespace ela_expert

using namespace ela_expert;

extern "C" {

int ela_expert_quantize(const void* weight, int dtype, int64_t E, int64_t K, int64_t N, int64_t stride_e, int64_t ldw,
                        int64_t group, int32_t* packed, void* scales, void* stream) {
    if (!sizes_4bit_ok(dtype, E, K, N, group) || stride_e < 0 || ldw < 0 || !weight || !packed || !scales ||
        !on_elements(2, weight, scales) || !on_elements(32, packed))
        return ELA_ERR_ARGUMENT;
    const int64_t blocks = pack_blocks(E, K, N);
    if (blocks > INT32_MAX) return ELA_ERR_UNSUPPORTED;
    const bool vec = aligned16(weight, ldw * 2) && (E == 1 || stride_e % 8 == 0) && K % 8 == 0;
    int rc = ELA_OK;
    ELA_BY_TYPE(dtype, {
        rc = launch(vec ? quantize_kernel<T_, true> : quantize_kernel<T_, false>, (unsigned)blocks, PACK_WARPS * 32, 0, reinterpret_cast<cudaStream_t>(stream),
                    (const T_*)weight, (int)K, (int)N, stride_e, ldw, group_shift(group), (int)q_words(K), (int)((K + group - 1) / group),
                    (uint32_t*)packed, (T_*)scales);
    })
    return rc;
}

int ela_expert_dequantize(const int32_t* packed, const void* scales, int dtype, int64_t E, int64_t K, int64_t N,
                          int64_t group, void* weight, void* stream) {
    if (!sizes_4bit_ok(dtype, E, K, N, group) || !weight || !packed || !scales || !on_elements(2, weight, scales) || !on_elements(32, packed))
        return ELA_ERR_ARGUMENT;
    const int64_t blocks = pack_blocks(E, K, N);
    if (blocks > INT32_MAX) return ELA_ERR_UNSUPPORTED;
    const bool vec = aligned16(weight, K * 2);
    int rc = ELA_OK;
    ELA_BY_TYPE(dtype, {
        rc = launch(vec ? dequantize_kernel<T_, true> : dequantize_kernel<T_, false>, (unsigned)blocks, PACK_WARPS * 32, 0, reinterpret_cast<cudaStream_t>(stream),
                    (const uint32_t*)packed, (const T_*)scales, (int)K, (int)N, group_shift(group), (int)q_words(K), (int)((K + group - 1) / group), (T_*)weight);
    })
    return rc;
}

size_t ela_expert_linear_4bit_workspace_bytes(int64_t R, int64_t E, int64_t K, int64_t N, int64_t group, int aligned) {
    if (few_rows_4bit(R, E, N) || group_shift(group) == 0) return 0;
    const Matrix x = {nullptr, 1, R, K, 0, 0}, scales = {nullptr, 1, E * ((K + group - 1) / group), N, 0, 0};
    return (aligned ? 0 : x.padded_bytes()) + (aligned && N % 8 == 0 ? 0 : scales.padded_bytes());
}

int ela_expert_linear_4bit(const void* x, const int32_t* packed, const void* scales, const void* bias,
                           const void* residual, const int32_t* offsets, int dtype, int64_t R, int64_t E, int64_t K,
                           int64_t N, int64_t group, int64_t ldx, int64_t ldr, int activation, void* y,
                           void* workspace, size_t workspace_bytes, void* stream) {
    if (!sizes_4bit_ok(dtype, E, K, N, group) || !linear_sizes_ok(dtype, R, E, K, N, offsets) || activation < 0 || activation > ELA_ACT_SILU ||
        ldx < 0 || ldr < 0)
        return ELA_ERR_ARGUMENT;
    if (R == 0) return ELA_OK;
    if (!x || !packed || !scales || !y || !on_elements(2, x, scales, bias, residual, y) || !on_elements(4, offsets) || !on_elements(32, packed))
        return ELA_ERR_ARGUMENT;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const int words = (int)q_words(K), parts = (int)((K + group - 1) / group), shift = group_shift(group);
    int rc = ELA_OK;
    if (few_rows_4bit(R, E, N)) {
        Stream4Params p = {x, (const uint32_t*)packed, scales, bias, residual, offsets, (int)R, (int)E, (int)K, (int)N, words, parts, shift, 0, 0,
                           activation, 0, ldx, ldr, y};
        const bool vec = aligned16(x, ldx * 2) && K % 8 == 0;
        ELA_BY_TYPE(dtype, { rc = stream4<T_>(p, vec, st); })
        return rc;
    }
    if (E * parts > INT32_MAX) return ELA_ERR_UNSUPPORTED;
    char* ws = reinterpret_cast<char*>(workspace);
    Matrix mx = {x, 1, R, K, ldx, 0}, ms = {scales, 1, E * parts, N, N, 0};
    if ((rc = readable(mx, ws, workspace_bytes, st)) != ELA_OK || (rc = readable(ms, ws, workspace_bytes, st)) != ELA_OK) return rc;
    MmaParams4 p = {};
    static_cast<MmaParams&>(p) = row_pass(offsets, R, E, N, K, true);
    p.bias = bias;
    p.parts = parts;
    p.shift = shift;
    p.residual = residual;
    p.ldr = ldr;
    p.out = y;
    p.vec = N % 2 == 0 && aligned4(y) && (!residual || (aligned4(residual) && ldr % 2 == 0));
    CUtensorMap a, b;
    if (!make_words_map(&a, packed, words, N, E) || !map_of(&b, dtype, mx, MMA_KB, p.bbox, false) ||
        !make_scales_map(&p.map_scales, ms.p, N, E * parts, ms.ld, 128 / (int)group))
        return ELA_ERR_CUDA;
    ELA_BY_TYPE(dtype, { ELA_BY_ACT(activation, rc = (mma_launch<PASS_4BIT, T_, A_>(a, b, p, row_tiles(p), st))) })
    return rc;
}

}  // extern "C"
