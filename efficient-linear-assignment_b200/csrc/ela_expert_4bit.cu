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
    uint16_t w[STEPS][8];
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
        unsigned most = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) most = max(most, w[i][j] & 0x7fffu);
        for (int o = 1; o < group_lanes; o <<= 1) most = max(most, __shfl_xor_sync(~0u, most, o));
        const uint16_t bits = (uint16_t)most;
        T largest;
        memcpy(&largest, &bits, 2);
        const T scale = El<T>::from(El<T>::to(largest) / 7.f);
        const float s = El<T>::to(scale);
        uint32_t word = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            T v;
            memcpy(&v, &w[i][j], 2);
            const float q = s > 0.f && s < INFINITY ? fminf(fmaxf(rintf(El<T>::to(v) / s), -8.f), 7.f) : 0.f;
            word |= (uint32_t)((int)q + 8) << (4 * (j / 2) + 16 * (j % 2));
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

template <typename T, bool VEC>
__global__ void __launch_bounds__(PACK_WARPS * 32) dequantize_kernel(const uint32_t* packed, const T* scales, int K, int N, int shift, int words,
                                                                     int parts, T* weight) {
    next_may_start();
    previous_done();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int chunks = (words * 8 + PACK_K - 1) / PACK_K, strips = (N + PACK_ROWS - 1) / PACK_ROWS;
    const int chunk = blockIdx.x % chunks, strip = blockIdx.x / chunks % strips, e = blockIdx.x / chunks / strips;
    const int k = chunk * PACK_K + 8 * lane;
    if (k >= K) return;
    constexpr int STEPS = PACK_ROWS / PACK_WARPS;
    uint32_t w[STEPS];
    T s[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int n = strip * PACK_ROWS + warp + PACK_WARPS * i;
        if (n < N) {
            w[i] = packed[((int64_t)e * N + n) * words + k / 8];
            s[i] = scales[((int64_t)e * parts + (k >> shift)) * N + n];
        }
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int n = strip * PACK_ROWS + warp + PACK_WARPS * i;
        if (n >= N) break;
        T* out = weight + ((int64_t)e * N + n) * K + k;
        uint32_t v[4];
        unpack<T>(w[i], scale_pair(s[i]), v);
        if (VEC) {
            *reinterpret_cast<uint4*>(out) = make_uint4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (k + j < K) reinterpret_cast<uint16_t*>(out)[j] = (uint16_t)(v[j / 2] >> (16 * (j & 1)));
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
        Stream4Params p = {x, (const uint32_t*)packed, scales, bias, residual, offsets, (int)R, (int)E, (int)K, (int)N, words, parts, shift, 0,
                           activation, 0, ldx, ldr, y};
        const bool vec = aligned16(x, ldx * 2) && K % 8 == 0;
        ELA_BY_TYPE(dtype, { rc = R <= 8 * E ? stream4_launch<T_, 1, 2, 2>(p, vec, st) : stream4_launch<T_, 4, 2, 2>(p, vec, st); })
        return rc;
    }
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
