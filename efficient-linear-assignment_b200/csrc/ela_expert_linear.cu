// ela_expert_linear.cu -- the product with each expert's weights and its
// gradient (include/ela_expert.h).
//
// Three products share one form, C[m,n] = sum_k A(m,k) B(n,k):
//   forward       C = z  (rows x N):  A = x rows,  B = W_e rows,     sum over K
//   input grad    C = dx (rows x K):  A = dz rows, B = W_e columns,  sum over N
//   weight grad   C = dW_e (N x K):   A = dz columns, B = x columns, sum over the expert's rows

#include "ela_expert.cuh"

namespace ela_expert {

// ------------------------------------------------- the product, simple form
// A 64 x 64 tile of C per CTA, fp32 sums in registers, operands of any stride
// staged 16 deep in shared memory.
#define ELA_TILE 64
#define ELA_DEPTH 16

struct Operand {
    const void* p;
    int64_t s_mn, s_k, s_e;  // distance along m (or n), along k, between experts
};

template <typename T, int ACT>
__device__ __forceinline__ void finish(float z, int64_t at, const T* bias, int64_t bias_at, const T* residual,
                                       int64_t res_at, T* y, T* zout) {
    if (bias) z += El<T>::to(bias[bias_at]);
    if (zout) zout[at] = El<T>::from(z);
    float v = act_value<ACT>(z);
    if (residual) v += El<T>::to(residual[res_at]);
    y[at] = El<T>::from(v);
}

// ROWS: C's rows are the expert's rows (forward, input grad); else the sum runs over them.
template <typename T, int ACT, bool ROWS>
__global__ void __launch_bounds__(256) simple_kernel(Operand A, Operand B, const int32_t* offsets, int R, int E, int M,
                                                     int N, int K, const T* bias, const T* residual, int64_t ldr,
                                                     T* C, T* zout) {
    __shared__ float as[ELA_DEPTH][ELA_TILE + 1], bs[ELA_DEPTH][ELA_TILE + 1];
    __shared__ int s_e, s_m;
    int e, m0, r0, r1;
    if (ROWS) {  // blockIdx.y counts the experts' row tiles
        if (threadIdx.x == 0) {
            int tile = blockIdx.y, f = 0, m = 0;
            for (; f < E; ++f) {
                int a, b;
                expert_rows(offsets, f, R, a, b);
                const int tiles = (b - a + ELA_TILE - 1) / ELA_TILE;
                if (tile < tiles) { m = a + tile * ELA_TILE; break; }
                tile -= tiles;
            }
            s_e = f;
            s_m = m;
        }
        __syncthreads();
        e = s_e;
        m0 = s_m;
        if (e >= E) return;
        expert_rows(offsets, e, R, r0, r1);
    } else {
        e = blockIdx.z;
        m0 = blockIdx.y * ELA_TILE;
        expert_rows(offsets, e, R, r0, r1);
    }
    const int n0 = blockIdx.x * ELA_TILE;
    const int m_end = ROWS ? r1 : M;
    const int k_begin = ROWS ? 0 : r0, k_end = ROWS ? K : r1;
    const T* a = reinterpret_cast<const T*>(A.p) + (int64_t)e * A.s_e;
    const T* b = reinterpret_cast<const T*>(B.p) + (int64_t)e * B.s_e;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float acc[4][4] = {};
    for (int k0 = k_begin; k0 < k_end; k0 += ELA_DEPTH) {
        for (int i = threadIdx.x; i < ELA_TILE * ELA_DEPTH; i += 256) {
            const int mn = A.s_k == 1 ? i / ELA_DEPTH : i % ELA_TILE, k = A.s_k == 1 ? i % ELA_DEPTH : i / ELA_TILE;
            as[k][mn] = m0 + mn < m_end && k0 + k < k_end ? El<T>::to(a[(m0 + mn) * A.s_mn + (k0 + k) * A.s_k]) : 0.f;
        }
        for (int i = threadIdx.x; i < ELA_TILE * ELA_DEPTH; i += 256) {
            const int mn = B.s_k == 1 ? i / ELA_DEPTH : i % ELA_TILE, k = B.s_k == 1 ? i % ELA_DEPTH : i / ELA_TILE;
            bs[k][mn] = n0 + mn < N && k0 + k < k_end ? El<T>::to(b[(n0 + mn) * B.s_mn + (k0 + k) * B.s_k]) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < ELA_DEPTH; ++k) {
            float av[4], bv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) { av[i] = as[k][ty * 4 + i]; bv[i] = bs[k][tx * 4 + i]; }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(av[i], bv[j], acc[i][j]);
        }
        __syncthreads();
    }
    T* c = C + (ROWS ? 0 : (int64_t)e * M * N);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
            if (m < m_end && n < N)
                finish<T, ACT>(acc[i][j], (int64_t)m * N + n, bias, (int64_t)e * N + n, residual, (int64_t)m * ldr + n, c, zout);
        }
}

// Rows of no expert: the residual, or 0.
template <typename T>
__global__ void __launch_bounds__(256) rest_kernel(const int32_t* offsets, int E, int R, int N, const T* residual,
                                                   int64_t ldr, T* y) {
    const int first = clampi(offsets[0], 0, R), last = clampi(offsets[E], 0, R);
    for (int r = blockIdx.x; r < R; r += gridDim.x) {
        if (r >= first && r < last) { r = last - 1 - (last - 1 - r) % (int)gridDim.x; continue; }
        for (int n = threadIdx.x; n < N; n += blockDim.x)
            y[(int64_t)r * N + n] = residual ? residual[(int64_t)r * ldr + n] : El<T>::from(0.f);
    }
}

// dz = dy * act'(z) and the bias gradient: a CTA owns 32 columns of an expert;
// 8 rows at a time, the 8 partial sums joined at the end.
template <typename T, int ACT>
__global__ void __launch_bounds__(256) grad_act_kernel(const T* dy, const T* z, const int32_t* offsets, int R, int N,
                                                       T* dz, T* dbias) {
    __shared__ float part[8][32];
    const int e = blockIdx.y, c = threadIdx.x & 31, w = threadIdx.x >> 5, n = blockIdx.x * 32 + c;
    int r0, r1;
    expert_rows(offsets, e, R, r0, r1);
    float sum = 0.f;
    if (n < N)
        for (int r = r0 + w; r < r1; r += 8) {
            const int64_t at = (int64_t)r * N + n;
            float g = El<T>::to(dy[at]);
            if (ACT != ELA_ACT_NONE) g *= act_slope<ACT>(El<T>::to(z[at]));
            if (dz) dz[at] = El<T>::from(g);
            sum += g;
        }
    part[w][c] = sum;
    __syncthreads();
    if (w == 0 && n < N && dbias) {
        for (int i = 1; i < 8; ++i) sum += part[i][c];
        dbias[(int64_t)e * N + n] = El<T>::from(sum);
    }
}

inline bool linear_sizes_ok(int dtype, int64_t R, int64_t E, int64_t K, int64_t N, const int32_t* offsets) {
    return (dtype == ELA_DTYPE_F16 || dtype == ELA_DTYPE_BF16) && R >= 0 && R <= (1ll << 30) && E >= 1 &&
           E <= ELA_EXPERT_MAX && K >= 1 && K <= (1ll << 30) && N >= 1 && N <= (1ll << 30) && (offsets || E == 1);
}
inline unsigned tiles(int64_t n) { return (unsigned)((n + ELA_TILE - 1) / ELA_TILE); }

#define ELA_BY_TYPE(dtype, ...)                               \
    if ((dtype) == ELA_DTYPE_F16) { typedef __half T_; __VA_ARGS__; } \
    else { typedef __nv_bfloat16 T_; __VA_ARGS__; }
#define ELA_BY_ACT(act, ...)                                          \
    switch (act) {                                                     \
    case ELA_ACT_RELU: { constexpr int A_ = ELA_ACT_RELU; __VA_ARGS__; break; } \
    case ELA_ACT_GELU: { constexpr int A_ = ELA_ACT_GELU; __VA_ARGS__; break; } \
    case ELA_ACT_SILU: { constexpr int A_ = ELA_ACT_SILU; __VA_ARGS__; break; } \
    default: { constexpr int A_ = ELA_ACT_NONE; __VA_ARGS__; break; }           \
    }

}  // namespace ela_expert

using namespace ela_expert;

extern "C" {

size_t ela_expert_linear_workspace_bytes(int, int64_t, int64_t, int64_t, int64_t, int) { return 0; }

int ela_expert_linear(const void* x, const void* weight, const void* bias, const void* residual,
                      const int32_t* offsets, int dtype, int64_t R, int64_t E, int64_t K, int64_t N, int64_t ldx,
                      int64_t stride_e, int64_t ldw, int64_t ldr, int activation, void* y, void* z, void*, size_t,
                      void* stream) {
    if (!linear_sizes_ok(dtype, R, E, K, N, offsets) || activation < 0 || activation > ELA_ACT_SILU || ldx < 0 ||
        stride_e < 0 || ldw < 0 || ldr < 0)
        return ELA_ERR_ARGUMENT;
    if (R == 0) return ELA_OK;
    if (!x || !weight || !y) return ELA_ERR_ARGUMENT;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const Operand A = {x, ldx, 1, 0}, B = {weight, ldw, 1, stride_e};
    const dim3 grid(tiles(N), tiles(R) + (unsigned)(E - 1));
    ELA_BY_TYPE(dtype, {
        if (offsets)
            rest_kernel<T_><<<(unsigned)(R < 592 ? R : 592), 256, 0, st>>>(offsets, (int)E, (int)R, (int)N, (const T_*)residual, ldr, (T_*)y);
        ELA_BY_ACT(activation, (simple_kernel<T_, A_, true><<<grid, 256, 0, st>>>(A, B, offsets, (int)R, (int)E, (int)R, (int)N, (int)K,
                                (const T_*)bias, (const T_*)residual, ldr, (T_*)y, (T_*)z)))
    })
    return launch_status();
}

int ela_expert_linear_grad_act(const void* dy, const void* z, const int32_t* offsets, int dtype, int64_t R,
                               int64_t E, int64_t N, int activation, void* dz, void* dbias, void*, size_t,
                               void* stream) {
    if (!linear_sizes_ok(dtype, R, E, 1, N, offsets) || activation < 0 || activation > ELA_ACT_SILU)
        return ELA_ERR_ARGUMENT;
    if ((R == 0 && !dbias) || (!dz && !dbias)) return ELA_OK;
    if (R > 0 && (!dy || (!z && activation != ELA_ACT_NONE))) return ELA_ERR_ARGUMENT;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)((N + 31) / 32), (unsigned)E);
    ELA_BY_TYPE(dtype, {
        ELA_BY_ACT(activation, (grad_act_kernel<T_, A_><<<grid, 256, 0, st>>>((const T_*)dy, (const T_*)z, offsets, (int)R, (int)N, (T_*)dz, (T_*)dbias)))
    })
    return launch_status();
}

int ela_expert_linear_grad_input(const void* dz, const void* weight, const int32_t* offsets, int dtype, int64_t R,
                                 int64_t E, int64_t K, int64_t N, int64_t stride_e, int64_t ldw, void* dx, void*,
                                 size_t, void* stream) {
    if (!linear_sizes_ok(dtype, R, E, K, N, offsets) || stride_e < 0 || ldw < 0) return ELA_ERR_ARGUMENT;
    if (R == 0) return ELA_OK;
    if (!dz || !weight || !dx) return ELA_ERR_ARGUMENT;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const Operand A = {dz, N, 1, 0}, B = {weight, 1, ldw, stride_e};
    const dim3 grid(tiles(K), tiles(R) + (unsigned)(E - 1));
    ELA_BY_TYPE(dtype, {
        if (offsets)
            rest_kernel<T_><<<(unsigned)(R < 592 ? R : 592), 256, 0, st>>>(offsets, (int)E, (int)R, (int)K, (const T_*)nullptr, 0, (T_*)dx);
        simple_kernel<T_, ELA_ACT_NONE, true><<<grid, 256, 0, st>>>(A, B, offsets, (int)R, (int)E, (int)R, (int)K, (int)N,
                                                                    (const T_*)nullptr, (const T_*)nullptr, 0, (T_*)dx, (T_*)nullptr);
    })
    return launch_status();
}

int ela_expert_linear_grad_weight(const void* dz, const void* x, const int32_t* offsets, int dtype, int64_t R,
                                  int64_t E, int64_t K, int64_t N, int64_t ldx, void* dweight, void*, size_t,
                                  void* stream) {
    if (!linear_sizes_ok(dtype, R, E, K, N, offsets) || ldx < 0) return ELA_ERR_ARGUMENT;
    if (!dweight || (R > 0 && (!dz || !x))) return ELA_ERR_ARGUMENT;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const Operand A = {dz, 1, N, 0}, B = {x, 1, ldx, 0};
    const dim3 grid(tiles(K), tiles(N), (unsigned)E);
    ELA_BY_TYPE(dtype, {
        simple_kernel<T_, ELA_ACT_NONE, false><<<grid, 256, 0, st>>>(A, B, offsets, (int)R, (int)E, (int)N, (int)K, (int)R,
                                                                     (const T_*)nullptr, (const T_*)nullptr, 0, (T_*)dweight, (T_*)nullptr);
    })
    return launch_status();
}

}  // extern "C"
