// ela_expert_linear.cu -- the product with each expert's weights and its
// gradient (include/ela_expert.h).
//
// The three products (forward, input gradient, weight gradient) are one
// tensor-core kernel, ela_expert_mma.cuh; the forward product of a few rows per
// expert streams the weights instead, ela_expert_stream.cuh; here are their entry points, the copies
// of operands that TMA cannot address, and the gradient of the activation with the
// bias gradient.

#include "ela_expert.cuh"
#include "ela_expert_mma.cuh"
#include "ela_expert_stream.cuh"

namespace ela_expert {

// Limit of every device-side wait: 2 s, and 4 us for each block of 64 k of a tile's sum, ten times
// what one takes, so that a sum of hundreds of millions of terms is not given up on.
inline unsigned long long wait_limit(int64_t k) { return 2000000000ull + 4000ull * (unsigned long long)(k / 64); }

// Rows of any stride and alignment copied to rows a multiple of 16 bytes apart
// (TMA's rule for strides and base).  Bits are moved, types do not matter.  A thread
// writes 16 bytes; where the source is off a 4-byte boundary it reads the five words
// around them (no word is touched that does not hold an element of the row).
__global__ void __launch_bounds__(256) realign_kernel(const uint16_t* src, int64_t rows, int cols, int64_t ld,
                                                      int64_t rows_per_matrix, int64_t stride_e, uint16_t* dst, int64_t ldd) {
    next_may_start();
    previous_done();
    const int pieces = (cols + 7) / 8;
    const int64_t all = rows * pieces;
    const int64_t step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t i0 = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i0 < all; i0 += 2 * step) {
        uint4 o[2];  // two pieces' loads before their stores
        uint16_t* to[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t i = i0 + h * step, r = i / pieces;
            to[h] = nullptr;
            if (i >= all) continue;
            const int c = (int)(i - r * pieces) * 8, left = cols - c;
            const uint16_t* s = src + r / rows_per_matrix * stride_e + r % rows_per_matrix * ld + c;
            const bool shift = (reinterpret_cast<uintptr_t>(s) & 3) != 0;
            const uint32_t* w = reinterpret_cast<const uint32_t*>(s - shift);
            uint32_t v[5];
#pragma unroll
            for (int k = 0; k < 5; ++k) v[k] = 2 * k - shift < left && (k < 4 || shift) ? w[k] : 0u;
            o[h].x = shift ? __funnelshift_r(v[0], v[1], 16) : v[0];
            o[h].y = shift ? __funnelshift_r(v[1], v[2], 16) : v[1];
            o[h].z = shift ? __funnelshift_r(v[2], v[3], 16) : v[2];
            o[h].w = shift ? __funnelshift_r(v[3], v[4], 16) : v[3];
            to[h] = dst + r * ldd + c;  // (ldd is cols rounded up to 8)
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (to[h]) *reinterpret_cast<uint4*>(to[h]) = o[h];
    }
}

inline int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }
inline size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// A matrix operand: (matrices, rows, cols), 16-bit.
struct Matrix {
    const void* p;
    int64_t matrices, rows, cols, ld, stride_e;
    size_t padded_bytes() const { return round256((size_t)(matrices * rows * round8(cols)) * 2); }
    bool ok() const { return aligned16(p, ld * 2) && (matrices == 1 || stride_e * 2 % 16 == 0); }
};

// The matrix itself where TMA can read it, else its copy in the workspace.
inline int readable(Matrix& m, char*& ws, size_t& left, cudaStream_t st) {
    if (m.ok()) return ELA_OK;
    const size_t need = m.padded_bytes();
    if (!ws || left < need || !aligned16(ws)) return ELA_ERR_ARGUMENT;
    const int64_t rows = m.matrices * m.rows, ld = round8(m.cols);
    const int64_t blocks = (rows * (ld / 8) + 255) / 256, most = 8 * (int64_t)sm_count();
    const int rc = launch(realign_kernel, (unsigned)(blocks < most ? blocks : most), 256, 0, st, (const uint16_t*)m.p, rows, (int)m.cols, m.ld, m.rows, m.stride_e, (uint16_t*)ws, ld);
    m.p = ws;
    m.ld = ld;
    m.stride_e = m.rows * ld;
    ws += need;
    left -= need;
    return rc;
}
inline bool map_of(CUtensorMap* map, int dtype, const Matrix& m, int box_cols, int box_rows, bool three) {
    const int64_t se = m.matrices > 1 ? m.stride_e : round8(m.ld * m.rows);
    return make_map(map, dtype, m.p, m.cols, m.rows, m.matrices, m.ld, se, box_cols, box_rows, three ? 3 : 2);
}

// ------------------------------------- gradient of the activation and the bias
// dz = dy * act'(z) in one pass over dy and z, with the column sums of dz (the bias
// gradient) taken on the way.  A CTA owns ACT_COLS columns of a block of rows; a warp
// takes every eighth row, a lane 8 columns (16 bytes; 8 single columns 32 apart where
// rows are not 16-byte aligned).  Row blocks cut across experts: the sums of block b
// for expert e are partial[b + e], a number no other pair on the path from (0, 0) to
// (last block, last expert) has, so nothing depends on where the experts end and no
// atomics are needed; sum_kernel adds an expert's partials in the order of its blocks.
constexpr int ACT_COLS = 256, ACT_WARPS = 8, ACT_ROWS = 2;  // rows a lane has in flight

// Two rows in flight at four CTAs an SM (64 registers): 16384 x 8192 GELU with its sums takes
// some 185 us, 1.07 GB with z in fp32 (5.8 TB/s).  Chosen with z in 16 bits, where it took 155,
// against 179 for four rows at two CTAs and 208 for two rows at five (spills).
template <typename T, int ACT, bool VEC>
__global__ void __launch_bounds__(ACT_WARPS * 32, 4) grad_act_kernel(const T* dy, const typename Kept<T, ACT>::Type* z, const int32_t* offsets, int R,
                                                                  int E, int N, int block_rows, T* dz, float* partial) {
    next_may_start();
    previous_done();
    typedef typename Kept<T, ACT>::Type Z;
    struct alignas(16) Eight { Z v[8]; };
    __shared__ float part[ACT_WARPS][ACT_COLS];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int strips = (N + ACT_COLS - 1) / ACT_COLS, strip = blockIdx.x % strips, block = blockIdx.x / strips;
    const int n0 = strip * ACT_COLS + (VEC ? lane * 8 : lane);
    constexpr int STEP = VEC ? 1 : 32;
    const int row0 = block * block_rows, row1 = (int)min((int64_t)row0 + block_rows, (int64_t)R);
    // the last expert that starts at or before row0
    int lo = 0, hi = E;
    while (offsets && hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (clampi(offsets[mid], 0, R) <= row0) lo = mid; else hi = mid;
    }
    for (int e = lo; e < E; ++e) {
        int r0, r1;
        expert_rows(offsets, e, R, r0, r1);
        if (r0 >= row1) break;
        r0 = max(r0, row0);
        r1 = min(r1, row1);
        if (r0 >= r1) continue;
        float sum[8] = {};
        if (VEC && n0 < N) {
            const T* gp = dy + (int64_t)(r0 + w) * N + n0;
            const Z* zp = z + (int64_t)(r0 + w) * N + n0;
            T* dp = dz + (int64_t)(r0 + w) * N + n0;
            const int64_t step = (int64_t)ACT_WARPS * N;
            auto row = [&](Pack<T>& g, const Eight& q, T* to) {
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    float v = El<T>::to(g.v[c]);
                    if (ACT != ELA_ACT_NONE) v *= act_slope<ACT>(El<Z>::to(q.v[c]));
                    sum[c] += v;
                    g.v[c] = El<T>::from(v);
                }
                if (dz) *reinterpret_cast<Pack<T>*>(to) = g;
            };
            int r = r0 + w;
            for (; r + (ACT_ROWS - 1) * ACT_WARPS < r1; r += ACT_WARPS * ACT_ROWS) {
                Pack<T> g[ACT_ROWS];
                Eight q[ACT_ROWS];
#pragma unroll
                for (int i = 0; i < ACT_ROWS; ++i) {
                    g[i] = *reinterpret_cast<const Pack<T>*>(gp + i * step);
                    if (ACT != ELA_ACT_NONE) q[i] = *reinterpret_cast<const Eight*>(zp + i * step);
                }
#pragma unroll
                for (int i = 0; i < ACT_ROWS; ++i) row(g[i], q[i], dp + i * step);
                gp += ACT_ROWS * step;
                zp += ACT_ROWS * step;
                dp += ACT_ROWS * step;
            }
            for (; r < r1; r += ACT_WARPS) {
                Pack<T> g = *reinterpret_cast<const Pack<T>*>(gp);
                Eight q;
                if (ACT != ELA_ACT_NONE) q = *reinterpret_cast<const Eight*>(zp);
                row(g, q, dp);
                gp += step;
                zp += step;
                dp += step;
            }
        } else if (!VEC) {
            for (int r = r0 + w; r < r1; r += 2 * ACT_WARPS) {  // two rows' loads before their stores: 4096 x 2051 33 -> 22 us, 300 x 1500 33 -> 15
                T g[2][8] = {};
                Z q[2][8] = {};
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        if (r + i * ACT_WARPS < r1 && n0 + c * 32 < N) {
                            const int64_t at = (int64_t)(r + i * ACT_WARPS) * N + n0 + c * 32;
                            g[i][c] = dy[at];
                            if (ACT != ELA_ACT_NONE) q[i][c] = z[at];
                        }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        if (r + i * ACT_WARPS < r1 && n0 + c * 32 < N) {
                            float v = El<T>::to(g[i][c]);
                            if (ACT != ELA_ACT_NONE) v *= act_slope<ACT>(El<Z>::to(q[i][c]));
                            sum[c] += v;
                            if (dz) dz[(int64_t)(r + i * ACT_WARPS) * N + n0 + c * 32] = El<T>::from(v);
                        }
            }
        }
        if (!partial) continue;
#pragma unroll
        for (int c = 0; c < 8; ++c) part[w][(VEC ? lane * 8 : lane) + c * STEP] = sum[c];
        __syncthreads();
        const int n = strip * ACT_COLS + threadIdx.x;
        float total = 0.f;
#pragma unroll
        for (int i = 0; i < ACT_WARPS; ++i) total += part[i][threadIdx.x];
        if (n < N) partial[(int64_t)(block + e) * N + n] = total;
        __syncthreads();
    }
}

// dbias[e][n]: 8 warps share the expert's row blocks, joined in a fixed order.
template <typename T>
__global__ void __launch_bounds__(256) sum_kernel(const float* partial, const int32_t* offsets, int R, int N, int block_rows,
                                                  T* dbias) {
    next_may_start();
    previous_done();
    __shared__ float part[8][32];
    const int strips = (N + 31) / 32, e = blockIdx.x / strips;
    const int c = threadIdx.x & 31, w = threadIdx.x >> 5, n = blockIdx.x % strips * 32 + c;
    int r0, r1;
    expert_rows(offsets, e, R, r0, r1);
    float sum = 0.f;
    if (r0 < r1 && n < N) {
        const int last = (r1 - 1) / block_rows;
#pragma unroll 4
        for (int b = r0 / block_rows + w; b <= last; b += 8) sum += partial[(int64_t)(b + e) * N + n];
    }
    part[w][c] = sum;
    __syncthreads();
    if (w == 0 && n < N) {
        for (int i = 1; i < 8; ++i) sum += part[i][c];
        dbias[(int64_t)e * N + n] = El<T>::from(sum);
    }
}

// Rows per block: 128, down to 32 while the grid is under eight blocks an SM, and on to a row a warp while it is
// under four: 300 rows of 1500 take 8 us with 8 rows a block, 15 with 32; 4096 x 2048 takes 15 us with 32 rows a
// block, 17 with 16.
inline int act_block_rows(int64_t R, int64_t N) {
    const int64_t strips = (N + ACT_COLS - 1) / ACT_COLS;
    int rows = 128;
    while (rows > ACT_WARPS && (R + rows - 1) / rows * strips < (rows > 32 ? 1184 : 592)) rows /= 2;
    return rows;
}

inline bool linear_sizes_ok(int dtype, int64_t R, int64_t E, int64_t K, int64_t N, const int32_t* offsets) {
    return (dtype == ELA_DTYPE_F16 || dtype == ELA_DTYPE_BF16) && R >= 0 && R <= (1ll << 30) && E >= 1 &&
           E <= ELA_EXPERT_MAX && K >= 1 && K <= (1ll << 30) && N >= 1 && N <= (1ll << 30) && (offsets || E == 1);
}
inline bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

// Parameters of a pass whose columns are the experts' rows: F features out, contraction length K.
inline MmaParams row_pass(const int32_t* offsets, int64_t R, int64_t E, int64_t F, int64_t K) {
    MmaParams p = {};
    p.offsets = offsets;
    p.R = (int)R; p.E = (int)E; p.F = (int)F; p.K = (int)K;
    p.f_tiles = (int)((F + MMA_PAIR_F - 1) / MMA_PAIR_F);
    p.bn = columns_per_tile(R, E, p.f_tiles, (K + MMA_KB - 1) / MMA_KB);
    // a CTA's half of a tile's columns is one box, or boxes of 64 where experts have fewer rows
    // than that makes (a box is loaded whole)
    p.bbox = p.bn % 128 == 0 && R < 256 * E ? 64 : p.bn / 2;
    p.stages = stages_for(p.bn, E);
    p.wait_ns = wait_limit(K);
    return p;
}
// At least as many tiles as the offsets can make.
inline int64_t row_tiles(const MmaParams& p) {
    const int64_t by_rows = p.R / p.bn + (p.E < p.R ? p.E : p.R);
    return (by_rows > 0 ? by_rows : 1) * p.f_tiles;
}

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

size_t ela_expert_linear_workspace_bytes(int pass, int64_t R, int64_t E, int64_t K, int64_t N, int aligned) {
    if (pass == ELA_LINEAR_GRAD_ACT) {
        const int rows = act_block_rows(R, N);
        return (size_t)((R + rows - 1) / rows + E) * N * 4;
    }
    if (aligned || (pass == ELA_LINEAR_FORWARD && few_rows(R, E, N))) return 0;
    const Matrix x = {nullptr, 1, R, K, 0, 0}, w = {nullptr, E, N, K, 0, 0}, dz = {nullptr, 1, R, N, 0, 0};
    return pass == ELA_LINEAR_FORWARD ? x.padded_bytes() + w.padded_bytes()
         : pass == ELA_LINEAR_GRAD_INPUT ? dz.padded_bytes() + w.padded_bytes()
                                         : dz.padded_bytes() + x.padded_bytes();
}

int ela_expert_status(int* status) {
    if (!status) return ELA_ERR_ARGUMENT;
    const int zero = ELA_OK;
    if (cudaDeviceSynchronize() != cudaSuccess) return ELA_ERR_CUDA;
    if (cudaMemcpyFromSymbol(status, g_expert_error, sizeof(int)) != cudaSuccess) return ELA_ERR_CUDA;
    if (*status != ELA_OK && cudaMemcpyToSymbol(g_expert_error, &zero, sizeof(int)) != cudaSuccess) return ELA_ERR_CUDA;
    return ELA_OK;
}

int ela_expert_linear(const void* x, const void* weight, const void* bias, const void* residual,
                      const int32_t* offsets, int dtype, int64_t R, int64_t E, int64_t K, int64_t N, int64_t ldx,
                      int64_t stride_e, int64_t ldw, int64_t ldr, int activation, void* y, void* z, void* workspace,
                      size_t workspace_bytes, void* stream) {
    if (!linear_sizes_ok(dtype, R, E, K, N, offsets) || activation < 0 || activation > ELA_ACT_SILU || ldx < 0 ||
        stride_e < 0 || ldw < 0 || ldr < 0)
        return ELA_ERR_ARGUMENT;
    if (R == 0) return ELA_OK;
    if (!x || !weight || !y) return ELA_ERR_ARGUMENT;
    const bool wide_z = activation == ELA_ACT_GELU || activation == ELA_ACT_SILU;
    if (!on_elements(2, x, weight, bias, residual, y) || !on_elements(wide_z ? 4 : 2, z) || !on_elements(4, offsets))
        return ELA_ERR_ARGUMENT;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (few_rows(R, E, N)) {
        if (E * ((N + 15) / 16) > INT32_MAX) return ELA_ERR_UNSUPPORTED;
        StreamParams q = {x, weight, bias, residual, offsets, (int)R, (int)E, (int)K, (int)N, 0, ldx, stride_e, ldw, ldr, y, z};
        const uint64_t bits = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(weight) | (uint64_t)(ldx * 2) | (uint64_t)(ldw * 2) |
                              (uint64_t)(E > 1 ? stride_e * 2 : 0) | (uint64_t)(K * 2);
        const int vb = bits % 32 == 0 ? 32 : bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 2;
        int rc = ELA_OK;
        ELA_BY_TYPE(dtype, { ELA_BY_ACT(activation, rc = R <= 4 * E || (E == 1 && R <= 8) ? (stream_launch<T_, A_, 1>(q, vb, st)) : R <= 16 * E ? (stream_launch<T_, A_, 2>(q, vb, st)) : (stream_launch<T_, A_, 4>(q, vb, st))) })
        if (rc == ELA_OK && z && activation == ELA_ACT_RELU) ELA_BY_TYPE(dtype, { rc = settle_launch<T_>(q, st); })
        return rc;
    }
    char* ws = reinterpret_cast<char*>(workspace);
    Matrix mx = {x, 1, R, K, ldx, 0}, mw = {weight, E, N, K, ldw, stride_e};
    int rc = readable(mx, ws, workspace_bytes, st);
    if (rc == ELA_OK) rc = readable(mw, ws, workspace_bytes, st);
    if (rc != ELA_OK) return rc;
    MmaParams p = row_pass(offsets, R, E, N, K);
    p.bias = bias;
    p.x = mx.p;
    p.ldx = mx.ld;
    p.weight = mw.p;
    p.ldw = mw.ld;
    p.stride_e = mw.stride_e;
    p.residual = residual;
    p.ldr = ldr;
    p.out = y;
    p.z = z;
    p.vec = N % 2 == 0 && aligned4(y) && (!z || (reinterpret_cast<uintptr_t>(z) & 7) == 0) && (!residual || (aligned4(residual) && ldr % 2 == 0));
    CUtensorMap a, b;
    if (!map_of(&a, dtype, mw, MMA_KB, MMA_F, true) || !map_of(&b, dtype, mx, MMA_KB, p.bbox, false)) return ELA_ERR_CUDA;
    ELA_BY_TYPE(dtype, { ELA_BY_ACT(activation, rc = z ? (mma_launch<PASS_FORWARD, T_, A_, true>(a, b, p, row_tiles(p), st)) : (mma_launch<PASS_FORWARD, T_, A_>(a, b, p, row_tiles(p), st))) })
    return rc;
}

int ela_expert_linear_grad_act(const void* dy, const void* z, const int32_t* offsets, int dtype, int64_t R,
                               int64_t E, int64_t N, int activation, void* dz, void* dbias, void* workspace,
                               size_t workspace_bytes, void* stream) {
    if (!linear_sizes_ok(dtype, R, E, 1, N, offsets) || activation < 0 || activation > ELA_ACT_SILU)
        return ELA_ERR_ARGUMENT;
    if ((R == 0 && !dbias) || (!dz && !dbias)) return ELA_OK;
    if (R > 0 && (!dy || (!z && activation != ELA_ACT_NONE))) return ELA_ERR_ARGUMENT;
    const int rows = act_block_rows(R, N);
    const int64_t blocks = (R + rows - 1) / rows;
    if (!on_elements(2, dy, dz, dbias) || !on_elements(activation == ELA_ACT_GELU || activation == ELA_ACT_SILU ? 4 : 2, z) ||
        !on_elements(4, offsets) || (dbias && !on_elements(4, workspace)))
        return ELA_ERR_ARGUMENT;
    if (dbias && (!workspace || workspace_bytes < (size_t)(blocks + E) * N * 4)) return ELA_ERR_ARGUMENT;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    float* partial = dbias ? reinterpret_cast<float*>(workspace) : nullptr;
    const bool vec = aligned16(dy, N * 2) && (!z || aligned16(z)) && (!dz || aligned16(dz));
    int rc = ELA_OK;
    ELA_BY_TYPE(dtype, {
        const unsigned grid = (unsigned)(blocks * ((N + ACT_COLS - 1) / ACT_COLS));  // strips of columns innermost
        if (R > 0)
            ELA_BY_ACT(activation, {
                auto kern = vec ? grad_act_kernel<T_, A_, true> : grad_act_kernel<T_, A_, false>;
                rc = launch(kern, grid, ACT_WARPS * 32, 0, st, (const T_*)dy, (const typename Kept<T_, A_>::Type*)z, offsets, (int)R, (int)E, (int)N, rows, (T_*)dz, partial);
            })
        if (dbias && rc == ELA_OK)
            rc = launch(sum_kernel<T_>, (unsigned)(E * ((N + 31) / 32)), 256, 0, st, (const float*)partial, offsets, (int)R, (int)N, rows, (T_*)dbias);
    })
    return rc;
}

int ela_expert_linear_grad_input(const void* dz, const void* weight, const int32_t* offsets, int dtype, int64_t R,
                                 int64_t E, int64_t K, int64_t N, int64_t stride_e, int64_t ldw, void* dx,
                                 void* workspace, size_t workspace_bytes, void* stream) {
    if (!linear_sizes_ok(dtype, R, E, K, N, offsets) || stride_e < 0 || ldw < 0) return ELA_ERR_ARGUMENT;
    if (R == 0) return ELA_OK;
    if (!dz || !weight || !dx || !on_elements(2, dz, weight, dx) || !on_elements(4, offsets)) return ELA_ERR_ARGUMENT;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    char* ws = reinterpret_cast<char*>(workspace);
    Matrix mz = {dz, 1, R, N, N, 0}, mw = {weight, E, N, K, ldw, stride_e};
    int rc = readable(mz, ws, workspace_bytes, st);
    if (rc == ELA_OK) rc = readable(mw, ws, workspace_bytes, st);
    if (rc != ELA_OK) return rc;
    MmaParams p = row_pass(offsets, R, E, K, N);
    p.out = dx;
    p.vec = K % 2 == 0 && aligned4(dx);
    CUtensorMap a, b;
    if (!map_of(&a, dtype, mw, 64, MMA_KB, true) || !map_of(&b, dtype, mz, MMA_KB, p.bbox, false)) return ELA_ERR_CUDA;
    ELA_BY_TYPE(dtype, { rc = (mma_launch<PASS_INPUT, T_, ELA_ACT_NONE>(a, b, p, row_tiles(p), st)); })
    return rc;
}

int ela_expert_linear_grad_weight(const void* dz, const void* x, const int32_t* offsets, int dtype, int64_t R,
                                  int64_t E, int64_t K, int64_t N, int64_t ldx, void* dweight, void* workspace,
                                  size_t workspace_bytes, void* stream) {
    if (!linear_sizes_ok(dtype, R, E, K, N, offsets) || ldx < 0) return ELA_ERR_ARGUMENT;
    if (!dweight || (R > 0 && (!dz || !x)) || !on_elements(2, dz, x, dweight) || !on_elements(4, offsets)) return ELA_ERR_ARGUMENT;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (R == 0) return cudaMemsetAsync(dweight, 0, (size_t)(E * N * K) * 2, st) == cudaSuccess ? ELA_OK : ELA_ERR_CUDA;
    char* ws = reinterpret_cast<char*>(workspace);
    Matrix mz = {dz, 1, R, N, N, 0}, mx = {x, 1, R, K, ldx, 0};
    int rc = readable(mz, ws, workspace_bytes, st);
    if (rc == ELA_OK) rc = readable(mx, ws, workspace_bytes, st);
    if (rc != ELA_OK) return rc;
    MmaParams p = {};
    p.offsets = offsets;
    p.R = (int)R; p.E = (int)E; p.F = (int)K; p.C = (int)N;
    p.bn = MMA_C;
    p.stages = stages_for(p.bn, E);
    p.f_tiles = (int)((K + MMA_PAIR_F - 1) / MMA_PAIR_F);
    p.c_tiles = (int)((N + MMA_C - 1) / MMA_C);
    p.out = dweight;
    p.vec = K % 2 == 0 && aligned4(dweight);
    p.wait_ns = wait_limit(R);
    CUtensorMap a, b;
    if (!map_of(&a, dtype, mx, 64, MMA_KB, false) || !map_of(&b, dtype, mz, 64, MMA_KB, false)) return ELA_ERR_CUDA;
    ELA_BY_TYPE(dtype, { rc = (mma_launch<PASS_WEIGHT, T_, ELA_ACT_NONE>(a, b, p, E * p.f_tiles * p.c_tiles, st)); })
    return rc;
}

}  // extern "C"
