// ela_expert.cu -- tokens sorted by expert and back (include/ela_expert.h): the
// plan (a stable counting sort), the dispatch of token rows into expert order
// and the weighted combine with its gradient.

#include "ela_expert.cuh"

namespace ela_expert {

// ------------------------------------------------------------------- plan
// A stable counting sort by one cluster of CTAs.  Every warp of the cluster owns a
// contiguous range of slots and walks it 32 at a time: the lanes of one bucket (found by
// a ballot for each bit of it; __match_any_sync took 80 cycles of an SM a time, five
// times as long) rank themselves in lane order behind the warp's counter of that bucket, so a slot's rank inside its warp's range is known when the ranges have been
// read once.  The first row of bucket b for a warp is then the slots of lower buckets
// anywhere, plus those of b in CTAs before this one (read from their shared memory),
// plus those of b in warps before this one.  Ranges up to 32 * PLAN_ITEMS slots stay in
// registers; longer ones park the rank in `position`.
constexpr int PLAN_THREADS = 1024, PLAN_ITEMS = 8, PLAN_CLUSTER = 16;

__device__ __forceinline__ int peer_read(const int* p, int rank) {
    uint32_t a;
    int v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void plan_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Rank of this lane's slot among the warp's slots of bucket b so far (all lanes call; b < 0:
// no slot).  bits: of the largest bucket plus one, so that -1 is no bucket in them.
__device__ __forceinline__ int plan_rank(int* mine, int b, int bits, int lane) {
    unsigned same = ~0u;
    for (int i = 0; i < bits; ++i) {
        const bool one = (b >> i) & 1;
        const unsigned with = __ballot_sync(~0u, one);
        same &= one ? with : ~with;
    }
    const int ahead = __popc(same & ((1u << lane) - 1));
    const int rank = b >= 0 ? mine[b] + ahead : 0;
    __syncwarp();
    if (b >= 0 && ahead == 0) mine[b] = rank + __popc(same);
    __syncwarp();
    return rank;
}

template <typename Id>
__global__ void __launch_bounds__(PLAN_THREADS, 1) plan_kernel(const Id* expert, int slots, int E, int nwarps, int per,
                                                               int32_t* offsets, int32_t* position, int32_t* source) {
    next_may_start();
    previous_done();
    extern __shared__ int shared[];  // [nwarps][E + 1] counts, [E + 1] totals of the CTA
    __shared__ int warp_sum[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = E + 1;
    const int rank = blockIdx.x, ctas = gridDim.x, bits = 32 - __clz(E + 1);
    int* total = shared + nwarps * B;
    for (int i = tid; i < nwarps * B; i += blockDim.x) shared[i] = 0;
    __syncthreads();
    const int64_t first = ((int64_t)rank * nwarps + warp) * per;
    // (unsigned: a step past the end of 2^31 - 1 slots must not come out negative)
    const unsigned s0 = warp < nwarps && first < slots ? (unsigned)first : slots;
    const unsigned s1 = (int64_t)s0 + per < slots ? s0 + per : slots;
    int* mine = shared + (warp < nwarps ? warp : 0) * B;
    const bool kept = per <= 32 * PLAN_ITEMS;
    int bucket[PLAN_ITEMS], local[PLAN_ITEMS];
    for (unsigned s = s0; s < s1; s += 32 * PLAN_ITEMS) {
#pragma unroll
        for (int i = 0; i < PLAN_ITEMS; ++i) {
            const unsigned at = s + 32 * i + lane;
            bucket[i] = -1;
            if (at < s1) {
                const Id e = expert[at];
                bucket[i] = e >= 0 && e < (Id)E ? (int)e : E;
            }
        }
#pragma unroll
        for (int i = 0; i < PLAN_ITEMS; ++i) {
            if (s + 32 * i >= s1) break;
            local[i] = plan_rank(mine, bucket[i], bits, lane);
            if (!kept && bucket[i] >= 0) position[s + 32 * i + lane] = local[i];
        }
    }
    __syncthreads();
    for (int b = tid; b < B; b += blockDim.x) {
        int sum = 0;
#pragma unroll 8
        for (int w = 0; w < nwarps; ++w) sum += shared[w * B + b];
        total[b] = sum;
    }
    if (ctas > 1) plan_cluster_sync(); else __syncthreads();
    // buckets in runs, one run a thread: slots of lower buckets, and of this one in earlier CTAs
    const int run = (B + blockDim.x - 1) / blockDim.x;
    const int b0 = min(tid * run, B), b1 = min(b0 + run, B);
    auto totals = [&](int b, int* c) {  // every CTA's, all reads in flight at once
#pragma unroll
        for (int r = 0; r < PLAN_CLUSTER; ++r) c[r] = r >= ctas ? 0 : r == rank ? total[b] : peer_read(total + b, r);
    };
    int sum = 0, c[PLAN_CLUSTER];
    for (int b = b0; b < b1; ++b) {
        totals(b, c);
#pragma unroll
        for (int r = 0; r < PLAN_CLUSTER; ++r) sum += c[r];
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(~0u, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    int base = incl - sum;
    for (int w = 0; w < warp; ++w) base += warp_sum[w];
    for (int b = b0; b < b1; ++b) {
        if (rank == 0) offsets[b] = base;
        if (run > 1) totals(b, c);
        int at = base;
#pragma unroll
        for (int r = 0; r < PLAN_CLUSTER; ++r) {
            if (r < rank) at += c[r];
            base += c[r];
        }
#pragma unroll 8
        for (int w = 0; w < nwarps; ++w) {
            const int n = shared[w * B + b];
            shared[w * B + b] = at;
            at += n;
        }
    }
    if (ctas > 1) plan_cluster_sync(); else __syncthreads();  // (peers have read this CTA's totals)
    if (kept) {
#pragma unroll
        for (int i = 0; i < PLAN_ITEMS; ++i) {
            const unsigned at = s0 + 32 * i + lane;
            if (at < s1) {
                const int row = mine[bucket[i]] + local[i];
                position[at] = row;
                source[row] = at;
            }
        }
    } else {
        for (unsigned s = s0; s < s1; s += 32 * PLAN_ITEMS) {
#pragma unroll
            for (int i = 0; i < PLAN_ITEMS; ++i) {
                const unsigned at = s + 32 * i + lane;
                if (at < s1) {
                    const Id e = expert[at];
                    local[i] = mine[e >= 0 && e < (Id)E ? (int)e : E] + position[at];
                }
            }
#pragma unroll
            for (int i = 0; i < PLAN_ITEMS; ++i) {
                const unsigned at = s + 32 * i + lane;
                if (at < s1) {
                    position[at] = local[i];
                    source[local[i]] = at;
                }
            }
        }
    }
}

template <typename Id>
int plan_launch(const Id* expert, int slots, int E, int32_t* offsets, int32_t* position, int32_t* source, cudaStream_t st) {
    const int fit = 200 * 1024 / (4 * (E + 1)) - 1, most = fit < 32 ? fit : 32;
    // a CTA for every 1024 slots (a step of its warps), up to 16: the scattered stores of a CTA
    // take as long as everything else, 32768 slots on 8 CTAs 9.5 us, a single CTA 52
    int ctas = 1;
    while (ctas < PLAN_CLUSTER && slots > ctas * most * 32) ctas *= 2;
    int nwarps = most;
    while (ctas == 1 && nwarps > 1 && (nwarps / 2) * 64 >= slots) nwarps /= 2;
    const int64_t all = (int64_t)ctas * nwarps;
    const int per = (int)((((int64_t)slots + all - 1) / all + 31) / 32 * 32);
    const size_t smem = (size_t)(nwarps + 1) * (E + 1) * 4;
    auto kern = plan_kernel<Id>;
    if (!allow_smem<&plan_kernel<Id>>(208 * 1024)) return ELA_ERR_CUDA;  // (48 KB without, the static part included)
    // the scan takes a thread per bucket; few slots need few warps
    int threads = nwarps * 32;
    while (threads < PLAN_THREADS && threads < E + 1) threads *= 2;
    if (threads > PLAN_THREADS) threads = PLAN_THREADS;
    if (ctas == 1) {
        return launch(kern, 1, threads, smem, st, expert, slots, E, nwarps, per, offsets, position, source);
    }
    if (ctas > 8 && !allow_wide_cluster<&plan_kernel<Id>>()) return ELA_ERR_CUDA;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    if (cudaLaunchKernelEx(&cfg, kern, expert, slots, E, nwarps, per, offsets, position, source) == cudaSuccess) return ELA_OK;
    cudaGetLastError();
    return ELA_ERR_CUDA;
}

// --------------------------------------------------------- dispatch, combine
// One pass over the rows: each is read once and written once, by the group of G threads
// (32 to 256, by the row's length) that owns the token, in pieces of VB bytes (the widest
// that every row's address allows), U pieces of a row and JC choices in flight per thread.
// Pieces stay packed in 32-bit words until they are used: kept as 16-bit elements they take
// a register each, and the rows in flight that hide the latency come from resident warps.
// 8192 tokens x 2 choices of 2048 bf16 rows (us; 32 bytes of a row in flight a thread, four
// CTAs an SM for combine, six for its gradient): 16.5, 20.6 and 32.9, that is 6.1, 4.9 and
// 5.1 TB/s with the launch; 16 bytes in flight 17.3, 22.7 and 41.1.
constexpr int ROUTE_THREADS = 256, JC = 2;

template <int VB> struct Piece;
template <> struct alignas(16) Piece<16> { uint32_t w[4]; };
template <> struct alignas(8) Piece<8> { uint32_t w[2]; };
template <> struct Piece<4> { uint32_t w[1]; };
template <> struct Piece<2> { uint16_t w[1]; };
template <int VB> struct Route { static constexpr int U = VB >= 4 ? 32 / VB : 4; };

template <int VB, typename T> __device__ __forceinline__ Piece<VB> load_piece(const T* p) { return *reinterpret_cast<const Piece<VB>*>(p); }
template <int VB, typename T> __device__ __forceinline__ void store_piece(T* p, const Piece<VB>& v) { *reinterpret_cast<Piece<VB>*>(p) = v; }

// A piece's elements in fp32, and a piece rounded from them.
template <typename T> struct Bits16;
template <> struct Bits16<__half> {
    static __device__ __forceinline__ float to(uint16_t b) { __half_raw h; h.x = b; return __half2float(__half(h)); }
    static __device__ __forceinline__ uint16_t from(float f) { return __half_raw(__float2half_rn(f)).x; }
    static __device__ __forceinline__ uint32_t pair(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
template <> struct Bits16<__nv_bfloat16> {
    static __device__ __forceinline__ float to(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }
    static __device__ __forceinline__ uint16_t from(float f) { return __nv_bfloat16_raw(__float2bfloat16_rn(f)).x; }
    static __device__ __forceinline__ uint32_t pair(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
template <typename T, int VB> struct Values {  // 16-bit elements
    static constexpr int N = VB / 2;
    static __device__ __forceinline__ void unpack(const Piece<VB>& p, float* f) {
        if constexpr (VB == 2) {
            f[0] = Bits16<T>::to(p.w[0]);
        } else {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                f[2 * i] = Bits16<T>::to((uint16_t)(p.w[i] & 0xffffu));
                f[2 * i + 1] = Bits16<T>::to((uint16_t)(p.w[i] >> 16));
            }
        }
    }
    static __device__ __forceinline__ Piece<VB> pack(const float* f) {
        Piece<VB> p;
        if constexpr (VB == 2) {
            p.w[0] = Bits16<T>::from(f[0]);
        } else {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) p.w[i] = Bits16<T>::pair(f[2 * i], f[2 * i + 1]);
        }
        return p;
    }
};
template <int VB> struct Values<float, VB> {
    static constexpr int N = VB / 4;
    static __device__ __forceinline__ void unpack(const Piece<VB>& p, float* f) {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = __uint_as_float(p.w[i]);
    }
    static __device__ __forceinline__ Piece<VB> pack(const float* f) {
        Piece<VB> p;
#pragma unroll
        for (int i = 0; i < N; ++i) p.w[i] = __float_as_uint(f[i]);
        return p;
    }
};

template <typename T, int VB>
__global__ void __launch_bounds__(ROUTE_THREADS) dispatch_kernel(const T* x, int T_, int k, int H, int64_t ldx, int G,
                                                                 const int32_t* position, const int32_t* offsets, int E,
                                                                 int rows, T* out) {
    next_may_start();
    previous_done();
    constexpr int N = VB / sizeof(T), U = Route<VB>::U;
    const int64_t t = (int64_t)blockIdx.x * (ROUTE_THREADS / G) + threadIdx.x / G;
    if (t >= T_) return;
    const int valid = offsets[E];
    const int32_t* pos = position + t * k;
    const T* from = x + t * ldx;
    for (int i = threadIdx.x % G * N; i < H; i += G * N * U) {
        Piece<VB> v[U];
        int at[2];  // positions (read before the stores, which might be to them for all the compiler knows)
        auto next = [&](int j0) {
#pragma unroll
            for (int j = 0; j < 2; ++j) at[j] = j0 + j < k ? pos[j0 + j] : -1;
        };
        next(0);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * G * N < H) v[u] = load_piece<VB>(from + i + u * G * N);
        for (int j0 = 0; j0 < k; j0 += 2) {
            if (j0) next(j0);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int p = at[j];
                if (p < 0 || p >= rows) continue;
                T* to = out + (int64_t)p * H + i;
                const Piece<VB> zero = {};
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (i + u * G * N < H) store_piece<VB>(to + u * G * N, p < valid ? v[u] : zero);
            }
        }
    }
}

template <typename T, typename Wt, int VB>
__global__ void __launch_bounds__(ROUTE_THREADS, 4) combine_kernel(const T* y, int T_, int k, int H, int64_t ldy,
                                                                            int G, const int32_t* position,
                                                                            const int32_t* offsets, int E, int rows,
                                                                            const Wt* weights, T* out) {
    next_may_start();
    previous_done();
    constexpr int N = VB / sizeof(T), U = Route<VB>::U;
    const int64_t t = (int64_t)blockIdx.x * (ROUTE_THREADS / G) + threadIdx.x / G;
    if (t >= T_) return;
    const int valid = min(offsets[E], rows);
    for (int i = threadIdx.x % G * N; i < H; i += G * N * U) {
        float acc[U][N] = {};
        for (int j0 = 0; j0 < k; j0 += JC) {
            Piece<VB> v[JC][U];
            float w[JC];
            bool has[JC];
#pragma unroll
            for (int j = 0; j < JC; ++j) {
                const int p = j0 + j < k ? position[t * k + j0 + j] : -1;
                has[j] = p >= 0 && p < valid;
                w[j] = has[j] && weights ? El<Wt>::to(weights[t * k + j0 + j]) : 1.f;
                if (has[j])
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (i + u * G * N < H) v[j][u] = load_piece<VB>(y + (int64_t)p * ldy + i + u * G * N);
            }
#pragma unroll
            for (int j = 0; j < JC; ++j)
                if (has[j])
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        float f[N];
                        Values<T, VB>::unpack(v[j][u], f);
#pragma unroll
                        for (int c = 0; c < N; ++c) acc[u][c] = fmaf(w[j], f[c], acc[u][c]);
                    }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * G * N < H) store_piece<VB>(out + t * H + i + u * G * N, Values<T, VB>::pack(acc[u]));
    }
}

// dy and dweights together: dout's piece is read once for JC choices, the JC dot products
// are joined at the end of the row, lanes first, then the group's warps in their order.
template <typename T, typename Wt, int VB>
__global__ void __launch_bounds__(ROUTE_THREADS, 6)
    combine_grad_kernel(const T* dout, const T* y, int T_, int k, int H, int64_t lddo, int64_t ldy, int G,
                        const int32_t* position, const int32_t* offsets, int E, int rows, const Wt* weights, T* dy,
                        Wt* dweights) {
    next_may_start();
    previous_done();
    constexpr int N = VB / sizeof(T);
    __shared__ float part[ROUTE_THREADS / 32][JC];
    const int64_t t = (int64_t)blockIdx.x * (ROUTE_THREADS / G) + threadIdx.x / G;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool in = t < T_;  // (no early return: the warps of a CTA share barriers)
    const int valid = min(offsets[E], rows);
    for (int j0 = 0; j0 < k; j0 += JC) {
        int p[JC];
        float w[JC], dot[JC] = {};
#pragma unroll
        for (int j = 0; j < JC; ++j) {
            p[j] = in && j0 + j < k ? position[t * k + j0 + j] : -1;
            if (p[j] >= rows) p[j] = -1;
            w[j] = p[j] < 0 || p[j] >= valid ? 0.f : weights ? El<Wt>::to(weights[t * k + j0 + j]) : 1.f;
        }
        for (int i = threadIdx.x % G * N; in && i < H; i += G * N) {
            const Piece<VB> dp = load_piece<VB>(dout + t * lddo + i);
            Piece<VB> v[JC];
            if (dweights)
#pragma unroll
                for (int j = 0; j < JC; ++j)
                    if (p[j] >= 0 && p[j] < valid) v[j] = load_piece<VB>(y + (int64_t)p[j] * ldy + i);
            float d[N];
            Values<T, VB>::unpack(dp, d);
#pragma unroll
            for (int j = 0; j < JC; ++j) {
                if (p[j] < 0) continue;
                const bool has = p[j] < valid;
                if (dy) {
                    float o[N];
#pragma unroll
                    for (int c = 0; c < N; ++c) o[c] = has ? w[j] * d[c] : 0.f;
                    store_piece<VB>(dy + (int64_t)p[j] * H + i, Values<T, VB>::pack(o));
                }
                if (dweights && has) {
                    float f[N];
                    Values<T, VB>::unpack(v[j], f);
#pragma unroll
                    for (int c = 0; c < N; ++c) dot[j] = fmaf(d[c], f[c], dot[j]);
                }
            }
        }
        if (dweights) {
#pragma unroll
            for (int j = 0; j < JC; ++j)
#pragma unroll
                for (int o = 16; o; o >>= 1) dot[j] += __shfl_xor_sync(~0u, dot[j], o);
            if (G > 32) {
                if (lane == 0)
#pragma unroll
                    for (int j = 0; j < JC; ++j) part[warp][j] = dot[j];
                __syncthreads();
            }
            const int j = threadIdx.x % G;
            if (in && j < JC && j0 + j < k) {
                float sum = 0.f;
                if (G > 32) {
                    for (int q = 0; q < G / 32; ++q) sum += part[warp + q][j];
                } else {
#pragma unroll
                    for (int q = 0; q < JC; ++q) if (q == j) sum = dot[q];
                }
                dweights[t * k + j0 + j] = El<Wt>::from(sum);
            }
            if (G > 32) __syncthreads();
        }
    }
}

// Bytes per piece: the widest power of two up to 16 that divides every address and row.
inline int piece_bytes(uint64_t bits) { return bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 2; }
// Threads per token: 32 to 256, of two to four pieces each where a row has as many.
inline int group_threads(int64_t H, int es, int vb) {
    const int64_t pieces = H * es / vb;
    int g = 32;
    while (g < ROUTE_THREADS && g * 4 <= pieces) g *= 2;
    return g;
}
inline unsigned route_grid(int64_t T, int G) { return (unsigned)((T * G + ROUTE_THREADS - 1) / ROUTE_THREADS); }
inline uint64_t address(const void* p) { return reinterpret_cast<uintptr_t>(p); }

inline bool sizes_ok(int dtype, int64_t T, int64_t k, int64_t H, int64_t E) {
    return dtype_bytes(dtype) != 0 && T >= 0 && k >= 0 && H >= 0 && H <= (1ll << 30) && E >= 1 && E <= ELA_EXPERT_MAX &&
           (k == 0 || T <= INT32_MAX / k) && T <= INT32_MAX;
}

#define ELA_BY_DTYPE(dtype, ...)                              \
    switch (dtype) {                                           \
    case ELA_DTYPE_F32: { typedef float T_; __VA_ARGS__; break; }     \
    case ELA_DTYPE_F16: { typedef __half T_; __VA_ARGS__; break; }    \
    default: { typedef __nv_bfloat16 T_; __VA_ARGS__; break; }        \
    }

#define ELA_BY_PIECE(vb, ...)                                                      \
    switch (vb) {                                                                  \
    case 16: { constexpr int V_ = 16; __VA_ARGS__; break; }                        \
    case 8: { constexpr int V_ = 8; __VA_ARGS__; break; }                          \
    case 4: { constexpr int V_ = 4; __VA_ARGS__; break; }                          \
    default: { constexpr int V_ = sizeof(T_) < 4 ? 2 : 4; __VA_ARGS__; break; }    \
    }

}  // namespace ela_expert

using namespace ela_expert;

extern "C" {

size_t ela_expert_plan_workspace_bytes(int64_t, int64_t) { return 0; }

int ela_expert_plan(const void* expert, int id_bytes, int64_t slots, int64_t num_experts, int32_t* offsets,
                    int32_t* position, int32_t* source, void*, size_t, void* stream) {
    if ((id_bytes != 4 && id_bytes != 8) || slots < 0 || slots > INT32_MAX || num_experts < 1 ||
        num_experts > ELA_EXPERT_MAX || !offsets || (slots > 0 && (!expert || !position || !source)) ||
        !on_elements(id_bytes, expert) || !on_elements(4, offsets, position, source))
        return ELA_ERR_ARGUMENT;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    return id_bytes == 4 ? plan_launch((const int32_t*)expert, (int)slots, (int)num_experts, offsets, position, source, st)
                         : plan_launch((const int64_t*)expert, (int)slots, (int)num_experts, offsets, position, source, st);
}

int ela_expert_dispatch(const void* x, int dtype, int64_t T, int64_t k, int64_t H, int64_t ldx,
                        const int32_t* position, const int32_t* offsets, int64_t num_experts, void* rows,
                        void* stream) {
    if (!sizes_ok(dtype, T, k, H, num_experts) || ldx < 0) return ELA_ERR_ARGUMENT;
    if (T == 0 || k == 0 || H == 0) return ELA_OK;
    if (!x || !position || !offsets || !rows || !on_elements(dtype_bytes(dtype), x, rows) || !on_elements(4, position, offsets))
        return ELA_ERR_ARGUMENT;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const int es = dtype_bytes(dtype);
    const int vb = piece_bytes(address(x) | address(rows) | (uint64_t)(ldx * es) | (uint64_t)(H * es));
    const int G = group_threads(H, es, vb);
    int rc = ELA_OK;
    ELA_BY_DTYPE(dtype, ELA_BY_PIECE(vb, {
        rc = launch(dispatch_kernel<T_, V_>, route_grid(T, G), ROUTE_THREADS, 0, st, (const T_*)x, (int)T, (int)k, (int)H, ldx, G, position, offsets,
                                                                          (int)num_experts, (int)(T * k), (T_*)rows);
    }))
    return rc;
}

int ela_expert_combine(const void* y, int dtype, int64_t T, int64_t k, int64_t H, int64_t ldy,
                       const int32_t* position, const int32_t* offsets, int64_t num_experts, const void* weights,
                       int weights_dtype, void* out, void* stream) {
    if (!sizes_ok(dtype, T, k, H, num_experts) || ldy < 0) return ELA_ERR_ARGUMENT;
    if (weights && weights_dtype != ELA_DTYPE_F32 && weights_dtype != dtype) return ELA_ERR_ARGUMENT;
    if (T == 0 || H == 0) return ELA_OK;
    if (!out || !offsets || (k > 0 && (!y || !position))) return ELA_ERR_ARGUMENT;
    if (!on_elements(dtype_bytes(dtype), y, out) || !on_elements(4, position, offsets) ||
        (weights && !on_elements(dtype_bytes(weights_dtype), weights)))
        return ELA_ERR_ARGUMENT;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const int es = dtype_bytes(dtype);
    const int vb = piece_bytes(address(y) | address(out) | (uint64_t)(ldy * es) | (uint64_t)(H * es));
    const int G = group_threads(H, es, vb);
    const bool w32 = !weights || weights_dtype == ELA_DTYPE_F32;
    int rc = ELA_OK;
    ELA_BY_DTYPE(dtype, ELA_BY_PIECE(vb, {
        if (w32)
            rc = launch(combine_kernel<T_, float, V_>, route_grid(T, G), ROUTE_THREADS, 0, st, (const T_*)y, (int)T, (int)k, (int)H, ldy, G, position, offsets,
                                                                                     (int)num_experts, (int)(T * k), (const float*)weights, (T_*)out);
        else
            rc = launch(combine_kernel<T_, T_, V_>, route_grid(T, G), ROUTE_THREADS, 0, st, (const T_*)y, (int)T, (int)k, (int)H, ldy, G, position, offsets,
                                                                                  (int)num_experts, (int)(T * k), (const T_*)weights, (T_*)out);
    }))
    return rc;
}

int ela_expert_combine_grad(const void* dout, const void* y, int dtype, int64_t T, int64_t k, int64_t H,
                            int64_t lddo, int64_t ldy, const int32_t* position, const int32_t* offsets,
                            int64_t num_experts, const void* weights, int weights_dtype, void* dy, void* dweights,
                            void* stream) {
    if (!sizes_ok(dtype, T, k, H, num_experts) || lddo < 0 || ldy < 0) return ELA_ERR_ARGUMENT;
    if ((weights || dweights) && weights_dtype != ELA_DTYPE_F32 && weights_dtype != dtype) return ELA_ERR_ARGUMENT;
    if (T == 0 || k == 0 || (!dy && !dweights)) return ELA_OK;
    if (!offsets || !position || (H > 0 && (!dout || (dweights && !y)))) return ELA_ERR_ARGUMENT;
    if (!on_elements(dtype_bytes(dtype), dout, y, dy) || !on_elements(4, position, offsets) ||
        ((weights || dweights) && !on_elements(dtype_bytes(weights_dtype), weights, dweights)))
        return ELA_ERR_ARGUMENT;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const int es = dtype_bytes(dtype);
    const int vb = piece_bytes(address(dout) | address(dy) | address(dweights ? y : nullptr) | (uint64_t)(lddo * es) |
                               (uint64_t)(dweights ? ldy * es : 0) | (uint64_t)(H * es));
    const int G = group_threads(H, es, vb);
    const bool w32 = (!weights && !dweights) || weights_dtype == ELA_DTYPE_F32;
    int rc = ELA_OK;
    ELA_BY_DTYPE(dtype, ELA_BY_PIECE(vb, {
        if (w32)
            rc = launch(combine_grad_kernel<T_, float, V_>, route_grid(T, G), ROUTE_THREADS, 0, st, 
                (const T_*)dout, (const T_*)y, (int)T, (int)k, (int)H, lddo, ldy, G, position, offsets, (int)num_experts, (int)(T * k),
                (const float*)weights, (T_*)dy, (float*)dweights);
        else
            rc = launch(combine_grad_kernel<T_, T_, V_>, route_grid(T, G), ROUTE_THREADS, 0, st, 
                (const T_*)dout, (const T_*)y, (int)T, (int)k, (int)H, lddo, ldy, G, position, offsets, (int)num_experts, (int)(T * k),
                (const T_*)weights, (T_*)dy, (T_*)dweights);
    }))
    return rc;
}

}  // extern "C"
