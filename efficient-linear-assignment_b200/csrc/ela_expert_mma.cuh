// ela_expert_mma.cuh -- the tensor-core product behind ela_expert_linear and its
// gradients (included by ela_expert_linear.cu).
//
// One persistent kernel computes out[c][f] = sum_k A(f,k) B(c,k), f contiguous in
// memory.  A pair of CTAs (cluster of 2, tcgen05 cta_group::2) owns a tile of 256
// features f by up to 256 columns c: each CTA loads 128 of the features and half of
// the columns, and keeps the accumulators of its 128 features by all columns.
//
//   pass           f (TMEM lanes)         c (MMA N)            k
//   forward        output feature n       row of the expert    input feature
//   input grad     input feature          row of the expert    output feature
//   weight grad    input feature          output feature       row of the expert
//
// Why a pair: one CTA's 128 x 256 tile loads 48 KB per 64 k, of which a CTA of a pair
// loads 32 KB for the same products: 4096^3 bf16 212 us by single CTAs, 94 us by pairs
// with the rest below, and 108 us in a loop at the power limit (1270 TFLOP/s, 0.92 of the
// measured sustained 1384; the library's product 90.5 and 104).  At full rounds a block of
// 64 k takes 386 ns against the 374 ns that the library's burst rate means; the rest is the
// last round, 34 tiles for 74 pairs.  Long products are held by the power limit, not by the
// schedule: 8192 rows by 8 experts of 8192 x 2048 take 203 us in a short run and 236 in a
// loop, and their input gradient keeps the tensor pipe 91 % busy.
//
// The rows of an expert are the MMA's N side, whose extent is a multiple of 32
// chosen per instruction: the last tile of an expert costs what its rows need, and
// the weights, the side with whole tiles, fill the 128 lanes.
//
// Operands are K-major where k is contiguous in memory (x and W in the forward
// pass, dz in the input gradient) and MN-major where it is not (W in the input
// gradient, both sides of the weight gradient); both come as 128-byte-swizzled TMA
// boxes, so no operand is ever transposed in memory.  Rows that belong to the next
// expert are harmless on the N side (their columns are not stored); in the weight
// gradient, where rows are summed over, the last block's rows past the expert are
// zeroed in shared memory, on both sides, since 0 * NaN is not 0.
//
// Roles, in each CTA: warp 0 issues the TMA loads of the CTA's halves, which count on the
// first CTA's barriers; warp 1 of the first CTA issues the MMAs of the pair; warp 2 owns the
// TMEM allocation and sums ReLU's z next to 0 again; warp 3 works out the tiles; warps 4-11
// run the epilogue while the next tile's MMAs fill the other half of TMEM (2 x 256 columns).
// Loads and MMAs are issued by one elected thread that runs the whole inner loop (a warp that
// polls, broadcasts and reconverges each block took 40 % longer), and no arrival of the inner
// loop crosses CTAs with cluster-scope ordering, whose fences cost 1000 cycles.  A warp reads
// 16 columns of its 32 features at a time, one feature a lane; bias, activation and residual
// are applied in fp32, and two neighbouring lanes swap halves so that each stores two
// consecutive features of one column: a store instruction writes 64 bytes of two columns,
// whole sectors, with no staging in shared memory and no barrier between the warps (staging
// fp32 chunks to store 256 bytes a row: 88 us instead of 46 for the weight gradient of 64
// experts of 1024 x 1024, whose tiles have two blocks of k each).  The residual of a chunk is
// loaded before its accumulators are waited for.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include "ela_expert.cuh"

namespace ela_expert {

enum { PASS_FORWARD = 0, PASS_INPUT = 1, PASS_WEIGHT = 2 };

constexpr int MMA_F = 128;              // features per CTA (TMEM lanes)
constexpr int MMA_PAIR_F = 256;         // features per tile
constexpr int MMA_C = 256;              // most columns per tile
constexpr int MMA_KB = 64;              // k per stage: 128 bytes, one swizzle span
constexpr int MMA_A_BYTES = MMA_F * MMA_KB * 2;
constexpr int MMA_CHUNK = 16;           // columns an epilogue warp takes at a time
constexpr int MMA_GROUPS = 2;           // epilogue warps per 32 TMEM lanes: 4 take 3 % less for the shortest
                                        // sums, but 2-4 % more for long ones at the power limit
constexpr int MMA_MAX_STAGES = 10;
constexpr int MMA_THREADS = 128 + MMA_GROUPS * 128;
constexpr int MMA_SMEM = 227 * 1024;
constexpr int MMA_SMEM_FIXED = 1024;    // alignment of the first stage
constexpr int MMA_TILES = 4;            // tiles the scheduling warp is ahead
constexpr int MMA_GROUP = 16;           // column tiles walked together, for L2 reuse of both operands

struct MmaParams {
    const int32_t* offsets;
    int R, E, F, C, K;      // C: columns of the weight gradient; K: contraction length of the row passes
    int bn, bbox, stages;   // columns per tile; rows per TMA box of the column operand; pipeline depth
    int f_tiles, c_tiles;   // c_tiles: weight gradient only
    int vec;                // two consecutive features may be loaded and stored together
    const void* bias;
    const void* residual;
    const void* x;          // forward with z: the operands again, for exact_z
    const void* weight;
    int64_t ldr, ldx, ldw, stride_e;
    void* out;
    void* z;
    unsigned long long wait_ns;
};

// Sticky error of the kernels below (a wait that ran out), read by ela_expert_status.
__device__ int g_expert_error;

// ------------------------------------------------------------- PTX wrappers
__device__ __forceinline__ uint32_t saddr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint64_t* b, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(saddr(b)), "r"(count) : "memory");
}
// The address of the same object in the pair's first CTA.
__device__ __forceinline__ uint32_t leader_addr(const void* p) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(saddr(p)));
    return r;
}
__device__ __forceinline__ void bar_expect(uint64_t* b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(saddr(b)), "r"(bytes) : "memory");
}
// Arrivals on another CTA's barrier.  Where the barrier orders TMEM or loads alone, the
// arrival is relaxed: a release at cluster scope is a fence that costs hundreds of cycles.
__device__ __forceinline__ void bar_arrive_at(uint32_t addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
__device__ __forceinline__ void bar_arrive_relaxed_at(uint32_t addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(saddr(b)) : "memory");
}
// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t yes;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
    return yes;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Bounded wait for the phase of this parity; false when the limit ran out or another role gave up.
__device__ __forceinline__ bool bar_wait(uint64_t* b, uint32_t parity, unsigned long long limit_ns,
                                         const volatile int* abort) {
    const uint32_t a = saddr(b);
    unsigned long long t0 = 0;
    for (uint32_t spins = 1;; ++spins) {
        uint32_t done;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(done) : "r"(a), "r"(parity), "r"(20000) : "memory");  // sleeps up to 20 us
        if (done) return true;
        if ((spins & 15u) == 0) {
            unsigned long long t;
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
            if (t0 == 0) t0 = t;
            if (*abort || t - t0 > limit_ns) return false;
        }
    }
}
// bar: shared::cluster address; it may be the pair's other CTA's.
__device__ __forceinline__ void tma_2d(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(saddr(dst)), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void tma_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(saddr(dst)), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
// Arrives on the barrier of this place in both CTAs when the products issued so far are done.
__device__ __forceinline__ void mma_commit(uint64_t* b) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(saddr(b)), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void mma_issue(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// Shared-memory operand descriptors, 128-byte swizzle (layout type 2, version 1).
// K-major: 8-row groups 1024 bytes apart; the k steps of 16 advance the start by 32 bytes.
// MN-major: blocks of 64 along MN 8192 bytes apart (one TMA box each), groups of 8
// along k 1024 bytes apart; the k steps of 16 advance the start by 2048 bytes.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, bool k_major) {
    const uint64_t lead = k_major ? 1 : 8192 >> 4, stride = 1024 >> 4;
    return (uint64_t)((addr >> 4) & 0x3fff) | (lead << 16) | (stride << 32) | (1ull << 46) | (2ull << 61);
}
template <typename T> __device__ __forceinline__ uint32_t instr_desc(int n, bool a_k_major, bool b_k_major) {
    const uint32_t ab = sizeof(T) == 2 && El<T>::BF16 ? 1u : 0u;
    return (1u << 4) | (ab << 7) | (ab << 10) | ((a_k_major ? 0u : 1u) << 15) | ((b_k_major ? 0u : 1u) << 16) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(MMA_PAIR_F >> 4) << 24);
}

// ------------------------------------------------------------- tile order
struct Tile {
    int e, f0, c0, nc;  // expert, first feature, first column, columns
    int k0, nk;         // contraction range (weight gradient: rows of the expert)
};

// The experts' rows and row tiles, in shared memory.
struct Plan {
    const int *row0, *row1, *tile0;  // [E]; tile0: tiles before expert e (row passes)
    int tiles;
};

// Row passes: experts in order; within an expert, groups of MMA_GROUP column tiles,
// feature tiles within a group, columns innermost.  Weight gradient: the same with the
// output features as columns.  The offsets, and so the tiles, are only known on the
// device.  The whole warp calls.
template <int PASS> __device__ __forceinline__ bool get_tile(const MmaParams& p, const Plan& plan, int t, Tile& out) {
    if (t >= plan.tiles) return false;
    int local, ct, r0, r1;
    if constexpr (PASS == PASS_WEIGHT) {
        ct = p.c_tiles;
        const int per = p.f_tiles * ct;
        out.e = t / per;
        local = t - out.e * per;
    } else {
        // the last expert whose tiles start at or before t: 32 probes a step
        const int lane = threadIdx.x & 31;
        int lo = 0, n = p.E;
        while (n > 1) {
            const int step = (n + 31) >> 5, at = lo + lane * step;
            const unsigned in = __ballot_sync(~0u, lane * step < n && plan.tile0[at < p.E ? at : p.E - 1] <= t);
            const int last = 31 - __clz(in);  // (probe 0 always holds)
            lo += last * step;
            n = min(step, n - last * step);
        }
        out.e = lo;
        local = t - plan.tile0[lo];
    }
    r0 = plan.row0[out.e];
    r1 = plan.row1[out.e];
    if constexpr (PASS != PASS_WEIGHT) ct = (r1 - r0 + p.bn - 1) / p.bn;
    const int group = local / (MMA_GROUP * p.f_tiles), g = min(MMA_GROUP, ct - group * MMA_GROUP);
    local -= group * MMA_GROUP * p.f_tiles;
    out.f0 = local / g * MMA_PAIR_F;
    const int c = (group * MMA_GROUP + local % g) * p.bn;
    if constexpr (PASS == PASS_WEIGHT) {
        out.c0 = c;
        out.nc = min(p.bn, p.C - c);
        out.k0 = r0;
        out.nk = r1 - r0;
    } else {
        out.c0 = r0 + c;
        out.nc = min(p.bn, r1 - out.c0);
        out.k0 = 0;
        out.nk = p.K;
    }
    return true;
}

// ------------------------------------------------------------- epilogue
// Lanes 2i and 2i+1 hold features f and f+1 of columns c (low half of p) and c+1 (high
// half).  After the swap the even lane has f, f+1 of column c, the odd lane of column
// c+1, which is how memory has them; it is its own inverse.
__device__ __forceinline__ uint32_t swap_pair(uint32_t p, uint32_t order) {
    return __byte_perm(p, __shfl_xor_sync(~0u, p, 1), order);
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t p);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t p) { return __half22float2(*reinterpret_cast<const __half2*>(&p)); }
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t p) {
    return make_float2(__uint_as_float(p << 16), __uint_as_float(p & 0xffff0000u));
}

// One chunk of a warp: v[j] is feature f (this lane's) of column c + j, j < left.  The
// lane's residual words are those of swap_pair's layout (loaded by load_residual).
// Addresses go from pair to pair of columns by one 64-bit addition: written as a product
// with j they made most of the epilogue's instructions.
template <typename T, int ACT, bool BIAS, bool Z, bool RES, bool ALL>
__device__ __forceinline__ void finish(float* v, float bias, const uint32_t* res, const MmaParams& p, int64_t c, int f, int left) {
    const bool odd = threadIdx.x & 1;
    const uint32_t order = odd ? 0x3276 : 0x5410;
    if (ALL || p.vec) {
        const int64_t at = (c + odd) * p.F + (f & ~1);
        char* out = reinterpret_cast<char*>(reinterpret_cast<T*>(p.out) + at);
        typedef typename Kept<T, ACT>::Type K;
        char* zout = reinterpret_cast<char*>(reinterpret_cast<K*>(p.z) + at);
        const int64_t step = 4 * (int64_t)p.F;
        // (F is even: both lanes of a pair are in or out)
        const int mine = ALL ? MMA_CHUNK : f < p.F ? left - odd : 0;
#pragma unroll
        for (int j = 0; j < MMA_CHUNK; j += 2) {
            float a = v[j], b = v[j + 1];
            if (BIAS) { a += bias; b += bias; }
            if (Z) {
                if constexpr (sizeof(K) == 4) {  // the same exchange with one float each way
                    const float other = __shfl_xor_sync(~0u, odd ? a : b, 1);
                    if (ALL || j < mine) *reinterpret_cast<float2*>(zout) = odd ? make_float2(other, b) : make_float2(a, other);
                } else {
                    const uint32_t w = swap_pair(ACT == ELA_ACT_RELU ? pack2<T>(sign_kept<T>(a), sign_kept<T>(b)) : pack2<T>(a, b), order);
                    if (ALL || j < mine) *reinterpret_cast<uint32_t*>(zout) = w;
                }
                zout += step * (sizeof(K) / 2);
            }
            a = act_value<ACT>(a);
            b = act_value<ACT>(b);
            if (RES) {
                const float2 r = unpack2<T>(swap_pair(res[j / 2], order));
                a += r.x;
                b += r.y;
            }
            const uint32_t w = swap_pair(pack2<T>(a, b), order);
            if (ALL || j < mine) *reinterpret_cast<uint32_t*>(out) = w;
            out += step;
        }
    } else if (f < p.F) {
#pragma unroll
        for (int j = 0; j < MMA_CHUNK; ++j)
            if (j < left) {
                const float a = BIAS ? v[j] + bias : v[j];
                const int64_t at = (c + j) * p.F + f;
                typedef typename Kept<T, ACT>::Type K;
                if (Z) reinterpret_cast<K*>(p.z)[at] = El<K>::from(ACT == ELA_ACT_RELU ? sign_kept<T>(a) : a);
                const float r = RES ? El<T>::to(reinterpret_cast<const T*>(p.residual)[(c + j) * p.ldr + f]) : 0.f;
                reinterpret_cast<T*>(p.out)[at] = El<T>::from(act_value<ACT>(a) + r);
            }
    }
}

// A z next to 0 (sign_band) to be summed again.  The epilogue warps leave them to warp 2,
// which has nothing else to do, in a queue each, and only do themselves what finds its queue
// full, and what is left when the tiles are done: done by the epilogue alone they held up the
// tiles (8192 rows of 64 experts of 1024 x 1024 43 -> 56 us, 16384 of 8 of 8192 x 2048 402 ->
// 564; so 43 and 427, and 37 and 369 without z).
struct Near { int e, row, f; };
constexpr int NEAR_QUEUE = 4;  // (static shared memory stays under the 1024 bytes left beside the stages)
struct NearQueues {
    Near at[4 * MMA_GROUPS][NEAR_QUEUE];
    uint32_t head[4 * MMA_GROUPS], tail[4 * MMA_GROUPS];  // entries put in, and taken out
    int ended[4 * MMA_GROUPS];                            // the epilogue warp has no more tiles
    uint32_t tile;                                        // counts tiles: a sign of life
};

template <bool SIGNS> struct Queues { typedef NearQueues Type; };
template <> struct Queues<false> { typedef int Type; };

// The whole warp: z of one row and feature, summed again.
template <typename T> __device__ __forceinline__ double exact_z(const MmaParams& p, const Near& n) {
    const double sum = exact_sum<T>(reinterpret_cast<const T*>(p.x) + (int64_t)n.row * p.ldx,
                                    reinterpret_cast<const T*>(p.weight) + (int64_t)n.e * p.stride_e + (int64_t)n.f * p.ldw, p.K);
    return sum + (p.bias ? (double)El<T>::to(reinterpret_cast<const T*>(p.bias)[(int64_t)n.e * p.F + n.f]) : 0.0);
}
template <typename T> __device__ __forceinline__ void settle_sign(const MmaParams& p, const Near& n) {
    const double z = exact_z<T>(p, n);
    if ((threadIdx.x & 31) == 0) reinterpret_cast<T*>(p.z)[(int64_t)n.row * p.F + n.f] = El<T>::from(sign_kept<T>((float)z));
}
// Takes the oldest entry out of a queue and settles it; false: the queue is empty.  (The entry
// is copied before it is claimed: only then may its place be filled again.)  The whole warp.
template <typename T> __device__ __forceinline__ bool settle_oldest(const MmaParams& p, NearQueues& queues, int w) {
    const int lane = threadIdx.x & 31;
    Near n = {};
    int got = 0;
    if (lane == 0) {
        for (;;) {  // (ends: another warp claimed an entry each time that this one did not)
            const uint32_t tail = *(volatile uint32_t*)&queues.tail[w];
            if (tail == *(volatile uint32_t*)&queues.head[w]) break;
            __threadfence_block();
            const volatile Near* at = &queues.at[w][tail % NEAR_QUEUE];
            n.e = at->e; n.row = at->row; n.f = at->f;
            __threadfence_block();
            if (atomicCAS(&queues.tail[w], tail, tail + 1) == tail) { got = 1; break; }
        }
    }
    if (!__shfl_sync(~0u, got, 0)) return false;
    n.e = __shfl_sync(~0u, n.e, 0);
    n.row = __shfl_sync(~0u, n.row, 0);
    n.f = __shfl_sync(~0u, n.f, 0);
    settle_sign<T>(p, n);
    return true;
}

// Whether a chunk may hold such a z, by the warp's largest: of |z| in its rounded form, two
// columns at a time, 16 instructions a chunk.
template <typename T> struct Two;
template <> struct Two<__half> { typedef __half2 V; };
template <> struct Two<__nv_bfloat16> { typedef __nv_bfloat162 V; };
template <typename T>
__device__ __forceinline__ bool may_be_near_zero(const float* v, float bias, const MmaParams& p, int f, int left) {
    if (left < MMA_CHUNK) return true;  // (what lies past the columns is not z)
    typedef typename Two<T>::V V;
    V big, least;
#pragma unroll
    for (int j = 0; j < MMA_CHUNK; j += 2) {
        const uint32_t w = pack2<T>(v[j] + bias, v[j + 1] + bias);
        const V z = __habs2(*reinterpret_cast<const V*>(&w));
        big = j ? __hmax2(big, z) : z;
        least = j ? __hmin2(least, z) : z;
    }
    const float most = f < p.F ? fmaxf(El<T>::to(big.x), El<T>::to(big.y)) + fabsf(bias) : 0.f;
    // (numbers from 0 on compare as their bits do; a NaN or an infinity is not "above" the band and is looked at)
    const float largest = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(most)));
    const float z = fminf(El<T>::to(least.x), El<T>::to(least.y));
    return __any_sync(~0u, f < p.F && !(z > sign_band(largest, p.K)));
}

// The lane's z within the band of their row, and its sums that are exactly 0, a bit a column.
__device__ __forceinline__ void near_columns(const float* v, float bias, int K, bool in, unsigned features, int left, unsigned& near, unsigned& zero) {
    const float bias_size = fabsf(bias) < INFINITY ? fabsf(bias) : 0.f;
    const bool few = __popc(features) < 8;  // too few features to tell a row's size: the largest of all rows
    float all = 0.f;
    if (few) {
#pragma unroll
        for (int j = 0; j < MMA_CHUNK; ++j) {
            const float z = fabsf(v[j] + bias);
            if (in && j < left && z < INFINITY) all = fmaxf(all, z + bias_size);
        }
        all = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(all)));
    }
    near = zero = 0;
#pragma unroll
    for (int j = 0; j < MMA_CHUNK; ++j) {
        const float z = fabsf(v[j] + bias);
        const bool here = in && j < left;
        float row = all;
        if (!few) row = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(here && z < INFINITY ? z + bias_size : 0.f)));
        const float band = sign_band(row, K);
        near |= (unsigned)(here && band > 0.f && z <= band) << j;
        zero |= (unsigned)(here && v[j] == 0.f) << j;
    }
}

// Hands the chunk's z next to 0 on to warp 2.  Exact zeros come by the hundred from rows of
// zeros, from features whose weights are zeros, and from products that are mostly zeros or
// small whole numbers; one by accident of rounding in 80000 chunks.  Whole rows and whole
// features of them are taken as they are, and so are two and more where the first one is 0
// summed again, too.
template <typename T>
__device__ __noinline__ void settle_signs(unsigned near, unsigned zero, const MmaParams& p, NearQueues& queues, int w, int e, int c, int f, int left) {
    const int lane = threadIdx.x & 31;
    const unsigned features = __ballot_sync(~0u, f < p.F), rows = left < MMA_CHUNK ? (1u << left) - 1 : (1u << MMA_CHUNK) - 1;
    const unsigned empty = __reduce_and_sync(~0u, f < p.F ? zero : ~0u);
    if (__popc(features) >= 8) near &= ~empty;
    if (left >= 8 && zero == rows) near = 0;
    if (__reduce_add_sync(~0u, __popc(near & zero)) >= 2) {
        const int from = __ffs(__ballot_sync(~0u, (near & zero) != 0)) - 1;
        const int j = __shfl_sync(~0u, __ffs(near & zero) - 1, from);
        if (exact_sum<T>(reinterpret_cast<const T*>(p.x) + (int64_t)(c + j) * p.ldx,
                         reinterpret_cast<const T*>(p.weight) + (int64_t)e * p.stride_e + (int64_t)(f - lane + from) * p.ldw, p.K) == 0.0)
            near &= ~zero;
    }
    __syncwarp();  // finish()'s stores come before those that replace them
    for (unsigned any = __reduce_or_sync(~0u, near); any; any &= any - 1) {
        const int j = __ffs(any) - 1;
        for (unsigned todo = __ballot_sync(~0u, near >> j & 1); todo; todo &= todo - 1) {
            const Near n = {e, c + j, f - lane + __ffs(todo) - 1};
            bool full = false;
            if (lane == 0) {
                const uint32_t head = queues.head[w];
                full = head - *(volatile uint32_t*)&queues.tail[w] >= NEAR_QUEUE;
                if (!full) {
                    queues.at[w][head % NEAR_QUEUE] = n;
                    __threadfence_block();
                    *(volatile uint32_t*)&queues.head[w] = head + 1;
                }
            }
            if (__any_sync(~0u, full)) settle_sign<T>(p, n);
        }
    }
}

template <typename T>
__device__ __forceinline__ void load_residual(uint32_t* res, const MmaParams& p, int64_t c, int f, int left) {
    const bool odd = threadIdx.x & 1;
    const uint32_t* at = reinterpret_cast<const uint32_t*>(reinterpret_cast<const T*>(p.residual) + (c + odd) * p.ldr + (f & ~1));
    const int mine = p.vec && f < p.F ? left - odd : 0;
#pragma unroll
    for (int j = 0; j < MMA_CHUNK; j += 2, at += p.ldr) res[j / 2] = j < mine ? *at : 0u;
}

// Z: the forward pass keeps z for the gradient.
template <int PASS, typename T, int ACT, bool Z>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(MMA_THREADS, 1)
    mma_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
               const __grid_constant__ MmaParams p) {
    constexpr bool A_K_MAJOR = PASS == PASS_FORWARD, B_K_MAJOR = PASS != PASS_WEIGHT;
    extern __shared__ unsigned char smem_raw[];
    // full, tempty, patched: the first CTA's are used; empty, tfull, landed: each CTA its own
    __shared__ __align__(8) uint64_t full[MMA_MAX_STAGES], empty[MMA_MAX_STAGES], tfull[2], tempty[2], sfull[MMA_TILES], sempty[MMA_TILES], patched[MMA_MAX_STAGES], landed, drained;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    __shared__ uint32_t s_issued;
    __shared__ int s_tiles;
    __shared__ Tile s_tile[MMA_TILES];
    constexpr bool SIGNS = Z && ACT == ELA_ACT_RELU;
    __shared__ typename Queues<SIGNS>::Type s_near;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    // the experts' tables, then the stages, each on a 1024-byte boundary
    int* table = reinterpret_cast<int*>(smem_raw);
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(table + 3 * p.E) + 1023) & ~(uintptr_t)1023);
    const int stage_bytes = MMA_A_BYTES + p.bn / 2 * MMA_KB * 2;
    const volatile int* abort = &s_abort;

    next_may_start();
    if (tid == 32) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b) : "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(saddr(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        s_abort = 0;
        for (int s = 0; s < p.stages; ++s) { bar_init(&full[s], 1); bar_init(&empty[s], 1); }
        for (int b = 0; b < 2; ++b) { bar_init(&tfull[b], 1); bar_init(&tempty[b], 2 * 4 * MMA_GROUPS); }
        for (int i = 0; i < MMA_TILES; ++i) { bar_init(&sfull[i], 1); bar_init(&sempty[i], 4 * MMA_GROUPS + 1 + (rank == 0)); }
        bar_init(&landed, 1);
        for (int s = 0; s < p.stages; ++s) bar_init(&patched[s], 1);
        bar_init(&drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if constexpr (SIGNS) {
        if (tid < 4 * MMA_GROUPS) s_near.head[tid] = s_near.tail[tid] = s_near.ended[tid] = 0;
        if (tid == 0) s_near.tile = 0;
    }
    previous_done();  // (no memory was touched before)
    for (int e = tid; e < p.E; e += MMA_THREADS) expert_rows(p.offsets, e, p.R, table[e], table[p.E + e]);
    __syncthreads();
    if (PASS != PASS_WEIGHT && warp == 3) {  // row tiles before each expert
        int before = 0;
        for (int e = lane; e - lane < p.E; e += 32) {
            const int mine = e < p.E ? (table[p.E + e] - table[e] + p.bn - 1) / p.bn * p.f_tiles : 0;
            int incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(~0u, incl, o);
                if (lane >= o) incl += v;
            }
            if (e < p.E) table[2 * p.E + e] = before + incl - mine;
            before += __shfl_sync(~0u, incl, 31);
        }
        if (lane == 0) s_tiles = before;
    }
    fence_before();
    __syncthreads();
    cluster_sync();  // the barriers of both CTAs are there before either is signalled
    fence_after();
    const uint32_t tmem = s_tmem;
    const Plan plan = {table, table + p.E, table + 2 * p.E, PASS == PASS_WEIGHT ? p.E * p.f_tiles * p.c_tiles : s_tiles};
    auto give_up = [&]() {
        *(volatile int*)&s_abort = 1;
        atomicExch(&g_expert_error, ELA_ERR_TIMEOUT);
    };

    // The i-th tile of this pair from the scheduling warp; false: none left, or a wait gave up (ok).
    auto fetch = [&](int i, Tile& t, bool& ok) {
        const int slot = i % MMA_TILES;
        int good = 0;
        if (lane == 0) good = bar_wait(&sfull[slot], (i / MMA_TILES) & 1, p.wait_ns, abort);
        ok = __shfl_sync(~0u, good, 0);
        __syncwarp();
        if (!ok) { if (lane == 0) give_up(); return false; }
        t = s_tile[slot];
        __syncwarp();
        if (lane == 0) bar_arrive(&sempty[slot]);
        return t.e >= 0;
    };

    uint32_t issued = 0;  // stages loaded (by the loading lane)
    if (warp == 3) {  // ---- tiles, a few ahead: their index arithmetic would cost each role 1000 cycles a tile
        bool ok = true, left = true;
        for (int i = 0, n = pair; ok && left; ++i, n += pairs) {
            const int slot = i % MMA_TILES;
            Tile t;
            left = get_tile<PASS>(p, plan, n, t);
            int good = 0;
            if (lane == 0) {
                good = bar_wait(&sempty[slot], ((i / MMA_TILES) & 1) ^ 1, p.wait_ns, abort);
                if (good) {
                    if (!left) t.e = -1;
                    s_tile[slot] = t;
                    bar_arrive(&sfull[slot]);
                } else {
                    give_up();
                }
            }
            ok = __shfl_sync(~0u, good, 0);
        }
    } else if (warp == 0) {  // ---- loads of this CTA's features and its half of the columns
        Tile t;
        int s = 0;
        uint32_t phase = 0, landings = 0, patches = 0;  // patches: bit s, the parity of stage s's patches
        bool ok = true;
        for (int i = 0; ok && fetch(i, t, ok); ++i) {
            const int f0 = t.f0 + rank * MMA_F;
            // column operand: boxes of p.bbox rows (K-major) or of 64 columns (MN-major)
            const int half = ((t.nc + 31) & ~31) >> 1, c0 = t.c0 + rank * half;
            const int boxes = B_K_MAJOR ? (half + p.bbox - 1) / p.bbox : (half + 63) / 64;
            const int box_bytes = B_K_MAJOR ? p.bbox * MMA_KB * 2 : 64 * MMA_KB * 2;
            const uint32_t bytes = MMA_A_BYTES + boxes * box_bytes;
            // Rows of the next expert in the last block of a sum over rows: that block's
            // loads land on a barrier of this CTA, the rows are zeroed, then the stage is full.
            const int tail = PASS == PASS_WEIGHT ? t.nk % MMA_KB : 0, blocks = (t.nk + MMA_KB - 1) / MMA_KB;
            const bool patch = (tail & 15) != 0;
            auto load = [&](int k, uint32_t bar) {  // one thread; into stage s
                unsigned char* a = smem + (size_t)s * stage_bytes;
                unsigned char* b = a + MMA_A_BYTES;
                if (PASS == PASS_FORWARD) {
                    tma_3d(a, &map_a, k, f0, t.e, bar);
                } else {
                    for (int h = 0; h < 2; ++h)
                        if (PASS == PASS_INPUT) tma_3d(a + h * 8192, &map_a, f0 + h * 64, k, t.e, bar);
                        else tma_2d(a + h * 8192, &map_a, f0 + h * 64, k, bar);
                }
                for (int i = 0; i < boxes; ++i)
                    if (B_K_MAJOR) tma_2d(b + i * box_bytes, &map_b, k, c0 + i * p.bbox, bar);
                    else tma_2d(b + i * box_bytes, &map_b, c0 + i * 64, k, bar);
                ++issued;
            };
            const int plain = blocks - patch;
            if (elect_one()) {
                for (int kb = 0; kb < plain; ++kb) {
                    ok = bar_wait(&empty[s], phase ^ 1, p.wait_ns, abort);
                    if (!ok) break;
                    if (rank == 0) bar_expect(&full[s], 2 * bytes);  // the pair's
                    load(t.k0 + kb * MMA_KB, leader_addr(&full[s]));
                    if (++s == p.stages) { s = 0; phase ^= 1; }
                }
                if (patch && ok) {
                    ok = bar_wait(&empty[s], phase ^ 1, p.wait_ns, abort);
                    if (ok) {
                        bar_expect(&landed, bytes);
                        load(t.k0 + plain * MMA_KB, saddr(&landed));
                        ok = bar_wait(&landed, landings & 1, p.wait_ns, abort);
                    }
                }
                if (!ok) give_up();
            }
            // the elected lane's place in the ring, to all (elect_one names the same lane again)
            const int who = __ffs(__ballot_sync(~0u, elect_one())) - 1;
            ok = __shfl_sync(~0u, (int)ok, who);
            s = __shfl_sync(~0u, s, who);
            phase = __shfl_sync(~0u, phase, who);
            __syncwarp();
            if (patch && ok) {
                ++landings;
                unsigned char* a = smem + (size_t)s * stage_bytes;
                const int pieces = (16 - (tail & 15)) * 8;  // A's two boxes, then B's, 8192 bytes each
                for (int j = lane; j < (2 + boxes) * pieces; j += 32)
                    *reinterpret_cast<uint4*>(a + (size_t)(j / pieces) * 8192 + tail * 128 + j % pieces * 16) = make_uint4(0, 0, 0, 0);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    // (a barrier per stage: the second CTA may be as many patches ahead as there are
                    // stages, and a phase of a single barrier would pass unseen)
                    if (rank == 1) {
                        bar_arrive_at(leader_addr(&patched[s]));
                    } else {
                        ok = bar_wait(&patched[s], (patches >> s) & 1, p.wait_ns, abort);
                        asm volatile("fence.acq_rel.cluster;" ::: "memory");
                        if (ok) bar_arrive(&full[s]);
                        else give_up();
                    }
                }
                ok = __shfl_sync(~0u, (int)ok, 0);
                patches ^= 1u << s;
                if (++s == p.stages) { s = 0; phase ^= 1; }
            }
        }
        s_issued = 0;
        __syncwarp();
        if (issued) s_issued = issued;
    } else if (warp == 1 && rank == 0) {  // ---- products of the pair
        Tile t;
        int s = 0, it = 0;
        uint32_t phase = 0;
        bool ok = true;
        const uint64_t a_desc = operand_desc(saddr(smem), A_K_MAJOR), b_desc = operand_desc(saddr(smem) + MMA_A_BYTES, B_K_MAJOR);
        constexpr int A_STEP = A_K_MAJOR ? 2 : 128, B_STEP = B_K_MAJOR ? 2 : 128;  // 16 k, in 16-byte units
        for (int i = 0; ok && fetch(i, t, ok); ++i) {
            const int blocks = (t.nk + MMA_KB - 1) / MMA_KB;
            if (blocks == 0) continue;  // an expert without rows: the epilogue writes its zeros
            if (elect_one()) {
                const int half = it & 1;
                const uint32_t d = tmem + half * MMA_C;
                const uint32_t idesc = instr_desc<T>((t.nc + 31) & ~31, A_K_MAJOR, B_K_MAJOR);
                ok = bar_wait(&tempty[half], ((it >> 1) & 1) ^ 1, p.wait_ns, abort);
                fence_after();
                for (int kb = 0; kb < blocks && ok; ++kb) {
                    ok = bar_wait(&full[s], phase, p.wait_ns, abort);
                    if (!ok) break;
                    fence_after();
                    const uint64_t off = (uint32_t)(s * stage_bytes) >> 4;
                    const int left = t.nk - kb * MMA_KB;
                    if (left >= MMA_KB) {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            mma_issue(d, a_desc + off + j * A_STEP, b_desc + off + j * B_STEP, idesc, kb + j > 0);
                    } else {
                        for (int j = 0; j < (left + 15) >> 4; ++j)
                            mma_issue(d, a_desc + off + j * A_STEP, b_desc + off + j * B_STEP, idesc, kb + j > 0);
                    }
                    mma_commit(&empty[s]);
                    if (++s == p.stages) { s = 0; phase ^= 1; }
                }
                if (ok) mma_commit(&tfull[half]);
                else give_up();
            }
            const int who = __ffs(__ballot_sync(~0u, elect_one())) - 1;
            ok = __shfl_sync(~0u, (int)ok, who);
            s = __shfl_sync(~0u, s, who);
            phase = __shfl_sync(~0u, phase, who);
            ++it;
        }
    } else if (SIGNS && warp == 2) {  // ---- z next to 0, as the epilogue finds them
        if constexpr (SIGNS) {
            const bool mine = lane < 4 * MMA_GROUPS;
            uint32_t tile = 0;
            unsigned long long t0 = 0, now;
            for (;;) {
                const bool ended = !mine || *(volatile int*)&s_near.ended[lane];
                __threadfence_block();
                const unsigned have = __ballot_sync(~0u, mine && *(volatile uint32_t*)&s_near.head[lane] != *(volatile uint32_t*)&s_near.tail[lane]);
                if (have) {
                    settle_oldest<T>(p, s_near, __ffs(have) - 1);
                    t0 = 0;
                    continue;
                }
                if (__all_sync(~0u, ended)) break;
                __nanosleep(500);
                asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
                const uint32_t seen = *(volatile uint32_t*)&s_near.tile;
                if (t0 == 0 || seen != tile) { t0 = now; tile = seen; }
                // (the epilogue's own waits end first: two of them at most between tiles)
                if (__any_sync(~0u, now - t0 > 4 * p.wait_ns)) {
                    if (lane == 0) give_up();
                    break;
                }
            }
        }
    } else if (warp >= 4) {  // ---- epilogue
        const int w = warp & 3, group = (warp - 4) >> 2;
        if constexpr (PASS != PASS_WEIGHT) {  // rows of no expert: the residual, or 0
            const int lo = p.offsets ? clampi(p.offsets[0], 0, p.R) : 0, hi = p.offsets ? clampi(p.offsets[p.E], 0, p.R) : p.R;
            for (int r = blockIdx.x; r < p.R; r += (int)gridDim.x) {
                if (r >= lo && r < hi) { r = hi - 1 - (hi - 1 - r) % (int)gridDim.x; continue; }
                for (int f = tid - 128; f < p.F; f += MMA_GROUPS * 128)
                    reinterpret_cast<T*>(p.out)[(int64_t)r * p.F + f] =
                        p.residual ? reinterpret_cast<const T*>(p.residual)[r * p.ldr + f] : El<T>::from(0.f);
            }
        }
        Tile t = {};
        int it = 0;
        bool ok = true;
        constexpr bool FWD = PASS == PASS_FORWARD;
        const bool with_res = PASS == PASS_FORWARD && p.residual;
        auto accumulators = [&](int half, int it) {  // waits for the tile's products
            if (lane == 0) ok = bar_wait(&tfull[half], (it >> 1) & 1, p.wait_ns, abort);
            ok = __shfl_sync(~0u, (int)ok, 0);
            if (!ok && lane == 0) give_up();
            __syncwarp();
            fence_after();
            return ok;
        };
        auto release = [&](int half) {  // this half of TMEM is free for the tile after next
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive_relaxed_at(leader_addr(&tempty[half]));
        };
        auto write = [&](float* v, float bias, const uint32_t* res, int64_t c, int f, int left) {
            if constexpr (Z) {
                if (with_res) finish<T, ACT, FWD, true, FWD, false>(v, bias, res, p, c, f, left);
                else finish<T, ACT, FWD, true, false, false>(v, bias, res, p, c, f, left);
                if constexpr (SIGNS)
                    if (may_be_near_zero<T>(v, bias, p, f, left)) {
                        unsigned near, zero;
                        near_columns(v, bias, p.K, f < p.F, __ballot_sync(~0u, f < p.F), left, near, zero);
                        if (__any_sync(~0u, near != 0)) settle_signs<T>(near, zero, p, s_near, warp - 4, t.e, (int)c, f, left);
                    }
            } else {
                if (with_res) finish<T, ACT, FWD, false, FWD, false>(v, bias, res, p, c, f, left);
                else if (p.vec && left >= MMA_CHUNK && (f | 31) < p.F) finish<T, ACT, FWD, false, false, true>(v, bias, res, p, c, f, left);
                else finish<T, ACT, FWD, false, false, false>(v, bias, res, p, c, f, left);
            }
        };
        for (int i = 0; ok && fetch(i, t, ok); ++i) {
            const bool product = t.nk > 0;
            const int half = it & 1;
            const int f = t.f0 + rank * MMA_F + 32 * w + lane;
            const float bias = PASS == PASS_FORWARD && p.bias && f < p.F
                                   ? El<T>::to(reinterpret_cast<const T*>(p.bias)[(int64_t)t.e * p.F + f]) : 0.f;
            const int64_t c_base = PASS == PASS_WEIGHT ? (int64_t)t.e * p.C + t.c0 : t.c0;
            uint32_t res[MMA_CHUNK / 2];
            if (with_res) load_residual<T>(res, p, c_base + group * MMA_CHUNK, f, t.nc - group * MMA_CHUNK);
            if (product && !accumulators(half, it)) break;
            for (int c = group * MMA_CHUNK; c < t.nc; c += MMA_GROUPS * MMA_CHUNK) {
                float v[MMA_CHUNK];
                __syncwarp();
                if (product) {
                    tmem_ld16(tmem + ((uint32_t)(32 * w) << 16) + half * MMA_C + c, v);
                } else {
#pragma unroll
                    for (int j = 0; j < MMA_CHUNK; ++j) v[j] = 0.f;
                }
                write(v, bias, res, c_base + c, f, t.nc - c);
                const int next = c + MMA_GROUPS * MMA_CHUNK;
                if (with_res && next < t.nc) load_residual<T>(res, p, c_base + next, f, t.nc - next);
            }
            if (product) release(half);
            it += product;
            if constexpr (SIGNS) {
                if (tid == 128) *(volatile uint32_t*)&s_near.tile = i + 1;
                // (off the tiles' path by now: the other half of TMEM is being filled)
                while (__shfl_sync(~0u, s_near.head[warp - 4] - *(volatile uint32_t*)&s_near.tail[warp - 4], 0) > NEAR_QUEUE / 2)
                    settle_oldest<T>(p, s_near, warp - 4);
            }
        }
        if constexpr (SIGNS) {
            __syncwarp();
            __threadfence_block();
            if (lane == 0) *(volatile int*)&s_near.ended[warp - 4] = 1;
            while (settle_oldest<T>(p, s_near, warp - 4)) {}
        }
    }
    __syncthreads();
    if (s_abort) {  // loads and products in flight end before the CTA gives back its memory
        int never = 0;
        if (tid == 0 && rank == 0) {
            const uint32_t last = s_issued < (uint32_t)p.stages ? s_issued : p.stages;
            for (uint32_t i = s_issued - last; i < s_issued; ++i)
                bar_wait(&full[i % p.stages], (i / p.stages) & 1, p.wait_ns, &never);
        }
        if (tid == 32 && rank == 0) {
            mma_commit(&drained);
            bar_wait(&drained, 0, p.wait_ns, &never);
        }
        if (tid == 0) {  // the other CTA's loads count on barriers that it cannot wait for
            unsigned long long t0, t1;
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
            do asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t1)); while (t1 - t0 < 1000000ull);
        }
        __syncthreads();
    }
    cluster_sync();  // neither CTA leaves while the other may signal it or read its shared memory
    fence_after();
    if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// ------------------------------------------------------------- host side
inline PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    }();
    return fn;
}

// A (d2, d1, d0) tensor of 16-bit elements, strides s1 and s2 in elements, read in
// boxes of b0 x b1 with 128-byte swizzle; what lies outside reads as 0.
inline bool make_map(CUtensorMap* map, int dtype, const void* base, int64_t d0, int64_t d1, int64_t d2, int64_t s1,
                     int64_t s2, int b0, int b1, int rank) {
    const auto fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)d0, (cuuint64_t)d1, (cuuint64_t)d2};
    const cuuint64_t strides[2] = {(cuuint64_t)s1 * 2, (cuuint64_t)s2 * 2};
    const cuuint32_t box[3] = {(cuuint32_t)b0, (cuuint32_t)b1, 1}, step[3] = {1, 1, 1};
    return fn(map, dtype == ELA_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank,
              const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int PASS, typename T, int ACT, bool Z = false>
int mma_launch(const CUtensorMap& a, const CUtensorMap& b, const MmaParams& p, int64_t max_tiles, cudaStream_t st) {
    auto kern = mma_kernel<PASS, T, ACT, Z>;
    const int sms = sm_count();
    if (sms == 0 || !allow_smem<&mma_kernel<PASS, T, ACT, Z>>(MMA_SMEM - 1024)) return ELA_ERR_CUDA;
    const int grid = 2 * (int)(max_tiles < sms / 2 ? max_tiles : sms / 2);
    return launch(kern, grid, MMA_THREADS, MMA_SMEM - 1024, st, a, b, p);
}

// Columns per tile of the row passes, a multiple of 32 up to 256: the one whose rounds of
// tiles over the pairs take least.  A block of 64 k takes the longer of its products (2
// cycles a column) and its loads (16 KB of weights and 64 bytes a column, at the 57
// bytes a cycle that an SM gets from the L2); a tile some 500 cycles more.  300 rows by
// 4096 x 4096: 20.7 us with 64 tiles of 96 columns, 28.4 with 32 of 256; 1500 rows of 4 experts
// of 1000 x 2048 16.8 and 20.0, 3000 of 64 of 1408 x 512 24.0 and 27.2.  Loads are uneven, so an
// expert is taken to have twice its share of the rows; on six such shapes with skewed loads
// that made 140 us in all, one and a half times 139, and the share itself 139.
inline int columns_per_tile(int64_t R, int64_t E, int64_t f_tiles, int64_t k_blocks) {
    const int64_t share = (R + E - 1) / E, rows = E == 1 ? share : 2 * share, pairs = sm_count() / 2 > 0 ? sm_count() / 2 : 1;
    int best = 256;
    int64_t least = INT64_MAX;
    for (int bn = 256; bn >= 32; bn -= 32) {
        const int64_t tiles = f_tiles * (E < R ? E : R) * ((rows + bn - 1) / bn), used = rows < bn ? (rows + 31) / 32 * 32 : bn;
        const int64_t loads = (16384 + 64 * used) / 57, block = 2 * used > loads ? 2 * used : loads;
        const int64_t time = (tiles + pairs - 1) / pairs * (k_blocks * block + 500);
        if (time < least || (time == least && rows <= bn)) { least = time; best = bn; }  // (a smaller stage leaves room for more)
    }
    return best;
}
inline int stages_for(int bn, int64_t E) {
    const int64_t n = (MMA_SMEM - 1024 - MMA_SMEM_FIXED - 12 * E) / (MMA_A_BYTES + bn / 2 * MMA_KB * 2);
    return (int)(n < MMA_MAX_STAGES ? n : MMA_MAX_STAGES);
}

}  // namespace ela_expert
