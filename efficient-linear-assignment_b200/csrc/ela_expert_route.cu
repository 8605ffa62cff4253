// ela_expert_route.cu -- a router's logits to the experts of each token and their
// weights, with the gradient (include/ela_expert.h).
//
// A row of logits belongs to a team of LANES threads, a part of a warp for up to 512
// experts, so that 32 / LANES rows share a warp, and a block of 256 for more.  A thread holds
// VPT consecutive experts in registers; one pass reads the row once, and everything else
// (softmax, groups, choice, weights) stays in registers, shuffles and a little shared memory.
//
// The k largest keys: the k-th largest of the threads' own two largest keys is a bound that at
// least k keys reach, and few others do (one or two for 8 of 256; with each thread's largest
// alone some 30 where groups leave half of the threads without a key).  Those that reach it are put
// side by side in shared memory, in the order of the experts, and each counts the keys above
// it, which is its rank.  8 of 256 experts take a third of the instructions of k rounds of
// "largest key left", each with a search by the thread that had it.
//
// The choice is settled as in 64 bits.  Without a bias a score grows with its logit, so logits
// are compared, which is exact.  Keys that are computed (score + bias, a group's sum) are
// formed in fp32 with a bound on their error; where two keys that decide something lie closer
// than that, the keys in question are formed again in fp64 (with all of the row's where groups
// decide).  That happens in a row of a thousand, and fp64 throughout would cost more than the
// rest of the kernel.
#include "ela_expert.cuh"

#include <type_traits>

namespace ela_expert {

constexpr int ROUTE_THREADS = 128, ROUTE_WIDE = 256;  // threads of a block; of a row's block past 512 experts

struct RouteParams {
    const void* logits;
    int64_t T, ld;
    int E, k, vec, vec_bias;  // vec: rows may be read 16 bytes at a time
    const float* bias;
    int groups, kept, top2;
    int sigmoid, renormalize;
    float scale;
    int32_t* expert;
    float* weights;
};
struct RouteGradParams {
    const void* logits;
    int64_t T, ld;
    int E, k, vec;
    int sigmoid, renormalize;
    float scale;
    const int32_t* expert;
    const float* dweights;
    void* dlogits;
};

// Numbers as unsigned whole numbers in the same order; NaN above all, -0 as 0.  0 is left
// for "not to be chosen".
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);  // (a sum that is NaN is 0x7fffffff)
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t ordered(double x) {
    const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0), top = 1ull << 63;
    return x != x ? ~0ull : b & top ? ~b : b | top;
}
__device__ __forceinline__ float number(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }
__device__ __forceinline__ double number(uint64_t u) {
    const uint64_t top = 1ull << 63;
    return __longlong_as_double((long long)(u & top ? u & ~top : ~u));
}
template <typename F> struct Ordered { typedef uint32_t U; };
template <> struct Ordered<double> { typedef uint64_t U; };

// What the threads of a row do together.  Every thread of the warp (of the block) calls.
template <int LANES> struct Team {
    static constexpr bool WIDE = LANES > 32;
    static constexpr int BLOCK = WIDE ? LANES : ROUTE_THREADS, ROWS = WIDE ? 1 : BLOCK / LANES;  // threads, rows of a block
    static __device__ __forceinline__ int lane() { return threadIdx.x % LANES; }
    static __device__ __forceinline__ int row() { return threadIdx.x / LANES; }
    static __device__ __forceinline__ void sync() { if (WIDE) __syncthreads(); else __syncwarp(); }
    static __device__ __forceinline__ bool any(bool v) { return WIDE ? __syncthreads_or(v) : __any_sync(~0u, v); }

    template <typename V, typename Op> static __device__ __forceinline__ V reduce(V v, Op op) {
#pragma unroll
        for (int o = (WIDE ? 32 : LANES) / 2; o; o >>= 1) v = op(v, __shfl_xor_sync(~0u, v, o));
        if constexpr (WIDE) {
            __shared__ V part[LANES / 32];
            __syncthreads();
            if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
            __syncthreads();
            v = part[0];
            for (int i = 1; i < LANES / 32; ++i) v = op(v, part[i]);
        }
        return v;
    }
    template <typename V> static __device__ __forceinline__ V sum(V v) { return reduce(v, [](V a, V b) { return a + b; }); }
    template <typename V> static __device__ __forceinline__ V most(V v) { return reduce(v, [](V a, V b) { return a > b ? a : b; }); }
    template <typename V> static __device__ __forceinline__ V least(V v) { return reduce(v, [](V a, V b) { return a < b ? a : b; }); }
    static __device__ __forceinline__ uint32_t most(uint32_t v) {
        if constexpr (LANES == 32) return __reduce_max_sync(~0u, v);
        return reduce(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
    }
    // The sum of v over the row's earlier threads, and over all.
    static __device__ __forceinline__ int before(int v, int& all) {
        constexpr int W = WIDE ? 32 : LANES;
        const int mine = v, at = threadIdx.x & (W - 1);
#pragma unroll
        for (int o = 1; o < W; o <<= 1) {
            const int u = __shfl_up_sync(~0u, v, o, W);
            if (at >= o) v += u;
        }
        all = __shfl_sync(~0u, v, W - 1, W);
        int base = 0;
        if constexpr (WIDE) {
            __shared__ int part[LANES / 32];
            __syncthreads();
            if (at == 0) part[threadIdx.x >> 5] = all;
            __syncthreads();
            all = 0;
            for (int i = 0; i < LANES / 32; ++i) {
                if (i == (int)(threadIdx.x >> 5)) base = all;
                all += part[i];
            }
        }
        return base + v - mine;
    }
};

// VPT logits of a row from expert e0 on; -inf past the last expert.
template <typename T, int VPT> __device__ __forceinline__ void load_logits(float* l, const T* row, int e0, int E, bool vec, bool in) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) l[i] = -INFINITY;
    if (!in) return;
    if (vec) {  // (E is a multiple of VPT: all of a thread's experts exist, or none)
        if (e0 < E)
#pragma unroll
            for (int i = 0; i < VPT; i += El<T>::W) {
                const Pack<T> q = *reinterpret_cast<const Pack<T>*>(row + e0 + i);
#pragma unroll
                for (int j = 0; j < El<T>::W; ++j) l[i + j] = El<T>::to(q.v[j]);
            }
    } else {
#pragma unroll
        for (int i = 0; i < VPT; ++i)
            if (e0 + i < E) l[i] = El<T>::to(row[e0 + i]);
    }
}

// A team's shared memory: the chosen experts, their logits and keys; the keys that reach the
// bound with their experts, or before them the values that groups are ranked by (each
// expert's, or each thread's two largest); with groups their ranks' values and the groups kept.
// (One word in 33 of the values unused: threads that walk groups of 32 side by side then hit
// different banks.)
__host__ __device__ inline int route_slot(int e) { return e + (e >> 5); }
struct RouteShared {
    int* at;
    float *logit, *key;
    void* value;       // [slots] keys of up to 8 bytes
    int* value_at;     // [slots]
    void* group;
    unsigned char* kept;
    static __host__ __device__ inline int even(int k) { return (k + 1) / 2 * 2; }
    // (in the gradient: the list alone, slots 0)
    static __host__ __device__ inline int bytes(int slots, int k, int groups) {
        return 12 * even(k) + 12 * slots + (groups > 1 ? 8 * groups + (groups + 7) / 8 * 8 : 0);
    }
    __device__ __forceinline__ RouteShared(unsigned char* p, int slots, int k, int groups) {
        at = reinterpret_cast<int*>(p);
        logit = reinterpret_cast<float*>(p + 4 * even(k));
        key = reinterpret_cast<float*>(p + 8 * even(k));
        p += 12 * even(k);
        value = p;
        value_at = reinterpret_cast<int*>(p + 8 * slots);
        group = p + 12 * slots;
        kept = p + 12 * slots + 8 * groups;
    }
};

// For keys, whose error is allowed for: 2^-22 of the result and |x| 2^-24.
__device__ __forceinline__ float exp_of(float x) { return exp2_fast(x * 1.4426950408889634f); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }
__device__ __forceinline__ float one_over(float x) { return reciprocal_fast(x); }
__device__ __forceinline__ double one_over(double x) { return 1 / x; }

// Two keys that differ by more than this are in the right order (of infinities: that differ).  size: what their
// scores may be off by together; each sum with a bias is off by 2^-24 of itself, and half a step more is for the
// arithmetic here.
__device__ __forceinline__ float apart(float size, float a, float b) {
    return fmaf(fminf(fmaxf(fabsf(a), fabsf(b)), 3.402823466e38f), 1.4901161193847656e-7f, size);
}
// A bound that also those keys reach that may do so in 64 bits.
__device__ __forceinline__ uint32_t lowered(uint32_t bound, float size) { return ordered(number(bound) - apart(size, number(bound), 0.f)); }

// Many keys reach the bound, as in a row of zeros: equal ones, which left the threads' two largest together
// and lowered the bound, perhaps to nothing.  Here they are counted as they leave, and of those
// that equal the first one at the bound in any arithmetic the first k alone stay in the list.  (Kept out of the
// kernel's registers, and of rows of up to 16 experts, whose keys rank as fast.)  8192 x 256 zeros with a bias 31 us, 192 by the ranks of all; 1024 x 4096 zeros 85 and 5530.
template <typename F, typename T, int LANES>
__device__ __noinline__ int route_thin(const RouteParams& p, int all, const T* row, float size, const RouteShared& s) {
    typedef Team<LANES> Tm;
    typedef typename Ordered<F>::U U;
    U* keys = reinterpret_cast<U*>(s.value);
    const int lane = Tm::lane();
    Tm::sync();
    U best = 0, second = 0, bound = 0;
    int taken = 0;
    for (int c = lane; c < all; c += LANES) {
        const U v = keys[c];
        second = v > best ? best : v > second ? v : second;
        best = v > best ? v : best;
    }
    while (true) {
        const U most = Tm::most(best);
        const bool open = taken < p.k && most != 0;
        if (!Tm::any(open)) break;
        if (open) bound = most;
        const bool leaves = open && best == bound;
        taken += Tm::sum((int)leaves);
        if (leaves) { best = second; second = 0; }
    }
    const bool enough = taken >= p.k;  // (else the threads' two largest are fewer than k, and no bound: all stay but the surplus of the last one's equals)
    U low = enough ? bound : 1;
    bool by_key = true;  // equal keys are equal in any arithmetic
    if constexpr (sizeof(F) == 4) {
        if (p.bias && enough) low = lowered(bound, size);
        by_key = !p.bias || !(fabsf(number(bound)) < INFINITY);
    }
    int first = INT32_MAX;
    for (int c = lane; c < all; c += LANES)
        if (keys[c] == bound) { first = s.value_at[c]; break; }
    first = Tm::least(first);  // (INT32_MAX: there are no keys)
    float logit = 0.f, bias = 0.f;
    if (first != INT32_MAX) {
        logit = El<T>::to(row[first]);
        if (p.bias) bias = p.bias[first];
    }
    int twins = 0, kept = 0, some;
    for (int c = lane; Tm::any(c - lane < all); c += LANES) {
        const U v = c < all ? keys[c] : 0;
        const int at = c < all ? s.value_at[c] : 0;
        const bool twin = c < all && v == bound && (by_key || (El<T>::to(row[at]) == logit && p.bias[at] == bias));
        const int rank = twins + Tm::before(twin, some);
        twins += some;
        const bool stays = c < all && v >= low && !(twin && rank >= p.k);
        const int to = kept + Tm::before(stays, some);
        kept += some;
        Tm::sync();
        if (stays) {
            keys[to] = v;
            s.value_at[to] = at;
        }
        Tm::sync();
    }
    return kept;
}

// The ranks of the `all` keys in s.value (into the upper half of their s.value_at), and the k
// experts of the first ranks with their logits and (fp32) keys.
template <typename F, typename T, int LANES>
__device__ __forceinline__ void route_ranks(int k, int all, const T* row, const RouteShared& s) {
    typedef Team<LANES> Tm;
    typedef typename Ordered<F>::U U;
    const U* keys = reinterpret_cast<const U*>(s.value);
    const int lane = Tm::lane();
    for (int j = lane; j < k; j += LANES) s.at[j] = -1;
    Tm::sync();
    for (int c = lane; c < all; c += LANES) {
        const U mine = keys[c];
        const int at = s.value_at[c];
        int rank = 0;
#pragma unroll 4
        for (int d = 0; d < all; ++d) rank += keys[d] > mine - (d < c);  // (of equal keys the first comes first; no key here is 0)
        s.value_at[c] = at | rank << 16;
        if (rank < k) {
            s.at[rank] = at;
            s.logit[rank] = El<T>::to(row[at]);
            if (sizeof(F) == 4) s.key[rank] = number((uint32_t)mine);
        }
    }
    Tm::sync();
}

// The keys in s.value formed again in 64 bits, and ranked.  (Kept out of the kernel's registers.)
template <typename T, int LANES, int VPT>
__device__ __noinline__ void route_settle(const RouteParams& p, int all, const T* row, const float (&l)[VPT], const RouteShared& s) {
    typedef Team<LANES> Tm;
    double m = 0, sum = 1;
    if (!p.sigmoid) {
        float most = -INFINITY;
#pragma unroll
        for (int i = 0; i < VPT; ++i) most = fmaxf(most, l[i]);
        m = Tm::most(most);
        sum = 0;
        for (int i = 0; i < VPT; ++i) sum += l[i] == -INFINITY ? 0 : exp((double)l[i] - m);
        sum = Tm::sum(sum);
    }
    Tm::sync();
    uint64_t* keys = reinterpret_cast<uint64_t*>(s.value);
    for (int c = Tm::lane(); c < all; c += LANES) {
        const int at = s.value_at[c] & 0xffff;
        const double x = El<T>::to(row[at]);
        keys[c] = ordered((p.sigmoid ? 1 / (1 + exp(-x)) : exp(x - m) / sum) + (double)p.bias[at]);
        s.value_at[c] = at;
    }
    Tm::sync();
    route_ranks<double, T, LANES>(p.k, all, row, s);
}

// Chooses the row's experts, in F, and leaves them in s, with their logits and (in fp32) keys.  True: the choice is
// not sure in fp32 (F double is always sure).
template <typename F, typename T, int LANES, int VPT>
__device__ __forceinline__ bool route_choose(const RouteParams& p, const T* row, const float (&l)[VPT], const RouteShared& s) {
    typedef Team<LANES> Tm;
    typedef typename Ordered<F>::U U;
    constexpr bool CHECK = sizeof(F) == 4;
    const int lane = Tm::lane(), e0 = lane * VPT;
    const bool computed = p.bias != nullptr;             // keys are scores and a bias, not logits
    const bool scores = computed || p.top2;
    float bias[VPT];
    if (computed) load_logits<float, VPT>(bias, p.bias, e0, p.E, p.vec_bias, true);
    F value[VPT];                                        // score + bias
    F size = 0;                                          // what two keys' scores may be off by together
    if (scores) {
        F m = 0, inv = 0;
        if (!p.sigmoid) {
            float most = -INFINITY;
#pragma unroll
            for (int i = 0; i < VPT; ++i) most = fmaxf(most, l[i]);
            m = Tm::most(most);
            if (m == -INFINITY) m = 0;  // (a row without experts)
        }
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            value[i] = p.sigmoid ? one_over(1 + exp_of(-(F)l[i])) : exp_of((F)l[i] - m);
            if (!p.sigmoid) inv += value[i];
        }
        if (!p.sigmoid) inv = one_over(Tm::sum(inv));
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            if (!p.sigmoid) value[i] *= inv;
            if (CHECK) size = value[i] > size ? value[i] : size;
            if (computed && e0 + i < p.E) value[i] += bias[i];
        }
        // A sigmoid's exponential is off by (1.5 |x| + 4) 2^-24 of itself (its exponent's rounding, its own error),
        // which moves the sigmoid by 1 - s of that, and the sum and the reciprocal move it by 3 * 2^-24.  For
        // x >= 0 that makes 3.4 * 2^-24, 5 * 2^-24 of the row's largest score S at most; below 0, where both the
        // score and its error grow with x, (1.5 |x| (1 - S) + 4 (1 - S) + 3) 2^-24 of S for the largest x.  Where S lies
        // in [2^e, 2^(e+1)), |x| is at most -0.7 e, and (5.6 + 2 (-1 - e)) 2^-24 of S is more for every e; it never
        // passes 3.4 * 2^-24.  A score below 2^-126 comes out as 0.  A softmax is off by 2^-22 of the largest for its exponential, and by the row's
        // sum, at most 29 additions one after the other of such terms, 2^-19; two of them by 2^-17.  A sum with
        // the bias is off by another 2^-24 of itself, which is allowed for key by key: one bias of -1e9
        // for an expert that is out of the question leaves the others their digits (by the row's largest
        // value every one was in doubt: 8192 x 256 took 120 and 260 us with and without groups, usual ones 17 and 14).
        if (CHECK) {
            size = Tm::most(size);
            const float below = (float)(126 - (int)(__float_as_uint((float)size) >> 23));  // -1 - e
            size = p.sigmoid ? fmaf(fminf((float)size * (5.6f + 2.f * fmaxf(below, 0.f)), 3.45f), 1.1920928955078125e-7f, 2.3509887e-38f) : size * (F)7.62939453125e-6;
        }
    }
    U key[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const bool there = l[i] != -INFINITY && !(computed && bias[i] == -INFINITY);  // (past the last expert both are)
        if (scores && !there) value[i] = -INFINITY;
        key[i] = there ? ordered(computed ? value[i] : (F)l[i]) : 0;
    }
    bool unsure = false;
    if (p.groups > 1) {
        U* vals = reinterpret_cast<U*>(s.value);
        U* group = reinterpret_cast<U*>(s.group);
        float* off = reinterpret_cast<float*>(group + p.groups);  // (in fp32, whose keys leave half of the place)
        const int S = p.E / p.groups;
        auto join = [](U v, U& a, U& b) {  // the largest and the second
            b = v > a ? a : v > b ? v : b;
            a = v > a ? v : a;
        };
        const bool whole = S % VPT == 0;  // a thread's experts are of one group: it joins them first
        U a = 0, b = 0;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const U v = p.top2 ? ordered(value[i]) : key[i] ? key[i] : ordered((F)-INFINITY);
            if (whole) join(v, a, b);
            else if (e0 + i < p.E) vals[route_slot(e0 + i)] = v;
        }
        if (whole && e0 < p.E) { vals[2 * lane] = a; vals[2 * lane + 1] = b; }
        Tm::sync();
        const int per = whole ? S / VPT * 2 : S;
        for (int g = lane; g < p.groups; g += LANES) {
            a = b = 0;
            for (int i = 0; i < per; ++i) join(vals[whole ? g * per + i : route_slot(g * per + i)], a, b);
            auto sum = number(a) + number(b);
            if (CHECK && p.top2 && fabsf(sum) == INFINITY && fabsf(number((uint32_t)a)) < INFINITY && fabsf(number((uint32_t)b)) < INFINITY)
                sum = sum > 0 ? 3.402823466e38f : -3.402823466e38f;  // (no infinity in 64 bits: in order with those, in doubt with its like)
            group[g] = p.top2 ? ordered(sum) : a;
            if (CHECK && scores) {  // what it may be off by: its two keys, and their sum
                const float x = number((uint32_t)a), y = p.top2 ? number((uint32_t)b) : 0.f;
                off[g] = (p.top2 ? 1.f : 0.5f) * (float)size + (fabsf(x) + fabsf(y) + (p.top2 ? fabsf(x + y) : 0.f)) * 5.9604708e-8f;
            }
        }
        Tm::sync();
        float last = INFINITY, next = -INFINITY;  // the least that a kept group may be, the most that one left out may be
        for (int g = lane; g < p.groups; g += LANES) {
            const U v = group[g];
            int before = 0;
            for (int h = 0; h < p.groups; ++h) before += group[h] > v || (group[h] == v && h < g);
            s.kept[g] = before < p.kept;
            if (CHECK && scores) {  // (an infinite sum is off by infinity: no doubt where closed groups, -inf, are left out)
                const float x = number((uint32_t)v);
                if (before < p.kept) last = fminf(last, __fsub_rd(x, off[g]));
                else next = fmaxf(next, __fadd_ru(x, off[g]));
            }
        }
        Tm::sync();
        if (CHECK && scores) {
            last = Tm::least(last);
            next = Tm::most(next);
            unsure = next > -INFINITY && last <= next;
        }
        int g = e0 / S, r = e0 - g * S;
        if (whole) {
            const bool stays = e0 < p.E && s.kept[g];
#pragma unroll
            for (int i = 0; i < VPT; ++i) key[i] = stays ? key[i] : 0;
        } else {
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                if (e0 + i < p.E && !s.kept[g]) key[i] = 0;
                if (++r == S) { r = 0; ++g; }
            }
        }
    }
    // the bound: the k-th of the threads' two largest keys each (equal ones leave together, which lowers it)
    U best = key[0], second = 0;
#pragma unroll
    for (int i = 1; i < VPT; ++i) {
        const U less = key[i] < best ? key[i] : best;
        second = less > second ? less : second;
        best = key[i] > best ? key[i] : best;
    }
    U bound = 0;
    for (int j = 0; j < p.k; ++j) {
        bound = Tm::most(best);
        if (best == bound) { best = second; second = 0; }
        if (LANES <= 32 && j >= 2 * LANES) break;  // (none left)
    }
    if (CHECK && computed && bound != 0) bound = lowered(bound, (float)size);
    if (bound == 0) bound = 1;
    int reach = 0, all;
#pragma unroll
    for (int i = 0; i < VPT; ++i) reach += key[i] >= bound;
    int to = Tm::before(reach, all);
    U* keys = reinterpret_cast<U*>(s.value);
#pragma unroll
    for (int i = 0; i < VPT; ++i)
        if (key[i] >= bound) {
            keys[to] = key[i];
            s.value_at[to++] = e0 + i;
        }
    constexpr int MANY = LANES < 16 ? 4 * LANES : 64;
    if (LANES >= 4 && Tm::any(all > MANY + 2 * p.k)) all = route_thin<F, T, LANES>(p, all, row, (float)size, s);
    route_ranks<F, T, LANES>(p.k, all, row, s);
    if (CHECK && computed) {
        auto same = [&](int a, int b) { return El<T>::to(row[a]) == El<T>::to(row[b]) && p.bias[a] == p.bias[b]; };  // equal keys in any arithmetic
        bool doubt = false;
        for (int c = lane; c < all; c += LANES) {  // each against the choice before it, or the last one
            const int rank = s.value_at[c] >> 16, at = s.value_at[c] & 0xffff, prev = min(rank, p.k) - 1;
            if (prev >= 0) doubt |= s.key[prev] - number(keys[c]) <= apart((float)size, s.key[prev], number(keys[c])) && !same(s.at[prev], at);
        }
        if (Tm::any(doubt)) route_settle<T, LANES, VPT>(p, all, row, l, s);
    }
    return unsure;
}

// 64 bits throughout, for the rows whose groups need them (kept out of the kernel's registers).
template <typename T, int LANES, int VPT>
__device__ __noinline__ void route_again(const RouteParams& p, const T* row, const float (&l)[VPT], const RouteShared& s) {
    Team<LANES>::sync();
    route_choose<double, T, LANES, VPT>(p, row, l, s);
}

// Weights of the chosen experts, in place of their logits.  Ratios of the chosen scores are
// formed from the exponents' differences, so that none is 0 / 0 however small the scores.
template <int LANES, int VPT>
__device__ __forceinline__ void route_weights(const RouteParams& p, const float (&l)[VPT], const RouteShared& s) {
    typedef Team<LANES> Tm;
    const int lane = Tm::lane();
    if (p.renormalize) {
        float most = -INFINITY, sum = 0.f;
        for (int j = lane; j < p.k; j += LANES)
            if (s.at[j] >= 0) most = fmaxf(most, p.sigmoid ? fminf(s.logit[j], 0.f) : s.logit[j]);
        most = Tm::most(most);
        auto part = [&](float x) { return p.sigmoid ? expf(fminf(x, 0.f) - most) / (1.f + expf(-fabsf(x))) : expf(x - most); };
        for (int j = lane; j < p.k; j += LANES)
            if (s.at[j] >= 0) sum += s.logit[j] = part(s.logit[j]);
        sum = Tm::sum(sum);
        if (!p.sigmoid && (p.bias || p.top2)) {  // a NaN or +inf that was not chosen: every score of its row is NaN
            float spoiled = 0.f;
#pragma unroll
            for (int i = 0; i < VPT; ++i) spoiled = l[i] < INFINITY ? spoiled : NAN;
            sum += Tm::sum(spoiled);
        }
        for (int j = lane; j < p.k; j += LANES) s.logit[j] = s.at[j] >= 0 ? p.scale * (s.logit[j] / sum) : 0.f;
    } else {
        float most = -INFINITY, sum = 0.f;
        if (!p.sigmoid) {
#pragma unroll
            for (int i = 0; i < VPT; ++i) most = fmaxf(most, l[i]);
            most = Tm::most(most);
            if (most == -INFINITY) most = 0.f;
#pragma unroll
            for (int i = 0; i < VPT; ++i) sum += expf(l[i] - most);
            sum = Tm::sum(sum);
        }
        for (int j = lane; j < p.k; j += LANES) {
            const float x = s.logit[j];
            s.logit[j] = s.at[j] < 0 ? 0.f : p.scale * (p.sigmoid ? 1.f / (1.f + expf(-x)) : expf(x - most) / sum);
        }
    }
    Tm::sync();
}

template <typename T, int LANES, int VPT>
__global__ void __launch_bounds__(Team<LANES>::BLOCK) route_kernel(const __grid_constant__ RouteParams p) {
    next_may_start();
    previous_done();
    typedef Team<LANES> Tm;
    extern __shared__ __align__(16) unsigned char shared[];
    const int64_t t = (int64_t)blockIdx.x * Tm::ROWS + Tm::row();
    const int bytes = RouteShared::bytes(LANES * VPT, p.k, p.groups);
    const RouteShared s(shared + Tm::row() * bytes, LANES * VPT, p.k, p.groups);
    float l[VPT];
    const T* row = reinterpret_cast<const T*>(p.logits) + (t < p.T ? t : 0) * p.ld;
    load_logits<T, VPT>(l, row, Tm::lane() * VPT, p.E, p.vec, t < p.T);
    if (Tm::any(route_choose<float, T, LANES, VPT>(p, row, l, s))) route_again<T, LANES, VPT>(p, row, l, s);
    route_weights<LANES, VPT>(p, l, s);
    if (t < p.T)
        for (int j = Tm::lane(); j < p.k; j += LANES) {
            p.expert[t * p.k + j] = s.at[j];
            p.weights[t * p.k + j] = s.logit[j];
        }
}

// Gradient.  With c_j = scale * dw_j and r_j the chosen ratios (p_i the softmax):
//   softmax           dl_i = p_i (c_i - sum_j c_j p_j), c_i = 0 where i is not chosen
//   softmax, ratios   dl_j = r_j (c_j - sum_j c_j r_j)
//   sigmoid           dl_j = c_j s_j (1 - s_j)
//   sigmoid, ratios   dl_j = r_j (c_j - sum_j c_j r_j) (1 - s_j)
// Only the first reads the whole row.  A choice outside [0, E) has no gradient.
template <typename T, int LANES, int VPT>
__global__ void __launch_bounds__(Team<LANES>::BLOCK) route_grad_kernel(const __grid_constant__ RouteGradParams p) {
    next_may_start();
    previous_done();
    typedef Team<LANES> Tm;
    extern __shared__ __align__(16) unsigned char shared[];
    const int lane = Tm::lane(), e0 = lane * VPT;
    const int64_t t = (int64_t)blockIdx.x * Tm::ROWS + Tm::row();
    const RouteShared s(shared + Tm::row() * RouteShared::bytes(0, p.k, 1), 0, p.k, 1);
    const T* row = reinterpret_cast<const T*>(p.logits) + (t < p.T ? t : 0) * p.ld;
    const bool dense = !p.sigmoid && !p.renormalize;
    float l[VPT], most = -INFINITY, sum = 0.f, mean = 0.f;
    if (dense) {
        load_logits<T, VPT>(l, row, e0, p.E, p.vec, t < p.T);
#pragma unroll
        for (int i = 0; i < VPT; ++i) most = fmaxf(most, l[i]);
        most = Tm::most(most);
        if (most == -INFINITY) most = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) sum += l[i] = expf(l[i] - most);
        sum = Tm::sum(sum);
#pragma unroll
        for (int i = 0; i < VPT; ++i) l[i] = sum > 0.f || sum != sum ? l[i] / sum : 0.f;
    }
    // the chosen experts, and what each adds to its logit's gradient
    for (int j = lane; j < p.k; j += LANES) {
        const int e = t < p.T ? p.expert[t * p.k + j] : -1;
        s.at[j] = e >= 0 && e < p.E ? e : -1;
        if (s.at[j] >= 0) {
            s.logit[j] = El<T>::to(row[e]);
            if (p.renormalize) most = fmaxf(most, p.sigmoid ? fminf(s.logit[j], 0.f) : s.logit[j]);
        }
    }
    if (p.renormalize) {
        most = Tm::most(most);
        for (int j = lane; j < p.k; j += LANES)
            if (s.at[j] >= 0) sum += p.sigmoid ? expf(fminf(s.logit[j], 0.f) - most) / (1.f + expf(-fabsf(s.logit[j]))) : expf(s.logit[j] - most);
        sum = Tm::sum(sum);
    }
    auto ratio = [&](float x) {  // the weight, without scale
        if (p.sigmoid) return p.renormalize ? expf(fminf(x, 0.f) - most) / (1.f + expf(-fabsf(x))) / sum : 1.f / (1.f + expf(-x));
        return expf(x - most) / sum;
    };
    // (rounded by itself: joined with the subtraction of the mean it left 2^-24 of a gradient that is 0)
    auto weighted = [&](int j) { return __fmul_rn(p.scale, p.dweights[t * p.k + j]); };
    if (!p.sigmoid || p.renormalize) {
        for (int j = lane; j < p.k; j += LANES)
            if (s.at[j] >= 0) mean = fmaf(weighted(j), ratio(s.logit[j]), mean);
        mean = Tm::sum(mean);
    }
    for (int j = lane; j < p.k; j += LANES)
        if (s.at[j] >= 0) {
            const float x = s.logit[j], c = weighted(j);
            s.logit[j] = dense ? c : ratio(x) * (c - mean) * (p.sigmoid ? 1.f / (1.f + expf(x)) : 1.f);
        }
    Tm::sync();
    float d[VPT] = {};
    for (int j = 0; j < p.k; ++j) {
        const int at = s.at[j];
#pragma unroll
        for (int i = 0; i < VPT; ++i)
            if (e0 + i == at) d[i] += s.logit[j];
    }
    if (dense)
#pragma unroll
        for (int i = 0; i < VPT; ++i) d[i] = l[i] * (d[i] - mean);
    if (t >= p.T) return;
    T* out = reinterpret_cast<T*>(p.dlogits) + t * p.E;
    if (p.vec) {
        if (e0 < p.E)
#pragma unroll
            for (int i = 0; i < VPT; i += El<T>::W) {
                Pack<T> q;
#pragma unroll
                for (int j = 0; j < El<T>::W; ++j) q.v[j] = El<T>::from(d[i + j]);
                *reinterpret_cast<Pack<T>*>(out + e0 + i) = q;
            }
    } else {
#pragma unroll
        for (int i = 0; i < VPT; ++i)
            if (e0 + i < p.E) out[e0 + i] = El<T>::from(d[i]);
    }
}

template <typename T, int LANES, int VPT> int route_launch(const RouteParams& p, cudaStream_t st) {
    typedef Team<LANES> Tm;
    const int bytes = Tm::ROWS * RouteShared::bytes(LANES * VPT, p.k, p.groups);
    const int64_t blocks = (p.T + Tm::ROWS - 1) / Tm::ROWS;
    if (blocks > INT32_MAX) return ELA_ERR_UNSUPPORTED;
    if (bytes > 48 * 1024 && !allow_smem<&route_kernel<T, LANES, VPT>>(100 * 1024)) return ELA_ERR_CUDA;
    return launch(route_kernel<T, LANES, VPT>, (unsigned)blocks, Tm::BLOCK, bytes, st, p);
}
template <typename T, int LANES, int VPT> int route_launch(const RouteGradParams& p, cudaStream_t st) {
    typedef Team<LANES> Tm;
    const int64_t blocks = (p.T + Tm::ROWS - 1) / Tm::ROWS;
    if (blocks > INT32_MAX) return ELA_ERR_UNSUPPORTED;
    return launch(route_grad_kernel<T, LANES, VPT>, (unsigned)blocks, Tm::BLOCK, Tm::ROWS * RouteShared::bytes(0, p.k, 1), st, p);
}

// Eight experts a thread, so that a row of 16-bit logits is one load each, on as few threads
// as that takes; sixteen past 128 experts.
template <typename T, typename P> int route_by_size(P p, cudaStream_t st) {
    const int per = p.E <= 128 ? 8 : 16;
    p.vec = p.vec && p.E % per == 0;
    if constexpr (std::is_same_v<P, RouteParams>) p.vec_bias = p.vec_bias && p.E % per == 0;
    return p.E <= 8 ? route_launch<T, 1, 8>(p, st) : p.E <= 16 ? route_launch<T, 2, 8>(p, st) : p.E <= 32 ? route_launch<T, 4, 8>(p, st)
         : p.E <= 64 ? route_launch<T, 8, 8>(p, st) : p.E <= 128 ? route_launch<T, 16, 8>(p, st) : p.E <= 256 ? route_launch<T, 16, 16>(p, st)
         : p.E <= 512 ? route_launch<T, 32, 16>(p, st) : route_launch<T, ROUTE_WIDE, 16>(p, st);
}
template <typename P> int route_by_type(const P& p, int dtype, cudaStream_t st) {
    return dtype == ELA_DTYPE_F32 ? route_by_size<float>(p, st) : dtype == ELA_DTYPE_F16 ? route_by_size<__half>(p, st) : route_by_size<__nv_bfloat16>(p, st);
}

inline bool route_sizes_ok(int dtype, int64_t T, int64_t E, int64_t ld, int64_t k, int score, float scale) {
    return dtype_bytes(dtype) != 0 && T >= 0 && E >= 1 && E <= ELA_EXPERT_MAX && ld >= 0 && k >= 1 && k <= E && k <= ELA_ROUTE_MAX_K &&
           T <= INT32_MAX / k && (score == ELA_SCORE_SOFTMAX || score == ELA_SCORE_SIGMOID) && scale - scale == 0.f;
}

}  // namespace ela_expert

using namespace ela_expert;

extern "C" {

int ela_expert_route(const void* logits, int dtype, int64_t T, int64_t E, int64_t ld, int64_t k, int score,
                     const float* bias, int64_t groups, int64_t groups_kept, int group_score, int renormalize,
                     float scale, int32_t* expert, float* weights, void* stream) {
    if (!route_sizes_ok(dtype, T, E, ld, k, score, scale) || groups < 1 || E % groups != 0 || groups_kept < 1 ||
        groups_kept > groups || k > groups_kept * (E / groups) ||
        (group_score != ELA_GROUP_MAX && group_score != ELA_GROUP_TOP2) || (groups > 1 && group_score == ELA_GROUP_TOP2 && E / groups < 2))
        return ELA_ERR_ARGUMENT;
    if (T == 0) return ELA_OK;
    if (!logits || !expert || !weights || !on_elements(dtype_bytes(dtype), logits) || !on_elements(4, bias, expert, weights)) return ELA_ERR_ARGUMENT;
    if (groups == groups_kept) groups = groups_kept = 1;  // all stay
    RouteParams p = {logits, T, ld, (int)E, (int)k, aligned16(logits, ld * dtype_bytes(dtype)), aligned16(bias), bias, (int)groups, (int)groups_kept,
                     groups > 1 && group_score == ELA_GROUP_TOP2, score == ELA_SCORE_SIGMOID, renormalize != 0, scale, expert, weights};
    return route_by_type(p, dtype, reinterpret_cast<cudaStream_t>(stream));
}

int ela_expert_route_grad(const void* logits, int dtype, int64_t T, int64_t E, int64_t ld, int64_t k, int score,
                          int renormalize, float scale, const int32_t* expert, const float* dweights, void* dlogits,
                          void* stream) {
    if (!route_sizes_ok(dtype, T, E, ld, k, score, scale)) return ELA_ERR_ARGUMENT;
    if (T == 0) return ELA_OK;
    if (!logits || !expert || !dweights || !dlogits || !on_elements(dtype_bytes(dtype), logits, dlogits) || !on_elements(4, expert, dweights))
        return ELA_ERR_ARGUMENT;
    const int size = dtype_bytes(dtype);
    RouteGradParams p = {logits, T, ld, (int)E, (int)k, aligned16(logits, ld * size) && aligned16(dlogits, E * size), score == ELA_SCORE_SIGMOID,
                         renormalize != 0, scale, expert, dweights, dlogits};
    return route_by_type(p, dtype, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
