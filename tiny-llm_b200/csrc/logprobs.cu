// Log probabilities of given tokens, entropy and largest alternatives of rows
// of logits, sm_100a. With z_j = (x_j - max x) / T and l = sum_j exp z_j:
//   logprob(t) = z_t - log l
//   entropy    = log l - (sum_j z_j exp z_j) / l
//   top        = the largest x_j, equal ones by their index
// One pass over a row: every thread keeps the maximum of its elements and,
// relative to it, the two sums (fp32, base 2), rescaled when the maximum
// grows, so the row is read from HBM once and nothing of it is kept. Many
// rows run near the stream: 2048 x 128256 without alternatives 92 us in fp16
// (packed arithmetic), 98 in bf16 (0.87 and 0.82 of the measured copy rate),
// 1024 rows of fp32 80 us (1.0). Rows too few to fill the machine are split
// over the CTAs of a cluster, which join in distributed shared memory.
//
// The alternatives add little to the pass: of the maxima of 8 to 128 groups
// of threads the n-th largest is a lower bound of the n-th largest logit, and
// only threads whose own maximum reaches it can hold one of the n. What comes
// after the pass is serial, and with few or short rows most of the call: their
// elements are looked at again (in registers where they fit, else those
// batches whose maximum, kept in shared memory, reaches the bound, from L2),
// the ones that reach the bound are listed and ranked by counting, a long list
// after a cut. One row of 128256 fp16 logits takes 4.9 us without
// alternatives, 8.0 with 5, 10.2 with 20, 16.8 with 64.
// A list that overflows is replaced by n searches of the slice for the largest
// element behind the last one found. Thousands of equal logits bring that
// about, a finite mask value that leaves fewer tokens than alternatives among
// them: 300 rows of 128256 with five tokens over the type's lowest value, 20
// alternatives, take 1.18 ms; with -inf in the mask's place 0.05.
//
// Sums are combined in a fixed order: a row's result does not depend on
// timing.
#include <algorithm>
#include <cfloat>
#include <cooperative_groups.h>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>

#include "kernels.h"
#include "ptx.cuh"

namespace tllm {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxTop = kLogprobMaxTop;
constexpr int kCand = 1024;
constexpr int kSlots = 16;             // of a thread's batches' maxima: 128256 fp32 logits in 256 threads
constexpr int kRank = 160;             // candidates ranked without a cut; above kMaxTop
constexpr int kMaxCluster = 8;
constexpr int kMaxWarps = 16;
constexpr int kMaxGroups = 128;        // of threads, for the bound; at least kMaxTop

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// 16 bytes of logits: values in fp32 and their maximum (NaN if one is).
template <typename T>
struct Vec;
template <>
struct Vec<__half> {
    static constexpr int kN = 8;
    static __device__ __forceinline__ void load(const uint4 &v, float (&f)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 t = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            f[2 * i] = t.x;
            f[2 * i + 1] = t.y;
        }
    }
    static __device__ __forceinline__ float max(const uint4 &v) {
        const __half2 *h = reinterpret_cast<const __half2 *>(&v);
        const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
        return max_nan(__low2float(m), __high2float(m));
    }
    static __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
    // Whether the packed pass holds, relative to a maximum m. An element at the
    // type's lowest value has to weigh nothing: then -inf may be taken for it,
    // which keeps every z finite without a comparison in fp32 for each. And
    // m c, rounded once for all elements, may be off by a half at most (below
    // 2^24 fp32's unit is one or less): the factor that puts the rounding
    // right, 2^shift, stays within [0.7, 1.42]. At a temperature of 1e-5 m c
    // reaches 9.4e9 and shift 432, whose power no fp32 number holds.
    static __device__ __forceinline__ bool packed_pass(float m, float c) {
        return (m + 65504.f) * c > 160.f && fabsf(m * c) < 16777216.f;
    }
    static __device__ __forceinline__ uint4 raise(uint4 v) {
        const __half2 low = __halves2half2(__ushort_as_half(0xFBFF), __ushort_as_half(0xFBFF));
        __half2 *h = reinterpret_cast<__half2 *>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __hmax2(h[i], low);
        return v;
    }
};
template <>
struct Vec<__nv_bfloat16> {
    static constexpr int kN = 8;
    static __device__ __forceinline__ void load(const uint4 &v, float (&f)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ float max(const uint4 &v) {
        const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&v);
        const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
        return max_nan(__low2float(m), __high2float(m));
    }
    static __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
    // (z of the lowest value is not finite for every c: clamped one by one)
    static __device__ __forceinline__ bool packed_pass(float, float) { return false; }
    static __device__ __forceinline__ uint4 raise(uint4 v) { return v; }
};
template <>
struct Vec<float> {
    static constexpr int kN = 4;
    static __device__ __forceinline__ void load(const uint4 &v, float (&f)[4]) {
        f[0] = __uint_as_float(v.x);
        f[1] = __uint_as_float(v.y);
        f[2] = __uint_as_float(v.z);
        f[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ float max(const uint4 &v) {
        return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)),
                       max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
    }
    static __device__ __forceinline__ float to_float(float v) { return v; }
    // (z of the lowest value is not finite for every c: clamped one by one)
    static __device__ __forceinline__ bool packed_pass(float, float) { return false; }
    static __device__ __forceinline__ uint4 raise(uint4 v) { return v; }
};

// Sums of a set of elements relative to their maximum m: l = sum 2^z and
// t = sum z 2^z with z = (x - m) c, c = log2(e) / T. An empty set, and one of
// -inf alone, has m = -inf, l = t = 0.
struct Sums {
    float m, l, t;
};

// z of x. -inf (a masked logit, a thread that has seen nothing), and what is
// far below, is held finite, so that 2^z = 0 and z 2^z = 0. kHalves, for c
// below kFlat (T above 1.4e36): x - m may pass fp32's range where (x - m) c
// does not, so it is taken by halves, which are exact and one FMA. From kFlat
// on such a difference is 340 and more in z and its weight 0 either way. Two
// instances of the kernel, since the FMA in place of the addition takes 8 %
// more (2048 x 128256 bf16 103 us instead of 96), a branch per batch as much.
constexpr float kFlat = 1e-36f;
template <bool kHalves>
__device__ __forceinline__ float z_of(float x, float m, float c) {
    return fmaxf(kHalves ? fmaf(x, 0.5f, -0.5f * m) * (2.f * c) : (x - m) * c, -1e30f);
}

// Moves s to the maximum m >= s.m.
template <bool kHalves>
__device__ __forceinline__ void rebase(Sums &s, float m, float c) {
    if (m == s.m) return;
    const float d = z_of<kHalves>(s.m, m, c), f = ptx::ex2(d);  // (nothing yet: l = t = 0 stay)
    s.t = f * fmaf(d, s.l, s.t);
    s.l *= f;
    s.m = m;
}

template <bool kHalves>
__device__ __forceinline__ Sums join(Sums a, Sums b, float c) {
    const float m = max_nan(a.m, b.m);
    rebase<kHalves>(a, m, c);
    rebase<kHalves>(b, m, c);
    return {m, a.l + b.l, a.t + b.t};
}

template <bool kHalves>
__device__ __forceinline__ void add(Sums &s, float x, float c) {
    const float z = z_of<kHalves>(x, s.m, c);
    const float e = ptx::ex2(z);
    s.l += e;
    s.t = fmaf(e, z, s.t);
}

// Two elements at a time, z by one packed FMA. nmc: -m c rounded once; what
// that rounding shifts every z by (packed_pass keeps it to a half) is put right
// at the end of each batch.
struct Sums2 {
    uint64_t l, t;
};
__device__ __forceinline__ void add2(Sums2 &s, float x0, float x1, uint64_t c2, uint64_t nmc2) {
    float z0, z1;
    ptx::f2_unpack(ptx::f2_fma(ptx::f2_pack(x0, x1), c2, nmc2), z0, z1);
    const uint64_t e = ptx::f2_pack(ptx::ex2(z0), ptx::ex2(z1));
    s.l = ptx::f2_add(s.l, e);
    s.t = ptx::f2_fma(e, ptx::f2_pack(z0, z1), s.t);
}

struct Best {
    float v;
    int i;
};
// Order of the alternatives: larger first, equal ones by index.
__device__ __forceinline__ bool before(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

struct Shared {
    Sums sums[kMaxWarps];
    Sums cta;                 // read by the cluster
    float gmax[kMaxGroups];
    float bound;
    int count;
    int found;                // entries of list
    Best list[kMaxTop];       // read by the cluster
    Best cand[kCand];         // candidates; then the cluster's lists
    Best red[kMaxWarps];
    int rank[kMaxCluster * kMaxTop];
    int tally[2][kMaxWarps];
};
static_assert(kMaxCluster * kMaxTop <= kCand, "the cluster's lists fit the candidates' place");

// kThreads: 512 where few CTAs share the device, 256 (four CTAs an SM) where
// the end of one row has to hide behind the passes of others.
template <typename T, int kThreads, bool kHalves>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) logprobs_kernel(const __grid_constant__ LogprobArgs a) {
    constexpr int N = Vec<T>::kN, kWarps = kThreads / 32;
    constexpr int kU = kThreads == 256 ? 8 : 4;  // vectors in flight per thread
    __shared__ Shared sh;
    __shared__ float batch_max[kSlots][kThreads];  // of a thread's batches b, b + kSlots, ...
    // Programmatic dependent launch: the kernel before may have written the
    // logits while this one was already started, so they are read by coherent
    // loads (ld.global.nc is for what no one writes in a kernel's lifetime),
    // and the next kernel is let in only after the wait: nothing older than
    // this kernel runs beside it.
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = a.split, rank = blockIdx.x % split;
    const int row = blockIdx.x / split;
    const T *x = static_cast<const T *>(a.logits) + (long long)row * a.row_stride;
    // this CTA's slice [lo, hi) of the row, and in it the 16-byte aligned part
    const int lo = (int)((long long)rank * a.vocab / split), hi = (int)((long long)(rank + 1) * a.vocab / split);
    const int mis = (int)((reinterpret_cast<uintptr_t>(x + lo) & 15) / sizeof(T));
    const int head = min(hi - lo, mis ? N - mis : 0);
    const int nvec = (hi - lo - head) / N;
    const uint4 *xv = reinterpret_cast<const uint4 *>(x + lo + head);
    const int tail0 = lo + head + nvec * N;  // [tail0, hi): what is left, < N elements
    const float c = a.scale_log2;

    if (tid == 0) {
        sh.count = 0;
        sh.bound = INFINITY;  // stays where a NaN leaves no group of the rank below
    }
    // elements that no vector holds: thread j < head has lo + j, thread 32 + j the tail's
    int single = -1;
    if (tid < head) single = lo + tid;
    if (tid >= 32 && tid - 32 < hi - tail0) single = tail0 + tid - 32;

    Sums s = {-INFINITY, 0.f, 0.f};
    float own = -INFINITY;  // the thread's maximum
    if (single >= 0) {
        const float v = Vec<T>::to_float(x[single]);
        own = v;
        rebase<kHalves>(s, max_nan(fmaxf(v, -FLT_MAX), v), c);
        add<kHalves>(s, v, c);
    }
    const bool once = nvec <= kThreads * kU;  // one round: the elements stay in registers
    uint4 v[kU];
    int batches = 0;
    for (int i0 = tid; i0 < nvec; i0 += kThreads * kU, ++batches) {
#pragma unroll
        for (int u = 0; u < kU; ++u)
            if (i0 + u * kThreads < nvec) v[u] = __ldcg(xv + i0 + u * kThreads);
        float m = -INFINITY;
#pragma unroll
        for (int u = 0; u < kU; ++u)
            if (i0 + u * kThreads < nvec) m = max_nan(m, Vec<T>::max(v[u]));
        own = max_nan(own, m);
        if (!once && a.top > 0) {
            float *slot = &batch_max[batches % kSlots][tid];
            *slot = batches < kSlots ? m : max_nan(*slot, m);
        }
        // a batch of -inf alone moves the maximum to -FLT_MAX, not to -inf:
        // differences to it stay numbers
        rebase<kHalves>(s, max_nan(s.m, max_nan(m, -FLT_MAX)), c);
        if (Vec<T>::packed_pass(s.m, c)) {
            const float nmc = -s.m * c, shift = fmaf(s.m, c, nmc);  // z of the maximum itself: the rounding of nmc
            const uint64_t c2 = ptx::f2_pack(c, c), nmc2 = ptx::f2_pack(nmc, nmc);
            Sums2 p = {0ull, 0ull}, q = {0ull, 0ull};
#pragma unroll
            for (int u = 0; u < kU; ++u)
                if (i0 + u * kThreads < nvec) {
                    float f[N];
                    Vec<T>::load(Vec<T>::raise(v[u]), f);
#pragma unroll
                    for (int e = 0; e < N; e += 4) {
                        add2(p, f[e], f[e + 1], c2, nmc2);
                        add2(q, f[e + 2], f[e + 3], c2, nmc2);
                    }
                }
            float l0, l1, t0, t1;
            ptx::f2_unpack(ptx::f2_add(p.l, q.l), l0, l1);
            ptx::f2_unpack(ptx::f2_add(p.t, q.t), t0, t1);
            // every weight came out 2^shift times too large, every z by shift
            const float l = l0 + l1, t = fmaf(-shift, l, t0 + t1), k = ptx::ex2(-shift);
            s.l = fmaf(l, k, s.l);
            s.t = fmaf(t, k, s.t);
        } else {
            // The batch's weights are summed apart: 500 alike ones added to one
            // running sum may all round the same way, up to 8e-6 of it; in
            // batches of 64 at most 1e-6. (2048 x 128256 bf16 98 us instead of
            // 96; t too apart 101. What t then loses stays below 1e-5 of the
            // entropy.)
            const float l = s.l;
            s.l = 0.f;
#pragma unroll
            for (int u = 0; u < kU; ++u)
                if (i0 + u * kThreads < nvec) {
                    float f[N];
                    Vec<T>::load(v[u], f);
#pragma unroll
                    for (int e = 0; e < N; ++e) add<kHalves>(s, f[e], c);
                }
            s.l += l;
        }
    }

    // ---- the CTA's sums, and the bound of its alternatives ----
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Sums b = {__shfl_down_sync(0xffffffffu, s.m, o), __shfl_down_sync(0xffffffffu, s.l, o),
                        __shfl_down_sync(0xffffffffu, s.t, o)};
        s = join<kHalves>(s, b, c);
    }
    if (lane == 0) sh.sums[warp] = s;
    const int top = a.top;
    // groups of 32 lanes or fewer: of those that hold elements half as many
    // again as alternatives, so that the bound is not far below the n-th
    // largest (with empty groups among the first n it would be -inf)
    int lanes = 32;
    while (lanes > 1 && min(nvec, kThreads) / lanes < top + top / 2) lanes >>= 1;
    const int groups = min(kThreads / lanes, kMaxGroups);
    if (top > 0) {
        float g = own;
        for (int o = 1; o < lanes; o <<= 1) g = max_nan(g, __shfl_xor_sync(0xffffffffu, g, o));
        if ((lane & (lanes - 1)) == 0 && tid / lanes < groups) sh.gmax[tid / lanes] = g;
    }
    __syncthreads();
    if (warp == 0) {
        Sums t = lane < kWarps ? sh.sums[lane] : Sums{-INFINITY, 0.f, 0.f};
#pragma unroll
        for (int o = kWarps / 2; o > 0; o >>= 1) {
            const Sums b = {__shfl_down_sync(0xffffffffu, t.m, o), __shfl_down_sync(0xffffffffu, t.l, o),
                            __shfl_down_sync(0xffffffffu, t.t, o)};
            t = join<kHalves>(t, b, c);
        }
        if (lane == 0) sh.cta = t;
    }
    if (top > 0) {
        const int at = tid - (kThreads - kMaxGroups);  // the last warps: warp 0 joins the sums
        if (at >= 0 && at < groups) {  // the group maximum of rank top - 1 (a NaN has rank 0: the row is answered with NaN)
            const float g = sh.gmax[at];
            int r = 0;
#pragma unroll 8
            for (int j = 0; j < groups; ++j) r += before(sh.gmax[j], j, g, at);
            if (r == top - 1) sh.bound = g;
        }
        __syncthreads();
        const float bound = sh.bound;
        auto offer = [&](float v, int i) {
            if (v >= bound && v > -INFINITY) {
                const int at = atomicAdd(&sh.count, 1);
                if (at < kCand) sh.cand[at] = {v, i};
            }
        };
        if (single >= 0) offer(Vec<T>::to_float(x[single]), single);
        const bool mine = own >= bound && own > -INFINITY;
        if (once) {
            if (mine) {
#pragma unroll
                for (int u = 0; u < kU; ++u) {
                    const int i = tid + u * kThreads;
                    if (i < nvec && Vec<T>::max(v[u]) >= bound) {
                        float f[N];
                        Vec<T>::load(v[u], f);
#pragma unroll
                        for (int e = 0; e < N; ++e) offer(f[e], lo + head + i * N + e);
                    }
                }
            }
        } else {
            // Few threads of the warp may hold one, and a thread's elements are
            // one load of the warp: the warp reads them, thread by thread.
            // Else a thread looks again at its batches that may hold one, the
            // lanes each at their next one together, so that their loads are
            // under way at once. 605 rows of 30079 fp16 logits, 5 alternatives:
            // 15.7 us the first way, 19.4 the second; 444 of 148663 fp32
            // logits, 64 alternatives: 104 and 56 us.
            unsigned todo = __ballot_sync(0xffffffffu, mine);
            const bool by_warp = nvec <= 32 * kThreads && __popc(todo) <= 3;
            if (by_warp)
                for (; todo; todo &= todo - 1) {
                    const int i = (warp << 5) + __ffs(todo) - 1 + lane * kThreads;
                    if (i >= nvec) continue;
                    v[0] = __ldcg(xv + i);
                    if (Vec<T>::max(v[0]) < bound) continue;
                    float f[N];
                    Vec<T>::load(v[0], f);
#pragma unroll
                    for (int e = 0; e < N; ++e) offer(f[e], lo + head + i * N + e);
                }
            unsigned hits = 0;
            if (mine && !by_warp)
                for (int b = 0; b < min(batches, kSlots); ++b) hits |= (unsigned)(batch_max[b][tid] >= bound) << b;
            while (__any_sync(0xffffffffu, hits != 0)) {
                if (hits)
                    for (int i0 = tid + (__ffs(hits) - 1) * kThreads * kU; i0 < nvec; i0 += kSlots * kThreads * kU) {
#pragma unroll
                        for (int u = 0; u < kU; ++u)
                            if (i0 + u * kThreads < nvec) v[u] = __ldcg(xv + i0 + u * kThreads);
#pragma unroll
                        for (int u = 0; u < kU; ++u)
                            if (i0 + u * kThreads < nvec && Vec<T>::max(v[u]) >= bound) {
                                float f[N];
                                Vec<T>::load(v[u], f);
#pragma unroll
                                for (int e = 0; e < N; ++e) offer(f[e], lo + head + (i0 + u * kThreads) * N + e);
                            }
                    }
                hits &= hits - 1;
            }
        }
        __syncthreads();
        int count = sh.count;
        if (count > kRank && count <= kCand) {
            // A long list (ties, or a row too short for a close bound): ranking
            // costs its square, so it is cut first, at a value found by halving
            // the range of the order-preserving integers. top or more stay.
            constexpr int kHold = kCand / kThreads;
            Best h[kHold];
            uint32_t key[kHold];
#pragma unroll
            for (int q = 0; q < kHold; ++q) {
                const int j = tid + q * kThreads;
                h[q] = j < count ? sh.cand[j] : Best{0.f, 0};
                const uint32_t u = __float_as_uint(h[q].v + 0.f);  // -0 orders as +0
                key[q] = j < count ? (u & 0x80000000u ? ~u : u | 0x80000000u) : 0u;
            }
            uint32_t from = 1u, to = 0xffffffffu;  // the cut: `from` leaves `left` >= top, above `to` fewer than top
            int left = count;
            for (int step = 0; from < to && left > kRank; ++step) {
                const uint32_t mid = from + (to - from) / 2 + 1;
                int c1 = 0;
#pragma unroll
                for (int q = 0; q < kHold; ++q) c1 += key[q] >= mid;
                c1 = __reduce_add_sync(0xffffffffu, c1);
                if (lane == 0) sh.tally[step & 1][warp] = c1;
                __syncthreads();
                int all = 0;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) all += sh.tally[step & 1][w];
                if (all >= top) {
                    from = mid;
                    left = all;
                } else {
                    to = mid - 1;
                }
            }
            __syncthreads();  // every candidate is held, every tally read
            if (tid == 0) sh.count = 0;
            __syncthreads();
#pragma unroll
            for (int q = 0; q < kHold; ++q)
                if (key[q] >= from) sh.cand[atomicAdd(&sh.count, 1)] = h[q];
            __syncthreads();
            count = sh.count;
        }
        if (count <= kCand) {
            for (int j = tid; j < count; j += kThreads) {
                const Best b = sh.cand[j];
                int r = 0;
                for (int q = 0; q < count; ++q) r += before(sh.cand[q].v, sh.cand[q].i, b.v, b.i);
                if (r < top) sh.list[r] = b;
            }
            if (tid == 0) sh.found = min(count, top);
        } else {
            // more elements reach the bound than the list holds: the largest
            // behind the last one found, top times
            Best last = {INFINITY, -1};
            for (int n = 0; n < top; ++n) {
                Best b = {-INFINITY, 0x7fffffff};
                for (int i = lo + tid; i < hi; i += kThreads) {
                    const float v = Vec<T>::to_float(x[i]);
                    if (before(last.v, last.i, v, i) && before(v, i, b.v, b.i)) b = {v, i};
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const Best d = {__shfl_xor_sync(0xffffffffu, b.v, o), __shfl_xor_sync(0xffffffffu, b.i, o)};
                    if (before(d.v, d.i, b.v, b.i)) b = d;
                }
                if (lane == 0) sh.red[warp] = b;
                __syncthreads();
                b = sh.red[0];
                for (int w = 1; w < kWarps; ++w)
                    if (before(sh.red[w].v, sh.red[w].i, b.v, b.i)) b = sh.red[w];
                __syncthreads();
                last = b;
                if (tid == 0) sh.list[n] = b;
            }
            if (tid == 0) sh.found = top;
        }
    } else if (tid == 0) {
        sh.found = 0;
    }
    __syncthreads();

    // ---- the row: rank 0 joins the cluster's sums and lists ----
    cg::cluster_group cluster = cg::this_cluster();
    Sums all = sh.cta;
    int found = sh.found;
    Best *merged = sh.list;
    if (split > 1) {
        cluster.sync();
        if (rank == 0) {
            // lane q has CTA q's sums; joined in a fixed order
            Sums t = lane < split ? *cluster.map_shared_rank(&sh.cta, lane) : Sums{-INFINITY, 0.f, 0.f};
#pragma unroll
            for (int o = kMaxCluster / 2; o > 0; o >>= 1) {
                const Sums b = {__shfl_down_sync(0xffffffffu, t.m, o), __shfl_down_sync(0xffffffffu, t.l, o),
                                __shfl_down_sync(0xffffffffu, t.t, o)};
                t = join<kHalves>(t, b, c);
            }
            all = {__shfl_sync(0xffffffffu, t.m, 0), __shfl_sync(0xffffffffu, t.l, 0), __shfl_sync(0xffffffffu, t.t, 0)};
            if (top > 0) {
                // every list in its place of `cand`, missing entries last; an
                // entry's rank is its own place and those before it in the
                // other lists, which are sorted
                int f = lane < split ? cluster.map_shared_rank(&sh, lane)->found : 0;
                for (int j = tid; j < split * top; j += kThreads) {
                    const int q = j / top, n = j % top;
                    const Shared *o = cluster.map_shared_rank(&sh, q);
                    sh.cand[j] = n < o->found ? o->list[n] : Best{-INFINITY, 0x7fffffff};
                    sh.rank[j] = n;
                }
#pragma unroll
                for (int o = kMaxCluster / 2; o > 0; o >>= 1) f += __shfl_xor_sync(0xffffffffu, f, o);
                found = min(__shfl_sync(0xffffffffu, f, 0), top);
                __syncthreads();
                for (int j = tid; j < split * top * split; j += kThreads) {
                    const int e = j / split, q = j % split;
                    const Best b = sh.cand[e];
                    if (q == e / top || b.i == 0x7fffffff) continue;
                    const Best *l = sh.cand + q * top;
                    int n = 0;
                    for (int step = kMaxTop; step > 0; step >>= 1)
                        if (n + step <= top && before(l[n + step - 1].v, l[n + step - 1].i, b.v, b.i)) n += step;
                    if (n > 0) atomicAdd(&sh.rank[e], n);
                }
                __syncthreads();
                for (int j = tid; j < split * top; j += kThreads)
                    if (sh.cand[j].i != 0x7fffffff && sh.rank[j] < top) sh.list[sh.rank[j]] = sh.cand[j];
                __syncthreads();
            }
        }
    }
    if (rank == 0) {
        constexpr float kLn2 = 0.69314718055994531f;
        const bool none = !(all.l > 0.f) && all.m <= -FLT_MAX;  // nothing but -inf
        const bool bad = !(all.m <= FLT_MAX);                   // NaN or +inf
        const float nan = __int_as_float(0x7fffffff);
        const float log2l = log2f(all.l);
        auto logprob = [&](float v) {
            if (bad) return nan;
            if (none || v == -INFINITY) return -INFINITY;
            // the difference may pass the type's end: by halves, and no log2 form
            return fmaf(v, 0.5f, -0.5f * all.m) * a.inv_temperature * 2.f - log2l * kLn2;
        };
        if (tid == 0) {
            if (a.logprobs) {
                const int t = a.tokens[row];
                a.logprobs[row] = t < 0 ? 0.f : t >= a.vocab ? nan : logprob(Vec<T>::to_float(x[t]));
            }
            if (a.entropy) a.entropy[row] = bad ? nan : none ? 0.f : (log2l - all.t / all.l) * kLn2;
        }
        for (int n = tid; n < top; n += kThreads) {
            const bool have = !bad && n < found;
            const long long at = (long long)row * top + n;
            if (a.top_tokens) a.top_tokens[at] = have ? merged[n].i : -1;
            if (a.top_logprobs) a.top_logprobs[at] = bad ? nan : have ? logprob(merged[n].v) : -INFINITY;
        }
    }
    __syncwarp();
    if (split > 1) cluster.sync();  // no CTA leaves while rank 0 may still read its shared memory
}

template <typename T, int kThreads, bool kHalves>
cudaError_t launch_n(const LogprobArgs &a, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.rows * (unsigned)a.split);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)a.split;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, logprobs_kernel<T, kThreads, kHalves>, a);
}

template <typename T>
cudaError_t launch_t(const LogprobArgs &a, int num_sms, cudaStream_t s) {
    if constexpr (!std::is_same_v<T, __half>)  // (fp16 differences stay inside fp32's range)
        if (a.scale_log2 < kFlat) return launch_n<T, 512, true>(a, s);
    return (long long)a.rows * a.split > 2ll * num_sms ? launch_n<T, 256, false>(a, s) : launch_n<T, 512, false>(a, s);
}

}  // namespace

cudaError_t launch_logprobs(LogprobArgs a, int dtype, int num_sms, cudaStream_t s) {
    if (a.rows <= 0) return cudaSuccess;
    // Rows split over a cluster until there is a CTA for every SM or two, as
    // long as a thread keeps two vectors (with twice as many CTAs 64 rows of
    // 128256 take 17.5 us instead of 14.8).
    const int per = dtype == 2 ? 4 : 8;
    a.split = 1;
    while (a.split < kMaxCluster && (long long)a.rows * a.split <= num_sms &&
           a.vocab / (a.split * 2) >= 2 * per * 512)
        a.split *= 2;
    switch (dtype) {
    case 0: return launch_t<__half>(a, num_sms, s);
    case 1: return launch_t<__nv_bfloat16>(a, num_sms, s);
    case 2: return launch_t<float>(a, num_sms, s);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace tllm
