// W8A16 projections with their epilogue, for up to 8 rows (a decode step):
//   y[r][n] = act(sum_k x[r][k] w[k][n] s[k / group][n] + bias[n]) + residual[r][n]
// and the gated pair act(gate) * up, sm_100a. The weights are packed once
// (linear_pack.cuh); tl_linear sends larger batches to linear_tc.cu.
//
// Every weight is read once, so the weight stream bounds it. A CTA owns one
// tile of 64 packed columns and a range of 128-row blocks of K (the whole K,
// or one of the equal parts that the CTAs of a cluster share). A producer
// warp streams units (weights and scales by one bulk copy, the rows'
// activations of the block by two TMA tiles, which also zero-fill past K and
// past the last row) through a ring of shared-memory stages, so the bytes in
// flight are the ring's and hold no registers; eight consumer warps take the
// units in turn, each from a stage of its own. The weights are the A side of
// mma.sync.m16n8k16, the 8 batch rows its N side, so a lane's 16-byte chunk of
// weights feeds four MMA steps and no transposition is needed. int8 -> fp16
// is exact and the scales multiply fp32 sums of at most 64 products, so no
// weight is rounded. tcgen05 is not used here: one UMMA covers 16 rows of K
// whatever the batch and takes longer to issue than the bytes it consumes
// take to arrive. With 16 rows the order turns: the same kernel for 16 took
// 143 us for 4096 x 128256, linear_tc.cu 98.
//
// The warps' sums meet in shared memory and, when K is split, the CTAs' in
// distributed shared memory, both in a fixed order: the result does not
// depend on timing. The mbarrier waits are bounded; a CTA whose wait gives up
// writes NaN. The barriers of the CTA and the cluster have no limit of their
// own: they wait for roles whose mbarrier waits all end.
#include <algorithm>
#include <atomic>
#include <cooperative_groups.h>
#include <cstdint>
#include <cuda_fp16.h>

#include "kernels.h"
#include "linear_pack.cuh"
#include "ptx.cuh"

namespace tllm {
namespace {

namespace cg = cooperative_groups;

constexpr int kRows = kLinearFewRows;              // 8: the N of one MMA
constexpr int kConsumers = 8;                      // warps
constexpr int kThreads = 32 * (kConsumers + 1);    // + the producer warp
constexpr int kMaxUnit = lin::unit_bytes(32);      // 8704
constexpr int kXHalf = kRows * 128;                // activations of 64 rows of K: [rows][128 B], swizzled
constexpr int kStage = (2 * kXHalf + kMaxUnit + 1023) / 1024 * 1024;
// One stage per consumer warp: a warp then meets every phase of its barrier in
// turn (with another count it could miss one and take the phase after it for
// the one before).
constexpr int kNS = kConsumers;
constexpr int kRing = kNS * kStage;
constexpr int kRowF = lin::kTileN + 4;             // floats of a row of sums (banks)
constexpr int kPart = kRows * kRowF * 4;           // the CTA's sums
constexpr int kSmem = 1024 + kRing + kPart + 2 * kNS * 8 + 16;
constexpr long long kWait = 4000000000ll;          // cycles: about 2 s
static_assert(kConsumers * kPart <= kRing, "every warp's sums, over the ring");
static_assert(2 * (kSmem + 1024) <= 227 * 1024, "two CTAs per SM");
static_assert(kRows == 8, "one MMA's N");

struct alignas(64) Map {  // a tensor map, opaque here
    unsigned char bytes[128];
};

template <bool G32>
__global__ void __launch_bounds__(kThreads, 2)
    linear_kernel(const __grid_constant__ LinearArgs a, const __grid_constant__ Map xmap) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float *part = reinterpret_cast<float *>(smem + kRing);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + kRing + kPart);
    const uint32_t full_u = ptx::smem_u32(bars), empty_u = full_u + 8 * kNS;
    __shared__ int s_failed;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int csplit = a.csplit, rank = blockIdx.x % csplit, tile = blockIdx.x / csplit;
    const int nblocks = lin::blocks(a.k);
    const int b0 = (int)((long long)rank * nblocks / csplit), b1 = (int)((long long)(rank + 1) * nblocks / csplit);
    const int count = b1 - b0;
    const int unit = lin::unit_bytes(a.group);

    if (threadIdx.x == 0) {
        for (int s = 0; s < kNS; ++s) {
            ptx::mbar_init(full_u + 8 * s, 1);
            ptx::mbar_init(empty_u + 8 * s, 1);
        }
        ptx::fence_barrier_init();
        s_failed = 0;
    }
    __syncthreads();
    // Programmatic dependent launch: until the kernel before has completed, only
    // a prefetch of the first weights to L2 (a later write of them still wins).
    // The next kernel is let in after the wait, so that nothing older than this
    // kernel runs beside it; its CTAs come as ours leave.
    const uint8_t *w = static_cast<const uint8_t *>(a.packed) + ((long long)tile * nblocks + b0) * unit;
    if (warp == kConsumers && lane == 0) {
        ptx::prefetch_tensormap(&xmap);
        ptx::bulk_prefetch_l2(w, (uint32_t)(min(kNS, count) * unit));
    }
    __syncwarp();
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();

    if (warp == kConsumers) {
        // ---- producer (one lane) ----
        if (lane == 0) {
            const uint64_t once = ptx::l2_policy_evict_first(), keep = ptx::l2_policy_evict_last();
            int issued = 0;
            for (int i = 0; i < count; ++i, ++issued) {
                const int s = i % kNS;
                if (i >= kNS && !ptx::mbar_wait_cycles(empty_u + 8 * s, (uint32_t)((i / kNS - 1) & 1), kWait)) {
                    s_failed = 1;
                    break;
                }
                const int k0 = (b0 + i) * lin::kBlockK;
                const uint32_t dst = ptx::smem_u32(smem + s * kStage), bar = full_u + 8 * s;
                ptx::mbar_arrive_expect_tx(bar, (uint32_t)(unit + 2 * kXHalf));
                ptx::bulk_load(dst + 2 * kXHalf, w + (long long)i * unit, (uint32_t)unit, bar, once);
                // (a half block past K lies wholly out of bounds: zeros)
                ptx::tma_load_2d(dst, &xmap, bar, k0, 0, keep);
                ptx::tma_load_2d(dst + kXHalf, &xmap, bar, k0 + 64, 0, keep);
            }
            // whoever gave up, the last copies land (or a bounded wait passes) before the CTA goes on
            for (int i = max(0, issued - kNS); i < issued; ++i)
                ptx::mbar_wait_cycles(full_u + 8 * (i % kNS), (uint32_t)((i / kNS) & 1), kWait);
        }
        __syncwarp();
    } else {
        // ---- consumers: warp w takes units w, w + 8, ... ----
        const int gid = lane >> 2, tig = lane & 3;
        float acc[4][4];
#pragma unroll
        for (int nb = 0; nb < 4; ++nb) acc[nb][0] = acc[nb][1] = acc[nb][2] = acc[nb][3] = 0.f;
        bool ok = true;
        for (int i = warp; i < count; i += kConsumers) {
            const int s = i % kNS;
            ok = __all_sync(0xffffffffu, ptx::mbar_wait_cycles(full_u + 8 * s, (uint32_t)((i / kNS) & 1), kWait));
            if (!ok) break;
            const uint8_t *st = smem + s * kStage;
            const uint8_t *wst = st + 2 * kXHalf;
            const __half *sc = reinterpret_cast<const __half *>(wst + 2 * lin::kHalfBytes);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                // row gid: k 8 tig..+7 and 32 + 8 tig..+7 of the half
                const uint8_t *p = st + h * kXHalf + gid * 128;
                const uint4 x0 = *reinterpret_cast<const uint4 *>(p + ((tig ^ gid) << 4));
                const uint4 x1 = *reinterpret_cast<const uint4 *>(p + (((4 + tig) ^ gid) << 4));
                const uint32_t xf[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
                const uint8_t *wp = wst + h * lin::kHalfBytes + tig * 1024;
#pragma unroll
                for (int nb = 0; nb < 4; ++nb) {
                    const int c0 = nb * 16 + gid;
                    const uint4 w0 = *reinterpret_cast<const uint4 *>(wp + (c0 ^ (2 * tig)) * 16);
                    const uint4 w1 = *reinterpret_cast<const uint4 *>(wp + ((c0 + 8) ^ (2 * tig)) * 16);
                    const uint32_t u0[4] = {w0.x, w0.y, w0.z, w0.w}, u1[4] = {w1.x, w1.y, w1.z, w1.w};
                    float d[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (j == 0 || (G32 && j == 2)) d[0] = d[1] = d[2] = d[3] = 0.f;
                        uint32_t a0, a1, a2, a3;
                        lin::to_h4(u0[j], a0, a2);
                        lin::to_h4(u1[j], a1, a3);
                        ptx::mma_16816(d, a0, a1, a2, a3, xf[2 * j], xf[2 * j + 1]);
                        if (j == 3 || (G32 && j == 1)) {
                            const int g = G32 ? 2 * h + (j >> 1) : h * 64 / a.group;
                            const float s0 = __half2float(sc[g * lin::kTileN + c0]);
                            const float s1 = __half2float(sc[g * lin::kTileN + c0 + 8]);
                            acc[nb][0] = fmaf(d[0], s0, acc[nb][0]);
                            acc[nb][1] = fmaf(d[1], s0, acc[nb][1]);
                            acc[nb][2] = fmaf(d[2], s1, acc[nb][2]);
                            acc[nb][3] = fmaf(d[3], s1, acc[nb][3]);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(empty_u + 8 * s);
        }
        if (!ok) s_failed = 1;
        ptx::named_barrier_sync(1, 32 * kConsumers);  // every unit consumed: the sums go over the ring
        float *sum = reinterpret_cast<float *>(smem) + warp * kRows * kRowF;
#pragma unroll
        for (int nb = 0; nb < 4; ++nb) {
            float *p = sum + 2 * tig * kRowF + nb * 16 + gid;
            p[0] = acc[nb][0];
            p[kRowF] = acc[nb][1];
            p[8] = acc[nb][2];
            p[kRowF + 8] = acc[nb][3];
        }
        ptx::named_barrier_sync(1, 32 * kConsumers);
        const float *all = reinterpret_cast<const float *>(smem);
        const int c = threadIdx.x & 63;
#pragma unroll
        for (int r = threadIdx.x >> 6; r < kRows; r += 4) {
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < kConsumers; ++w) v += all[(w * kRows + r) * kRowF + c];
            part[r * kRowF + c] = v;
        }
    }

    // ---- the CTAs' parts of K, in rank order, and the epilogue ----
    __syncthreads();
    if (s_failed) {  // a wait gave up: NaN, not a wrong number
        for (int i = threadIdx.x; i < kRows * kRowF; i += kThreads) part[i] = __int_as_float(0x7fffffff);
        __syncthreads();
    }
    cg::cluster_group cluster = cg::this_cluster();
    if (csplit > 1) cluster.sync();
    auto total = [&](int r, int c) {
        if (csplit == 1) return part[r * kRowF + c];
        float v = 0.f;
        for (int q = 0; q < csplit; ++q) v += *cluster.map_shared_rank(part + r * kRowF + c, q);
        return v;
    };
    const int oc = a.gated ? lin::kTileN / 2 : lin::kTileN;  // output columns of the tile
    const __half *bias = static_cast<const __half *>(a.bias), *bias2 = static_cast<const __half *>(a.bias2);
    for (int i = rank * kThreads + threadIdx.x; i < a.rows * oc; i += csplit * kThreads) {
        const int r = i / oc, c = i % oc;
        const long long n = (long long)tile * oc + c;
        if (n >= a.n) continue;
        float v;
        if (a.gated) {
            const int p = (c >> 3) * 16 + (c & 7);
            float g = total(r, p), u = total(r, p + 8);
            if (bias) g += __half2float(bias[n]);
            if (bias2) u += __half2float(bias2[n]);
            v = lin::activate(a.act, g) * u;
        } else {
            v = total(r, c);
            if (bias) v += __half2float(bias[n]);
            v = lin::activate(a.act, v);
            if (a.residual)
                v += __half2float(static_cast<const __half *>(a.residual)[(long long)r * a.residual_stride + n]);
        }
        static_cast<__half *>(a.y)[(long long)r * a.y_stride + n] = __float2half_rn(v);
    }
    __syncwarp();
    if (csplit > 1) cluster.sync();  // no CTA leaves while another may still read its shared memory
}

// One thread per 16-byte chunk (and, past those, per scale) of the packed
// weights. Runs once per weight at load; no tuning.
__global__ void linear_pack_kernel(const int8_t *w, const __half *s, const int8_t *w2, const __half *s2, int k, int n,
                                   int group, uint8_t *out) {
    const bool gated = w2 != nullptr;
    const int unit = lin::unit_bytes(group), nblocks = lin::blocks(k);
    const int per = 512 + lin::kTileN * (lin::kBlockK / group);  // chunks and scales of a unit
    const long long total = lin::tiles(n, gated) * nblocks * per;
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
        const long long u = i / per;
        const int j = (int)(i % per);
        const long long tile = u / nblocks;
        const int block = (int)(u % nblocks);
        const int c = j & 63;
        const long long p = tile * lin::kTileN + c;  // packed column
        const bool up = gated && (p & 8);
        const long long col = gated ? (p >> 4) * 8 + (p & 7) : p;
        const int8_t *src = up ? w2 : w;
        uint8_t *dst = out + u * unit;
        if (j < 512) {
            const int h = j >> 8, ch = (j >> 6) & 3;
            uint32_t word[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t v = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const long long row = (long long)block * lin::kBlockK + h * 64 + (q >> 1) * 32 + 8 * ch + (q & 1) * 4 + e;
                    const int b = row < k && col < n ? src[row * n + col] : 0;
                    v |= (uint32_t)((b + 128) & 255) << (8 * e);
                }
                word[q] = v;
            }
            *reinterpret_cast<uint4 *>(dst + h * lin::kHalfBytes + ch * 1024 + (c ^ (2 * ch)) * 16) =
                make_uint4(word[0], word[1], word[2], word[3]);
        } else {
            const int g = (j - 512) >> 6;
            const long long grp = (long long)block * (lin::kBlockK / group) + g;
            const long long row = grp * group;
            const __half v = row < k && col < n ? (up ? s2 : s)[grp * n + col] : __half(0.f);
            reinterpret_cast<__half *>(dst + 2 * lin::kHalfBytes)[g * lin::kTileN + c] = v;
        }
    }
}

template <bool G32>
cudaError_t launch_t(const LinearArgs &a, cudaStream_t s) {
    static std::atomic<unsigned long long> done{0};  // devices whose shared-memory limit is set
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(done.load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(linear_kernel<G32>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
        if (e != cudaSuccess) return e;
        done.fetch_or(bit, std::memory_order_acq_rel);
    }
    const long long ntiles = lin::tiles(a.n, a.gated != 0);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(ntiles * a.csplit));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)a.csplit;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    Map xmap;
    e = encode_tensor_map_2d(&xmap, true, a.x, (unsigned long long)a.k, (unsigned long long)a.rows,
                             (unsigned long long)a.x_stride * 2, 64, kRows);
    if (e != cudaSuccess) return e;
    return cudaLaunchKernelEx(&cfg, linear_kernel<G32>, a, xmap);
}

}  // namespace

cudaError_t launch_linear(LinearArgs a, int num_sms, cudaStream_t s) {
    // K split over a cluster until the tiles fill the SMs' CTA slots, as long
    // as every CTA keeps a unit for each of its warps.
    const long long tiles = lin::tiles(a.n, a.gated != 0), slots = 2ll * num_sms;
    const int nblocks = lin::blocks(a.k);
    a.csplit = 1;
    while (a.csplit < 8 && tiles * a.csplit * 2 <= slots && nblocks / (a.csplit * 2) >= kConsumers) a.csplit *= 2;
    return a.group == 32 ? launch_t<true>(a, s) : launch_t<false>(a, s);
}

cudaError_t launch_linear_pack(const int8_t *w, const void *s, const int8_t *w2, const void *s2, int k, int n, int group,
                               void *out, int num_sms, cudaStream_t st) {
    linear_pack_kernel<<<num_sms * 8, 256, 0, st>>>(w, static_cast<const __half *>(s), w2,
                                                   static_cast<const __half *>(s2), k, n, group,
                                                   static_cast<uint8_t *>(out));
    return cudaGetLastError();
}

}  // namespace tllm
