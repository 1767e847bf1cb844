// W8A16 projections with their epilogue on the 5th-generation tensor cores
// (tcgen05), sm_100a: tl_linear / tl_linear_gated for more rows than
// linear.cu takes. Same operation, same packed weights (linear_pack.cuh).
//
// The packed weight columns are the M side of the UMMA (128 per tile: two
// tiles of 64 of the packed layout), a tile of up to 128 batch rows the N
// side, K in steps of 128 (a block of the packed layout). The int8 weights
// become the fp16 A operand on the way, exactly and in TMEM; their scales
// multiply the fp32 sums of one scale group, so no weight is rounded and no
// fp16 copy of the weights exists in HBM or shared memory. Per CTA:
//   producer    one lane: per step two 8 KB bulk copies of packed weights and
//               two TMA tiles of activations [rows][64] (128-byte swizzle,
//               zeros past K and the last row) into a ring of stages;
//   converters  thread = weight column: 64 bytes from shared memory, to 64
//               fp16, one tcgen05.st of 32 columns: the K-major A operand of
//               half a step (four warps do both halves, eight one each);
//   MMA         one thread each of one or two warps: eight UMMAs (K = 16) per step, A
//               in TMEM, B in shared memory; the scale groups take two
//               accumulators in turn, with two warps each its own;
//   drains      thread = weight column (TMEM lane): when a group is complete,
//               acc += scale * sum for the thread's rows, in registers; after
//               the last group the epilogue from them.
// So one accumulator is filled while the other is scaled, and the CTAs are
// persistent: the next tile's first groups run while a tile's outputs are
// written. The chain conversion - UMMAs - drain sets the pace, not the tensor
// pipe (39 % active at 1024 x 4096 x 14336 gated).
//
// A wait that succeeds at once costs an issuing thread about 110 cycles, a
// commit 80, a UMMA 75 or its pipe time (rows / 2) while the pipe's queue is
// full. So a step is as deep as the layout's block, the stage and the A
// operand are released by one commit, the issuing threads do not wait for the
// activations (the converters waited for the same barrier before they
// arrived), and one thread's waits pass while the other's UMMAs run.
//
// Too few tiles for the SMs: a cluster's CTAs share a tile's K and add their
// sums in distributed shared memory, in rank order. No atomics, no workspace:
// results do not depend on timing. The mbarrier waits are bounded; a CTA whose
// wait gives up writes NaN. What has no limit of its own ends because what it
// waits for does: the barriers of the CTA and the cluster wait for roles whose
// mbarrier waits all end, and tcgen05.alloc for CTAs of the SM that hold
// columns and wait for nobody who still needs some. (A kernel that waits for
// this one was let in after every CTA here had its columns, and columns are
// given back before the cluster's barriers.)
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

constexpr int kM = 128;            // packed columns of a tile
constexpr int kStepK = lin::kBlockK;  // rows of K per ring stage
constexpr int kACols = kStepK / 2;  // TMEM columns of one (fp16 pairs along K)
constexpr int kRaw = 2 * 2 * lin::kHalfBytes;  // packed weights of a step
constexpr int kMaxStages = 8;
constexpr int kMaxSplit = 8;       // CTAs of a cluster that share K
constexpr int kOutRows = 16;       // rows a drain warp writes at a time
constexpr int kOutPitch = 36;      // floats of such a row: 32 columns, padded to 16 bytes and other banks
constexpr long long kWait = 4000000000ll;  // cycles: about 2 s

struct alignas(64) Map {  // a tensor map, opaque here
    unsigned char bytes[128];
};

// kRows: most rows of a tile. kNA: A operand stages in TMEM. kCW, kDW:
// converter and drain warps (sets of four, one per TMEM lane quarter). kIssue:
// warps that issue UMMAs. kPerSm: CTAs per SM.
template <int kRows_, int kNA_, int kCW_, int kDW_, int kIssue_, int kPerSm_>
struct Cfg {
    static constexpr int kNA = kNA_;
    static constexpr int kIssue = kIssue_;
    static constexpr int kRows = kRows_, kCW = kCW_, kDW = kDW_, kPerSm = kPerSm_;
    static constexpr int kConvSets = kCW / 4, kDrainSets = kDW / 4;
    static constexpr int kProd = kDW + kCW, kMma = kProd + 1;  // warps
    static constexpr int kThreads = 32 * (kDW + kCW + 1 + kIssue);
    static constexpr int kAcc = kRows / kDrainSets;  // rows per drain thread
    static constexpr uint32_t kTmemCols = 2 * kRows + kNA * kACols <= 256 ? 256 : 512;
    static constexpr int kRing = (kPerSm == 2 ? 96 : 192) * 1024;
    static constexpr int kOut = kDW * kOutRows * kOutPitch * 4;  // the drain warps' rows on their way out
    static constexpr int kBars = (2 * kMaxStages + kNA + 5) * 8;
    static constexpr int kSmem = 1024 + kRing + kOut + kBars + 16;
    static_assert(kIssue == 1 || kNA % 2 == 0, "an issuing warp meets every phase of its A stages");
    static_assert(kRing / (kRows * 256 + kRaw) > kNA, "a converter meets every phase it waits for");
    static_assert(kAcc % 16 == 0 && kPerSm * kTmemCols <= 512, "tile");
};

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
                   "=r"(r[15])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float *p) {
    uint32_t r[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(p[i]);
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
                 "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
// Waits for this thread's TMEM loads; r is read after it.
__device__ __forceinline__ void tmem_wait_ld16(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                   "+r"(r[15])::"memory");
}

// Tile t of the launch: bands of 16 column tiles, in a band the row tiles in
// turn, so that the tiles in flight share both operands in L2.
struct TilePos {
    int nt, rt;
};
__device__ __forceinline__ TilePos tile_pos(int t, int ntiles, int nrt) {
    const int band = t / (16 * nrt), left = t - band * 16 * nrt;
    const int width = min(16, ntiles - band * 16);
    return {band * 16 + left % width, left / width};
}

// A ring position: the stage and the parity of its current round.
struct Ring {
    int s = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void advance(int by, int size) {
        s += by;
        if (s >= size) {
            s -= size;
            parity ^= 1u;
        }
    }
};

// One drain warp's [16 rows][32 packed columns] of sums, in shared memory, to
// the output: lane = (row, half of the columns). q0, q1: the lane's residuals
// where `have_res`.
template <int ACT, bool GATED>
__device__ __forceinline__ void write_rows(const LinearArgs &a, const float *st, int lane, long long row0, int nrows,
                                        long long packed0, bool have_res, uint4 q0, uint4 q1) {
    constexpr int W = GATED ? 8 : 16;  // outputs of the lane
    const int r = lane >> 1, h = lane & 1;
    const long long n0 = (GATED ? packed0 / 2 : packed0) + h * W;
    const int valid = (int)min((long long)W, a.n - n0);
    if (r >= nrows || valid <= 0) return;
    const float *v = st + r * kOutPitch + h * 16;
    const __half *bias = static_cast<const __half *>(a.bias), *bias2 = static_cast<const __half *>(a.bias2);
    const __half *res =
        a.residual ? static_cast<const __half *>(a.residual) + (row0 + r) * a.residual_stride + n0 : nullptr;
    __half *y = static_cast<__half *>(a.y) + (row0 + r) * a.y_stride + n0;
    const uint32_t q[8] = {q0.x, q0.y, q0.z, q0.w, q1.x, q1.y, q1.z, q1.w};
    uint32_t o[W / 2];
#pragma unroll
    for (int j = 0; j < W; j += 2) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int at = min(j + e, valid - 1);  // (outputs past the last column are not written)
            float x = v[j + e];
            if (bias) x += __half2float(bias[n0 + at]);
            x = lin::activate(ACT, x);
            if constexpr (GATED) {
                float u = v[8 + j + e];
                if (bias2) u += __half2float(bias2[n0 + at]);
                x *= u;
            } else if (have_res) {
                x += __half2float(__ushort_as_half((unsigned short)(q[j / 2] >> (16 * e))));
            } else if (res) {
                x += __half2float(res[at]);
            }
            f[e] = x;
        }
        o[j / 2] = ptx::pack_half2(f[0], f[1]);
    }
    if (valid == W && (reinterpret_cast<uintptr_t>(y) & 15) == 0) {
        *reinterpret_cast<uint4 *>(y) = make_uint4(o[0], o[1], o[2], o[3]);
        if constexpr (!GATED) *reinterpret_cast<uint4 *>(y + 8) = make_uint4(o[4], o[5], o[6], o[7]);
    } else {
#pragma unroll
        for (int j = 0; j < W; ++j)
            if (j < valid) y[j] = __ushort_as_half((unsigned short)(o[j / 2] >> (16 * (j & 1))));
    }
}

template <bool GATED>
__device__ __forceinline__ void write_rows_act(const LinearArgs &a, const float *st, int lane, long long row0, int nrows,
                                               long long packed0, bool have_res, uint4 q0, uint4 q1) {
    switch (a.act) {
    case 1: return write_rows<1, GATED>(a, st, lane, row0, nrows, packed0, have_res, q0, q1);
    case 2: return write_rows<2, GATED>(a, st, lane, row0, nrows, packed0, have_res, q0, q1);
    case 3: return write_rows<3, GATED>(a, st, lane, row0, nrows, packed0, have_res, q0, q1);
    case 4: return write_rows<4, GATED>(a, st, lane, row0, nrows, packed0, have_res, q0, q1);
    default: return write_rows<0, GATED>(a, st, lane, row0, nrows, packed0, have_res, q0, q1);
    }
}

// Four outputs of a row from their sums (v, and u of a gated pair).
template <int ACT>
__device__ __forceinline__ void finish4(const LinearArgs &a, const float (&v)[4], const float (&u)[4], long long row,
                                        long long n0) {
    const int valid = (int)min(4ll, a.n - n0);
    const __half *bias = static_cast<const __half *>(a.bias), *bias2 = static_cast<const __half *>(a.bias2);
    const __half *res = a.residual ? static_cast<const __half *>(a.residual) + row * a.residual_stride + n0 : nullptr;
    __half *y = static_cast<__half *>(a.y) + row * a.y_stride + n0;
    uint32_t o[2];
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int at = min(j + e, valid - 1);  // (outputs past the last column are not written)
            float x = v[j + e];
            if (bias) x += __half2float(bias[n0 + at]);
            x = lin::activate(ACT, x);
            if (a.gated) x *= u[j + e] + (bias2 ? __half2float(bias2[n0 + at]) : 0.f);
            else if (res) x += __half2float(res[at]);
            f[e] = x;
        }
        o[j / 2] = ptx::pack_half2(f[0], f[1]);
    }
    if (valid == 4 && (reinterpret_cast<uintptr_t>(y) & 7) == 0) {
        *reinterpret_cast<uint2 *>(y) = make_uint2(o[0], o[1]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < valid) y[j] = __ushort_as_half((unsigned short)(o[j / 2] >> (16 * (j & 1))));
    }
}

// GPS: scale groups of a step (128 / group).
template <typename C, int GPS>
__global__ void __launch_bounds__(C::kThreads, C::kPerSm)
    linear_tc_kernel(const __grid_constant__ LinearArgs a, const __grid_constant__ Map xmap) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float *out_rows = reinterpret_cast<float *>(smem + C::kRing);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::kRing + C::kOut);
    const uint32_t full_u = ptx::smem_u32(bars);           // [stages] weights and activations landed
    const uint32_t empty_u = full_u + 8 * kMaxStages;      // [stages] multiplied: the stage and its A operand are free
    const uint32_t afull_u = empty_u + 8 * kMaxStages;     // [kNA] A operand in TMEM
    const uint32_t dfull_u = afull_u + 8 * C::kNA;            // [2] a group's sums complete
    const uint32_t dempty_u = dfull_u + 16;                // [2] ... and drained
    const uint32_t done_u = dempty_u + 16;                 // every UMMA complete
    __shared__ uint32_t s_tmem;
    __shared__ int s_failed;  // a drain's wait gave up (csplit > 1)

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int RT = a.row_tile;  // rows of a tile, a multiple of 32
    const int nrt = (a.rows + RT - 1) / RT;
    const int tiles64 = (int)lin::tiles(a.n, a.gated != 0);
    const int ntiles = (tiles64 + 1) / 2, total = ntiles * nrt;
    const int csplit = a.csplit, rank = blockIdx.x % csplit;
    const int nblocks = lin::blocks(a.k), unit = lin::unit_bytes(a.group);
    // this CTA's part of K, in blocks of 128: its steps
    const int b0 = (int)((long long)rank * nblocks / csplit), b1 = (int)((long long)(rank + 1) * nblocks / csplit);
    const int steps = b1 - b0;
    const int first = blockIdx.x / csplit, stride = gridDim.x / csplit;
    const int xhalf = RT * 128, stage_bytes = 2 * xhalf + kRaw;
    const int NS = min(kMaxStages, C::kRing / stage_bytes);  // > kNA: a converter meets every phase it waits for

    if (threadIdx.x == 0) {
        for (int s = 0; s < kMaxStages; ++s) {
            ptx::mbar_init(full_u + 8 * s, 1);
            ptx::mbar_init(empty_u + 8 * s, GPS == 1 ? 1 : C::kIssue);  // commits: of the warp(s) that had a part of the step
        }
        for (int s = 0; s < C::kNA; ++s) ptx::mbar_init(afull_u + 8 * s, C::kCW);
        for (int s = 0; s < 2; ++s) {
            ptx::mbar_init(dfull_u + 8 * s, 1);
            ptx::mbar_init(dempty_u + 8 * s, C::kDW);
        }
        ptx::mbar_init(done_u, C::kIssue);
        ptx::fence_barrier_init();
        s_failed = 0;
    }
    if (warp == C::kMma) ptx::tmem_alloc(ptx::smem_u32(&s_tmem), C::kTmemCols);
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tbase = s_tmem;             // accumulators at 0 and kRows, then the A stages
    const uint32_t acol = 2 * C::kRows;
    // Programmatic dependent launch: until the kernel before has completed, only
    // a prefetch of the first weights to L2 (a later write of them still wins).
    // The next kernel is let in after the wait, so that nothing older than this
    // kernel runs beside it.
    if (warp == C::kProd && lane == 0) {
        ptx::prefetch_tensormap(&xmap);
        if (first < total) {
            const TilePos p = tile_pos(first, ntiles, nrt);
            const uint8_t *w = static_cast<const uint8_t *>(a.packed) + ((long long)(2 * p.nt) * nblocks + b0) * unit;
            const uint32_t bytes = (uint32_t)(min(NS, steps) * unit);
            ptx::bulk_prefetch_l2(w, bytes);
            if (2 * p.nt + 1 < tiles64) ptx::bulk_prefetch_l2(w + (long long)nblocks * unit, bytes);
        }
    }
    __syncwarp();
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();

    // (A wait for "empty" starts on the parity of the round before: a fresh
    // barrier answers it at once.)
    if (warp == C::kProd) {
        if (lane == 0) {
            // ---- producer ----
            const uint64_t keep = ptx::l2_policy_evict_last();
            const uint64_t wpol = nrt > 1 ? keep : ptx::l2_policy_evict_first();  // weights: read once per row tile
            const uint8_t *packed = static_cast<const uint8_t *>(a.packed);
            const uint32_t ring_u = ptx::smem_u32(smem);
            Ring r;
            int issued = 0;
            bool ok = true;
            for (int t = first; t < total && ok; t += stride) {
                const TilePos p = tile_pos(t, ntiles, nrt);
                const bool both = 2 * p.nt + 1 < tiles64;
                const uint8_t *w0 = packed + ((long long)(2 * p.nt) * nblocks + b0) * unit;
                const uint8_t *w1 = w0 + (long long)nblocks * unit;
                const uint32_t bytes = (uint32_t)(2 * xhalf + (both ? 2 : 1) * 2 * lin::kHalfBytes);
                for (int i = 0; i < steps; ++i, r.advance(1, NS), ++issued) {
                    if (!ptx::mbar_wait_cycles(empty_u + 8 * r.s, r.parity ^ 1u, kWait)) {
                        ok = false;
                        break;
                    }
                    const uint32_t dst = ring_u + (uint32_t)(r.s * stage_bytes), bar = full_u + 8 * r.s;
                    ptx::mbar_arrive_expect_tx(bar, bytes);
                    ptx::bulk_load(dst + 2 * xhalf, w0, 2 * lin::kHalfBytes, bar, wpol);
                    if (both) ptx::bulk_load(dst + 2 * xhalf + 2 * lin::kHalfBytes, w1, 2 * lin::kHalfBytes, bar, wpol);
                    // the block's scales, on their way to L2 for the drains: a
                    // load of them is asked for one group ahead, less than HBM takes
                    ptx::bulk_prefetch_l2(w0 + 2 * lin::kHalfBytes, (uint32_t)(unit - 2 * lin::kHalfBytes));
                    if (both) ptx::bulk_prefetch_l2(w1 + 2 * lin::kHalfBytes, (uint32_t)(unit - 2 * lin::kHalfBytes));
                    const int k0 = (b0 + i) * kStepK;  // (a half past K lies wholly out of bounds: zeros)
                    ptx::tma_load_2d(dst, &xmap, bar, k0, p.rt * RT, keep);
                    ptx::tma_load_2d(dst + xhalf, &xmap, bar, k0 + 64, p.rt * RT, keep);
                    w0 += unit;
                    w1 += unit;
                }
            }
            // whoever gave up, the last copies land (or a bounded wait passes) before the CTA goes on
            for (int i = max(0, issued - NS); i < issued; ++i)
                ptx::mbar_wait_cycles(full_u + 8 * (i % NS), (uint32_t)((i / NS) & 1), kWait);
        }
    } else if (warp >= C::kMma) {
        if (lane == 0) {
            // ---- UMMA issue: one warp for all groups, or warp m of two for
            // every second one, with accumulator m ----
            const int m = warp - C::kMma;
            const uint32_t idesc = (1u << 4) | ((uint32_t)(RT >> 3) << 17) | ((uint32_t)(kM >> 4) << 24);
            const uint64_t desc0 = ptx::umma_desc_sw128(ptx::smem_u32(smem), 16, 1024);
            const uint32_t half = (uint32_t)xhalf >> 4;  // descriptors count 16 bytes
            const int my_steps = first < total ? ((total - first + stride - 1) / stride) * steps : 0;
            constexpr int kBy = C::kIssue == 2 && GPS == 1 ? 2 : 1;          // steps from one of this warp's to the next
            constexpr int kMine = C::kIssue == 2 ? (GPS + 1) / 2 : GPS;      // its groups of a step
            Ring r, aa, dd;
            r.s = aa.s = kBy == 2 ? m : 0;
            dd.s = m;
            bool ok = true;
            for (int it = r.s; it < my_steps && ok; it += kBy) {
                const uint64_t bd = desc0 + (uint64_t)((uint32_t)(r.s * stage_bytes) >> 4);
                const uint32_t at = tbase + acol + (uint32_t)(aa.s * kACols);
#pragma unroll
                for (int gg = 0; gg < kMine; ++gg) {
                    ok = ok && ptx::mbar_wait_cycles(dempty_u + 8 * dd.s, dd.parity ^ 1u, kWait);
                    if (gg == 0) ok = ok && ptx::mbar_wait_cycles(afull_u + 8 * aa.s, aa.parity, kWait);
                    if (!ok) break;
                    ptx::tc_fence_after_sync();
                    const uint32_t dt = tbase + (uint32_t)(dd.s * C::kRows);
                    // the group's first 16 rows of K
                    const int ks0 = (GPS == 1 ? 0 : C::kIssue == 2 ? 2 * gg + m : gg) * (8 / GPS);
#pragma unroll
                    for (int j = 0; j < 8 / GPS; ++j) {
                        const int ks = ks0 + j;
                        ptx::umma_f16_ta(dt, at + (uint32_t)(8 * ks), bd + (uint32_t)(ks >> 2) * half + (uint32_t)(ks & 3) * 2,
                                         idesc, j == 0 ? 0u : 1u);
                    }
                    ptx::umma_commit(dfull_u + 8 * dd.s);
                    dd.advance(C::kIssue, 2);
                }
                if (ok) ptx::umma_commit(empty_u + 8 * r.s);
                r.advance(kBy, NS);
                aa.advance(kBy, C::kNA);
            }
            // every UMMA issued is complete before TMEM is freed
            ptx::umma_commit(done_u);
            ptx::mbar_wait_cycles(done_u, 0u, kWait);
        }
    } else if (warp >= C::kDW) {
        // ---- converters: both halves of every step, or (two sets) one ----
        const int set = (warp - C::kDW) >> 2, q = warp & 3;
        const int n64 = (q & 1) * 32 + lane;
        const uint8_t *raw0 = smem + 2 * xhalf + (q >> 1) * 2 * lin::kHalfBytes;
        const uint32_t at0 = tbase + ((uint32_t)(32 * q) << 16) + acol;
        const int my_steps = first < total ? ((total - first + stride - 1) / stride) * steps : 0;
        Ring r, aa, old;  // the step's stage and A stage; the stage of the step that used the A stage before
        for (int it = 0; it < my_steps; ++it) {
            bool ok = ptx::mbar_wait_cycles(full_u + 8 * r.s, r.parity, kWait);
            if (it >= C::kNA) {
                ok = ok && ptx::mbar_wait_cycles(empty_u + 8 * old.s, old.parity, kWait);
                old.advance(1, NS);
            }
            if (!__all_sync(0xffffffffu, ok)) break;
            ptx::tc_fence_after_sync();
#pragma unroll
            for (int hh = 0; hh < 2 / C::kConvSets; ++hh) {
                const int h = C::kConvSets == 2 ? set : hh;
                const uint8_t *raw = raw0 + r.s * stage_bytes + h * lin::kHalfBytes;
                uint32_t f[32];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(raw + c * 1024 + ((n64 ^ (2 * c)) << 4));
                    lin::to_h4(v.x, f[4 * c], f[4 * c + 1]);
                    lin::to_h4(v.y, f[4 * c + 2], f[4 * c + 3]);
                    lin::to_h4(v.z, f[16 + 4 * c], f[16 + 4 * c + 1]);
                    lin::to_h4(v.w, f[16 + 4 * c + 2], f[16 + 4 * c + 3]);
                }
                ptx::tmem_st32(at0 + (uint32_t)(aa.s * kACols + h * 32), f);
            }
            ptx::tmem_wait_st();
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(afull_u + 8 * aa.s);
            r.advance(1, NS);
            aa.advance(1, C::kNA);
        }
    } else {
        // ---- drains ----
        const int q = warp & 3, set = warp >> 2;
        const int col = 32 * q + lane;              // packed column of the tile
        const int per = RT / C::kDrainSets;         // rows of a drain thread, a multiple of 16
        const int row_off = set * per;
        const uint32_t tlane = tbase + ((uint32_t)(32 * q) << 16) + (uint32_t)row_off;
        float *st = out_rows + warp * kOutRows * kOutPitch;
        Ring dd;
        bool ok = true;
        for (int t = first; t < total; t += stride) {
            const TilePos p = tile_pos(t, ntiles, nrt);
            const int t64 = 2 * p.nt + (q >> 1);
            // this column's scales, one per group (a tile's missing second half: any)
            const uint8_t *sp = static_cast<const uint8_t *>(a.packed) +
                                ((long long)(t64 < tiles64 ? t64 : 0) * nblocks + b0) * unit + 2 * lin::kHalfBytes +
                                (col & 63) * 2;
            int sub = 0;
            auto next_scale = [&]() -> unsigned short {  // converted where it is used, a group after it was asked for
                const unsigned short v = __ldcg(reinterpret_cast<const unsigned short *>(sp));
                if (GPS == 1 || ++sub == GPS) {
                    sub = 0;
                    sp += unit - (GPS - 1) * (lin::kTileN * 2);
                } else {
                    sp += lin::kTileN * 2;
                }
                return v;
            };
            const long long row0 = (long long)p.rt * RT + row_off, packed0 = (long long)p.nt * kM + 32 * q;
            const int nrows = (int)max(0ll, min((long long)per, a.rows - row0));
            // residuals by 16 bytes where the addresses allow it
            const __half *res = static_cast<const __half *>(a.residual) + row0 * a.residual_stride + packed0;
            const bool vec_res = a.residual && packed0 + 32 <= a.n && a.residual_stride % 8 == 0 &&
                                 (reinterpret_cast<uintptr_t>(a.residual) & 15) == 0;
            if (vec_res)  // on their way to L2 while the tile is computed
                for (int r = lane; r < nrows; r += 32)
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(res + (long long)r * a.residual_stride));
            float acc[C::kAcc];
#pragma unroll
            for (int i = 0; i < C::kAcc; ++i) acc[i] = 0.f;
            unsigned short sc = next_scale();
            const int ngroups = steps * GPS;
            for (int g = 0; g < ngroups; ++g, dd.advance(1, 2)) {
                const unsigned short sraw = sc;
                if (g + 1 < ngroups) sc = next_scale();
                ok = ok && __all_sync(0xffffffffu, ptx::mbar_wait_cycles(dfull_u + 8 * dd.s, dd.parity, kWait));
                if (!ok) continue;
                ptx::tc_fence_after_sync();
                const float sf = __half2float(__ushort_as_half(sraw));
#pragma unroll
                for (int c = 0; c < C::kAcc / 16; ++c) {
                    if (c * 16 < per) {
                        uint32_t v[16];
                        tmem_ld16(tlane + (uint32_t)(dd.s * C::kRows + c * 16), v);
                        tmem_wait_ld16(v);
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            acc[c * 16 + i] = fmaf(__uint_as_float(v[i]), sf, acc[c * 16 + i]);
                    }
                }
                if (g + 1 == ngroups && csplit == 1) break;  // the accumulator stays until the tile is written
                ptx::tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(dempty_u + 8 * dd.s);
            }
            if (csplit > 1) {  // the CTA's one tile: its sums to the ring (every step is consumed)
                if (!ok) s_failed = 1;
                float *part = reinterpret_cast<float *>(smem);
#pragma unroll
                for (int i = 0; i < C::kAcc; ++i)
                    if (i < per) part[(row_off + i) * kM + col] = acc[i];
                break;
            }
            // ---- epilogue: the sums back to the last group's accumulator, then
            // 16 rows at a time through shared memory, in a loop that is not
            // unrolled: from registers it would have to be, and its code with
            // the activations then outgrows the instruction cache (94,000
            // cycles a tile) ----
            const uint32_t tsum = tlane + (uint32_t)(dd.s * C::kRows);
#pragma unroll
            for (int c = 0; c < C::kAcc / 16; ++c)
                if (c * 16 < per) tmem_st16(tsum + (uint32_t)(c * 16), acc + c * 16);
            ptx::tmem_wait_st();
            const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
            uint4 q0 = zero, q1 = zero;
            auto load_res = [&](int c) {
                const int r = c * 16 + (lane >> 1);
                if (vec_res && r < nrows) {
                    const uint4 *src = reinterpret_cast<const uint4 *>(res + (long long)r * a.residual_stride + (lane & 1) * 16);
                    q0 = src[0];
                    q1 = src[1];
                }
            };
            load_res(0);
#pragma unroll 1
            for (int c = 0; c * 16 < nrows; ++c) {
                uint32_t v[16];
                tmem_ld16(tsum + (uint32_t)(c * 16), v);
                tmem_wait_ld16(v);
                if (!ok)  // not from TMEM, where a UMMA may still be adding
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = 0x7fffffffu;
#pragma unroll
                for (int i = 0; i < 16; ++i) st[i * kOutPitch + lane] = __uint_as_float(v[i]);
                __syncwarp();
                const uint4 p0 = q0, p1 = q1;
                load_res(c + 1);  // the next rows' residuals
                if (a.gated)
                    write_rows_act<true>(a, st, lane, row0 + c * 16, min(16, nrows - c * 16), packed0, false, p0, p1);
                else
                    write_rows_act<false>(a, st, lane, row0 + c * 16, min(16, nrows - c * 16), packed0, vec_res, p0, p1);
                __syncwarp();
            }
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(dempty_u + 8 * dd.s);
            dd.advance(1, 2);
        }
    }

    __syncwarp();
    ptx::tc_fence_before_sync();
    __syncthreads();
    if (warp == C::kMma) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc(tbase, C::kTmemCols);
    }
    if (csplit > 1) {
        // ---- the parts of K, in rank order, and the epilogue ----
        cg::cluster_group cluster = cg::this_cluster();
        if (s_failed)  // NaN, not a wrong number; here, where no copy lands in the ring any more
            for (int i = threadIdx.x; i < RT * kM; i += C::kThreads)
                reinterpret_cast<float *>(smem)[i] = __int_as_float(0x7fffffff);
        __syncwarp();
        cluster.sync();
        const TilePos p = tile_pos(first, ntiles, nrt);
        const float *part = reinterpret_cast<const float *>(smem);
        const int nrows = min(RT, a.rows - p.rt * RT), chunks = a.gated ? kM / 8 : kM / 4;  // fours of outputs
        // every CTA's four sums asked for at once, added in rank order
        auto total4 = [&](const float *mine, float (&t)[4]) {
            float4 x[kMaxSplit];
#pragma unroll
            for (int k = 0; k < kMaxSplit; ++k)
                if (k < csplit) x[k] = *reinterpret_cast<const float4 *>(cluster.map_shared_rank(mine, k));
            t[0] = t[1] = t[2] = t[3] = 0.f;
#pragma unroll
            for (int k = 0; k < kMaxSplit; ++k)
                if (k < csplit) {
                    t[0] += x[k].x;
                    t[1] += x[k].y;
                    t[2] += x[k].z;
                    t[3] += x[k].w;
                }
        };
        for (int i = rank * C::kThreads + threadIdx.x; i < nrows * chunks; i += csplit * C::kThreads) {
            const int r = i / chunks, c = i % chunks;
            const long long n0 = ((long long)p.nt * chunks + c) * 4, row = (long long)p.rt * RT + r;
            if (n0 >= a.n) continue;
            const float *mine = part + r * kM + (a.gated ? (c >> 1) * 16 + (c & 1) * 4 : 4 * c);
            float v[4], u[4] = {0.f, 0.f, 0.f, 0.f};
            total4(mine, v);
            if (a.gated) total4(mine + 8, u);
            switch (a.act) {
            case 1: finish4<1>(a, v, u, row, n0); break;
            case 2: finish4<2>(a, v, u, row, n0); break;
            case 3: finish4<3>(a, v, u, row, n0); break;
            case 4: finish4<4>(a, v, u, row, n0); break;
            default: finish4<0>(a, v, u, row, n0);
            }
        }
        __syncwarp();
        cluster.sync();  // no CTA leaves while another may still read its shared memory
    }
}

template <typename C, int GPS>
cudaError_t launch_g(const LinearArgs &a, unsigned grid, cudaStream_t s) {
    static std::atomic<unsigned long long> done{0};  // devices whose shared-memory limit is set
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(done.load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(linear_tc_kernel<C, GPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
        if (e != cudaSuccess) return e;
        done.fetch_or(bit, std::memory_order_acq_rel);
    }
    Map xmap;
    e = encode_tensor_map_2d(&xmap, true, a.x, (unsigned long long)a.k, (unsigned long long)a.rows,
                             (unsigned long long)a.x_stride * 2, 64, (unsigned)a.row_tile);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)a.csplit;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, linear_tc_kernel<C, GPS>, a, xmap);
}

template <typename C>
cudaError_t launch_t(const LinearArgs &a, unsigned grid, cudaStream_t s) {
    return a.group == 32 ? launch_g<C, 4>(a, grid, s) : a.group == 64 ? launch_g<C, 2>(a, grid, s) : launch_g<C, 1>(a, grid, s);
}

// Few rows: the weight stream asks for two CTAs' converters and issuers per SM
// (10 warps of 96 registers each; 32 rows x 4096 x 14336 gated 27 us against
// 31.6 with two issuers a CTA, whose 80 registers spill, and 36 with one CTA,
// measured beside one another; the present build takes 28.7 to 33 by box and
// clocks).
// Many: the sums ask for drains (64 rows a thread; 80 and 96 measured 5 % and
// more slower at 8192 x 4096 x 4096 and ragged sizes).
using Small = Cfg<32, 2, 4, 4, 1, 2>;
using Medium = Cfg<64, 2, 8, 4, 2, 1>;
using Large = Cfg<128, 2, 4, 8, 2, 1>;

}  // namespace

cudaError_t launch_linear_tc(LinearArgs a, int num_sms, cudaStream_t s) {
    const int nrt = (a.rows + Large::kRows - 1) / Large::kRows;
    a.row_tile = ((a.rows + nrt - 1) / nrt + 31) / 32 * 32;
    const long long ntiles = (lin::tiles(a.n, a.gated != 0) + 1) / 2;
    const long long total = ntiles * ((a.rows + a.row_tile - 1) / a.row_tile);
    const bool small = a.row_tile <= Small::kRows;
    const long long slots = (long long)num_sms * (small ? Small::kPerSm : Large::kPerSm);
    const int nblocks = lin::blocks(a.k);
    a.csplit = 1;
    while (a.csplit < kMaxSplit && total * a.csplit * 2 <= slots && nblocks / (a.csplit * 2) >= 4) a.csplit *= 2;
    const unsigned grid = (unsigned)(a.csplit > 1 ? total * a.csplit : std::min<long long>(total, slots));
    return small ? launch_t<Small>(a, grid, s)
           : a.row_tile <= Medium::kRows ? launch_t<Medium>(a, grid, s)
                                         : launch_t<Large>(a, grid, s);
}

}  // namespace tllm
