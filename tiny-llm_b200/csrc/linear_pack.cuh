// Layout of the weights of tl_linear / tl_linear_gated, as tl_linear_pack
// writes them and both product kernels read them.
//
// The packed columns come in tiles of 64 and K in blocks of 128; unit
// (tile t, block b) is kUnit(group) contiguous bytes at
// (t * blocks + b) * kUnit(group): first the two 64-row halves of the block,
// 4096 bytes each, then the block's scales, fp16 [128 / group][64]. In a half,
// column c of the tile has four 16-byte chunks; chunk j holds rows 8j..8j+7
// and 32+8j..32+8j+7 at byte j * 1024 + (c ^ 2j) * 16, each weight as its
// value plus 128. A chunk is what one lane feeds to four m16n8k16 steps (two
// in each 32 rows, so that a scale group of 32 ends between steps), the XOR
// spreads the eight lanes of a shared-memory phase over all banks, and the
// excess-128 form turns into fp16 with one byte permute and one subtraction.
// Rows and columns past the matrix hold weight 0 and scale 0.
//
// A gated pair shares the columns: packed columns 16i..16i+7 are the gate's
// 8i..8i+7, 16i+8..16i+15 the same columns of the other projection, so one
// MMA tile (and one lane of it) holds both numbers of an output.
#pragma once

#include <cstdint>
#ifdef __CUDACC__
#include <cuda_fp16.h>
#endif

namespace tllm {
namespace lin {

constexpr int kTileN = 64;    // packed columns of a tile
constexpr int kBlockK = 128;  // rows of a block
constexpr int kHalfBytes = 4096;

__host__ __device__ constexpr int unit_bytes(int group) { return 2 * kHalfBytes + kTileN * 2 * (kBlockK / group); }
__host__ __device__ constexpr long long packed_columns(int n, bool gated) {
    return gated ? 16ll * ((n + 7ll) / 8) : (long long)n;
}
__host__ __device__ constexpr long long tiles(int n, bool gated) {
    return (packed_columns(n, gated) + kTileN - 1) / kTileN;
}
__host__ __device__ constexpr int blocks(int k) { return (int)((k + (long long)kBlockK - 1) / kBlockK); }

#ifdef __CUDACC__
// 4 excess-128 bytes (one word) -> 4 fp16 (two words), exactly: the byte in
// the mantissa of 1024.0, minus 1152.
__device__ __forceinline__ void to_h4(uint32_t w, uint32_t &lo, uint32_t &hi) {
    uint32_t a, b;
    asm("prmt.b32 %0, %1, %2, 0x5140;" : "=r"(a) : "r"(w), "r"(0x64646464u));
    asm("prmt.b32 %0, %1, %2, 0x7362;" : "=r"(b) : "r"(w), "r"(0x64646464u));
    const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
    const __half2 ha = __hsub2(*reinterpret_cast<const __half2 *>(&a), off);
    const __half2 hb = __hsub2(*reinterpret_cast<const __half2 *>(&b), off);
    lo = *reinterpret_cast<const uint32_t *>(&ha);
    hi = *reinterpret_cast<const uint32_t *>(&hb);
}

// The activations of the epilogue, in fp32.
__device__ __forceinline__ float activate(int act, float v) {
    switch (act) {
    case 1: return v > 0.f ? v : (v != v ? v : 0.f);  // relu; NaN stays NaN
    // 1 + erf(t) = erfc(-t) and (1 + tanh(t)) / 2 = 1 / (1 + exp(-2t)): no
    // cancellation where the result is small
    case 2: return 0.5f * v * erfcf(-0.70710678118654752f * v);
    // (the exponential and the division by the fast forms: a few fp32 units,
    // next to the output's 2^-11)
    case 3: return __fdividef(v, 1.f + __expf(-1.5957691216057308f * (v + 0.044715f * v * v * v)));
    case 4: return __fdividef(v, 1.f + __expf(-v));
    default: return v;
    }
}

#endif  // __CUDACC__

}  // namespace lin
}  // namespace tllm
