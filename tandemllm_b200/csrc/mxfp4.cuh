// Matrices in microscaled 4-bit numbers (MXFP4 of the Open Compute Project's MX formats): 32 consecutive values of a row share a
// power of two 2^(s - 127), held in a byte s (E8M0, 255: not a number), and each value is a 4-bit number (E2M1: sign, 0 1/2 1 3/2 2 3 4 6).
//
// Layout, made for the products: tiles of 8 rows by 128 k, [matrix][N / 8][K / 128], both rounded up (rows and values past the matrix
// are zeros). A tile's codes are 512 bytes, [k-block of 32][row][16 bytes], so that 32 lanes that take a row's 32 values each read them
// in one go, whether as 8 rows by 4 blocks (the MMA fragments of a warp) or as 32 rows of one block (the lanes of tensor memory); its
// scales are 32 bytes, [row][k-block].
//
// A 32-bit word holds eight consecutive values; of the pair j (values 2 j and 2 j + 1) the first lies in the lower and the second in the
// upper half of the word, at the bits where a bfloat16 has its sign, its two lowest exponent bits and its highest mantissa bit, moved
// down by 3 j (j < 3): a shift and a mask make a pair of bfloat16 numbers that are value * 2^-126 (E2M1's subnormal falls on bfloat16's), and one
// multiplication by 2^(s - 1) makes them the values, exactly. What is left for pair 3 is bit 14 (sign) and 13, 11, 10.
#pragma once
#include "common.cuh"

namespace tl {
namespace mx {

constexpr int BLOCK = 32;           // values a scale
constexpr int TILE_ROWS = 8;
constexpr int TILE_K = 128;
constexpr int TILE_CODES = TILE_ROWS * TILE_K / 2;             // bytes
constexpr int TILE_SCALES = TILE_ROWS * TILE_K / BLOCK;

// The factors of a block with scale code s: 2^(min(s, 128) - 1) twice in a word; and what is left where s > 128 (not a number for 255).
__device__ __forceinline__ uint32_t factor(uint32_t s) { return (min(s, 128u) + 126u) * 0x00800080u; }
__device__ __forceinline__ uint32_t factor_left(uint32_t s) {
  return s <= 128u ? 0x3F803F80u : s == 255u ? 0x7FFF7FFFu : (s - 1u) * 0x00800080u;
}

__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// The four pairs of a word, times `f`.
__device__ __forceinline__ void values(uint32_t w, uint32_t f, uint32_t (&v)[4]) {
  constexpr uint32_t MASK = 0x81C081C0u;
  v[0] = mul2(w & MASK, f);
  v[1] = mul2((w << 3) & MASK, f);
  v[2] = mul2((w << 6) & MASK, f);
  v[3] = mul2(((w << 1) & 0x80008000u) | ((w >> 4) & 0x00C000C0u) | ((w >> 5) & 0x01000100u), f);
}

// The word of eight E2M1 codes that lie as four in each half, pair j at bits 4 j .. 4 j + 3.
__device__ __forceinline__ uint32_t placed(uint32_t n) {
  return ((n & 0x00080008u) << 12) | ((n & 0x00070007u) << 6) |            // pair 0
         ((n & 0x00800080u) << 5) | ((n & 0x00700070u) >> 1) |             // pair 1
         ((n & 0x08000800u) >> 2) | ((n & 0x07000700u) >> 8) |             // pair 2
         ((n & 0xC000C000u) >> 1) | ((n & 0x30003000u) >> 2);              // pair 3
}

}  // namespace mx
}  // namespace tl
