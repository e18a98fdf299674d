// Matrices in microscaled 4-bit numbers (MXFP4 of the Open Compute Project's MX formats): 32 consecutive values of a row share a
// power of two 2^(s - 127), held in a byte s (E8M0, 255: not a number), and each value is a 4-bit number (E2M1: sign, 0 1/2 1 3/2 2 3 4 6).
//
// Layout, made for the products: tiles of 8 rows by 128 k, [matrix][N / 8][K / 128], both rounded up (rows and values past the matrix
// are zeros). A word of codes holds eight consecutive values of a row, those of even places in its lower half, those of odd places in its
// upper one. A tile's codes are 512 bytes, [row r][quarter t of 4][block b of 4]: the word of row r's values 32 b + 8 t .. + 7. So 16 bytes at (r, t)
// are what lane (r, t) of a warp multiplies in an MMA of each of the tile's four blocks, and 64 bytes what a lane of tensor memory needs. Behind the
// codes of all tiles come their scales, 32 bytes a tile, [row][block], as t = s + 1 (255 stays): the exponent of a 32-bit number, 2^(t - 127), which
// is twice the scale and a normal number for every s.
#pragma once
#include "common.cuh"

namespace tl {
namespace mx {

constexpr int BLOCK = 32;           // values a scale
constexpr int TILE_ROWS = 8;
constexpr int TILE_K = 128;
constexpr int TILE_CODES = TILE_ROWS * TILE_K / 2;             // bytes
constexpr int TILE_SCALES = TILE_ROWS * TILE_K / BLOCK;

__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// As bfloat16 numbers, exactly. With a code's lower three bits at the lowest exponent bits and the highest mantissa bit a bfloat16 number is
// value * 2^-126 (E2M1's subnormal falls on bfloat16's), and one multiplication by 2^(t - 2) makes it the value. `factor` is 2^(min(t, NEAR) - 2)
// twice in a word, `factor_left` what is missing where t > NEAR (not a number for 255).
constexpr uint32_t NEAR = 129;
__device__ __forceinline__ uint32_t factor(uint32_t t) { return (min(t, NEAR) + 125u) * 0x00800080u; }
__device__ __forceinline__ uint32_t factor_left(uint32_t t) {
  return t <= NEAR ? 0x3F803F80u : t == 255u ? 0x7FFF7FFFu : (t - 2u) * 0x00800080u;
}
// The four pairs of a word, times `f`: pair j is values 2 j (lower half) and 2 j + 1. A pair alone in its word times two powers of two is its sign at a
// half's top and its other bits at their place, beside copies that the mask takes away: a multiplication, which another pipe than the logic does.
__device__ __forceinline__ void values(uint32_t w, uint32_t f, uint32_t (&v)[4]) {
  constexpr uint32_t SIGN = 0x80008000u, REST = 0x01C001C0u;
  const uint32_t y = w >> 6;
  v[0] = mul2((w & 0x000F000Fu) * (4096u + 64u) & (SIGN | REST), f);
  v[1] = mul2((w & 0x00F000F0u) * (256u + 4u) & (SIGN | REST), f);
  v[2] = mul2((y & 0x003C003Cu) * (1024u + 16u) & (SIGN | REST), f);
  v[3] = mul2((w & SIGN) | (y & REST), f);
}

// As float16 numbers without their scale, pairs as the conversion finds them in the word's bytes: values (0, 2), (4, 6), (1, 3), (5, 7).
__device__ __forceinline__ void values16(uint32_t w, uint32_t (&v)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\tcvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(w));
}
// Twice the scale of block b from a row's four in a word, in 32 bits; infinite for 255, which the zeros that such a block has for codes make a NaN.
__device__ __forceinline__ float scale32(uint32_t four, int b) {
  return __uint_as_float((b < 3 ? four << (23 - 8 * b) : four >> 1) & 0x7F800000u);
}

// A launch that, with `behind`, may begin before the kernel in front of it in the stream has ended (programmatic dependent launch); the kernel waits
// for that one's end itself (chain_wait). For the kernels of one call behind one another: the second's CTAs are on their SMs when the first's leave.
template <typename... KernelArgs, typename... Args>
inline int launch_behind(bool behind, void (*kernel)(KernelArgs...), dim3 grid, int threads, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = behind || chained_launches() ? 1 : 0;
  return (int)cudaLaunchKernelEx(&cfg, kernel, static_cast<KernelArgs>(args)...);
}

}  // namespace mx
}  // namespace tl
