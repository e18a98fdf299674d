// Matrices into MXFP4 (mxfp4.cuh has the format and the layout) and back.
//
//   s = max(floor(log2(max |v|)) - 2, -127)       over a block of 32 values of a row
//   code = nearest of 0 1/2 1 3/2 2 3 4 6, ties to even, to |v| / 2^s, the largest beyond 6, with v's sign
//
// A block that holds an infinity or a NaN gets the scale that is not a number. All of it is exact: dividing by a power of two is a
// multiplication, and the rounding is the conversion instruction's.
#include "mxfp4.cuh"

namespace tl {
namespace mx {

// codes of a (upper four bits) and b (lower four)
__device__ __forceinline__ uint32_t encode4(float a0, float b0, float a1, float b1, float a2, float b2, float a3, float b3) {
  uint32_t d;
  asm("{\n\t.reg .b8 c0, c1, c2, c3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c0, %1, %2;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c1, %3, %4;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c2, %5, %6;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c3, %7, %8;\n\t"
      "mov.b32 %0, {c0, c1, c2, c3};\n\t}"
      : "=r"(d) : "f"(a0), "f"(b0), "f"(a1), "f"(b1), "f"(a2), "f"(b2), "f"(a3), "f"(b3));
  return d;
}

template <typename T> struct Piece;                                 // 16 bytes of a row
template <> struct Piece<float> { static constexpr int COUNT = 4; };
template <> struct Piece<bf16> { static constexpr int COUNT = 8; };

// One warp a tile of 8 rows by 128 k: lane (g, t) takes block t of row g.
template <typename T, bool WHOLE>
__global__ void __launch_bounds__(256) quantize_kernel(const T* __restrict__ w, long long ld, long long ld_group, uint8_t* __restrict__ codes,
                                                       uint8_t* __restrict__ scales, int N, int K, int row_tiles, int k_tiles,
                                                       long long tiles) {
  const long long tile = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (tile >= tiles) return;
  const int lane = threadIdx.x & 31, g = lane & 7, t = lane >> 3;
  const long long rows_at = tile / k_tiles;
  const int k0 = (int)(tile - rows_at * k_tiles) * TILE_K + t * BLOCK;
  const long long group = rows_at / row_tiles;
  const int row = (int)(rows_at - group * row_tiles) * TILE_ROWS + g;
  const T* from = w + group * ld_group + (long long)row * ld + k0;
  float v[BLOCK];
  if (WHOLE && row < N && k0 + BLOCK <= K) {
#pragma unroll
    for (int i = 0; i < BLOCK; i += Piece<T>::COUNT) {
      const uint4 u = *reinterpret_cast<const uint4*>(from + i);
      if constexpr (sizeof(T) == 2) {
        float f[8];
        unpack8(u, f);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i + j] = f[j];
      } else {
        v[i] = __uint_as_float(u.x), v[i + 1] = __uint_as_float(u.y), v[i + 2] = __uint_as_float(u.z), v[i + 3] = __uint_as_float(u.w);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < BLOCK; ++i) v[i] = row < N && k0 + i < K ? to_f32(from[i]) : 0.f;
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < BLOCK; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);       // (a NaN's bits are above an infinity's)
  const uint32_t e = top >> 23;
  const bool finite = e < 255u;
  const uint32_t s = finite ? max(e, 2u) - 2u : 255u;
  const float inverse = finite ? __uint_as_float((254u - s) << 23) : 0.f;                     // 2^(127 - s), a normal number: s <= 252
  uint32_t out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = finite ? v[8 * i + j] * inverse : 0.f;
    out[i] = placed(encode4(y[2], y[0], y[6], y[4], y[3], y[1], y[7], y[5]));
  }
  reinterpret_cast<uint4*>(codes + tile * TILE_CODES)[t * TILE_ROWS + g] = make_uint4(out[0], out[1], out[2], out[3]);
  scales[tile * TILE_SCALES + g * (TILE_K / BLOCK) + t] = (uint8_t)s;
}

template <typename T>
__global__ void __launch_bounds__(256) values_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, T* __restrict__ out,
                                                     int N, int K, int row_tiles, int k_tiles, long long tiles, int whole) {
  const long long tile = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (tile >= tiles) return;
  const int lane = threadIdx.x & 31, g = lane & 7, t = lane >> 3;
  const long long rows_at = tile / k_tiles;
  const int k0 = (int)(tile - rows_at * k_tiles) * TILE_K + t * BLOCK;
  const long long group = rows_at / row_tiles;
  const int row = (int)(rows_at - group * row_tiles) * TILE_ROWS + g;
  if (row >= N || k0 >= K) return;
  const uint4 c = reinterpret_cast<const uint4*>(codes + tile * TILE_CODES)[t * TILE_ROWS + g];
  const uint32_t s = scales[tile * TILE_SCALES + g * (TILE_K / BLOCK) + t];
  const uint32_t f = factor(s), left = factor_left(s), word[4] = {c.x, c.y, c.z, c.w};
  T* to = out + (group * N + row) * (long long)K + k0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t v[4];
    values(word[i], f, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = mul2(v[j], left);
    if (whole && k0 + BLOCK <= K) {
      if constexpr (sizeof(T) == 2) {
        reinterpret_cast<uint4*>(to)[i] = make_uint4(v[0], v[1], v[2], v[3]);
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j)
          reinterpret_cast<uint4*>(to)[2 * i + j] =
              make_uint4(v[2 * j] << 16, v[2 * j] & 0xFFFF0000u, v[2 * j + 1] << 16, v[2 * j + 1] & 0xFFFF0000u);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t bits = j & 1 ? v[j >> 1] & 0xFFFF0000u : v[j >> 1] << 16;
        if (k0 + 8 * i + j < K) to[8 * i + j] = from_f32<T>(__uint_as_float(bits));
      }
    }
  }
}

}  // namespace mx
}  // namespace tl

using namespace tl;

extern "C" const char* tl_mx_last_error() { return tl_error_text; }

// w [groups, N, K] of 32-bit (TL_FP32) or bfloat16 numbers, rows `ld` and matrices `ld_group` elements apart, into codes and scales.
extern "C" int tl_mxfp4_quantize(const void* w, long long ld, long long ld_group, int dtype, void* codes, void* scales, int groups, int N,
                                 int K, cudaStream_t stream) {
  if (groups == 0 || N == 0 || K == 0) return 0;
  TL_REQUIRE(groups > 0 && N > 0 && K > 0 && K <= 0x7FFFFF00, "mxfp4: %d matrices of %d x %d", groups, N, K);
  TL_REQUIRE(dtype == TL_FP32 || dtype == TL_BF16, "mxfp4: elements of type %d", dtype);
  const int row_tiles = ceil_div(N, mx::TILE_ROWS), k_tiles = ceil_div(K, mx::TILE_K);
  const long long tiles = (long long)groups * row_tiles * k_tiles, blocks = ceil_div64(tiles, 8);
  TL_REQUIRE(blocks <= 0x7FFFFFFF, "mxfp4: %lld tiles are too many", tiles);
  const int size = dtype == TL_FP32 ? 4 : 2;
  const bool whole = ((uintptr_t)w % 16) == 0 && ld * size % 16 == 0 && ld_group * size % 16 == 0;
#define TL_QUANTIZE(T_, W_)                                                                                                        \
  mx::quantize_kernel<T_, W_><<<(unsigned)blocks, 256, 0, stream>>>((const T_*)w, ld, ld_group, (uint8_t*)codes, (uint8_t*)scales, N, K, \
                                                                    row_tiles, k_tiles, tiles)
  if (dtype == TL_FP32) {
    if (whole) TL_QUANTIZE(float, true);
    else TL_QUANTIZE(float, false);
  } else {
    if (whole) TL_QUANTIZE(bf16, true);
    else TL_QUANTIZE(bf16, false);
  }
#undef TL_QUANTIZE
  TL_LAUNCH_CHECK();
  return 0;
}

// out [groups, N, K], contiguous: the values that codes and scales stand for.
extern "C" int tl_mxfp4_values(const void* codes, const void* scales, void* out, int dtype, int groups, int N, int K, cudaStream_t stream) {
  if (groups == 0 || N == 0 || K == 0) return 0;
  TL_REQUIRE(groups > 0 && N > 0 && K > 0 && K <= 0x7FFFFF00, "mxfp4: %d matrices of %d x %d", groups, N, K);
  TL_REQUIRE(dtype == TL_FP32 || dtype == TL_BF16, "mxfp4: elements of type %d", dtype);
  const int row_tiles = ceil_div(N, mx::TILE_ROWS), k_tiles = ceil_div(K, mx::TILE_K);
  const long long tiles = (long long)groups * row_tiles * k_tiles, blocks = ceil_div64(tiles, 8);
  TL_REQUIRE(blocks <= 0x7FFFFFFF, "mxfp4: %lld tiles are too many", tiles);
  const int whole = ((uintptr_t)out % 16) == 0 && (long long)K * (dtype == TL_FP32 ? 4 : 2) % 16 == 0;
  if (dtype == TL_FP32)
    mx::values_kernel<float><<<(unsigned)blocks, 256, 0, stream>>>((const uint8_t*)codes, (const uint8_t*)scales, (float*)out, N, K,
                                                                   row_tiles, k_tiles, tiles, whole);
  else
    mx::values_kernel<bf16><<<(unsigned)blocks, 256, 0, stream>>>((const uint8_t*)codes, (const uint8_t*)scales, (bf16*)out, N, K,
                                                                  row_tiles, k_tiles, tiles, whole);
  TL_LAUNCH_CHECK();
  return 0;
}
