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

// Eight consecutive numbers of a row as they lie.
template <typename T> struct Eight;
template <> struct Eight<bf16> {
  uint4 v;
  __device__ __forceinline__ void load(const bf16* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float (&f)[8]) const { unpack8(v, f); }
};
template <> struct Eight<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const float4*>(p);
    b = *reinterpret_cast<const float4*>(p + 4);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  }
};

// A block of 8 warps 8 rows, a warp every eighth of their tiles of 128 k, two rows at a time: 16 lanes a row, four lanes a block of values,
// eight values and one word of codes a lane. Both sides of memory are then read and written in whole sectors.
constexpr int CODER_WARPS = 8;
struct Place {
  unsigned row_tile, group;   // among all matrices' row tiles; the matrix
  int row, k, at, scale_at;   // the lane's first row and, in a tile, its first value, the word of codes that holds it, its block's scale
  __device__ __forceinline__ explicit Place(int row_tiles) {
    row_tile = blockIdx.x;
    group = row_tile / (unsigned)row_tiles;
    const int lane = threadIdx.x & 31, piece = lane & 15;
    row = (int)(row_tile - group * (unsigned)row_tiles) * TILE_ROWS + (lane >> 4);
    k = piece * 8;
    at = (lane >> 4) * 16 + (piece & 3) * 4 + (piece >> 2);
    scale_at = (lane >> 4) * (TILE_K / BLOCK) + (piece >> 2);
  }
};

template <typename T, bool WHOLE>
__global__ void __launch_bounds__(CODER_WARPS * 32, 4) quantize_kernel(const T* __restrict__ w, long long ld, long long ld_group,
                                                                    uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int N, int K,
                                                                       int row_tiles, int k_tiles) {
  const Place to(row_tiles);
  const T* from = w + to.group * ld_group + (long long)to.row * ld + to.k;
  for (int c = threadIdx.x >> 5; c < k_tiles; c += CODER_WARPS) {
    const long long tile = (long long)to.row_tile * k_tiles + c;
    const int left = K - c * TILE_K - to.k;
    float v[4][8];
    if (WHOLE && left >= 8 && to.row + 6 < N) {
      Eight<T> e[4];                            // (all four loads on their way before the first is looked at)
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i].load(from + 2 * i * ld + c * TILE_K);
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i].get(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = to.row + 2 * i < N && j < left ? to_f32(from[2 * i * ld + c * TILE_K + j]) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[i][j]) & 0x7FFFFFFFu);      // (a NaN's bits are above an infinity's)
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const uint32_t e = top >> 23;
      const bool finite = e < 255u;
      const uint32_t t = finite ? max(e, 2u) - 1u : 255u;
      const float inverse = __uint_as_float((255u - min(t, 254u)) << 23);                       // 2^(128 - t), a normal number
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = v[i][j] * inverse;
      const uint32_t word = finite ? encode4(y[2], y[0], y[6], y[4], y[3], y[1], y[7], y[5]) : 0u;
      reinterpret_cast<uint32_t*>(codes + tile * TILE_CODES)[to.at + 32 * i] = word;
      if ((threadIdx.x & 3) == 0) scales[tile * TILE_SCALES + to.scale_at + 2 * i * (TILE_K / BLOCK)] = (uint8_t)t;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(CODER_WARPS * 32) values_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                                  T* __restrict__ out, int N, int K, int row_tiles, int k_tiles, int whole) {
  const Place at(row_tiles);
  T* to = out + ((long long)at.group * N + at.row) * K + at.k;
  for (int c = threadIdx.x >> 5; c < k_tiles; c += CODER_WARPS) {
    const long long tile = (long long)at.row_tile * k_tiles + c;
    const int left = K - c * TILE_K - at.k;
    uint32_t word[4], s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      word[i] = reinterpret_cast<const uint32_t*>(codes + tile * TILE_CODES)[at.at + 32 * i];
      s[i] = scales[tile * TILE_SCALES + at.scale_at + 2 * i * (TILE_K / BLOCK)];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (at.row + 2 * i >= N) continue;
      const uint32_t more = factor_left(s[i]);
      uint32_t v[4];
      values(word[i], factor(s[i]), v);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = mul2(v[j], more);
      T* p = to + 2 * i * (long long)K + c * TILE_K;
      if (whole && left >= 8) {
        if constexpr (sizeof(T) == 2) {
          *reinterpret_cast<uint4*>(p) = make_uint4(v[0], v[1], v[2], v[3]);
        } else {
          reinterpret_cast<uint4*>(p)[0] = make_uint4(v[0] << 16, v[0] & 0xFFFF0000u, v[1] << 16, v[1] & 0xFFFF0000u);
          reinterpret_cast<uint4*>(p)[1] = make_uint4(v[2] << 16, v[2] & 0xFFFF0000u, v[3] << 16, v[3] & 0xFFFF0000u);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < left) p[j] = from_f32<T>(__uint_as_float(j & 1 ? v[j >> 1] & 0xFFFF0000u : v[j >> 1] << 16));
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
  const long long blocks = (long long)groups * row_tiles;
  TL_REQUIRE(blocks <= 0x7FFFFFFF, "mxfp4: %lld tiles of rows are too many", blocks);
  const int size = dtype == TL_FP32 ? 4 : 2;
  const bool whole = ((uintptr_t)w % 16) == 0 && ld * size % 16 == 0 && ld_group * size % 16 == 0;
#define TL_QUANTIZE(T_, W_)                                                                                                        \
  mx::quantize_kernel<T_, W_><<<(unsigned)blocks, 256, 0, stream>>>((const T_*)w, ld, ld_group, (uint8_t*)codes, (uint8_t*)scales, N, K, \
                                                                    row_tiles, k_tiles)
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
  const long long blocks = (long long)groups * row_tiles;
  TL_REQUIRE(blocks <= 0x7FFFFFFF, "mxfp4: %lld tiles of rows are too many", blocks);
  const int whole = ((uintptr_t)out % 16) == 0 && (long long)K * (dtype == TL_FP32 ? 4 : 2) % 16 == 0;
  if (dtype == TL_FP32)
    mx::values_kernel<float><<<(unsigned)blocks, 256, 0, stream>>>((const uint8_t*)codes, (const uint8_t*)scales, (float*)out, N, K,
                                                                   row_tiles, k_tiles, whole);
  else
    mx::values_kernel<bf16><<<(unsigned)blocks, 256, 0, stream>>>((const uint8_t*)codes, (const uint8_t*)scales, (bf16*)out, N, K,
                                                                  row_tiles, k_tiles, whole);
  TL_LAUNCH_CHECK();
  return 0;
}
