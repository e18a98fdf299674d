// Products of a few bfloat16 rows with MXFP4 weights (mxfp4.cuh), for decode steps:
//
//   few_kernel      C = X W^T (+ bias), or gated C = act(X G^T + b_g) * (X U^T + b_u)
//   first_kernel    the experts' first half for up to 8 rows: a[p] = act(G_e x) * (U_e x) of every (row, slot) pair p, times the pair's weight
//   second_kernel   their second half: out[r] = sum over r's pairs of D_e a[p], all experts in one sum
//
// Such a product reads every weight once and does little with it, so its time is the weights' bytes or, for a few MB, the length of its
// chain of dependent steps. As in the bfloat16 form (gemm_skinny_mma.cu) there is no staging: a lane loads 32 values of a row and their scale
// (16 bytes and 1), makes them bfloat16 numbers in its registers (15 instructions for eight) and multiplies them with mma.sync m16n8k16 by the
// same 32 numbers of a token row, which it loads as they lie; k's order within an MMA is any, as long as both operands have the same.
// The warps of a CTA split k in tiles of 128, and their 32-bit sums are added in warp order through shared memory, so results do not
// depend on timing.
#include "mxfp4.cuh"

namespace tl {
namespace mx {

constexpr int WARPS = 8;
constexpr int MAX_PAIRS = 256;      // of the experts' form
constexpr int MAX_ROWS = 8;

__device__ __forceinline__ void mma_16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes where valid, else zeros. Volatile: a round's loads stay in front of its MMAs, all in flight together.
__device__ __forceinline__ uint4 load16(const void* p, bool valid) {
  uint4 v;
  asm volatile(
      "{\n\t.reg .pred ok;\n\t"
      "setp.ne.b32 ok, %5, 0;\n\t"
      "mov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
      "@ok ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
      : "l"(p), "r"((int)valid));
  return v;
}
// Eight numbers of a token row from its element k on, zeros past K and where not valid. WHOLE: rows begin at multiples of 16 bytes and K is a
// multiple of 8, so the eight are in or out; else they are fetched one by one.
template <bool WHOLE>
__device__ __forceinline__ uint4 load_row(const bf16* row, int k, int K, bool valid) {
  if constexpr (WHOLE) return load16(row + k, valid && k < K);
  uint32_t v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool lo = valid && k + 2 * i < K, hi = valid && k + 2 * i + 1 < K;
    const uint32_t a = lo ? __bfloat16_as_ushort(row[k + 2 * i]) : 0u, b = hi ? __bfloat16_as_ushort(row[k + 2 * i + 1]) : 0u;
    v[i] = a | b << 16;
  }
  return make_uint4(v[0], v[1], v[2], v[3]);
}
// 16 bytes of weights, which no kernel writes and no other CTA reads.
__device__ __forceinline__ uint4 load_codes(const uint8_t* p, bool valid) {
  uint4 v;
  asm volatile(
      "{\n\t.reg .pred ok;\n\t"
      "setp.ne.b32 ok, %5, 0;\n\t"
      "mov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
      "@ok ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
      : "l"(p), "r"((int)valid));
  return v;
}
__device__ __forceinline__ uint32_t load_scale(const uint8_t* p, bool valid) {
  uint32_t v;
  asm volatile(
      "{\n\t.reg .pred ok;\n\t"
      "setp.ne.b32 ok, %2, 0;\n\t"
      "mov.b32 %0, 0;\n\t"
      "@ok ld.global.nc.u8 %0, [%1];\n\t}"
      : "=r"(v) : "l"(p), "r"((int)valid));
  return v;
}

// A lane's share of 16 rows by 128 k: 32 values of row g and of row g + 8.
struct Fragment {
  uint4 lo, hi;
  uint32_t s_lo, s_hi;
};

// Lane (g = lane / 4, t = lane % 4) of the tiles at row tile `at` (a tile's place counted in all matrices) and the one below it.
__device__ __forceinline__ void load_fragment(Fragment& f, const uint8_t* codes, const uint8_t* scales, long long tile_lo, long long tile_hi,
                                              int g, int t, bool ok_lo, bool ok_hi) {
  f.lo = load_codes(codes + tile_lo * TILE_CODES + (t * TILE_ROWS + g) * 16, ok_lo);
  f.hi = load_codes(codes + tile_hi * TILE_CODES + (t * TILE_ROWS + g) * 16, ok_hi);
  f.s_lo = load_scale(scales + tile_lo * TILE_SCALES + g * 4 + t, ok_lo);
  f.s_hi = load_scale(scales + tile_hi * TILE_SCALES + g * 4 + t, ok_hi);
}

// acc[j] += the fragment times the 32 numbers a lane holds of its token row in every tile j of eight rows.
template <int NT>
__device__ __forceinline__ void multiply(float (&acc)[NT][4], const Fragment& f, const uint4 (&x)[NT][4]) {
  const uint32_t f_lo = factor(f.s_lo), f_hi = factor(f.s_hi);
  const bool far = __any_sync(0xffffffffu, max(f.s_lo, f.s_hi) > 128u);       // blocks of 8 and more: one multiplication more
  const uint32_t lo[4] = {f.lo.x, f.lo.y, f.lo.z, f.lo.w}, hi[4] = {f.hi.x, f.hi.y, f.hi.z, f.hi.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t a[4], b[4];
    values(lo[i], f_lo, a);
    values(hi[i], f_hi, b);
    if (far) {
      const uint32_t l_lo = factor_left(f.s_lo), l_hi = factor_left(f.s_hi);
#pragma unroll
      for (int j = 0; j < 4; ++j) a[j] = mul2(a[j], l_lo), b[j] = mul2(b[j], l_hi);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      mma_16816(acc[j], a[0], b[0], a[1], b[1], x[j][i].x, x[j][i].y);
      mma_16816(acc[j], a[2], b[2], a[3], b[3], x[j][i].z, x[j][i].w);
    }
  }
}

template <int RT, int NT>
__device__ __forceinline__ void keep(float (&part)[RT][16][8 * NT + 1], const float (&acc)[RT][NT][4], int g, int t) {
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      part[r][g][8 * j + 2 * t] = acc[r][j][0];
      part[r][g][8 * j + 2 * t + 1] = acc[r][j][1];
      part[r][g + 8][8 * j + 2 * t] = acc[r][j][2];
      part[r][g + 8][8 * j + 2 * t + 1] = acc[r][j][3];
    }
}

// 16 outputs a CTA for up to 8 NT rows. `gate` != 0: the second matrix holds the up rows, and `bias` its numbers behind the gate's.
template <int NT, bool GATED, bool WHOLE, int UNROLL, typename TOut>
__global__ void __launch_bounds__(WARPS * 32) few_kernel(const bf16* __restrict__ x, long long ldx, const uint8_t* __restrict__ codes,
                                                         const uint8_t* __restrict__ scales, const float* __restrict__ bias, TOut* __restrict__ out,
                                                         long long ldc, int M, int N, int K, int act, float ga0, float ga1) {
  constexpr int RT = GATED ? 2 : 1;
  __shared__ float part[WARPS][RT][16][8 * NT + 1];
  chain_next();
  chain_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int k_tiles = ceil_div(K, TILE_K), row_tiles = ceil_div(N, TILE_ROWS), row_tile = blockIdx.x * 2;
  const bool ok_hi = row_tile + 1 < row_tiles;
  float acc[RT][NT][4] = {};
  for (int c0 = warp; c0 < k_tiles; c0 += WARPS * UNROLL) {
    Fragment f[UNROLL][RT];
    uint4 b[UNROLL][NT][4];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int c = c0 + u * WARPS;
      const bool in = c < k_tiles;
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const long long at = ((long long)r * row_tiles + row_tile) * k_tiles + (in ? c : 0);
        load_fragment(f[u][r], codes, scales, at, ok_hi ? at + k_tiles : at, g, t, in, in && ok_hi);
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int m = j * 8 + g, k = c * TILE_K + t * BLOCK;
        const bf16* row = x + (long long)(m < M ? m : 0) * ldx;
#pragma unroll
        for (int i = 0; i < 4; ++i) b[u][j][i] = load_row<WHOLE>(row, k + 8 * i, K, m < M);
      }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int r = 0; r < RT; ++r) multiply<NT>(acc[r], f[u][r], b[u]);
  }
  keep<RT, NT>(part[warp], acc, g, t);
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * 8 * NT; i += WARPS * 32) {
    const int row = i & 15, m = i >> 4, n = blockIdx.x * 16 + row;
    if (m >= M || n >= N) continue;
    float v[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      v[r] = 0.f;
#pragma unroll
      for (int s = 0; s < WARPS; ++s) v[r] += part[s][r][row][m];
      if (bias) v[r] += bias[r * N + n];
    }
    out[(long long)m * ldc + n] = from_f32<TOut>(GATED ? gated(v[0], v[RT - 1], act, ga0, ga1) : (act < 0 ? gate_activation(v[0], -act) : v[0]));
  }
}

// ------------------------------------------------------------------------------------------ experts
// The experts of a small step, found by every CTA from the ids: item i is an expert and, for every row that chose it, the pair (row, slot)
// that did. A row that names an expert twice has its second time in an item of its own. Items come in the order in which they first appear.
struct Items {
  int count;
  short expert[MAX_PAIRS];
  short pair[MAX_PAIRS][MAX_ROWS];        // -1: the row did not choose it
  int key[MAX_PAIRS];
  uint32_t firsts[MAX_PAIRS / 32];
};

// All of the CTA's threads (at least MAX_PAIRS where the pairs are more than a warp's); ends with a barrier. An id that names no expert is
// recorded in `status` and its pair counts for nothing.
__device__ __forceinline__ void find_items(Items& s, const int* __restrict__ ids, int pairs, int top, int experts, int* status) {
  const int p = threadIdx.x, lane = p & 31, warp = p >> 5;
  if (pairs <= 32) {
    if (warp == 0) {
      const int id = lane < pairs ? ids[lane] : -1, row = lane / top;
      const bool ok = id >= 0 && id < experts;
      if (lane < pairs && !ok) atomicExch(status, 6);
      for (int i = lane; i < pairs * MAX_ROWS; i += 32) (&s.pair[0][0])[i] = -1;
      const uint32_t same = __match_any_sync(0xffffffffu, ok ? id : -1), before = (1u << lane) - 1u;
      const int again = __popc(same & before & ~((1u << (row * top & 31)) - 1u));      // earlier slots of this row with this expert
      const uint32_t item = __match_any_sync(0xffffffffu, ok ? id * 32 + again : -1);
      const int leader = __ffs(item) - 1;
      const uint32_t firsts = __ballot_sync(0xffffffffu, ok && leader == lane);
      __syncwarp();
      if (ok) {
        const int at = __popc(firsts & ((1u << leader) - 1u));
        s.pair[at][row] = (short)lane;
        if (leader == lane) s.expert[at] = (short)id;
      }
      if (lane == 0) s.count = __popc(firsts);
    }
    __syncthreads();
    return;
  }
  int id = -1, key = -1;
  if (p < pairs) {
    id = ids[p];
    if (id >= 0 && id < experts) {
      int again = 0;
      for (int q = p - p % top; q < p; ++q) again += ids[q] == id;
      key = id * 32 + again;
    } else {
      atomicExch(status, 6);
    }
    s.key[p] = key;
#pragma unroll
    for (int r = 0; r < MAX_ROWS; ++r) s.pair[p][r] = -1;
  }
  __syncthreads();
  int leader = p;
  if (key >= 0)
    for (leader = 0; s.key[leader] != key;) ++leader;
  const uint32_t firsts = __ballot_sync(0xffffffffu, key >= 0 && leader == p);
  if (lane == 0 && warp < MAX_PAIRS / 32) s.firsts[warp] = firsts;
  __syncthreads();
  if (key >= 0) {
    int at = __popc(s.firsts[leader >> 5] & ((1u << (leader & 31)) - 1u));
    for (int i = 0; i < leader >> 5; ++i) at += __popc(s.firsts[i]);
    s.pair[at][p / top] = (short)p;
    if (leader == p) s.expert[at] = (short)id;
  }
  if (p == 0) {
    int n = 0;
    for (int i = 0; i < MAX_PAIRS / 32; ++i) n += __popc(s.firsts[i]);
    s.count = n;
  }
  __syncthreads();
}

// grid (16 outputs, items at most): a CTA takes an item's expert and the rows that chose it. `out` [pairs, ldc], outputs up to ldc (those
// past N come from rows of zeros). `before`: the pair's weight multiplies the sums, in front of the activation, else what comes of them.
template <bool GATED, bool WHOLE, int UNROLL>
__global__ void __launch_bounds__(WARPS * 32) first_kernel(const bf16* __restrict__ x, long long ldx, const uint8_t* __restrict__ codes,
                                                           const uint8_t* __restrict__ scales, bf16* __restrict__ out, int ldc, int N, int K,
                                                           const int* __restrict__ ids, const float* __restrict__ wts, int before, int pairs,
                                                           int top, int experts, int act, float ga0, float ga1, int* status) {
  constexpr int RT = GATED ? 2 : 1;
  __shared__ float part[WARPS][RT][16][8 + 1];
  __shared__ Items items;
  chain_next();
  chain_wait();
  find_items(items, ids, pairs, top, experts, status);
  const int item = blockIdx.y;
  if (item >= items.count) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int k_tiles = ceil_div(K, TILE_K), row_tiles = ceil_div(N, TILE_ROWS), row_tile = blockIdx.x * 2;
  const bool ok_hi = row_tile + 1 < row_tiles;
  const long long matrix = (long long)items.expert[item] * RT;
  const int pair = items.pair[item][g];
  const bf16* row = x + (long long)(pair >= 0 ? pair / top : 0) * ldx;
  float acc[RT][1][4] = {};
  for (int c0 = warp; c0 < k_tiles; c0 += WARPS * UNROLL) {
    Fragment f[UNROLL][RT];
    uint4 b[UNROLL][1][4];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int c = c0 + u * WARPS, k = c * TILE_K + t * BLOCK;
      const bool in = c < k_tiles;
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const long long at = ((matrix + r) * row_tiles + row_tile) * k_tiles + (in ? c : 0);
        load_fragment(f[u][r], codes, scales, at, ok_hi ? at + k_tiles : at, g, t, in, in && ok_hi);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) b[u][0][i] = load_row<WHOLE>(row, k + 8 * i, K, pair >= 0);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int r = 0; r < RT; ++r) multiply<1>(acc[r], f[u][r], b[u]);
  }
  keep<RT, 1>(part[warp], acc, g, t);
  __syncthreads();
  if (threadIdx.x < 16 * MAX_ROWS) {
    const int i = threadIdx.x & 15, m = threadIdx.x >> 4, n = blockIdx.x * 16 + i, p = items.pair[item][m];
    if (p >= 0 && n < ldc) {
      const float weight = wts[p];
      float v[RT];
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        v[r] = 0.f;
#pragma unroll
        for (int s = 0; s < WARPS; ++s) v[r] += part[s][r][i][m];
        if (before) v[r] *= weight;
      }
      const float a = GATED ? gated(v[0], v[RT - 1], act, ga0, ga1) : gate_activation(v[0], act);
      out[(long long)p * ldc + n] = __float2bfloat16_rn(before ? a : a * weight);
    }
  }
}

// 16 outputs a CTA: all experts' products of all rows are one sum, whose terms are the items' tiles of 128 k one item after the other; a
// row that did not choose an item's expert has zeros there.
template <int UNROLL, typename TOut>
__global__ void __launch_bounds__(WARPS * 32) second_kernel(const bf16* __restrict__ a, int lda, const uint8_t* __restrict__ codes,
                                                            const uint8_t* __restrict__ scales, TOut* __restrict__ out, long long ldc, int rows,
                                                            int N, int K, const int* __restrict__ ids, int pairs, int top, int experts,
                                                            int* status) {
  __shared__ float part[WARPS][1][16][8 + 1];
  __shared__ Items items;
  chain_next();
  chain_wait();
  find_items(items, ids, pairs, top, experts, status);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int k_tiles = ceil_div(K, TILE_K), row_tiles = ceil_div(N, TILE_ROWS), row_tile = blockIdx.x * 2;
  const bool ok_hi = row_tile + 1 < row_tiles;
  const int total = items.count * k_tiles;
  float acc[1][1][4] = {};
  for (int u0 = warp; u0 < total; u0 += WARPS * UNROLL) {
    Fragment f[UNROLL];
    uint4 b[UNROLL][1][4];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int unit = u0 + u * WARPS;
      const bool in = unit < total;
      const int item = in ? unit / k_tiles : 0, c = in ? unit - item * k_tiles : 0, k = c * TILE_K + t * BLOCK;
      const long long at = ((long long)(in ? items.expert[item] : 0) * row_tiles + row_tile) * k_tiles + c;
      load_fragment(f[u], codes, scales, at, ok_hi ? at + k_tiles : at, g, t, in, in && ok_hi);
      const int pair = in ? items.pair[item][g] : -1;
      const bf16* row = a + (long long)(pair >= 0 ? pair : 0) * lda + k;
#pragma unroll
      for (int i = 0; i < 4; ++i) b[u][0][i] = load16(row + 8 * i, pair >= 0 && k + 8 * i < lda);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) multiply<1>(acc[0], f[u], b[u]);
  }
  keep<1, 1>(part[warp], acc, g, t);
  __syncthreads();
  if (threadIdx.x < 16 * MAX_ROWS) {
    const int i = threadIdx.x & 15, m = threadIdx.x >> 4, n = blockIdx.x * 16 + i;
    if (m < rows && n < N) {
      float v = 0.f;
#pragma unroll
      for (int s = 0; s < WARPS; ++s) v += part[s][0][i][m];
      out[(long long)m * ldc + n] = from_f32<TOut>(v);
    }
  }
}

}  // namespace mx
}  // namespace tl

using namespace tl;

// x [M, K] bfloat16 (row stride ldx), M <= 32; the matrix N x K (gated: two, gate and up); bias [N] (gated: [2 N]) 32-bit or null; out [M, N]
// (row stride ldc) bfloat16 or 32-bit. `act`: the gate's activation TL_ACT_*, 0 for a plain product, negated an activation on its results.
extern "C" int tl_mxfp4_few(const void* x, long long ldx, const void* codes, const void* scales, const float* bias, void* out, long long ldc,
                            int M, int N, int K, int act, float a0, float a1, int out_dtype, cudaStream_t stream) {
  if (M == 0 || N == 0) return 0;
  TL_REQUIRE(M >= 1 && M <= 32 && N >= 1 && K >= 1, "mxfp4 product of few rows: %d rows x (%d x %d)", M, N, K);
  TL_REQUIRE(act <= 0 ? act >= -TL_ACT_IDENTITY : tl_is_gate(act), "mxfp4 product: gate activation %d is none (nor an ungated one, negated)", act);
  TL_REQUIRE(act <= 0 || out_dtype == TL_BF16, "mxfp4 product: gated outputs of type %d", out_dtype);
  const dim3 grid(ceil_div(N, 16)), block(mx::WARPS * 32);
  const int nt = ceil_div(M, 8);
  const bool whole = K % 8 == 0 && ldx % 8 == 0 && ((uintptr_t)x % 16) == 0;
#define TL_FEW(NT_, G_, W_, U_, T_)                                                                                               \
  return (int)launch_chained(mx::few_kernel<NT_, G_, W_, U_, T_>, grid, block, 0, stream, (const bf16*)x, ldx, (const uint8_t*)codes, \
                             (const uint8_t*)scales, bias, (T_*)out, ldc, M, N, K, act, a0, a1)
#define TL_FEW_(NT_, W_, U_)                                     \
  do {                                                           \
    if (act > 0) TL_FEW(NT_, true, W_, U_, bf16);                \
    if (out_dtype == TL_FP32) TL_FEW(NT_, false, W_, U_, float); \
    TL_FEW(NT_, false, W_, U_, bf16);                            \
  } while (0)
  if (whole) {
    if (nt == 1) TL_FEW_(1, true, 2);
    if (nt == 2) TL_FEW_(2, true, 1);
    TL_FEW_(4, true, 1);
  }
  if (nt == 1) TL_FEW_(1, false, 1);
  if (nt == 2) TL_FEW_(2, false, 1);
  TL_FEW_(4, false, 1);
#undef TL_FEW_
#undef TL_FEW
}

// Routed experts of up to 8 rows and 256 pairs, first half: x [rows, K]; matrices [experts] (or gated [2 experts], gate and up in turn) of N x K;
// out [rows * top, ldc] bfloat16 with ldc = N rounded up to 8.
extern "C" int tl_mxfp4_experts_first(const void* x, long long ldx, const void* codes, const void* scales, void* out, int ldc, int rows, int N,
                                      int K, const int* ids, const float* wts, int before, int top, int experts, int act, float a0, float a1,
                                      int* status, cudaStream_t stream) {
  if (rows == 0 || N == 0) return 0;
  TL_REQUIRE(rows >= 1 && rows <= mx::MAX_ROWS && top >= 1 && rows * top <= mx::MAX_PAIRS && top <= 32 && experts >= 1 && experts <= 1024,
             "mxfp4 experts: %d rows, top-%d of %d", rows, top, experts);
  TL_REQUIRE(N >= 1 && K >= 1 && ldc == ceil_div(N, 8) * 8, "mxfp4 experts: %d x %d, row stride %d", N, K, ldc);
  TL_REQUIRE(act < 0 ? act >= -TL_ACT_IDENTITY : tl_is_gate(act), "mxfp4 experts: gate activation %d is none (nor an ungated one, negated)", act);
  const dim3 grid(ceil_div(N, 16), rows * top), block(mx::WARPS * 32);
#define TL_FIRST(G_, W_, U_)                                                                                                                      \
  return (int)launch_chained(mx::first_kernel<G_, W_, U_>, grid, block, 0, stream, (const bf16*)x, ldx, (const uint8_t*)codes,                    \
                             (const uint8_t*)scales, (bf16*)out, ldc, N, K, ids, wts, before, rows * top, top, experts, act < 0 ? -act : act, \
                             a0, a1, status)
  if (K % 8 == 0 && ldx % 8 == 0 && ((uintptr_t)x % 16) == 0) {
    if (act > 0) TL_FIRST(true, true, 2);
    TL_FIRST(false, true, 2);
  }
  if (act > 0) TL_FIRST(true, false, 1);
  TL_FIRST(false, false, 1);
#undef TL_FIRST
}

// Second half: a [rows * top, lda] (what the first half left, K rounded up to 8); matrices [experts] of N x K; out [rows, N] (row stride ldc).
extern "C" int tl_mxfp4_experts_second(const void* a, int lda, const void* codes, const void* scales, void* out, long long ldc, int rows, int N,
                                       int K, const int* ids, int top, int experts, int out_dtype, int* status, cudaStream_t stream) {
  if (rows == 0 || N == 0) return 0;
  TL_REQUIRE(rows >= 1 && rows <= mx::MAX_ROWS && top >= 1 && rows * top <= mx::MAX_PAIRS && top <= 32 && experts >= 1 && experts <= 1024,
             "mxfp4 experts: %d rows, top-%d of %d", rows, top, experts);
  TL_REQUIRE(N >= 1 && K >= 1 && lda == ceil_div(K, 8) * 8 && ((uintptr_t)a % 16) == 0, "mxfp4 experts: %d x %d, row stride %d", N, K, lda);
  const dim3 grid(ceil_div(N, 16)), block(mx::WARPS * 32);
#define TL_SECOND(T_)                                                                                                        \
  return (int)launch_chained(mx::second_kernel<4, T_>, grid, block, 0, stream, (const bf16*)a, lda, (const uint8_t*)codes,   \
                             (const uint8_t*)scales, (T_*)out, ldc, rows, N, K, ids, rows * top, top, experts, status)
  if (out_dtype == TL_FP32) TL_SECOND(float);
  TL_SECOND(bf16);
#undef TL_SECOND
}
