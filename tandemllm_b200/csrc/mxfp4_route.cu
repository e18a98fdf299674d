// Around the routed experts' products of a step that is too large for the two-kernel form (mxfp4_few.cu): which pairs (row, slot) an expert
// has, its token rows side by side, and the weighed sum of what the experts made of a row.
//
// The kernels begin before the ones in front of them have ended. What those leave is read behind chain_wait() and through pointers that promise
// nothing: of a `const __restrict__` one the compiler may read early, and by the read-only path.
#include "mxfp4.cuh"

namespace tl {
namespace mx {

constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_EXPERTS = 1024;
constexpr int SUM_TOP = 32;

// The sum of `v` over the threads before this one; `total` gets all of it. `scratch`: 33 of them.
__device__ __forceinline__ long long before_me(long long v, long long* scratch, long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long run = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += a;
  }
  if (lane == 31) scratch[warp] = run;
  __syncthreads();
  if (warp == 0) {
    const long long mine = scratch[lane];
    long long sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long a = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += a;
    }
    scratch[lane] = sum - mine;
    if (lane == 31) scratch[32] = sum;
  }
  __syncthreads();
  total = scratch[32];
  return scratch[warp] + run - v;
}

// One block. Pairs of an expert lie together, in any order among themselves: a row's products do not depend on the rows beside it, so the
// order, which the atomics leave open, changes no result. Pairs without an expert come last and are in no tile.
__global__ void __launch_bounds__(PLAN_THREADS) plan_kernel(const int* ids, int pairs, int experts, int tile_rows_at_most, int* sorted, int* place,
                                                            int* tile_group, int* tile_row0, int* tile_rows, int* n_tiles, int* status) {
  __shared__ int at[PLAN_EXPERTS + 1];
  __shared__ long long scratch[33];
  chain_wait();               // (first: what comes behind takes tensor memory before it waits, so nothing in front of the layer may still need any)
  chain_next();
  const int tid = threadIdx.x;
  // Eight ids a thread at once, on their way together; up to 8192 pairs they stay for the second pass. -1: none, else what names no expert is `experts`.
  constexpr int HELD = 8;
  int held[HELD];
  auto load = [&](int p0) {
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
      const int p = p0 + j * PLAN_THREADS;
      held[j] = p < pairs ? ids[p] : -1;
    }
#pragma unroll
    for (int j = 0; j < HELD; ++j)
      if (p0 + j * PLAN_THREADS < pairs && (unsigned)held[j] >= (unsigned)experts) held[j] = experts;
  };
  for (int e = tid; e <= experts; e += PLAN_THREADS) at[e] = 0;
  load(tid);
  __syncthreads();
  for (int p0 = tid; p0 < pairs; p0 += HELD * PLAN_THREADS) {
    if (p0 != tid) load(p0);
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
      if (held[j] >= 0) atomicAdd(&at[held[j]], 1);
      if (held[j] == experts) atomicExch(status, 6);
    }
  }
  __syncthreads();
  // (two sums in one: pairs above, tiles below)
  const int mine = tid < experts ? at[tid] : 0, tiles = (mine + tile_rows_at_most - 1) / tile_rows_at_most;
  long long total;
  const long long before = before_me((long long)mine << 32 | tiles, scratch, total);
  const int first = (int)(before >> 32), first_tile = (int)(before & 0x7FFFFFFF), all = (int)(total >> 32), all_tiles = (int)(total & 0x7FFFFFFF);
  if (tid < experts) {
    at[tid] = first;
    for (int t = 0; t < tiles; ++t) {
      tile_group[first_tile + t] = tid;
      tile_row0[first_tile + t] = first + t * tile_rows_at_most;
      tile_rows[first_tile + t] = min(tile_rows_at_most, mine - t * tile_rows_at_most);
    }
  }
  if (tid == 0) {
    at[experts] = all;
    *n_tiles = all_tiles;
  }
  __syncthreads();
  for (int p0 = tid; p0 < pairs; p0 += HELD * PLAN_THREADS) {
    if (pairs > HELD * PLAN_THREADS) load(p0);
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
      if (held[j] < 0) continue;
      const int p = p0 + j * PLAN_THREADS, to = atomicAdd(&at[held[j]], 1);
      sorted[to] = p;
      place[p] = to;
    }
  }
}

// to[i] = from[order[i] / div] (without an order from[i]), eight numbers a thread; those past `width` stay as they are.
template <bool WHOLE>
__global__ void __launch_bounds__(256) gather_kernel(const bf16* from, long long ld, const int* order, int div, bf16* to, int ld_to, int width,
                                                     long long total) {
  chain_next();
  chain_wait();
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  const long long row = i / (ld_to / 8);
  const int at = (int)(i - row * (ld_to / 8)) * 8;
  const bf16* src = from + (order ? order[row] / div : row) * ld + at;
  bf16* dst = to + row * ld_to + at;
  if (WHOLE) {
    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
  } else {
    for (int j = 0; j < 8 && at + j < width; ++j) dst[j] = src[j];
  }
}

// out[r] = sum over r's slots, one after the other, of wts * y[place]; without weights the rows as they are. Four outputs a thread.
template <bool WHOLE, typename TOut>
__global__ void __launch_bounds__(256) sum_kernel(const float* y, long long ldy, const int* place, const int* ids, const float* wts, TOut* out, int N,
                                                  int top, int experts) {
  __shared__ int s_place[SUM_TOP];
  __shared__ float s_weight[SUM_TOP];
  chain_next();
  chain_wait();
  const long long r = blockIdx.x;
  if (threadIdx.x < top) {
    const long long p = r * top + threadIdx.x;
    s_place[threadIdx.x] = (unsigned)ids[p] < (unsigned)experts ? place[p] : -1;
    s_weight[threadIdx.x] = wts ? wts[p] : 1.f;
  }
  __syncthreads();
  const int n = (blockIdx.y * 256 + threadIdx.x) * 4;
  if (n >= N) return;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < top; ++j) {
    if (s_place[j] < 0) continue;
    const float* from = y + s_place[j] * ldy + n;
    const float w = s_weight[j];
    if (WHOLE) {
      const float4 f = *reinterpret_cast<const float4*>(from);
      v[0] = fmaf(w, f.x, v[0]), v[1] = fmaf(w, f.y, v[1]), v[2] = fmaf(w, f.z, v[2]), v[3] = fmaf(w, f.w, v[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < N) v[i] = fmaf(w, from[i], v[i]);
    }
  }
  TOut* to = out + r * N + n;
  if (WHOLE) {
    store4(to, v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < N) to[i] = from_f32<TOut>(v[i]);
  }
}

}  // namespace mx
}  // namespace tl

using namespace tl;

extern "C" int tl_mxfp4_plan(const int* ids, int pairs, int experts, int tile_rows_at_most, int* sorted, int* place, int* tile_group, int* tile_row0,
                             int* tile_rows, int* n_tiles, int* status, cudaStream_t stream) {
  if (pairs == 0) return 0;
  TL_REQUIRE(pairs > 0 && pairs <= 1 << 30 && experts >= 1 && experts <= mx::PLAN_EXPERTS && tile_rows_at_most >= 1,
             "mxfp4 experts: %d pairs of %d experts", pairs, experts);
  return mx::launch_behind(false, mx::plan_kernel, dim3(1), mx::PLAN_THREADS, 0, stream, ids, pairs, experts, tile_rows_at_most, sorted, place,
                             tile_group, tile_row0, tile_rows, n_tiles, status);
}

// to [rows, width] bfloat16 (row stride ld_to, a multiple of 8, 16-byte aligned) from x (row stride ldx): row i is x[order[i] / div], or x[i].
extern "C" int tl_mxfp4_gather(const void* x, long long ldx, const int* order, int div, void* to, long long ld_to, int rows, int width,
                               cudaStream_t stream) {
  if (rows == 0 || width == 0) return 0;
  TL_REQUIRE(rows > 0 && div >= 1 && width > 0 && ld_to % 8 == 0 && ld_to >= width && ld_to <= 0x7FFFFFF8 && ((uintptr_t)to % 16) == 0,
             "mxfp4 product: rows of %d numbers to rows %lld apart", width, ld_to);
  const long long total = (long long)rows * (ld_to / 8), blocks = ceil_div64(total, 256);
  TL_REQUIRE(blocks <= 0x7FFFFFFF, "mxfp4 product: %d rows of %d numbers are too many", rows, width);
  const bool whole = width % 8 == 0 && width == ld_to && ldx % 8 == 0 && ((uintptr_t)x % 16) == 0;
#define TL_GATHER(W_)                                                                                                                       \
  return mx::launch_behind(order != nullptr, mx::gather_kernel<W_>, dim3((unsigned)blocks), 256, 0, stream, (const bf16*)x, ldx, order, div, \
                           (bf16*)to, (int)ld_to, width, total)
  if (whole) TL_GATHER(true);
  TL_GATHER(false);
#undef TL_GATHER
}

// y [pairs, N] 32-bit, out [rows, N] contiguous, bfloat16 or 32-bit.
extern "C" int tl_mxfp4_sum(const float* y, const int* place, const int* ids, const float* wts, void* out, int out_dtype, int rows, int N, int top,
                            int experts, cudaStream_t stream) {
  if (rows == 0 || N == 0) return 0;
  TL_REQUIRE(rows > 0 && N > 0 && top >= 1 && top <= mx::SUM_TOP, "mxfp4 experts: %d rows of %d, top-%d", rows, N, top);
  TL_REQUIRE(N <= 65535 * 1024, "mxfp4 experts: %d outputs exceed the grid limit", N);
  const bool whole = N % 4 == 0 && ((uintptr_t)y % 16) == 0 && ((uintptr_t)out % 16) == 0;
  const dim3 grid(rows, ceil_div(N, 1024));
#define TL_SUM(W_, T_) \
  return mx::launch_behind(true, mx::sum_kernel<W_, T_>, grid, 256, 0, stream, y, (long long)N, place, ids, wts, (T_*)out, N, top, experts)
  if (out_dtype == TL_FP32) {
    if (whole) TL_SUM(true, float);
    TL_SUM(false, float);
  }
  if (whole) TL_SUM(true, bf16);
  TL_SUM(false, bf16);
#undef TL_SUM
}
