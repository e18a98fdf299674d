// Products of a few bfloat16 rows with MXFP4 weights (mxfp4.cuh), for decode steps:
//
//   DENSE   C = X W^T (+ bias), or gated C = act(X G^T + b_g) * (X U^T + b_u)
//   FIRST   the experts' first half for up to 8 rows: a[p] = act(G_e x) * (U_e x) of every (row, slot) pair p, times the pair's weight
//   SECOND  their second half: out[r] = sum over r's pairs of D_e a[p], all experts in one sum
//
// a[p] is rounded to bfloat16 between the halves, as the bfloat16 path's rows are: in 32 bits a step's rows would not fit shared memory beside the
// weights' stages, and a layer's result, which is rounded to bfloat16 itself (1.7e-3 of it), is off by 2.3e-3 so.
//
// Such a product reads every weight once and does little with it: its bounds are the weights' stream and their conversion. Codes become float16
// numbers two at a time by a conversion of the GPU's, and a block's 32 products are two mma.sync m16n8k16 whose sum joins the others times the block's
// scale, in 32 bits. (As bfloat16 numbers made of bits and times their scale, a word of eight codes takes 32 cycles of a scheduler with its MMA;
// converted and times a float16 scale 19; so about 12.) The token rows become float16 numbers relative to their largest, which becomes 2^14 or a
// little more: that keeps all bits of a bfloat16 number down to 2^-31 of it, and nothing below 2^-39; the power of two comes back with the sum (which
// weights of 2^112 / K, 2^95 for the longest rows taken, can make infinite before).
//
// A persistent CTA an SM has four groups of four warps. A group's producer (one thread of a warp of its own) keeps a ring of stages full
// with bulk copies, which the layout's tiles make long: a stage is 16 weight rows by up to `slice` tiles of 128 k. The group's four warps take
// every fourth tile of a stage, and a sixth warp makes results of their sums while they are at the next ones. The token rows lie in shared
// memory for good.
//
// The unit of work is 16 weight rows (gated: 8 gate rows and the 8 up rows of the same outputs) of one matrix. It belongs to a team of one, two or
// four groups, the larger the fewer units there are. The warps' 32-bit sums are added in the order of the warps, so results do not depend on
// timing.
//
// Every wait on an mbarrier is bounded: when a bound is hit the CTA records status 11, its warps stop, wait (bounded again) for the copies
// in flight, and return.
#include <cuda_fp16.h>

#include "mxfp4.cuh"
#include "tma.cuh"

namespace tl {
namespace mx {

constexpr int GROUPS = 4;
constexpr int GROUP_WARPS = 4;
constexpr int WARPS = GROUPS * GROUP_WARPS;           // that multiply; a group has one more that copies and one that finishes
constexpr int THREADS = (WARPS + 2 * GROUPS) * 32;
constexpr int MAX_PAIRS = 256;                        // of the experts' form
constexpr int MAX_ROWS = 8;                           // token rows: the N side of the MMA

// Token rows in shared memory: a row's length is 64 modulo 128 bytes, so that the 16 bytes of eight lanes (two rows, four quarters of a
// block) fall on all banks. Eight numbers lie as the codes' conversion leaves theirs: 0 2, 4 6, 1 3, 5 7. (64 bits: it is asked of any length.)
__host__ __device__ __forceinline__ long long row_bytes(int k_tiles) { return k_tiles * (TILE_K * 2ll) + 64; }

__device__ __forceinline__ void mma_16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same from zero.
__device__ __forceinline__ void mma_16816_first(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ void copy_bulk(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

// 2^e for e in -126 .. 127
__device__ __forceinline__ float power(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// The exponent of a row whose largest number has the bits `top` (without the sign): its numbers times `to_half` are float16 numbers, and sums of
// these times twice the blocks' scales (scale32) are what they are times `from_half`.
__device__ __forceinline__ int row_exponent(uint32_t top) { return max((int)(top >> 23) - 127, -111); }
__device__ __forceinline__ float to_half(uint32_t top) { return power(14 - row_exponent(top)); }
__device__ __forceinline__ float from_half(uint32_t top) { return power(row_exponent(top) - 15); }

// acc += 16 weight rows by 128 k times eight token rows. `lo` and `hi`: a lane's words of the four blocks in row g and in row g + 8; `s_lo` and `s_hi`
// these rows' scales.
__device__ __forceinline__ void multiply(float (&acc)[4], const uint4& lo4, const uint4& hi4, uint32_t s_lo, uint32_t s_hi, const uint8_t* row) {
  const uint32_t lo[4] = {lo4.x, lo4.y, lo4.z, lo4.w}, hi[4] = {hi4.x, hi4.y, hi4.z, hi4.w};
  uint4 x[4];
#pragma unroll
  for (int b = 0; b < 4; ++b) x[b] = *reinterpret_cast<const uint4*>(row + 64 * b);
  // two blocks side by side: an MMA's sum is there 30 cycles later
#pragma unroll
  for (int b0 = 0; b0 < 4; b0 += 2) {
    uint32_t u[2][4], v[2][4];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      values16(lo[b0 + b], u[b]);
      values16(hi[b0 + b], v[b]);
    }
    float c[2][4];
#pragma unroll
    for (int b = 0; b < 2; ++b) mma_16816_first(c[b], u[b][0], v[b][0], u[b][1], v[b][1], x[b0 + b].x, x[b0 + b].y);
#pragma unroll
    for (int b = 0; b < 2; ++b) mma_16816(c[b], u[b][2], v[b][2], u[b][3], v[b][3], x[b0 + b].z, x[b0 + b].w);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const float f_lo = scale32(s_lo, b0 + b), f_hi = scale32(s_hi, b0 + b);
      acc[0] = fmaf(c[b][0], f_lo, acc[0]);
      acc[1] = fmaf(c[b][1], f_lo, acc[1]);
      acc[2] = fmaf(c[b][2], f_hi, acc[2]);
      acc[3] = fmaf(c[b][3], f_hi, acc[3]);
    }
  }
}

// ------------------------------------------------------------------------------------------ experts
// The experts of a small step, found by every CTA from the ids: item i is an expert and, for every row that chose it, the pair (row, slot)
// that did. A row that names an expert twice has its second time in an item of its own. Items come in the order in which they first appear.
struct Items {
  int count;
  short expert[MAX_PAIRS];
  short pair[MAX_PAIRS][MAX_ROWS];        // -1: the row did not choose it
  alignas(16) int key[MAX_PAIRS];
  short leader[MAX_PAIRS];                // the id, until the leaders are known
  uint32_t firsts[MAX_PAIRS / 32];
  float weight[MAX_PAIRS];
};

// From L2: what the SM has held of this memory since an earlier kernel does not count.
__device__ __forceinline__ int load_id(const int* p) {
  int v;
  asm volatile("ld.relaxed.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// All of the CTA's threads; ends with a barrier. `mine`: with up to 32 pairs, the id of pair `lane` in the first copying warp. An id that names no
// expert is recorded in `status` and its pair counts for nothing.
__device__ __forceinline__ void find_items(Items& s, const int* ids, int mine, int pairs, int top, int experts, int* status) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (pairs <= 32) {
    if (warp == WARPS) {                    // (the others may be at the token rows meanwhile)
      const int id = mine, row = lane / top;
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
  for (int p = threadIdx.x; p < pairs; p += THREADS) {
    const int id = load_id(ids + p);
    s.leader[p] = (short)(id >= 0 && id < experts ? id : -1);
#pragma unroll
    for (int r = 0; r < MAX_ROWS; ++r) s.pair[p][r] = -1;
  }
  __syncthreads();
  for (int p = threadIdx.x; p < MAX_PAIRS; p += THREADS) {
    int key = -1;
    if (p < pairs) {
      const int id = s.leader[p];
      if (id >= 0) {
        int again = 0;
        for (int q = p - p % top; q < p; ++q) again += s.leader[q] == id;
        key = id * 32 + again;
      } else {
        atomicExch(status, 6);
      }
    }
    s.key[p] = key;
  }
  __syncthreads();
  for (int p = threadIdx.x; p < MAX_PAIRS; p += THREADS) {
    const int key = s.key[p];
    int leader = 0;
    for (bool found = key < 0; !found; leader += found ? 0 : 4) {       // (four at a time, at the latest its own)
      const int4 four = *reinterpret_cast<const int4*>(s.key + leader);
      found = four.x == key || four.y == key || four.z == key || four.w == key;
      if (found) leader += four.x == key ? 0 : four.y == key ? 1 : four.z == key ? 2 : 3;
    }
    s.leader[p] = (short)leader;
    const uint32_t firsts = __ballot_sync(0xffffffffu, key >= 0 && leader == p);
    if (lane == 0) s.firsts[p >> 5] = firsts;
  }
  __syncthreads();
  for (int p = threadIdx.x; p < pairs; p += THREADS) {
    const int key = s.key[p], leader = s.leader[p];
    if (key < 0) continue;
    int at = __popc(s.firsts[leader >> 5] & ((1u << (leader & 31)) - 1u));
    for (int i = 0; i < leader >> 5; ++i) at += __popc(s.firsts[i]);
    s.pair[at][p / top] = (short)p;
    if (leader == p) s.expert[at] = (short)(key >> 5);
  }
  if (threadIdx.x == 0) {
    int n = 0;
    for (int i = 0; i < MAX_PAIRS / 32; ++i) n += __popc(s.firsts[i]);
    s.count = n;
  }
  __syncthreads();
}

struct FewParams {
  const void* x;              // DENSE, FIRST: token rows; SECOND: a row a pair
  long long ldx;
  const uint8_t* codes;
  const uint8_t* scales;
  const float* bias;          // DENSE (or null)
  void* out;                  // FIRST: what SECOND reads, K rounded up to 128
  long long ldc;
  float* largest;             // FIRST, SECOND: [pairs][parts], the largest numbers of each part of a row between the two
  int parts;
  int M, N, K;                // SECOND: M the pairs
  int act;                    // the gate's activation; a plain product: negated an activation on its results, or 0
  float ga0, ga1;
  const int* ids;             // FIRST, SECOND
  const float* wts;           // FIRST
  int before;                 // FIRST: the weight multiplies the sums, in front of the activation, else what comes of them
  int rows, top, experts;     // FIRST, SECOND
  int team, slice, stages;    // groups a unit, tiles a stage, stages a ring
  int* status;
  int skip;                   // -1; a test sets the group's stage whose copies are left out, so that a wait runs out
};

inline int& skip_stage_for_test() {
  static int stage = -1;
  return stage;
}

enum Kind { DENSE, FIRST, SECOND };

template <Kind KIND> struct Place { typedef Items Type; };
template <> struct Place<DENSE> { typedef int Type; };              // (never looked into)

__host__ __device__ __forceinline__ int stage_bytes(int slice) { return 2 * slice * (TILE_CODES + TILE_SCALES); }
// Dynamic shared memory: token rows (SECOND: and one of zeros), rings, two sets of the warps' sums, barriers (full and empty ones of the rings,
// of the sums two each a group, and one of SECOND's rows), the rows' largest numbers.
__host__ __device__ __forceinline__ long long rows_bytes(Kind kind, int m, int k_tiles) { return (m + (kind == SECOND ? 1 : 0)) * row_bytes(k_tiles); }
inline long long few_bytes(Kind kind, int m, int k_tiles, int slice, int stages) {
  return rows_bytes(kind, m, k_tiles) + GROUPS * stages * stage_bytes(slice) + 2 * WARPS * 16 * (MAX_ROWS + 1) * 4 + (GROUPS * (2 * stages + 4) + 1) * 8 +
         m * 4;
}

// Eight numbers of a token row from element k on, zeros past K and where there is no row. ALIGNED: rows begin at multiples of 16 bytes and K is a
// multiple of 8, so the eight are in or out; the load then stands alone (a branch around it would wait for it), else one by one.
template <bool ALIGNED>
__device__ __forceinline__ uint4 load_piece(const bf16* row, int k, int K, bool there) {
  uint4 v;
  if constexpr (ALIGNED) {
    asm volatile(
        "{\n\t.reg .pred ok;\n\t"
        "setp.ne.b32 ok, %5, 0;\n\t"
        "mov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
        "@ok ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
        : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(row + k), "r"((int)(there && k < K)) : "memory");
  } else {
    uint32_t u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t lo = there && k + 2 * j < K ? __bfloat16_as_ushort(row[k + 2 * j]) : 0u;
      const uint32_t hi = there && k + 2 * j + 1 < K ? __bfloat16_as_ushort(row[k + 2 * j + 1]) : 0u;
      u[j] = lo | hi << 16;
    }
    v = make_uint4(u[0], u[1], u[2], u[3]);
  }
  return v;
}

template <bool GATED, Kind KIND, bool ALIGNED, typename TOut>
__global__ void __launch_bounds__(THREADS, 1) few_kernel(const FewParams p) {
  constexpr int OUTS = GATED ? 8 : 16, COLS = MAX_ROWS;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ typename Place<KIND>::Type place;
  __shared__ int aborted_;
  volatile int* aborted = &aborted_;
  // SECOND starts behind FIRST's end on its SM, not behind all of it (programmatic dependent launch): it sets itself up, finds its items and has its
  // first weights on their way before it waits for the rows that FIRST makes. The ids that it reads in front of its wait are another kernel's results.
  // They are final by then, because FIRST opens the door only behind its own wait, and they are read where all SMs see the same (load_id).
  if (KIND != SECOND) chain_wait();
  chain_next();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = warp < WARPS ? warp / GROUP_WARPS : (warp - WARPS) % GROUPS;
  int my_id = -1;
  if (KIND != DENSE && warp == WARPS && lane < p.rows * p.top) my_id = load_id(p.ids + lane);
  const int k_tiles = ceil_div(p.K, TILE_K), row_tiles = ceil_div(p.N, TILE_ROWS);
  const int x_bytes = (int)row_bytes(k_tiles), one_stage = stage_bytes(p.slice);
  // The token rows: a warp takes 256 numbers of a row at a time, ROUND such pieces on their way. Their largest numbers come first; what fits one
  // round stays in registers until these are known, the rest is read again.
  constexpr int ROUND = 4;
  const int a_row = ceil_div(k_tiles, 2), all_pieces = p.M * a_row;
  uint4 raw[ROUND];
  int m_of[ROUND], k_of[ROUND];
  int next_m = 0, next_c = warp;
  auto load_round = [&]() {
#pragma unroll
    for (int j = 0; j < ROUND; ++j) {
      while (next_c >= a_row) next_c -= a_row, ++next_m;
      m_of[j] = next_m, k_of[j] = next_c * 256 + lane * 8;
      raw[j] = load_piece<ALIGNED>(static_cast<const bf16*>(p.x) + next_m * p.ldx, k_of[j], p.K, next_m < p.M);
      next_c += WARPS;
    }
  };
  if (KIND != SECOND && warp < WARPS) load_round();
  uint8_t* xs = smem;
  uint8_t* rings = smem + (int)rows_bytes(KIND, p.M, k_tiles);
  uint8_t* ring = rings + group * p.stages * one_stage;
  float (*part)[WARPS][16][COLS + 1] = reinterpret_cast<float (*)[WARPS][16][COLS + 1]>(rings + GROUPS * p.stages * one_stage);
  uint64_t* full = reinterpret_cast<uint64_t*>(part + 2);       // [stages][GROUPS], and so on
  uint64_t* empty = full + p.stages * GROUPS;
  uint64_t* summed = empty + p.stages * GROUPS;                 // [2][GROUPS]: a team's sums are there
  uint64_t* taken = summed + 2 * GROUPS;                        // and read
  uint64_t* rows_there = taken + 2 * GROUPS;                    // SECOND
  uint32_t* tops = reinterpret_cast<uint32_t*>(rows_there + 1);           // the bits of a token row's largest number
  if (threadIdx.x < (2 * p.stages + 4) * GROUPS) {
    const int i = threadIdx.x / GROUPS - p.stages;
    mbar_init(&full[threadIdx.x], i < 0 ? 1 : i < p.stages ? GROUP_WARPS : i < p.stages + 2 ? p.team * GROUP_WARPS : p.team);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (KIND == SECOND && threadIdx.x == THREADS - 1) {
    mbar_init(rows_there, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x == 0) aborted_ = 0;
  for (int m = threadIdx.x; m < p.M; m += THREADS) tops[m] = 0u;
  __syncthreads();
  if constexpr (KIND == FIRST)
    for (int i = threadIdx.x - (WARPS + GROUPS) * 32; i >= 0 && i < p.rows * p.top; i += GROUPS * 32)
      reinterpret_cast<Items*>(&place)->weight[i] = p.wts[i];
  if (KIND != SECOND && warp < WARPS) {
    for (int done = 0; done < all_pieces; done += ROUND * WARPS) {
      if (done) load_round();
#pragma unroll
      for (int j = 0; j < ROUND; ++j) {
        if (m_of[j] >= p.M) break;
        const uint32_t a = __vmaxu2(raw[j].x & 0x7FFF7FFFu, raw[j].y & 0x7FFF7FFFu), b = __vmaxu2(raw[j].z & 0x7FFF7FFFu, raw[j].w & 0x7FFF7FFFu);
        const uint32_t c = __vmaxu2(a, b), top = __reduce_max_sync(0xffffffffu, max(c << 16, c & 0xFFFF0000u));
        if (lane == 0) atomicMax(&tops[m_of[j]], top);
      }
    }
  }
  Items* items = reinterpret_cast<Items*>(&place);
  int count = 1;
  if constexpr (KIND != DENSE) {
    find_items(*items, p.ids, my_id, p.rows * p.top, p.top, p.experts, p.status);
    count = items->count;
  }
  // What all roles go through, in the same order: this team's units, and of a unit the slices that are this group's.
  const int blocks = ceil_div(p.N, OUTS), units = KIND == FIRST ? blocks * count : blocks;
  const int teams = gridDim.x * (GROUPS / p.team), member = group % p.team, team0 = group - member;
  const int parts = ceil_div(k_tiles, p.slice), slices = KIND == SECOND ? parts * count : parts;
  const int first_unit = blockIdx.x * (GROUPS / p.team) + group / p.team;
  auto give_up = [&]() {
    *aborted = 1;
    atomicExch(p.status, 11);
  };

  if (warp >= WARPS && warp < WARPS + GROUPS) {
    // ---- copies ----
    if (lane == 0) {
      int it = 0;
      for (int unit = first_unit; unit < units && !*aborted; unit += teams) {
        const int item0 = KIND == FIRST ? unit / blocks : 0, block = unit - item0 * blocks;
        const int row_lo = GATED ? block : 2 * block, row_hi = GATED ? block : min(row_lo + 1, row_tiles - 1);
        for (int sl = member; sl < slices; sl += p.team, ++it) {
          const int item = KIND == SECOND ? sl / parts : item0, tile0 = (sl - (KIND == SECOND ? item * parts : 0)) * p.slice;
          const int n = min(p.slice, k_tiles - tile0), s = it % p.stages;
          uint64_t* bar = &full[s * GROUPS + group];
          if (it >= p.stages && !mbar_wait(&empty[s * GROUPS + group], ((it / p.stages) - 1) & 1)) give_up();
          if (*aborted) break;
          uint8_t* to = ring + s * one_stage;
          uint8_t* to_scales = to + p.slice * 2 * TILE_CODES;
          const long long matrix = KIND == DENSE ? 0 : (long long)items->expert[item] * (GATED ? 2 : 1);
          const long long lo = (matrix * row_tiles + row_lo) * k_tiles + tile0;
          const long long hi = ((matrix + (GATED ? 1 : 0)) * row_tiles + row_hi) * k_tiles + tile0;
          if (it == p.skip) continue;
          mbar_expect_tx(bar, 2 * n * (TILE_CODES + TILE_SCALES));
          copy_bulk(to, p.codes + lo * TILE_CODES, n * TILE_CODES, bar);
          copy_bulk(to + p.slice * TILE_CODES, p.codes + hi * TILE_CODES, n * TILE_CODES, bar);
          copy_bulk(to_scales, p.scales + lo * TILE_SCALES, n * TILE_SCALES, bar);
          copy_bulk(to_scales + p.slice * TILE_SCALES, p.scales + hi * TILE_SCALES, n * TILE_SCALES, bar);
        }
      }
      // no CTA leaves with copies under way, whether it gave up or not
      for (int i = max(0, it - p.stages); i < it; ++i)
        if (i != p.skip) mbar_wait(&full[(i % p.stages) * GROUPS + group], (i / p.stages) & 1);
      if (KIND == SECOND) mbar_wait(rows_there, 0);
    }
    return;
  }

  if (warp >= WARPS + GROUPS) {
    // ---- results ----
    if (KIND == SECOND) chain_wait();
    int nth = 0;
    for (int unit = first_unit; unit < units; unit += teams, ++nth) {
      const int item = KIND == FIRST ? unit / blocks : 0, block = unit - item * blocks, buffer = nth & 1;
      const bool ok = __all_sync(0xffffffffu, !*aborted && mbar_wait(&summed[buffer * GROUPS + team0], (nth >> 1) & 1));
      if (!ok) {
        if (lane == 0) give_up();
        break;
      }
#pragma unroll 2
      for (int i = member * 32 + lane; i < OUTS * COLS; i += p.team * 32) {
        const int o = i & (OUTS - 1), m = i / OUTS, n = block * OUTS + o;
        int row = m;
        bool mine = m < (KIND == SECOND ? p.rows : p.M) && n < p.N;
        float weight = 1.f;
        if (KIND == FIRST) {
          row = items->pair[item][m];
          mine = row >= 0;
          if (mine) weight = items->weight[row];
        }
        float v = 0.f, u = 0.f;
        for (int s = team0 * GROUP_WARPS; s < (team0 + p.team) * GROUP_WARPS; ++s) {
          v += part[buffer][s][o][m];
          if (GATED) u += part[buffer][s][o + 8][m];
        }
        if (KIND != SECOND && mine) {
          const float f = from_half(tops[m]);
          v *= f;
          if (GATED) u *= f;
        }
        if (KIND == FIRST && n >= p.N) v = u = 0.f;             // (what lies behind the last output meets codes of zeros)
        if (KIND == FIRST && p.before) v *= weight, u *= weight;
        if (KIND == DENSE && p.bias && mine) {
          v += p.bias[n];
          if (GATED) u += p.bias[p.N + n];
        }
        float out = GATED ? gated(v, u, p.act, p.ga0, p.ga1) : p.act < 0 ? gate_activation(v, -p.act) : v;
        if (KIND == FIRST && !p.before) out *= weight;
        const TOut rounded = from_f32<TOut>(out);
        if (mine) static_cast<TOut*>(p.out)[row * p.ldc + n] = rounded;
        if (KIND == FIRST) {                                      // (bits: a NaN's are above all others)
          uint32_t top = mine ? __float_as_uint(to_f32(rounded)) & 0x7FFFFFFFu : 0u;
#pragma unroll
          for (int d = 1; d < OUTS; d *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
          if (mine && o == 0) p.largest[(long long)row * p.parts + block] = __uint_as_float(top);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&taken[buffer * GROUPS + team0]);
    }
    return;
  }

  // ---- token rows into shared memory ----
  if (KIND == SECOND) {
    // whole rows by bulk copies, which no register waits for, made float16 numbers where they lie
    const uint32_t bytes = k_tiles * TILE_K * 2;
    chain_wait();
    if (lane == 0) {
      asm volatile("fence.proxy.async;" ::: "memory");          // (the rows were written by ordinary stores)
      for (int m = warp; m < p.M; m += WARPS) copy_bulk(xs + m * x_bytes, static_cast<const bf16*>(p.x) + m * p.ldx, bytes, rows_there);
      if (warp == 0) mbar_expect_tx(rows_there, p.M * bytes);
    }
    __syncwarp();
    for (int m = warp; m < p.M; m += WARPS) {
      uint32_t top = 0u;
      for (int i0 = lane; i0 < p.parts; i0 += 8 * 32) {
        uint32_t some[8];                                       // on their way together
#pragma unroll
        for (int j = 0; j < 8; ++j) some[j] = i0 + 32 * j < p.parts ? __float_as_uint(p.largest[(long long)m * p.parts + i0 + 32 * j]) : 0u;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, some[j]);
      }
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane == 0) tops[m] = top;
    }
  }
  asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory");
  auto put_piece = [&](int m, int k, const uint4& eight, float f) {
    float v[8];
    unpack8(eight, v);
    __half2 h[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int at = (e & 1) * 4 + (e >> 1);
      h[e] = __floats2half2_rn(v[at] * f, v[at + 2] * f);
    }
    *reinterpret_cast<uint4*>(xs + m * x_bytes + k * 2) = *reinterpret_cast<const uint4*>(h);
  };
  if constexpr (KIND == SECOND) {
    if (!__all_sync(0xffffffffu, mbar_wait(rows_there, 0)) && lane == 0) give_up();
    auto in_place = [&](int m, int k, float f) {
      if (k < k_tiles * TILE_K) put_piece(m, k, *reinterpret_cast<const uint4*>(xs + m * x_bytes + k * 2), f);
    };
    if (p.M >= WARPS) {                                         // a warp whole rows
      for (int m = warp; m < p.M; m += WARPS) {
        const float f = to_half(tops[m]);
#pragma unroll 4
        for (int k = lane * 8; k < k_tiles * TILE_K; k += 256) in_place(m, k, f);
      }
    } else {
      for (int piece = warp; piece < all_pieces; piece += WARPS) {
        const int m = piece / a_row;
        in_place(m, (piece - m * a_row) * 256 + lane * 8, to_half(tops[m]));
      }
    }
  } else {
    if (all_pieces > ROUND * WARPS) {
      next_m = 0, next_c = warp;
      load_round();
    }
    for (int done = 0; done < all_pieces; done += ROUND * WARPS) {
      if (done) load_round();
#pragma unroll
      for (int j = 0; j < ROUND; ++j)
        if (m_of[j] < p.M && k_of[j] < k_tiles * TILE_K) put_piece(m_of[j], k_of[j], raw[j], to_half(tops[m_of[j]]));
    }
  }
  if (KIND == SECOND)
    for (int i = threadIdx.x; i < x_bytes / 16; i += WARPS * 32) reinterpret_cast<uint4*>(xs + p.M * x_bytes)[i] = make_uint4(0u, 0u, 0u, 0u);
  asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory");

  // ---- products ----
  const int g = lane >> 2, t = lane & 3, w = warp % GROUP_WARPS;
  const unsigned lane_codes = lane * 16;
  int it = 0, nth = 0;
  for (int unit = first_unit; unit < units; unit += teams, ++nth) {
    float acc[4] = {};
    bool ok = true;
    for (int sl = member; sl < slices; sl += p.team, ++it) {
      const int item = KIND == SECOND ? sl / parts : 0, tile0 = (sl - (KIND == SECOND ? item * parts : 0)) * p.slice;
      const int n = min(p.slice, k_tiles - tile0), s = it % p.stages;
      const uint8_t* from = ring + s * one_stage;
      int m = min(g, p.M - 1);
      if (KIND == SECOND) {
        const int pair = items->pair[item][g];
        m = pair >= 0 ? pair : p.M;
      }
      const uint8_t* row = xs + m * x_bytes + tile0 * (TILE_K * 2) + t * 16;
      ok = __all_sync(0xffffffffu, !*aborted && mbar_wait(&full[s * GROUPS + group], (it / p.stages) & 1));
      if (!ok) break;
      float sum[4] = {};
      for (int c = (w + it) & (GROUP_WARPS - 1); c < n; c += GROUP_WARPS) {
        const uint8_t* codes = from + c * TILE_CODES + lane_codes;
        const uint8_t* scales = from + p.slice * 2 * TILE_CODES + c * TILE_SCALES + g * 4;
        multiply(KIND == SECOND ? sum : acc, *reinterpret_cast<const uint4*>(codes), *reinterpret_cast<const uint4*>(codes + p.slice * TILE_CODES),
                 *reinterpret_cast<const uint32_t*>(scales), *reinterpret_cast<const uint32_t*>(scales + p.slice * TILE_SCALES),
                 row + c * (TILE_K * 2));
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s * GROUPS + group]);
      if (KIND == SECOND) {       // every pair has an exponent of its own; the rows that did not choose the expert have nothing to add
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int pair = items->pair[item][2 * t + c];
          if (pair >= 0) {
            const float f = from_half(tops[pair]);
            acc[c] = fmaf(sum[c], f, acc[c]);
            acc[c + 2] = fmaf(sum[c + 2], f, acc[c + 2]);
          }
        }
      }
    }
    // ---- the unit's end ----
    const int buffer = nth & 1;
    if (ok && nth >= 2) ok = __all_sync(0xffffffffu, !*aborted && mbar_wait(&taken[buffer * GROUPS + team0], ((nth >> 1) - 1) & 1));
    if (!ok) {
      if (lane == 0) give_up();
      break;
    }
    float (&mine)[16][COLS + 1] = part[buffer][warp];
    mine[g][2 * t] = acc[0];
    mine[g][2 * t + 1] = acc[1];
    mine[g + 8][2 * t] = acc[2];
    mine[g + 8][2 * t + 1] = acc[3];
    __syncwarp();
    if (lane == 0) mbar_arrive(&summed[buffer * GROUPS + team0]);
  }
  if (KIND == FIRST) {        // and the rest of the last tile of 128, in every pair's row
    const int from = blocks * OUTS, rest = (int)p.ldc - from;
    for (int i = blockIdx.x * WARPS * 32 + threadIdx.x; i < p.rows * p.top * rest; i += gridDim.x * WARPS * 32)
      static_cast<TOut*>(p.out)[(i / rest) * p.ldc + from + i % rest] = from_f32<TOut>(0.f);
  }
}

}  // namespace mx
}  // namespace tl

using namespace tl;

namespace {

constexpr int FEW_SMEM = 226 * 1024;
constexpr int few_dynamic(mx::Kind kind) { return FEW_SMEM - (kind == mx::DENSE ? 0 : (int)sizeof(mx::Items)) - 64; }

// Tiles a stage and stages a ring that fit beside the token rows, or false. Stages of 16 tiles where a slice is as long, so that a wait and an
// arrival serve four tiles a warp, else of 8 or 4.
bool few_fits(mx::Kind kind, int m, int k_tiles, mx::FewParams& p) {
  const int share = kind == mx::SECOND ? k_tiles : ceil_div(k_tiles, p.team);
  for (int slice = 16; slice >= 4; slice /= 2) {
    if (slice > 4 && slice / 2 >= share) continue;
    for (int stages = 6; stages >= 2; --stages)
      if (mx::few_bytes(kind, m, k_tiles, slice, stages) <= few_dynamic(kind) && (stages <= 3 || stages * slice <= 32)) {
        p.slice = slice, p.stages = stages;
        return true;
      }
  }
  return false;
}

template <auto kernel>
int launch_few(mx::FewParams& p, mx::Kind kind, long long units, cudaStream_t stream) {
  p.skip = mx::skip_stage_for_test();
  static thread_local int set_on = -1;              // the device whose function has its shared memory
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (set_on != dev) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, few_dynamic(kind));
    if (e != cudaSuccess) return (int)e;
    set_on = dev;
  }
  const long long ctas = ceil_div64(units, mx::GROUPS / p.team);
  const int bytes = (int)mx::few_bytes(kind, p.M, ceil_div(p.K, mx::TILE_K), p.slice, p.stages);        // (few_fits has passed it)
  const dim3 grid((unsigned)(ctas < sm_count() ? ctas : sm_count()));
  return mx::launch_behind(kind == mx::SECOND, kernel, grid, mx::THREADS, bytes, stream, p);
}

// Groups a unit: one where the groups of the GPU have units enough each, else two or four.
int team_of(long long units) {
  const long long groups = (long long)mx::GROUPS * sm_count();
  return units >= groups ? 1 : 2 * units >= groups ? 2 : 4;
}

bool a_few(int rows, int top, int experts) {
  return rows >= 1 && rows <= mx::MAX_ROWS && top >= 1 && rows * top <= mx::MAX_PAIRS && top <= 32 && experts >= 1 && experts <= 1024;
}

}  // namespace

// Whether `M` rows of K elements go through the form below.
extern "C" int tl_mxfp4_few_fits(int M, int N, int K, int act) {
  if (M < 1 || M > mx::MAX_ROWS || N < 1 || K < 1) return 0;
  mx::FewParams p = {};
  p.team = team_of(ceil_div(N, act > 0 ? 8 : 16));
  return few_fits(mx::DENSE, M, ceil_div(K, mx::TILE_K), p);
}

// x [M, K] bfloat16 (row stride ldx), M <= 8; the matrix N x K (gated: two, gate and up); bias [N] (gated: [2 N]) 32-bit or null; out [M, N]
// (row stride ldc) bfloat16 or 32-bit. `act`: the gate's activation TL_ACT_*, 0 for a plain product, negated an activation on its results.
extern "C" int tl_mxfp4_few(const void* x, long long ldx, const void* codes, const void* scales, const float* bias, void* out, long long ldc,
                            int M, int N, int K, int act, float a0, float a1, int out_dtype, int* status, cudaStream_t stream) {
  if (M == 0 || N == 0) return 0;
  TL_REQUIRE(M >= 1 && M <= mx::MAX_ROWS && N >= 1 && K >= 1, "mxfp4 product of few rows: %d rows x (%d x %d)", M, N, K);
  TL_REQUIRE(act <= 0 ? act >= -TL_ACT_IDENTITY : tl_is_gate(act), "mxfp4 product: gate activation %d is none (nor an ungated one, negated)", act);
  TL_REQUIRE(act <= 0 || out_dtype == TL_BF16, "mxfp4 product: gated outputs of type %d", out_dtype);
  mx::FewParams p = {};
  p.x = x, p.ldx = ldx, p.codes = (const uint8_t*)codes, p.scales = (const uint8_t*)scales, p.bias = bias, p.out = out, p.ldc = ldc;
  p.M = M, p.N = N, p.K = K, p.act = act, p.ga0 = a0, p.ga1 = a1, p.status = status;
  const bool aligned = K % 8 == 0 && ldx % 8 == 0 && ((uintptr_t)x % 16) == 0;
  const int units = ceil_div(N, act > 0 ? 8 : 16);
  p.team = team_of(units);
  TL_REQUIRE(few_fits(mx::DENSE, M, ceil_div(K, mx::TILE_K), p), "mxfp4 product of few rows: %d rows of %d elements are too many", M, K);
#define TL_FEW(G_, T_)                                                                                       \
  do {                                                                                                       \
    if (aligned) return launch_few<mx::few_kernel<G_, mx::DENSE, true, T_>>(p, mx::DENSE, units, stream);    \
    return launch_few<mx::few_kernel<G_, mx::DENSE, false, T_>>(p, mx::DENSE, units, stream);                \
  } while (0)
  if (act > 0) TL_FEW(true, bf16);
  if (out_dtype == TL_FP32) TL_FEW(false, float);
  TL_FEW(false, bf16);
#undef TL_FEW
}

// Whether `rows` rows of K elements and what top experts of `inter` outputs each make of them go through the two kernels below; and the bytes
// of what lies between the two.
extern "C" int tl_mxfp4_experts_fit(int rows, int top, int K, int inter) {
  if (!a_few(rows, top, 1) || K < 1 || inter < 1) return 0;
  mx::FewParams p = {};
  p.team = 4;
  return few_fits(mx::FIRST, rows, ceil_div(K, mx::TILE_K), p) && few_fits(mx::SECOND, rows * top, ceil_div(inter, mx::TILE_K), p);
}
static int between_row(int inter) { return ceil_div(inter, mx::TILE_K) * mx::TILE_K; }
extern "C" long long tl_mxfp4_experts_between(int pairs, int inter) {
  return (long long)pairs * (between_row(inter) * 2 + ceil_div(inter, 8) * 4);
}

// Routed experts of up to 8 rows and 256 pairs, first half: x [rows, K]; matrices [experts] (or gated [2 experts], gate and up in turn) of N x K;
// `between` (16-byte aligned) receives a bfloat16 row of N numbers, rounded up to 128, for every pair, and behind them the rows' largest numbers.
extern "C" int tl_mxfp4_experts_first(const void* x, long long ldx, const void* codes, const void* scales, void* between, int rows, int N, int K,
                                      const int* ids, const float* wts, int before, int top, int experts, int act, float a0, float a1, int* status,
                                      cudaStream_t stream) {
  if (rows == 0 || N == 0) return 0;
  TL_REQUIRE(a_few(rows, top, experts), "mxfp4 experts: %d rows, top-%d of %d", rows, top, experts);
  TL_REQUIRE(N >= 1 && K >= 1 && ((uintptr_t)between % 16) == 0, "mxfp4 experts: %d x %d", N, K);
  TL_REQUIRE(act < 0 ? act >= -TL_ACT_IDENTITY : tl_is_gate(act), "mxfp4 experts: gate activation %d is none (nor an ungated one, negated)", act);
  mx::FewParams p = {};
  p.x = x, p.ldx = ldx, p.codes = (const uint8_t*)codes, p.scales = (const uint8_t*)scales, p.out = between;
  p.ldc = between_row(N), p.M = rows, p.N = N, p.K = K, p.act = act, p.ga0 = a0, p.ga1 = a1;
  p.parts = ceil_div(N, act > 0 ? 8 : 16), p.largest = (float*)((uint8_t*)between + rows * top * p.ldc * 2);
  p.ids = ids, p.wts = wts, p.before = before, p.rows = rows, p.top = top, p.experts = experts, p.status = status;
  const bool aligned = K % 8 == 0 && ldx % 8 == 0 && ((uintptr_t)x % 16) == 0;
  const long long units = (long long)p.parts * (top < experts ? top : experts);       // (at least so many)
  p.team = team_of(units);
  TL_REQUIRE(few_fits(mx::FIRST, rows, ceil_div(K, mx::TILE_K), p), "mxfp4 experts: %d rows of %d elements are too many", rows, K);
#define TL_FIRST(G_)                                                                                                     \
  do {                                                                                                                   \
    if (aligned) return launch_few<mx::few_kernel<G_, mx::FIRST, true, bf16>>(p, mx::FIRST, units * rows, stream); \
    return launch_few<mx::few_kernel<G_, mx::FIRST, false, bf16>>(p, mx::FIRST, units * rows, stream);             \
  } while (0)
  if (act > 0) TL_FIRST(true);
  TL_FIRST(false);
#undef TL_FIRST
}

// Second half: `between` as the first half (of the same `act`) left it for pairs of K numbers; matrices [experts] of N x K; out [rows, N] (row
// stride ldc).
extern "C" int tl_mxfp4_experts_second(void* between, const void* codes, const void* scales, void* out, long long ldc, int rows, int N, int K,
                                       const int* ids, int top, int experts, int act, int out_dtype, int* status, cudaStream_t stream) {
  if (rows == 0 || N == 0) return 0;
  TL_REQUIRE(a_few(rows, top, experts), "mxfp4 experts: %d rows, top-%d of %d", rows, top, experts);
  TL_REQUIRE(N >= 1 && K >= 1 && ((uintptr_t)between % 16) == 0, "mxfp4 experts: %d x %d", N, K);
  mx::FewParams p = {};
  p.x = between, p.ldx = between_row(K), p.codes = (const uint8_t*)codes, p.scales = (const uint8_t*)scales, p.out = out, p.ldc = ldc;
  p.M = rows * top, p.N = N, p.K = (int)p.ldx;
  p.parts = ceil_div(K, act > 0 ? 8 : 16), p.largest = (float*)((uint8_t*)between + rows * top * p.ldx * 2);
  p.ids = ids, p.rows = rows, p.top = top, p.experts = experts, p.status = status;
  const int units = ceil_div(N, 16);
  p.team = team_of(units);
  TL_REQUIRE(few_fits(mx::SECOND, p.M, ceil_div(K, mx::TILE_K), p), "mxfp4 experts: %d pairs of %d elements are too many", p.M, K);
  if (out_dtype == TL_FP32) return launch_few<mx::few_kernel<false, mx::SECOND, true, float>>(p, mx::SECOND, units, stream);
  return launch_few<mx::few_kernel<false, mx::SECOND, true, bf16>>(p, mx::SECOND, units, stream);
}

// For tests of the bounded waits: the polls after which a wait of this file's kernels gives up (0 puts the default back), and the stage of
// weights, counted over a group's work, that is not copied (-1: none).
extern "C" int tl_mxfp4_few_set_wait_limit(unsigned int polls) {
  const uint32_t v = polls ? polls : (1u << 22);
  return (int)cudaMemcpyToSymbol(wait_limit, &v, sizeof(v));
}
extern "C" void tl_mxfp4_few_test_skip_stage(int stage) { mx::skip_stage_for_test() = stage; }
