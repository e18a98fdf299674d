// Products of bfloat16 rows with MXFP4 weights (mxfp4.cuh) on the 5th-generation tensor cores, for more rows than mxfp4_few.cu takes:
//
//   C[m, n] = sum_k X[m, k] * W[n, k] (+ bias[n])      or, gated:  C[m, n] = act(X . G[n] + b_g[n]) * (X . U[n] + b_u[n])
//
// A CTA computes 128 weight rows (gated: 64 outputs, 8 gate rows and the 8 up rows of the same outputs in turn) by BN token rows. The
// weights are the MMA's M side and come from tensor memory: lane r of it is weight row r, so the thread that owns a lane loads that
// row's 64 values of a k-block (32 bytes of codes and two scales), makes them bfloat16 numbers in its registers and stores them to its
// lane with one tcgen05.st. The 4-bit weights thus cross from L2 once, as they are, and no shared memory is spent on them. The token rows are the N
// side: boxes of 64 k-elements that TMA brings into a ring of stages (128-byte swizzle, no multicast).
//
//   warp 0       one thread keeps the ring of token boxes full
//   warp 1       one thread issues the MMAs (kind::f16, A in tensor memory, B in shared memory) and releases both operands' stages
//   warps 2..9   two groups of four that take every other tile of 128 k of the weights; then the epilogue, each group every other 16 columns
//
// The products of a tile of 128 k with 128 token rows take 512 cycles of the tensor pipe and its weights' conversion 290 of each scheduler's integer
// pipe (nine operations a word, at half rate), so with as many rows the conversion runs under the products; two CTAs an SM run under each other's ends.
//
// SPLIT: a cluster of CTAs shares a tile, each with a run of k; each leaves its accumulator in its shared memory, the cluster meets, and
// every CTA adds the sums of some of the tokens in rank order and stores them, so the result does not depend on timing.
//
// Every wait on an mbarrier is bounded: when a bound is hit the CTA records status 11, stops issuing work, waits (bounded again) for the
// copies and products in flight, meets its cluster, frees its tensor memory and returns. The copies' barriers also count the warps that convert
// weights; for one that leaves early its arrivals are made up at the CTA's end.
#include "mxfp4.cuh"
#include "tma.cuh"

namespace tl {
namespace mx {

constexpr int ROWS = 128;                   // weight rows a CTA: the MMA's M side
constexpr int KB = TMA_BOX_COLS;            // k-elements a block
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 64 + 32 * EPI_WARPS;
constexpr int MAX_SPLITS = 8;

struct TcParams {
  const uint8_t* codes;
  const uint8_t* scales;
  const float* bias;
  void* C;
  long long ldc;
  int M, N, K;                // tokens, outputs, reduction length
  int matrices;               // matrices a group: 1, or 2 where gate and up matrix come in turn
  int tiles_a_split;          // tiles of 128 k a CTA of a cluster takes
  const int* tile_group;      // grouped, persistent (or null): per token tile its group, first row and rows, `*n_tiles` of them
  const int* tile_row0;
  const int* tile_rows;
  const int* n_tiles;
  int act;                    // the gate's activation (TL_ACT_*), 0 for a plain product; negated: an activation on a plain product's results
  float ga0, ga1;
  const float* row_weight;    // grouped (or null): a (row, slot) pair's own weight on its sums, row_weight[weight_index[position]]
  const int* weight_index;
  int* status;
  int copies, products;       // a test's: the tiles of 128 k, counted over a CTA's work, behind which no token rows are copied any more, and
};                            // those behind which the products give up as if their wait had run out

struct StopForTest {
  int copies = 0x7fffffff, products = 0x7fffffff;
};
inline StopForTest& stop_for_test() {
  static StopForTest stop;
  return stop;
}

__device__ __forceinline__ float weight_of(const TcParams& p, long long position) {
  return p.row_weight[p.weight_index ? (long long)p.weight_index[position] : position];
}

template <int BN>
struct Tc {
  static constexpr int HALF_BYTES = BN * KB * 2;
  static constexpr int B_BYTES = 2 * HALF_BYTES;                // a stage of token rows: a tile of 128 k, its two k-blocks one after the other
  static constexpr int B_STAGES = BN >= 128 ? 3 : 4;
  static constexpr int A_COLS = TILE_K / 2;                     // columns of tensor memory a stage of weights takes: a tile of 128 k
  static constexpr int A_STAGES = 2;
  static constexpr int TMEM_COLS = 256;
  static constexpr int TOTAL = B_STAGES * B_BYTES + 1024 /* alignment slack */ + 256 /* barriers */;
  // What a launch with clusters asks for at least. A CTA of a cluster that waits for tensor memory keeps the others waiting, who keep
  // theirs; beside another kernel of clusters that could close a circle. With this much shared memory no SM has room for more CTAs of such kernels
  // (tc_gemm_pair.cu: 90 KB and more with half of tensor memory, 192 KB and more with all of it) than its tensor memory has.
  static constexpr int SPLIT_TOTAL = TOTAL > 72 * 1024 ? TOTAL : 72 * 1024;
  static_assert(BN + A_STAGES * A_COLS <= TMEM_COLS, "accumulator and weights share half of tensor memory");
  static_assert(B_STAGES * B_BYTES >= BN * ROWS * 4, "an accumulator fits the ring of token boxes");
};

// The CTA's nth tile of 128 k has two barriers, full[nth % SLOTS] and done[nth % SLOTS]. Its weights (an arrival of each of the four warps that bring
// them) and its token rows (the copying warp's arrival and their bytes) complete a phase of the one, its products a phase of the other: then its stages
// of weights and of token rows are free. Whoever fills a stage again waits for the tile that had it, at most SLOTS before its own, so no phase
// is missed and none of two tiles mixes.
constexpr int SLOTS = 8;
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity);
__device__ __forceinline__ bool wait_nth(uint64_t* bars, int nth) { return nth < 0 || wait_for(&bars[nth % SLOTS], (nth / SLOTS) & 1); }

// The stage of a ring, tile by tile.
template <int STAGES>
struct Ring {
  int stage = 0;
  __device__ __forceinline__ void next() { stage = stage + 1 == STAGES ? 0 : stage + 1; }
};

// A shared-memory operand, K-major with 128-byte rows and swizzle (8-row groups 1024 bytes apart), from 16 bytes' number `at16` on.
__device__ __forceinline__ uint64_t desc(uint32_t at16) {
  constexpr uint64_t FIXED = (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
  return FIXED | at16;
}

// The whole warp goes through the loops that copy and multiply, and where something is issued, the one lane that `elected` names does it: in a branch of
// a lane that the compiler cannot tell to be alone, every operand would first have to be made uniform (a k-block's four MMAs and two waits took
// 1100 cycles so, more than the products themselves).
__device__ __forceinline__ bool elected() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one;
}

__device__ __forceinline__ void mma_a_tmem(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Whether the phase with this parity is complete, without waiting.
__device__ __forceinline__ uint32_t look(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return done;
}

// mbar_wait behind one look, which mostly suffices
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return done || mbar_wait(bar, parity);
}

__device__ __forceinline__ void tmem_store32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
      "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]),
      "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_load16(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float load_from(const float* p, uint32_t rank) {     // `p` in the shared memory of the cluster's CTA `rank`
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The codes and scales of a thread's row in one tile of 128 k: the words of its four blocks in each of the tile's quarters.
struct RowTile {
  uint4 c[4];
  uint32_t s;
};
__device__ __forceinline__ void load_row_tile(RowTile& q, const uint8_t* codes, const uint8_t* scales, bool valid) {
#pragma unroll
  for (int t = 0; t < 4; ++t)
    asm volatile(
        "{\n\t.reg .pred ok;\n\t"
        "setp.ne.b32 ok, %5, 0;\n\t"
        "mov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
        "@ok ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
        : "=r"(q.c[t].x), "=r"(q.c[t].y), "=r"(q.c[t].z), "=r"(q.c[t].w) : "l"(codes + t * 16), "r"((int)valid));
  asm volatile("{\n\t.reg .pred ok;\n\tsetp.ne.b32 ok, %2, 0;\n\tmov.b32 %0, 0;\n\t@ok ld.global.nc.u32 %0, [%1];\n\t}"
               : "=r"(q.s) : "l"(scales), "r"((int)valid));
}

// Copies to shared memory that the thread waits for itself; zeros where there is nothing.
__device__ __forceinline__ void copy_16(uint32_t to, const void* from, bool there) {
  asm volatile("{\n\t.reg .pred no;\n\tsetp.eq.b32 no, %2, 0;\n\tcp.async.cg.shared.global [%0], [%1], 16, no;\n\t}"
               ::"r"(to), "l"(from), "r"((int)there) : "memory");
}
__device__ __forceinline__ void copy_4(uint32_t to, const void* from, bool there) {
  asm volatile("{\n\t.reg .pred no;\n\tsetp.eq.b32 no, %2, 0;\n\tcp.async.ca.shared.global [%0], [%1], 4, no;\n\t}"
               ::"r"(to), "l"(from), "r"((int)there) : "memory");
}
__device__ __forceinline__ uint4 load_shared16(uint32_t from) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(from) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t load_shared4(uint32_t from) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(from) : "memory");
  return v;
}

// The values of the tile's first or second 64 k, two a register.
template <int HALF>
__device__ __forceinline__ void convert(const RowTile& q, uint32_t (&v)[32]) {
  const uint32_t s[2] = {(q.s >> (16 * HALF)) & 255u, (q.s >> (16 * HALF + 8)) & 255u};
  const bool far = __any_sync(0xffffffffu, max(s[0], s[1]) > NEAR);
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const uint32_t w[2] = {HALF ? q.c[t].z : q.c[t].x, HALF ? q.c[t].w : q.c[t].y};
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      uint32_t x[4];
      values(w[b], factor(s[b]), x);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[b * 16 + t * 4 + j] = x[j];
    }
  }
  if (far) {
    const uint32_t left[2] = {factor_left(s[0]), factor_left(s[1])};
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      v[j] = mul2(v[j], left[j >> 4]);
      asm volatile("" : "+r"(v[j]));          // (a branch of its own, not 32 instructions that mostly do nothing)
    }
  }
}

// A box from (x, y) where `one` is true: predicated, because behind a branch the operands would be made uniform first (see `elected`).
__device__ __forceinline__ void tma_load_if(bool one, void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "@p cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n\t}"
      ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"((int)one) : "memory");
}

// A tile's values to a stage of tensor memory, once the products of the tile that had it (`before`; negative: none) are done; `then` runs when
// the tile's codes are used up. False where the wait ran out or somebody gave up.
template <typename Then>
__device__ __forceinline__ bool give_tile(uint32_t taddr, const RowTile& q, uint64_t* full, uint64_t* done, int before, volatile uint32_t* aborted,
                                          Then then) {
  uint32_t v[32];
  convert<0>(q, v);
  if (!__all_sync(0xffffffffu, wait_nth(done, before) && *aborted == 0)) return false;
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  tmem_store32(taddr, v);
  convert<1>(q, v);
  tmem_store32(taddr + KB / 2, v);
  then();
  tmem_stored();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(full);
  return true;
}

// At a CTA's end, where somebody gave up: of the `copied` tiles the last `STAGES` may not be there yet, and they land before the CTA's shared memory
// goes away. A converting warp that left early (of a tile's group of four, in place `left` of the CTA's tiles) owes its arrivals from there on.
template <int STAGES, int GROUPS>
__device__ __forceinline__ void drain(uint64_t* full, int copied, int k_tiles, volatile int* left, int lane) {
  for (int c = max(0, copied - STAGES); c < copied; ++c) {
    if (lane < 4 && left[c % k_tiles % GROUPS * 4 + lane] <= c) mbar_arrive(&full[c % SLOTS]);
    __syncwarp();
    mbar_wait(&full[c % SLOTS], (c / SLOTS) & 1);
  }
}

// The products of a tile of 128 k (of its first 64 where there is no `second`): weights at `a` in tensor memory, token rows at 16 bytes' number `b` in
// shared memory, the second 64 k `half16` behind the first. Their end arrives at `done`.
__device__ __forceinline__ void multiply_tile(uint32_t d, uint32_t a, uint32_t b, uint32_t half16, uint32_t idesc, bool add, bool second,
                                              uint64_t* done) {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (elected()) {
#pragma unroll
    for (int k = 0; k < KB / 16; ++k) mma_a_tmem(d, a + k * 8, desc(b + k * 2), idesc, (add || k > 0) ? 1u : 0u);
    if (second) {
#pragma unroll
      for (int k = 0; k < KB / 16; ++k) mma_a_tmem(d, a + KB / 2 + k * 8, desc(b + half16 + k * 2), idesc, 1u);
    }
    commit(done);
  }
  __syncwarp();
}

template <typename TOut> __device__ __forceinline__ void store_one(TOut* p, float v) { *p = from_f32<TOut>(v); }

template <int BN, bool GATED, bool SPLIT, typename TOut>
__global__ void __launch_bounds__(THREADS, 2) tc_kernel(const __grid_constant__ CUtensorMap tmX, TcParams p) {
  using S = Tc<BN>;
  constexpr int OUTS = GATED ? ROWS / 2 : ROWS;
  chain_wait();
  const int tok0 = blockIdx.y * BN, tok_rows = min(BN, p.M - tok0);
  const int n0 = blockIdx.x * OUTS;
  const int k_tiles = ceil_div(p.K, TILE_K);
  const int tile0 = SPLIT ? (int)blockIdx.z * p.tiles_a_split : 0;              // first tile of 128 k
  const int kb0 = 2 * tile0, num_kb = min(ceil_div(p.K, KB), SPLIT ? kb0 + 2 * p.tiles_a_split : 0x7fffffff) - kb0;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* boxes = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = (uint64_t*)(boxes + S::B_STAGES * S::B_BYTES);
  uint64_t* done = full + SLOTS;
  uint64_t* acc_full = done + SLOTS;
  uint32_t* tmem_slot = (uint32_t*)(acc_full + 1);
  volatile uint32_t* aborted = tmem_slot + 1;
  volatile int* copied = (int*)(tmem_slot + 2);
  volatile int* left = copied + 1;                              // see drain()

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&full[s], 5);
      mbar_init(&done[s], 1);
    }
    mbar_init(acc_full, 1);
    *aborted = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x < EPI_WARPS) left[threadIdx.x] = 0x7fffffff;
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)S::TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = *tmem_slot;
  chain_next();               // (only now: see the persistent form)
  auto give_up = [&]() {
    *aborted = 1;
    atomicExch(p.status, 11);
  };

  const int tiles = ceil_div(num_kb, 2);
  if (warp == 0) {
    // ---- token rows ----
    Ring<S::B_STAGES> ring;
    int issued = 0;
    const int copies = min(tiles, p.copies);
    for (int c = 0; c < copies; ++c, ring.next()) {
      if (!__all_sync(0xffffffffu, wait_nth(done, c - S::B_STAGES) && *aborted == 0)) {
        give_up();
        break;
      }
      const int blocks = min(2, num_kb - 2 * c);
      if (elected()) {
        mbar_expect_tx(&full[c % SLOTS], blocks * S::HALF_BYTES);
        for (int i = 0; i < blocks; ++i)
          tma_load_2d(boxes + ring.stage * S::B_BYTES + i * S::HALF_BYTES, &tmX, &full[c % SLOTS], (kb0 + 2 * c + i) * KB, tok0);
      }
      __syncwarp();
      issued = c + 1;
    }
    *copied = issued;
  } else if (warp == 1) {
    // ---- products: f32 sums, bf16 operands, both K-major, M = 128, N = BN ----
    constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(ROWS >> 4) << 24);
    Ring<S::A_STAGES> ra;
    Ring<S::B_STAGES> rb;
    bool there = false;
    const int products = min(tiles, p.products);
    for (int c = 0; c < products; ++c, ra.next(), rb.next()) {
      if (!there && !__all_sync(0xffffffffu, wait_nth(full, c))) {
        give_up();
        break;
      }
      const uint32_t next = look(&full[(c + 1) % SLOTS], ((c + 1) / SLOTS) & 1);
      multiply_tile(tmem_base, tmem_base + BN + ra.stage * S::A_COLS, smem_u32(boxes + rb.stage * S::B_BYTES) >> 4, S::HALF_BYTES >> 4, idesc, c > 0,
                    2 * c + 1 < num_kb, &done[c % SLOTS]);
      there = __all_sync(0xffffffffu, next);
    }
    if (products < tiles) give_up();
    if (elected()) commit(acc_full);
    __syncwarp();
    mbar_wait(acc_full, 0);                 // the products have left tensor memory and shared memory before anybody frees them
  } else {
    // ---- weights: tensor-memory lanes 32 (warp % 4) .. + 31, tiles of 128 k of this group's parity ----
    const int half = (warp - 2) >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t t_lane = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
    const int eight = r >> 3, row_tiles = ceil_div(p.N, TILE_ROWS);
    const int row_tile = (n0 >> 3) + (GATED ? eight >> 1 : eight);
    const bool valid = row_tile < row_tiles;
    const long long first = ((GATED ? (long long)(eight & 1) * row_tiles : 0) + (valid ? row_tile : 0)) * k_tiles + tile0;
    const uint8_t* codes = p.codes + first * TILE_CODES + (r & 7) * (TILE_K / 2);
    const uint8_t* scales = p.scales + first * TILE_SCALES + (r & 7) * (TILE_K / BLOCK);
    constexpr int AHEAD = 2;                                    // tiles of codes a thread has at hand or on their way
    RowTile q[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      load_row_tile(q[u], codes + (half + 2 * u) * TILE_CODES, scales + (half + 2 * u) * TILE_SCALES, valid && half + 2 * u < tiles);
    bool ok = true;
    for (int c0 = half; c0 < tiles && ok; c0 += 2 * AHEAD) {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int c = c0 + 2 * u;
        if (c < tiles && ok) {
          ok = give_tile(t_lane + BN + half * S::A_COLS, q[u], &full[c % SLOTS], done, c - S::A_STAGES, aborted, [&]() {
            const int after = c + 2 * AHEAD;
            load_row_tile(q[u], codes + (long long)after * TILE_CODES, scales + (long long)after * TILE_SCALES, valid && after < tiles);
          });
          if (!ok && lane == 0) {
            give_up();
            left[warp - 2] = c;
          }
        }
      }
    }
    // ---- epilogue ----
    if (!__all_sync(0xffffffffu, mbar_wait(acc_full, 0))) {
      if (lane == 0) give_up();
    }
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    ok = __all_sync(0xffffffffu, *aborted == 0);
    if (ok) {
      float* part = (float*)boxes;                              // SPLIT: [BN][128]; the products have read the boxes
      TOut* C = (TOut*)p.C;
      const int n = n0 + (GATED ? (r >> 4) * 8 + (r & 7) : r);
      const bool mine = n < p.N, up = GATED && (eight & 1);
      float bias = 0.f;
      if (!SPLIT && p.bias && mine) bias = p.bias[up ? p.N + n : n];
#pragma unroll 1
      for (int c0 = half * 16; c0 < min(BN, tok_rows); c0 += 32) {
        float v[16];
        tmem_load16(t_lane + c0, v);
        const int left = tok_rows - c0;
        if constexpr (SPLIT) {
#pragma unroll
          for (int j = 0; j < 16; ++j) part[(c0 + j) * ROWS + r] = v[j];
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] += bias;
          if constexpr (GATED) {
            // of two tokens the lane with the gate row finishes the first and the one with the up row the second
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
              const float other = __shfl_xor_sync(0xffffffffu, up ? v[j] : v[j + 1], 8);
              const float out = gated(up ? other : v[j], up ? v[j + 1] : other, p.act, p.ga0, p.ga1);
              const int m = up ? j + 1 : j;
              if (mine && m < left) store_one(C + (long long)(tok0 + c0 + m) * p.ldc + n, out);
            }
          } else {
            if (p.act < 0) {
#pragma unroll
              for (int j = 0; j < 16; ++j) v[j] = gate_activation(v[j], -p.act);
            }
            if (mine) {
              TOut* to = C + (long long)(tok0 + c0) * p.ldc + n;
#pragma unroll
              for (int j = 0; j < 16; ++j)
                if (j < left) store_one(to + (long long)j * p.ldc, v[j]);
            }
          }
        }
      }
    }
  }
  if constexpr (SPLIT) {
    __syncthreads();
    __syncwarp();
    cluster_sync();
    if (warp >= 2 && *aborted == 0) {
      const float* part = (const float*)boxes;
      TOut* C = (TOut*)p.C;
      const int rank = (int)cluster_rank(), ranks = gridDim.z, at = threadIdx.x - 64;
      const int o = at & (OUTS - 1), n = n0 + o;
      const int r = GATED ? (o >> 3) * 16 + (o & 7) : o;
      if (n < p.N) {
        for (int m = rank + ranks * (at / OUTS); m < tok_rows; m += ranks * (32 * EPI_WARPS / OUTS)) {
          float v = 0.f, u = 0.f;
          for (int s = 0; s < ranks; ++s) {
            v += load_from(part + m * ROWS + r, s);
            if (GATED) u += load_from(part + m * ROWS + r + 8, s);
          }
          if (p.bias) {
            v += p.bias[n];
            if (GATED) u += p.bias[p.N + n];
          }
          const float out = GATED ? gated(v, u, p.act, p.ga0, p.ga1) : p.act < 0 ? gate_activation(v, -p.act) : v;
          store_one(C + (long long)(tok0 + m) * p.ldc + n, out);
        }
      }
    }
    __syncwarp();
    cluster_sync();                                             // no CTA leaves while another reads its sums
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 0 && *aborted) drain<S::B_STAGES, 2>(full, *copied, tiles, left, lane);
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)S::TMEM_COLS));
  }
}

// ---------------------------------------------------------------------------------------------------------------
// The same for prompts and routed experts: a persistent CTA an SM, whose token tiles are up to MAXN rows high, so that the conversion of a tile of
// weights hides under its products (4 cycles a token row; both with what they wait for: 0.45 us a tile up to 200 rows). Tensor memory holds two
// accumulators of 160 columns and three stages of weights, or one of 256 and four where that saves a round, or (few rows an expert) two of 64 and
// six: the way of a stage, from its values to its products' end and back, takes some 2000 cycles, of which every stage more hides a part (2048
// rows, 7168 gated outputs of 2048: 103 us with two stages beside two accumulators of 192 where these took 99; 92 since). Eight warps of their own
// finish a tile while the next one's products run. The N side of an MMA is as many token rows as the tile has, rounded up to 16, and they come in
// boxes of 256, 80 or 16.
//
// With few rows an expert the converting warps are what takes longest: sixteen of them, and four that finish (a layer of 64 experts with 4 rows
// each, 768 by 2048: 87 us with eight, 76 with twelve, 74 with sixteen; 72 with the sign and the rest of a pair put in place by one multiplication,
// which took 5 to 10 % off all of these products; 69 with a tile's codes read from shared memory while the stores of the one before are under way).
// Tiles as low of one matrix have the form of 160 rows, whose eight finishing warps are sooner done when nothing runs beside them (150 rows, 2500
// gated outputs of 1096: 10.8 us, 13.4 with four).
template <int MAXN>
struct Many {
  static constexpr int BOX_ROWS = MAXN > 160 ? 256 : MAXN > 64 ? 80 : 16;      // token rows a TMA box
  static constexpr int BOX_BYTES = BOX_ROWS * KB * 2;
  static constexpr int HALF_BYTES = MAXN * KB * 2;
  static constexpr int B_BYTES = 2 * HALF_BYTES;                 // a stage of token rows: a tile of 128 k, its two k-blocks one after the other
  static constexpr int B_STAGES = MAXN > 160 ? 3 : MAXN > 64 ? 4 : 5;
  static constexpr int A_COLS = TILE_K / 2;                      // a stage of weights: a tile of 128 k
  static constexpr int A_STAGES = MAXN > 160 ? 4 : MAXN > 64 ? 3 : 6;
  static constexpr int ACCS = MAXN > 160 ? 1 : 2;
  static constexpr int A_AT = 512 - A_STAGES * A_COLS;           // the accumulators come first
  static constexpr int CONVERT_WARPS = MAXN > 64 ? 8 : 16;
  static constexpr int FINISH_WARPS = MAXN > 64 ? 8 : 4;
  static constexpr int GROUPS = CONVERT_WARPS / 4;
  static constexpr int THREADS = (2 + CONVERT_WARPS + FINISH_WARPS) * 32;
  // Tiles of codes that a converting warp has on their way to its part of shared memory (more gain nothing); 0: two in registers,
  // where the token rows leave no room. Through shared memory a warp's copies are whole lines: 768 rows to 32 experts 133 -> 122 us.
  static constexpr int AHEAD = MAXN > 160 ? 0 : MAXN > 64 ? 3 : 2;
  static constexpr int SLOT_BYTES = 4 * (TILE_CODES + TILE_SCALES);
  static constexpr int TOTAL = B_STAGES * B_BYTES + CONVERT_WARPS * AHEAD * SLOT_BYTES + 1024 /* alignment slack */ + 256 /* barriers */;
  static_assert(TOTAL <= 227 * 1024, "a CTA's shared memory");
  static_assert(ACCS * MAXN <= A_AT, "accumulators and weights share tensor memory");
  static_assert(BOX_BYTES % 1024 == 0, "a box begins where the swizzle does");
  static_assert(A_STAGES <= SLOTS && B_STAGES <= SLOTS, "see SLOTS");
};

__device__ __forceinline__ void gate_all(float (&g)[8], const float (&u)[8], const TcParams& p) {
  if (p.act == TL_ACT_SILU) {          // (the fast exponential and division: the result is rounded to bfloat16, far coarser than their error)
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = __fdividef(g[j], 1.f + __expf(-g[j])) * u[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = gated(g[j], u[j], p.act, p.ga0, p.ga1);
  }
}

template <int MAXN, bool GATED, typename TOut>
__global__ void __launch_bounds__(Many<MAXN>::THREADS, 1) tc_many_kernel(const __grid_constant__ CUtensorMap tmX, TcParams p, int tile_at_most) {
  using S = Many<MAXN>;
  constexpr int OUTS = GATED ? ROWS / 2 : ROWS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* boxes = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* slots = boxes + S::B_STAGES * S::B_BYTES;
  uint64_t* full = (uint64_t*)(slots + S::CONVERT_WARPS * S::AHEAD * S::SLOT_BYTES);
  uint64_t* done = full + SLOTS;
  uint64_t* acc_full = done + SLOTS;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = (uint32_t*)(acc_empty + 2);
  volatile uint32_t* aborted = tmem_slot + 1;
  volatile int* copied = (int*)(tmem_slot + 2);
  volatile int* left = copied + 1;                              // see drain()

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&full[s], 5);
      mbar_init(&done[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], S::FINISH_WARPS);                // one arrival each
    }
    *aborted = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x < S::CONVERT_WARPS) left[threadIdx.x] = 0x7fffffff;
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = *tmem_slot;
  // The next kernel of a layer may come only when every CTA of this one has its tensor memory: it takes its own before it waits for this kernel's end,
  // and a CTA here that waited for what a cluster of another stream holds, while that cluster waits for what the next kernel holds, would close a circle.
  chain_next();
  chain_wait();
  auto give_up = [&]() {
    *aborted = 1;
    atomicExch(p.status, 11);
  };

  const int k_tiles = ceil_div(p.K, TILE_K), num_kb = ceil_div(p.K, KB), row_tiles = ceil_div(p.N, TILE_ROWS);
  const int tiles_n = ceil_div(p.N, OUTS), tiles_m = p.tile_group ? *p.n_tiles : ceil_div(p.M, tile_at_most);
  const int work = tiles_n * tiles_m;
  // work item w: token tile w / tiles_n, weight tile w % tiles_n (neighbouring CTAs share token rows). What is to be known of the next item is
  // read while this one is at work: a read's 700 cycles an item would be as long as one or two of its tiles.
  struct Tokens {
    int first, rows;
  };
  auto tokens_of = [&](int w) {
    Tokens t = {0, 0};
    if (w < work) {
      const int tm = w / tiles_n;
      t.first = p.tile_group ? p.tile_row0[tm] : tm * tile_at_most;
      t.rows = p.tile_group ? p.tile_rows[tm] : min(tile_at_most, p.M - t.first);
    }
    return t;
  };

  if (warp == 0) {
    // ---- token rows ----
    Ring<S::B_STAGES> ring;
    int issued = 0;
    bool ok = true;
    Tokens coming = tokens_of(blockIdx.x);
    for (int w = blockIdx.x; w < work && ok; w += gridDim.x) {
      const int tok0 = coming.first, tok_rows = min(coming.rows, MAXN);
      coming = tokens_of(w + gridDim.x);
      const int boxes_here = ceil_div(tok_rows, S::BOX_ROWS);
      const int copies = min(k_tiles, p.copies - issued);
      for (int c = 0; c < copies; ++c, ring.next()) {
        if (!__all_sync(0xffffffffu, wait_nth(done, issued - S::B_STAGES) && *aborted == 0)) {
          give_up();
          ok = false;
          break;
        }
        const int blocks = min(2, num_kb - 2 * c);
        const bool one = elected();
        uint64_t* bar = &full[issued % SLOTS];
        uint8_t* at = boxes + ring.stage * S::B_BYTES;
        if (one) mbar_expect_tx(bar, blocks * boxes_here * S::BOX_BYTES);
        for (int b = 0; b < boxes_here; ++b) {
          tma_load_if(one, at + b * S::BOX_BYTES, &tmX, bar, 2 * c * KB, tok0 + b * S::BOX_ROWS);
          if (blocks == 2) tma_load_if(one, at + S::HALF_BYTES + b * S::BOX_BYTES, &tmX, bar, 2 * c * KB + KB, tok0 + b * S::BOX_ROWS);
        }
        __syncwarp();
        ++issued;
      }
      if (copies < k_tiles) break;
    }
    *copied = issued;
  } else if (warp == 1) {
    // ---- products ----
    Ring<S::A_STAGES> ra;
    Ring<S::B_STAGES> rb;
    Ring<S::ACCS> rd;
    int tile = 0, items = 0;
    bool ok = true, there = false;
    Tokens coming = tokens_of(blockIdx.x);
    for (int w = blockIdx.x; w < work && ok; w += gridDim.x, rd.next()) {
      const int tok_rows = min(coming.rows, MAXN);
      coming = tokens_of(w + gridDim.x);
      const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(ceil_div(tok_rows, 16) * 2) << 17) | ((uint32_t)(ROWS >> 4) << 24);
      if (!__all_sync(0xffffffffu, (items < S::ACCS || wait_for(&acc_empty[rd.stage], (items / S::ACCS - 1) & 1)) && *aborted == 0)) {
        give_up();
        break;
      }
      const uint32_t d = tmem_base + rd.stage * MAXN;
      const int products = min(k_tiles, p.products - tile);
      for (int c = 0; c < products; ++c, ++tile, ra.next(), rb.next()) {
        if (!there && !__all_sync(0xffffffffu, wait_nth(full, tile))) {
          give_up();
          ok = false;
          break;
        }
        // A look at the next tile's operands in front of this one's products, which costs the tensor pipe nothing there; a wait behind them would
        // leave it idle.
        const uint32_t next = look(&full[(tile + 1) % SLOTS], ((tile + 1) / SLOTS) & 1);
        multiply_tile(d, tmem_base + S::A_AT + ra.stage * S::A_COLS, smem_u32(boxes + rb.stage * S::B_BYTES) >> 4, S::HALF_BYTES >> 4, idesc, c > 0,
                      2 * c + 1 < num_kb, &done[tile % SLOTS]);
        there = __all_sync(0xffffffffu, next);
      }
      if (products < k_tiles) {
        give_up();
        ok = false;
      }
      if (elected()) commit(&acc_full[rd.stage]);      // (also where it gave up: whoever waits learns of it)
      __syncwarp();
      ++items;
    }
    // the last products have left tensor memory and shared memory before anybody frees them
    if (items > 0) mbar_wait(&acc_full[(items - 1) % S::ACCS], ((items - 1) / S::ACCS) & 1);
  } else if (warp < 2 + S::CONVERT_WARPS) {
    // ---- weights: tensor-memory lanes 32 (warp % 4) .. + 31, every GROUPS-th tile of 128 k ----
    const int turn = (warp - 2) >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t t_lane = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + S::A_AT;
    // The warp's 32 rows are four tiles of 8 rows: two and two, or gated two of the gate and two of the up matrix in turn.
    const int eight0 = (warp & 3) * 4, eight = r >> 3;
    auto row_tile_of = [&](int n0, int e) { return (n0 >> 3) + (GATED ? e >> 1 : e); };
    const long long line = (long long)k_tiles * TILE_CODES, matrix_bytes = row_tiles * line;
    // where a thread is: the work item, the tile of 128 k, and that tile of its row (AHEAD: its 16 bytes of the warp's first row tile)
    struct Cursor {
      int w, c, row_tile, group;                                // (the group: the next item's)
      const uint8_t* codes;
      const uint8_t* scales;
    };
    auto group_of = [&](int w) { return p.tile_group && w < work ? p.tile_group[w / tiles_n] : 0; };
    auto enter = [&](Cursor& q, int w) {
      q.w = w;
      q.c = turn;
      q.row_tile = row_tiles;
      q.codes = p.codes, q.scales = p.scales;
      if (w >= work || turn >= k_tiles) return;
      const int n0 = w % tiles_n * OUTS, group = q.group;
      q.group = group_of(w + gridDim.x);
      const int mine = row_tile_of(n0, eight), first = row_tile_of(n0, eight0);
      q.row_tile = S::AHEAD ? first : mine;
      const long long matrix = (long long)group * p.matrices * row_tiles;
      const long long own = (matrix + (GATED ? (long long)(eight & 1) * row_tiles : 0) + min(mine, row_tiles - 1)) * k_tiles;
      q.codes = S::AHEAD ? p.codes + (matrix + min(first, row_tiles - 1)) * k_tiles * TILE_CODES + lane * 16
                         : p.codes + own * TILE_CODES + (r & 7) * (TILE_K / 2);
      q.scales = p.scales + own * TILE_SCALES + (r & 7) * (TILE_K / BLOCK);
      q.codes += turn * TILE_CODES, q.scales += turn * TILE_SCALES;
    };
    auto advance = [&](Cursor& q) {
      q.c += S::GROUPS, q.codes += S::GROUPS * TILE_CODES, q.scales += S::GROUPS * TILE_SCALES;
      if (q.c >= k_tiles) enter(q, q.w + gridDim.x);
    };
    constexpr int BUFFERS = S::AHEAD ? 1 : 2;
    RowTile q[BUFFERS];
    Cursor next, now;
    next.group = group_of(blockIdx.x);
    enter(next, blockIdx.x);
    now = next;
    // A slot is four tiles' codes and their rows' scales. A row's 16 bytes of quarter t lie at t ^ (row / 2 % 4), so that both the copies (a lane
    // 16 bytes of a tile) and the reads (a lane a row) fall on all banks.
    const uint32_t my_slots = smem_u32(slots + (warp - 2) * (S::AHEAD * S::SLOT_BYTES));
    const uint32_t put = (lane >> 2) * 64 + (((lane & 3) ^ ((lane >> 3) & 3)) << 4);
    const uint32_t take = (lane >> 3) * TILE_CODES + (lane & 7) * 64, turned = ((lane & 7) >> 1) << 4;
    int to = 0, from = 0;                                       // slots' offsets
    auto fetch = [&](RowTile& q) {                              // the tile at `next`, on its way
      if constexpr (S::AHEAD > 0) {
        __syncwarp();                                           // (all lanes have read what the slot held)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          copy_16(my_slots + to + j * TILE_CODES + put, next.codes + (GATED ? (j & 1) * matrix_bytes + (j >> 1) * line : j * line),
                  next.row_tile + (GATED ? j >> 1 : j) < row_tiles);
        copy_4(my_slots + to + 4 * TILE_CODES + lane * 4, next.scales, next.row_tile + (GATED ? lane >> 4 : lane >> 3) < row_tiles);
        asm volatile("cp.async.commit_group;" ::: "memory");
        to = to + S::SLOT_BYTES == S::AHEAD * S::SLOT_BYTES ? 0 : to + S::SLOT_BYTES;
      } else {
        load_row_tile(q, next.codes, next.scales, next.row_tile < row_tiles);
      }
      advance(next);
    };
#pragma unroll
    for (int u = 0; u < (S::AHEAD ? S::AHEAD : BUFFERS); ++u) fetch(q[u % BUFFERS]);
    auto read = [&](RowTile& q) {                               // the oldest tile of those on their way
      if constexpr (S::AHEAD > 0) {
        asm volatile("cp.async.wait_group %0;" ::"n"(S::AHEAD > 0 ? S::AHEAD - 1 : 0) : "memory");
        __syncwarp();
#pragma unroll
        for (int t = 0; t < 4; ++t) q.c[t] = load_shared16(my_slots + from + take + ((t << 4) ^ turned));
        q.s = load_shared4(my_slots + from + 4 * TILE_CODES + lane * 4);
        from = from + S::SLOT_BYTES == S::AHEAD * S::SLOT_BYTES ? 0 : from + S::SLOT_BYTES;
      }
    };
    read(q[0]);
    // The tiles of all of the CTA's work items are one sequence; this group's are every GROUPS-th of an item, so the stage of one is its place
    // in the sequence, and how often the stage was used before it that place's round.
    int at = turn;                                              // the place of the tile at hand
    bool ok = true;
    while (ok && now.w < work && turn < k_tiles) {
#pragma unroll
      for (int u = 0; u < BUFFERS; ++u) {
        if (!ok || now.w >= work) break;
        const int stage = at % S::A_STAGES;
        ok = give_tile(t_lane + stage * S::A_COLS, q[u], &full[at % SLOTS], done, at - S::A_STAGES, aborted, [&]() {
          fetch(q[u]);
          read(q[u]);
        });
        if (!ok && lane == 0) {
          give_up();
          left[warp - 2] = at;
        }
        const int before = now.c;
        now.c += S::GROUPS;
        if (now.c >= k_tiles) {
          now.c = turn, now.w += gridDim.x;
          at += k_tiles - before + turn;
        } else {
          at += S::GROUPS;
        }
      }
    }
    // (also where it gave up: nothing may arrive in shared memory that is another CTA's by then)
    if constexpr (S::AHEAD > 0) asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    // ---- results: accumulator rows 32 (warp % 4) .. + 31 ----
    const int r = (warp & 3) * 32 + lane, eight = r >> 3;
    const bool up = GATED && (eight & 1);
    const int other = (warp - 2 - S::CONVERT_WARPS) >> 2;       // of the warps of a quarter of the rows, which take 16 columns in turn
    int nth = 0;
    Tokens coming = tokens_of(blockIdx.x);
    for (int w = blockIdx.x; w < work; w += gridDim.x, ++nth) {
      const int tok0 = coming.first, tok_rows = min(coming.rows, MAXN);
      coming = tokens_of(w + gridDim.x);
      const int acc = nth % S::ACCS, n = (w % tiles_n) * OUTS + (GATED ? (r >> 4) * 8 + (r & 7) : r);
      const bool mine = n < p.N;
      const float bias = p.bias && mine ? p.bias[up ? p.N + n : n] : 0.f;
      if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[acc], (nth / S::ACCS) & 1) && *aborted == 0)) {
        if (lane == 0) give_up();
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t from = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + acc * MAXN;
      TOut* C = (TOut*)p.C;
#pragma unroll 1
      for (int c0 = other * 16; c0 < tok_rows; c0 += S::FINISH_WARPS * 4) {
        float v[16];
        tmem_load16(from + c0, v);
        const int left = tok_rows - c0;
        if (p.row_weight) {
          const float weight = (lane & 15) < left ? weight_of(p, (long long)tok0 + c0 + (lane & 15)) : 1.f;
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] *= __shfl_sync(0xffffffffu, weight, j);
        }
        if (p.bias) {
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] += bias;
        }
        if constexpr (GATED) {
          // of two tokens the lane with the gate row finishes the first and the one with the up row the second
          float g[8], u[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float theirs = __shfl_xor_sync(0xffffffffu, up ? v[2 * j] : v[2 * j + 1], 8);
            g[j] = up ? theirs : v[2 * j];
            u[j] = up ? v[2 * j + 1] : theirs;
          }
          gate_all(g, u, p);
          if (mine) {
            TOut* to = C + (long long)(tok0 + c0 + (up ? 1 : 0)) * p.ldc + n;
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (2 * j + (up ? 1 : 0) < left) store_one(to + (long long)(2 * j) * p.ldc, g[j]);
          }
        } else {
          if (p.act < 0) {
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = gate_activation(v[j], -p.act);
          }
          if (mine) {
            TOut* to = C + (long long)(tok0 + c0) * p.ldc + n;
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (j < left) store_one(to + (long long)j * p.ldc, v[j]);
          }
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[acc]);
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 0 && *aborted) drain<S::B_STAGES, S::GROUPS>(full, *copied, k_tiles, left, lane);
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u));
  }
}

template <int MAXN, bool GATED, typename TOut>
int launch_many(const CUtensorMap& tmX, const TcParams& p, int tile_at_most, long long work, cudaStream_t stream) {
  using S = Many<MAXN>;
  auto kernel = tc_many_kernel<MAXN, GATED, TOut>;
  static thread_local int set_on = -1;              // the device whose function has its shared memory
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (set_on != dev) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::TOTAL);
    if (e != cudaSuccess) return (int)e;
    set_on = dev;
  }
  const dim3 grid((unsigned)(work < sm_count() ? work : sm_count()));
  return launch_behind(p.tile_group != nullptr, kernel, grid, S::THREADS, S::TOTAL, stream, tmX, p, tile_at_most);
}

template <int BN, bool GATED, bool SPLIT, typename TOut>
int launch_tc(const CUtensorMap& tmX, const TcParams& p, dim3 grid, cudaStream_t stream) {
  constexpr int BYTES = SPLIT ? Tc<BN>::SPLIT_TOTAL : Tc<BN>::TOTAL;
  auto kernel = tc_kernel<BN, GATED, SPLIT, TOut>;
  static thread_local int set_on = -1;              // the device whose function has its shared memory
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (set_on != dev) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES);
    if (e != cudaSuccess) return (int)e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return (int)e;
    set_on = dev;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = grid.z;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = BYTES;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = SPLIT ? 1 : 0;
  return (int)cudaLaunchKernelEx(&cfg, kernel, tmX, p);
}

}  // namespace mx
}  // namespace tl

using namespace tl;

// x [x_rows, K] bfloat16 (row stride ldx); the matrix N x K, or gated a gate and an up matrix; grouped (tile_group ..., `splits` 0): as many for
// every group, x in the plan's order, tiles of at most `bn` rows. bias [N] (gated: [2 N]) 32-bit or null. out [M, N] (row stride ldc). `act`
// as in tl_mxfp4_few. `splits` 0: the persistent form, in
// tiles of up to `bn` <= 256 token rows; else token tiles of `bn` rows, 16, 32, 64 or 128, and the CTAs, 1 to 8, that share a tile's k.
extern "C" int tl_mxfp4_tc(const void* x, long long ldx, long long x_rows, const void* codes, const void* scales, const float* bias, void* out,
                           long long ldc, int M, int N, int K, int act, float a0, float a1, int out_dtype, int bn, int splits,
                           const int* tile_group, const int* tile_row0, const int* tile_rows, const int* n_tiles, int max_tiles,
                           const float* row_weight, const int* weight_index, int* status, cudaStream_t stream) {
  if (M == 0 || N == 0 || (tile_group && max_tiles == 0)) return 0;
  TL_REQUIRE(M >= 1 && N >= 1 && K >= 1 && ldx % 8 == 0 && ((uintptr_t)x % 16) == 0, "mxfp4 product: %d rows x (%d x %d), row stride %lld",
             M, N, K, ldx);
  TL_REQUIRE(act <= 0 ? act >= -TL_ACT_IDENTITY : tl_is_gate(act), "mxfp4 product: gate activation %d is none (nor an ungated one, negated)", act);
  TL_REQUIRE(act <= 0 || out_dtype == TL_BF16, "mxfp4 product: gated outputs of type %d", out_dtype);
  const int k_tiles = ceil_div(K, mx::TILE_K);
  TL_REQUIRE(splits >= 0 && splits <= mx::MAX_SPLITS && splits <= k_tiles, "mxfp4 product: k %d in %d runs", K, splits);
  TL_REQUIRE(!tile_group || (tile_row0 && tile_rows && n_tiles), "mxfp4 product: an incomplete plan (%d tiles)", max_tiles);
  TL_REQUIRE((!tile_group && !row_weight) || (tile_group && splits == 0), "mxfp4 product: groups and rows' weights in %d runs of k; the persistent form "
             "alone has them", splits);
  TL_REQUIRE(splits == 0 || bn == 16 || bn == 32 || bn == 64 || bn == 128, "mxfp4 product: token tiles of %d rows; 16, 32, 64 or 128", bn);
  mx::TcParams p = {};
  p.codes = (const uint8_t*)codes, p.scales = (const uint8_t*)scales, p.bias = bias, p.C = out, p.ldc = ldc, p.M = M, p.N = N, p.K = K;
  p.matrices = act > 0 ? 2 : 1;
  if (splits) {
    p.tiles_a_split = ceil_div(k_tiles, splits);
    splits = ceil_div(k_tiles, p.tiles_a_split);                // (rounding up may leave the last ones nothing)
  }
  p.tile_group = tile_group, p.tile_row0 = tile_row0, p.tile_rows = tile_rows, p.n_tiles = n_tiles;
  p.copies = mx::stop_for_test().copies, p.products = mx::stop_for_test().products;
  p.act = act, p.ga0 = a0, p.ga1 = a1, p.row_weight = row_weight, p.weight_index = weight_index, p.status = status;
  if (splits == 0) {
    TL_REQUIRE(bn >= 1 && bn <= 256, "mxfp4 product: token tiles of %d rows", bn);
    const long long work = (long long)ceil_div(N, act > 0 ? mx::ROWS / 2 : mx::ROWS) * (tile_group ? max_tiles : ceil_div(M, bn));
    TL_REQUIRE(work <= 0x7FFFFFFF, "mxfp4 product: %lld tiles are too many", work);
    CUtensorMap tmX;
    const int box = bn <= 64 && tile_group ? mx::Many<64>::BOX_ROWS : bn <= 160 ? mx::Many<160>::BOX_ROWS : mx::Many<256>::BOX_ROWS;
    const int r = tensor_map(x, x_rows, K, ldx, box, &tmX);
    if (r) return r;
#define TL_MX_MANY(N_)                                                                                \
  do {                                                                                                \
    if (act > 0) return mx::launch_many<N_, true, bf16>(tmX, p, bn, work, stream);                    \
    if (out_dtype == TL_FP32) return mx::launch_many<N_, false, float>(tmX, p, bn, work, stream);     \
    return mx::launch_many<N_, false, bf16>(tmX, p, bn, work, stream);                                \
  } while (0)
    if (bn <= 64 && tile_group) TL_MX_MANY(64);
    if (bn <= 160) TL_MX_MANY(160);
    TL_MX_MANY(256);
#undef TL_MX_MANY
  }
  const dim3 grid(ceil_div(N, act > 0 ? mx::ROWS / 2 : mx::ROWS), ceil_div(M, bn), splits);
  TL_REQUIRE(grid.y <= 65535, "mxfp4 product: %d token tiles exceed the grid limit", (int)grid.y);
  CUtensorMap tmX;
  const int r = tensor_map(x, x_rows, K, ldx, bn, &tmX);
  if (r) return r;
#define TL_MX_TC_(BN_, S_)                                                                            \
  do {                                                                                                \
    if (act > 0) return mx::launch_tc<BN_, true, S_, bf16>(tmX, p, grid, stream);                     \
    if (out_dtype == TL_FP32) return mx::launch_tc<BN_, false, S_, float>(tmX, p, grid, stream);      \
    return mx::launch_tc<BN_, false, S_, bf16>(tmX, p, grid, stream);                                 \
  } while (0)
#define TL_MX_TC(BN_)                 \
  do {                                \
    if (splits > 1) TL_MX_TC_(BN_, true); \
    TL_MX_TC_(BN_, false);            \
  } while (0)
  if (bn == 16) TL_MX_TC(16);
  if (bn == 32) TL_MX_TC(32);
  if (bn == 64) TL_MX_TC(64);
  TL_MX_TC(128);
#undef TL_MX_TC
#undef TL_MX_TC_
}

// For tests of the bounded waits: the polls after which a wait of this file's kernels gives up (0 puts the default back), and the tiles of 128 k,
// counted over a CTA's work, behind which no token rows are copied and behind which the products give up (-1: none).
extern "C" int tl_mxfp4_tc_set_wait_limit(unsigned int polls) {
  const uint32_t v = polls ? polls : (1u << 22);
  return (int)cudaMemcpyToSymbol(wait_limit, &v, sizeof(v));
}
extern "C" void tl_mxfp4_tc_test_stop(int copies, int products) {
  mx::stop_for_test() = {copies < 0 ? 0x7fffffff : copies, products < 0 ? 0x7fffffff : products};
}
