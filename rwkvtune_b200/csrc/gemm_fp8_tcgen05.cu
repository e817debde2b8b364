// 8-bit GEMM on pairs of SMs: C[M,N] = op(A) op(B) for operands in the block format of fp8_format.cuh, one 256x256 output
// tile per cluster of two CTAs, issued as tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale with fp32 accumulation.
//
// Scales.  The format's scales are powers of two, so the tensor core applies them: its instruction takes one E8M0 byte per
// row and 32 contraction elements, and the byte of a 128-block is simply named by the four instructions that cover the
// block.  The accumulator is never rescaled by ordinary threads (which, at 128 columns of contraction a step, would cost
// as long as the step's products themselves).  A scale warp in each CTA gathers the bytes of four blocks (512 elements of
// the contraction) into the 32-lane layout that tcgen05.cp copies into tensor memory.
//
// Operands may be K-major or MN-major; tiles of 128 x 128 have the same scale in either direction, so one packed copy of an
// activation, a gradient or a weight serves every product it takes part in:  y = x W^T (NT), dx = dy W (NN),
// dW = dy^T x (TN).  Every operand tile is 128 rows of 128 bytes in shared memory, whatever its direction.
// Blocks of one row (a_rows = 1) exist for a K-major A.
//
// Epilogues: store bf16; add a bf16 residual; and two that put the result back into the block format without writing it in
// 16 bits - relu(x)^2 (the forward activation that is kept for backward) and x * 2 sqrt(h) with h the kept activation (its
// derivative).  A CTA owns 128 rows and two blocks of 128 columns, so a tile's scale is a maximum inside one CTA; a thread
// owns a row, so the scale of a row block is a maximum inside one thread.
//
// Tensor memory holds two 256-column accumulators that overlap by 64 columns plus four 16-column sets of scales.  The
// epilogue of a tile reads the shared 64 columns first and releases them; the products of the next tile start there, so
// the overlap costs one 64-column read per tile instead of a whole drained accumulator.  Two groups of four warps drain a
// tile, 128 columns each.
//
// What bounds it.  A step of 128 contraction elements is 512 cycles of the tensor pipe.  Measured over whole kernels it takes
// 519 cycles in dW 8192 x 2048 x 32768 (TN), 534 in 32768 x 2048 x 8192 (NN), and 606 to 628 at a contraction of 2048, where
// the 650 cycles between two tiles' products weigh most (accumulator complete, shared columns read, both CTAs told).  With
// that many products a cycle the power cap sets the clock: 1.32 to 1.45 GHz on random data against 1.75 to 1.8 on zeros.
// 32768 x 2048 x 2048 in 94 to 109 us, x 8192 in 365 us (3.0 PFLOP/s), relu^2 packed 32768 x 8192 x 2048 in 383 to 405 us, its
// derivative 411 to 440, dW 8192 x 2048 x 32768 in 396; in a run of seconds (1.28 GHz) 1.15 times that.  Four or three ring
// stages instead of five: NN x 8192 433 and 524 us against 411.
//
// Every mbarrier wait is bounded as in gemm_tcgen05_2cta.cu: on expiry a code goes to `status`, all roles leave, the CTAs
// meet, tensor memory is released and the kernel returns.
#include <cuda.h>

#include <atomic>

#include "fp8_format.cuh"
#include "fp8_steps.cuh"
#include "tensormap_cache.cuh"

namespace {

constexpr int TM = 128;                        // rows of C per CTA; the pair covers 256
constexpr int TN = 256;                        // columns of C per pair
constexpr int TK = 128;                        // contraction elements (bytes) per ring stage: one scale block
constexpr int STAGES = 5;
constexpr int OP_BYTES = 128 * 128;            // one operand tile of one CTA
constexpr int STAGE_BYTES = 2 * OP_BYTES;
constexpr int OUT_BYTES = TM * 128;            // 128 rows x 64 bf16, or x 128 packed bytes
constexpr int SF_STAGES = 4;
constexpr int SF_GROUP = 4;                    // scale blocks per set
constexpr int SF_BYTES = 512 * 3;              // 128 rows of A, 256 of B, four bytes each
constexpr int WARP_TMA = 0, WARP_MMA = 1, WARP_SCALE = 2, WARP_EPI = 3;
constexpr int EPI_GROUPS = 2;                  // each drains 128 columns of the tile
constexpr int NUM_THREADS = 32 * (WARP_EPI + 4 * EPI_GROUPS);
constexpr int TMEM_COLS = 512, ACC1_COL = 192, SF_COL = 448, SF_COLS = 16, SF_B_OFFSET = 8;
constexpr unsigned long long WAIT_NS = 4000000000ull;

enum Epilogue { EPI_STORE = 0, EPI_RESIDUAL = 1, EPI_RELU_SQ = 2, EPI_RELU_SQ_GRAD = 3, EPI_PARTIAL = 4 };

struct Barriers {
  uint64_t full[STAGES];         // leader: both CTAs' operand loads have landed
  uint64_t empty[STAGES];        // every CTA: the products that read the stage are done
  uint64_t sf_full[SF_STAGES];   // leader: both CTAs' scale warps have written the set
  uint64_t sf_empty[SF_STAGES];  // every CTA: the products that use the set are done
  uint64_t acc_full[2];          // every CTA: accumulator complete
  uint64_t acc_free;             // leader: the shared columns of the tile, and all of the tile before, have been read
  uint64_t in_full[EPI_GROUPS];  // every CTA: the tile that the epilogue reads (kept activation) has landed in its staging buffer
  uint32_t tmem_base;
  int abort_flag;
  uint32_t block_max[EPI_GROUPS][2][4];   // epilogue: maxima of a group's four warps, two tiles in flight
};

constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 2 * OUT_BYTES + SF_STAGES * SF_BYTES + 512 + 1024;

struct Args {
  int M, N;
  const uint8_t* a_exp;
  const uint8_t* b_exp;
  int a_rows;                    // 1 or 128
  long long a_ld;                // a_rows = 1: exponents of one column block
  int a_sm, a_sk, b_sn, b_sk;    // strides of the tile exponents along M / N and along the contraction
  bf16* c;
  const bf16* residual;
  long long ldc, ldr;
  int direct;                    // rows of C or of the residual do not start on 16 bytes: no TMA for either
  const uint8_t* h_exp;          // exponents of the kept activation, packed like the result
  uint8_t* q_exp;
  long long q_ldv, q_lde;        // leading dimensions of the packed result (and of h)
  int* status;
};
// One product, or two of the same kind in one launch: their tiles follow one another, so the second fills the SMs that the
// first's last round leaves idle (the two weight gradients of a feed-forward half: 2 x 256 tiles of 74 at a time in 7 rounds
// instead of 2 x 4).
struct alignas(64) Problem {
  CUtensorMap a, b, out, in;
  Args g;
  int tiles_n, tiles, num_kb;
  int splits, kb_split, rows_split;  // EPI_PARTIAL: slices of the contraction, blocks of a slice, rows of a slice in the workspace
};
template <int COUNT>
struct Problems {
  Problem p[COUNT];
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t map_to_cta(uint32_t addr, uint32_t rank) {
  uint32_t out;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(addr), "r"(rank));
  return out;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
// Arrive on an mbarrier of either CTA of the pair.  At CTA scope: what is announced is read by the tensor core (shared memory
// of the writer's own CTA, behind a proxy fence) or has left tensor memory.  A release at cluster scope waits for the
// thread's earlier stores all the way and costs 1650 cycles between two tiles' products (32768 x 2048 x 8192: 405 -> 490 us).
__device__ __forceinline__ void mbar_arrive_at(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t ok;
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "elect.sync _|p, 0xffffffff;\n"
      "selp.b32 %0, 1, 0, p;\n"
      "}\n"
      : "=r"(ok));
  return ok != 0;
}
// What these barriers announce is read by the tensor core and the copy engine, or lies in tensor memory: an acquire at
// cluster scope would only slow the issuing warp (NN 32768 x 2048 x 8192: 387 against 381 us).
__device__ __forceinline__ bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      "selp.b32 %0, 1, 0, p;\n"
      "}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ unsigned long long globaltimer_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, Barriers* bars, int* status, int code) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long deadline = globaltimer_ns() + WAIT_NS;
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 0x3ff) == 0) {
      if (*reinterpret_cast<volatile int*>(&bars->abort_flag)) return false;
      if (globaltimer_ns() > deadline) break;
    }
  }
  *reinterpret_cast<volatile int*>(&bars->abort_flag) = 1;
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(map_to_cta(smem_u32(&bars->abort_flag), cluster_ctarank() ^ 1u)), "r"(1)
               : "memory");
  if (status) atomicCAS(status, 0, code);
  return false;
}
// the same answer in every lane of a warp whose lanes all wait
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, Barriers* bars, int* status, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, bars, status, code));
}
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar_cluster_addr, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar_cluster_addr), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
               ::"l"(map), "r"(src), "r"(x), "r"(y)
               : "memory");
}
// operand tile: 128 rows of 128 bytes, 128-byte swizzle, 8-row groups 1024 bytes apart (either direction)
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// scale set: 32 rows of 16 bytes, no swizzle, 8-row groups 128 bytes apart
__device__ __forceinline__ uint64_t scale_desc(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)1 << 16 | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}
__device__ __forceinline__ void umma_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa,
                                          uint32_t sfb, uint32_t acc) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %6, 0;\n"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n"
      "}\n"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
      ::"r"(smem_u32(bar)), "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// Waits for the loads into v.  The empty statements make every later use of v depend on something behind the wait: without
// them the compiler may copy a destination register before its value has arrived.
template <int COUNT>
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&v)[COUNT]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < COUNT; ++i) asm volatile("" : "+r"(v[i]));
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// barrier of a group; true if `ok` holds in all its threads
__device__ __forceinline__ bool epi_all(int group, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.b32 p, %1, 0;\n"
      "barrier.cta.red.and.pred q, %2, 128, p;\n"
      "selp.b32 %0, 1, 0, q;\n"
      "}\n"
      : "=r"(r)
      : "r"((uint32_t)ok), "r"(1 + group)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void epi_sync(int group) { asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory"); }
// a tile of 128 rows by 128 bytes into a staging buffer, once the store out of that buffer has been read
__device__ __forceinline__ void fetch_input(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  mbar_expect_tx(bar, OUT_BYTES);
  tma_load_2d(dst, map, bar, x, y);
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_shared16(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

template <bool A_MN, bool B_MN, int EPI, int Q_ROWS, int COUNT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(NUM_THREADS, 1)
gemm_fp8_kernel(const __grid_constant__ Problems<COUNT> all) {
  extern __shared__ unsigned char smem_dyn[];
  const uint32_t raw = smem_u32(smem_dyn);
  const uint32_t base = (raw + 1023u) & ~1023u;
  const uint32_t out_stage = base + STAGES * STAGE_BYTES;
  const uint32_t sf_stage = out_stage + 2 * OUT_BYTES;
  Barriers* bars = reinterpret_cast<Barriers*>(smem_dyn + (sf_stage - raw) + SF_STAGES * SF_BYTES);
  static_assert(sizeof(Barriers) <= 512, "room for the barriers");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();            // 0 = leader
  const int pair = (int)blockIdx.x >> 1, n_pairs = (int)gridDim.x >> 1;
  constexpr bool SPLIT = EPI == EPI_PARTIAL;
  const int tiles0 = all.p[0].tiles * (SPLIT ? all.p[0].splits : 1);
  const int num_tiles = tiles0 + (COUNT > 1 ? all.p[COUNT - 1].tiles * (SPLIT ? all.p[COUNT - 1].splits : 1) : 0);
  int* const status = all.p[0].g.status;
  // the problem of a tile, its first row, its first column and (split: tile = slice * tiles + tile) its blocks of the contraction
  const auto locate = [&](int tile, int& m0, int& n0, int& kb0, int& num_kb) -> const Problem& {
    const bool second = COUNT > 1 && tile >= tiles0;
    const Problem& p = second ? all.p[COUNT - 1] : all.p[0];
    if (second) tile -= tiles0;
    kb0 = 0;
    num_kb = p.num_kb;
    if (SPLIT) {
      kb0 = tile / p.tiles * p.kb_split;
      num_kb = min(p.kb_split, p.num_kb - kb0);
      tile %= p.tiles;
    }
    // eight rows of tiles at a time, column by column: what runs at once shares its operands in L2 (2902 -> 2870 us for a
    // feed-forward half of 32768 x 2048 under the power cap)
    const int band = tile / (8 * p.tiles_n), rest = tile - band * (8 * p.tiles_n);
    const int height = min(8, p.tiles / p.tiles_n - band * 8);
    m0 = (band * 8 + rest % height) * (2 * TM) + (int)rank * TM;
    n0 = rest / height * TN;
    return p;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&bars->full[s], 1); mbar_init(&bars->empty[s], 1); }
    for (int s = 0; s < SF_STAGES; ++s) { mbar_init(&bars->sf_full[s], 2); mbar_init(&bars->sf_empty[s], 1); }
    mbar_init(&bars->acc_full[0], 1);
    mbar_init(&bars->acc_full[1], 1);
    for (int i = 0; i < EPI_GROUPS; ++i) mbar_init(&bars->in_full[i], 1);
    mbar_init(&bars->acc_free, 2 * 4 * EPI_GROUPS);
    bars->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == WARP_MMA) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem_base)),
                 "r"(TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;

  if (warp == WARP_TMA) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = pair; tile < num_tiles && ok; tile += n_pairs) {
        int m0, n0, kb0, num_kb;
        const Problem& p = locate(tile, m0, n0, kb0, num_kb);
        n0 += (int)rank * 128;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&bars->empty[stage], phase ^ 1, bars, status, 211)) { ok = false; break; }
          if (rank == 0) mbar_expect_tx(&bars->full[stage], 2 * STAGE_BYTES);
          const uint32_t full_leader = map_to_cta(smem_u32(&bars->full[stage]), 0);
          const uint32_t sa = base + stage * STAGE_BYTES, sb = sa + OP_BYTES;
          const int k0 = (kb0 + kb) * TK;
          tma_load_2d_pair(sa, &p.a, full_leader, A_MN ? m0 : k0, A_MN ? k0 : m0);
          tma_load_2d_pair(sb, &p.b, full_leader, B_MN ? n0 : k0, B_MN ? k0 : n0);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == WARP_MMA) {
    if (rank == 0) {           // the whole warp runs the loop, one elected thread issues: operands stay in uniform registers
      // kind::mxf8f6f4: A and B e4m3 (0), E8M0 scales (bit 23), directions, N = 256, M = 256 across the pair
      constexpr uint32_t idesc = ((A_MN ? 1u : 0u) << 15) | ((B_MN ? 1u : 0u) << 16) | ((uint32_t)(TN >> 3) << 17) | (1u << 23) |
                                 ((uint32_t)((2 * TM) >> 7) << 27);
      // 32 contraction elements further: 32 bytes along a K-major row, 32 rows of an MN-major tile
      constexpr uint32_t a_adv = (A_MN ? 32 * 128 : 32) >> 4, b_adv = (B_MN ? 32 * 128 : 32) >> 4;
      int stage = 0, sf = 0, local = 0;
      uint32_t phase = 0, sf_phase = 0;
      bool ok = true;
      for (int tile = pair; tile < num_tiles && ok; tile += n_pairs, ++local) {
        const uint32_t d_tmem = tmem_base + (local & 1) * ACC1_COL;
        int m0, n0, kb0, num_kb;
        locate(tile, m0, n0, kb0, num_kb);
        for (int kb = 0; kb < num_kb; ++kb) {
          const uint32_t sfa = tmem_base + SF_COL + sf * SF_COLS, sfb = sfa + SF_B_OFFSET;
          const uint32_t id = kb % SF_GROUP;
          if (id == 0) {       // (a tile's first set does not wait for the accumulator)
            if (!warp_wait(&bars->sf_full[sf], sf_phase, bars, status, 213)) { ok = false; break; }
            tc_fence_after();
            if (elect_one()) {
              const uint32_t src = sf_stage + sf * SF_BYTES;
              scales_to_tmem(sfa, scale_desc(src));
              scales_to_tmem(sfb, scale_desc(src + 512));
              scales_to_tmem(sfb + 4, scale_desc(src + 1024));
            }
            __syncwarp();
          }
          if (!warp_wait(&bars->full[stage], phase, bars, status, 214)) { ok = false; break; }
          if (kb == 0 && local > 0 && !warp_wait(&bars->acc_free, (local - 1) & 1, bars, status, 212)) { ok = false; break; }
          tc_fence_after();
          if (elect_one()) {
            const uint32_t sa = base + stage * STAGE_BYTES;
            const uint64_t adesc = operand_desc(sa), bdesc = operand_desc(sa + OP_BYTES);
            const uint32_t desc = idesc | (id << 4) | (id << 29);
#pragma unroll
            for (int k = 0; k < TK / 32; ++k)
              umma_pair(d_tmem, adesc + (uint64_t)(k * a_adv), bdesc + (uint64_t)(k * b_adv), desc, sfa, sfb, (kb | k) ? 1u : 0u);
            umma_commit_pair(&bars->empty[stage]);
            if (id == SF_GROUP - 1 || kb == num_kb - 1) umma_commit_pair(&bars->sf_empty[sf]);
            if (kb == num_kb - 1) umma_commit_pair(&bars->acc_full[local & 1]);
          }
          __syncwarp();
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
          if (id == SF_GROUP - 1 || kb == num_kb - 1)
            if (++sf == SF_STAGES) { sf = 0; sf_phase ^= 1; }
        }
      }
    }
  } else if (warp == WARP_SCALE) {
    // Sets of scales: word r of an operand holds the bytes of rows r (128 of A, 256 of B) for four blocks of the
    // contraction; word r goes to lane r % 32, column r / 32.
    const bool by_row = !A_MN && COUNT == 1 && all.p[0].g.a_rows == 1;
    int sf = 0;
    uint32_t sf_phase = 0;
    // lanes 0-3: A, 4-7 and 8-11: the two column blocks of B; blocks of one row: four rows a lane
    auto fetch = [&](int tile, int set, uint32_t& byte, uint32_t (&rows4)[4]) {
      int m0, n0, kb0, num_kb;
      const Problem& p = locate(tile, m0, n0, kb0, num_kb);
      const Args& g = p.g;
      const int which = lane >> 2, kb = kb0 + set * SF_GROUP + (lane & 3);
      byte = 0;
      if (kb < kb0 + num_kb) {
        if (which == 0 && !by_row && m0 < g.M) byte = __ldg(g.a_exp + (long long)(m0 >> 7) * g.a_sm + (long long)kb * g.a_sk);
        if ((which == 1 || which == 2) && n0 + (which - 1) * 128 < g.N)
          byte = __ldg(g.b_exp + (long long)((n0 >> 7) + which - 1) * g.b_sn + (long long)kb * g.b_sk);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        rows4[i] = 0;
        if (by_row && set * SF_GROUP + i < num_kb && m0 + 4 * lane < g.a_ld)
          rows4[i] = __ldg(reinterpret_cast<const uint32_t*>(g.a_exp + (long long)(kb0 + set * SF_GROUP + i) * g.a_ld + m0 + 4 * lane));
      }
      return (num_kb + SF_GROUP - 1) / SF_GROUP;
    };
    uint32_t next_byte, next_rows[4];
    int tile = pair, set = 0, sets = 0;
    if (tile < num_tiles) sets = fetch(tile, 0, next_byte, next_rows);
    while (tile < num_tiles) {
      uint32_t byte = next_byte, rows4[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) rows4[i] = next_rows[i];
      if (++set == sets) { set = 0; tile += n_pairs; }
      if (tile < num_tiles) sets = fetch(tile, set, next_byte, next_rows);      // one set ahead of the one that is written
      if (!warp_wait(&bars->sf_empty[sf], sf_phase ^ 1, bars, status, 215)) break;
      byte <<= 8 * (lane & 3);
      byte |= __shfl_xor_sync(0xffffffffu, byte, 1);
      byte |= __shfl_xor_sync(0xffffffffu, byte, 2);
      const uint32_t wa = __shfl_sync(0xffffffffu, byte, 0), wb0 = __shfl_sync(0xffffffffu, byte, 4),
                     wb1 = __shfl_sync(0xffffffffu, byte, 8);
      const uint32_t dst = sf_stage + sf * SF_BYTES;
      if (by_row) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {      // word of row 4 * lane + i: byte i of the four blocks
          const uint32_t lo = __byte_perm(rows4[0], rows4[1], i | ((4 + i) << 4));
          const uint32_t hi = __byte_perm(rows4[2], rows4[3], i | ((4 + i) << 4));
          const int r = 4 * lane + i;
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(dst + (r & 31) * 16 + (r >> 5) * 4), "r"(__byte_perm(lo, hi, 0x5410))
                       : "memory");
        }
      } else {
        st_shared16(dst + lane * 16, make_uint4(wa, wa, wa, wa));
      }
      st_shared16(dst + 512 + lane * 16, make_uint4(wb0, wb0, wb0, wb0));
      st_shared16(dst + 1024 + lane * 16, make_uint4(wb1, wb1, wb1, wb1));
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive_at(map_to_cta(smem_u32(&bars->sf_full[sf]), 0));
      if (++sf == SF_STAGES) { sf = 0; sf_phase ^= 1; }
    }
  } else {
    const int quarter = warp & 3;                 // tensor-memory lanes [32q, 32q + 32)
    const int row = quarter * 32 + lane;          // row of this CTA's 128 owned by this thread
    const int group = (warp - WARP_EPI) >> 2;     // columns [128 * group, 128 * group + 128) of the tile
    const bool elected = threadIdx.x == 32 * (WARP_EPI + 4 * group);
    const uint32_t stage_addr = out_stage + group * OUT_BYTES;
    const uint32_t free_leader = map_to_cta(smem_u32(&bars->acc_free), 0);
    int local = 0;
    for (int tile = pair; tile < num_tiles; tile += n_pairs, ++local) {
      int m0, gn0, kb0, num_kb;
      const Problem& p = locate(tile, m0, gn0, kb0, num_kb);
      gn0 += group * 128;
      const Args& g = p.g;
      const int M = g.M, N = g.N;
      const int gm = m0 + row;
      const int acc = local & 1;
      const bool shared_columns = group != acc;    // accumulator 0 shares its last 64 columns, accumulator 1 its first
      // What the epilogue reads - the kept activation, or the first half of the residual - is fetched while the products run
      // and replaced in place by the result.
      const bool residual_by_tma = EPI == EPI_RESIDUAL && !g.direct;
      if ((EPI == EPI_RELU_SQ_GRAD || residual_by_tma) && elected)
        fetch_input(stage_addr, &p.in, &bars->in_full[group], gn0 + (EPI == EPI_RESIDUAL && acc == 0 ? 64 : 0), m0);
      if (!epi_all(group, mbar_wait(&bars->acc_full[acc], (local >> 1) & 1, bars, status, 216))) break;
      tc_fence_after();
      // a group without shared columns arrives at once: it has read all of the tile before
      if (!shared_columns && lane == 0) mbar_arrive_at(free_leader);
      const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * ACC1_COL + group * 128;
      if constexpr (EPI == EPI_STORE || EPI == EPI_RESIDUAL) {
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
          const int chunk = acc == 0 ? 1 - i : i;      // the columns shared with the other accumulator first
          const int c0 = gn0 + chunk * 64;
          uint32_t v[64];
          tmem_ld32(t_row + chunk * 64, v);
          tmem_ld32(t_row + chunk * 64 + 32, v + 32);
          if (residual_by_tma && i == 1 && elected) fetch_input(stage_addr, &p.in, &bars->in_full[group], c0, m0);
          tmem_wait_ld(v);
          if (i == 0 && shared_columns) {
            tc_fence_before();
            if (lane == 0) mbar_arrive_at(free_leader);
          }
          if (residual_by_tma) {
            if (!epi_all(group, mbar_wait(&bars->in_full[group], i, bars, status, 217))) break;
          } else {
            if (elected) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            epi_sync(group);
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t at = stage_addr + row * 128 + ((j ^ (row & 7)) << 4);
            float f[8];
            if (residual_by_tma) {
              unpack8(ld_shared16(at), f);
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                f[e] = EPI == EPI_RESIDUAL && gm < M && c0 + j * 8 + e < N
                           ? __bfloat162float(g.residual[(long long)gm * g.ldr + c0 + j * 8 + e]) : 0.f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] += __uint_as_float(v[j * 8 + e]);
            st_shared16(at, pack8(f));
          }
          if (!g.direct) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            epi_sync(group);
            if (elected && m0 < M && c0 < N) {
              tma_store_2d(&p.out, stage_addr, c0, m0);
              asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
          } else {                                                // unaligned rows: copied out value by value
            epi_sync(group);
            for (int r = quarter; r < TM && m0 + r < M; r += 4)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int col = lane + h * 32;
                uint16_t val;
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(val)
                             : "r"(stage_addr + r * 128 + (((col >> 3) ^ (r & 7)) << 4) + (col & 7) * 2)
                             : "memory");
                if (c0 + col < N) reinterpret_cast<uint16_t*>(g.c)[(long long)(m0 + r) * g.ldc + c0 + col] = val;
              }
          }
        }
      } else if constexpr (EPI == EPI_PARTIAL) {      // fp32 rows of this slice, 32 columns at a time
        const int out_row = kb0 / p.kb_split * p.rows_split + m0;
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
          const int chunk = acc == 0 ? 1 - i : i;      // the columns shared with the other accumulator first
          uint32_t v[64];
          tmem_ld32(t_row + chunk * 64, v);
          tmem_ld32(t_row + chunk * 64 + 32, v + 32);
          tmem_wait_ld(v);
          if (i == 0 && shared_columns) {
            tc_fence_before();
            if (lane == 0) mbar_arrive_at(free_leader);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int c0 = gn0 + chunk * 64 + h * 32;
            if (elected) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            epi_sync(group);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const uint32_t* w = v + h * 32 + j * 4;
              st_shared16(stage_addr + row * 128 + ((j ^ (row & 7)) << 4), make_uint4(w[0], w[1], w[2], w[3]));
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            epi_sync(group);
            if (elected && m0 < M && c0 < N) {
              tma_store_2d(&p.out, stage_addr, c0, out_row);
              asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
          }
        }
      } else {
        const int nb = gn0 >> 7;
        const bool partial = m0 + TM > M || gn0 + 128 > N;
        float c_in = 1.f, c_out = 0.f;             // 2 sqrt(q 2^s) = c_out sqrt(c_in q)
        if (EPI == EPI_RELU_SQ_GRAD && gm < M && gn0 < N) {
          const uint32_t he = Q_ROWS == 1 ? g.h_exp[(long long)nb * g.q_lde + gm] : g.h_exp[(long long)(m0 >> 7) * g.q_lde + nb];
          const int s = (int)he - 127;
          c_in = s & 1 ? 2.f : 1.f;
          c_out = __uint_as_float((uint32_t)((s >> 1) + 1 + 127) << 23);
        }
        uint32_t v[128];
#pragma unroll
        for (int j = 0; j < 4; ++j) tmem_ld32(t_row + j * 32, v + j * 32);
        tmem_wait_ld(v);
        if (shared_columns) {
          tc_fence_before();
          if (lane == 0) mbar_arrive_at(free_leader);
        }
        if (EPI == EPI_RELU_SQ_GRAD && !epi_all(group, mbar_wait(&bars->in_full[group], local & 1, bars, status, 217))) break;
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float h[16];
          if (EPI == EPI_RELU_SQ_GRAD) {
            const uint4 q = ld_shared16(stage_addr + row * 128 + ((j ^ (row & 7)) << 4));
            fp8_unpack4(q.x, h); fp8_unpack4(q.y, h + 4); fp8_unpack4(q.z, h + 8); fp8_unpack4(q.w, h + 12);
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float x = __uint_as_float(v[j * 16 + e]);
            if (EPI == EPI_RELU_SQ) {
              x = x < 0.f ? 0.f : x;             // a NaN stays one
              x *= x;
            } else {
              x *= c_out * sqrtf(h[e] * c_in);
            }
            v[j * 16 + e] = __float_as_uint(x);
          }
        }
        if (partial) {
#pragma unroll
          for (int e = 0; e < 128; ++e)
            if (gm >= M || gn0 + e >= N) v[e] = 0u;
        }
#pragma unroll
        for (int e = 0; e < 128; ++e) top = max(top, v[e] & 0x7fffffffu);
        if (Q_ROWS == 128) {
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
          if (lane == 0) bars->block_max[group][acc][quarter] = top;
        }
        if (EPI == EPI_RELU_SQ && elected) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        epi_sync(group);
        if (Q_ROWS == 128) {
          const uint32_t* b = bars->block_max[group][acc];
          top = max(max(b[0], b[1]), max(b[2], b[3]));
        }
        const uint32_t e = fp8_block_exponent(top);
        const float s = fp8_inverse_scale(e == 255u ? 127u : e);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t w[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const uint32_t* p = v + j * 16 + t * 4;
            w[t] = fp8_pack4(__uint_as_float(p[0]) * s, __uint_as_float(p[1]) * s, __uint_as_float(p[2]) * s, __uint_as_float(p[3]) * s);
            if (e == 255u) w[t] = 0x7f7f7f7fu;
          }
          st_shared16(stage_addr + row * 128 + ((j ^ (row & 7)) << 4), make_uint4(w[0], w[1], w[2], w[3]));
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        epi_sync(group);
        if (m0 < M && gn0 < N) {
          if (elected) {
            tma_store_2d(&p.out, stage_addr, gn0, m0);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            if (Q_ROWS == 128) g.q_exp[(long long)(m0 >> 7) * g.q_lde + nb] = (uint8_t)e;
          }
          if (Q_ROWS == 1 && gm < M) g.q_exp[(long long)nb * g.q_lde + gm] = (uint8_t)e;
        }
      }
    }
    if (elected) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }

  __syncwarp();
  if (warp == WARP_TMA && *reinterpret_cast<volatile int*>(&bars->abort_flag)) {
    const unsigned long long until = globaltimer_ns() + 1000000ull;      // loads in flight land before the memory is given up
    while (globaltimer_ns() < until) {}
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();            // neither CTA leaves (or frees tensor memory) while the other may still signal or read it
  if (warp == WARP_MMA) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS));
  }
}

// Tensor map over [rows, cols] of 1- or 2-byte elements, box of 128 rows x 128 bytes, 128-byte swizzle.
int encode(CUtensorMap* map, CUtensorMapDataType type, int elem, const void* ptr, long long rows, long long cols, long long ld) {
  if (((uintptr_t)ptr & 15) || (ld * elem) % 16) return RWKV_ERR_BAD_ALIGNMENT;
  rwkv_tmap::EncodeTiledFn enc = rwkv_tmap::get_encode();
  if (!enc) return RWKV_ERR_NOT_INITIALISED;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)(ld * elem)};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / elem), 128}, estr[2] = {1, 1};
  CUresult r = CUDA_SUCCESS;
  for (int attempt = 0; attempt < 2; ++attempt) {
    r = enc(map, type, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_ERROR_INVALID_CONTEXT) break;
    cudaFree(nullptr);       // a thread without CUDA work so far (an autograd worker): binds the device's context
  }
  return r == CUDA_SUCCESS ? RWKV_OK : RWKV_ERR_CUDA_BASE + 900 + (int)r;
}

template <bool A_MN, bool B_MN, int EPI, int Q_ROWS, int COUNT = 1>
int launch(const Problems<COUNT>& all, cudaStream_t st) {
  auto kern = gemm_fp8_kernel<A_MN, B_MN, EPI, Q_ROWS, COUNT>;
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return RWKV_ERR_CUDA_BASE + (int)e;
  static std::atomic<unsigned long long> configured{0};          // devices whose copy of the kernel may use the memory
  const unsigned long long bit = 1ull << (dev & 63);
  if (!(configured.load() & bit)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
    if (e != cudaSuccess) return RWKV_ERR_CUDA_BASE + (int)e;
    configured.fetch_or(bit);
  }
  long long tiles = 0;
  for (int i = 0; i < COUNT; ++i) tiles += (long long)all.p[i].tiles * all.p[i].splits;
  const int pairs = tiles < sms / 2 ? (int)tiles : sms / 2;
  kern<<<2 * pairs, NUM_THREADS, SMEM_BYTES, st>>>(all);
  return rwkv_launch_status();
}

inline int up(int n, int m) { return (n + m - 1) / m * m; }

// Slices of the contraction: few tiles and a long contraction leave most SM pairs idle, so the contraction is cut into
// slices of at least eight blocks whose fp32 sums a second kernel adds in a fixed order.  A block takes 0.3 us, the second
// kernel and its traffic 4 to 6: slices are used where they save a tile 24 blocks or more, on at most half the pairs
// (M x N x K, in one piece and in slices: 222 x 64 x 23302 61.7 and 12.7 us, 1024 x 1024 x 32768 78.1 and 35.2,
// 2304 x 1024 x 8192 25.3 and 22.9; below the rule 2048 x 1024 x 4096 16.0 and 17.2, 512 x 2048 x 2048 10.6 and 13.1).
int splits_for(int M, int N, int K) {
  const long long tiles = (long long)(up(M, 2 * TM) / (2 * TM)) * (up(N, TN) / TN);
  const int kb = up(K, TK) / TK;
  if (tiles > 37 || kb < 32) return 1;
  const int s = (int)(74 / tiles) < kb / 8 ? (int)(74 / tiles) : kb / 8;
  const int per = up((kb + s - 1) / s, SF_GROUP);            // whole sets of scales
  return kb - per >= 24 ? (kb + per - 1) / per : 1;
}
inline int kb_of_slice(int K, int splits) { return up((up(K, TK) / TK + splits - 1) / splits, SF_GROUP); }

// c = (residual +) the sum of the slices' rows
__global__ void __launch_bounds__(256)
fp8_sum_slices_kernel(const float* __restrict__ ws, int splits, long long slice, int ldw, int M, int N, const bf16* __restrict__ residual,
                      long long ldr, bf16* __restrict__ c, long long ldc, int vec) {
  const int quads = (N + 3) / 4;
  const long long total = (long long)M * quads;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const int m = (int)(i / quads), n = (int)(i % quads) * 4;
    float f[4] = {0.f, 0.f, 0.f, 0.f};
    const float* p = ws + (long long)m * ldw + n;
    for (int s = 0; s < splits; ++s) {
      const float4 v = *reinterpret_cast<const float4*>(p + s * slice);
      f[0] += v.x; f[1] += v.y; f[2] += v.z; f[3] += v.w;
    }
    if (vec) {
      if (residual) {
        const uint2 r = *reinterpret_cast<const uint2*>(residual + m * ldr + n);
        f[0] += bf16_lo(r.x); f[1] += bf16_hi(r.x); f[2] += bf16_lo(r.y); f[3] += bf16_hi(r.y);
      }
      *reinterpret_cast<uint2*>(c + m * ldc + n) = make_uint2(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < N) c[m * ldc + n + e] = __float2bfloat16_rn(f[e] + (residual ? __bfloat162float(residual[m * ldr + n + e]) : 0.f));
    }
  }
}
int sum_slices(const Fp8Step& s, int splits, cudaStream_t st) {
  const int ldw = up(s.N, 4);
  const long long total = (long long)s.M * ((s.N + 3) / 4), ctas = (total + 255) / 256;
  const int vec = !(s.N % 4) && !((uintptr_t)s.c & 7) && !(s.ldc % 4) && !((uintptr_t)s.residual & 7) && !(s.ldr % 4);
  fp8_sum_slices_kernel<<<(int)(ctas < 148 * 16 ? ctas : 148 * 16), 256, 0, st>>>(
      (const float*)s.workspace, splits, (long long)up(s.M, TM) * ldw, ldw, s.M, s.N, (const bf16*)s.residual, s.ldr, (bf16*)s.c,
      s.ldc, vec);
  return rwkv_launch_status();
}

// Checks a record and fills in a problem; with a workspace the result goes there in slices.
int describe(const Fp8Step& s, Problem& p) {
  const int M = s.M, N = s.N, K = s.K, a_mn = s.a_mn, b_mn = s.b_mn, epilogue = s.epilogue, q_rows = s.q_rows;
  if (M <= 0 || N <= 0 || K <= 0 || M > 0x7ffffe00 || N > 0x7ffffe00 || K > 0x7ffffe00) return RWKV_ERR_BAD_SHAPE;
  if (!(s.a_rows == 128 || (s.a_rows == 1 && !a_mn)) || epilogue < 0 || epilogue > 3) return RWKV_ERR_BAD_SHAPE;
  if (epilogue <= 1 ? (!s.c || s.ldc < N || (epilogue == 1 && (!s.residual || s.ldr < N)))
                    : (!s.q_val || !s.q_exp || !(q_rows == 1 || q_rows == 128) ||
                       (epilogue == 3 && (!s.h_val || !s.h_exp || ((uintptr_t)s.h_val & 15)))))
    return RWKV_ERR_BAD_SHAPE;
  const CUtensorMapDataType u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8, b16 = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  int r = a_mn ? encode(&p.a, u8, 1, s.a_val, K, M, up(M, 16)) : encode(&p.a, u8, 1, s.a_val, M, K, up(K, 16));
  if (r) return r;
  r = b_mn ? encode(&p.b, u8, 1, s.b_val, K, N, up(N, 16)) : encode(&p.b, u8, 1, s.b_val, N, K, up(K, 16));
  if (r) return r;
  const int mb_n = up(M, 128) / 128, nb_n = up(N, 128) / 128, kb_n = up(K, 128) / 128;
  const long long tiles = (long long)(up(M, 2 * TM) / (2 * TM)) * (up(N, TN) / TN);
  if (tiles > 0x1fffffff) return RWKV_ERR_TOO_LARGE;
  p.tiles = (int)tiles; p.tiles_n = up(N, TN) / TN; p.num_kb = kb_n;
  Args& g = p.g;
  g = {};
  g.M = M; g.N = N;
  g.a_exp = (const uint8_t*)s.a_exp; g.b_exp = (const uint8_t*)s.b_exp;
  g.a_rows = s.a_rows;
  g.a_ld = up(M, 16);
  g.a_sm = a_mn ? 1 : kb_n; g.a_sk = a_mn ? mb_n : 1;
  g.b_sn = b_mn ? 1 : kb_n; g.b_sk = b_mn ? nb_n : 1;
  g.c = (bf16*)s.c; g.residual = (const bf16*)s.residual; g.ldc = s.ldc; g.ldr = s.ldr;
  g.h_exp = (const uint8_t*)s.h_exp; g.q_exp = (uint8_t*)s.q_exp;
  g.q_ldv = up(N, 16);
  g.q_lde = q_rows == 1 ? up(M, 16) : nb_n;
  g.status = (int*)s.status;
  p.out = p.in = p.a;                  // maps that the epilogue does not use are never read
  p.splits = 1; p.kb_split = kb_n; p.rows_split = up(M, TM);
  if (epilogue <= 1 && s.workspace) {
    p.splits = splits_for(M, N, K);
    p.kb_split = kb_of_slice(K, p.splits);
    r = encode(&p.out, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, s.workspace, (long long)p.splits * p.rows_split, N, up(N, 4));
  } else if (epilogue <= 1) {
    g.direct = ((uintptr_t)s.c & 15) || (s.ldc & 7) || (epilogue == 1 && (((uintptr_t)s.residual & 15) || (s.ldr & 7)));
    if (!g.direct) r = encode(&p.out, b16, 2, s.c, M, N, s.ldc);
    if (!r && epilogue == 1 && !g.direct) r = encode(&p.in, b16, 2, s.residual, M, N, s.ldr);
  } else {
    r = encode(&p.out, u8, 1, s.q_val, M, N, g.q_ldv);
    if (!r && epilogue == 3) r = encode(&p.in, u8, 1, s.h_val, M, N, g.q_ldv);
  }
  return r;
}

}  // namespace

// C[M,N] = op(A) op(B) of packed operands (fp8_format.cuh).
//   a_mn = 0: A is [M,K], a_rows 1 or 128;  a_mn = 1: A is stored [K,M], a_rows 128
//   b_mn = 0: B is [N,K];  b_mn = 1: B is stored [K,N]; both in tiles
//   epilogue 0: c = bf16 result (row stride ldc);  1: c = result + residual (bf16, row stride ldr), NT only;
//            2: (q_val, q_exp) = packed relu(result)^2, NT only;  3: = packed result * 2 sqrt(h), NN only;
//            the packed result and h are [M,N] with blocks of q_rows rows
//   workspace (epilogues 0 and 1): rwkv_fp8_workspace(M, N, K) bytes, the contraction runs in slices; null: it does not
//   status: device int, set non-zero if a device-side wait expired
int rwkv_fp8_gemm(const Fp8Step& s, cudaStream_t st) {
  Problems<1> all;
  int r = describe(s, all.p[0]);
  if (r) return r;
  const bool a_mn = s.a_mn, b_mn = s.b_mn;
  if (s.workspace && s.epilogue <= 1) {
    if (a_mn && !b_mn) return RWKV_ERR_BAD_SHAPE;
    r = a_mn ? launch<true, true, EPI_PARTIAL, 0>(all, st)
             : b_mn ? launch<false, true, EPI_PARTIAL, 0>(all, st) : launch<false, false, EPI_PARTIAL, 0>(all, st);
    return r ? r : sum_slices(s, all.p[0].splits, st);
  }
  switch (s.epilogue) {
    case EPI_RELU_SQ:
      if (a_mn || b_mn) return RWKV_ERR_BAD_SHAPE;
      return s.q_rows == 1 ? launch<false, false, EPI_RELU_SQ, 1>(all, st) : launch<false, false, EPI_RELU_SQ, 128>(all, st);
    case EPI_RELU_SQ_GRAD:
      if (a_mn || !b_mn) return RWKV_ERR_BAD_SHAPE;
      return s.q_rows == 1 ? launch<false, true, EPI_RELU_SQ_GRAD, 1>(all, st) : launch<false, true, EPI_RELU_SQ_GRAD, 128>(all, st);
    case EPI_RESIDUAL:
      return a_mn || b_mn ? RWKV_ERR_BAD_SHAPE : launch<false, false, EPI_RESIDUAL, 0>(all, st);
    default:
      if (a_mn) return b_mn ? launch<true, true, EPI_STORE, 0>(all, st) : RWKV_ERR_BAD_SHAPE;
      return b_mn ? launch<false, true, EPI_STORE, 0>(all, st) : launch<false, false, EPI_STORE, 0>(all, st);
  }
}

// Two products of the kind a^T b (a_mn = b_mn = 1, epilogue 0) in one launch.
int rwkv_fp8_gemm_two(const Fp8Step& s, const Fp8Step& t, cudaStream_t st) {
  if (!s.a_mn || !s.b_mn || s.epilogue || !t.a_mn || !t.b_mn || t.epilogue) return RWKV_ERR_BAD_SHAPE;
  Problems<2> all;
  int r = describe(s, all.p[0]);
  if (!r) r = describe(t, all.p[1]);
  if (r || !s.workspace != !t.workspace) return r ? r : RWKV_ERR_BAD_SHAPE;
  if (!s.workspace) return launch<true, true, EPI_STORE, 0, 2>(all, st);
  r = launch<true, true, EPI_PARTIAL, 0, 2>(all, st);
  if (!r) r = sum_slices(s, all.p[0].splits, st);
  return r ? r : sum_slices(t, all.p[1].splits, st);
}

// Bytes of workspace that a product wants (0: none).  Depends on sizes only.
RWKV_EXPORT long long rwkv_fp8_workspace(int M, int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0 || M > 0x7ffffe00 || N > 0x7ffffe00 || K > 0x7ffffe00) return 0;
  const int splits = splits_for(M, N, K);
  return splits > 1 ? (long long)splits * up(M, TM) * up(N, 4) * 4 : 0;
}
