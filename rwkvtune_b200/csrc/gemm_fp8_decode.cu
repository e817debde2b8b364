// 8-bit product for few rows: y[M, N] = x[M, K] W[N, K]^T with M <= 128 and W packed in tiles (fp8_format.cuh).
//
// Bound by streaming W once, one byte a weight, and below a few megabytes by latency.  As in gemm_decode_tcgen05.cu the
// weight tile is the 128-row operand A of the instruction and the tokens are its columns (M rounded up to 16), so the
// accumulator's lanes are full whatever M is; a column block of 128 weights is one CTA's and its contraction is cut over a
// cluster of S CTAs.  Token m of the sum belongs to CTA m % S: the others write their partial rows into its shared memory,
// and after one cluster barrier it adds them in a fixed order.  S depends on N and K alone, so a row's result does not
// depend on how many others there are (of these 128; larger batches run the pair kernel, with other sums).
//
// The tokens come either in bf16 - then each CTA packs its part of the contraction itself, row by row, into the
// shared-memory tiles the tensor core reads, which saves a launch and a round trip - or already packed, fetched by TMA in
// the same ring as the weights.  Packing in the kernel repeats the work in every CTA: it is used up to 16 rows (feed-forward
// half of 2048 channels, weights in L2, packed in the kernel and by a launch before it: 32 rows 14.7 and 13.4 us, 64 rows 20.0
// and 15.8; one row 12.0 and 14.2).
//
// Epilogues: store bf16, add a bf16 residual, or relu(y)^2 packed again: a CTA owns exactly one block of 128 columns of
// every token, so a block's scale is a maximum over one warp.
//
// A launch may be chained to its predecessor (programmatic dependent launch): it requests its first weight tiles, which no
// kernel of the chain writes, before it waits for the predecessor's results.  The workers' wait stands behind the CTA's
// barrier for that: in front of it, it held back the weight stream too (feed-forward half of one row, chained, weights from
// HBM: 12.9 us, behind it 11.9; 8 rows 13.1 and 12.4).
//
// Back to back in a graph that cycles through more weights than L2 holds, as the blocks of a decode step do: 2048 -> 2048 for
// one row 7.4 us (4 MB: latency, 4700 cycles of it between the first instruction and the accumulator), the head 2048 -> 65536
// 25.9 us for one row (5.2 TB/s) and 30.5 with the packing launch for 64 (4.4 TB/s); a feed-forward half of 2048 channels 14.1
// us for one row (2.4 TB/s), 19.5 for 64.  The same half on one pair of weights, which then lies in L2: 12.4 and 16.1 us.
//
// Shared memory is at least 112 KB per CTA, so an SM holds at most two of these, and with 256 columns of tensor memory each
// they never wait for one another's allocation (CTAs of different clusters that did could wait in a circle).
#include <cuda.h>

#include <atomic>

#include "fp8_format.cuh"
#include "fp8_steps.cuh"
#include "tensormap_cache.cuh"

namespace {

constexpr int WORKERS = 8;                       // warps that pack the tokens and drain the accumulator
constexpr int WARP_TMA = WORKERS, WARP_MMA = WORKERS + 1;
constexpr int THREADS = 32 * (WORKERS + 2);
constexpr int W_BYTES = 128 * 128;
constexpr int MAX_STAGES = 8;
constexpr int MAX_GROUPS = 16;                   // sets of four scale blocks: 64 blocks of the contraction per CTA
// Tensor memory: accumulator in columns 0..127 (two in turn if mpad <= 64), then the scales: four columns per set of tokens
// and four per set and column block of weights, all of them resident.
constexpr int TMEM_COLS = 256, SF_COL = 128, MAX_SETS = (TMEM_COLS - SF_COL) / 4;
constexpr int SMEM_MIN = 112 * 1024, SMEM_MAX = 224 * 1024;
constexpr unsigned long long WAIT_NS = 2000000000ull;

struct Barriers {
  uint64_t full[MAX_STAGES], empty[MAX_STAGES];
  uint64_t x_ready[MAX_GROUPS];                  // tokens (or their scales) of a set are in shared memory
  uint64_t acc_full[2], acc_free[2];
  uint32_t tmem_base;
  int abort_flag;
};

struct Args {
  int M, N, K, mpad, stages;
  int tiles;                                     // column blocks of a CTA, one after another (S = 1)
  int split_log, m_log;                          // log2 of S, and of M rounded up to a power of two
  const uint8_t* w_exp;
  const bf16* x;                                 // null: packed tokens
  long long ldx;
  const uint8_t* x_exp;
  long long x_lde;
  bf16* c;
  const bf16* residual;
  long long ldc, ldr;
  int vec;                                       // rows of c and of the residual start on 8 bytes and N is a multiple of 4
  uint8_t *q_val, *q_exp;
  long long q_ldv, q_lde;
  int* status;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
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
  if (status) atomicCAS(status, 0, code);
  return false;
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ uint64_t scale_desc(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)1 << 16 | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}
__device__ __forceinline__ void umma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                     uint32_t acc) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %6, 0;\n"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n"
      "}\n"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, float* v) {
  uint32_t r[8];
  // one statement: a copy of a destination register must not move between the load and its wait
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n"
               "tcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
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
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

enum Epilogue { EPI_STORE = 0, EPI_RESIDUAL = 1, EPI_RELU_SQ = 2 };

// Tokens z, z + S, ... of a column block: sums the S partial rows, applies the epilogue and stores; one warp a token, four
// columns a lane.
template <int EPI>
__device__ __forceinline__ void finish(const Args& g, uint32_t part, int slab, int warp, int lane, int z, int slog, int own_tokens) {
  const int n = slab * 128 + lane * 4;
  for (int m = z + (warp << slog); m < g.M; m += WORKERS << slog) {
    float f[4] = {0.f, 0.f, 0.f, 0.f};
    for (int r = 0; r < 1 << slog; ++r) {
      float4 p;
      asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(p.x), "=f"(p.y), "=f"(p.z), "=f"(p.w)
                   : "r"(part + (r * own_tokens + (m >> slog)) * 512 + lane * 16) : "memory");
      f[0] += p.x; f[1] += p.y; f[2] += p.z; f[3] += p.w;
    }
    if (EPI == EPI_RELU_SQ) {
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[e] = f[e] < 0.f || n + e >= g.N ? 0.f : f[e];
        f[e] *= f[e];
        top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      const uint32_t e = fp8_block_exponent(top);
      const float s = fp8_inverse_scale(e == 255u ? 127u : e);
      if (n < g.q_ldv)
        *reinterpret_cast<uint32_t*>(g.q_val + (long long)m * g.q_ldv + n) =
            e == 255u ? 0x7f7f7f7fu : fp8_pack4(f[0] * s, f[1] * s, f[2] * s, f[3] * s);
      if (lane == 0) g.q_exp[(long long)slab * g.q_lde + m] = (uint8_t)e;
    } else if (g.vec) {
      if (n < g.N) {
        if (EPI == EPI_RESIDUAL) {
          const uint2 p = *reinterpret_cast<const uint2*>(g.residual + m * g.ldr + n);
          f[0] += bf16_lo(p.x); f[1] += bf16_hi(p.x); f[2] += bf16_lo(p.y); f[3] += bf16_hi(p.y);
        }
        *reinterpret_cast<uint2*>(g.c + m * g.ldc + n) = make_uint2(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]));
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < g.N)
          g.c[m * g.ldc + n + e] =
              __float2bfloat16_rn(f[e] + (EPI == EPI_RESIDUAL ? __bfloat162float(g.residual[m * g.ldr + n + e]) : 0.f));
    }
  }
}

// grid: (column blocks of 128 / tiles, S), clusters of (1, S, 1)
template <bool PACKED, int EPI>
__global__ void __launch_bounds__(THREADS, 2)
fp8_decode_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                  const __grid_constant__ Args g) {
  extern __shared__ unsigned char smem_dyn[];
  const uint32_t raw = smem_u32(smem_dyn);
  const uint32_t base = (raw + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slog = g.split_log, S = 1 << slog, z = (int)blockIdx.y;
  // column blocks of this CTA: tiles of them, the last CTA's may be fewer
  const int slab0 = (int)blockIdx.x * g.tiles, slabs = (g.N + 127) >> 7, tiles = min(g.tiles, slabs - slab0);
  const int accs = g.mpad <= 64 ? 2 : 1;          // accumulators in turn, mpad <= 64 columns apart
  // the first all_kb % S CTAs of a cluster take one block of the contraction more
  const int all_kb = (g.K + 127) >> 7, more = all_kb & (S - 1), kb0 = z * (all_kb >> slog) + min(z, more);
  const int nkb = (all_kb >> slog) + (z < more ? 1 : 0);
  const int groups = (nkb + 3) >> 2, x_bytes = g.mpad * 128;
  const int stage_bytes = W_BYTES + (PACKED ? x_bytes : 0);
  const uint32_t xs = base + g.stages * stage_bytes;                       // tokens packed here (not PACKED)
  const int max_kb = (all_kb + S - 1) >> slog;
  const int max_groups = (max_kb + 3) >> 2;
  const uint32_t sf = xs + (PACKED ? 0 : max_kb * x_bytes);                // 512 bytes per set: tokens, then weights by block
  const uint32_t part = sf + max_groups * (1 + g.tiles) * 512;             // [CTA][own token][128 columns] in fp32
  const int own_tokens = (g.mpad + S - 1) >> slog;
  Barriers* bars = reinterpret_cast<Barriers*>(smem_dyn + (part - raw) + own_tokens * S * 512);

  rwkv_chain_trigger();
  if (warp == WARP_TMA) {                        // a lane a barrier
    if (lane < MAX_STAGES) { mbar_init(&bars->full[lane], 1); mbar_init(&bars->empty[lane], 1); }
    if (lane < MAX_GROUPS) mbar_init(&bars->x_ready[lane], WORKERS);
    if (lane >= MAX_GROUPS && lane < MAX_GROUPS + 2) {
      mbar_init(&bars->acc_full[lane - MAX_GROUPS], 1);
      mbar_init(&bars->acc_free[lane - MAX_GROUPS], WORKERS);
    }
    if (lane == 31) bars->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // scales of the weights, one byte per block: requested before anything is waited for
  uint32_t w_scale = 0;
  const int w_sets = groups * tiles;                            // set i: column block i / groups, blocks of the contraction i % groups
  const auto weight_scale = [&](int i) {
    const int t = i / groups, kb = kb0 + (i - t * groups) * 4 + (lane & 3);
    return kb < all_kb ? (uint32_t)g.w_exp[(long long)(slab0 + t) * all_kb + kb] << (8 * (lane & 3)) : 0u;
  };
  if (warp < WORKERS && warp < w_sets) w_scale = weight_scale(warp);
  // tokens: eight threads a block of 128, DEEP blocks a thread in flight; the first set's are requested before anything else
  constexpr int DEEP = 4;
  const int sub = lane & 7;
  uint4 v[DEEP][2];
  const auto fetch = [&](int i, int u0) {
    const int units = (nkb - i * 4 < 4 ? nkb - i * 4 : 4) << g.m_log;
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
      const int u = u0 + d * WORKERS * 4, row = u & ((1 << g.m_log) - 1), col = (kb0 + i * 4 + (u >> g.m_log)) * 128 + sub * 16;
      v[d][0] = v[d][1] = make_uint4(0u, 0u, 0u, 0u);
      if (u < units && row < g.M) {
        const uint4* p = reinterpret_cast<const uint4*>(g.x + row * g.ldx + col);
        if (col < g.K) v[d][0] = p[0];
        if (col + 8 < g.K) v[d][1] = p[1];
      }
    }
  };
  __syncthreads();
  if (S > 1) cluster_arrive_relaxed();       // waited for before the first write to another CTA: it has started by then

  if (warp == WARP_TMA) {
    if (lane == 0) {
      const int all = nkb * tiles, first = all < g.stages ? all : g.stages;
      int kb = 0, n0 = slab0 * 128;
      for (int i = 0; i < first; ++i) {
        mbar_expect_tx(&bars->full[i], stage_bytes);
        tma_load_2d(base + i * stage_bytes, &map_w, &bars->full[i], (kb0 + kb) * 128, n0);
        if (++kb == nkb) { kb = 0; n0 += 128; }
      }
      rwkv_chain_wait();
      if (PACKED)
        for (int i = 0, k = 0; i < first; ++i) {
          tma_load_2d(base + i * stage_bytes + W_BYTES, &map_x, &bars->full[i], (kb0 + k) * 128, 0);
          if (++k == nkb) k = 0;
        }
      int s = 0;
      uint32_t phase = 0;
      for (int i = first; i < all; ++i) {
        if (!mbar_wait(&bars->empty[s], phase, bars, g.status, 221)) break;
        mbar_expect_tx(&bars->full[s], stage_bytes);
        tma_load_2d(base + s * stage_bytes, &map_w, &bars->full[s], (kb0 + kb) * 128, n0);
        if (PACKED) tma_load_2d(base + s * stage_bytes + W_BYTES, &map_x, &bars->full[s], (kb0 + kb) * 128, 0);
        if (++kb == nkb) { kb = 0; n0 += 128; }
        if (++s == g.stages) { s = 0; phase ^= 1; }
      }
    }
  } else if (warp == WARP_MMA) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem_base)),
                 "r"(TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    __syncwarp();
    tc_fence_before();
    asm volatile("bar.arrive 2, 288;" ::: "memory");           // the workers read the address before they read the accumulator
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&bars->tmem_base);
    // kind::mxf8f6f4: e4m3 operands, both K-major, E8M0 scales, M = 128, N = mpad
    const uint32_t idesc = ((uint32_t)(g.mpad >> 3) << 17) | (1u << 23) | (1u << 27);
    bool ok = true;
    int s = 0;
    uint32_t phase = 0;
    for (int t = 0; t < tiles && ok; ++t) {
      const int a = t & (accs - 1);
      const uint32_t d = tmem + a * 64;
      if (t >= accs) ok = __all_sync(0xffffffffu, mbar_wait(&bars->acc_free[a], ((t - accs) / accs) & 1, bars, g.status, 225));
      for (int i = 0; i < nkb && ok; ++i) {
        const uint32_t id = i & 3, set = i >> 2, sfb = tmem + SF_COL + set * 4, w_set = max_groups + t * groups + set;
        const uint32_t sfa = tmem + SF_COL + w_set * 4;
        if (id == 0 && t == 0) ok = __all_sync(0xffffffffu, mbar_wait(&bars->x_ready[set], 0, bars, g.status, 222));
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&bars->full[s], phase, bars, g.status, 223));
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          if (id == 0) {
            scales_to_tmem(sfa, scale_desc(sf + w_set * 512));
            if (t == 0) scales_to_tmem(sfb, scale_desc(sf + set * 512));
          }
          const uint32_t sa = base + s * stage_bytes, sb = PACKED ? sa + W_BYTES : xs + i * x_bytes;
          const uint64_t da = operand_desc(sa), db = operand_desc(sb);
          const uint32_t desc = idesc | (id << 4) | (id << 29);
#pragma unroll
          for (int k = 0; k < 4; ++k) umma(d, da + k * 2, db + k * 2, desc, sfa, sfb, (i | k) ? 1u : 0u);
          umma_commit(&bars->empty[s]);
          if (i == nkb - 1) umma_commit(&bars->acc_full[a]);
        }
        __syncwarp();
        if (++s == g.stages) { s = 0; phase ^= 1; }
      }
    }
  } else {
    if (!PACKED) {                               // behind the barrier: the other two warps do not wait for the predecessor
      rwkv_chain_wait();
      fetch(0, warp * 4 + (lane >> 3));
    }
    for (int i = warp; i < w_sets; i += WORKERS) {
      uint32_t w = i == warp ? w_scale : weight_scale(i);
      w |= __shfl_xor_sync(0xffffffffu, w, 1);
      w |= __shfl_xor_sync(0xffffffffu, w, 2);
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sf + (max_groups + i) * 512 + lane * 16), "r"(w) : "memory");
    }
    if (PACKED) {
      // ---- scales of the tokens: word of row r holds the bytes of four blocks
      rwkv_chain_wait();
      for (int u = threadIdx.x; u < groups << g.m_log; u += 32 * WORKERS) {
        const int i = u >> g.m_log, r = u & ((1 << g.m_log) - 1);
        if (r >= g.M) continue;
        uint32_t w = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b)
          if (i * 4 + b < nkb) w |= (uint32_t)g.x_exp[(long long)(kb0 + i * 4 + b) * g.x_lde + r] << (8 * b);
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(sf + i * 512 + (r & 31) * 16 + (r >> 5) * 4), "r"(w) : "memory");
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0)
        for (int i = 0; i < groups; ++i) mbar_arrive(&bars->x_ready[i]);
    } else {
      for (int i = 0; i < groups; ++i) {
        const int units = (nkb - i * 4 < 4 ? nkb - i * 4 : 4) << g.m_log;
        for (int u0 = warp * 4 + (lane >> 3); u0 - (lane >> 3) < units; u0 += WORKERS * 4 * DEEP) {
          if (i > 0 || u0 >= WORKERS * 4) fetch(i, u0);
#pragma unroll
          for (int d = 0; d < DEEP; ++d) {
            const int u = u0 + d * WORKERS * 4, row = u & ((1 << g.m_log) - 1), b = u >> g.m_log;
            float f[16];
            unpack8(v[d][0], f);
            unpack8(v[d][1], f + 8);
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 16; ++j) top = max(top, __float_as_uint(f[j]) & 0x7fffffffu);
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            if (u < units && row < g.M) {
              const uint32_t e = fp8_block_exponent(top);
              uint32_t q[4];
              const float s = fp8_inverse_scale(e == 255u ? 127u : e);
#pragma unroll
              for (int j = 0; j < 4; ++j)
                q[j] = e == 255u ? 0x7f7f7f7fu : fp8_pack4(f[4 * j] * s, f[4 * j + 1] * s, f[4 * j + 2] * s, f[4 * j + 3] * s);
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                           ::"r"(xs + (i * 4 + b) * x_bytes + row * 128 + ((sub ^ (row & 7)) << 4)), "r"(q[0]), "r"(q[1]), "r"(q[2]),
                             "r"(q[3])
                           : "memory");
              if (sub == 0)
                asm volatile("st.shared.u8 [%0], %1;" ::"r"(sf + i * 512 + (row & 31) * 16 + (row >> 5) * 4 + b), "r"(e)
                             : "memory");
            }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->x_ready[i]);
      }
    }
    asm volatile("bar.sync 2, 288;" ::: "memory");
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&bars->tmem_base);
    const int quarter = warp & 3;
    const uint32_t column = (quarter * 32 + lane) * 4;
    for (int t = 0; t < tiles; ++t) {
      // ---- partial rows to the CTAs that own the tokens (all mpad of them: rows beyond M are never read)
      const int a = t & (accs - 1);
      const bool ok = mbar_wait(&bars->acc_full[a], (t / accs) & 1, bars, g.status, 224);
      __syncwarp();
      tc_fence_after();
      if (S > 1) cluster_wait();                 // (S > 1: one column block)
#pragma unroll 1
      for (int m = (warp >> 2) * 8; m < g.mpad; m += 16) {
        float p[8];
        tmem_ld8(tmem + ((uint32_t)(quarter * 32) << 16) + a * 64 + m, p);
        if (S == 1) {
#pragma unroll
          for (int e = 0; e < 8; ++e) asm volatile("st.shared.f32 [%0], %1;" ::"r"(part + (m + e) * 512 + column), "f"(p[e]) : "memory");
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int at = z * own_tokens + ((m + e) >> slog);
            uint32_t dst;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(dst) : "r"(part + at * 512 + column), "r"((m + e) & (S - 1)));
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst), "f"(p[e]) : "memory");
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->acc_free[a]);
      if (S > 1) {
        cluster_arrive();
        cluster_wait();
      } else {
        asm volatile("bar.sync 1, 256;" ::: "memory");
      }
      if (ok) finish<EPI>(g, part, slab0 + t, warp, lane, z, slog, own_tokens);
      if (t + 1 < tiles) asm volatile("bar.sync 1, 256;" ::: "memory");
    }
  }

  __syncwarp();
  if (warp == WARP_TMA && *reinterpret_cast<volatile int*>(&bars->abort_flag)) {
    const unsigned long long until = globaltimer_ns() + 1000000ull;      // loads in flight land before the memory is given up
    while (globaltimer_ns() < until) {}
  }
  if (S > 1 && warp >= WORKERS) {                // the other two warps' part in both cluster barriers
    cluster_wait();
    cluster_arrive();
    cluster_wait();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == WARP_MMA) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;"
                 ::"r"(*reinterpret_cast<volatile uint32_t*>(&bars->tmem_base)), "r"(TMEM_COLS));
  }
}

int encode(CUtensorMap* map, const void* ptr, long long rows, long long cols, long long ld, int box_rows) {
  if (((uintptr_t)ptr & 15) || ld % 16) return RWKV_ERR_BAD_ALIGNMENT;
  rwkv_tmap::EncodeTiledFn enc = rwkv_tmap::get_encode();
  if (!enc) return RWKV_ERR_NOT_INITIALISED;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, estr[2] = {1, 1};
  CUresult r = CUDA_SUCCESS;
  for (int attempt = 0; attempt < 2; ++attempt) {
    r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_ERROR_INVALID_CONTEXT) break;
    cudaFree(nullptr);       // a thread without CUDA work so far: binds the device's context
  }
  return r == CUDA_SUCCESS ? RWKV_OK : RWKV_ERR_CUDA_BASE + 900 + (int)r;
}

template <bool PACKED, int EPI>
int launch(const CUtensorMap& mw, const CUtensorMap& mx, const Args& g, int smem, int chained, cudaStream_t st) {
  auto kern = fp8_decode_kernel<PACKED, EPI>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  static std::atomic<unsigned long long> configured{0};
  const unsigned long long bit = 1ull << (dev & 63);
  if (e == cudaSuccess && !(configured.load() & bit)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX);
    if (e == cudaSuccess) configured.fetch_or(bit);
  }
  if (e != cudaSuccess) return RWKV_ERR_CUDA_BASE + (int)e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(((g.N + 127) / 128 + g.tiles - 1) / g.tiles), 1u << g.split_log);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = 1u << g.split_log;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = chained ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kern, mw, mx, g);
  return rwkv_launch_status();
}

// CTAs that share a column block: as many as bring the launch to at least 120 of the 148 SMs, eight at most
int split_for(int N, int K) {
  const int slabs = (N + 127) / 128, kb = (K + 127) / 128;
  int s = 1;
  while (s < 8 && slabs * s < 120 && s * 2 <= kb) s *= 2;
  return s;
}
// Column blocks of a CTA: with more blocks than two CTAs on every SM, a CTA takes several and its ring runs on from one to
// the next, so the weights keep streaming through the epilogues.
int tiles_for(int N, int K, int split) {
  const int slabs = (N + 127) / 128, groups = ((K + 127) / 128 + 3) / 4;
  if (split > 1) return 1;
  const int fit = MAX_SETS / groups - 1, want = (slabs + 2 * 148 - 1) / (2 * 148);
  return want < fit ? want : fit < 1 ? 1 : fit;
}

struct Layout {
  int stages, smem;          // stages = 0: does not fit
};
Layout layout_for(int mpad, int K, int split, int tiles, bool packed) {
  const int kb = ((K + 127) / 128 + split - 1) / split, groups = (kb + 3) / 4;
  if (groups > MAX_GROUPS) return {0, 0};
  const int stage = W_BYTES + (packed ? mpad * 128 : 0);
  const int fixed = (packed ? 0 : kb * mpad * 128) + groups * (1 + tiles) * 512 + (mpad + split - 1) / split * split * 512 +
                    (int)sizeof(Barriers) + 1024 + 64;
  for (int budget = SMEM_MIN; budget <= SMEM_MAX; budget += SMEM_MAX - SMEM_MIN) {
    int stages = (budget - fixed) / stage;
    if (stages > MAX_STAGES) stages = MAX_STAGES;
    if (stages >= (kb < 3 ? kb : 3)) return {stages, budget};
  }
  return {0, 0};
}

}  // namespace

// How a product of M tokens with a packed [N, K] weight is run: 0 - not by this kernel, 1 - on packed tokens,
// 2 - on bf16 tokens that it packs itself (never if `packed`: the tokens are packed already).  Depends on sizes only.
RWKV_EXPORT int rwkv_fp8_decode_form(int M, int N, int K, int packed) {
  if (M < 1 || M > 128 || N < 1 || K < 1 || N > 0x7ffffe00 || K > 0x7ffffe00) return 0;
  const int mpad = (M + 15) / 16 * 16, split = split_for(N, K), tiles = tiles_for(N, K, split);
  if (!packed && K % 8 == 0 && M <= 16 && layout_for(mpad, K, split, tiles, false).stages) return 2;
  return layout_for(mpad, K, split, tiles, true).stages ? 1 : 0;
}

// x: bf16 rows (16-byte aligned, K a multiple of 8) or, if null, packed tokens in (a_val, a_exp) with blocks of one row;
// epilogue 0, 1 (packed tokens only), 2 as in gemm_fp8_tcgen05.cu with q_rows = 1.  chained: may start before its predecessor in the stream has
// finished; the weights must not be written by it.
int rwkv_fp8_decode(const Fp8Step& s, cudaStream_t st) {
  const int M = s.M, N = s.N, K = s.K;
  if (M < 1 || M > 128 || N < 1 || K < 1 || N > 0x7ffffe00 || K > 0x7ffffe00 || s.epilogue < 0 || s.epilogue > 2)
    return RWKV_ERR_BAD_SHAPE;
  const bool packed = !s.x;
  if (packed ? !s.a_val || !s.a_exp || s.a_rows != 1 : (K % 8 || s.ldx < K || s.epilogue == 1)) return RWKV_ERR_BAD_SHAPE;
  if (!packed && (((uintptr_t)s.x & 15) || s.ldx % 8)) return RWKV_ERR_BAD_ALIGNMENT;
  if (s.epilogue == 2 ? !s.q_val || !s.q_exp || s.q_rows != 1 : !s.c || s.ldc < N || (s.epilogue == 1 && (!s.residual || s.ldr < N)))
    return RWKV_ERR_BAD_SHAPE;
  const int mpad = (M + 15) / 16 * 16, split = split_for(N, K), tiles = tiles_for(N, K, split);
  const Layout lay = layout_for(mpad, K, split, tiles, packed);
  if (!lay.stages) return RWKV_ERR_TOO_LARGE;
  const int ldk = (K + 15) / 16 * 16;
  CUtensorMap mw, mx;
  int r = encode(&mw, s.b_val, N, K, ldk, 128);
  if (r) return r;
  if (packed) r = encode(&mx, s.a_val, M, K, ldk, mpad); else mx = mw;
  if (r) return r;
  Args g = {};
  g.M = M; g.N = N; g.K = K; g.mpad = mpad; g.stages = lay.stages; g.tiles = tiles;
  while ((1 << g.split_log) < split) ++g.split_log;
  while ((1 << g.m_log) < M) ++g.m_log;
  g.w_exp = (const uint8_t*)s.b_exp;
  g.x = (const bf16*)s.x; g.ldx = s.ldx;
  g.x_exp = (const uint8_t*)s.a_exp; g.x_lde = (M + 15) / 16 * 16;
  g.c = (bf16*)s.c; g.residual = (const bf16*)s.residual; g.ldc = s.ldc; g.ldr = s.ldr;
  g.vec = !(N % 4) && !((uintptr_t)s.c & 7) && !(s.ldc % 4) && !((uintptr_t)s.residual & 7) && !(s.ldr % 4);
  g.q_val = (uint8_t*)s.q_val; g.q_exp = (uint8_t*)s.q_exp;
  g.q_ldv = (N + 15) / 16 * 16; g.q_lde = (M + 15) / 16 * 16;
  g.status = (int*)s.status;
  const bool next = rwkv_chain_next(st);
  const int ch = s.chained && (next || !rwkv_chain().on);      // in a chain: not its first launch
  if (packed) {
    if (s.epilogue == 2) return launch<true, EPI_RELU_SQ>(mw, mx, g, lay.smem, ch, st);
    return s.epilogue == 1 ? launch<true, EPI_RESIDUAL>(mw, mx, g, lay.smem, ch, st) : launch<true, EPI_STORE>(mw, mx, g, lay.smem, ch, st);
  }
  return s.epilogue == 2 ? launch<false, EPI_RELU_SQ>(mw, mx, g, lay.smem, ch, st) : launch<false, EPI_STORE>(mw, mx, g, lay.smem, ch, st);
}
