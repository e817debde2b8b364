// 8-bit product for few rows: y[M, N] = x[M, K] W[N, K]^T with M <= 128 and W packed in tiles (fp8_format.cuh).
//
// Bound by streaming W once, one byte a weight, and below a few megabytes by latency.  As in gemm_decode_tcgen05.cu the
// weight tile is the 128-row operand A of the instruction and the tokens are its columns (M rounded up to 16), so the
// accumulator's lanes are full whatever M is; a column block of 128 weights is one CTA's, its contraction is cut over a
// cluster of S CTAs, and the partial tiles are summed through distributed shared memory in a fixed order.  S depends on N
// and K alone, so a row's result does not depend on how many others there are.
//
// The tokens come either in bf16 - then each CTA packs its part of the contraction itself, row by row, into the
// shared-memory tiles the tensor core reads, which saves a launch and a round trip - or already packed, fetched by TMA in
// the same ring as the weights.  Packing in the kernel repeats the work in every CTA, so it is used while a CTA's tokens fit
// a small part of its shared memory (see rwkv_fp8_decode).
//
// Epilogues: store bf16, add a bf16 residual, or relu(y)^2 packed again: a CTA owns exactly one block of 128 columns of
// every token, so a block's scale is a maximum over one warp.
//
// A launch may be chained to its predecessor (programmatic dependent launch): it requests its first weight tiles, which no
// kernel of the chain writes, before it waits for the predecessor's results.
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
constexpr int TMEM_COLS = 256, SF_COL = 128;     // accumulator in columns 0..127, eight columns of scales per set behind it
constexpr int SMEM_MIN = 112 * 1024, SMEM_MAX = 224 * 1024;
constexpr unsigned long long WAIT_NS = 2000000000ull;

struct Barriers {
  uint64_t full[MAX_STAGES], empty[MAX_STAGES];
  uint64_t x_ready[MAX_GROUPS];                  // tokens (or their scales) of a set are in shared memory
  uint64_t acc_full;
  uint32_t tmem_base;
  int abort_flag;
};

struct Args {
  int M, N, K, mpad, stages, split;
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
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}

enum Epilogue { EPI_STORE = 0, EPI_RESIDUAL = 1, EPI_RELU_SQ = 2 };

// grid: (column blocks of 128, S), clusters of (1, S, 1)
template <bool PACKED, int EPI>
__global__ void __launch_bounds__(THREADS)
fp8_decode_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                  const __grid_constant__ Args g) {
  extern __shared__ unsigned char smem_dyn[];
  const uint32_t raw = smem_u32(smem_dyn);
  const uint32_t base = (raw + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = g.split, z = (int)blockIdx.y, n0 = (int)blockIdx.x * 128;
  const int all_kb = (g.K + 127) / 128, kb0 = (int)((long long)all_kb * z / S), nkb = (int)((long long)all_kb * (z + 1) / S) - kb0;
  const int groups = (nkb + 3) / 4, x_bytes = g.mpad * 128;
  const int stage_bytes = W_BYTES + (PACKED ? x_bytes : 0);
  const uint32_t xs = base + g.stages * stage_bytes;                       // tokens packed here (not PACKED)
  const int max_kb = (all_kb + S - 1) / S;
  const uint32_t sf = xs + (PACKED ? 0 : max_kb * x_bytes);                // 512 bytes of A, 512 of B per set
  Barriers* bars = reinterpret_cast<Barriers*>(smem_dyn + (sf - raw) + (max_kb + 3) / 4 * 1024);

  if (threadIdx.x == 0) {
    for (int s = 0; s < g.stages; ++s) { mbar_init(&bars->full[s], 1); mbar_init(&bars->empty[s], 1); }
    for (int i = 0; i < groups; ++i) mbar_init(&bars->x_ready[i], WORKERS);
    mbar_init(&bars->acc_full, 1);
    bars->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == WARP_MMA) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem_base)),
                 "r"(TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  rwkv_chain_trigger();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;

  if (warp == WARP_TMA) {
    if (lane == 0) {
      const int first = nkb < g.stages ? nkb : g.stages;
      for (int i = 0; i < first; ++i) {
        mbar_expect_tx(&bars->full[i], stage_bytes);
        tma_load_2d(base + i * stage_bytes, &map_w, &bars->full[i], (kb0 + i) * 128, n0);
      }
      rwkv_chain_wait();
      if (PACKED)
        for (int i = 0; i < first; ++i)
          tma_load_2d(base + i * stage_bytes + W_BYTES, &map_x, &bars->full[i], (kb0 + i) * 128, 0);
      for (int i = first; i < nkb; ++i) {
        const int s = i % g.stages;
        if (!mbar_wait(&bars->empty[s], (i / g.stages - 1) & 1, bars, g.status, 221)) break;
        mbar_expect_tx(&bars->full[s], stage_bytes);
        tma_load_2d(base + s * stage_bytes, &map_w, &bars->full[s], (kb0 + i) * 128, n0);
        if (PACKED) tma_load_2d(base + s * stage_bytes + W_BYTES, &map_x, &bars->full[s], (kb0 + i) * 128, 0);
      }
    }
  } else if (warp == WARP_MMA) {
    if (lane == 0) {
      // kind::mxf8f6f4: e4m3 operands, both K-major, E8M0 scales, M = 128, N = mpad
      const uint32_t idesc = ((uint32_t)(g.mpad >> 3) << 17) | (1u << 23) | (1u << 27);
      bool ok = true;
      for (int i = 0; i < nkb && ok; ++i) {
        const int s = i % g.stages;
        const uint32_t id = i & 3, sfa = tmem + SF_COL + (i >> 2) * 8, sfb = sfa + 4;
        if (id == 0) {
          if (!mbar_wait(&bars->x_ready[i >> 2], 0, bars, g.status, 222)) break;
          tc_fence_after();
          scales_to_tmem(sfa, scale_desc(sf + (i >> 2) * 1024));
          scales_to_tmem(sfb, scale_desc(sf + (i >> 2) * 1024 + 512));
        }
        ok = mbar_wait(&bars->full[s], (i / g.stages) & 1, bars, g.status, 223);
        if (!ok) break;
        tc_fence_after();
        const uint32_t sa = base + s * stage_bytes, sb = PACKED ? sa + W_BYTES : xs + i * x_bytes;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma(tmem, operand_desc(sa) + k * 2, operand_desc(sb) + k * 2, idesc | (id << 4) | (id << 29), sfa, sfb, (i | k) ? 1u : 0u);
        umma_commit(&bars->empty[s]);
      }
      umma_commit(&bars->acc_full);
    }
  } else {
    // ---- scales of the weights: one byte per block, the same for all 128 rows
    for (int i = warp; i < groups; i += WORKERS) {
      const int kb = kb0 + i * 4 + (lane & 3);
      uint32_t w = kb < all_kb ? (uint32_t)g.w_exp[(long long)blockIdx.x * all_kb + kb] << (8 * (lane & 3)) : 0u;
      w |= __shfl_xor_sync(0xffffffffu, w, 1);
      w |= __shfl_xor_sync(0xffffffffu, w, 2);
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sf + i * 1024 + lane * 16), "r"(w) : "memory");
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");
    rwkv_chain_wait();
    if (PACKED) {
      // ---- scales of the tokens: word of row r holds the bytes of four blocks
      for (int u = threadIdx.x; u < groups * g.M; u += 32 * WORKERS) {
        const int i = u / g.M, r = u % g.M;
        uint32_t w = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b)
          if (i * 4 + b < nkb) w |= (uint32_t)g.x_exp[(long long)(kb0 + i * 4 + b) * g.x_lde + r] << (8 * b);
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(sf + i * 1024 + 512 + (r & 31) * 16 + (r >> 5) * 4), "r"(w) : "memory");
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0)
        for (int i = 0; i < groups; ++i) mbar_arrive(&bars->x_ready[i]);
    } else {
      // ---- pack the tokens: eight threads a block of 128, four blocks a thread in flight
      constexpr int DEEP = 4;
      const int part = lane & 7;
      for (int i = 0; i < groups; ++i) {
        const int blocks = nkb - i * 4 < 4 ? nkb - i * 4 : 4, units = blocks * g.M;
        for (int u0 = warp * 4 + (lane >> 3); u0 - (lane >> 3) < units; u0 += WORKERS * 4 * DEEP) {
          uint4 v[DEEP][2];
#pragma unroll
          for (int d = 0; d < DEEP; ++d) {
            const int u = u0 + d * WORKERS * 4, row = u % g.M, kb = kb0 + i * 4 + u / g.M, col = kb * 128 + part * 16;
            v[d][0] = v[d][1] = make_uint4(0u, 0u, 0u, 0u);
            if (u < units) {
              const uint4* p = reinterpret_cast<const uint4*>(g.x + row * g.ldx + col);
              if (col < g.K) v[d][0] = p[0];
              if (col + 8 < g.K) v[d][1] = p[1];
            }
          }
#pragma unroll
          for (int d = 0; d < DEEP; ++d) {
            const int u = u0 + d * WORKERS * 4, row = u % g.M, b = u / g.M;
            float f[16];
            unpack8(v[d][0], f);
            unpack8(v[d][1], f + 8);
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 16; ++j) top = max(top, __float_as_uint(f[j]) & 0x7fffffffu);
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            if (u < units) {
              const uint32_t e = fp8_block_exponent(top);
              uint32_t q[4];
              const float s = fp8_inverse_scale(e == 255u ? 127u : e);
#pragma unroll
              for (int j = 0; j < 4; ++j)
                q[j] = e == 255u ? 0x7f7f7f7fu : fp8_pack4(f[4 * j] * s, f[4 * j + 1] * s, f[4 * j + 2] * s, f[4 * j + 3] * s);
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                           ::"r"(xs + (i * 4 + b) * x_bytes + row * 128 + ((part ^ (row & 7)) << 4)), "r"(q[0]), "r"(q[1]), "r"(q[2]),
                             "r"(q[3])
                           : "memory");
              if (part == 0)
                asm volatile("st.shared.u8 [%0], %1;" ::"r"(sf + i * 1024 + 512 + (row & 31) * 16 + (row >> 5) * 4 + b), "r"(e)
                             : "memory");
            }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->x_ready[i]);
      }
    }
    // ---- this CTA's partial tile, [token][128 columns] in fp32, over the ring (every load of it has been consumed)
    mbar_wait(&bars->acc_full, 0, bars, g.status, 224);
    __syncwarp();
    tc_fence_after();
    const int quarter = warp & 3;
    // All mpad rows are stored: with the store under a test of the row, nvcc 12.9 dropped that of the last row of an unrolled
    // iteration.
#pragma unroll 1
    for (int m = (warp >> 2) * 8; m < g.mpad; m += 16) {
      float v[8];
      tmem_ld8(tmem + ((uint32_t)(quarter * 32) << 16) + m, v);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(base + (m + e) * 512 + (quarter * 32 + lane) * 4), "f"(v[e]) : "memory");
    }
  }

  __syncwarp();
  if (warp == WARP_TMA && *reinterpret_cast<volatile int*>(&bars->abort_flag)) {
    const unsigned long long until = globaltimer_ns() + 1000000ull;      // loads in flight land before the memory is given up
    while (globaltimer_ns() < until) {}
  }
  tc_fence_before();
  if (S > 1) cluster_sync(); else __syncthreads();
  if (warp == WARP_MMA) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS));
  }
  if (warp < WORKERS && !*reinterpret_cast<volatile int*>(&bars->abort_flag)) {
    // ---- tokens z, z + S, ... of the cluster's sum, one warp a token, four columns a lane
    const int n = n0 + lane * 4;
    for (int m = z + warp * S; m < g.M; m += WORKERS * S) {
      float f[4] = {0.f, 0.f, 0.f, 0.f};
      for (int r = 0; r < S; ++r) {
        uint32_t at;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(base + m * 512 + lane * 16), "r"(r));
        float4 p;
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(p.x), "=f"(p.y), "=f"(p.z), "=f"(p.w) : "r"(at));
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
        if (lane == 0) g.q_exp[(long long)blockIdx.x * g.q_lde + m] = (uint8_t)e;
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
  if (S > 1) cluster_sync();           // no CTA leaves while another reads its partial tile
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
  cfg.gridDim = dim3((unsigned)((g.N + 127) / 128), (unsigned)g.split);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = g.split;
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

struct Layout {
  int stages, smem;          // stages = 0: does not fit
};
Layout layout_for(int mpad, int K, int split, bool packed) {
  const int kb = ((K + 127) / 128 + split - 1) / split;
  if ((kb + 3) / 4 > MAX_GROUPS) return {0, 0};
  const int stage = W_BYTES + (packed ? mpad * 128 : 0);
  const int fixed = (packed ? 0 : kb * mpad * 128) + (kb + 3) / 4 * 1024 + (int)sizeof(Barriers) + 1024 + 64;
  const int need = mpad * 512;                                       // the partial tile lies over the ring
  for (int budget = SMEM_MIN; budget <= SMEM_MAX; budget += SMEM_MAX - SMEM_MIN) {
    int stages = (budget - fixed) / stage;
    if (stages > MAX_STAGES) stages = MAX_STAGES;
    if (stages >= 3 && stages * stage >= need) return {stages, budget};
  }
  return {0, 0};
}

}  // namespace

// How a product of M tokens with a packed [N, K] weight is run: 0 - not by this kernel, 1 - on packed tokens,
// 2 - on bf16 tokens that it packs itself (never if `packed`: the tokens are packed already).  Depends on sizes only.
RWKV_EXPORT int rwkv_fp8_decode_form(int M, int N, int K, int packed) {
  if (M < 1 || M > 128 || N < 1 || K < 1 || N > 0x7ffffe00 || K > 0x7ffffe00) return 0;
  const int mpad = (M + 15) / 16 * 16, split = split_for(N, K);
  if (!packed && K % 8 == 0 && M <= 16 && layout_for(mpad, K, split, false).stages) return 2;
  return layout_for(mpad, K, split, true).stages ? 1 : 0;
}

// x: bf16 rows (16-byte aligned, K a multiple of 8) or, if null, packed tokens in (a_val, a_exp) with blocks of one row;
// epilogue 0, 1, 2 as in gemm_fp8_tcgen05.cu with q_rows = 1.  chained: may start before its predecessor in the stream has
// finished; the weights must not be written by it.
int rwkv_fp8_decode(const Fp8Step& s, cudaStream_t st) {
  const int M = s.M, N = s.N, K = s.K;
  if (M < 1 || M > 128 || N < 1 || K < 1 || N > 0x7ffffe00 || K > 0x7ffffe00 || s.epilogue < 0 || s.epilogue > 2)
    return RWKV_ERR_BAD_SHAPE;
  const bool packed = !s.x;
  if (packed ? !s.a_val || !s.a_exp || s.a_rows != 1 : (K % 8 || s.ldx < K)) return RWKV_ERR_BAD_SHAPE;
  if (!packed && (((uintptr_t)s.x & 15) || s.ldx % 8)) return RWKV_ERR_BAD_ALIGNMENT;
  if (s.epilogue == 2 ? !s.q_val || !s.q_exp || s.q_rows != 1 : !s.c || s.ldc < N || (s.epilogue == 1 && (!s.residual || s.ldr < N)))
    return RWKV_ERR_BAD_SHAPE;
  const int mpad = (M + 15) / 16 * 16, split = split_for(N, K);
  const Layout lay = layout_for(mpad, K, split, packed);
  if (!lay.stages) return RWKV_ERR_TOO_LARGE;
  const int ldk = (K + 15) / 16 * 16;
  CUtensorMap mw, mx;
  int r = encode(&mw, s.b_val, N, K, ldk, 128);
  if (r) return r;
  if (packed) r = encode(&mx, s.a_val, M, K, ldk, mpad); else mx = mw;
  if (r) return r;
  Args g = {};
  g.M = M; g.N = N; g.K = K; g.mpad = mpad; g.stages = lay.stages; g.split = split;
  g.w_exp = (const uint8_t*)s.b_exp;
  g.x = (const bf16*)s.x; g.ldx = s.ldx;
  g.x_exp = (const uint8_t*)s.a_exp; g.x_lde = (M + 15) / 16 * 16;
  g.c = (bf16*)s.c; g.residual = (const bf16*)s.residual; g.ldc = s.ldc; g.ldr = s.ldr;
  g.vec = !(N % 4) && !((uintptr_t)s.c & 7) && !(s.ldc % 4) && !((uintptr_t)s.residual & 7) && !(s.ldr % 4);
  g.q_val = (uint8_t*)s.q_val; g.q_exp = (uint8_t*)s.q_exp;
  g.q_ldv = (N + 15) / 16 * 16; g.q_lde = (M + 15) / 16 * 16;
  g.status = (int*)s.status;
  const int ch = s.chained;
  if (packed) {
    if (s.epilogue == 2) return launch<true, EPI_RELU_SQ>(mw, mx, g, lay.smem, ch, st);
    return s.epilogue == 1 ? launch<true, EPI_RESIDUAL>(mw, mx, g, lay.smem, ch, st) : launch<true, EPI_STORE>(mw, mx, g, lay.smem, ch, st);
  }
  if (s.epilogue == 2) return launch<false, EPI_RELU_SQ>(mw, mx, g, lay.smem, ch, st);
  return s.epilogue == 1 ? launch<false, EPI_RESIDUAL>(mw, mx, g, lay.smem, ch, st) : launch<false, EPI_STORE>(mw, mx, g, lay.smem, ch, st);
}
