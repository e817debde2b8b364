// Packing to and from the 8-bit block format (fp8_format.cuh): activation checkpoints, and the operands of the 8-bit GEMMs.
//
// Both directions are bound by memory: 2 + 1 bytes a value for bf16.  Eight threads own the 128 columns of a block's row, 16
// values each, in pieces as wide as the row pitch and the address allow (32 to 2 bytes), neighbouring threads on
// neighbouring pieces.  The values stay in registers between the maximum and the rounding, so the input is read once:
//   rows = 1  : the maximum is three shuffles among the eight threads; one block a thread and many CTAs (two or four blocks
//               a thread in flight were slower: 32768 x 2048 in 35.0, 39.1 and 46.0 us);
//   rows = 128: a CTA of 512 threads walks over tiles with the next one's loads in flight; warp maxima meet in shared
//               memory (one CTA a tile: 43.2 us, walking: 33.3 us, 6.06 TB/s).
//
// Launched through rwkv_launch: inside a chain of decode launches they are part of it.  Tiles may be weights, which products of
// the chain fetch before they wait: the launch after them is an ordinary one.
//
// Arithmetic in the rest of the library flushes numbers below 2^-126 to zero, and so do these kernels.
#include <cuda_fp16.h>

#include <type_traits>

#include "fp8_format.cuh"
#include "fp8_steps.cuh"

namespace {

__device__ __forceinline__ float to_f32(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ bf16 from_f32<bf16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
// largest finite value: the rounding to e4m3 may lift a value next to it by half a step, and a finite input reads back finite
template <typename T> __device__ __forceinline__ float largest();
template <> __device__ __forceinline__ float largest<bf16>() { return 3.3895313892515355e38f; }
template <> __device__ __forceinline__ float largest<__half>() { return 65504.f; }
template <> __device__ __forceinline__ float largest<float>() { return 3.4028234663852886e38f; }
// smallest exponent byte of a block with a value of T's largest power of two or more: 256 * 2^(E - 127) reaches it
template <typename T> __device__ __forceinline__ constexpr uint32_t first_overflow() { return 127 + 127 - 8; }
template <> __device__ __forceinline__ constexpr uint32_t first_overflow<__half>() { return 127 + 15 - 8; }

// 16 neighbouring values as they lie in memory
template <typename T> struct Raw16 {
  union {
    uint32_t w[4 * sizeof(T)];
    T t[16];
  };
};
template <int V> __device__ __forceinline__ void load_word(const void* p, uint32_t* w);
template <> __device__ __forceinline__ void load_word<4>(const void* p, uint32_t* w) { w[0] = __ldcs((const uint32_t*)p); }
template <> __device__ __forceinline__ void load_word<8>(const void* p, uint32_t* w) {
  const uint2 v = __ldcs((const uint2*)p);
  w[0] = v.x; w[1] = v.y;
}
template <> __device__ __forceinline__ void load_word<16>(const void* p, uint32_t* w) {
  const uint4 v = __ldcs((const uint4*)p);
  w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
}
template <> __device__ __forceinline__ void load_word<32>(const void* p, uint32_t* w) {
  asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p));
}
template <int V> __device__ __forceinline__ void store_word(void* p, const uint32_t* w);
template <> __device__ __forceinline__ void store_word<4>(void* p, const uint32_t* w) { *(uint32_t*)p = w[0]; }
template <> __device__ __forceinline__ void store_word<8>(void* p, const uint32_t* w) { *(uint2*)p = make_uint2(w[0], w[1]); }
template <> __device__ __forceinline__ void store_word<16>(void* p, const uint32_t* w) {
  *(uint4*)p = make_uint4(w[0], w[1], w[2], w[3]);
}
template <> __device__ __forceinline__ void store_word<32>(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
               "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// A thread's 16 values of a block's row: pieces of PER values, piece i of thread `part` at (8 i + part) PER.
// The first n values of the row are in range (n may be <= 0 or above 128), the others read as zero.
template <typename T, int V>
__device__ __forceinline__ void load16(const T* p, int part, int n, Raw16<T>& r) {
  constexpr int PER = V / (int)sizeof(T);
#pragma unroll
  for (int i = 0; i < 16 / PER; ++i) {
    const int at = (8 * i + part) * PER;
    if (V > 2 && at + PER <= n) {
      load_word<(V > 2 ? V : 4)>(p + at, r.w + i * V / 4);
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j) r.t[i * PER + j] = at + j < n ? p[at + j] : from_f32<T>(0.f);
    }
  }
}
template <typename T>
__device__ __forceinline__ void widen16(const Raw16<T>& r, float* f) {
#pragma unroll
  for (int i = 0; i < 16; ++i) f[i] = to_f32(r.t[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store16(T* p, int part, int n, const float* f) {
  constexpr int PER = V / (int)sizeof(T);
  Raw16<T> r;
#pragma unroll
  for (int i = 0; i < 16; ++i) r.t[i] = from_f32<T>(f[i]);
#pragma unroll
  for (int i = 0; i < 16 / PER; ++i) {
    const int at = (8 * i + part) * PER;
    if (V > 2 && at + PER <= n) {
      store_word<(V > 2 ? V : 4)>(p + at, r.w + i * V / 4);
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (at + j < n) p[at + j] = r.t[i * PER + j];
    }
  }
}
// the same pieces of a packed row, n columns of which exist (a multiple of 16)
union Packed16 {
  uint32_t w[4];
  uint16_t h[8];
  uint8_t b[16];
};
template <int PER>
__device__ __forceinline__ void store_packed(uint8_t* p, int part, int n, const Packed16& q) {
#pragma unroll
  for (int i = 0; i < 16 / PER; ++i) {
    const int at = (8 * i + part) * PER;
    if (at >= n) continue;
    if constexpr (PER >= 4) store_word<(PER >= 4 ? PER : 4)>(p + at, q.w + i * PER / 4);
    if constexpr (PER == 2) *reinterpret_cast<uint16_t*>(p + at) = q.h[i];
    if constexpr (PER == 1) p[at] = q.b[i];
  }
}
template <int PER>
__device__ __forceinline__ void load_packed(const uint8_t* p, int part, int n, Packed16& q) {
#pragma unroll
  for (int i = 0; i < 16 / PER; ++i) {
    const int at = (8 * i + part) * PER;
    const bool live = at < n;
    if constexpr (PER >= 4) {
      if (live) load_word<(PER >= 4 ? PER : 4)>(p + at, q.w + i * PER / 4);
    }
    if constexpr (PER == 2) q.h[i] = live ? *reinterpret_cast<const uint16_t*>(p + at) : 0;
    if constexpr (PER == 1) q.b[i] = live ? p[at] : 0;
  }
}

__device__ __forceinline__ uint32_t abs_bits16(const float* f) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
  return m;
}
__device__ __forceinline__ Packed16 quantise16(const float* f, uint32_t e) {
  Packed16 q;
  const float s = fp8_inverse_scale(e == 255u ? 127u : e);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    q.w[i] = e == 255u ? 0x7f7f7f7fu : fp8_pack4(f[4 * i] * s, f[4 * i + 1] * s, f[4 * i + 2] * s, f[4 * i + 3] * s);
  return q;
}

constexpr int ROW_THREADS = 256;

template <typename T, int V>
__global__ void __launch_bounds__(ROW_THREADS)
fp8_pack_rows_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ values, uint8_t* __restrict__ exps,
                     uint32_t units, int C, int ldv, int lde, uint32_t blocks) {
  rwkv_chain_begin();         // a chained decode product may fetch its weights meanwhile
  const int part = threadIdx.x & 7;
  const uint32_t step = gridDim.x * (ROW_THREADS / 8);
  Raw16<T> next;
  auto fetch = [&](uint32_t u) {
    const uint32_t row = u < units ? u / blocks : 0, col = u < units ? (u - row * blocks) * FP8_BLOCK : 0;
    load16<T, V>(x + row * ldx + col, part, u < units ? C - (int)col : 0, next);
  };
  // the first block of a warp decides for all of it: the shuffles need whole warps
  uint32_t base = blockIdx.x * (ROW_THREADS / 8) + (threadIdx.x >> 5) * 4;
  const uint32_t mine = (threadIdx.x >> 3) & 3;
  if (base < units) fetch(base + mine);
  for (; base < units; base += step) {
    float f[16];
    widen16(next, f);
    if (base + step < units) fetch(base + step + mine);
    uint32_t m = abs_bits16(f);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const uint32_t u = base + mine, e = fp8_block_exponent(m);
    if (u < units) {
      const uint32_t row = u / blocks, kb = u - row * blocks;
      const int col = kb * FP8_BLOCK;
      store_packed<V / sizeof(T)>(values + (long long)row * ldv + col, part, ldv - col, quantise16(f, e));
      if (part == 0) exps[(long long)kb * lde + row] = (uint8_t)e;
    }
  }
}

constexpr int TILE_THREADS = 512;

// Up to three matrices whose tiles follow one another: the operands of one pass in one launch.
struct TileJob {
  const void* x;
  long long ldx;
  uint8_t *values, *exps;
  int R, C, ldv;
  uint32_t blocks, end;           // column blocks; number of tiles up to and with this matrix
};
constexpr int MAX_JOBS = 3;
struct TileJobs {
  TileJob job[MAX_JOBS];
  int count;
};

// A CTA walks over tiles and has the next one in flight while it works on the present one.  MANY: more than one matrix
// (looking a tile's matrix up costs a single one 34.0 -> 36.8 us at 32768 x 2048).
template <typename T, int V, bool MANY>
__global__ void __launch_bounds__(TILE_THREADS, sizeof(T) == 4 ? 1 : 2)
fp8_pack_tiles_kernel(const __grid_constant__ TileJobs all) {
  rwkv_chain_begin();
  __shared__ uint32_t warp_max[2][TILE_THREADS / 32];
  const uint32_t tiles = MANY ? all.job[all.count - 1].end : all.job[0].end;
  const int part = threadIdx.x & 7;
  // the matrix of a tile, the tile's number in it, and this thread's first row and the tile's first column
  const auto locate = [&](uint32_t tile, uint32_t& own, int& row, int& col) -> const TileJob& {
    int j = 0;
    while (MANY && j + 1 < all.count && tile >= all.job[j].end) ++j;
    const TileJob& m = MANY ? all.job[j] : all.job[0];
    own = tile - (j ? all.job[j - 1].end : 0);
    row = (int)(own / m.blocks) * FP8_BLOCK + (threadIdx.x >> 3);
    col = (int)(own % m.blocks) * FP8_BLOCK;
    return m;
  };
  Raw16<T> next[2];
  const auto fetch = [&](uint32_t tile) {
    uint32_t own;
    int row0, col;
    const TileJob& m = locate(tile, own, row0, col);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = row0 + i * (TILE_THREADS / 8);
      load16<T, V>((const T*)m.x + min(row, m.R - 1) * m.ldx + col, part, row < m.R ? m.C - col : 0, next[i]);
    }
  };
  uint32_t tile = blockIdx.x;
  if (tile < tiles) fetch(tile);
  for (int turn = 0; tile < tiles; turn ^= 1) {
    float f[2][16];
    widen16(next[0], f[0]);
    widen16(next[1], f[1]);
    const uint32_t now = tile;
    tile += gridDim.x;
    if (tile < tiles) fetch(tile);
    uint32_t top = max(abs_bits16(f[0]), abs_bits16(f[1]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) warp_max[turn][threadIdx.x >> 5] = top;
    __syncthreads();
    top = warp_max[turn][threadIdx.x & (TILE_THREADS / 32 - 1)];
#pragma unroll
    for (int o = TILE_THREADS / 64; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const uint32_t e = fp8_block_exponent(top);
    uint32_t own;
    int row0, col;
    const TileJob& m = locate(now, own, row0, col);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = row0 + i * (TILE_THREADS / 8);
      if (row < m.R)
        store_packed<V / sizeof(T)>(m.values + (long long)row * m.ldv + col, part, m.ldv - col, quantise16(f[i], e));
    }
    if (threadIdx.x == 0) m.exps[own] = (uint8_t)e;
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(ROW_THREADS)
fp8_unpack_kernel(const uint8_t* __restrict__ values, const uint8_t* __restrict__ exps, T* __restrict__ y, long long ldy,
                  uint32_t units, int C, int ldv, int lde, int rows, uint32_t blocks) {
  rwkv_chain_begin();
  const int part = threadIdx.x & 7;
  for (uint32_t u = blockIdx.x * (ROW_THREADS / 8) + (threadIdx.x >> 3); u < units; u += gridDim.x * (ROW_THREADS / 8)) {
    const uint32_t row = u / blocks, kb = u - row * blocks;
    const int col = kb * FP8_BLOCK;
    const uint32_t e = rows == 1 ? exps[(long long)kb * lde + row] : exps[(long long)(row / FP8_BLOCK) * lde + kb];
    Packed16 q;
    load_packed<V / sizeof(T)>(values + (long long)row * ldv + col, part, ldv - col, q);
    float f[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) fp8_unpack4(q.w[i], f + 4 * i);
    // one multiplication, but for blocks whose scale is no normal number and for those that may end above the largest one
    if (e != 0u && e < first_overflow<T>()) {
      const float s = __uint_as_float(e << 23);
#pragma unroll
      for (int i = 0; i < 16; ++i) f[i] *= s;
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        f[i] = fp8_scaled(f[i], e);
        if (e < 255u) f[i] = fminf(fmaxf(f[i], -largest<T>()), largest<T>());
      }
    }
    store16<T, V>(y + row * ldy + col, part, C - col, f);
  }
}

// widest access that every row start allows
int access_bytes(const void* p, long long pitch_bytes) {
  for (int v = 32; v > 2; v /= 2)
    if ((uintptr_t)p % v == 0 && pitch_bytes % v == 0) return v;
  return 2;
}
inline int up(int n, int m) { return (n + m - 1) / m * m; }
int grid_for(long long ctas, int per_sm) { return (int)(ctas < 148 * per_sm ? ctas : 148 * per_sm); }
// Rows of one launch: the kernels count in 32 bits.
int rows_at_once(int R, int per_row) {
  const long long most = 0x40000000ll / per_row / FP8_BLOCK * FP8_BLOCK;
  return R < most ? R : (int)most;
}

template <typename T, int V>
int pack_rows_v(const Fp8Step& s, cudaStream_t st) {
  const int R = s.M, C = s.N, blocks = (C + FP8_BLOCK - 1) / FP8_BLOCK, ldv = up(C, 16), most = rows_at_once(R, blocks);
  for (long long r0 = 0; r0 < R; r0 += most) {
    const int n = R - r0 < most ? (int)(R - r0) : most;
    const long long ctas = ((long long)n * blocks + ROW_THREADS / 8 - 1) / (ROW_THREADS / 8);
    rwkv_launch(fp8_pack_rows_kernel<T, V>, dim3(grid_for(ctas, 16)), dim3(ROW_THREADS), 0, st, (const T*)s.x + r0 * s.ldx, s.ldx,
                (uint8_t*)s.q_val + r0 * ldv, (uint8_t*)s.q_exp + r0, (uint32_t)n * blocks, C, ldv, up(R, 16), (uint32_t)blocks);
  }
  return rwkv_launch_status();
}
template <typename T, int V>
int pack_tiles_v(const Fp8Step* s, int count, cudaStream_t st) {
  TileJobs all = {};
  uint32_t tiles = 0;
  const auto launch = [&] {
    if (!all.count) return;
    auto kern = fp8_pack_tiles_kernel<T, V, false>;
    if constexpr (std::is_same<T, bf16>::value)           // only the products' operands come several at a time
      if (all.count > 1) kern = fp8_pack_tiles_kernel<T, V, true>;
    rwkv_launch(kern, dim3(grid_for(tiles, sizeof(T) == 4 ? 1 : 2)), dim3(TILE_THREADS), 0, st, all);
    all.count = 0;
    tiles = 0;
  };
  for (int i = 0; i < count; ++i) {
    const int R = s[i].M, C = s[i].N, blocks = (C + FP8_BLOCK - 1) / FP8_BLOCK, ldv = up(C, 16), most = rows_at_once(R, blocks);
    for (long long r0 = 0; r0 < R; r0 += most) {
      const int n = R - r0 < most ? (int)(R - r0) : most;
      const uint32_t own = (uint32_t)((n + FP8_BLOCK - 1) / FP8_BLOCK) * blocks;
      if (all.count == (std::is_same<T, bf16>::value ? MAX_JOBS : 1) || tiles + own > 0x40000000u) launch();
      tiles += own;
      all.job[all.count++] = {(const T*)s[i].x + r0 * s[i].ldx, s[i].ldx, (uint8_t*)s[i].q_val + r0 * ldv,
                              (uint8_t*)s[i].q_exp + r0 / FP8_BLOCK * blocks, n, C, ldv, (uint32_t)blocks, tiles};
    }
  }
  launch();
  rwkv_chain_restart();
  return rwkv_launch_status();
}
template <typename T>
int pack_t(const Fp8Step* s, int count, cudaStream_t st) {
  int v = 32;
  for (int i = 0; i < count; ++i) {
    const int w = access_bytes(s[i].x, s[i].ldx * (long long)sizeof(T));
    if (w < v) v = w;
  }
  const bool by_row = s[0].q_rows == 1;
  switch (v) {
    case 32: return by_row ? pack_rows_v<T, 32>(*s, st) : pack_tiles_v<T, 32>(s, count, st);
    case 16: return by_row ? pack_rows_v<T, 16>(*s, st) : pack_tiles_v<T, 16>(s, count, st);
    case 8: return by_row ? pack_rows_v<T, 8>(*s, st) : pack_tiles_v<T, 8>(s, count, st);
    case 4: return by_row ? pack_rows_v<T, 4>(*s, st) : pack_tiles_v<T, 4>(s, count, st);
    default: return by_row ? pack_rows_v<T, sizeof(T)>(*s, st) : pack_tiles_v<T, sizeof(T)>(s, count, st);
  }
}
template <typename T, int V>
int unpack_v(const uint8_t* values, const uint8_t* exps, T* y, long long ldy, int R, int C, int rows, cudaStream_t st) {
  const int ldv = up(C, 16), blocks = (C + FP8_BLOCK - 1) / FP8_BLOCK;
  const int lde = rows == 1 ? up(R, 16) : blocks;
  const int most = rows_at_once(R, blocks);
  for (long long r0 = 0; r0 < R; r0 += most) {
    const int n = R - r0 < most ? (int)(R - r0) : most;
    const long long ctas = ((long long)n * blocks + ROW_THREADS / 8 - 1) / (ROW_THREADS / 8);
    rwkv_launch(fp8_unpack_kernel<T, V>, dim3(grid_for(ctas, 32)), dim3(ROW_THREADS), 0, st, values + r0 * ldv,
                exps + (rows == 1 ? r0 : r0 / FP8_BLOCK * blocks), y + r0 * ldy, ldy, (uint32_t)n * blocks, C,
                ldv, lde, rows, (uint32_t)blocks);
  }
  return rwkv_launch_status();
}
template <typename T>
int unpack_t(const uint8_t* values, const uint8_t* exps, void* y, long long ldy, int R, int C, int rows, cudaStream_t st) {
  T* p = (T*)y;
  switch (access_bytes(y, ldy * (long long)sizeof(T))) {
    case 32: return unpack_v<T, 32>(values, exps, p, ldy, R, C, rows, st);
    case 16: return unpack_v<T, 16>(values, exps, p, ldy, R, C, rows, st);
    case 8: return unpack_v<T, 8>(values, exps, p, ldy, R, C, rows, st);
    case 4: return unpack_v<T, 4>(values, exps, p, ldy, R, C, rows, st);
    default: return unpack_v<T, sizeof(T)>(values, exps, p, ldy, R, C, rows, st);
  }
}
bool args_ok(const void* values, long long ld, int dtype, int R, int C, int rows) {
  return R > 0 && C > 0 && C <= 0x3fffff00 && ld >= C && (rows == 1 || rows == FP8_BLOCK) && dtype >= 0 && dtype <= 2 &&
         (uintptr_t)values % 16 == 0;
}

}  // namespace

// Pack: x [M, N] (row stride ldx, dtype 0 bf16, 1 fp16, 2 fp32) -> q_val [M, N rounded up to 16], q_exp as in fp8_format.cuh,
// blocks of q_rows rows.  More than one record: tiles of one type each, one launch for up to three.
int rwkv_fp8_pack(const Fp8Step* s, int count, cudaStream_t st) {
  for (int i = 0; i < count; ++i) {
    if (!args_ok(s[i].q_val, s[i].ldx, s[i].dtype, s[i].M, s[i].N, s[i].q_rows)) return RWKV_ERR_BAD_SHAPE;
    if (count > 1 && (s[i].q_rows != FP8_BLOCK || s[i].dtype != s[0].dtype)) return RWKV_ERR_BAD_SHAPE;
  }
  if (s[0].dtype == 0) return pack_t<bf16>(s, count, st);
  return s[0].dtype == 1 ? pack_t<__half>(s, count, st) : pack_t<float>(s, count, st);
}

// Unpack: the values that (a_val, a_exp) [M, N] stands for -> c (row stride ldc)
int rwkv_fp8_unpack(const Fp8Step& s, cudaStream_t st) {
  if (!args_ok(s.a_val, s.ldc, s.dtype, s.M, s.N, s.a_rows)) return RWKV_ERR_BAD_SHAPE;
  const uint8_t *v = (const uint8_t*)s.a_val, *e = (const uint8_t*)s.a_exp;
  if (s.dtype == 0) return unpack_t<bf16>(v, e, s.c, s.ldc, s.M, s.N, s.a_rows, st);
  if (s.dtype == 1) return unpack_t<__half>(v, e, s.c, s.ldc, s.M, s.N, s.a_rows, st);
  return unpack_t<float>(v, e, s.c, s.ldc, s.M, s.N, s.a_rows, st);
}
