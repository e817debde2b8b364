// Packing to and from the 8-bit block format (fp8_format.cuh): activation checkpoints, and the operands of the 8-bit GEMMs.
//
// Both directions are bound by memory: 2 + 1 bytes a value for bf16.  A thread owns 16 neighbouring values (two 16-byte
// loads, one 16-byte store for bf16), eight threads a block of 128 columns.  The values stay in registers between the
// maximum and the rounding, so the input is read once:
//   rows = 1  : the maximum is three shuffles among the eight threads of a block;
//   rows = 128: a CTA of 512 threads owns a tile, 32 values a thread; warp maxima meet in shared memory.
// Loads and stores take the widest of 16 / 8 / 4 / 2 bytes that the row pitch and the address allow.
//
// Arithmetic in the rest of the library flushes numbers below 2^-126 to zero, and so do these kernels.
#include <cuda_fp16.h>

#include "fp8_format.cuh"

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

template <int BYTES> struct Word;
template <> struct Word<2> { typedef uint16_t type; };
template <> struct Word<4> { typedef uint32_t type; };
template <> struct Word<8> { typedef uint2 type; };
template <> struct Word<16> { typedef uint4 type; };

// 16 values from p, the first n of them in range (n may be <= 0 or above 16); V: bytes of one load
template <typename T, int V>
__device__ __forceinline__ void load16(const T* p, int n, float* f) {
  constexpr int PER = V / (int)sizeof(T);
  union { typename Word<V>::type w[16 / PER]; T t[16]; } u;
#pragma unroll
  for (int i = 0; i < 16 / PER; ++i) {
    if ((i + 1) * PER <= n) {
      u.w[i] = __ldcs(reinterpret_cast<const typename Word<V>::type*>(p) + i);
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j) u.t[i * PER + j] = i * PER + j < n ? p[i * PER + j] : from_f32<T>(0.f);
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) f[i] = to_f32(u.t[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store16(T* p, int n, const float* f) {
  constexpr int PER = V / (int)sizeof(T);
  union { typename Word<V>::type w[16 / PER]; T t[16]; } u;
#pragma unroll
  for (int i = 0; i < 16; ++i) u.t[i] = from_f32<T>(f[i]);
#pragma unroll
  for (int i = 0; i < 16 / PER; ++i) {
    if ((i + 1) * PER <= n) {
      reinterpret_cast<typename Word<V>::type*>(p)[i] = u.w[i];
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (i * PER + j < n) p[i * PER + j] = u.t[i * PER + j];
    }
  }
}

__device__ __forceinline__ uint32_t abs_bits16(const float* f) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
  return m;
}
__device__ __forceinline__ uint4 quantise16(const float* f, uint32_t e) {
  if (e == 255u) return make_uint4(0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu);
  const float s = fp8_inverse_scale(e);
  return make_uint4(fp8_pack4(f[0] * s, f[1] * s, f[2] * s, f[3] * s), fp8_pack4(f[4] * s, f[5] * s, f[6] * s, f[7] * s),
                    fp8_pack4(f[8] * s, f[9] * s, f[10] * s, f[11] * s), fp8_pack4(f[12] * s, f[13] * s, f[14] * s, f[15] * s));
}

constexpr int ROW_THREADS = 256;

template <typename T, int V>
__global__ void __launch_bounds__(ROW_THREADS)
fp8_pack_rows_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ values, uint8_t* __restrict__ exps,
                     int R, int C, int ldv, int lde, int blocks) {
  rwkv_chain_trigger();       // a chained decode product may fetch its weights meanwhile
  const long long units = (long long)R * blocks, stride = (long long)gridDim.x * (ROW_THREADS / 8);
  const int part = threadIdx.x & 7;
  const long long rounds = (units + stride - 1) / stride;          // the same for every thread: the shuffles need whole warps
  long long u = (long long)blockIdx.x * (ROW_THREADS / 8) + (threadIdx.x >> 3);
  for (long long i = 0; i < rounds; ++i, u += stride) {
    const bool live = u < units;
    const int row = live ? (int)(u / blocks) : 0, kb = live ? (int)(u % blocks) : 0;
    const int col = kb * FP8_BLOCK + part * 16;
    float f[16];
    load16<T, V>(x + row * ldx + col, live ? C - col : 0, f);
    uint32_t m = abs_bits16(f);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const uint32_t e = fp8_block_exponent(m);
    if (live) {
      if (col < ldv) *reinterpret_cast<uint4*>(values + (long long)row * ldv + col) = quantise16(f, e);
      if (part == 0) exps[(long long)kb * lde + row] = (uint8_t)e;
    }
  }
}

constexpr int TILE_THREADS = 512;

template <typename T, int V>
__global__ void __launch_bounds__(TILE_THREADS)
fp8_pack_tiles_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ values, uint8_t* __restrict__ exps,
                      int R, int C, int ldv, int blocks) {
  __shared__ uint32_t warp_max[TILE_THREADS / 32];
  const int rb = (int)(blockIdx.x / blocks), kb = (int)(blockIdx.x % blocks);
  const int col = kb * FP8_BLOCK + (threadIdx.x & 7) * 16;
  const int row0 = rb * FP8_BLOCK + (threadIdx.x >> 3);
  float f[2][16];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = row0 + i * (TILE_THREADS / 8);
    load16<T, V>(x + (long long)min(row, R - 1) * ldx + col, row < R ? C - col : 0, f[i]);
  }
  uint32_t m = max(abs_bits16(f[0]), abs_bits16(f[1]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
  __syncthreads();
  m = warp_max[threadIdx.x & (TILE_THREADS / 32 - 1)];
#pragma unroll
  for (int o = TILE_THREADS / 64; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  const uint32_t e = fp8_block_exponent(m);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = row0 + i * (TILE_THREADS / 8);
    if (row < R && col < ldv) *reinterpret_cast<uint4*>(values + (long long)row * ldv + col) = quantise16(f[i], e);
  }
  if (threadIdx.x == 0) exps[blockIdx.x] = (uint8_t)e;
}

template <typename T, int V>
__global__ void __launch_bounds__(ROW_THREADS)
fp8_unpack_kernel(const uint8_t* __restrict__ values, const uint8_t* __restrict__ exps, T* __restrict__ y, long long ldy,
                  int R, int C, int ldv, int lde, int rows, int chunks) {
  const long long units = (long long)R * chunks, stride = (long long)gridDim.x * ROW_THREADS;
  for (long long u = (long long)blockIdx.x * ROW_THREADS + threadIdx.x; u < units; u += stride) {
    const int row = (int)(u / chunks), col = (int)(u % chunks) * 16, kb = col / FP8_BLOCK;
    const uint4 q = __ldcs(reinterpret_cast<const uint4*>(values + (long long)row * ldv + col));
    const uint32_t e = rows == 1 ? exps[(long long)kb * lde + row] : exps[(long long)(row / FP8_BLOCK) * lde + kb];
    float f[16];
    fp8_unpack4(q.x, f); fp8_unpack4(q.y, f + 4); fp8_unpack4(q.z, f + 8); fp8_unpack4(q.w, f + 12);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      f[i] = fp8_scaled(f[i], e);
      if (e < 255u) f[i] = fminf(fmaxf(f[i], -largest<T>()), largest<T>());
    }
    store16<T, V>(y + row * ldy + col, C - col, f);
  }
}

// widest access that every row start allows
int access_bytes(const void* p, long long pitch_bytes, int elem) {
  for (int v = 16; v > elem; v /= 2)
    if ((uintptr_t)p % v == 0 && pitch_bytes % v == 0) return v;
  return elem;
}
unsigned grid_for(long long ctas) { return (unsigned)(ctas < 148 * 8 * 4 ? ctas : 148 * 8 * 4); }

template <typename T, int V>
int pack_v(const void* x, long long ld, uint8_t* values, uint8_t* exps, int R, int C, int rows, cudaStream_t st) {
  const int blocks = (C + FP8_BLOCK - 1) / FP8_BLOCK, ldv = (C + 15) / 16 * 16;
  if (rows == 1) {
    const int lde = (R + 15) / 16 * 16;
    const long long ctas = ((long long)R * blocks + ROW_THREADS / 8 - 1) / (ROW_THREADS / 8);
    fp8_pack_rows_kernel<T, V><<<grid_for(ctas), ROW_THREADS, 0, st>>>((const T*)x, ld, values, exps, R, C, ldv, lde, blocks);
  } else {
    const long long tiles = (long long)((R + FP8_BLOCK - 1) / FP8_BLOCK) * blocks;
    if (tiles > 0x7fffffffll) return RWKV_ERR_TOO_LARGE;
    fp8_pack_tiles_kernel<T, V><<<(unsigned)tiles, TILE_THREADS, 0, st>>>((const T*)x, ld, values, exps, R, C, ldv, blocks);
  }
  return rwkv_launch_status();
}
template <typename T>
int pack_t(const void* x, long long ld, uint8_t* values, uint8_t* exps, int R, int C, int rows, cudaStream_t st) {
  switch (access_bytes(x, ld * (long long)sizeof(T), sizeof(T))) {
    case 16: return pack_v<T, 16>(x, ld, values, exps, R, C, rows, st);
    case 8: return pack_v<T, 8>(x, ld, values, exps, R, C, rows, st);
    case 4: return pack_v<T, 4>(x, ld, values, exps, R, C, rows, st);
    default: return pack_v<T, sizeof(T)>(x, ld, values, exps, R, C, rows, st);
  }
}
template <typename T, int V>
int unpack_v(const uint8_t* values, const uint8_t* exps, void* y, long long ldy, int R, int C, int rows, cudaStream_t st) {
  const int ldv = (C + 15) / 16 * 16, chunks = ldv / 16;
  const int lde = rows == 1 ? (R + 15) / 16 * 16 : (C + FP8_BLOCK - 1) / FP8_BLOCK;
  const long long ctas = ((long long)R * chunks + ROW_THREADS - 1) / ROW_THREADS;
  fp8_unpack_kernel<T, V><<<grid_for(ctas), ROW_THREADS, 0, st>>>(values, exps, (T*)y, ldy, R, C, ldv, lde, rows, chunks);
  return rwkv_launch_status();
}
template <typename T>
int unpack_t(const uint8_t* values, const uint8_t* exps, void* y, long long ldy, int R, int C, int rows, cudaStream_t st) {
  switch (access_bytes(y, ldy * (long long)sizeof(T), sizeof(T))) {
    case 16: return unpack_v<T, 16>(values, exps, y, ldy, R, C, rows, st);
    case 8: return unpack_v<T, 8>(values, exps, y, ldy, R, C, rows, st);
    case 4: return unpack_v<T, 4>(values, exps, y, ldy, R, C, rows, st);
    default: return unpack_v<T, sizeof(T)>(values, exps, y, ldy, R, C, rows, st);
  }
}
bool args_ok(const void* values, long long ld, int dtype, int R, int C, int rows) {
  return R > 0 && C > 0 && C <= 0x7fffff00 && ld >= C && (rows == 1 || rows == FP8_BLOCK) && dtype >= 0 && dtype <= 2 &&
         (uintptr_t)values % 16 == 0;
}

}  // namespace

// x [R, C] (row stride ldx, dtype 0 bf16, 1 fp16, 2 fp32) -> values [R, C rounded up to 16], exponents as in fp8_format.cuh
RWKV_EXPORT int rwkv_fp8_pack(const void* x, int dtype, long long ldx, void* values, void* exps, int R, int C, int rows,
                              void* stream) {
  if (!args_ok(values, ldx, dtype, R, C, rows)) return RWKV_ERR_BAD_SHAPE;
  cudaStream_t st = (cudaStream_t)stream;
  uint8_t *v = (uint8_t*)values, *e = (uint8_t*)exps;
  if (dtype == 0) return pack_t<bf16>(x, ldx, v, e, R, C, rows, st);
  if (dtype == 1) return pack_t<__half>(x, ldx, v, e, R, C, rows, st);
  return pack_t<float>(x, ldx, v, e, R, C, rows, st);
}

// the values a packed matrix stands for, y [R, C] (row stride ldy)
RWKV_EXPORT int rwkv_fp8_unpack(const void* values, const void* exps, void* y, int dtype, long long ldy, int R, int C, int rows,
                                void* stream) {
  if (!args_ok(values, ldy, dtype, R, C, rows)) return RWKV_ERR_BAD_SHAPE;
  cudaStream_t st = (cudaStream_t)stream;
  const uint8_t *v = (const uint8_t*)values, *e = (const uint8_t*)exps;
  if (dtype == 0) return unpack_t<bf16>(v, e, y, ldy, R, C, rows, st);
  if (dtype == 1) return unpack_t<__half>(v, e, y, ldy, R, C, rows, st);
  return unpack_t<float>(v, e, y, ldy, R, C, rows, st);
}
