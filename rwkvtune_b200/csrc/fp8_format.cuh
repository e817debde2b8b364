// The 8-bit block format shared by the packing kernels and the 8-bit GEMMs.
//
// A matrix [R, C] is held as e4m3 bytes, row-major with a leading dimension of C rounded up to 16 (so that every row can be
// the start of a TMA copy), and one exponent byte E per block: the block's values are e4m3 * 2^(E - 127).  E is the smallest
// non-negative byte with  max|x| <= 448 * 2^(E - 127).  A block that holds an infinity or a NaN gets E = 255 (the NaN of the
// E8M0 scale type of the tensor cores) and NaN bytes: it reads back as NaN and so does every product it takes part in.
//   rows = 1  : a block is 128 columns of one row.  Exponents are stored [ceil(C / 128)][R rounded up to 16]: the bytes of
//               neighbouring rows are neighbours, which is how the GEMM gathers them.
//   rows = 128: a block is a tile of 128 x 128.  Exponents are stored [ceil(R / 128)][ceil(C / 128)].
// Power-of-two scales make packing exact apart from the one rounding to e4m3, and they are what the tensor cores apply
// themselves while they multiply; with a scale found by division each value would be rounded twice.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

constexpr int FP8_BLOCK = 128;

// exponent byte of a block from the largest bit pattern of |x| in it (as fp32; NaN > infinity > finite)
__device__ __forceinline__ uint32_t fp8_block_exponent(uint32_t max_bits) {
  if (max_bits >= 0x7f800000u) return 255u;
  // max|x| = 1.m * 2^(f - 127) <= 1.75 * 2^8 * 2^(E - 127)
  const int e = (int)(max_bits >> 23) - 8 + ((max_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e > 0 ? (uint32_t)e : 0u;
}
// 2^(127 - E) for E <= 247 (the largest a finite block has): a normal number
__device__ __forceinline__ float fp8_inverse_scale(uint32_t e) { return __uint_as_float((254u - e) << 23); }
// q * 2^(E - 127) in two exact factors, each a normal number for every E (2^-127 alone would be flushed to zero)
__device__ __forceinline__ float fp8_scaled(float q, uint32_t e) {
  const uint32_t half = e >> 1;
  return q * __uint_as_float((half + 64u) << 23) * __uint_as_float((e - half + 63u) << 23);
}
// four fp32 values -> four e4m3 bytes, round to nearest even
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(lo) : "f"(a), "f"(b));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(hi) : "f"(c), "f"(d));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}
__device__ __forceinline__ void fp8_unpack4(uint32_t p, float* f) {
  uint32_t lo, hi;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"((uint16_t)(p & 0xffffu)));
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"((uint16_t)(p >> 16)));
  const float2 a = __half22float2(*reinterpret_cast<__half2*>(&lo)), b = __half22float2(*reinterpret_cast<__half2*>(&hi));
  f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
}
