// The record that describes one launch of an 8-bit operator to rwkv_fp8_run (the host side packs it field by field).
#pragma once
#include "common.cuh"

enum Fp8StepKind : int { FP8_STEP_PACK = 0, FP8_STEP_UNPACK = 1, FP8_STEP_GEMM = 2, FP8_STEP_DECODE = 3 };

struct Fp8Step {
  int kind;
  int M, N, K;               // pack, unpack: M rows, N columns
  int a_rows, q_rows;        // rows of a block of A (unpack: of the input) and of the packed result
  int dtype;                 // pack, unpack: type of the plain side (0 bf16, 1 fp16, 2 fp32)
  int a_mn, b_mn, epilogue;  // gemm: see gemm_fp8_tcgen05.cu
  int chained;               // decode: may start before its predecessor has finished (see gemm_fp8_decode.cu)
  int with_next;             // gemm: this record and the next are one launch
  long long ldx, ldc, ldr;   // row strides of x (pack), c and the residual
  const void* x;
  const void *a_val, *a_exp, *b_val, *b_exp;
  void* c;
  const void* residual;
  const void *h_val, *h_exp;
  void *q_val, *q_exp;
  void* workspace;           // gemm: see gemm_fp8_tcgen05.cu
  void* status;
};

int rwkv_fp8_pack(const Fp8Step* s, int count, cudaStream_t stream);
int rwkv_fp8_unpack(const Fp8Step& s, cudaStream_t stream);
int rwkv_fp8_gemm(const Fp8Step& s, cudaStream_t stream);
int rwkv_fp8_gemm_two(const Fp8Step& s, const Fp8Step& t, cudaStream_t stream);
int rwkv_fp8_decode(const Fp8Step& s, cudaStream_t stream);
