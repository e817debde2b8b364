// One library call for the launches of an 8-bit operator.  A forward or backward pass is three to six kernels of a few
// microseconds on small batches, and a foreign call with twenty arguments costs about as much as a launch; the host side
// therefore describes the launches in one array of plain records.
#include "fp8_steps.cuh"

// Runs `count` steps in order on `stream`; returns the status of the first that was refused or failed to launch.
RWKV_EXPORT int rwkv_fp8_run(const Fp8Step* steps, int count, void* stream) {
  if (count < 0 || (count > 0 && !steps)) return RWKV_ERR_BAD_SHAPE;
  for (int i = 0; i < count; ++i) {
    const Fp8Step& s = steps[i];
    int r = RWKV_ERR_BAD_SHAPE;
    switch (s.kind) {
      case FP8_STEP_PACK: {                   // tiles of one type that follow one another go out together
        int n = 1;
        while (s.q_rows == 128 && i + n < count && steps[i + n].kind == FP8_STEP_PACK && steps[i + n].q_rows == 128 &&
               steps[i + n].dtype == s.dtype)
          ++n;
        r = rwkv_fp8_pack(steps + i, n, (cudaStream_t)stream);
        i += n - 1;
        break;
      }
      case FP8_STEP_UNPACK: r = rwkv_fp8_unpack(s, (cudaStream_t)stream); break;
      case FP8_STEP_GEMM:
        if (!s.with_next) {
          r = rwkv_fp8_gemm(s, (cudaStream_t)stream);
        } else if (i + 1 < count && steps[i + 1].kind == FP8_STEP_GEMM) {
          r = rwkv_fp8_gemm_two(s, steps[++i], (cudaStream_t)stream);
        }
        break;
      case FP8_STEP_DECODE: r = rwkv_fp8_decode(s, (cudaStream_t)stream); break;
      default: break;
    }
    if (r) return r;
  }
  return RWKV_OK;
}
