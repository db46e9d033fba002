// Shared pieces of the kernels over an 8-bit KV cache (fp8_write.cu,
// fp8_decode.cu, fp8_prefill.cu).
//
// The cache holds float8 e4m3 codes, [num_blocks, KH, BS, D] for the keys and
// the values, and kv_scale float32 [num_blocks, KH, 2]: the scale of the keys
// and the scale of the values of each (block, KV head).  An element stands for
// code * scale.  Every e4m3 value is exact in f16 (4 exponent and 3 mantissa
// bits against 5 and 10), so the attention kernels feed the codes to f16
// tensor-core products and apply the scales to the 32-bit results.
#pragma once

#include <cuda_fp8.h>

#include "mvb_common.cuh"

namespace mvb {

constexpr float kFp8Max = 448.f;       // largest e4m3 value
constexpr int kFp8MinScaleExp = -100;  // the smallest scale is 2^-100 (a block of zeros)
constexpr int kFp8MinBlock = 16;       // tokens of the smallest block: a 16-token tile lies in one block
constexpr int kFp8MaxBlock = 1024;

// The smallest power of two s >= 2^-100 with amax <= 448 s, for a finite amax >= 0:
// amax = f * 2^e with 1 <= f < 2 and 448 = 1.75 * 2^8.
__host__ __device__ __forceinline__ float fp8_scale_for(float amax) {
#ifdef __CUDA_ARCH__
  const uint32_t u = __float_as_uint(amax);
#else
  union { float f; uint32_t u; } cv;
  cv.f = amax;
  const uint32_t u = cv.u;
#endif
  int e = (int)(u >> 23) - 127 - 8;                // a subnormal amax gives -135: clamped below
  if ((u & 0x7fffffu) > 0x600000u) e += 1;         // f > 1.75
  if (e < kFp8MinScaleExp) e = kFp8MinScaleExp;
  const uint32_t r = (uint32_t)(e + 127) << 23;
#ifdef __CUDA_ARCH__
  return __uint_as_float(r);
#else
  cv.u = r;
  return cv.f;
#endif
}

// Four codes (one word) as two f16 pairs.
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
// Four floats as four codes (first in the low byte), rounded to nearest even;
// beyond +-448 the largest code, NaN the NaN code.
__device__ __forceinline__ uint32_t f32x4_to_e4m3(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
      "mov.b32 %0, {lo, hi};\n\t}"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}

}  // namespace mvb
