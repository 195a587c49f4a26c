// The 4-bit cache format: E2M1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), two to a byte (the even element in
// the low nibble), with one E4M3 scale for every 16 consecutive values of a row.
//
// A value times its scale has at most 6 significant bits (2 + 4) and lies between 2^-10 and 2 688, so FP16 holds
// every product exactly, subnormal scales included: widening a cache to FP16 loses nothing.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

namespace atrex_sm100 {

constexpr int kFp4Block = 16;   // values per E4M3 scale

// Four bytes (eight values) -> four FP16 pairs, low nibble in the low half.
__device__ __forceinline__ void e2m1x8_to_f16x2(uint32_t word, uint32_t (&out)[4]) {
  asm("{\n"
      ".reg .b8 b0, b1, b2, b3;\n"
      "mov.b32 {b0, b1, b2, b3}, %4;\n"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n"
      "}\n"
      : "=r"(out[0]), "=r"(out[1]), "=r"(out[2]), "=r"(out[3])
      : "r"(word));
}
// Two E4M3 bytes (low 16 bits of `pair`) -> an FP16 pair.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t pair) {
  uint32_t d;
  asm("{\n"
      ".reg .b16 lo, hi;\n"
      "mov.b32 {lo, hi}, %1;\n"
      "cvt.rn.f16x2.e4m3x2 %0, lo;\n"
      "}\n"
      : "=r"(d)
      : "r"(pair));
  return d;
}
// Eight FP32 -> eight E2M1 codes, round to nearest even, saturating at 6 (a NaN becomes +6: the format has no NaN).
__device__ __forceinline__ uint32_t f32x8_to_e2m1(const float (&x)[8]) {
  uint32_t d;
  asm("{\n"
      ".reg .b8 b0, b1, b2, b3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
      "mov.b32 %0, {b0, b1, b2, b3};\n"
      "}\n"
      : "=r"(d)
      : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]));
  return d;
}
__device__ __forceinline__ uint32_t hmul2_u32(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// a times the low / high half of b (the instruction broadcasts a half by itself).
__device__ __forceinline__ uint32_t hmul2_low(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), __low2half2(*reinterpret_cast<const __half2*>(&b)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hmul2_high(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), __high2half2(*reinterpret_cast<const __half2*>(&b)));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// A query row scaled into FP16's range: the power of two that brings the row's largest element (BF16 magnitude bits
// `top`) to 2^13 .. 2^14, and its inverse, which joins the row's score factor.
__device__ __forceinline__ void row_power(uint32_t top, float& up, float& down) {
  const int e = top == 0u ? 127 : min(254, max(1, 267 - (int)(top >> 7)));
  up = __int_as_float(e << 23);
  down = e == 254 ? 0x1p-127f : __int_as_float((254 - e) << 23);
}
// Score factor of a row: positive (a negative scale goes into the sign of Q) and never zero, so that a masked score
// stays -inf when it is multiplied by it.  A NaN stays, and makes the scores of the row NaN, unless the row sees no key: it
// is empty whatever its scale.  `sees_keys` is asked about NaN scales only (the decode kernel pays 1 - 2 % for asking always).
template <typename SeesKeys>
__device__ __forceinline__ float score_factor(float scale, const SeesKeys& sees_keys) {
  if (scale != scale && !sees_keys()) scale = 0.f;
  const float a = fabsf(scale);
  return a < 1.2e-38f ? 1.2e-38f : a;
}

}  // namespace atrex_sm100
