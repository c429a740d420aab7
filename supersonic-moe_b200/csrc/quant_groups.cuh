// A group's scale and payload, as every row quantiser here makes them.
#pragma once
#include <stdint.h>

namespace smoe {

// ---- 1x32, powers of two (rule: see quant.cu)
__device__ __forceinline__ int q_e8m0_of(float amax) {
  const int bits = __float_as_int(amax);
  const int bexp = (bits >> 23) & 0xFF;
  const int e = bexp - 8 + ((bits & 0x7FFFFF) > 0x600000 ? 1 : 0);
  return bexp > 0 ? max(e, 0) : 0;
}
__device__ __forceinline__ float q_scale_of(int e8m0) {
  return __int_as_float(min(max(254 - e8m0, 1), 254) << 23);
}
__device__ __forceinline__ uint32_t q_pack4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}
__device__ __forceinline__ void bf16x8_to_f32(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}

// larger of two pairs of bf16, a number before a NaN
__device__ __forceinline__ uint32_t q_max_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// max of the magnitudes of two bf16 pairs, element by element; the sign bits are those of the product
__device__ __forceinline__ uint32_t q_max_abs_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// A bf16 pair times a pair of powers of two, in f32: exact, one instruction a value where unpacking and multiplying take two, and
// on another pipe than the conversions; adding -0 keeps the sign of a zero
__device__ __forceinline__ float2 q_scaled(uint32_t w, uint32_t qs) {
  float2 r;
  asm("{\n\t.reg .b16 a, b, c, d;\n\t"
      "mov.b32 {a, b}, %2;\n\tmov.b32 {c, d}, %3;\n\t"
      "fma.rn.f32.bf16 %0, a, c, %4;\n\tfma.rn.f32.bf16 %1, b, d, %4;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "r"(w), "r"(qs), "f"(-0.0f));
  return r;
}
// four bf16 values of a row, each with its scale -> four e4m3 bytes
__device__ __forceinline__ uint32_t q_pack4_scaled(uint32_t a, uint32_t b, uint32_t qa, uint32_t qb) {
  const float2 x = q_scaled(a, qa), y = q_scaled(b, qb);
  return q_pack4(x.x, x.y, y.x, y.y);
}
__device__ __forceinline__ uint32_t q_bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// ---- 1x128, f32 (rule: see quant128.cu)
constexpr float kE4m3Max = 448.f;
constexpr float kAmaxFloor = 7.888609052210118e-31f;      // 2^-100: 448 / a stays finite, a / 448 normal

}  // namespace smoe
