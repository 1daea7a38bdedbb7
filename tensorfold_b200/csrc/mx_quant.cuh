// Rounding to microscaled 4-bit floating point: what the quantising kernels and the epilogues share.
//
// A block of 32 values with largest magnitude a has the scale 2^(floor(log2 a) - 2), 2 being the largest exponent of e2m1 (OCP
// microscaling formats, conversion with the shared exponent of the largest value).  In bits: the scale's biased exponent is a's
// less 2, clamped at 0; the values times 2^(127 - code) are exact, below 8 in magnitude, and are rounded to nearest even onto
// 0, 0.5, 1, 1.5, 2, 3, 4, 6 with saturation, which is what the conversion instruction does.  A block that holds an infinity
// or a NaN gets the scale code 255, a NaN, and zero codes.
#pragma once

#include <stdint.h>

namespace tf {

// Eight values to eight codes, the first in the low bits.
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n.reg .b8 a, b, c, d;\n"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\ncvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\ncvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
      "mov.b32 %0, {a, b, c, d};\n}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// Four neighbouring lanes hold a block, eight values each (all lanes of the warp call): this lane's codes, and the block's scale.
__device__ __forceinline__ uint32_t quantize_block(float (&v)[8], uint32_t& scale) {
  uint32_t top = 0;                                          // magnitudes compare as integers, NaN above infinity
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
  top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
  // no branch: several blocks in one thread would run one after another
  const bool bad = top >= 0x7F800000u;
  const int e = static_cast<int>(top >> 23);
  scale = bad ? 255u : static_cast<uint32_t>(max(e - 2, 0));
  const float inverse = __uint_as_float((254u - min(scale, 254u)) << 23);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= inverse;
  const uint32_t codes = e2m1x8(v);
  return bad ? 0u : codes;
}

__device__ __forceinline__ void widen8(uint4 p, float (&v)[8]) {
  const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
}

// The same from eight bf16 values as they lie in memory: their magnitudes compare two at a time as 16-bit integers.
__device__ __forceinline__ uint32_t quantize_block(uint4 p, uint32_t& scale) {
  constexpr uint32_t MAGNITUDE = 0x7FFF7FFFu;
  uint32_t m = __vmaxu2(__vmaxu2(p.x & MAGNITUDE, p.y & MAGNITUDE), __vmaxu2(p.z & MAGNITUDE, p.w & MAGNITUDE));
  m = __vmaxu2(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
  m = __vmaxu2(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
  const uint32_t top = max(m >> 16, m & 0xFFFFu);
  const bool bad = top >= 0x7F80u;
  scale = bad ? 255u : static_cast<uint32_t>(max(static_cast<int>(top >> 7) - 2, 0));
  const float inverse = __uint_as_float((254u - min(scale, 254u)) << 23);
  float v[8];
  widen8(p, v);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= inverse;
  const uint32_t codes = e2m1x8(v);
  return bad ? 0u : codes;
}

}  // namespace tf
