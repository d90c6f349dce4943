// The packed form's element codes made on the device from float32: the formats, a block's scale byte (floor(log2
// amax) - emax by the exponent field) and the rounding of two values to two codes by sm_100's conversions.
#pragma once
#include <stdint.h>

namespace mxq {

enum { kFmtE4M3 = 0, kFmtE5M2, kFmtE3M2, kFmtE2M3, kFmtE2M1, kFmtNone = -1 };

inline int format_of(int e, int m) {
  if (e == 4 && m == 3) return kFmtE4M3;
  if (e == 5 && m == 2) return kFmtE5M2;
  if (e == 3 && m == 2) return kFmtE3M2;
  if (e == 2 && m == 3) return kFmtE2M3;
  if (e == 2 && m == 1) return kFmtE2M1;
  return kFmtNone;
}

__device__ __forceinline__ int emax_of(int fmt) { return fmt == kFmtE4M3 ? 8 : fmt == kFmtE5M2 ? 15 : fmt == kFmtE3M2 ? 4 : 2; }

// The scale byte of a block whose largest |value| has these bits: floor(log2) - emax by the exponent field (a
// subnormal or zero block gets the lowest scale), 0xFF (NaN) when the block holds an Inf or a NaN.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits, int fmt) {
  const int ex = (int)(amax_bits >> 23);
  if (ex == 255) return 255u;
  const int b = ex - emax_of(fmt);
  return (uint32_t)(b < 0 ? 0 : b);
}
// 2^(127 - byte), exact; 0 for a NaN block, whose codes are then zeros
__device__ __forceinline__ float scale_inverse(uint32_t byte) {
  if (byte == 255u) return 0.0f;
  const uint32_t e = 254u - byte;
  return __uint_as_float(e == 0u ? 0x00400000u : e << 23);
}
__device__ __forceinline__ float scaled(float v, float inv) { return inv == 0.0f ? 0.0f : __fmul_rn(v, inv); }

// two values -> two codes (round to nearest even, saturating), the first in the low byte; FP4: in the low nibble
__device__ __forceinline__ uint32_t encode2(int fmt, float lo, float hi) {
  uint16_t q;
  switch (fmt) {
    case kFmtE4M3: asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(q) : "f"(hi), "f"(lo)); break;
    case kFmtE5M2: asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(q) : "f"(hi), "f"(lo)); break;
    case kFmtE3M2: asm("cvt.rn.satfinite.e3m2x2.f32 %0, %1, %2;" : "=h"(q) : "f"(hi), "f"(lo)); break;
    case kFmtE2M3: asm("cvt.rn.satfinite.e2m3x2.f32 %0, %1, %2;" : "=h"(q) : "f"(hi), "f"(lo)); break;
    default:
      asm("{\n .reg .b8 t;\n cvt.rn.satfinite.e2m1x2.f32 t, %1, %2;\n cvt.u16.u8 %0, t;\n}" : "=h"(q) : "f"(hi), "f"(lo));
  }
  return q;
}

// two FP6 or FP4 codes (the first in the low byte) as the E4M3 codes of the same values, exactly: 8-bit E4M3 holds
// every value of the smaller grids
__device__ __forceinline__ uint32_t widen2(int fmt, uint32_t codes) {
  uint32_t h;
  const uint16_t c = (uint16_t)codes;
  if (fmt == kFmtE3M2)
    asm("cvt.rn.f16x2.e3m2x2 %0, %1;" : "=r"(h) : "h"(c));
  else if (fmt == kFmtE2M3)
    asm("cvt.rn.f16x2.e2m3x2 %0, %1;" : "=r"(h) : "h"(c));
  else                                                       // both nibbles of one byte
    asm("{\n .reg .b8 t;\n cvt.u8.u16 t, %1;\n cvt.rn.f16x2.e2m1x2 %0, t;\n}" : "=r"(h) : "h"(c));
  uint16_t q;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(q) : "r"(h));
  return q;
}

}  // namespace mxq
