// The 8-bit K/V cache: e4m3 codes with one FP32 power-of-two scale per (block of 64 slots, head). Shared by the store
// (kv8.cu) and the attention that reads it (kv8_attention.cu).
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace morj {
namespace kv8 {

constexpr int BLOCK = 64;            // slots that share a scale
constexpr int BLOCK_SHIFT = 6;
constexpr int MIN_EXP = -100;        // the smallest scale is 2^-100

// the two e4m3 codes in the low half of `two` (low byte first) as FP16 values; exact (e4m3's range and precision lie inside FP16's)
MORJ_DEV uint32_t codes2_f16(uint32_t two) {
  uint32_t r;
  asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(r) : "r"(two));
  return r;
}
MORJ_DEV float2 codes2_f32(uint32_t two) {
  const uint32_t h = codes2_f16(two);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// two FP32 values as e4m3 codes (round to nearest even, saturated), `lo` in the low byte
MORJ_DEV uint32_t f32_codes2(float lo, float hi) {
  uint32_t r;
  asm("{\n\t.reg .b16 t;\n\tcvt.rn.satfinite.e4m3x2.f32 t, %2, %1;\n\tcvt.u32.u16 %0, t;\n\t}"
      : "=r"(r)
      : "f"(lo), "f"(hi));
  return r;
}
MORJ_DEV float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // 2^e, -126 <= e <= 127

// The smallest power of two s >= 2^MIN_EXP with a <= 448 s. a finite, >= 0: a = m 2^x with m in [1, 2), 448 = 1.75 * 2^8.
MORJ_DEV float scale_for(float a) {
  const uint32_t bits = __float_as_uint(a);
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);
  return exp2_int(e < MIN_EXP ? MIN_EXP : e);
}

}  // namespace kv8
}  // namespace morj
