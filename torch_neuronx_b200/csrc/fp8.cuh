// 8-bit cached rows: e4m3 values and the biased exponent of a power of two for each row (cache_rows.cu has the format).
#pragma once

#include "common.cuh"
#include "report.cuh"

namespace b200 {

// Biased exponent of the least power of two 2^e with top <= 448 * 2^e (448 = 1.75 * 2^8), from the bits of the row's
// largest magnitude: 127 (e = 0) for zero, 255 (NaN) for an infinity or NaN, never below 0 (e = -127).
__device__ __forceinline__ int scale_code(uint32_t top_bits) {
  if (top_bits == 0u) return 127;
  if (top_bits >= 0x7f800000u) return 255;
  const int code = static_cast<int>(top_bits >> 23) - ((top_bits & 0x7fffffu) <= 0x600000u ? 8 : 7);
  return code < 0 ? 0 : code;
}
// 2^-e and 2^e of a code; NaN for 255.
__device__ __forceinline__ float scale_inverse(int code) {
  return code == 255 ? CUDART_NAN_F : __int_as_float((254 - code) << 23);   // (codes written here are at most 247)
}
__device__ __forceinline__ float scale_value(int code) {
  return code == 255 ? CUDART_NAN_F : __int_as_float(code == 0 ? 1 << 22 : code << 23);
}

// Two fp32 values rounded to e4m3, the first in the low byte.
__device__ __forceinline__ uint32_t pack_e4m3(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Four e4m3 values as two fp16 pairs (exact).
__device__ __forceinline__ void unpack_e4m3_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t"
      ".reg .b16 a, b;\n\t"
      "mov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n\t"
      "}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
__device__ __forceinline__ void unpack_e4m3x4(uint32_t w, float (&f)[4]) {
  uint32_t lo, hi;
  unpack_e4m3_f16(w, lo, hi);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  f[0] = a.x;
  f[1] = a.y;
  f[2] = b.x;
  f[3] = b.y;
}

template <bool BF16> __device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if (BF16) {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  } else {
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  }
  return r;
}
template <bool BF16> __device__ __forceinline__ float half_to_f32(uint16_t x) {
  if (BF16) return __uint_as_float(static_cast<uint32_t>(x) << 16);
  return __half2float(__ushort_as_half(x));
}

__device__ __forceinline__ uint4 ld_stream_16B(const void* ptr) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(ptr));
  return r;
}

}  // namespace b200
