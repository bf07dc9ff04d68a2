// dcn_fp8.h — rounding of a block to e4m3 with a power-of-two exponent (include/dcn.h, 8-bit
// pointwise products), shared by dcn_fp8.hip and dcn_fp8_gemm.hip.
#pragma once
#include "dcn_philox.h"

namespace dcn {

// largest finite magnitude so far, as bits (ordered like the values)
__device__ __forceinline__ unsigned mag_max(unsigned m, float v) {
  const unsigned u = __float_as_uint(v) & 0x7fffffffu;
  return u < 0x7f800000u ? max(m, u) : m;
}
// exponent byte of a block: smallest e >= -126 with amax <= 448 · 2^e = 1.75 · 2^(e + 8)
__device__ __forceinline__ unsigned exp_byte(unsigned amax) {
  const int e = (int)(amax >> 23) - 127 - 8 + ((amax & 0x7fffffu) > 0x600000u);
  return (unsigned)(max(e, -126) + 127);
}
// 2^-e of an exponent byte
__device__ __forceinline__ float exp_inv(unsigned byte) {
  return __uint_as_float((254u - byte) << 23);
}
// four values to four bytes; an infinity becomes NaN like a NaN itself
__device__ __forceinline__ unsigned to_fp8x4(float a, float b, float c, float d) {
  int q = 0;
  q = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, q, false);
  q = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, q, true);
  return (unsigned)q;
}

}  // namespace dcn
