// dcn_fp8.h — rounding of a block to e4m3 with a power-of-two exponent (include/dcn.h, 8-bit
// pointwise products), shared by dcn_fp8.hip and dcn_fp8_gemm.hip.
#pragma once
#include "dcn_philox.h"

namespace dcn {

// Largest finite magnitudes. fp32 values count as their 31 magnitude bits, which are ordered like
// the values; bf16 values as pairs of 15 bits, two to an instruction. Non-finite ones are rare:
// the maxima are taken with them first and again without (CLEAN) where one turned up.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ unsigned max2(unsigned a, unsigned b) {  // of either half
  return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a),
                                                                __builtin_bit_cast(u16x2, b)));
}
template <typename T>
struct Mag;
template <>
struct Mag<float> {
  static constexpr unsigned kInf = 0x7f800000u;
  template <bool CLEAN>
  static __device__ __forceinline__ unsigned of(unsigned u) {
    u &= 0x7fffffffu;
    return CLEAN && u >= kInf ? 0u : u;
  }
  static __device__ __forceinline__ unsigned join(unsigned a, unsigned b) { return max(a, b); }
  static __device__ __forceinline__ bool odd(unsigned m) { return m >= kInf; }
  // exponent byte of a block with this maximum: smallest e >= -126 with amax <= 448 · 2^e =
  // 1.75 · 2^(e + 8); a mantissa above 1.75 carries into the exponent
  static __device__ __forceinline__ unsigned exp_byte(unsigned m) {
    return (unsigned)max((int)((m + 0x1fffffu) >> 23) - 8, 1);
  }
};
template <>
struct Mag<bf16_t> {
  template <bool CLEAN>
  static __device__ __forceinline__ unsigned of(unsigned u) {
    u &= 0x7fff7fffu;
    if (CLEAN && (u & 0xffffu) >= 0x7f80u) u &= 0xffff0000u;
    if (CLEAN && u >= 0x7f800000u) u &= 0xffffu;
    return u;
  }
  static __device__ __forceinline__ unsigned join(unsigned a, unsigned b) { return max2(a, b); }
  static __device__ __forceinline__ bool odd(unsigned m) {
    return max(m >> 16, m & 0xffffu) >= 0x7f80u;
  }
  static __device__ __forceinline__ unsigned exp_byte(unsigned m) {  // m: one magnitude
    return (unsigned)max((int)((m + 0x1fu) >> 7) - 8, 1);
  }
};

// 2^e of an exponent byte
__device__ __forceinline__ float exp_scale(unsigned byte) { return __uint_as_float(byte << 23); }

// Four values · 2^-e to four bytes, rounded to nearest even, scaled on the way
// (v_cvt_scalef32_pk_fp8: equal to the exact product and v_cvt_pk_fp8_f32 for every bf16 value and
// exponent); an infinity becomes NaN like a NaN itself.
typedef short s16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ unsigned to_fp8x4(float a, float b, float c, float d, float scale) {
  s16x2 q = {0, 0};
  q = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(q, a, b, scale, false);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(q, c, d, scale, true);
  return __builtin_bit_cast(unsigned, q);
}
__device__ __forceinline__ unsigned to_fp8x4(unsigned ab, unsigned cd, float scale) {  // bf16 pairs
  s16x2 q = {0, 0};
  q = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(q, __builtin_bit_cast(bf16v2, ab), scale, false);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(q, __builtin_bit_cast(bf16v2, cd), scale, true);
  return __builtin_bit_cast(unsigned, q);
}

}  // namespace dcn
