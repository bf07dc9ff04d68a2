// dcn_philox.h — counter-based random bits and element-vector access shared by the residual
// block's kernels (dcn_dropout.hip, dcn_block_norm.hip).
//
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3",
// 2011): ten rounds of two 32x32 -> 64-bit products. One call gives four words = eight 16-bit
// draws, so eight neighbouring elements (one 16-byte bf16 vector) share a call. 16 bits per
// draw instead of 32 halves the integer work (ten dependent rounds of two 64-bit products a
// call), which at 32 bits would exceed what the memory side of a bf16 stream takes; the price is
// p in steps of 1/65536, with the kept values scaled by the exact reciprocal of that p.
#pragma once
#include "dcn_device.h"

namespace dcn {

// What a kernel needs to draw masks: threshold, kept scale, and the seed / offset (or where
// they lie on the device).
struct DropArgs {
  const uint64_t* rng;  // {seed, offset} or null
  uint64_t seed, offset;
  unsigned thr;  // dropped where draw < thr; 0 = no dropout
  float scale;   // 65536 / (65536 - thr), 0 when everything is dropped
};

struct PhiloxKey {
  unsigned k0, k1, o0, o1;
};

__device__ __forceinline__ PhiloxKey philox_key(const DropArgs& a) {
  uint64_t seed = a.seed, off = a.offset;
  if (a.rng) {
    seed = a.rng[0];
    off = a.rng[1];
  }
  return PhiloxKey{(unsigned)seed, (unsigned)(seed >> 32), (unsigned)off, (unsigned)(off >> 32)};
}

__device__ __forceinline__ unsigned xor3(unsigned a, unsigned b, unsigned c) {
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);  // one instruction
}

__device__ __forceinline__ uint4 philox10(uint64_t block, const PhiloxKey& k) {
  unsigned x0 = (unsigned)block, x1 = (unsigned)(block >> 32), x2 = k.o0, x3 = k.o1;
  unsigned k0 = k.k0, k1 = k.k1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)x0 * 0xD2511F53u, p1 = (uint64_t)x2 * 0xCD9E8D57u;
    const unsigned n0 = xor3((unsigned)(p1 >> 32), x1, k0), n2 = xor3((unsigned)(p0 >> 32), x3, k1);
    x1 = (unsigned)p1;
    x3 = (unsigned)p0;
    x0 = n0;
    x2 = n2;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(x0, x1, x2, x3);
}

// bit j = draw j of the block is kept
__device__ __forceinline__ unsigned keep8(uint64_t block, const PhiloxKey& k, unsigned thr) {
  const uint4 w = philox10(block, k);
  const unsigned v[4] = {w.x, w.y, w.z, w.w};
  unsigned m = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    m |= (unsigned)((v[j] & 0xffffu) >= thr) << (2 * j);
    m |= (unsigned)((v[j] >> 16) >= thr) << (2 * j + 1);
  }
  return m;
}

__device__ __forceinline__ bool keep1(uint64_t draw, const PhiloxKey& k, unsigned thr) {
  return (keep8(draw >> 3, k, thr) >> (draw & 7)) & 1u;
}

// Vectors of 16 bytes at any element alignment: global memory takes unaligned accesses, so rows
// of odd length and sliced tensors need no scalar path (only their last partial vector does).
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16v2 __attribute__((ext_vector_type(2)));
typedef u32x4 u32x4_any __attribute__((aligned(2), may_alias));

template <typename T>
struct ElemVec;
template <>
struct ElemVec<bf16_t> {
  static constexpr int N = 8;
};
template <>
struct ElemVec<float> {
  static constexpr int N = 4;
};

// one 16-byte vector as it lies in memory; elements past `valid` are zero
template <typename T>
__device__ __forceinline__ u32x4 ldv_raw(const T* p, int valid) {
  constexpr int N = ElemVec<T>::N;
  if (valid >= N) return *reinterpret_cast<const u32x4_any*>(p);
  u32x4 r = {0u, 0u, 0u, 0u};
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < valid) r[j >> 1] |= (unsigned)p[j] << (16 * (j & 1));
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < valid) r[j] = __float_as_uint(p[j]);
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void unpack(const u32x4& r, float (&v)[ElemVec<T>::N]) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = __uint_as_float(r[j] << 16);
      v[2 * j + 1] = __uint_as_float(r[j] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(r[j]);
  }
}
template <typename T>
__device__ __forceinline__ u32x4 pack(const float (&v)[ElemVec<T>::N]) {
  u32x4 r;
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x2 p = {v[2 * j], v[2 * j + 1]};
      r[j] = __builtin_bit_cast(unsigned, __builtin_convertvector(p, bf16v2));  // one cvt_pk
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = __float_as_uint(v[j]);
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void stv_raw(T* p, const u32x4& r, int valid) {
  constexpr int N = ElemVec<T>::N;
  if (valid >= N) {
    *reinterpret_cast<u32x4_any*>(p) = r;
    return;
  }
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (j < valid) {
      if constexpr (sizeof(T) == 2)
        p[j] = (bf16_t)(r[j >> 1] >> (16 * (j & 1)));
      else
        p[j] = __uint_as_float(r[j]);
    }
}
template <typename T>
__device__ __forceinline__ void ldv(const T* p, int valid, float (&v)[ElemVec<T>::N]) {
  unpack<T>(ldv_raw(p, valid), v);
}
template <typename T>
__device__ __forceinline__ void stv(T* p, int valid, const float (&v)[ElemVec<T>::N]) {
  stv_raw(p, pack<T>(v), valid);
}
__device__ __forceinline__ float from_f32(float v, float) { return v; }
__device__ __forceinline__ bf16_t from_f32(float v, bf16_t) { return f2bf(v); }

}  // namespace dcn
