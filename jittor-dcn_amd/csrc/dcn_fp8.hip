// dcn_fp8.hip — rounding of maps and weights to e4m3 with one power-of-two exponent per block
// of 128 along the contracted axis (include/dcn.h, 8-bit pointwise products).
//
// Power-of-two scales: v · 2^-e is exact, so a value is rounded once (round to nearest even,
// v_cvt_pk_fp8_f32), and the MFMA applies the exponents itself (dcn_fp8_gemm.hip). A block
// loses no relative precision to that, at most one of e4m3's 18 binades of range.
//
// Memory is read once: a workgroup holds a 128 x 128 tile in registers (rows r of the tensor's
// outer axis, columns s of its contiguous one), takes the maxima it needs (per row of the tile
// for blocks along s, per column for blocks along r, over the tile for weights) and writes the
// straight bytes from registers, the transposed ones through LDS.
#include "dcn_block.h"
#include "dcn_fp8.h"

namespace dcn {

namespace {

constexpr int kThreads = 256;
constexpr int kRows = 8;  // consecutive rows of a thread

// One matrix [R][S] per image; see include/dcn.h for the two results.
struct QuantArgs {
  const void* v;
  unsigned char *q, *s;    // blocks along S: q[r][img · kimg + s], row stride qk; s[k / 128][sstr]
  unsigned char *qt, *st;  // blocks along R: qt[img · S + s][r], row stride tk; st[r / 128][tstr]
  int R, S;
  long qk, kimg, sstr, tk, tstr;
  int tiles_s, tiles_r;
};

// BLOCK2D: one exponent per tile, for both results (weights)
template <typename T, bool BLOCK2D>
__global__ __launch_bounds__(kThreads) void fp8_quantize(QuantArgs a) {
  constexpr int V = ElemVec<T>::N, LPR = 128 / V;     // lanes across a row of the tile
  constexpr int GROUPS = kThreads / LPR;              // row groups of kRows rows at a time
  constexpr int PASS = 128 / (GROUPS * kRows);        // 1 (bf16), 2 (f32)
  constexpr int PITCH = 136;                          // LDS row: 128 bytes of r, padded
  __shared__ __attribute__((aligned(16))) unsigned char tile[128 * PITCH];
  __shared__ unsigned colmax[GROUPS][128];
  const int lane = threadIdx.x % LPR, grp = threadIdx.x / LPR;
  const int ts = blockIdx.x % a.tiles_s, tr = (blockIdx.x / a.tiles_s) % a.tiles_r;
  const int img = blockIdx.x / (a.tiles_s * a.tiles_r);
  const int s0 = ts * 128, r0 = tr * 128, s = s0 + lane * V;
  const T* src = static_cast<const T*>(a.v) + (size_t)img * a.R * a.S;

  u32x4 raw[PASS][kRows];
#pragma unroll
  for (int p = 0; p < PASS; ++p)
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int r = r0 + (p * GROUPS + grp) * kRows + i;
      raw[p][i] = r < a.R ? ldv_raw(src + (size_t)r * a.S + s, a.S - s) : u32x4{0u, 0u, 0u, 0u};
    }

  unsigned rowmax[PASS][kRows], cmax[V];
#pragma unroll
  for (int j = 0; j < V; ++j) cmax[j] = 0;
#pragma unroll
  for (int p = 0; p < PASS; ++p)
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      float v[V];
      unpack<T>(raw[p][i], v);
      unsigned m = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        m = mag_max(m, v[j]);
        cmax[j] = mag_max(cmax[j], v[j]);
      }
#pragma unroll
      for (int o = 1; o < LPR; o <<= 1) m = max(m, (unsigned)__shfl_xor((int)m, o));
      rowmax[p][i] = m;
    }
  if (BLOCK2D || a.qt) {
#pragma unroll
    for (int j = 0; j < V; ++j) colmax[grp][lane * V + j] = cmax[j];
    __syncthreads();
    if (threadIdx.x < 128) {
      unsigned m = 0;
      for (int g = 0; g < GROUPS; ++g) m = max(m, colmax[g][threadIdx.x]);
      colmax[0][threadIdx.x] = m;
    }
    __syncthreads();
  }
  unsigned whole = 0;
  if (BLOCK2D) {
    for (int j = threadIdx.x & 63; j < 128; j += 64) whole = max(whole, colmax[0][j]);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) whole = max(whole, (unsigned)__shfl_xor((int)whole, o));
    whole = exp_byte(whole);
  }

  if (a.q) {
    const size_t k = (size_t)img * a.kimg + s;  // the row's tail up to the next 128 is zeros
#pragma unroll
    for (int p = 0; p < PASS; ++p)
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int r = r0 + (p * GROUPS + grp) * kRows + i;
        if (r >= a.R) continue;
        const unsigned e = BLOCK2D ? whole : exp_byte(rowmax[p][i]);
        const float f = exp_inv(e);
        float v[V];
        unpack<T>(raw[p][i], v);
        unsigned* dst = reinterpret_cast<unsigned*>(a.q + (size_t)r * a.qk + k);
#pragma unroll
        for (int j = 0; j < V; j += 4)
          dst[j / 4] = to_fp8x4(v[j] * f, v[j + 1] * f, v[j + 2] * f, v[j + 3] * f);
        if (!BLOCK2D && lane == 0)
          a.s[(((size_t)img * a.kimg + s0) / 128) * a.sstr + r] = (unsigned char)e;
      }
    if (BLOCK2D && threadIdx.x == 0) a.s[(size_t)ts * a.sstr + tr] = (unsigned char)whole;
  }
  if (!a.qt) return;  // uniform

  float f[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const unsigned e = BLOCK2D ? whole : exp_byte(colmax[0][lane * V + j]);
    f[j] = exp_inv(e);
    if (!BLOCK2D && grp == 0 && s + j < a.S)
      a.st[(size_t)tr * a.tstr + (size_t)img * a.S + s + j] = (unsigned char)e;
  }
  if (BLOCK2D && threadIdx.x == 0) a.st[(size_t)tr * a.tstr + ts] = (unsigned char)whole;
#pragma unroll
  for (int p = 0; p < PASS; ++p) {
    float v[kRows][V];
#pragma unroll
    for (int i = 0; i < kRows; ++i) unpack<T>(raw[p][i], v[i]);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const uint2 b = make_uint2(
          to_fp8x4(v[0][j] * f[j], v[1][j] * f[j], v[2][j] * f[j], v[3][j] * f[j]),
          to_fp8x4(v[4][j] * f[j], v[5][j] * f[j], v[6][j] * f[j], v[7][j] * f[j]));
      *reinterpret_cast<uint2*>(&tile[(lane * V + j) * PITCH + (p * GROUPS + grp) * kRows]) = b;
    }
  }
  __syncthreads();
  // 8 lanes of 16 bytes a row, 32 rows a pass
  for (int row = threadIdx.x / 8; row < 128 && s0 + row < a.S; row += kThreads / 8) {
    const unsigned char* t = &tile[row * PITCH + (threadIdx.x % 8) * 16];
    const uint2 lo = *reinterpret_cast<const uint2*>(t), hi = *reinterpret_cast<const uint2*>(t + 8);
    *reinterpret_cast<uint4*>(a.qt + ((size_t)img * a.S + s0 + row) * a.tk + r0 +
                              (threadIdx.x % 8) * 16) = make_uint4(lo.x, lo.y, hi.x, hi.y);
  }
}

long up128(long v) { return (v + 127) / 128 * 128; }

hipError_t launch(QuantArgs a, int images, int dtype, bool block2d, hipStream_t s) {
  a.tiles_s = (a.S + 127) / 128;
  a.tiles_r = (a.R + 127) / 128;
  const unsigned grid = (unsigned)((size_t)a.tiles_s * a.tiles_r * images);
  const dim3 g(grid), t(kThreads);
  if (dtype == DCN_BF16 && block2d)
    hipLaunchKernelGGL((fp8_quantize<bf16_t, true>), g, t, 0, s, a);
  else if (dtype == DCN_BF16)
    hipLaunchKernelGGL((fp8_quantize<bf16_t, false>), g, t, 0, s, a);
  else if (block2d)
    hipLaunchKernelGGL((fp8_quantize<float, true>), g, t, 0, s, a);
  else
    hipLaunchKernelGGL((fp8_quantize<float, false>), g, t, 0, s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_fp8_quantize(int B, int C, int P, int layout, int dtype, const void* v,
                               void* q_tok, void* s_tok, void* q_ch, void* s_ch, hipStream_t s) {
  QuantArgs a{};
  a.v = v;
  auto u8 = [](void* p) { return static_cast<unsigned char*>(p); };
  const long T = (long)B * P;
  if (layout == DCN_NHWC) {
    a.R = (int)T;
    a.S = C;
    a.q = u8(q_tok);
    a.s = u8(s_tok);
    a.qk = up128(C);
    a.sstr = up128(T);
    a.qt = u8(q_ch);
    a.st = u8(s_ch);
    a.tk = up128(T);
    a.tstr = up128(C);
    return launch(a, 1, dtype, false, s);
  }
  a.R = C;
  a.S = P;
  a.q = u8(q_ch);
  a.s = u8(s_ch);
  a.kimg = up128(P);
  a.qk = B * a.kimg;
  a.sstr = up128(C);
  a.qt = u8(q_tok);
  a.st = u8(s_tok);
  a.tk = up128(C);
  a.tstr = up128(T);
  return launch(a, B, dtype, false, s);
}

hipError_t launch_fp8_quantize_weight(int O, int C, int dtype, const void* w, void* q, void* sq,
                                      void* qT, void* sT, hipStream_t s) {
  QuantArgs a{};
  auto u8 = [](void* p) { return static_cast<unsigned char*>(p); };
  a.v = w;
  a.R = O;
  a.S = C;
  a.q = u8(q);
  a.s = u8(sq);
  a.qk = up128(C);
  a.sstr = (O + 127) / 128;
  a.qt = u8(qT);
  a.st = u8(sT);
  a.tk = up128(O);
  a.tstr = (C + 127) / 128;
  return launch(a, 1, dtype, true, s);
}

}  // namespace dcn
