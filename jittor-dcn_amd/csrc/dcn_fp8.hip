// dcn_fp8.hip — rounding of maps and weights to e4m3 with one power-of-two exponent per block
// of 128 along the contracted axis (include/dcn.h, 8-bit pointwise products).
//
// Power-of-two scales: v · 2^-e is exact, so a value is rounded once (round to nearest even,
// v_cvt_scalef32_pk_fp8), and the MFMA applies the exponents itself (dcn_fp8_gemm.hip). A block
// loses no relative precision to that, at most one of e4m3's 18 binades of range.
//
// Memory is read once: a workgroup holds a 128 x 128 tile in registers (rows r of the tensor's
// outer axis, columns s of its contiguous one), takes the maxima it needs (per row of the tile
// for blocks along s, per column for blocks along r, over the tile for weights) and writes the
// straight bytes from registers, the transposed ones through LDS. bf16 values stay in pairs
// throughout: maxima and conversions take two at a time.
#include <type_traits>

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

// max over aligned groups of LPR (16 or 32) lanes; JOIN: both halves apart, or whole
template <int LPR, typename F>
__device__ __forceinline__ unsigned lanes_max(unsigned v, F join) {
  auto dpp = [](unsigned u, auto ctrl) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)u, decltype(ctrl)::value, 0xf, 0xf, false);
  };
  v = join(v, dpp(v, std::integral_constant<int, 0xB1>()));   // quad_perm [1,0,3,2]
  v = join(v, dpp(v, std::integral_constant<int, 0x4E>()));   // quad_perm [2,3,0,1]
  v = join(v, dpp(v, std::integral_constant<int, 0x141>()));  // row_half_mirror
  v = join(v, dpp(v, std::integral_constant<int, 0x140>()));  // row_mirror
  if constexpr (LPR == 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = join(r[0], r[1]);
  }
  return v;
}

// LDS row of the transposed tile: 16 chunks of 8 bytes, chunk c at c ^ 2 ((row >> 4) & 7), rows
// padded by 16 bytes: a wave's writes (rows V apart) meet every bank equally often
constexpr int PITCH = 144;
template <typename T>
struct QuantShared {
  static constexpr int LPR = 128 / ElemVec<T>::N;
  unsigned char tile[128 * PITCH];
  unsigned colmax[kThreads / LPR][LPR][4];  // as raw: pairs, or one
};

// Tile `bid` of one matrix. BLOCK2D: one exponent per tile, for both results (weights)
template <typename T, bool BLOCK2D>
__device__ __forceinline__ void quantize_tile(const QuantArgs& a, int bid, QuantShared<T>& sh) {
  using M = Mag<T>;
  constexpr bool PAIRS = sizeof(T) == 2;
  constexpr int V = ElemVec<T>::N, LPR = 128 / V;     // lanes across a row of the tile
  constexpr int GROUPS = kThreads / LPR;              // row groups of kRows rows at a time
  constexpr int PASS = 128 / (GROUPS * kRows);        // 1 (bf16), 2 (f32)
  auto& tile = sh.tile;
  auto& colmax = sh.colmax;
  const int lane = threadIdx.x % LPR, grp = threadIdx.x / LPR;
  const int ts = bid % a.tiles_s, tr = (bid / a.tiles_s) % a.tiles_r;
  const int img = bid / (a.tiles_s * a.tiles_r);
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

  unsigned rmax[PASS][kRows], cmax[4];  // this thread's share of rows and columns
  auto maxima = [&](auto clean) {
    constexpr bool CLEAN = decltype(clean)::value;
#pragma unroll
    for (int j = 0; j < 4; ++j) cmax[j] = 0;
#pragma unroll
    for (int p = 0; p < PASS; ++p)
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        unsigned m[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          m[j] = M::template of<CLEAN>(raw[p][i][j]);
          cmax[j] = M::join(cmax[j], m[j]);
        }
        rmax[p][i] = M::join(M::join(m[0], m[1]), M::join(m[2], m[3]));
      }
  };
  maxima(std::false_type());
  if (__any(M::odd(M::join(M::join(cmax[0], cmax[1]), M::join(cmax[2], cmax[3])))))
    maxima(std::true_type());

  if (BLOCK2D || a.qt) {
    *reinterpret_cast<u32x4*>(colmax[grp][lane]) = u32x4{cmax[0], cmax[1], cmax[2], cmax[3]};
    __syncthreads();
    if (threadIdx.x < LPR * 4) {
      unsigned* c = &colmax[0][0][0] + threadIdx.x;
      unsigned m = 0;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) m = M::join(m, c[g * LPR * 4]);
      *c = m;
    }
    __syncthreads();
  }
  unsigned whole = 0;
  if (BLOCK2D) {
    const unsigned* c = &colmax[0][0][0];
    for (int j = threadIdx.x & 63; j < LPR * 4; j += 64) whole = M::join(whole, c[j]);
    if (PAIRS) whole = max(whole >> 16, whole & 0xffffu);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) whole = max(whole, (unsigned)__shfl_xor((int)whole, o));
    whole = M::exp_byte(whole);
  }

  if (a.q) {
    if constexpr (!BLOCK2D) {  // exponent bytes of the rows into rmax
#pragma unroll
      for (int p = 0; p < PASS; ++p) {
        if constexpr (PAIRS) {  // two rows in one register
#pragma unroll
          for (int i = 0; i < kRows; i += 2) {
            const unsigned x = rmax[p][i], y = rmax[p][i + 1];
            const unsigned m = lanes_max<LPR>(
                max2(__builtin_amdgcn_perm(y, x, 0x05040100u), __builtin_amdgcn_perm(y, x, 0x07060302u)),
                max2);
            rmax[p][i] = M::exp_byte(m & 0xffffu);
            rmax[p][i + 1] = M::exp_byte(m >> 16);
          }
        } else {
#pragma unroll
          for (int i = 0; i < kRows; ++i)
            rmax[p][i] = M::exp_byte(lanes_max<LPR>(
                rmax[p][i], [](unsigned u, unsigned v) { return max(u, v); }));
        }
      }
    }
    const size_t k = (size_t)img * a.kimg + s;  // the row's tail up to the next 128 is zeros
#pragma unroll
    for (int p = 0; p < PASS; ++p)
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int r = r0 + (p * GROUPS + grp) * kRows + i;
        if (r >= a.R) continue;
        const unsigned e = BLOCK2D ? whole : rmax[p][i];
        const float sc = exp_scale(e);
        const u32x4 v = raw[p][i];
        unsigned char* dst = a.q + (size_t)r * a.qk + k;
        if constexpr (PAIRS)
          *reinterpret_cast<uint2*>(dst) =
              make_uint2(to_fp8x4(v[0], v[1], sc), to_fp8x4(v[2], v[3], sc));
        else
          *reinterpret_cast<unsigned*>(dst) =
              to_fp8x4(__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2]),
                       __uint_as_float(v[3]), sc);
        if (!BLOCK2D && lane == 0)
          a.s[(((size_t)img * a.kimg + s0) / 128) * a.sstr + r] = (unsigned char)e;
      }
    if (BLOCK2D && threadIdx.x == 0) a.s[(size_t)ts * a.sstr + tr] = (unsigned char)whole;
  }
  if (!a.qt) return;  // uniform

  float f[V];
  const u32x4 cm = *reinterpret_cast<const u32x4*>(colmax[0][lane]);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const unsigned m = PAIRS ? (cm[j / 2] >> (16 * (j & 1))) & 0xffffu : cm[j % 4];
    const unsigned e = BLOCK2D ? whole : M::exp_byte(m);
    f[j] = exp_scale(e);
    if (!BLOCK2D && grp == 0 && s + j < a.S)
      a.st[(size_t)tr * a.tstr + (size_t)img * a.S + s + j] = (unsigned char)e;
  }
  if (BLOCK2D && threadIdx.x == 0) a.st[(size_t)tr * a.tstr + ts] = (unsigned char)whole;
#pragma unroll
  for (int p = 0; p < PASS; ++p)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const u32x4(&v)[kRows] = raw[p];
      uint2 b;
      if constexpr (PAIRS) {  // column j of two rows, side by side
        const unsigned sel = j & 1 ? 0x07060302u : 0x05040100u;
        auto two = [&](int i) { return __builtin_amdgcn_perm(v[i + 1][j / 2], v[i][j / 2], sel); };
        b = make_uint2(to_fp8x4(two(0), two(2), f[j]), to_fp8x4(two(4), two(6), f[j]));
      } else {
        auto one = [&](int i) { return __uint_as_float(v[i][j % 4]); };
        b = make_uint2(to_fp8x4(one(0), one(1), one(2), one(3), f[j]),
                       to_fp8x4(one(4), one(5), one(6), one(7), f[j]));
      }
      const int row = lane * V + j, c = (p * GROUPS + grp) ^ (((row >> 4) & 7) << 1);
      *reinterpret_cast<uint2*>(&tile[row * PITCH + c * 8]) = b;
    }
  __syncthreads();
  // 8 lanes of 16 bytes a row, 32 rows a pass
  for (int row = threadIdx.x / 8; row < 128 && s0 + row < a.S; row += kThreads / 8) {
    const int c = threadIdx.x % 8;
    *reinterpret_cast<u32x4*>(a.qt + ((size_t)img * a.S + s0 + row) * a.tk + r0 + c * 16) =
        *reinterpret_cast<const u32x4*>(&tile[row * PITCH + (c ^ ((row >> 4) & 7)) * 16]);
  }
}

template <typename T, bool BLOCK2D>
__global__ __launch_bounds__(kThreads) void fp8_quantize(QuantArgs a) {
  __shared__ __attribute__((aligned(16))) QuantShared<T> sh;
  quantize_tile<T, BLOCK2D>(a, blockIdx.x, sh);
}

// A weight's tiles and a tensor's in one launch (a launch and its gap are about 5 us, as long as
// the rounding of 8 MB)
template <typename T>
__global__ __launch_bounds__(kThreads) void fp8_quantize_both(QuantArgs w, QuantArgs x, int w_tiles) {
  __shared__ __attribute__((aligned(16))) QuantShared<T> sh;
  if ((int)blockIdx.x < w_tiles)
    quantize_tile<T, true>(w, blockIdx.x, sh);
  else
    quantize_tile<T, false>(x, blockIdx.x - w_tiles, sh);
}

long up128(long v) { return (v + 127) / 128 * 128; }

// fills in the tiles and gives their number
unsigned tiles(QuantArgs& a, int images) {
  a.tiles_s = (a.S + 127) / 128;
  a.tiles_r = (a.R + 127) / 128;
  return (unsigned)((size_t)a.tiles_s * a.tiles_r * images);
}

hipError_t launch(QuantArgs a, int images, int dtype, bool block2d, hipStream_t s) {
  const dim3 g(tiles(a, images)), t(kThreads);
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

QuantArgs tensor_args(int B, int C, int P, int layout, const void* v, void* q_tok, void* s_tok,
                      void* q_ch, void* s_ch) {
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
    return a;
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
  return a;
}

QuantArgs weight_args(int O, int C, const void* w, void* q, void* sq, void* qT, void* sT) {
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
  return a;
}

}  // namespace

hipError_t launch_fp8_quantize(int B, int C, int P, int layout, int dtype, const void* v,
                               void* q_tok, void* s_tok, void* q_ch, void* s_ch, hipStream_t s) {
  return launch(tensor_args(B, C, P, layout, v, q_tok, s_tok, q_ch, s_ch),
                layout == DCN_NHWC ? 1 : B, dtype, false, s);
}

hipError_t launch_fp8_quantize_weight(int O, int C, int dtype, const void* w, void* q, void* sq,
                                      void* qT, void* sT, hipStream_t s) {
  return launch(weight_args(O, C, w, q, sq, qT, sT), 1, dtype, true, s);
}

hipError_t launch_fp8_quantize_both(int B, int C, int P, int layout, int dtype, const void* v,
                                    void* q_tok, void* s_tok, void* q_ch, void* s_ch, int O,
                                    const void* w, void* q, void* sq, void* qT, void* sT,
                                    hipStream_t s) {
  QuantArgs x = tensor_args(B, C, P, layout, v, q_tok, s_tok, q_ch, s_ch);
  QuantArgs a = weight_args(O, C, w, q, sq, qT, sT);
  const unsigned nw = tiles(a, 1), nx = tiles(x, layout == DCN_NHWC ? 1 : B);
  const dim3 g(nw + nx), t(kThreads);
  if (dtype == DCN_BF16)
    hipLaunchKernelGGL((fp8_quantize_both<bf16_t>), g, t, 0, s, a, x, (int)nw);
  else
    hipLaunchKernelGGL((fp8_quantize_both<float>), g, t, 0, s, a, x, (int)nw);
  return hipGetLastError();
}

}  // namespace dcn
