// dcn_fp8_gemm.hip — out = a · bᵀ over 8-bit matrices with one exponent per block of 128 along
// K (include/dcn.h, dcn_fp8_matmul), on the scaled MFMA of gfx950.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes K = 128 at once, one block of both operands, and
// multiplies by both exponents on the way into the fp32 accumulator, so the scales cost no
// arithmetic. Both operands are K-contiguous; which 32 of the 128 k's a lane holds does not
// matter as long as a's and b's lanes agree, because one exponent covers all 128.
//
// The 8-bit MFMA does not add in 32 bits throughout: measured on the builtin, in every group of
// 8 neighbouring k's the products are cut below 2^-13 of the largest one's power of two before
// they are added (then fp32). A sum is off by less than 7 · 2^-13 = 8.5e-4 of its Σ|a b|, 1e-5 to
// 7e-5 of the result in practice: inside the half step 2^-9 of a bf16 result unless the sum cancels
// (and the bytes are worth their values to 2^-4 only), so those use it. An fp32 result (WIDE)
// multiplies the same bytes as bf16 on the bf16 MFMA (fp32 sums, 1e-7), at half the rate and a
// conversion per byte (v_cvt_scalef32_pk_bf16_fp8). bf16 holds every byte with its exponent but
// for the ends of the range: below 2^-133 bits are lost (exponents under -124), and 448 · 2^120
// covers values that e4m3 rounds up to 2^128, infinite there.
//
// Rows of a 64-row group are dealt to the fragments in turn (fragment f, lane r = row 4r + f):
// one aligned dword of exponents then serves a lane's four fragments (the instruction picks the
// byte), and a lane's four columns of the result are neighbours, stored as one vector.
#include <type_traits>

#include "dcn_block.h"
#include "dcn_fp8.h"

namespace dcn {

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(1))) void gvoid;
typedef __attribute__((address_space(3))) void lvoid;

struct GemmArgs {
  const unsigned char *a, *sa, *b, *sb;
  void* out;
  float* part;  // split K: fp32 partials [split][M][N]
  int M, N, nkb, P, nchw, a_shift, b_shift;  // shift: log2 of rows per exponent
  long K, sa_str, sb_str;
  int kb_split;    // k blocks of a split
  const void* x;   // the short side before its rounding, rows of x_cols
  int x_cols;
  int tiles_m, tiles_n;
};

// row of a tile that LDS row `slot` holds
__device__ __forceinline__ int slot_row(int slot) {
  return (slot & ~63) + 4 * (slot & 15) + ((slot >> 4) & 3);
}

// exponents of rows 4r .. 4r + 3 of the 64-row group at row0, for k block kb
__device__ __forceinline__ int exps4(const unsigned char* s, long str, int shift, int kb, int row0,
                                     int r) {
  const unsigned char* p = s + (size_t)kb * str;
  if (shift) return (int)p[min((long)(row0 >> shift), str - 1)];  // one for all four: spread()
  return *reinterpret_cast<const int*>(p + min((long)(row0 + 4 * r), str - 4));
}
// what exps4 loaded as four bytes (apart from the load, so that the load is waited for here)
__device__ __forceinline__ int spread(int e, int shift) {
  return shift ? (int)((unsigned)e * 0x01010101u) : e;
}

// eight bytes (dwords 2p, 2p + 1 of a fragment) as bf16, with the exponent `e`
__device__ __forceinline__ bf16x8 widen(const i32x8& v, int p, unsigned e) {
  const float sc = __uint_as_float(e << 23);
  bf16x2 w[4];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    w[2 * j] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)v[2 * p + j], sc, false);
    w[2 * j + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)v[2 * p + j], sc, true);
  }
  return bf16x8{w[0][0], w[0][1], w[1][0], w[1][1], w[2][0], w[2][1], w[3][0], w[3][1]};
}

template <int I, int J>
__device__ __forceinline__ f32x4 mfma8(const i32x8& a, const i32x8& b, f32x4 c, int ea, int eb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, I, ea, J, eb);
}

// four fragments of a times four of b (one 64-row group of either)
template <bool WIDE>
__device__ __forceinline__ void quad(const i32x8 (&a)[4], const i32x8 (&b)[4], int ea, int eb,
                                     f32x4 (&c)[4][4]) {
  if constexpr (WIDE) {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      bf16x8 xa[4], xb[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        xa[i] = widen(a[i], p, ((unsigned)ea >> (8 * i)) & 255u);
        xb[i] = widen(b[i], p, ((unsigned)eb >> (8 * i)) & 255u);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          c[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xa[i], xb[j], c[i][j], 0, 0, 0);
    }
  } else {
#define DCN_ROW(i)                                \
  c[i][0] = mfma8<i, 0>(a[i], b[0], c[i][0], ea, eb); \
  c[i][1] = mfma8<i, 1>(a[i], b[1], c[i][1], ea, eb); \
  c[i][2] = mfma8<i, 2>(a[i], b[2], c[i][2], ea, eb); \
  c[i][3] = mfma8<i, 3>(a[i], b[3], c[i][3], ea, eb);
    DCN_ROW(0)
    DCN_ROW(1)
    DCN_ROW(2)
    DCN_ROW(3)
#undef DCN_ROW
  }
}

// where element (m, n) of the result lies
__device__ __forceinline__ size_t out_at(const GemmArgs& g, int m, int n) {
  if (!g.nchw) return (size_t)m * g.N + n;
  const int b = n / g.P;
  return ((size_t)b * g.M + m) * g.P + (n - b * g.P);
}
template <bool WIDE>
__device__ __forceinline__ void put(const GemmArgs& g, size_t at, float v) {
  if constexpr (WIDE)
    static_cast<float*>(g.out)[at] = v;
  else
    static_cast<bf16_t*>(g.out)[at] = f2bf(v);
}
typedef f32x4 f32x4_any __attribute__((aligned(4), may_alias));
typedef unsigned u32x2_any __attribute__((ext_vector_type(2), aligned(2), may_alias));
// columns n .. n + 3 of row m, one store where they are neighbours (any alignment will do)
struct Column {  // column n's place in row 0, the rows' stride, and whether n .. n + 3 are neighbours
  size_t at, stride;
  bool four;
};
__device__ __forceinline__ Column column(const GemmArgs& g, int n) {
  if (!g.nchw) return {(size_t)n, (size_t)g.N, n + 4 <= g.N};
  const int b = n / g.P, p = n - b * g.P;
  return {(size_t)b * g.M * g.P + p, (size_t)g.P, n + 4 <= g.N && p + 4 <= g.P};
}
template <bool WIDE>
__device__ __forceinline__ void put4(const GemmArgs& g, const Column& c, int m, int n, f32x4 v) {
  if (c.four) {
    const size_t at = c.at + m * c.stride;
    if constexpr (WIDE) {
      *reinterpret_cast<f32x4_any*>(static_cast<float*>(g.out) + at) = v;
    } else {
      const u32x2_any u = {__builtin_bit_cast(unsigned, __builtin_convertvector(
                               __builtin_shufflevector(v, v, 0, 1), bf16x2)),
                           __builtin_bit_cast(unsigned, __builtin_convertvector(
                               __builtin_shufflevector(v, v, 2, 3), bf16x2))};
      *reinterpret_cast<u32x2_any*>(static_cast<bf16_t*>(g.out) + at) = u;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (n + j < g.N) put<WIDE>(g, out_at(g, m, n + j), v[j]);
}

// ---- tiles: WM x WN waves, each GA x GB groups of 64 x 64, K in stages of 128 through two LDS
// buffers: while one is multiplied, LDS-DMA fills the other.
template <int GA, int GB, int WM, int WN, int WPE, int STAGES, bool WIDE, bool SPLIT>
__global__ __launch_bounds__(WM* WN * 64, WPE) void fp8_gemm(GemmArgs g) {
  constexpr int BM = WM * GA * 64, BN = WN * GB * 64, NW = WM * WN, STAGE = (BM + BN) * 128;
  constexpr int PER = STAGE / 1024 / NW;  // 1 KiB DMA instructions of a wave and stage
  __shared__ __attribute__((aligned(1024))) char ring0[STAGE], ring1[STAGES == 2 ? STAGE : 16];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // neighbouring tiles on one XCD, in bands of 8 tile rows, share their operands through its L2
  const int nwg = g.tiles_m * g.tiles_n, bid = blockIdx.x, xcd = bid & 7, q8 = nwg >> 3, r8 = nwg & 7;
  const int lid = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (bid >> 3);
  const int width = 8 * g.tiles_n, band = lid / width, in = lid % width;
  const int rows = min(8, g.tiles_m - band * 8);
  const int m0 = (band * 8 + in % rows) * BM, n0 = in / rows * BN;
  const int k0 = SPLIT ? (int)blockIdx.y * g.kb_split : 0;
  const int nkb = SPLIT ? min(g.kb_split, g.nkb - k0) : g.nkb;

  // LDS rows of 128 bytes, a's then b's; 16-byte chunk c of row t sits at c ^ (t >> 1)
  const unsigned char* src[PER];
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int i = u * NW + w, t = i * 8 + (lane >> 3), c = (lane & 7) ^ ((t >> 1) & 7);
    const bool isb = i >= BM / 8;
    const int row = isb ? min(n0 + slot_row(t - BM), g.N - 1) : min(m0 + slot_row(t), g.M - 1);
    src[u] = (isb ? g.b : g.a) + (size_t)row * g.K + (size_t)k0 * 128 + c * 16;
  }
  auto issue = [&](int kb, char* slot) {
#pragma unroll
    for (int u = 0; u < PER; ++u)
      __builtin_amdgcn_global_load_lds((gvoid*)(src[u] + (size_t)kb * 128),
                                       (lvoid*)(slot + (u * NW + w) * 1024), 16, 0, 0);
  };
  const int wm = w / WN, wn = w % WN, r = lane & 15, q = lane >> 4, x = (r >> 1) & 7;
  const int lo = r * 128 + ((q ^ x) << 4), hi = r * 128 + (((q + 4) ^ x) << 4);
  auto frag = [&](const char* base, int f) {  // f: fragment of 16 LDS rows
    const i32x4 l = *reinterpret_cast<const i32x4*>(base + f * 2048 + lo);
    const i32x4 h = *reinterpret_cast<const i32x4*>(base + f * 2048 + hi);
    return __builtin_shufflevector(l, h, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  f32x4 acc[GA][GB][4][4];
#pragma unroll
  for (int i = 0; i < GA * GB * 16; ++i)
    (&acc[0][0][0][0])[i] = f32x4{0.f, 0.f, 0.f, 0.f};

  int ea[GA], eb[GB], na[GA], nb[GB];  // this stage's exponents and the next's
  auto exps = [&](int kb) {
#pragma unroll
    for (int i = 0; i < GA; ++i)
      na[i] = exps4(g.sa, g.sa_str, g.a_shift, k0 + kb, m0 + (wm * GA + i) * 64, r);
#pragma unroll
    for (int j = 0; j < GB; ++j)
      nb[j] = exps4(g.sb, g.sb_str, g.b_shift, k0 + kb, n0 + (wn * GB + j) * 64, r);
  };
  auto compute = [&](const char* slot) {
    i32x8 fb[GB][4];
#pragma unroll
    for (int j = 0; j < GB; ++j)
#pragma unroll
      for (int f = 0; f < 4; ++f) fb[j][f] = frag(slot + BM * 128, (wn * GB + j) * 4 + f);
#pragma unroll
    for (int i = 0; i < GA; ++i) {
      i32x8 fa[4];
#pragma unroll
      for (int f = 0; f < 4; ++f) fa[f] = frag(slot, (wm * GA + i) * 4 + f);
#pragma unroll
      for (int j = 0; j < GB; ++j) quad<WIDE>(fa, fb[j], ea[i], eb[j], acc[i][j]);
    }
  };
  auto step = [&](int kb, const char* cur, char* other) {
    __syncthreads();  // stage kb and its exponents landed; every wave is done with `other`
#pragma unroll
    for (int i = 0; i < GA; ++i) ea[i] = spread(na[i], g.a_shift);
#pragma unroll
    for (int j = 0; j < GB; ++j) eb[j] = spread(nb[j], g.b_shift);
    if (kb + 1 < nkb) {
      exps(kb + 1);
      issue(kb + 1, other);
    }
    compute(cur);
  };
  exps(0);
  issue(0, ring0);
  if constexpr (STAGES == 2) {
    for (int kb = 0; kb < nkb; kb += 2) {
      step(kb, ring0, ring1);
      if (kb + 1 < nkb) step(kb + 1, ring1, ring0);
    }
  } else {
    for (int kb = 0; kb < nkb; ++kb) {
      __syncthreads();  // the stage landed
#pragma unroll
      for (int i = 0; i < GA; ++i) ea[i] = spread(na[i], g.a_shift);
#pragma unroll
      for (int j = 0; j < GB; ++j) eb[j] = spread(nb[j], g.b_shift);
      compute(ring0);
      if (kb + 1 == nkb) break;
      __syncthreads();  // every wave has read it
      exps(kb + 1);
      issue(kb + 1, ring0);
    }
  }

  // acc[..][i][j][e]: row 4 (4q + e) + i, column 4r + j of its 64 x 64
#pragma unroll
  for (int ga = 0; ga < GA; ++ga)
#pragma unroll
    for (int gb = 0; gb < GB; ++gb) {
      const int n = n0 + (wn * GB + gb) * 64 + 4 * r;
      const Column col = column(g, n);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int m = m0 + (wm * GA + ga) * 64 + 4 * (4 * q + e) + i;
          if (m >= g.M || n >= g.N) continue;
          const f32x4 v = {acc[ga][gb][i][0][e], acc[ga][gb][i][1][e], acc[ga][gb][i][2][e],
                           acc[ga][gb][i][3][e]};
          if constexpr (SPLIT) {
            float* p = g.part + ((size_t)blockIdx.y * g.M + m) * g.N + n;
            if (n + 4 <= g.N) {
              *reinterpret_cast<f32x4_any*>(p) = v;
            } else {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (n + j < g.N) p[j] = v[j];
            }
          } else {
            put4<WIDE>(g, col, m, n, v);
          }
        }
    }
}

// ---- large tiles, two groups of waves in turn: 256 x 256, eight waves of 128 x 64. Waves 0..3 and
// 4..7 (one of each on every SIMD) run half a stage apart: while one group's fragments come out of
// LDS the other multiplies, so the matrix cores never wait for LDS; a barrier ends every half.
//   phase 2k: group 0 reads stage k, group 1 multiplies stage k - 1; 2k + 1: the other way round.
// Stage k + 1 replaces stage k - 1, which group 1 has read in phase 2k - 1: both groups fetch their
// shares from phase 2k on and have waited for them by the end of phase 2k + 1. A stage's LDS traffic
// (24 KB read by each wave, 64 KB written) takes about as long as its products; all waves in step
// waited for the one and then the other (16384 x 8192 x 8192 1.08 ms, in turns 0.94).
// A128, B128: an exponent per 128 rows (known here, so that the stages have no branches).
template <bool A128, bool B128>
__global__ __launch_bounds__(512, 2) void fp8_gemm_turns(GemmArgs g) {
  constexpr int BM = 256, BN = 256, STAGE = (BM + BN) * 128, PER = STAGE / 1024 / 8;
  __shared__ __attribute__((aligned(1024))) char ring0[STAGE], ring1[STAGE];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = w & 3;
  const bool second = w >> 2;  // group, and which half of the rows
  const int nwg = g.tiles_m * g.tiles_n, bid = blockIdx.x, xcd = bid & 7, q8 = nwg >> 3, r8 = nwg & 7;
  const int lid = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (bid >> 3);
  const int width = 8 * g.tiles_n, band = lid / width, in = lid % width;
  const int rows = min(8, g.tiles_m - band * 8);
  const int m0 = (band * 8 + in % rows) * BM, n0 = in / rows * BN;
  const int nkb = g.nkb;

  // Unit u fetches LDS rows 64 u + 8 w ..+ 7 (u < PER / 2: a's, else b's; laid out as in fp8_gemm),
  // at 64 rows a unit from one lane offset. Through buffer descriptors that end with the matrix:
  // rows past it read as zeros. (256 rows stay below 2^31 bytes: K <= 2^22.)
  const auto ra = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<unsigned char*>(g.a) + (size_t)m0 * g.K, 0, (int)(min(g.M - m0, BM) * g.K), 0x00020000);
  const auto rb = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<unsigned char*>(g.b) + (size_t)n0 * g.K, 0, (int)(min(g.N - n0, BN) * g.K), 0x00020000);
  const int t0 = w * 8 + (lane >> 3);
  const unsigned off = (unsigned)slot_row(t0) * (unsigned)g.K + (((lane & 7) ^ ((t0 >> 1) & 7)) << 4);
  auto issue = [&](int kb, char* slot) {
    const int k = min(kb, nkb - 1) * 128;  // (past the end the last once more, unread)
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const unsigned at = off + (unsigned)(u % (PER / 2)) * 64u * (unsigned)g.K;
      lvoid* to = (lvoid*)(slot + (u * 8 + w) * 1024);
      if (u < PER / 2)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, to, 16, at, k, 0, 0);
      else
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, to, 16, at, k, 0, 0);
    }
  };
  const int r = lane & 15, q = lane >> 4, x = (r >> 1) & 7;
  const int lo = r * 128 + ((q ^ x) << 4), hi = r * 128 + (((q + 4) ^ x) << 4);
  auto frag = [&](const char* base, int f) {
    const i32x4 l = *reinterpret_cast<const i32x4*>(base + f * 2048 + lo);
    const i32x4 h = *reinterpret_cast<const i32x4*>(base + f * 2048 + hi);
    return __builtin_shufflevector(l, h, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  f32x4 acc[2][4][4];
#pragma unroll
  for (int i = 0; i < 32; ++i) (&acc[0][0][0])[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  int na[2], nb, ea[2], eb;
  auto exps = [&](int kb) {
    const int k = min(kb, nkb - 1);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      na[i] = exps4(g.sa, g.sa_str, A128 ? 7 : 0, k, m0 + (second * 2 + i) * 64, r);
    nb = exps4(g.sb, g.sb_str, B128 ? 7 : 0, k, n0 + wn * 64, r);
  };
  auto landed = [] {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  };
  auto turn = [] {
    __builtin_amdgcn_sched_barrier(0);
    lds_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  auto stage = [&](auto group, int kb, char* cur, char* other) {
    constexpr bool SECOND = decltype(group)::value;
#pragma unroll
    for (int i = 0; i < 2; ++i) ea[i] = spread(na[i], A128);
    eb = spread(nb, B128);
    i32x8 fb[4], fa[2][4];
#pragma unroll
    for (int f = 0; f < 4; ++f) fb[f] = frag(cur + BM * 128, wn * 4 + f);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int f = 0; f < 4; ++f) fa[i][f] = frag(cur, (SECOND * 2 + i) * 4 + f);
    __builtin_amdgcn_sched_barrier(0);  // LDS first: the other group's turn waits for it
    if (!SECOND) issue(kb + 1, other);
    if (SECOND) landed();
    exps(kb + 1);
    turn();
    if (SECOND) issue(kb + 2, cur);
#pragma unroll
    for (int i = 0; i < 2; ++i) quad<false>(fa[i], fb, ea[i], eb, acc[i]);
    if (!SECOND) landed();
    turn();
  };
  auto stages = [&](auto group) {
    for (int kb = 0; kb + 1 < nkb; kb += 2) {
      stage(group, kb, ring0, ring1);
      stage(group, kb + 1, ring1, ring0);
    }
    if (nkb & 1) stage(group, nkb - 1, ring0, ring1);
  };
  exps(0);
  issue(0, ring0);
  landed();
  turn();
  if (second) {
    issue(1, ring1);
    turn();
    stages(std::true_type());
  } else {
    stages(std::false_type());
    turn();
  }
  landed();  // nothing may arrive in LDS after the workgroup has ended

#pragma unroll
  for (int ga = 0; ga < 2; ++ga) {
    const int n = n0 + wn * 64 + 4 * r;
    const Column col = column(g, n);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int m = m0 + (second * 2 + ga) * 64 + 4 * (4 * q + e) + i;
        if (m >= g.M || n >= g.N) continue;
        put4<false>(g, col, m, n, f32x4{acc[ga][i][0][e], acc[ga][i][1][e], acc[ga][i][2][e],
                                        acc[ga][i][3][e]});
      }
  }
}

// the splits' partials, added in order, four columns a thread
template <bool WIDE>
__global__ __launch_bounds__(256) void fp8_gemm_join(GemmArgs g, int splits) {
  const size_t total = (size_t)g.M * g.N;
  const unsigned quads = (g.N + 3) / 4;
  const size_t all = (size_t)g.M * quads;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (size_t)gridDim.x * 256) {
    const int m = (int)(i / quads), n = 4 * (int)(i - (size_t)m * quads);
    const float* p = g.part + (size_t)m * g.N + n;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (n + 4 <= g.N) {
      s = *reinterpret_cast<const f32x4_any*>(p);
#pragma unroll 4
      for (int k = 1; k < splits; ++k) s += *reinterpret_cast<const f32x4_any*>(p + k * total);
    } else {
      for (int j = 0; n + j < g.N; ++j) {
        float t = p[j];
        for (int k = 1; k < splits; ++k) t += p[j + k * total];
        s[j] = t;
      }
    }
    put4<WIDE>(g, column(g, n), m, n, s);
  }
}

// The same for many splits of a small result: 16 threads share four columns, each adds every 16th
// split in order, then theirs are added in order (256 x 64 in 128 splits 12.6 -> 4 us).
template <bool WIDE>
__global__ __launch_bounds__(256) void fp8_gemm_join_many(GemmArgs g, int splits) {
  __shared__ f32x4 part[16][16];
  const unsigned quads = (g.N + 3) / 4;
  const size_t total = (size_t)g.M * g.N, all = (size_t)g.M * quads;
  const int l = threadIdx.x >> 4, c = threadIdx.x & 15;
  for (size_t i0 = (size_t)blockIdx.x * 16; i0 < all; i0 += (size_t)gridDim.x * 16) {
    const size_t i = i0 + c;
    const int m = (int)(i / quads), n = 4 * (int)(i - (size_t)m * quads);
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (i < all) {
      const float* p = g.part + (size_t)m * g.N + n;
      if (n + 4 <= g.N) {
#pragma unroll 4
        for (int k = l; k < splits; k += 16) s += *reinterpret_cast<const f32x4_any*>(p + k * total);
      } else {
        for (int j = 0; n + j < g.N; ++j)
          for (int k = l; k < splits; k += 16) s[j] += p[j + k * total];
      }
    }
    part[l][c] = s;
    __syncthreads();
    if (l == 0 && i < all) {
#pragma unroll
      for (int k = 1; k < 16; ++k) s += part[k][c];
      put4<WIDE>(g, column(g, n), m, n, s);
    }
    __syncthreads();
  }
}

// ---- few rows on one side (tokens being served): nothing to reuse, so no LDS for the operands.
// A workgroup takes 16 rows of the long side and all of K; its waves take the k blocks in
// turn, each lane loading its 32 bytes of a block straight into MFMA operands (whole 128-byte
// lines per four lanes), AHEAD blocks in flight; the waves' sums meet in LDS, in wave order.
//
// F: fragments (16 rows) of the short side. FUSED: the short side is not yet rounded; every
// workgroup rounds its 16 rows of x [S][C] on the way in, four lanes to a block of 128, which
// is cheaper than a launch for it (4096 x 4096, bf16: one token 6.4 us, 16 tokens 9.0 us, against
// 5.2 us behind a rounding kernel of 5).
template <int F, bool WIDE, bool FUSED>
__global__ __launch_bounds__(512) void fp8_gemm_few(GemmArgs g, int swap) {
  using T = std::conditional_t<WIDE, float, bf16_t>;
  static_assert(!FUSED || F == 1, "one fragment");
  constexpr int NW = 8, AHEAD = F > 1 || (FUSED && WIDE) ? 2 : 4;
  constexpr int V = ElemVec<T>::N, XV = FUSED ? 32 / V : 1;  // vectors of x a lane and block
  __shared__ float sum[NW][F][256];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  // short side s (F * 16 rows), long side l
  const unsigned char *sp = swap ? g.b : g.a, *lp = swap ? g.a : g.b;
  const unsigned char *se = swap ? g.sb : g.sa, *le = swap ? g.sa : g.sb;
  const long sstr = swap ? g.sb_str : g.sa_str, lstr = swap ? g.sa_str : g.sb_str;
  const int ssh = swap ? g.b_shift : g.a_shift, lsh = swap ? g.a_shift : g.b_shift;
  const int S = swap ? g.N : g.M, L = swap ? g.M : g.N;
  const int l0 = blockIdx.x * 16, lrow = min(l0 + r, L - 1);
  const unsigned char* lsrc = lp + (size_t)lrow * g.K + q * 16;
  const unsigned char* lexp = le + (lrow >> lsh);
  const unsigned char *ssrc[F], *sexp[F];
#pragma unroll
  for (int f = 0; f < F; ++f) {
    const int row = min(f * 16 + r, S - 1);
    ssrc[f] = sp + (size_t)row * g.K + q * 16;
    sexp[f] = se + (row >> ssh);
  }
  const T* xrow = FUSED ? static_cast<const T*>(g.x) + (size_t)min(r, S - 1) * g.x_cols : nullptr;
  f32x4 acc[F];
#pragma unroll
  for (int f = 0; f < F; ++f) acc[f] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto ld = [](const unsigned char* p) {
    const i32x4 l = *reinterpret_cast<const i32x4*>(p);
    const i32x4 h = *reinterpret_cast<const i32x4*>(p + 64);
    return __builtin_shufflevector(l, h, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  // U blocks from kb0: all their loads, then their products
  auto blocks = [&](int kb0, auto count) {
    constexpr int U = decltype(count)::value;
    i32x8 lv[U], sv[U][F];
    int el[U], es[U][F];
    u32x4 xv[U][XV];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      lv[u] = ld(lsrc + (size_t)(kb0 + u) * 128);
      el[u] = lexp[(size_t)(kb0 + u) * lstr];
      if constexpr (FUSED) {  // k 16q .. 16q + 15 of the block's lower half, then of its upper
#pragma unroll
        for (int i = 0; i < XV; ++i) {
          const int c = (kb0 + u) * 128 + (i / (XV / 2)) * 64 + q * 16 + (i % (XV / 2)) * V;
          xv[u][i] = c < g.x_cols ? ldv_raw(xrow + c, g.x_cols - c) : u32x4{0u, 0u, 0u, 0u};
        }
        continue;
      }
#pragma unroll
      for (int f = 0; f < F; ++f) {
        sv[u][f] = ld(ssrc[f] + (size_t)(kb0 + u) * 128);
        es[u][f] = sexp[f][(size_t)(kb0 + u) * sstr];
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (FUSED) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        using M = Mag<T>;
        auto largest = [&](auto clean) {
          unsigned m = 0;
#pragma unroll
          for (int i = 0; i < XV; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              m = M::join(m, M::template of<decltype(clean)::value>(xv[u][i][j]));
          return m;
        };
        unsigned m = largest(std::false_type());
        if (__any(M::odd(m))) m = largest(std::true_type());
        if constexpr (!WIDE) m = max(m >> 16, m & 0xffffu);
        const auto h = __builtin_amdgcn_permlane16_swap(m, m, false, false);
        m = max(h[0], h[1]);
        const auto g = __builtin_amdgcn_permlane32_swap(m, m, false, false);
        m = max(g[0], g[1]);
        es[u][0] = (int)M::exp_byte(m);
        const float sc = exp_scale((unsigned)es[u][0]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if constexpr (WIDE) {
            auto x = [&](int j) { return __uint_as_float(xv[u][i][j]); };
            sv[u][0][i] = (int)to_fp8x4(x(0), x(1), x(2), x(3), sc);
          } else {
            const u32x4 v = xv[u][i / 2];
            sv[u][0][i] = (int)to_fp8x4(v[2 * (i & 1)], v[2 * (i & 1) + 1], sc);
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int f = 0; f < F; ++f) {
        if constexpr (WIDE) {
#pragma unroll
          for (int p = 0; p < 4; ++p)
            acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                widen(sv[u][f], p, es[u][f]), widen(lv[u], p, el[u]), acc[f], 0, 0, 0);
        } else {
          acc[f] = mfma8<0, 0>(sv[u][f], lv[u], acc[f], es[u][f], el[u]);
        }
      }
  };
  const int whole = g.nkb / AHEAD;
  for (int c = w; c < whole; c += NW) blocks(c * AHEAD, std::integral_constant<int, AHEAD>());
  for (int kb = whole * AHEAD; kb < g.nkb; ++kb)
    if ((whole + kb) % NW == w) blocks(kb, std::integral_constant<int, 1>());
#pragma unroll
  for (int f = 0; f < F; ++f)
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[w][f][(4 * q + e) * 16 + r] = acc[f][e];
  __syncthreads();
  for (int i = threadIdx.x; i < F * 256; i += 512) {
    float t = 0.f;
#pragma unroll
    for (int v = 0; v < NW; ++v) t += sum[v][i >> 8][i & 255];
    const int s = i >> 4, l = l0 + (i & 15);
    if (s < S && l < L) put<WIDE>(g, swap ? out_at(g, l, s) : out_at(g, s, l), t);
  }
}

// How a product runs; the same for the workspace query and the call.
struct Plan {
  enum { FEW, SHORT, TILE128, TILE256 } kind;
  int splits, kb_split;
};

Plan plan(const dcn_fp8_matmul_desc& d) {
  const int few = std::min(d.M, d.N), nkb = d.K / 128;
  // One workgroup per 16 rows of the long side, all of K in it: a few tokens through a weight, as
  // long as fragments x k blocks x rounds of the card stay below 128. us, and in tiles: 16 tokens
  // 4096 x 4096 6.6, 12.7, 8192 x 8192 18, 20; 32 tokens 4096 x 4096 8.7, 12.9, 8192 x 8192 25, 21;
  // 64 tokens 4096 x 4096 12.7, 14.0, 4096 x 8192 22, 15.
  // Nor the weight gradient of few channels (few workgroups, the tokens as K) nor many tokens to
  // few channels (a workgroup reads the short side whole, and up to eight k blocks keep one wave
  // each): 64 x 256 channels over 200704 tokens, weight gradient 471 -> 27 us, input gradient
  // 94 -> 18; 64 x 64 over 50176 132 -> 13, 24 -> 6.
  const long wgs = (std::max(d.M, d.N) + 15L) / 16, frags = few <= 16 ? 1 : few <= 32 ? 2 : 4;
  if (few <= 64 && wgs <= 1024 && nkb <= 64 &&
      frags * std::max(nkb, 8) * std::max(256L, wgs) <= 128 * 256)
    return {Plan::FEW, 1, nkb};
  auto tiles = [&](int b) { return (long)((d.M + b - 1) / b) * ((d.N + b - 1) / b); };
  // A short K is all prologue and epilogue: three small workgroups a CU that take turns at them
  // beat one large one that overlaps its own stages (50176 x 1024 bf16 results, K = 256 / 512 /
  // 1024: 30 / 40 / 64 us, one stage in LDS; two stages 35 / 49 / 78; 256 x 256 tiles 36 / 47 / 66).
  if (nkb <= 8 && tiles(128) >= 768) return {Plan::SHORT, 1, nkb};
  // 256 x 256: half the LDS reads per product (16384 x 8192 x 8192, bf16: 0.94 ms; 128 x 128 1.7 ms)
  if (few > 128 && tiles(256) >= 192) return {Plan::TILE256, 1, nkb};
  // Fewer tiles than CUs: parts of K, at least eight k blocks each, up to one workgroup a CU. (More
  // parts cost more in the joining than they save: 2048 x 2048 x 2048, 256 tiles, whole 16 us, in two
  // parts 16 + 7.5; 300 x 4096 x 4096, 96 tiles, whole 25, in two 17 + 4, in five 15 + 5.5;
  // 1777 x 1500 x 1000 in fp32, 168 tiles, whole 14, in two 15 + 6.)
  const long t = tiles(128);
  int splits = (int)std::min<long>(std::max<long>(1, 256 / t), std::max(1, nkb / 8));
  const int kb = (nkb + splits - 1) / splits;
  splits = (nkb + kb - 1) / kb;
  return {Plan::TILE128, splits, kb};
}

template <int GA, int GB, int WM, int WN, int WPE, int STAGES>
hipError_t run_tiles(GemmArgs g, const Plan& p, bool wide, hipStream_t s) {
  g.tiles_m = (g.M + WM * GA * 64 - 1) / (WM * GA * 64);
  g.tiles_n = (g.N + WN * GB * 64 - 1) / (WN * GB * 64);
  g.kb_split = p.kb_split;
  const dim3 grid((unsigned)g.tiles_m * g.tiles_n, p.splits), block(WM * WN * 64);
  if (p.splits == 1) {
    if (wide)
      hipLaunchKernelGGL((fp8_gemm<GA, GB, WM, WN, WPE, STAGES, true, false>), grid, block, 0, s, g);
    else
      hipLaunchKernelGGL((fp8_gemm<GA, GB, WM, WN, WPE, STAGES, false, false>), grid, block, 0, s, g);
    return hipGetLastError();
  }
  if (wide)
    hipLaunchKernelGGL((fp8_gemm<GA, GB, WM, WN, WPE, STAGES, true, true>), grid, block, 0, s, g);
  else
    hipLaunchKernelGGL((fp8_gemm<GA, GB, WM, WN, WPE, STAGES, false, true>), grid, block, 0, s, g);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const size_t quads = (size_t)g.M * ((g.N + 3) / 4);
  if (p.splits > 16) {
    const dim3 n((unsigned)std::min<size_t>((quads + 15) / 16, 4096));
    if (wide)
      hipLaunchKernelGGL(fp8_gemm_join_many<true>, n, dim3(256), 0, s, g, p.splits);
    else
      hipLaunchKernelGGL(fp8_gemm_join_many<false>, n, dim3(256), 0, s, g, p.splits);
  } else {
    const dim3 n((unsigned)std::min<size_t>((quads + 255) / 256, 4096));
    if (wide)
      hipLaunchKernelGGL(fp8_gemm_join<true>, n, dim3(256), 0, s, g, p.splits);
    else
      hipLaunchKernelGGL(fp8_gemm_join<false>, n, dim3(256), 0, s, g, p.splits);
  }
  return hipGetLastError();
}

template <int F, bool FUSED>
hipError_t run_few(const GemmArgs& g, bool wide, hipStream_t s) {
  const int swap = !FUSED && g.N < g.M, longest = swap ? g.M : g.N;
  const dim3 grid((longest + 15) / 16), block(512);
  if (wide)
    hipLaunchKernelGGL((fp8_gemm_few<F, true, FUSED>), grid, block, 0, s, g, swap);
  else
    hipLaunchKernelGGL((fp8_gemm_few<F, false, FUSED>), grid, block, 0, s, g, swap);
  return hipGetLastError();
}

GemmArgs gemm_args(const dcn_fp8_matmul_desc& d) {
  GemmArgs g{};
  g.M = d.M;
  g.N = d.N;
  g.K = d.K;
  g.nkb = d.K / 128;
  g.P = d.P;
  g.nchw = d.layout == DCN_NCHW;
  g.a_shift = d.a_block == 128 ? 7 : 0;
  g.b_shift = d.b_block == 128 ? 7 : 0;
  g.sa_str = d.a_block == 128 ? (d.M + 127) / 128 : (d.M + 127) / 128 * 128;
  g.sb_str = d.b_block == 128 ? (d.N + 127) / 128 : (d.N + 127) / 128 * 128;
  return g;
}

const unsigned char* u8(const void* p) { return static_cast<const unsigned char*>(p); }

}  // namespace

size_t fp8_matmul_ws_bytes(const dcn_fp8_matmul_desc& d) {
  const Plan p = plan(d);
  return p.splits > 1 ? (size_t)p.splits * d.M * d.N * sizeof(float) : 0;
}

hipError_t launch_fp8_matmul(const dcn_fp8_matmul_desc& d, const void* a, const void* sa,
                             const void* b, const void* sb, void* out, void* ws, hipStream_t s) {
  GemmArgs g = gemm_args(d);
  g.a = u8(a);
  g.sa = u8(sa);
  g.b = u8(b);
  g.sb = u8(sb);
  g.out = out;
  g.part = static_cast<float*>(ws);
  const bool wide = d.out_dtype == DCN_F32;
  const Plan p = plan(d);
  if (p.kind == Plan::FEW) {
    const int few = std::min(d.M, d.N);
    return few <= 16 ? run_few<1, false>(g, wide, s) : few <= 32 ? run_few<2, false>(g, wide, s)
                                                          : run_few<4, false>(g, wide, s);
  }
  if (p.kind == Plan::TILE256 && !wide && d.K <= 1 << 22) {
    g.tiles_m = (g.M + 255) / 256;
    g.tiles_n = (g.N + 255) / 256;
    const dim3 grid((unsigned)g.tiles_m * g.tiles_n), block(512);
    if (g.a_shift && g.b_shift)
      hipLaunchKernelGGL((fp8_gemm_turns<true, true>), grid, block, 0, s, g);
    else if (g.a_shift)
      hipLaunchKernelGGL((fp8_gemm_turns<true, false>), grid, block, 0, s, g);
    else if (g.b_shift)
      hipLaunchKernelGGL((fp8_gemm_turns<false, true>), grid, block, 0, s, g);
    else
      hipLaunchKernelGGL((fp8_gemm_turns<false, false>), grid, block, 0, s, g);
    return hipGetLastError();
  }
  if (p.kind == Plan::TILE256) return run_tiles<2, 1, 2, 4, 2, 2>(g, p, wide, s);
  if (p.kind == Plan::SHORT) return run_tiles<1, 1, 2, 2, 3, 1>(g, p, wide, s);
  return run_tiles<1, 1, 2, 2, 2, 2>(g, p, wide, s);
}

bool fp8_few_tokens(size_t tokens) { return tokens <= 16; }

hipError_t launch_fp8_few_tokens(const dcn_fp8_matmul_desc& d, int cols, const void* x,
                                 const void* w, const void* sw, void* out, hipStream_t s) {
  GemmArgs g = gemm_args(d);
  g.x = x;
  g.x_cols = cols;
  g.b = u8(w);
  g.sb = u8(sw);
  g.out = out;
  return run_few<1, true>(g, d.out_dtype == DCN_F32, s);
}

}  // namespace dcn
