// dcn_block_norm.h — kernels of the operator between two residual blocks (include/dcn.h, block norms):
//   t = drop(alpha · scale[c] · act(gate) · N_post(x)), out = residual + t, y = N_pre(out)
// over the C channels of every position, and its backward.
//
// Backward, with h = (v - m) · r the normalised values of a norm and a = g · w:
//   N'(g) = r · (a - [layer] mean(a) - h · mean(a h)),  ∂w = Σ g h,  ∂b = Σ g
//   G  = ∂out + N_pre'(∂y)                 (= ∂residual)
//   dt = keep ? G · drop scale : 0
//   ∂gate = dt · N_post(x) · alpha · scale · act'(gate),  ∂scale = Σ dt · N_post(x) · alpha · act
//   ∂x = N_post'(dt · alpha · scale · act)
// What dropout drops reaches no gradient, NaN and infinities neither: x and a full gate count as 0
// in those products, an image gate's are left out (a dropped image's are not even read).
// out is computed again from x and the residual (the residual is read instead of out, so that
// costs no bytes), which keeps the backward free of out's rounding. The statistics come from
// the forward where the caller kept them: 16 bytes a position, against two of the four rounds
// of sums that a position's workgroup goes through.
#pragma once
#include <algorithm>
#include <cstdlib>

#include "dcn_block.h"
#include "dcn_philox.h"

namespace dcn {

// register-resident variants (dcn_block_map_*.hip, dcn_block_row_*.hip): false where there is
// none for this many channels, else *e is the launch's result
bool block_map_fwd(const BlockArgs& a, hipStream_t s, hipError_t* e);
bool block_map_bwd(const BlockArgs& a, hipStream_t s, hipError_t* e);
bool block_row_fwd(const BlockArgs& a, hipStream_t s, hipError_t* e);
bool block_row_bwd(const BlockArgs& a, hipStream_t s, hipError_t* e);

namespace {

// sigmoid(g) and 1 - sigmoid(g), both from e = exp(-|g|): e / (1 + e) and 1 / (1 + e) cancel
// nowhere, and 1 + e lies in [1, 2], where the hardware's reciprocal (1 ulp) has its full range.
// fp32: expf (1 ulp), so each is within 8 · 2^-24 of its value for every finite g. bf16: exp2 of a
// rounded product, (9 + 2 |g|) 2^-24 down to g = -87 and 0 below, 300 times finer than the result's
// half step (with expf 8x1024x4096 rows with a full gate 78 -> 83 us forward, 123 -> 145 backward).
template <typename T>
__device__ __forceinline__ void sigmoids(float g, float& s, float& rest) {
  const float e = sizeof(T) == 2 ? __expf(-fabsf(g)) : expf(-fabsf(g));
  const float r = __builtin_amdgcn_rcpf(1.f + e), er = e * r;
  s = g < 0.f ? er : r;
  rest = g < 0.f ? r : er;
}
// act(g) and act'(g)
template <typename T>
__device__ __forceinline__ float gate_act(float g, int act) {
  if (act == DCN_ACT_LINEAR) return g;
  float s, rest;
  sigmoids<T>(g, s, rest);
  return act == DCN_ACT_SIGMOID ? s : g * s;
}
template <typename T>
__device__ __forceinline__ void gate_act_grad(float g, int act, float& a, float& d) {
  a = g;
  d = 1.f;
  if (act == DCN_ACT_LINEAR) return;
  float s, rest;
  sigmoids<T>(g, s, rest);
  a = act == DCN_ACT_SIGMOID ? s : g * s;
  d = act == DCN_ACT_SIGMOID ? s * rest : s * fmaf(g, rest, 1.f);
}

// ---- one pass: the channels of a tile of positions stay in registers ----------------------
// Both layouts share the plan: work is cut into tiles (maps: TP neighbouring positions of an
// image, rows: one row per LPR lanes), a workgroup's tiles lie in one run of neighbours, and a
// thread keeps the same channels in every tile, so its parameter gradients add up in registers.
// They leave once per workgroup as partials [workgroup][5][C] (scale, w1, b1, w2, b2), an image
// gate's once per workgroup and image, and block_fold adds them in a fixed order.
//
// `group` workgroups share a run and take its tiles in turn. Neighbouring tiles of maps share
// the cache lines that straddle them (a channel's row starts anywhere, and 32 bf16 positions
// are half a line); taken at the same time they are fetched once (64x256x28x28 backward, runs of
// one workgroup against interleaved: bf16 68 -> 54 us, fp32 107 -> 94 us).
struct Plan {
  int tpi;            // tiles of an image
  long tiles;         // of the call
  int wgs, group;     // run g of wgs / group has tiles [first_tile(g), first_tile(g + 1))
  int images, P;      // rows without an image gate count as one image
  bool image_gate;    // ∂gate sums over positions
  // [wgs][5][C], and a row of C for workgroup j of run g at image b in slot (g + b) · group + j
  // (g + b grows along the runs and their images, so no two share a slot)
  float *part, *gpart;
  float* rowst;  // [6][rows]: m1, r1, m2, r2, mean(a2), mean(a2 h2) of long rows (N_pre's a and h)
};

__host__ __device__ __forceinline__ long first_tile(const Plan& q, int run) {
  return q.tiles * run / (q.wgs / q.group);
}

// the workgroups that share an XCD (equal index mod 8) take neighbouring ranges
__device__ __forceinline__ int xcd_wg(int n) {
  const int bid = blockIdx.x, q = n >> 3, r = n & 7, x = bid & 7;
  return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (bid >> 3);
}

// Σ over aligned groups of LPR lanes; every lane gets the sum. VALU only (DPP mirrors and
// lane-row swaps), fixed order.
template <int LPR>
__device__ __forceinline__ float group_sum(float v) {
  if constexpr (LPR >= 2) v += dpp_f<0xB1>(v);
  if constexpr (LPR >= 4) v += dpp_f<0x4E>(v);
  if constexpr (LPR >= 8) v += dpp_f<0x141>(v);
  if constexpr (LPR >= 16) v += dpp_f<0x140>(v);
  if constexpr (LPR >= 32) v = swap_fold16(v);
  if constexpr (LPR >= 64) v = swap_fold32(v);
  return v;
}
// keep bits of the V elements from i
template <int V>
__device__ __forceinline__ unsigned keepv(uint64_t i, const PhiloxKey& k, unsigned thr) {
  const unsigned s = (unsigned)(i & 7);
  unsigned m = keep8(i >> 3, k, thr) >> s;
  if (s + V > 8) m |= keep8((i >> 3) + 1, k, thr) << (8 - s);
  return m;
}

// ---- maps [B][C][P]: PL lanes of one vector along the positions, NT / PL channel groups, channels
// cg + CG · i of a thread, i < CPT.
//
// Sums over the channels of every position. A thread's partial sums of its V positions go
// through LDS twice: inside the wave (its GPW channel groups x TP positions, each lane then adds
// a column's share), then between the waves; finally every wave finishes all TP positions for
// itself, one lane each, and the threads read their V results back. Done in registers instead
// (V values through DPP rotations, every thread finishing all its positions) the same sums took
// two thirds of the kernel's instructions.
template <int NT, int PL, int V, int CPT>
struct MapSums {
  static constexpr int TP = PL * V, NW = NT / 64, GPW = 64 / PL, CG = NT / PL;
  static constexpr int SHARE = 64 / TP, EACH = GPW / SHARE;  // lanes a position, groups a lane
  static_assert(TP <= 64 && SHARE * TP == 64 && EACH * SHARE == GPW, "lanes cover the positions");
  struct Shared {
    float wave[NW][2][GPW][TP];  // a wave's partials (two quantities)
    float join[2][NW][2][TP];    // waves' sums, alternating: read in a round, written in the next
                                 // but one
    float res[NW][6][TP];        // a wave's copy of m1, r1, m2, r2 and of a pair of sums
    float2 num[NW];              // channels of every wave and 1 / that (0 of 0)
  };
  Shared& sh;
  int w, lane, pl, gl, C, phase = 0;
  float inw;  // 1 / channels of this wave
  __device__ MapSums(Shared& s, int c) : sh(s), C(c) {
    w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    lane = threadIdx.x & 63;
    pl = threadIdx.x % PL;
    gl = lane / PL;
    const float n = count(w);
    inw = n > 0.f ? 1.f / n : 0.f;
    if (lane == 0) sh.num[w] = make_float2(n, inw);  // read behind the first join's barrier
  }
  __device__ float count(int wave) const {  // channels of a wave
    int n = 0;
#pragma unroll
    for (int i = 0; i < CPT; ++i) n += min(max(C - (CG * i + wave * GPW), 0), GPW);
    return (float)n;
  }
  // LDS accesses of one wave happen in order; this keeps the compiler to it
  static __device__ __forceinline__ void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  __device__ void put(int k, const float (&v)[V]) {
    float* d = &sh.wave[w][k][gl][pl * V];
#pragma unroll
    for (int e = 0; e < V; e += 4)
      *reinterpret_cast<float4*>(d + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
  }
  // the wave's sum of quantity k at position lane % TP
  __device__ float column(int k) const {
    const float* d = &sh.wave[w][k][(lane / TP) * EACH][lane % TP];
    float t = d[0];
#pragma unroll
    for (int i = 1; i < EACH; ++i) t += d[i * TP];
    if constexpr (SHARE >= 2) t = swap_fold32(t);
    if constexpr (SHARE >= 4) t = swap_fold16(t);
    return t;
  }
  __device__ void get(int k, float (&v)[V]) const {
    const float* d = &sh.res[w][k][pl * V];
#pragma unroll
    for (int e = 0; e < V; e += 4) {
      const float4 f = *reinterpret_cast<const float4*>(d + e);
      v[e] = f.x;
      v[e + 1] = f.y;
      v[e + 2] = f.z;
      v[e + 3] = f.w;
    }
  }
  __device__ void give(int k, float v) {
    if (lane < TP) sh.res[w][k][lane] = v;
  }
  // Σ over all channels, a times fa, b times fb
  __device__ void sum2(float (&a)[V], float (&b)[V], float fa, float fb) {
    put(0, a);
    put(1, b);
    wave_order();
    float ta = column(0), tb = column(1);
    if constexpr (NW > 1) {
      phase ^= 1;
      if (lane < TP) {
        sh.join[phase][w][0][lane] = ta;
        sh.join[phase][w][1][lane] = tb;
      }
      lds_barrier();
      ta = tb = 0.f;
#pragma unroll
      for (int v = 0; v < NW; ++v) {
        ta += sh.join[phase][v][0][lane % TP];
        tb += sh.join[phase][v][1][lane % TP];
      }
    }
    give(4, ta * fa);
    give(5, tb * fb);
    wave_order();
    get(4, a);
    get(5, b);
    wave_order();
  }
  // Mean and 1/sqrt(var + eps) of each position (0 past the map's end, `left` = positions of
  // the tile, so that nothing from there reaches the parameter sums); mk: 1 for a channel, 0
  // past the last (its v is 0). Layer: every wave takes its own mean and the squares about it;
  // the waves' are joined about the whole mean, so large means cancel nowhere.
  // The results go to rows k and k + 1 of the wave's copies, and to `stats` where wanted.
  __device__ void moments(const float (&v)[CPT][V], const float (&mk)[CPT], int kind, float eps,
                          int left, int k, float* stats, size_t rows) {
    float t[V], m[V], s = 0.f, q;
    if (kind == DCN_NORM_LAYER) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        t[e] = v[0][e];
#pragma unroll
        for (int i = 1; i < CPT; ++i) t[e] += v[i][e];
      }
      put(0, t);
      wave_order();
      s = column(0);
      give(4, s * inw);
      wave_order();
      get(4, m);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        t[e] = 0.f;
#pragma unroll
        for (int i = 0; i < CPT; ++i) {
          const float d = fmaf(-m[e], mk[i], v[i][e]);
          t[e] = fmaf(d, d, t[e]);
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        t[e] = v[0][e] * v[0][e];
#pragma unroll
        for (int i = 1; i < CPT; ++i) t[e] = fmaf(v[i][e], v[i][e], t[e]);
      }
    }
    put(1, t);
    wave_order();
    q = column(1);
    const float ic = 1.f / (float)C;
    if constexpr (NW > 1) {
      phase ^= 1;
      if (lane < TP) {
        sh.join[phase][w][0][lane] = s;
        sh.join[phase][w][1][lane] = q;
      }
      lds_barrier();
      q = 0.f;
#pragma unroll
      for (int x = 0; x < NW; ++x) q += sh.join[phase][x][1][lane % TP];
      if (kind == DCN_NORM_LAYER) {
        float sx[NW];
        s = 0.f;
#pragma unroll
        for (int x = 0; x < NW; ++x) {
          sx[x] = sh.join[phase][x][0][lane % TP];
          s += sx[x];
        }
#pragma unroll
        for (int x = 0; x < NW; ++x) {
          const float2 n = sh.num[x];
          const float d = fmaf(sx[x], n.y, -s * ic);  // a wave without channels: s and n are 0
          q = fmaf(n.x * d, d, q);
        }
      }
    }
    const float mean = s * ic, rs = lane % TP < left ? rsqrtf(fmaf(q, ic, eps)) : 0.f;
    give(k, mean);
    give(k + 1, rs);
    wave_order();
    if (stats && w == 0 && lane < TP && lane < left) {
      stats[k * rows + lane] = mean;
      stats[(k + 1) * rows + lane] = rs;
    }
  }
  // kept statistics of a tile: lane + 64 i of the 4 x TP values, fetched ahead of their use
  static constexpr int KEPT = TP / 16;
  __device__ void fetch(const float* stats, size_t rows, int left, float (&st)[KEPT]) const {
#pragma unroll
    for (int i = 0; i < KEPT; ++i) {
      const int j = lane + 64 * i, p = j % TP;
      st[i] = p < left ? stats[(j / TP) * rows + p] : 0.f;
    }
  }
  __device__ void keep(const float (&st)[KEPT]) {
#pragma unroll
    for (int i = 0; i < KEPT; ++i) {
      const int j = lane + 64 * i;
      sh.res[w][j / TP][j % TP] = st[i];
    }
    wave_order();
  }
};

template <typename T>
__device__ __forceinline__ float par(const void* t, int c, float none) {
  return t ? to_f32(static_cast<const T*>(t)[c]) : none;
}

template <typename T, int NT, int PL, int CPT, int WPE, bool AHEAD, bool BWD, bool FULL, bool DROP>
__global__ __launch_bounds__(NT, WPE) void block_map(BlockArgs a, Plan q) {
  constexpr int V = ElemVec<T>::N, TP = PL * V, CG = NT / PL;
  using Sums = MapSums<NT, PL, V, CPT>;
  __shared__ __attribute__((aligned(16))) typename Sums::Shared shared;
  const PhiloxKey key = philox_key(a.drop);
  const int pl = threadIdx.x % PL, cg = threadIdx.x / PL;
  Sums sums(shared, a.C);
  const int wg = xcd_wg(q.wgs);
  const T *xp = static_cast<const T*>(a.x), *rp = static_cast<const T*>(a.res);
  const T* gp = static_cast<const T*>(a.gate);

  bool inc[CPT];
  float mk[CPT];
  float sc[CPT], w1[CPT], b1[CPT], w2[CPT], b2[CPT];
  // accd: Σ dt · N_post(x) under one gate (an image's, or none), from which its ∂gate and ∂scale
  // follow at its end; seen: channels of which anything was kept
  float acc[5][CPT], accd[CPT];
  unsigned seen = 0u;
#pragma unroll
  for (int i = 0; i < CPT; ++i) {
    const int c = cg + CG * i;
    inc[i] = c < a.C;
    mk[i] = inc[i] ? 1.f : 0.f;
    sc[i] = a.alpha * (inc[i] ? par<T>(a.scale, c, 1.f) : 0.f);
    w1[i] = inc[i] ? par<T>(a.w1, c, 1.f) : 0.f;
    b1[i] = inc[i] ? par<T>(a.b1, c, 0.f) : 0.f;
    w2[i] = inc[i] ? par<T>(a.w2, c, 1.f) : 0.f;
    b2[i] = inc[i] ? par<T>(a.b2, c, 0.f) : 0.f;
#pragma unroll
    for (int k = 0; k < 5; ++k) acc[k][i] = 0.f;
    accd[i] = 0.f;
  }
  const int run = wg / q.group, turn = wg % q.group;
  const long t0 = first_tile(q, run) + turn, t1 = first_tile(q, run + 1), ts = q.group;
  struct Raw {
    u32x4 x[CPT], r[CPT], g[CPT], y[CPT], o[CPT];
    float st[Sums::KEPT];
    bool gone;  // the image is dropped
  } nx;
  const size_t rows = (size_t)a.B * a.P;
  auto load = [&](long t, Raw& w) {
    const int p = (int)(t % q.tpi) * TP + pl * V, valid = a.P - p;
    if (BWD && a.stats)
      sums.fetch(a.stats + (t / q.tpi) * a.P + t % q.tpi * TP, rows,
                 a.P - (int)(t % q.tpi) * TP, w.st);
    const size_t base = (size_t)(t / q.tpi) * a.C * a.P + p;
    const u32x4 zero = {0u, 0u, 0u, 0u};
    w.gone = false;
    if constexpr (DROP) w.gone = a.drop_image && !keep1(t / q.tpi, key, a.drop.thr);
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const bool ok = inc[i] && valid > 0;
      const size_t at = base + (size_t)(cg + CG * i) * a.P;
      w.x[i] = ok && xp && !w.gone ? ldv_raw(xp + at, valid) : zero;
      w.r[i] = ok && rp ? ldv_raw(rp + at, valid) : zero;
      if constexpr (FULL) w.g[i] = ok && !w.gone ? ldv_raw(gp + at, valid) : zero;
      if constexpr (BWD) {
        w.y[i] = ok && a.gy ? ldv_raw(static_cast<const T*>(a.gy) + at, valid) : zero;
        w.o[i] = ok && a.go ? ldv_raw(static_cast<const T*>(a.go) + at, valid) : zero;
      }
    }
  };
  // an image gate's act and act', kept while the tiles stay in one image (read for every tile
  // they cost 64x256x28x28 10 us of 45)
  float gv[CPT], gd[CPT];
  int gb = -1;
#pragma unroll
  for (int i = 0; i < CPT; ++i) {
    gv[i] = 1.f;
    gd[i] = 0.f;
  }
  if (AHEAD && t0 < t1) load(t0, nx);
  for (long t = t0; t < t1; t += ts) {
    const int b = (int)(t / q.tpi), p = (int)(t % q.tpi) * TP + pl * V, valid = a.P - p;
    const int left = a.P - (int)(t % q.tpi) * TP;
    const size_t base = (size_t)b * a.C * a.P + p;
    bool ok[CPT];
    size_t at[CPT];
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      ok[i] = inc[i] && valid > 0;
      at[i] = base + (size_t)(cg + CG * i) * a.P;
    }
    if (!AHEAD) load(t, nx);
    const Raw in = nx;
    if (AHEAD && t + ts < t1) load(t + ts, nx);
    if (a.gate_kind == DCN_GATE_IMAGE && b != gb) {
      gb = b;
#pragma unroll
      for (int i = 0; i < CPT; ++i) {
        gv[i] = 1.f;  // (a dropped image's gate: nothing of another image's may stay)
        gd[i] = 0.f;
        if (inc[i] && !in.gone)
          gate_act_grad<T>(to_f32(gp[(size_t)b * a.C + cg + CG * i]), a.act, gv[i], gd[i]);
      }
    }
    unsigned keep[CPT];
    if constexpr (DROP) {
      // past the map's end nothing is kept (a gate that is not finite may not reach the sums there)
      const unsigned img = in.gone ? 0u : 0xffu, in_map = valid < V ? (1u << max(valid, 0)) - 1u : ~0u;
#pragma unroll
      for (int i = 0; i < CPT; ++i)
        keep[i] = (a.drop_image ? img : keepv<V>(at[i], key, a.drop.thr)) & in_map;
    }
    auto kept = [&](int i, int e, float t) {
      if constexpr (DROP) return (keep[i] >> e) & 1u ? t : 0.f;
      return t;
    };
    auto drop = [&](int i, int e, float t) {
      if constexpr (DROP) return kept(i, e, t * a.drop.scale);
      return t;
    };

    float* st = a.stats && !BWD ? a.stats + (size_t)b * a.P + (t % q.tpi) * TP : nullptr;
    const bool known = BWD && a.stats;
    if (known) sums.keep(in.st);
    auto post = [&](float (&m)[V], float (&r)[V]) {
      if (a.post && !in.gone) {
        sums.get(0, m);
        sums.get(1, r);
        return;
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {  // no post norm: N_post(x) = x (a dropped image's x is 0)
        m[e] = 0.f;
        r[e] = 1.f;
      }
    };
    float o[CPT][V];
    if (xp) {
      if (a.post && !known) {
        float xv[CPT][V];
#pragma unroll
        for (int i = 0; i < CPT; ++i) unpack<T>(in.x[i], xv[i]);
        sums.moments(xv, mk, a.post, a.eps1, left, 0, st, rows);
      }
      float m1[V], r1[V];
      post(m1, r1);
#pragma unroll
      for (int i = 0; i < CPT; ++i) {
        float xv[V], rv[V], fv[V];
        const float k = sc[i] * gv[i];
        unpack<T>(in.x[i], xv);
        unpack<T>(in.r[i], rv);
        if constexpr (FULL) unpack<T>(in.g[i], fv);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float v = fmaf((xv[e] - m1[e]) * r1[e], w1[i], b1[i]);
          o[i][e] = rv[e] + drop(i, e, v * (FULL ? sc[i] * gate_act<T>(fv[e], a.act) : k));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < CPT; ++i) unpack<T>(in.r[i], o[i]);
    }
    if (a.pre && !known) sums.moments(o, mk, a.pre, a.eps2, left, 2, st, rows);

    if constexpr (!BWD) {
      float m2[V], r2[V];
      if (a.pre) {
        sums.get(2, m2);
        sums.get(3, r2);
      }
      Sums::wave_order();  // read before the next tile's are written
#pragma unroll
      for (int i = 0; i < CPT; ++i) {
        if (!ok[i]) continue;
        if (a.pre) {
          float y[V];
#pragma unroll
          for (int e = 0; e < V; ++e) y[e] = fmaf((o[i][e] - m2[e]) * r2[e], w2[i], b2[i]);
          stv(static_cast<T*>(a.y) + at[i], valid, y);
        }
        if (a.out) stv(static_cast<T*>(a.out) + at[i], valid, o[i]);
      }
    } else {
      // G into o
      if (a.pre) {
        float s1[V], s2[V], m2[V], r2[V];
        sums.get(2, m2);
        sums.get(3, r2);
#pragma unroll
        for (int e = 0; e < V; ++e) s1[e] = s2[e] = 0.f;
#pragma unroll
        for (int i = 0; i < CPT; ++i) {
          float gy[V];
          unpack<T>(in.y[i], gy);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float h = (o[i][e] - m2[e]) * r2[e], w = gy[e] * w2[i];
            o[i][e] = h;
            s1[e] += w;
            s2[e] = fmaf(w, h, s2[e]);
            acc[3][i] = fmaf(gy[e], h, acc[3][i]);
            acc[4][i] += gy[e];
          }
        }
        const float ic = 1.f / (float)a.C;
        sums.sum2(s1, s2, a.pre == DCN_NORM_LAYER ? ic : 0.f, ic);
#pragma unroll
        for (int i = 0; i < CPT; ++i) {
          float gy[V], go[V];
          unpack<T>(in.y[i], gy);
          unpack<T>(in.o[i], go);
#pragma unroll
          for (int e = 0; e < V; ++e)
            o[i][e] = fmaf(r2[e], gy[e] * w2[i] - s1[e] - o[i][e] * s2[e], go[e]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < CPT; ++i) unpack<T>(in.o[i], o[i]);
      }
      if (a.gr) {
#pragma unroll
        for (int i = 0; i < CPT; ++i)
          if (ok[i]) stv(static_cast<T*>(a.gr) + at[i], valid, o[i]);
      }
      if (xp) {
        // dt, ∂gate, ∂scale; dv into o
        float s3[V], s4[V], m1[V], r1[V];
        post(m1, r1);
        Sums::wave_order();  // read before the next tile's are written
#pragma unroll
        for (int e = 0; e < V; ++e) s3[e] = s4[e] = 0.f;
#pragma unroll
        for (int i = 0; i < CPT; ++i) {
          float xv[V], fv[V], gg[V];
          const float k = sc[i] * gv[i];
          unpack<T>(in.x[i], xv);
          if constexpr (DROP && !FULL) seen |= (unsigned)(keep[i] != 0u) << i;
          if constexpr (FULL) unpack<T>(in.g[i], fv);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float h = kept(i, e, (xv[e] - m1[e]) * r1[e]), v = fmaf(h, w1[i], b1[i]);
            const float dt = drop(i, e, o[i][e]), dtv = dt * v;
            float dv;
            if constexpr (FULL) {
              float av, ad;
              gate_act_grad<T>(kept(i, e, fv[e]), a.act, av, ad);
              dv = dt * (sc[i] * av);
              gg[e] = dtv * (sc[i] * ad);
              acc[0][i] = fmaf(dtv, a.alpha * av, acc[0][i]);
            } else {
              dv = kept(i, e, dt * k);  // (0 times a gate that is not finite is not 0)
              accd[i] += dtv;
            }
            acc[1][i] = fmaf(dv, h, acc[1][i]);
            acc[2][i] += dv;
            o[i][e] = dv;
            const float w = dv * w1[i];
            s3[e] += w;
            s4[e] = fmaf(w, h, s4[e]);
          }
          if (FULL && a.gg && ok[i])
            stv(static_cast<T*>(a.gg) + at[i], valid, gg);
        }
        if (a.gx) {
          if (a.post) {
            const float ic = 1.f / (float)a.C;
            sums.sum2(s3, s4, a.post == DCN_NORM_LAYER ? ic : 0.f, ic);
          }
#pragma unroll
          for (int i = 0; i < CPT; ++i) {
            if (!ok[i]) continue;
            if (a.post) {
              float xv[V];
              unpack<T>(in.x[i], xv);
#pragma unroll
              for (int e = 0; e < V; ++e) {
                const float h = (xv[e] - m1[e]) * r1[e];
                o[i][e] = r1[e] * (o[i][e] * w1[i] - s3[e] - h * s4[e]);
              }
            }
            stv(static_cast<T*>(a.gx) + at[i], valid, o[i]);
          }
        }
        // the last tile of this gate
        if (!FULL && (t + ts >= t1 || (a.gate_kind == DCN_GATE_IMAGE && (t + ts) / q.tpi != b))) {
          float* dst =
              q.image_gate ? q.gpart + ((size_t)(run + b) * q.group + turn) * a.C : nullptr;
#pragma unroll
          for (int i = 0; i < CPT; ++i) {
            const bool any = !DROP || (seen >> i & 1u);
            acc[0][i] = any ? fmaf(accd[i], a.alpha * gv[i], acc[0][i]) : acc[0][i];
            if (q.image_gate) {
              const float g = group_sum<PL>(any ? accd[i] * (sc[i] * gd[i]) : 0.f);
              if (inc[i] && pl == 0) dst[cg + CG * i] = g;
            }
            accd[i] = 0.f;
          }
          seen = 0u;
        }
      }
    }
  }
  if constexpr (BWD) {
    if (!q.part) return;
#pragma unroll
    for (int i = 0; i < CPT; ++i)
#pragma unroll
      for (int k = 0; k < 5; ++k) {
        const float g = group_sum<PL>(acc[k][i]);
        if (inc[i] && pl == 0) q.part[((size_t)wg * 5 + k) * a.C + cg + CG * i] = g;
      }
  }
}

// ---- rows [B][P][C]: LPR lanes a row, NV vectors a lane (channels (lane + LPR · j) · V ..), NT / LPR
// rows of one image at a time. LPR <= 64: a row stays inside a wave and its sums are lane
// exchanges; above, a workgroup holds one row and the waves join through LDS.
template <int NT, int LPR, int V, int NV>
struct RowSums {
  static constexpr int NW = LPR > 64 ? LPR / 64 : 1, GR = NT / LPR;
  struct Shared {
    float join[2][GR][NW][2];  // alternating, as in MapSums
    float2 num[NW];
  };
  Shared& sh;
  int lane, g, w, C, phase = 0;
  float inw = 0.f;
  bool tail;  // some lane's last vector is not full
  __device__ RowSums(Shared& s, int c) : sh(s), C(c) {
    lane = threadIdx.x % LPR;
    g = threadIdx.x / LPR;
    w = lane >> 6;
    tail = c != LPR * NV * V;
    if constexpr (NW > 1) {
      int n = 0;
#pragma unroll
      for (int j = 0; j < NV; ++j) n += min(max(c - (LPR * j + w * 64) * V, 0), 64 * V);
      inw = n > 0 ? 1.f / (float)n : 0.f;
      if ((lane & 63) == 0) sh.num[w] = make_float2((float)n, inw);
    }
  }
  __device__ void sum2(float& a, float& b) {
    constexpr int G = LPR < 64 ? LPR : 64;
    a = group_sum<G>(a);
    b = group_sum<G>(b);
    if constexpr (NW > 1) {
      phase ^= 1;
      if ((lane & 63) == 0) {
        sh.join[phase][g][w][0] = a;
        sh.join[phase][g][w][1] = b;
      }
      lds_barrier();
      a = b = 0.f;
#pragma unroll
      for (int x = 0; x < NW; ++x) {
        a += sh.join[phase][g][x][0];
        b += sh.join[phase][g][x][1];
      }
    }
  }
  // v is 0 past the last channel
  __device__ void moments(const float (&v)[NV][V], int kind, float eps, bool live, float& m,
                          float& r) {
    constexpr int G = LPR < 64 ? LPR : 64;
    const float ic = 1.f / (float)C;
    float s = 0.f, q = 0.f, mu = 0.f;
    if (kind == DCN_NORM_LAYER) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) s += v[j][e];
      s = group_sum<G>(s);
      mu = s * (NW > 1 ? inw : ic);
    }
    if (tail && kind == DCN_NORM_LAYER) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = (lane + LPR * j) * V + e < C ? v[j][e] - mu : 0.f;
          q = fmaf(d, d, q);
        }
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = v[j][e] - mu;
          q = fmaf(d, d, q);
        }
    }
    q = group_sum<G>(q);
    m = mu;
    if constexpr (NW > 1) {
      phase ^= 1;
      if ((lane & 63) == 0) {
        sh.join[phase][g][w][0] = s;
        sh.join[phase][g][w][1] = q;
      }
      lds_barrier();
      s = q = 0.f;
#pragma unroll
      for (int x = 0; x < NW; ++x) {
        s += sh.join[phase][g][x][0];
        q += sh.join[phase][g][x][1];
      }
      m = s * ic;
      if (kind == DCN_NORM_LAYER) {
#pragma unroll
        for (int x = 0; x < NW; ++x) {
          const float2 n = sh.num[x];
          const float d = fmaf(sh.join[phase][g][x][0], n.y, -m);
          q = fmaf(n.x * d, d, q);
        }
      }
    }
    r = live ? rsqrtf(fmaf(q, ic, eps)) : 0.f;
  }
};

// PAR: the backward adds up the parameters' gradients here; without, it leaves each row's six
// numbers (below) for block_row_params.
template <typename T, int NT, int LPR, int NV, int WPE, bool AHEAD, bool BWD, bool FULL, bool DROP,
          bool PAR>
__global__ __launch_bounds__(NT, WPE) void block_row(BlockArgs a, Plan q) {
  constexpr int V = ElemVec<T>::N, GR = NT / LPR;
  using Sums = RowSums<NT, LPR, V, NV>;
  __shared__ __attribute__((aligned(16))) typename Sums::Shared shared;
  constexpr bool SUMS = BWD && PAR;
  __shared__ float fold[SUMS ? GR : 1][SUMS ? LPR * NV * V : 1];
  const PhiloxKey key = philox_key(a.drop);
  Sums sums(shared, a.C);
  const int lane = sums.lane, g = threadIdx.x / LPR;
  const int wg = xcd_wg(q.wgs);
  auto ptr = [](const void* p) { return static_cast<const T*>(p); };

  int cv[NV];  // valid elements of a vector
  // The parameters of this lane's channels: kept beside a prefetched row, read again (from the
  // caches) for every row where the registers are needed for the sums. Past the last channel they
  // are 0, given or not: x is 0 there, but its normalised value -m r is not, and the factors' zeros
  // keep it out of out, of N_pre's moments and of the backward's sums.
  const void* const pars[5] = {a.scale, a.w1, a.b1, a.w2, a.b2};
  u32x4 kept[AHEAD ? (BWD ? 4 : 5) : 1][NV];
  auto fetch = [&](int k, int j) {
    const u32x4 zero = {0u, 0u, 0u, 0u};
    if (cv[j] <= 0) return zero;
    if (pars[k]) return ldv_raw(ptr(pars[k]) + (lane + LPR * j) * V, cv[j]);
    float t[V];
#pragma unroll
    for (int e = 0; e < V; ++e) t[e] = k == 2 || k == 4 || e >= cv[j] ? 0.f : 1.f;
    return pack<T>(t);
  };
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    cv[j] = a.C - (lane + LPR * j) * V;
    if constexpr (AHEAD) {
#pragma unroll
      for (int k = 0; k < (BWD ? 4 : 5); ++k) kept[k][j] = fetch(k, j);
    }
  }
  enum { SC, W1, B1, W2, B2 };
  auto param = [&](int k, int j, float (&v)[V]) {
    if constexpr (AHEAD)
      unpack<T>(kept[k][j], v);
    else
      unpack<T>(fetch(k, j), v);
  };
  const u32x4 zero = {0u, 0u, 0u, 0u};
  float acc[SUMS ? 5 : 1][NV][V], accg[SUMS && !FULL ? NV : 1][V];
  if constexpr (SUMS) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e) {
#pragma unroll
        for (int k = 0; k < 5; ++k) acc[k][j][e] = 0.f;
        if constexpr (!FULL) accg[j][e] = 0.f;
      }
  }
  // Σ of v over the row groups of the workgroup, to dst[C]
  auto fold_groups = [&](const float (&v)[NV][V], float* dst) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e) fold[g][(lane + LPR * j) * V + e] = v[j][e];
    __syncthreads();
    for (int c = threadIdx.x; c < a.C; c += NT) {
      float s = fold[0][c];
#pragma unroll
      for (int x = 1; x < GR; ++x) s += fold[x][c];
      dst[c] = s;
    }
  };

  const long t0 = first_tile(q, wg), t1 = first_tile(q, wg + 1);  // (group 1)
  struct Raw {
    u32x4 x[NV], r[NV], g[NV], y[NV], o[NV];
    float st[4];
    bool gone;  // the row's image is dropped
  } nx;
  const size_t rows = (size_t)q.images * q.P;
  auto load = [&](long t, Raw& w) {
    const int b = (int)(t / q.tpi), p = (int)(t % q.tpi) * GR + g;
    const size_t base = ((size_t)b * q.P + p) * a.C;
    if (BWD && a.stats) {
#pragma unroll
      for (int k = 0; k < 4; ++k)  // 0 past the last row: nothing there may reach the sums
        w.st[k] = p < q.P ? a.stats[k * rows + (size_t)b * q.P + p] : 0.f;
    }
    w.gone = false;
    if constexpr (DROP) {
      if (a.drop_image) {
        const int image = q.images == a.B ? b : (int)(((size_t)b * q.P + p) / a.P);
        w.gone = !keep1(image, key, a.drop.thr);
      }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const bool ok = p < q.P && cv[j] > 0;
      const size_t at = base + (lane + LPR * j) * V;
      w.x[j] = ok && a.x && !w.gone ? ldv_raw(ptr(a.x) + at, cv[j]) : zero;
      w.r[j] = ok && a.res ? ldv_raw(ptr(a.res) + at, cv[j]) : zero;
      if constexpr (FULL) w.g[j] = ok && !w.gone ? ldv_raw(ptr(a.gate) + at, cv[j]) : zero;
      if constexpr (BWD) {
        w.y[j] = ok && a.gy ? ldv_raw(ptr(a.gy) + at, cv[j]) : zero;
        w.o[j] = ok && a.go ? ldv_raw(ptr(a.go) + at, cv[j]) : zero;
      }
    }
  };
  // an image gate's act and act', kept while the rows stay in one image (with the registers for a
  // prefetched row there are some for these); read for every row otherwise
  constexpr bool KEEP = !FULL && AHEAD;
  float gv[KEEP ? NV : 1][V], gd[KEEP && BWD ? NV : 1][V];
  int gb = -1;
  if constexpr (KEEP) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        gv[j][e] = 1.f;
        gd[BWD ? j : 0][e] = 0.f;
      }
  }
  if (AHEAD && t0 < t1) load(t0, nx);
  for (long t = t0; t < t1; ++t) {
    const int b = (int)(t / q.tpi), p = (int)(t % q.tpi) * GR + g;
    const bool live = p < q.P;
    const size_t base = ((size_t)b * q.P + p) * a.C;
    if (!AHEAD) load(t, nx);
    const Raw in = nx;
    if (AHEAD && t + 1 < t1) load(t + 1, nx);

    unsigned keep[NV];
    if constexpr (DROP) {
      // nothing of a row behind the last is kept, as past a map's end
      const unsigned img = in.gone ? 0u : 0xffu, in_rows = live ? ~0u : 0u;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        keep[j] = (a.drop_image ? img : keepv<V>(base + (lane + LPR * j) * V, key, a.drop.thr)) &
                  in_rows;
    }
    auto kept_or_0 = [&](int j, int e, float v) {
      if constexpr (DROP) return (keep[j] >> e) & 1u ? v : 0.f;
      return v;
    };
    auto drop = [&](int j, int e, float v) {
      if constexpr (DROP) return kept_or_0(j, e, v * a.drop.scale);
      return v;
    };
    if constexpr (KEEP) {
      if (a.gate_kind == DCN_GATE_IMAGE && b != gb) {
        gb = b;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const bool read = cv[j] > 0 && !in.gone;
          float f[V];
          if (read) ldv(ptr(a.gate) + (size_t)b * a.C + (lane + LPR * j) * V, cv[j], f);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            gv[j][e] = 1.f;  // (a dropped image's gate: nothing of another image's may stay)
            gd[BWD ? j : 0][e] = 0.f;
            if (read) gate_act_grad<T>(f[e], a.act, gv[j][e], gd[BWD ? j : 0][e]);
          }
        }
      }
    }
    // the gate's value and slope
    auto gate = [&](int j, float (&av)[V], float (&ad)[V]) {
      if constexpr (KEEP) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          av[e] = gv[j][e];
          ad[e] = gd[BWD ? j : 0][e];
        }
        return;
      }
      float f[V];
      if constexpr (FULL) {
        unpack<T>(in.g[j], f);
        if constexpr (BWD) {
#pragma unroll
          for (int e = 0; e < V; ++e) f[e] = kept_or_0(j, e, f[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          av[e] = 1.f;
          ad[e] = 0.f;
        }
        if (a.gate_kind == DCN_GATE_NONE || cv[j] <= 0 || in.gone) return;
        ldv(ptr(a.gate) + (size_t)b * a.C + (lane + LPR * j) * V, cv[j], f);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) gate_act_grad<T>(f[e], a.act, av[e], ad[e]);
    };

    float m1 = 0.f, r1 = 1.f, m2 = 0.f, r2 = 1.f;
    const bool known = BWD && a.stats;
    if (known) {
      if (a.post) {
        m1 = in.st[0];
        r1 = in.st[1];
      }
      m2 = in.st[2];
      r2 = in.st[3];
    }
    float o[NV][V];
    if (a.x) {
      if (a.post && !known) {
        float xv[NV][V];
#pragma unroll
        for (int j = 0; j < NV; ++j) unpack<T>(in.x[j], xv[j]);
        sums.moments(xv, a.post, a.eps1, live, m1, r1);
      }
      if (in.gone) {
        m1 = 0.f;
        r1 = 1.f;
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float xv[V], rv[V], sc[V], w1[V], b1[V], av[V], ad[V];
        unpack<T>(in.x[j], xv);
        unpack<T>(in.r[j], rv);
        param(SC, j, sc);
        param(W1, j, w1);
        param(B1, j, b1);
        gate(j, av, ad);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float v = fmaf((xv[e] - m1) * r1, w1[e], b1[e]);
          o[j][e] = rv[e] + drop(j, e, v * (a.alpha * sc[e] * av[e]));
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j) unpack<T>(in.r[j], o[j]);
    }
    if (a.pre && !known) sums.moments(o, a.pre, a.eps2, live, m2, r2);

    if constexpr (!BWD) {
      if (a.stats && live && lane == 0) {
        float* st = a.stats + (size_t)b * q.P + p;
        st[0] = m1;
        st[rows] = r1;
        st[2 * rows] = m2;
        st[3 * rows] = r2;
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (!live || cv[j] <= 0) continue;
        const size_t at = base + (lane + LPR * j) * V;
        if (a.pre) {
          float w2[V], b2[V], y[V];
          param(W2, j, w2);
          param(B2, j, b2);
#pragma unroll
          for (int e = 0; e < V; ++e) y[e] = fmaf((o[j][e] - m2) * r2, w2[e], b2[e]);
          stv(static_cast<T*>(a.y) + at, cv[j], y);
        }
        if (a.out) stv(static_cast<T*>(a.out) + at, cv[j], o[j]);
      }
    } else {
      const float ic = 1.f / (float)a.C;
      float s1 = 0.f, s2 = 0.f;
      // G into o
      if (a.pre) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          float gy[V], w2[V];
          unpack<T>(in.y[j], gy);
          param(W2, j, w2);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float h = (o[j][e] - m2) * r2, w = gy[e] * w2[e];
            o[j][e] = h;
            s1 += w;
            s2 = fmaf(w, h, s2);
            if constexpr (SUMS) {
              acc[3][j][e] = fmaf(gy[e], h, acc[3][j][e]);
              acc[4][j][e] += gy[e];
            }
          }
        }
        sums.sum2(s1, s2);
        s1 = a.pre == DCN_NORM_LAYER ? s1 * ic : 0.f;
        s2 *= ic;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          float gy[V], go[V], w2[V];
          unpack<T>(in.y[j], gy);
          unpack<T>(in.o[j], go);
          param(W2, j, w2);
#pragma unroll
          for (int e = 0; e < V; ++e)
            o[j][e] = fmaf(r2, gy[e] * w2[e] - s1 - o[j][e] * s2, go[e]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < NV; ++j) unpack<T>(in.o[j], o[j]);
      }
      if constexpr (!PAR) {
        if (q.rowst && live && lane == 0) {
          const float st[6] = {m1, r1, m2, r2, s1, s2};
#pragma unroll
          for (int k = 0; k < 6; ++k) q.rowst[k * rows + (size_t)b * q.P + p] = st[k];
        }
      }
      if (a.gr) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if (live && cv[j] > 0)
            stv(static_cast<T*>(a.gr) + base + (lane + LPR * j) * V, cv[j], o[j]);
      }
      if (a.x) {
        float s3 = 0.f, s4 = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          float xv[V], sc[V], w1[V], b1[V], av[V], ad[V], gg[V];
          unpack<T>(in.x[j], xv);
          param(SC, j, sc);
          param(W1, j, w1);
          param(B1, j, b1);
          gate(j, av, ad);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float h = kept_or_0(j, e, (xv[e] - m1) * r1), v = fmaf(h, w1[e], b1[e]);
            const float dt = drop(j, e, o[j][e]), dtv = dt * v, k = a.alpha * sc[e];
            // (selected: 0 times an image gate that is not finite is not 0; a full one counts as 0)
            float dv = dt * (k * av[e]);
            gg[e] = dtv * (k * ad[e]);
            if constexpr (!FULL) {
              dv = kept_or_0(j, e, dv);
              gg[e] = kept_or_0(j, e, gg[e]);
            }
            if constexpr (SUMS) {
              const float sum = fmaf(dtv, a.alpha * av[e], acc[0][j][e]);
              if constexpr (DROP && !FULL)
                acc[0][j][e] = (keep[j] >> e) & 1u ? sum : acc[0][j][e];
              else
                acc[0][j][e] = sum;
              acc[1][j][e] = fmaf(dv, h, acc[1][j][e]);
              acc[2][j][e] += dv;
              if constexpr (!FULL) accg[j][e] += gg[e];
            }
            o[j][e] = dv;
            const float w = dv * w1[e];
            s3 += w;
            s4 = fmaf(w, h, s4);
          }
          if (FULL && a.gg && live && cv[j] > 0)
            stv(static_cast<T*>(a.gg) + base + (lane + LPR * j) * V, cv[j], gg);
        }
        if (a.gx) {
          if (a.post) {
            sums.sum2(s3, s4);
            s3 = a.post == DCN_NORM_LAYER ? s3 * ic : 0.f;
            s4 *= ic;
          }
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            if (!live || cv[j] <= 0) continue;
            if (a.post) {
              float xv[V], w1[V];
              unpack<T>(in.x[j], xv);
              param(W1, j, w1);
#pragma unroll
              for (int e = 0; e < V; ++e) {
                const float h = (xv[e] - m1) * r1;
                o[j][e] = r1 * (o[j][e] * w1[e] - s3 - h * s4);
              }
            }
            stv(static_cast<T*>(a.gx) + base + (lane + LPR * j) * V, cv[j], o[j]);
          }
        }
        if constexpr (SUMS && !FULL) {
          if (q.image_gate && (t + 1 == t1 || (t + 1) % q.tpi == 0)) {
            fold_groups(accg, q.gpart + (size_t)(wg + b) * a.C);
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
              for (int e = 0; e < V; ++e) accg[j][e] = 0.f;
          }
        }
      }
    }
  }
  if constexpr (SUMS) {
    if (!q.part) return;
#pragma unroll
    for (int k = 0; k < 5; ++k) fold_groups(acc[k], q.part + ((size_t)wg * 5 + k) * a.C);
  }
}

// The parameters' gradients of long rows, in a second pass: with 16 channels a lane their five sums
// do not fit beside the row (1024 x 8192 bf16, spilling, in one pass 65 us; in two 30 and 23, and 5
// for the fold). A workgroup takes 64 vectors of channels and a run of rows, kParamRows / V of them
// to a wave at a time; what a row needs besides its values are the six numbers that block_row left.
constexpr int kParamRows = 16;  // channels times rows of a lane at a time
template <typename T, bool FULL, bool DROP>
__global__ __launch_bounds__(256) void block_row_params(BlockArgs a, Plan q) {
  constexpr int V = ElemVec<T>::N, GR = 4, U = kParamRows / V;
  __shared__ float fold[GR][64 * V];
  const PhiloxKey key = philox_key(a.drop);
  const int lane = threadIdx.x & 63, g = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = ((int)blockIdx.y * 64 + lane) * V, cv = a.C - c, wg = blockIdx.x;
  auto ptr = [](const void* p) { return static_cast<const T*>(p); };
  auto param = [&](const void* p, float none, float (&v)[V]) {
    if (p && cv > 0) return ldv(ptr(p) + c, cv, v);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = none;
  };
  float sc[V], w1[V], b1[V], w2[V], gv[V], gd[V], acc[5][V], accg[V];
  param(a.scale, 1.f, sc);
  param(a.w1, 1.f, w1);
  param(a.b1, 0.f, b1);
  param(a.w2, 1.f, w2);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    gv[e] = 1.f;
    gd[e] = accg[e] = 0.f;
#pragma unroll
    for (int k = 0; k < 5; ++k) acc[k][e] = 0.f;
  }
  auto fold_waves = [&](const float (&v)[V], float* dst) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < V; ++e) fold[g][lane * V + e] = v[e];
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * V; i += 256) {
      const int at = (int)blockIdx.y * 64 * V + i;
      if (at < a.C) dst[at] = (fold[0][i] + fold[1][i]) + (fold[2][i] + fold[3][i]);
    }
  };
  int gb = -1;
  const size_t rows = (size_t)q.images * q.P;
  const long t1 = first_tile(q, wg + 1);
  for (long t = first_tile(q, wg); t < t1; ++t) {
    const int b = (int)(t / q.tpi), p0 = (int)(t % q.tpi) * GR * U + g * U;
    // U rows' loads in flight at a time; a row behind the last is zeros and adds nothing
    u32x4 x[U], o[U], f[U], gy[U], go[U];
    float st[U][6];
    unsigned keep[U];
    bool gone = false;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool live = p0 + u < q.P && cv > 0;
      const size_t row = (size_t)b * q.P + p0 + u, at = row * a.C + c;
      keep[u] = 0xffu;
      if constexpr (DROP) {
        if (a.drop_image) {
          gone = !keep1(q.images == a.B ? b : (int)(row / a.P), key, a.drop.thr);
          keep[u] = gone ? 0u : 0xffu;
        } else {
          keep[u] = keepv<V>(at, key, a.drop.thr);
        }
        if (!live) keep[u] = 0u;
      }
      auto read = [&](const void* t) {
        return t && live ? ldv_raw(ptr(t) + at, cv) : u32x4{0u, 0u, 0u, 0u};
      };
      x[u] = read(gone ? nullptr : a.x);
      o[u] = read(a.res);
      gy[u] = read(a.gy);
      go[u] = read(a.go);
      if constexpr (FULL) f[u] = read(gone ? nullptr : a.gate);
#pragma unroll
      for (int k = 0; k < 6; ++k) st[u][k] = live ? q.rowst[k * rows + row] : 0.f;
    }
    if (a.gate_kind == DCN_GATE_IMAGE && b != gb) {
      gb = b;
      float w[V];
      if (!gone && cv > 0) ldv(ptr(a.gate) + (size_t)b * a.C + c, cv, w);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        gv[e] = 1.f;
        gd[e] = 0.f;
        if (!gone && cv > 0) gate_act_grad<T>(w[e], a.act, gv[e], gd[e]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float xv[V], ov[V], fv[V], gyv[V], gov[V];
      unpack<T>(x[u], xv);
      unpack<T>(o[u], ov);
      unpack<T>(gy[u], gyv);
      unpack<T>(go[u], gov);
      if constexpr (FULL) unpack<T>(f[u], fv);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const bool kept = !DROP || (keep[u] >> e & 1u);
        float av = gv[e], ad = gd[e];
        if constexpr (FULL) gate_act_grad<T>(kept ? fv[e] : 0.f, a.act, av, ad);
        const float h = kept ? (xv[e] - st[u][0]) * st[u][1] : 0.f, v = fmaf(h, w1[e], b1[e]);
        const float k = a.alpha * sc[e], ds = kept ? (DROP ? a.drop.scale : 1.f) : 0.f;
        float G = gov[e];
        if (a.pre) {
          const float h2 = (ov[e] + (a.x && kept ? v * (k * av) * ds : 0.f) - st[u][2]) * st[u][3];
          acc[3][e] = fmaf(gyv[e], h2, acc[3][e]);
          acc[4][e] += gyv[e];
          G = fmaf(st[u][3], gyv[e] * w2[e] - st[u][4] - h2 * st[u][5], G);
        }
        const float dt = kept ? G * ds : 0.f, dv = kept ? dt * (k * av) : 0.f;
        const float s0 = fmaf(dt * v, a.alpha * av, acc[0][e]);
        acc[0][e] = kept ? s0 : acc[0][e];
        acc[1][e] = fmaf(dv, h, acc[1][e]);
        acc[2][e] += dv;
        if constexpr (!FULL) {
          const float sg = fmaf(dt * v, k * ad, accg[e]);
          accg[e] = kept ? sg : accg[e];
        }
      }
    }
    if (q.image_gate && (t + 1 == t1 || (t + 1) % q.tpi == 0)) {  // uniform
      fold_waves(accg, q.gpart + (size_t)(wg + b) * a.C);
#pragma unroll
      for (int e = 0; e < V; ++e) accg[e] = 0.f;
    }
  }
  if (!q.part) return;
#pragma unroll
  for (int k = 0; k < 5; ++k) fold_waves(acc[k], q.part + ((size_t)wg * 5 + k) * a.C);
}

// The partials of one parameter (k < 5) or of one image's gate (k = 5 + image), 64 channels
// per workgroup, added in workgroup order: 16 threads a channel, then a tree over them.
template <typename T>
__global__ __launch_bounds__(1024) void block_fold(BlockArgs a, Plan q, int k0) {
  __shared__ float red[16][64];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), g = threadIdx.x >> 6, k = k0 + blockIdx.y;
  void* dst[5] = {a.gs, a.gw1, a.gb1, a.gw2, a.gb2};
  T* out = k < 5 ? static_cast<T*>(dst[k]) : static_cast<T*>(a.gg) + (size_t)(k - 5) * a.C;
  if (k < 5 && !dst[k]) return;
  float s = 0.f;
  if (c < a.C) {
    if (k < 5) {
#pragma unroll 4
      for (int w = g; w < q.wgs; w += 16) s += q.part[((size_t)w * 5 + k) * a.C + c];
    } else {
      // the runs that meet this image's tiles [lo, hi), and in them the turns that took one
      const long lo = (long)(k - 5) * q.tpi, hi = lo + q.tpi;
      const int runs = q.wgs / q.group;
      int r0 = (int)(lo * runs / q.tiles);
      while (r0 > 0 && first_tile(q, r0) > lo) --r0;
      while (first_tile(q, r0 + 1) <= lo) ++r0;
      for (int i = g;; i += 16) {
        const int r = r0 + i / q.group, j = i % q.group;
        if (r >= runs || first_tile(q, r) >= hi) break;
        const long c0 = first_tile(q, r), from = max(lo, c0), to = min(hi, first_tile(q, r + 1));
        const long t = c0 + j >= from ? c0 + j : from + (q.group - (from - c0 - j) % q.group) % q.group;
        if (t < to) s += q.gpart[((size_t)(r + k - 5) * q.group + j) * a.C + c];
      }
    }
  }
  red[g][threadIdx.x & 63] = s;
  __syncthreads();
  for (int o = 8; o > 0; o >>= 1) {
    if (g < o) red[g][threadIdx.x & 63] += red[g + o][threadIdx.x & 63];
    __syncthreads();
  }
  if (g == 0 && c < a.C) out[c] = from_f32(red[0][threadIdx.x], T());
}

constexpr int kMaxWgs = 1024;   // workgroups with partials, maps
constexpr int kRowWgs = 512;    // and rows
constexpr int kLongWgs = 256;   // and rows of more than
constexpr int kRowSums = 4096;  // channels: beside those the parameters' sums fit
constexpr int kInterleave = 8;  // workgroups that share a run of map tiles

// Workgroups that leave partials, at most: those of the variant, and no more than a call has tiles
// (of a row, or of 16 positions of a map, at least). The workspace's size and layout go by it.
inline int long_columns(const BlockArgs& a) {  // workgroups across the channels in block_row_params
  const int per = 64 * (a.dtype == DCN_BF16 ? ElemVec<bf16_t>::N : ElemVec<float>::N);
  return (a.C + per - 1) / per;
}
inline int partial_wgs(const BlockArgs& a) {
  const bool rows = a.layout == DCN_NHWC || a.P == 1;
  const long tiles = (long)a.B * (rows ? a.P : (a.P + 15) / 16);
  long wgs = kMaxWgs;
  if (rows && a.C <= kRowSums) wgs = kRowWgs;
  if (rows && a.C > kRowSums) {
    const bool gated = a.dtype == DCN_BF16 && a.C <= 8192 && a.gate_kind == DCN_GATE_FULL;
    wgs = gated ? kLongWgs : std::min(kLongWgs, std::max(1, 1024 / long_columns(a)));
  }
  return (int)std::min(wgs, tiles);
}

// adds up the partials; a parameter without a destination ends at once
template <typename T>
hipError_t fold_partials(const BlockArgs& a, const Plan& q, hipStream_t s) {
  const int rows = 5 + (q.image_gate ? a.B : 0);  // an image gate's start at 5
  for (int k = q.part ? 0 : 5, n; k < rows; k += n) {
    n = std::min(rows - k, 32768);
    hipLaunchKernelGGL((block_fold<T>), dim3((a.C + 63) / 64, n), dim3(1024), 0, s, a, q, k);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// Fills the plan for tiles of `per` positions, launches `kernel(full gate, dropout)` and the fold.
template <typename T, bool BWD, typename K>
hipError_t run_tiles(const BlockArgs& a, int images, int P, int per, int wgs, int threads, bool maps,
                     K kernel, hipStream_t s) {
  Plan q{};
  q.images = images;
  q.P = P;
  q.tpi = (P + per - 1) / per;
  q.tiles = (long)q.tpi * images;
  const bool params = BWD && (a.gs || a.gw1 || a.gb1 || a.gw2 || a.gb2);
  q.image_gate = BWD && a.gg && a.gate_kind == DCN_GATE_IMAGE;
  // wgs: > 0 with a prefetch, < 0 without, 0 without and one a tile as far as partials allow
  q.wgs = (int)std::min<long>(
      q.tiles, wgs ? std::abs(wgs) : params || q.image_gate ? kMaxWgs : 1 << 20);
  q.group = maps && q.tpi >= kInterleave && q.wgs % kInterleave == 0 ? kInterleave : 1;
  if (params) q.part = a.ws;
  if (q.image_gate) q.gpart = a.ws + (size_t)partial_wgs(a) * 5 * a.C;
  auto* fn = kernel(a.gate_kind == DCN_GATE_FULL, a.drop.thr != 0);
  hipLaunchKernelGGL(fn, dim3(q.wgs), dim3(threads), 0, s, a, q);
  const hipError_t e = hipGetLastError();
  return e != hipSuccess || !(params || q.image_gate) ? e : fold_partials<T>(a, q, s);
}

template <typename T, int NT, int PL, int CPT, int WPE, int WGS, bool BWD>
hipError_t run_map(const BlockArgs& a, hipStream_t s) {
  auto pick = [](bool full, bool drop) {
    return full ? (drop ? block_map<T, NT, PL, CPT, WPE, (WGS > 0), BWD, true, true>
                        : block_map<T, NT, PL, CPT, WPE, (WGS > 0), BWD, true, false>)
                : (drop ? block_map<T, NT, PL, CPT, WPE, (WGS > 0), BWD, false, true>
                        : block_map<T, NT, PL, CPT, WPE, (WGS > 0), BWD, false, false>);
  };
  return run_tiles<T, BWD>(a, a.B, a.P, PL * ElemVec<T>::N, WGS, NT, true, pick, s);
}

// images matter to an image gate only; else all rows are one run (up to int)
inline bool one_run(const BlockArgs& a) {
  return a.gate_kind != DCN_GATE_IMAGE && (size_t)a.B * a.P < (1u << 30);
}

template <typename T, int NT, int LPR, int NV, int WPE, int WGS, bool BWD>
hipError_t run_row(const BlockArgs& a, hipStream_t s) {
  auto pick = [](bool full, bool drop) {
    return full ? (drop ? block_row<T, NT, LPR, NV, WPE, (WGS > 0), BWD, true, true, true>
                        : block_row<T, NT, LPR, NV, WPE, (WGS > 0), BWD, true, false, true>)
                : (drop ? block_row<T, NT, LPR, NV, WPE, (WGS > 0), BWD, false, true, true>
                        : block_row<T, NT, LPR, NV, WPE, (WGS > 0), BWD, false, false, true>);
  };
  const bool one = one_run(a);
  return run_tiles<T, BWD>(a, one ? 1 : a.B, one ? a.B * a.P : a.P, NT / LPR, WGS, NT, false, pick,
                           s);
}

// A full gate's backward of rows of 16 channels a lane in one pass after all: with nothing fetched
// ahead and the parameters read again for every row the sums fit (run_long_row).
template <typename T, int NT, int NV, int WPE, int WGS>
hipError_t run_gated_row(const BlockArgs& a, hipStream_t s) {
  static_assert(WGS <= kLongWgs, "partials");
  auto pick = [](bool, bool drop) {
    return drop ? block_row<T, NT, NT, NV, WPE, false, true, true, true, true>
                : block_row<T, NT, NT, NV, WPE, false, true, true, false, true>;
  };
  return run_tiles<T, true>(a, 1, a.B * a.P, 1, WGS, NT, false, pick, s);
}

// A backward in two passes: every row's gradients, then the parameters'.
template <typename T, int NT, int NV, int WPE, bool AHEAD, int WGS>
hipError_t run_long_row(const BlockArgs& a, hipStream_t s) {
  Plan q{};
  const bool one = one_run(a), image_gate = a.gg && a.gate_kind == DCN_GATE_IMAGE;
  const bool params = a.gs || a.gw1 || a.gb1 || a.gw2 || a.gb2, full = a.gate_kind == DCN_GATE_FULL;
  q.images = one ? 1 : a.B;
  q.P = one ? a.B * a.P : a.P;
  q.tpi = q.P;  // one row a tile
  q.tiles = (long)q.tpi * q.images;
  q.wgs = (int)std::min<long>(q.tiles, WGS);
  q.group = 1;
  if (params || image_gate) q.rowst = a.ws;
  const bool drop = a.drop.thr != 0;
  auto* fn = full ? (drop ? block_row<T, NT, NT, NV, WPE, AHEAD, true, true, true, false>
                          : block_row<T, NT, NT, NV, WPE, AHEAD, true, true, false, false>)
                  : (drop ? block_row<T, NT, NT, NV, WPE, AHEAD, true, false, true, false>
                          : block_row<T, NT, NT, NV, WPE, AHEAD, true, false, false, false>);
  if (a.gx || a.gr || (a.gg && full) || q.rowst) {
    hipLaunchKernelGGL(fn, dim3(q.wgs), dim3(NT), 0, s, a, q);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !q.rowst) return e;
  }
  float* rest = a.ws + ((size_t)a.B * a.P * 6 + 63) / 64 * 64;
  const int columns = long_columns(a);
  const int per = 4 * kParamRows / ElemVec<T>::N;
  q.tpi = (q.P + per - 1) / per;
  q.tiles = (long)q.tpi * q.images;
  q.wgs = (int)std::min<long>(q.tiles, partial_wgs(a));
  q.image_gate = image_gate;
  if (params) q.part = rest;
  if (image_gate) q.gpart = rest + (size_t)partial_wgs(a) * 5 * a.C;
  auto* pn = full ? (drop ? block_row_params<T, true, true> : block_row_params<T, true, false>)
                  : (drop ? block_row_params<T, false, true> : block_row_params<T, false, false>);
  hipLaunchKernelGGL(pn, dim3(q.wgs, columns), dim3(256), 0, s, a, q);
  const hipError_t e = hipGetLastError();
  return e != hipSuccess ? e : fold_partials<T>(a, q, s);
}

}  // namespace

}  // namespace dcn
