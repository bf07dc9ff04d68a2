// dcn_block_norm.hip — the operator between two residual blocks (include/dcn.h, block norms):
//   t = drop(alpha · scale[c] · act(gate) · N_post(x)), out = residual + t, y = N_pre(out)
// over the C channels of every position, and its backward.
//
// Backward, with h = (v - m) · r the normalised values of a norm and a = g · w:
//   N'(g) = r · (a - [layer] mean(a) - h · mean(a h)),  ∂w = Σ g h,  ∂b = Σ g
//   G  = ∂out + N_pre'(∂y)                 (= ∂residual)
//   dt = keep ? G · drop scale : 0
//   ∂gate = dt · N_post(x) · alpha · scale · act'(gate),  ∂scale = Σ dt · N_post(x) · alpha · act
//   ∂x = N_post'(dt · alpha · scale · act)
// out and the statistics are computed again from x and the residual (the residual is read
// instead of out, so that costs no bytes), which keeps the backward free of out's rounding.
#include "dcn_block.h"
#include "dcn_philox.h"

namespace dcn {

namespace {

constexpr int kThreads = 256;

// act(g) and act'(g)
__device__ __forceinline__ float gate_act(float g, int act) {
  if (act == DCN_ACT_LINEAR) return g;
  const float s = 1.f / (1.f + expf(-g));
  return act == DCN_ACT_SIGMOID ? s : g * s;
}
__device__ __forceinline__ void gate_act_grad(float g, int act, float& a, float& d) {
  a = g;
  d = 1.f;
  if (act == DCN_ACT_LINEAR) return;
  const float s = 1.f / (1.f + expf(-g));
  a = act == DCN_ACT_SIGMOID ? s : g * s;
  d = act == DCN_ACT_SIGMOID ? s * (1.f - s) : s * (1.f + g * (1.f - s));
}

// ---- any size: one position per LP lanes, several passes over its channels ----------------
// Addresses of one position's channels and the values of one element.
template <typename T>
struct Pos {
  const BlockArgs& a;
  const PhiloxKey& key;
  size_t base, cs;  // element (b, c, p) at base + c · cs
  int b;
  bool drop_all;  // this image's draw (drop_image)
  float m1 = 0.f, r1 = 1.f, m2 = 0.f, r2 = 1.f;

  __device__ Pos(const BlockArgs& a_, const PhiloxKey& k_, int b_, int p) : a(a_), key(k_), b(b_) {
    const bool maps = a.layout == DCN_NCHW;
    cs = maps ? a.P : 1;
    base = maps ? (size_t)b * a.C * a.P + p : ((size_t)b * a.P + p) * a.C;
    drop_all = a.drop.thr && a.drop_image && !keep1(b, key, a.drop.thr);
  }
  __device__ float ld(const void* t, size_t i) const { return to_f32(static_cast<const T*>(t)[i]); }
  __device__ float par(const void* t, int c, float none) const { return t ? ld(t, c) : none; }
  __device__ float x(int c) const { return ld(a.x, base + c * cs); }
  __device__ float h1(int c) const { return (x(c) - m1) * r1; }
  __device__ float v(int c) const {
    return a.post ? h1(c) * par(a.w1, c, 1.f) + par(a.b1, c, 0.f) : x(c);
  }
  __device__ float gate(int c) const {
    return ld(a.gate, a.gate_kind == DCN_GATE_FULL ? base + c * cs : (size_t)b * a.C + c);
  }
  __device__ float act(int c) const { return a.gate_kind ? gate_act(gate(c), a.act) : 1.f; }
  __device__ float k(int c) const { return a.alpha * par(a.scale, c, 1.f) * act(c); }
  __device__ float drop(float t, int c) const {
    if (!a.drop.thr) return t;
    const bool keep = a.drop_image ? !drop_all : keep1(base + c * cs, key, a.drop.thr);
    return keep ? t * a.drop.scale : 0.f;
  }
  __device__ float out(int c) const {
    const float r = a.res ? ld(a.res, base + c * cs) : 0.f;
    return a.x ? r + drop(v(c) * k(c), c) : r;
  }
  __device__ float h2(int c) const { return (out(c) - m2) * r2; }
  __device__ float gy(int c) const { return a.gy ? ld(a.gy, base + c * cs) : 0.f; }
};

// Σ over the LP lanes of a position
template <int LP>
__device__ __forceinline__ float lane_sum(float v) {
#pragma unroll
  for (int o = 1; o < LP; o <<= 1) v += __shfl_xor(v, o);
  return v;
}

// mean and 1/sqrt(var + eps) of f(c), in two passes: the second about the first's mean
template <int LP, typename F>
__device__ __forceinline__ void moments(F f, int lane, int C, int kind, float eps, float& m,
                                        float& r) {
  m = 0.f;
  if (kind == DCN_NORM_LAYER) {
    float s = 0.f;
    for (int c = lane; c < C; c += LP) s += f(c);
    m = lane_sum<LP>(s) / (float)C;
  }
  float s = 0.f;
  for (int c = lane; c < C; c += LP) {
    const float d = f(c) - m;
    s = fmaf(d, d, s);
  }
  r = 1.f / sqrtf(lane_sum<LP>(s) / (float)C + eps);
}

template <typename T, int LP>
__device__ __forceinline__ void pos_moments(Pos<T>& q, int lane) {
  const BlockArgs& a = q.a;
  if (a.x && a.post)
    moments<LP>([&](int c) { return q.x(c); }, lane, a.C, a.post, a.eps1, q.m1, q.r1);
  if (a.pre) moments<LP>([&](int c) { return q.out(c); }, lane, a.C, a.pre, a.eps2, q.m2, q.r2);
}

template <typename T, int LP>
__global__ __launch_bounds__(kThreads) void block_any_fwd(BlockArgs a) {
  const PhiloxKey key = philox_key(a.drop);
  const int lane = threadIdx.x % LP;
  const size_t rows = (size_t)a.B * a.P, step = (size_t)gridDim.x * (kThreads / LP);
  for (size_t row = (size_t)blockIdx.x * (kThreads / LP) + threadIdx.x / LP; row < rows;
       row += step) {
    Pos<T> q(a, key, (int)(row / a.P), (int)(row % a.P));
    pos_moments<T, LP>(q, lane);
    for (int c = lane; c < a.C; c += LP) {
      const float o = q.out(c);
      const size_t i = q.base + c * q.cs;
      if (a.pre)
        static_cast<T*>(a.y)[i] = from_f32(
            (o - q.m2) * q.r2 * q.par(a.w2, c, 1.f) + q.par(a.b2, c, 0.f), T());
      if (a.out) static_cast<T*>(a.out)[i] = from_f32(o, T());
    }
  }
}

// The elementwise gradients, and each position's statistics for block_any_params:
// ws[k][rows], k = m1, r1, m2, r2, mean(a2), mean(a2 h2).
template <typename T, int LP>
__global__ __launch_bounds__(kThreads) void block_any_bwd(BlockArgs a) {
  const PhiloxKey key = philox_key(a.drop);
  const int lane = threadIdx.x % LP;
  const size_t rows = (size_t)a.B * a.P, step = (size_t)gridDim.x * (kThreads / LP);
  for (size_t row = (size_t)blockIdx.x * (kThreads / LP) + threadIdx.x / LP; row < rows;
       row += step) {
    Pos<T> q(a, key, (int)(row / a.P), (int)(row % a.P));
    pos_moments<T, LP>(q, lane);
    float s1 = 0.f, s2 = 0.f;
    if (a.pre) {
      for (int c = lane; c < a.C; c += LP) {
        const float w = q.gy(c) * q.par(a.w2, c, 1.f);
        s1 += w;
        s2 = fmaf(w, q.h2(c), s2);
      }
      s1 = a.pre == DCN_NORM_LAYER ? lane_sum<LP>(s1) / (float)a.C : 0.f;
      s2 = lane_sum<LP>(s2) / (float)a.C;
    }
    auto total = [&](int c) {
      float g = a.go ? q.ld(a.go, q.base + c * q.cs) : 0.f;
      if (a.pre) g += q.r2 * (q.gy(c) * q.par(a.w2, c, 1.f) - s1 - q.h2(c) * s2);
      return g;
    };
    float s3 = 0.f, s4 = 0.f;
    if (a.x && a.post) {
      for (int c = lane; c < a.C; c += LP) {
        const float w = q.drop(total(c), c) * q.k(c) * q.par(a.w1, c, 1.f);
        s3 += w;
        s4 = fmaf(w, q.h1(c), s4);
      }
      s3 = a.post == DCN_NORM_LAYER ? lane_sum<LP>(s3) / (float)a.C : 0.f;
      s4 = lane_sum<LP>(s4) / (float)a.C;
    }
    for (int c = lane; c < a.C; c += LP) {
      const size_t i = q.base + c * q.cs;
      const float g = total(c);
      if (a.gr) static_cast<T*>(a.gr)[i] = from_f32(g, T());
      if (!a.x) continue;
      const float dt = q.drop(g, c);
      if (a.gg && a.gate_kind == DCN_GATE_FULL) {
        float av, ad;
        gate_act_grad(q.gate(c), a.act, av, ad);
        static_cast<T*>(a.gg)[i] =
            from_f32(dt * q.v(c) * (a.alpha * q.par(a.scale, c, 1.f)) * ad, T());
      }
      if (a.gx) {
        const float dv = dt * q.k(c);
        const float gx =
            a.post ? q.r1 * (dv * q.par(a.w1, c, 1.f) - s3 - q.h1(c) * s4) : dv;
        static_cast<T*>(a.gx)[i] = from_f32(gx, T());
      }
    }
    if (lane == 0) {
      const float st[6] = {q.m1, q.r1, q.m2, q.r2, s1, s2};
#pragma unroll
      for (int k = 0; k < 6; ++k) a.ws[k * rows + row] = st[k];
    }
  }
}

// One channel's parameter gradients (and its gates' over each image): sums over positions in a
// fixed order.
template <typename T>
__global__ __launch_bounds__(kThreads) void block_any_params(BlockArgs a) {
  __shared__ float red[6][kThreads / 64];
  const PhiloxKey key = philox_key(a.drop);
  const int c = blockIdx.x;
  const size_t rows = (size_t)a.B * a.P;
  float sum[5] = {0.f, 0.f, 0.f, 0.f, 0.f};  // scale, w1, b1, w2, b2
  for (int b = 0; b < a.B; ++b) {
    float sg = 0.f;
    for (int p = threadIdx.x; p < a.P; p += kThreads) {
      Pos<T> q(a, key, b, p);
      const size_t row = (size_t)b * a.P + p;
      q.m1 = a.ws[row];
      q.r1 = a.ws[rows + row];
      q.m2 = a.ws[2 * rows + row];
      q.r2 = a.ws[3 * rows + row];
      float g = a.go ? q.ld(a.go, q.base + c * q.cs) : 0.f;
      if (a.pre) {
        const float gy = q.gy(c), h2 = q.h2(c);
        g += q.r2 * (gy * q.par(a.w2, c, 1.f) - a.ws[4 * rows + row] - h2 * a.ws[5 * rows + row]);
        sum[3] = fmaf(gy, h2, sum[3]);
        sum[4] += gy;
      }
      if (!a.x) continue;
      const float dt = q.drop(g, c), v = q.v(c);
      float av = 1.f, ad = 0.f;
      if (a.gate_kind) gate_act_grad(q.gate(c), a.act, av, ad);
      sum[0] = fmaf(dt * v, a.alpha * av, sum[0]);
      sg = fmaf(dt * v * (a.alpha * q.par(a.scale, c, 1.f)), ad, sg);
      if (a.post) {
        const float dv = dt * q.k(c);
        sum[1] = fmaf(dv, q.h1(c), sum[1]);
        sum[2] += dv;
      }
    }
    if (a.gg && a.gate_kind == DCN_GATE_IMAGE) {  // uniform
      sg = wave_sum(sg);
      __syncthreads();
      if (threadIdx.x % 64 == 0) red[5][threadIdx.x / 64] = sg;
      __syncthreads();
      if (threadIdx.x == 0)
        static_cast<T*>(a.gg)[(size_t)b * a.C + c] =
            from_f32(red[5][0] + red[5][1] + red[5][2] + red[5][3], T());
    }
  }
#pragma unroll
  for (int k = 0; k < 5; ++k) {
    const float s = wave_sum(sum[k]);
    if (threadIdx.x % 64 == 0) red[k][threadIdx.x / 64] = s;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    void* dst[5] = {a.gs, a.gw1, a.gb1, a.gw2, a.gb2};
#pragma unroll
    for (int k = 0; k < 5; ++k)
      if (dst[k])
        static_cast<T*>(dst[k])[c] =
            from_f32(red[k][0] + red[k][1] + red[k][2] + red[k][3], T());
  }
}

// ---- one pass: the channels of a tile of positions stay in registers ----------------------
// Both layouts share the plan: work is cut into tiles (maps: TP neighbouring positions of an
// image, rows: one row per LPR lanes), the tiles of one workgroup are neighbours, and a thread
// keeps the same channels in every tile, so its parameter gradients add up in registers. They
// leave once per workgroup as partials [workgroup][5][C] (scale, w1, b1, w2, b2), an image
// gate's once per workgroup and image, and block_fold adds them in workgroup order.
struct Plan {
  int tpi;            // tiles of an image
  long tiles;         // of the call
  int wgs;            // workgroups; workgroup w takes tiles [w · tiles / wgs, (w + 1) · tiles / wgs)
  int images, P;      // rows without an image gate count as one image
  bool image_gate;    // ∂gate sums over positions
  float *part, *gpart;  // [wgs][5][C], [wgs + images][C]: slot wg + image is written once
};

__device__ __forceinline__ long first_tile(const Plan& q, int w) { return q.tiles * w / q.wgs; }

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
    float res[NW][2][TP];        // a wave's copy of the results
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
    give(0, ta * fa);
    give(1, tb * fb);
    wave_order();
    get(0, a);
    get(1, b);
    wave_order();
  }
  // Mean and 1/sqrt(var + eps) of each position (0 past the map's end, `left` = positions of
  // the tile, so that nothing from there reaches the parameter sums); mk: 1 for a channel, 0
  // past the last (its v is 0). Layer: every wave takes its own mean and the squares about it;
  // the waves' are joined about the whole mean, so large means cancel nowhere.
  __device__ void moments(const float (&v)[CPT][V], const float (&mk)[CPT], int kind, float eps,
                          int left, float (&m)[V], float (&r)[V]) {
    float t[V], s = 0.f, q;
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
      give(0, s * inw);
      wave_order();
      get(0, m);
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
    give(0, s * ic);
    give(1, lane % TP < left ? rsqrtf(fmaf(q, ic, eps)) : 0.f);
    wave_order();
    get(0, m);
    get(1, r);
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
  float acc[5][CPT], accg[CPT];
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
    accg[i] = 0.f;
  }
  const long t0 = first_tile(q, wg), t1 = first_tile(q, wg + 1);
  struct Raw {
    u32x4 x[CPT], r[CPT], g[CPT], y[CPT], o[CPT];
  } nx;
  auto load = [&](long t, Raw& w) {
    const int p = (int)(t % q.tpi) * TP + pl * V, valid = a.P - p;
    const size_t base = (size_t)(t / q.tpi) * a.C * a.P + p;
    const u32x4 zero = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      const bool ok = inc[i] && valid > 0;
      const size_t at = base + (size_t)(cg + CG * i) * a.P;
      w.x[i] = ok && xp ? ldv_raw(xp + at, valid) : zero;
      w.r[i] = ok && rp ? ldv_raw(rp + at, valid) : zero;
      if constexpr (FULL) w.g[i] = ok ? ldv_raw(gp + at, valid) : zero;
      if constexpr (BWD) {
        w.y[i] = ok && a.gy ? ldv_raw(static_cast<const T*>(a.gy) + at, valid) : zero;
        w.o[i] = ok && a.go ? ldv_raw(static_cast<const T*>(a.go) + at, valid) : zero;
      }
    }
  };
  if (AHEAD && t0 < t1) load(t0, nx);
  for (long t = t0; t < t1; ++t) {
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
    if (AHEAD && t + 1 < t1) load(t + 1, nx);
    float gv[CPT], gd[CPT];  // an image gate's act and act'
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      gv[i] = 1.f;
      gd[i] = 0.f;
      if (a.gate_kind == DCN_GATE_IMAGE && inc[i])
        gate_act_grad(to_f32(gp[(size_t)b * a.C + cg + CG * i]), a.act, gv[i], gd[i]);
    }
    unsigned keep[CPT];
    if constexpr (DROP) {
      const unsigned img = a.drop_image && keep1(b, key, a.drop.thr) ? 0xffu : 0u;
#pragma unroll
      for (int i = 0; i < CPT; ++i) keep[i] = a.drop_image ? img : keepv<V>(at[i], key, a.drop.thr);
    }
    auto drop = [&](int i, int e, float t) {
      if constexpr (DROP) return (keep[i] >> e) & 1u ? t * a.drop.scale : 0.f;
      return t;
    };

    float m1[V], r1[V], m2[V], r2[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {  // no post norm: N_post(x) = x
      m1[e] = 0.f;
      r1[e] = 1.f;
    }
    float o[CPT][V];
    if (xp) {
      if (a.post) {
        float xv[CPT][V];
#pragma unroll
        for (int i = 0; i < CPT; ++i) unpack<T>(in.x[i], xv[i]);
        sums.moments(xv, mk, a.post, a.eps1, left, m1, r1);
      }
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
          o[i][e] = rv[e] + drop(i, e, v * (FULL ? sc[i] * gate_act(fv[e], a.act) : k));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < CPT; ++i) unpack<T>(in.r[i], o[i]);
    }
    if (a.pre) sums.moments(o, mk, a.pre, a.eps2, left, m2, r2);

    if constexpr (!BWD) {
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
        float s1[V], s2[V];
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
        float s3[V], s4[V];
#pragma unroll
        for (int e = 0; e < V; ++e) s3[e] = s4[e] = 0.f;
#pragma unroll
        for (int i = 0; i < CPT; ++i) {
          float xv[V], fv[V], gg[V];
          const float ka = a.alpha * gv[i], kd = sc[i] * gd[i], k = sc[i] * gv[i];
          unpack<T>(in.x[i], xv);
          if constexpr (FULL) unpack<T>(in.g[i], fv);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float h = (xv[e] - m1[e]) * r1[e], v = fmaf(h, w1[i], b1[i]);
            const float dt = drop(i, e, o[i][e]), dtv = dt * v;
            float dv;
            if constexpr (FULL) {
              float av, ad;
              gate_act_grad(fv[e], a.act, av, ad);
              dv = dt * (sc[i] * av);
              gg[e] = dtv * (sc[i] * ad);
              acc[0][i] = fmaf(dtv, a.alpha * av, acc[0][i]);
            } else {
              dv = dt * k;
              accg[i] = fmaf(dtv, kd, accg[i]);
              acc[0][i] = fmaf(dtv, ka, acc[0][i]);
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
        if (q.image_gate && (t + 1 == t1 || (t + 1) % q.tpi == 0)) {
#pragma unroll
          for (int i = 0; i < CPT; ++i) {
            const float g = group_sum<PL>(accg[i]);
            if (inc[i] && pl == 0) q.gpart[(size_t)(wg + b) * a.C + cg + CG * i] = g;
            accg[i] = 0.f;
          }
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

// The partials of one parameter (blockIdx.y < 5) or of one image's gate (5 + image), 64 channels
// per workgroup, added in workgroup order: 16 threads a channel, then a tree over them.
template <typename T>
__global__ __launch_bounds__(1024) void block_fold(BlockArgs a, Plan q) {
  __shared__ float red[16][64];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), g = threadIdx.x >> 6, k = blockIdx.y;
  void* dst[5] = {a.gs, a.gw1, a.gb1, a.gw2, a.gb2};
  T* out = k < 5 ? static_cast<T*>(dst[k]) : static_cast<T*>(a.gg) + (size_t)(k - 5) * a.C;
  if (k < 5 && !dst[k]) return;
  float s = 0.f;
  if (c < a.C) {
    if (k < 5) {
#pragma unroll 4
      for (int w = g; w < q.wgs; w += 16) s += q.part[((size_t)w * 5 + k) * a.C + c];
    } else {
      // workgroups whose range meets this image's tiles
      const long lo = (long)(k - 5) * q.tpi, hi = lo + q.tpi;
      int w0 = (int)(lo * q.wgs / q.tiles);
      while (w0 > 0 && first_tile(q, w0) > lo) --w0;
      while (first_tile(q, w0 + 1) <= lo) ++w0;
      for (int w = w0 + g; w < q.wgs && first_tile(q, w) < hi; w += 16)
        if (first_tile(q, w + 1) > first_tile(q, w)) s += q.gpart[(size_t)(w + k - 5) * a.C + c];
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

constexpr int kMaxWgs = 1024;

// floats of the partials, then the gate's
size_t plan_floats(const BlockArgs& a) {
  return (size_t)kMaxWgs * 5 * a.C + (size_t)(kMaxWgs + a.B) * a.C;
}

template <typename T, int NT, int PL, int CPT, int WPE, int WGS, bool BWD>
hipError_t run_map(const BlockArgs& a, hipStream_t s) {
  constexpr int TP = PL * ElemVec<T>::N;
  Plan q{};
  q.tpi = (a.P + TP - 1) / TP;
  q.tiles = (long)q.tpi * a.B;
  q.images = a.B;
  q.P = a.P;
  const bool params = BWD && (a.gs || a.gw1 || a.gb1 || a.gw2 || a.gb2);
  q.image_gate = BWD && a.gg && a.gate_kind == DCN_GATE_IMAGE;
  q.wgs = (int)std::min<long>(q.tiles, WGS ? WGS : params || q.image_gate ? kMaxWgs : 1 << 20);
  if (params) q.part = a.ws;
  if (q.image_gate) q.gpart = a.ws + (size_t)kMaxWgs * 5 * a.C;
  const bool full = a.gate_kind == DCN_GATE_FULL, drop = a.drop.thr != 0;
  const dim3 grid(q.wgs), block(NT);
  if (full && drop)
    hipLaunchKernelGGL((block_map<T, NT, PL, CPT, WPE, WGS != 0, BWD, true, true>), grid, block, 0, s, a, q);
  else if (full)
    hipLaunchKernelGGL((block_map<T, NT, PL, CPT, WPE, WGS != 0, BWD, true, false>), grid, block, 0, s, a, q);
  else if (drop)
    hipLaunchKernelGGL((block_map<T, NT, PL, CPT, WPE, WGS != 0, BWD, false, true>), grid, block, 0, s, a, q);
  else
    hipLaunchKernelGGL((block_map<T, NT, PL, CPT, WPE, WGS != 0, BWD, false, false>), grid, block, 0, s, a, q);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !(params || q.image_gate)) return e;
  // without parameter gradients the first five rows have no destination and end at once
  hipLaunchKernelGGL((block_fold<T>), dim3((a.C + 63) / 64, 5 + (q.image_gate ? a.B : 0)),
                     dim3(1024), 0, s, a, q);
  return hipGetLastError();
}

// Threads, lanes along the positions, channels a thread, waves per SIMD and workgroups that
// prefetch their next tile (0: a workgroup per tile, or 1024 of them where parameters add up)
// by channels and direction, the fastest of those tried at 64 images (us, the best two):
//   bf16 forward   64x3136: 30, 44    128x784: 23, 25    256x784: 35, 35   512x196: 32, 36
//   bf16 backward  64x3136: 52, 79    128x784: 42, 47    256x784: 72, 89   512x196: 62, 147
//   f32 forward    64x3136: 46, 55    128x784: 31, 34    256x784: 57, 66   512x196: 46, 52
//   f32 backward   64x3136: 83, 108   128x784: 61, 100   256x784: 112, 191 512x196: 103, 168
// More channels than a workgroup's registers hold take narrower tiles (32-byte runs of a
// channel at 1024), which costs less than a second pass. false: no variant (C > 2048).
template <bool BWD>
bool map_variant(const BlockArgs& a, hipStream_t s, hipError_t* e) {
  const int C = a.C;
  if (a.dtype == DCN_BF16) {
    if (C <= 32) *e = run_map<bf16_t, 256, 8, 1, 3, 0, BWD>(a, s);
    else if (C <= 64) *e = run_map<bf16_t, 256, 8, 2, 2, 512, BWD>(a, s);
    else if (C <= 128) *e = run_map<bf16_t, 256, 4, 2, 2, 512, BWD>(a, s);
    else if (C <= 256 && !BWD) *e = run_map<bf16_t, 512, 4, 2, 4, 0, false>(a, s);
    else if (C <= 256) *e = run_map<bf16_t, 512, 4, 2, 2, 256, BWD>(a, s);
    else if (C <= 512 && !BWD) *e = run_map<bf16_t, 1024, 4, 2, 4, 0, false>(a, s);
    else if (C <= 512) *e = run_map<bf16_t, 512, 2, 2, 2, 256, BWD>(a, s);
    else if (C <= 1024) *e = run_map<bf16_t, 512, 2, 4, 2, 256, BWD>(a, s);
    else if (C <= 2048) *e = run_map<bf16_t, 1024, 2, 4, 4, 256, BWD>(a, s);
    else return false;
  } else {
    if (C <= 32) *e = run_map<float, 256, 8, 1, 3, 0, BWD>(a, s);
    else if (C <= 64) *e = run_map<float, 256, 8, 2, 4, 0, BWD>(a, s);
    else if (C <= 128) *e = run_map<float, 256, 8, 4, 2, 512, BWD>(a, s);
    else if (C <= 256 && !BWD) *e = run_map<float, 512, 8, 4, 4, 0, false>(a, s);
    else if (C <= 256) *e = run_map<float, 512, 8, 4, 2, 256, BWD>(a, s);
    else if (C <= 512) *e = run_map<float, 512, 4, 4, 2, 256, BWD>(a, s);
    else if (C <= 1024 && !BWD) *e = run_map<float, 512, 4, 8, 2, 256, false>(a, s);
    else if (C <= 1024) *e = run_map<float, 1024, 4, 4, 4, 0, BWD>(a, s);
    else if (C <= 2048) *e = run_map<float, 1024, 4, 8, 4, 256, BWD>(a, s);
    else return false;
  }
  return true;
}

template <typename T, int LP>
hipError_t any_fwd(const BlockArgs& a, hipStream_t s) {
  const size_t rows = (size_t)a.B * a.P, per = kThreads / LP;
  const unsigned grid = (unsigned)std::min<size_t>((rows + per - 1) / per, 1u << 20);
  hipLaunchKernelGGL((block_any_fwd<T, LP>), dim3(grid), dim3(kThreads), 0, s, a);
  return hipGetLastError();
}
template <typename T, int LP>
hipError_t any_bwd(const BlockArgs& a, hipStream_t s) {
  const size_t rows = (size_t)a.B * a.P, per = kThreads / LP;
  const unsigned grid = (unsigned)std::min<size_t>((rows + per - 1) / per, 1u << 20);
  hipLaunchKernelGGL((block_any_bwd<T, LP>), dim3(grid), dim3(kThreads), 0, s, a);
  hipError_t e = hipGetLastError();
  const bool image_gate = a.gg && a.gate_kind == DCN_GATE_IMAGE;
  if (e != hipSuccess || !(a.gs || a.gw1 || a.gb1 || a.gw2 || a.gb2 || image_gate)) return e;
  hipLaunchKernelGGL((block_any_params<T>), dim3(a.C), dim3(kThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace

size_t block_norm_ws_floats(const BlockArgs& a) {
  return std::max(6 * (size_t)a.B * a.P, plan_floats(a));
}

hipError_t launch_block_norm_fwd(const BlockArgs& a, hipStream_t s) {
  hipError_t e;
  if (a.layout == DCN_NCHW && map_variant<false>(a, s, &e)) return e;
  if (a.layout == DCN_NCHW)
    return a.dtype == DCN_BF16 ? any_fwd<bf16_t, 1>(a, s) : any_fwd<float, 1>(a, s);
  return a.dtype == DCN_BF16 ? any_fwd<bf16_t, 64>(a, s) : any_fwd<float, 64>(a, s);
}

hipError_t launch_block_norm_bwd(const BlockArgs& a, hipStream_t s) {
  hipError_t e;
  if (a.layout == DCN_NCHW && map_variant<true>(a, s, &e)) return e;
  if (a.layout == DCN_NCHW)
    return a.dtype == DCN_BF16 ? any_bwd<bf16_t, 1>(a, s) : any_bwd<float, 1>(a, s);
  return a.dtype == DCN_BF16 ? any_bwd<bf16_t, 64>(a, s) : any_bwd<float, 64>(a, s);
}

}  // namespace dcn
