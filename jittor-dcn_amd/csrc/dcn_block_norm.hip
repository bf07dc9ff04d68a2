// dcn_block_norm.hip — block norms of any size (dcn_block_norm.h has the formulas): the variant
// that keeps the channels in registers where there is one, else several passes over them.
#include "dcn_block_norm.h"

namespace dcn {

namespace {

constexpr int kThreads = 256;

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
  __device__ float x(int c) const { return drop_all ? 0.f : ld(a.x, base + c * cs); }
  __device__ float h1(int c) const { return (x(c) - m1) * r1; }
  __device__ float v(int c) const {
    return a.post ? h1(c) * par(a.w1, c, 1.f) + par(a.b1, c, 0.f) : x(c);
  }
  __device__ float gate(int c) const {
    return drop_all ? 0.f : ld(a.gate, a.gate_kind == DCN_GATE_FULL ? base + c * cs : (size_t)b * a.C + c);
  }
  __device__ float act(int c) const { return a.gate_kind ? gate_act<T>(gate(c), a.act) : 1.f; }
  __device__ float k(int c) const { return a.alpha * par(a.scale, c, 1.f) * act(c); }
  __device__ bool kept(int c) const {
    return !a.drop.thr || (a.drop_image ? !drop_all : keep1(base + c * cs, key, a.drop.thr));
  }
  __device__ float drop(float t, int c) const {
    return kept(c) ? (a.drop.thr ? t * a.drop.scale : t) : 0.f;
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
__device__ __forceinline__ void pos_moments(Pos<T>& q, int lane, size_t row, bool known) {
  const BlockArgs& a = q.a;
  const size_t rows = (size_t)a.B * a.P;
  if (known) {
    if (a.x && a.post && !q.drop_all) {
      q.m1 = a.stats[row];
      q.r1 = a.stats[rows + row];
    }
    if (a.pre) {
      q.m2 = a.stats[2 * rows + row];
      q.r2 = a.stats[3 * rows + row];
    }
    return;
  }
  if (a.x && a.post && !q.drop_all)
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
    pos_moments<T, LP>(q, lane, row, false);
    if (a.stats && lane == 0) {
      const float st[4] = {q.m1, q.r1, q.m2, q.r2};
#pragma unroll
      for (int k = 0; k < 4; ++k) a.stats[k * rows + row] = st[k];
    }
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
    pos_moments<T, LP>(q, lane, row, a.stats != nullptr);
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
        if (!q.kept(c)) continue;
        const float g = total(c), dt = a.drop.thr ? g * a.drop.scale : g;
        const float w = dt * q.k(c) * q.par(a.w1, c, 1.f);
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
      const bool kept = q.kept(c);
      const float dt = a.drop.thr ? g * a.drop.scale : g;
      if (a.gg && a.gate_kind == DCN_GATE_FULL) {
        float av, ad;
        gate_act_grad<T>(q.gate(c), a.act, av, ad);
        const float gg = dt * q.v(c) * (a.alpha * q.par(a.scale, c, 1.f)) * ad;
        static_cast<T*>(a.gg)[i] = from_f32(kept ? gg : 0.f, T());
      }
      if (a.gx) {
        const float dv = kept ? dt * q.k(c) : 0.f;
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
      if (!a.x || !q.kept(c)) continue;
      const float dt = a.drop.thr ? g * a.drop.scale : g, v = q.v(c);
      float av = 1.f, ad = 0.f;
      if (a.gate_kind) gate_act_grad<T>(q.gate(c), a.act, av, ad);
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

// channels that the register-resident variants take
constexpr int kMapChannels = 2048, kRowChannels = 16384;

size_t block_norm_ws_floats(const BlockArgs& a) {
  const bool rows = a.layout == DCN_NHWC || a.P == 1;  // a one-position map is a row
  // six numbers a position for the passes, or partials of the parameters and of an image gate
  // (interleaved where an image has kInterleave tiles, of 16 positions at least)
  if (a.C > (rows ? kRowChannels : kMapChannels)) return 6 * (size_t)a.B * a.P;
  const int wgs = partial_wgs(a);
  const int group = rows || a.P <= 16 * (kInterleave - 1) ? 1 : kInterleave;
  size_t partials = (size_t)wgs * 5 * a.C;
  if (a.gate_kind == DCN_GATE_IMAGE) partials += (wgs + (size_t)a.B * group) * a.C;
  if (rows && a.C > kRowSums) partials += ((size_t)a.B * a.P * 6 + 63) / 64 * 64;
  return partials;
}

hipError_t launch_block_norm_fwd(const BlockArgs& a, hipStream_t s) {
  hipError_t e;
  const bool rows = a.layout == DCN_NHWC || a.P == 1;
  if (rows ? block_row_fwd(a, s, &e) : block_map_fwd(a, s, &e)) return e;
  if (!rows) return a.dtype == DCN_BF16 ? any_fwd<bf16_t, 1>(a, s) : any_fwd<float, 1>(a, s);
  return a.dtype == DCN_BF16 ? any_fwd<bf16_t, 64>(a, s) : any_fwd<float, 64>(a, s);
}

hipError_t launch_block_norm_bwd(const BlockArgs& a, hipStream_t s) {
  hipError_t e;
  const bool rows = a.layout == DCN_NHWC || a.P == 1;
  if (rows ? block_row_bwd(a, s, &e) : block_map_bwd(a, s, &e)) return e;
  if (!rows) return a.dtype == DCN_BF16 ? any_bwd<bf16_t, 1>(a, s) : any_bwd<float, 1>(a, s);
  return a.dtype == DCN_BF16 ? any_bwd<bf16_t, 64>(a, s) : any_bwd<float, 64>(a, s);
}

}  // namespace dcn
