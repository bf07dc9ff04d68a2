// dcn_dropout.hip — dropout whose mask is drawn from (seed, offset, element) and never stored:
// y = residual + keep(i) ? x · scale : 0, and the same map on the gradient (include/dcn.h).
//
// A stream: x (and residual) read once, y written once, no other memory. Eight elements per
// thread and step, one Philox call for them; the draws of a group > 1 (channel maps, images)
// come from the group's index, two groups at most inside one vector unless groups are tiny.
#include "dcn_philox.h"

namespace dcn {

namespace {

constexpr int kThreads = 256;

template <typename T>
__device__ __forceinline__ void ld8(const T* p, int valid, float (&v)[8]) {
  constexpr int N = ElemVec<T>::N;
#pragma unroll
  for (int h = 0; h < 8; h += N) {
    float t[N];
    ldv(p + h, valid - h, t);
#pragma unroll
    for (int j = 0; j < N; ++j) v[h + j] = t[j];
  }
}
template <typename T>
__device__ __forceinline__ void st8(T* p, int valid, const float (&v)[8]) {
  constexpr int N = ElemVec<T>::N;
#pragma unroll
  for (int h = 0; h < 8; h += N) {
    float t[N];
#pragma unroll
    for (int j = 0; j < N; ++j) t[j] = v[h + j];
    stv(p + h, valid - h, t);
  }
}

// keep bits of the eight elements from i0 (a multiple of 8), `group` elements to a draw
__device__ unsigned keep_grouped(uint64_t i0, uint64_t group, const PhiloxKey& k, unsigned thr) {
  uint64_t d, r;
  if ((i0 >> 32) == 0 && (group >> 32) == 0) {  // 32-bit division where it is enough
    d = (unsigned)i0 / (unsigned)group;
    r = i0 - d * group;
  } else {
    d = i0 / group;
    r = i0 - d * group;
  }
  uint64_t blk = d >> 3;
  unsigned cur = keep8(blk, k, thr), m = 0;
  for (int j = 0; j < 8; ++j) {
    m |= ((cur >> (d & 7)) & 1u) << j;
    if (++r == group) {
      r = 0;
      ++d;
      if ((d >> 3) != blk && j < 7) {
        blk = d >> 3;
        cur = keep8(blk, k, thr);
      }
    }
  }
  return m;
}

template <typename T, bool GROUPED, bool RES>
__global__ __launch_bounds__(kThreads) void dropout_kernel(DropArgs a, const T* x, const T* res,
                                                           T* y, uint64_t n, uint64_t group) {
  const PhiloxKey k = philox_key(a);
  const uint64_t step = (uint64_t)gridDim.x * kThreads * 8;
  for (uint64_t i = ((uint64_t)blockIdx.x * kThreads + threadIdx.x) * 8; i < n; i += step) {
    const int valid = (int)min((uint64_t)8, n - i);
    float v[8], r[8];
    ld8(x + i, valid, v);
    if (RES) ld8(res + i, valid, r);
    const unsigned m = GROUPED ? keep_grouped(i, group, k, a.thr) : keep8(i >> 3, k, a.thr);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float t = (m >> j) & 1u ? v[j] * a.scale : 0.f;
      v[j] = RES ? r[j] + t : t;
    }
    st8(y + i, valid, v);
  }
}

template <typename T, bool GROUPED>
void launch_t(const DropArgs& a, const void* x, const void* res, void* y, uint64_t n,
              uint64_t group, unsigned grid, hipStream_t s) {
  const T* xt = static_cast<const T*>(x);
  T* yt = static_cast<T*>(y);
  if (res)
    hipLaunchKernelGGL((dropout_kernel<T, GROUPED, true>), dim3(grid), dim3(kThreads), 0, s, a, xt,
                       static_cast<const T*>(res), yt, n, group);
  else
    hipLaunchKernelGGL((dropout_kernel<T, GROUPED, false>), dim3(grid), dim3(kThreads), 0, s, a,
                       xt, static_cast<const T*>(nullptr), yt, n, group);
}

}  // namespace

hipError_t launch_dropout(const DropArgs& a, int dtype, const void* x, const void* res, void* y,
                          uint64_t n, uint64_t group, hipStream_t s) {
  if (n == 0) return hipSuccess;
  const uint64_t blocks = (n + 8ull * kThreads - 1) / (8ull * kThreads);
  const unsigned grid = (unsigned)std::min<uint64_t>(blocks, 1u << 20);
  if (dtype == DCN_BF16)
    group > 1 ? launch_t<bf16_t, true>(a, x, res, y, n, group, grid, s)
              : launch_t<bf16_t, false>(a, x, res, y, n, group, grid, s);
  else
    group > 1 ? launch_t<float, true>(a, x, res, y, n, group, grid, s)
              : launch_t<float, false>(a, x, res, y, n, group, grid, s);
  return hipGetLastError();
}

}  // namespace dcn
