// dcn_block.h — launchers of the residual block's operators (include/dcn.h, "residual block
// around a DeformConv2d"): dcn_dropout.hip, dcn_block_norm.hip, dcn_fp8.hip, dcn_fp8_gemm.hip.
// dcn_block.cpp holds the entry points and their checks.
#pragma once
#include "dcn_internal.h"
#include "dcn_philox.h"

namespace dcn {

// y = res + drop(x) (res may be null); n elements, `group` to a draw
hipError_t launch_dropout(const DropArgs& a, int dtype, const void* x, const void* res, void* y,
                          uint64_t n, uint64_t group, hipStream_t s);

// One block-norm call (dcn_block_desc / dcn_block_io): 1 = post, 2 = pre.
struct BlockArgs {
  const void *x, *res, *gate, *scale, *w1, *b1, *w2, *b2;
  void *out, *y;
  const void *go, *gy;
  void *gx, *gr, *gg, *gs, *gw1, *gb1, *gw2, *gb2;
  float* ws;
  float* stats;  // [4][B · P]: m1, r1, m2, r2 of every position, or null
  DropArgs drop;
  int B, C, P, layout, dtype, post, pre, gate_kind, act, drop_image;
  float eps1, eps2, alpha;
};
size_t block_norm_ws_floats(const BlockArgs& a);
hipError_t launch_block_norm_fwd(const BlockArgs& a, hipStream_t s);
hipError_t launch_block_norm_bwd(const BlockArgs& a, hipStream_t s);

hipError_t launch_fp8_quantize(int B, int C, int P, int layout, int dtype, const void* v,
                               void* q_tok, void* s_tok, void* q_ch, void* s_ch, hipStream_t s);
hipError_t launch_fp8_quantize_weight(int O, int C, int dtype, const void* w, void* q, void* sq,
                                      void* qT, void* sT, hipStream_t s);
// both in one launch (x [B][C][P] or tokens, w [O][C])
hipError_t launch_fp8_quantize_both(int B, int C, int P, int layout, int dtype, const void* v,
                                    void* q_tok, void* s_tok, void* q_ch, void* s_ch, int O,
                                    const void* w, void* q, void* sq, void* qT, void* sT,
                                    hipStream_t s);
size_t fp8_matmul_ws_bytes(const dcn_fp8_matmul_desc& d);
hipError_t launch_fp8_matmul(const dcn_fp8_matmul_desc& d, const void* a, const void* sa,
                             const void* b, const void* sb, void* out, void* ws, hipStream_t s);
// The product of few tokens x [d.M][cols] that are not rounded yet with b, in one launch.
bool fp8_few_tokens(size_t tokens);
hipError_t launch_fp8_few_tokens(const dcn_fp8_matmul_desc& d, int cols, const void* x,
                                 const void* w, const void* sw, void* out, hipStream_t s);

}  // namespace dcn
