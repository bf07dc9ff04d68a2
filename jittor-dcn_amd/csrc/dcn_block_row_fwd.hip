// dcn_block_row_fwd.hip — block norms on token rows, forward: which variant of block_row runs.
#include "dcn_block_norm.h"

namespace dcn {

// Threads, lanes a row, vectors a lane, waves per SIMD, workgroups (each prefetches its next
// rows; negative: does not). 16 channels a lane and two waves per SIMD: with four, or 32 channels
// a lane, the registers spill (8192 x 1024 bf16: 15.8 us against 20.7 and 25.4). Above 8192
// channels a row leaves no room for the next (512 x 16384 bf16 58 us with the prefetch, 32
// without, fp32 103, 76; 1024 x 8192 bf16 19, 24, fp32 37, 47). Up to 128 channels fewer lanes,
// or one vector a lane: those without a channel cost more than the width saves (50176 x 64 bf16
// 20 us on 16 lanes of two vectors, 10 on 8 of one; 200704 x 32 58, 15 on 4; 50176 x 128 20, 16 on
// 16 of one; fp32 23, 12 and 67, 26). false: no variant.
bool block_row_fwd(const BlockArgs& a, hipStream_t s, hipError_t* e) {
  const int C = a.C;
  if (a.dtype == DCN_BF16) {
    if (C <= 32) *e = run_row<bf16_t, 256, 4, 1, 4, 1024, false>(a, s);
    else if (C <= 64) *e = run_row<bf16_t, 256, 8, 1, 4, 1024, false>(a, s);
    else if (C <= 128) *e = run_row<bf16_t, 256, 16, 1, 4, 1024, false>(a, s);
    else if (C <= 256) *e = run_row<bf16_t, 256, 16, 2, 2, 512, false>(a, s);
    else if (C <= 512) *e = run_row<bf16_t, 256, 32, 2, 2, 512, false>(a, s);
    else if (C <= 1024) *e = run_row<bf16_t, 256, 64, 2, 2, 512, false>(a, s);
    else if (C <= 2048) *e = run_row<bf16_t, 256, 128, 2, 2, 512, false>(a, s);
    else if (C <= 4096) *e = run_row<bf16_t, 256, 256, 2, 2, 512, false>(a, s);
    else if (C <= 8192) *e = run_row<bf16_t, 512, 512, 2, 2, 256, false>(a, s);
    else if (C <= 16384) *e = run_row<bf16_t, 1024, 1024, 2, 4, -512, false>(a, s);
    else return false;
  } else {
    if (C <= 32) *e = run_row<float, 256, 8, 1, 4, 1024, false>(a, s);
    else if (C <= 64) *e = run_row<float, 256, 16, 1, 4, 1024, false>(a, s);
    else if (C <= 128) *e = run_row<float, 256, 16, 2, 4, 1024, false>(a, s);
    else if (C <= 256) *e = run_row<float, 256, 16, 4, 2, 512, false>(a, s);
    else if (C <= 512) *e = run_row<float, 256, 32, 4, 2, 512, false>(a, s);
    else if (C <= 1024) *e = run_row<float, 256, 64, 4, 2, 512, false>(a, s);
    else if (C <= 2048) *e = run_row<float, 256, 128, 4, 2, 512, false>(a, s);
    else if (C <= 4096) *e = run_row<float, 256, 256, 4, 2, 512, false>(a, s);
    else if (C <= 8192) *e = run_row<float, 512, 512, 4, 2, 256, false>(a, s);
    else if (C <= 16384) *e = run_row<float, 1024, 1024, 4, 4, -512, false>(a, s);
    else return false;
  }
  return true;
}

}  // namespace dcn
