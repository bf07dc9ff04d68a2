// dcn_block_row_bwd.hip — block norms on token rows, backward: which variant of block_row runs.
#include "dcn_block_norm.h"

namespace dcn {

// As forward, with 8 channels a lane: the five parameter sums of every channel stay in
// registers beside the rows (8192 x 1024 bf16: 37 us; 75 us with 16 channels a lane, 83 us
// with four waves per SIMD). Few channels take fewer lanes (64 x 3136 x 32 bf16 64 us on 16 lanes a
// row, 28 on 4; fp32 64, 41). Above 4096 channels the parameters' sums take a pass of their own
// (us, one pass with its spills against two: bf16 2048 x 5120 92, 66, 1024 x 8192 65, 57,
// 512 x 16384 253, 91; fp32 188, 118, 130, 101, 357, 182; the first pass prefetches in bf16, 68
// against 86, and not in fp32, 118 against 125), save beside a full gate in bf16 up to 8192, which
// adds a tensor to the second pass and spares the gate's sums in the first (76, 90 and 62, 72).
// false: no variant.
bool block_row_bwd(const BlockArgs& a, hipStream_t s, hipError_t* e) {
  const int C = a.C;
  if (a.dtype == DCN_BF16) {
    if (C <= 32) *e = run_row<bf16_t, 256, 4, 1, 2, 512, true>(a, s);
    else if (C <= 64) *e = run_row<bf16_t, 256, 8, 1, 2, 512, true>(a, s);
    else if (C <= 128) *e = run_row<bf16_t, 256, 16, 1, 2, 512, true>(a, s);
    else if (C <= 256) *e = run_row<bf16_t, 256, 32, 1, 2, 512, true>(a, s);
    else if (C <= 512) *e = run_row<bf16_t, 256, 64, 1, 2, 512, true>(a, s);
    else if (C <= 1024) *e = run_row<bf16_t, 256, 128, 1, 2, 512, true>(a, s);
    else if (C <= 2048) *e = run_row<bf16_t, 256, 256, 1, 2, 512, true>(a, s);
    else if (C <= 4096) *e = run_row<bf16_t, 512, 512, 1, 2, 256, true>(a, s);
    else if (C <= 8192 && a.gate_kind == DCN_GATE_FULL && one_run(a))
      *e = run_gated_row<bf16_t, 512, 2, 2, 256>(a, s);
    else if (C <= 8192) *e = run_long_row<bf16_t, 512, 2, 2, true, 512>(a, s);
    else if (C <= 16384) *e = run_long_row<bf16_t, 1024, 2, 4, false, 512>(a, s);
    else return false;
  } else {
    if (C <= 32) *e = run_row<float, 256, 8, 1, 4, 512, true>(a, s);
    else if (C <= 64) *e = run_row<float, 256, 16, 1, 4, 512, true>(a, s);
    else if (C <= 128) *e = run_row<float, 256, 16, 2, 2, 512, true>(a, s);
    else if (C <= 256) *e = run_row<float, 256, 32, 2, 2, 512, true>(a, s);
    else if (C <= 512) *e = run_row<float, 256, 64, 2, 2, 512, true>(a, s);
    else if (C <= 1024) *e = run_row<float, 256, 128, 2, 2, 512, true>(a, s);
    else if (C <= 2048) *e = run_row<float, 256, 256, 2, 2, 512, true>(a, s);
    else if (C <= 4096) *e = run_row<float, 512, 512, 2, 2, 256, true>(a, s);
    else if (C <= 8192) *e = run_long_row<float, 512, 4, 2, false, 512>(a, s);
    else if (C <= 16384) *e = run_long_row<float, 1024, 4, 4, false, 512>(a, s);
    else return false;
  }
  return true;
}

}  // namespace dcn
