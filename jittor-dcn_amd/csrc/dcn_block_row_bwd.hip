// dcn_block_row_bwd.hip — block norms on token rows, backward: which variant of block_row runs.
#include "dcn_block_norm.h"

namespace dcn {

// As forward, with 8 channels a lane: the five parameter sums of every channel stay in
// registers beside the rows (8192 x 1024 bf16: 37 us; 75 us with 16 channels a lane, 83 us
// with four waves per SIMD). Above 4096 bf16 channels (or 8192 fp32) 16 a lane are needed: without the
// prefetch and the kept parameters (a negative count) less spills (1024 x 8192 bf16: 66 us
// against 150, fp32 139 against 191). false: no variant.
bool block_row_bwd(const BlockArgs& a, hipStream_t s, hipError_t* e) {
  const int C = a.C;
  if (a.dtype == DCN_BF16) {
    if (C <= 128) *e = run_row<bf16_t, 256, 16, 1, 2, 512, true>(a, s);
    else if (C <= 256) *e = run_row<bf16_t, 256, 32, 1, 2, 512, true>(a, s);
    else if (C <= 512) *e = run_row<bf16_t, 256, 64, 1, 2, 512, true>(a, s);
    else if (C <= 1024) *e = run_row<bf16_t, 256, 128, 1, 2, 512, true>(a, s);
    else if (C <= 2048) *e = run_row<bf16_t, 256, 256, 1, 2, 512, true>(a, s);
    else if (C <= 4096) *e = run_row<bf16_t, 512, 512, 1, 2, 256, true>(a, s);
    else if (C <= 8192) *e = run_row<bf16_t, 512, 512, 2, 2, -256, true>(a, s);
    else if (C <= 16384) *e = run_row<bf16_t, 1024, 1024, 2, 4, -256, true>(a, s);
    else return false;
  } else {
    if (C <= 128) *e = run_row<float, 256, 16, 2, 2, 512, true>(a, s);
    else if (C <= 256) *e = run_row<float, 256, 32, 2, 2, 512, true>(a, s);
    else if (C <= 512) *e = run_row<float, 256, 64, 2, 2, 512, true>(a, s);
    else if (C <= 1024) *e = run_row<float, 256, 128, 2, 2, 512, true>(a, s);
    else if (C <= 2048) *e = run_row<float, 256, 256, 2, 2, 512, true>(a, s);
    else if (C <= 4096) *e = run_row<float, 512, 512, 2, 2, 256, true>(a, s);
    else if (C <= 8192) *e = run_row<float, 1024, 1024, 2, 4, -256, true>(a, s);
    else if (C <= 16384) *e = run_row<float, 1024, 1024, 4, 4, -256, true>(a, s);
    else return false;
  }
  return true;
}

}  // namespace dcn
