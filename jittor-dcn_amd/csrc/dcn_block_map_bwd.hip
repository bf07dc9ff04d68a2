// dcn_block_map_bwd.hip — block norms on maps, backward: which variant of block_map runs.
#include "dcn_block_norm.h"

namespace dcn {

// Threads, lanes along the positions, channels a thread, waves per SIMD and workgroups that
// prefetch their next tile (0: up to 1024 that do not) by channels; the fastest of those tried
// at 64 images (us, the best two, tiles not yet interleaved):
//   bf16  64x3136: 52, 79   128x784: 42, 47   256x784: 72, 89   512x196: 62, 147
//   fp32  64x3136: 83, 108  128x784: 61, 100  256x784: 112, 191  512x196: 103, 168
// false: no variant (C > 2048).
bool block_map_bwd(const BlockArgs& a, hipStream_t s, hipError_t* e) {
  const int C = a.C;
  if (a.dtype == DCN_BF16) {
    if (C <= 32) *e = run_map<bf16_t, 256, 8, 1, 3, 0, true>(a, s);
    else if (C <= 64) *e = run_map<bf16_t, 256, 8, 2, 2, 512, true>(a, s);
    else if (C <= 128) *e = run_map<bf16_t, 256, 4, 2, 2, 512, true>(a, s);
    else if (C <= 256) *e = run_map<bf16_t, 512, 4, 2, 2, 256, true>(a, s);
    else if (C <= 512) *e = run_map<bf16_t, 512, 2, 2, 2, 256, true>(a, s);
    else if (C <= 1024) *e = run_map<bf16_t, 512, 2, 4, 2, 256, true>(a, s);
    else if (C <= 2048) *e = run_map<bf16_t, 1024, 2, 4, 4, 256, true>(a, s);
    else return false;
  } else {
    if (C <= 32) *e = run_map<float, 256, 8, 1, 3, 0, true>(a, s);
    else if (C <= 64) *e = run_map<float, 256, 8, 2, 4, 0, true>(a, s);
    else if (C <= 128) *e = run_map<float, 256, 8, 4, 2, 512, true>(a, s);
    else if (C <= 256) *e = run_map<float, 512, 8, 4, 2, 256, true>(a, s);
    else if (C <= 512) *e = run_map<float, 512, 4, 4, 2, 256, true>(a, s);
    else if (C <= 1024) *e = run_map<float, 1024, 4, 4, 4, 0, true>(a, s);
    else if (C <= 2048) *e = run_map<float, 1024, 4, 8, 4, 256, true>(a, s);
    else return false;
  }
  return true;
}

}  // namespace dcn
