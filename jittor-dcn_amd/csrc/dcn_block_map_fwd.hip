// dcn_block_map_fwd.hip — block norms on maps, forward: which variant of block_map runs.
#include "dcn_block_norm.h"

namespace dcn {

// Threads, lanes along the positions, channels a thread, waves per SIMD and workgroups that
// prefetch their next tile (0: one workgroup per tile) by channels; the fastest of those tried
// at 64 images (us, the best two):
//   bf16  64x3136: 30, 44   128x784: 23, 25   256x784: 31, 34   512x196: 28, 36
//   fp32  64x3136: 46, 55   128x784: 31, 34   256x3136: 178, 179   512x196: 35, 52
// 256 bf16 channels want four waves per SIMD more than the prefetch with dropout (64x256x196 17 us,
// 21; 64x200x784 36, 41) and where 256 workgroups would get three tiles of 32 positions or fewer
// (64x256x196 12.4 us, 14.4; 32x256x784, 800 tiles, 17.6, 17.8; 64x256x784 34, 31).
// Above 512 channels fp32, above 1024 bf16 spill beside a prefetched tile (64x1024x196 fp32 with a
// full gate 143 us with it, 103 without; 64x2048x49 bf16 44, 30).
// More channels than a workgroup's registers hold take narrower tiles (32-byte runs of a
// channel at 1024), which costs less than a second pass. false: no variant (C > 2048).
bool block_map_fwd(const BlockArgs& a, hipStream_t s, hipError_t* e) {
  const int C = a.C;
  if (a.dtype == DCN_BF16) {
    if (C <= 32) *e = run_map<bf16_t, 256, 8, 1, 3, 0, false>(a, s);
    else if (C <= 64) *e = run_map<bf16_t, 256, 8, 2, 2, 512, false>(a, s);
    else if (C <= 128) *e = run_map<bf16_t, 256, 4, 2, 2, 512, false>(a, s);
    else if (C <= 256 && (a.drop.thr || (long)a.B * ((a.P + 31) / 32) <= 3 * 256))
      *e = run_map<bf16_t, 512, 4, 2, 4, 0, false>(a, s);
    else if (C <= 256) *e = run_map<bf16_t, 512, 4, 2, 2, 256, false>(a, s);
    else if (C <= 512) *e = run_map<bf16_t, 1024, 4, 2, 4, 0, false>(a, s);
    else if (C <= 1024) *e = run_map<bf16_t, 512, 2, 4, 2, 256, false>(a, s);
    else if (C <= 2048) *e = run_map<bf16_t, 512, 2, 8, 2, 0, false>(a, s);
    else return false;
  } else {
    if (C <= 32) *e = run_map<float, 256, 8, 1, 3, 0, false>(a, s);
    else if (C <= 64) *e = run_map<float, 256, 8, 2, 4, 0, false>(a, s);
    else if (C <= 128) *e = run_map<float, 256, 8, 4, 2, 512, false>(a, s);
    else if (C <= 256) *e = run_map<float, 512, 8, 4, 2, 256, false>(a, s);
    else if (C <= 512) *e = run_map<float, 512, 4, 4, 2, 256, false>(a, s);
    else if (C <= 1024) *e = run_map<float, 512, 4, 8, 2, 0, false>(a, s);
    else if (C <= 2048) *e = run_map<float, 512, 4, 16, 2, 0, false>(a, s);
    else return false;
  }
  return true;
}

}  // namespace dcn
