// dcn_block_map_bwd.hip — block norms on maps, backward: which variant of block_map runs.
#include "dcn_block_norm.h"

namespace dcn {

// Threads, lanes along the positions, channels a thread, waves per SIMD and workgroups that
// prefetch their next tile (negative: that do not; 0: up to 1024 that do not) by channels; the
// fastest of those tried at 64 images. The prefetch, us with and without (layer norms, no gate;
// then a full gate): bf16 256x784 54, 67; 74, 88   512x196 46, 50; 63, 72   1024x196 130, 97;
// 182, 136   fp32 128x784 50, 48; 70, 66   256x784 92, 86; 134, 122   512x196 61, 59; 84, 82
// 1024x196 226, 159; 254, 224: a second tile in registers costs fp32 and wide maps spills that
// cost more than the wait. false: no variant (C > 2048).
bool block_map_bwd(const BlockArgs& a, hipStream_t s, hipError_t* e) {
  const int C = a.C;
  if (a.dtype == DCN_BF16) {
    if (C <= 32) *e = run_map<bf16_t, 256, 8, 1, 3, 0, true>(a, s);
    else if (C <= 64) *e = run_map<bf16_t, 256, 8, 2, 2, 512, true>(a, s);
    else if (C <= 128) *e = run_map<bf16_t, 256, 4, 2, 2, 512, true>(a, s);
    else if (C <= 256) *e = run_map<bf16_t, 512, 4, 2, 2, 256, true>(a, s);
    else if (C <= 512) *e = run_map<bf16_t, 512, 2, 2, 2, 256, true>(a, s);
    else if (C <= 1024) *e = run_map<bf16_t, 512, 2, 4, 2, -256, true>(a, s);
    else if (C <= 2048) *e = run_map<bf16_t, 512, 2, 8, 2, 0, true>(a, s);
    else return false;
  } else {
    if (C <= 32) *e = run_map<float, 256, 8, 1, 3, 0, true>(a, s);
    else if (C <= 64) *e = run_map<float, 256, 8, 2, 4, 0, true>(a, s);
    else if (C <= 128) *e = run_map<float, 256, 8, 4, 2, -512, true>(a, s);
    else if (C <= 256) *e = run_map<float, 512, 8, 4, 2, -256, true>(a, s);
    else if (C <= 512) *e = run_map<float, 512, 4, 4, 2, -256, true>(a, s);
    else if (C <= 1024) *e = run_map<float, 512, 4, 8, 2, -256, true>(a, s);
    else if (C <= 2048) *e = run_map<float, 512, 4, 16, 2, -256, true>(a, s);
    else return false;
  }
  return true;
}

}  // namespace dcn
