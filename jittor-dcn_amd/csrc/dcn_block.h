// dcn_block.h — launchers of the residual block's operators (include/dcn.h, "residual block
// around a DeformConv2d"): dcn_dropout.hip, dcn_block_norm.hip, dcn_fp8.hip, dcn_fp8_gemm.hip.
// dcn_block.cpp holds the entry points and their checks.
#pragma once
#include "dcn_internal.h"

namespace dcn {

struct DropArgs;
// y = res + drop(x) (res may be null); n elements, `group` to a draw
hipError_t launch_dropout(const DropArgs& a, int dtype, const void* x, const void* res, void* y,
                          uint64_t n, uint64_t group, hipStream_t s);

}  // namespace dcn
