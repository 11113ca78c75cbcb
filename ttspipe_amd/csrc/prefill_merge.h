// The joining launch of attention whose keys are split over workgroups (prefill_attn.hip).
#pragma once

#include <hip/hip_runtime.h>

namespace ttsp {

// Y [S][nh][128] of `dtype` from `splits` (2 to 16) workgroups' sums: per split, row and head 128
// unnormalised values, behind all of them the reference (log2 units) and the sum of the weights.
void prefill_merge(const float* work, int splits, int S, int nh, void* Y, int dtype, hipStream_t stream);

}  // namespace ttsp
