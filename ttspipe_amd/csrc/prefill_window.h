// The launch of prefill_window.hip, for the entry point in prefill_attn.hip.
#pragma once

#include <hip/hip_runtime.h>

namespace ttsp {

// Workgroups from which on the rows' tiles are 128 rows, and below it 64.
constexpr int PW_FULL = 256, PW_LEAST = 1;

// The kernel's tiles (32 rows each) a workgroup for these shapes, 0: too few rows for it.
int prompt_window_tiles(int S, int nh, int nkv);

// The arguments are checked by the entry point; hipErrorInvalidValue where a launch cannot count its workgroups.
int prompt_window_launch(const void* Q, long long q_ss, long long q_sh, const void* K, long long k_ss, long long k_sh,
                         const void* V, long long v_ss, long long v_sh, const long long* pos, void* Y, int S, int nh,
                         int nkv, int L, int window, int sinks, float scale, int dtype, int tiles, hipStream_t stream);

}  // namespace ttsp
