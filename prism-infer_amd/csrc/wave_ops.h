// Scans and reductions over the lanes of a wave, by DPP (no LDS round trips).
#pragma once

#include "common.h"

namespace prism {

// A uniform value in an SGPR.
__device__ __forceinline__ int uniform_int(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Inclusive scan with f over lanes of non-negative values (0 is f's neutral
// element): row shifts, then the row ends broadcast onwards.
template <typename F>
__device__ __forceinline__ int wave_scan(int v, F f) {
  v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false));  // row_shr:1
  v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false));  // row_shr:2
  v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false));  // row_shr:4
  v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false));  // row_shr:8
  v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false));  // row_bcast:15 into rows 1 and 3
  return f(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false));  // row_bcast:31 into rows 2 and 3
}

struct Add {
  __device__ int operator()(int x, int y) const { return x + y; }
};
struct Max {
  __device__ int operator()(int x, int y) const { return max(x, y); }
};

template <typename F>
__device__ __forceinline__ int wave_reduce(int v, F f) {
  return __builtin_amdgcn_readlane(wave_scan(v, f), 63);
}

}  // namespace prism
