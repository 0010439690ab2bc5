// The caller's offsets of sorted rows.
#pragma once
#include "../common/sm100.cuh"

namespace abacus {
namespace ragged {

// Called by one warp of a launch: offsets that do not start at 0, decrease, or end after the rows are the caller's mistake.
// The kernels clamp what they read of them, so it shows in the device status, and in results that say nothing.
__device__ __forceinline__ void check_offsets(const int* offsets, int experts, int rows, int lane, int* status) {
  bool bad = lane == 0 && (offsets[0] != 0 || offsets[experts] > rows);
  for (int e = lane; e < experts; e += 32) bad = bad || offsets[e + 1] < offsets[e];
  if (bad) atomicCAS(status, kStatusOk, kStatusBadArgs);
}

}  // namespace ragged
}  // namespace abacus
