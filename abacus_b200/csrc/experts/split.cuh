// fp32 numbers as sums of bf16 parts.
#pragma once
#include <cuda_bf16.h>

namespace abacus {
namespace ragged {

// x = part[0] + part[1] + part[2], each part the rounded remainder of those before. An infinite or NaN x is part[0]
// alone; a finite one too large to round up to bf16 is cut instead, so that it stays finite.
__device__ __forceinline__ void split(float x, __nv_bfloat16 (&part)[3]) {
  const bool finite = isfinite(x);
  float h = __bfloat162float(__float2bfloat16_rn(x));
  if (finite && !isfinite(h)) h = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
  part[0] = __float2bfloat16_rn(h);
  const float r = finite ? x - h : 0.f;
  const float m = __bfloat162float(__float2bfloat16_rn(r));
  part[1] = __float2bfloat16_rn(m);
  part[2] = __float2bfloat16_rn(r - m);
}

}  // namespace ragged
}  // namespace abacus
