// fp32 numbers as sums of bf16 parts.
#pragma once
#include <cuda_bf16.h>
#include <cstdint>

namespace abacus {
namespace ragged {

// Magnitudes (as bits) from which on rounding to bf16 gives infinity; infinities and NaN are above too.
constexpr uint32_t kRoundsToInfinity = 0x7f7f8000u;

__device__ __forceinline__ uint32_t bits_of(__nv_bfloat162 x) { return *reinterpret_cast<const uint32_t*>(&x); }

// x = part 0 + part 1 + part 2 for two numbers at once (a in the low halves), each part the rounded remainder of those
// before. Both below kRoundsToInfinity.
__device__ __forceinline__ void split_two(float a, float b, uint32_t (&part)[3]) {
  part[0] = bits_of(__floats2bfloat162_rn(a, b));
  a -= __uint_as_float(part[0] << 16);
  b -= __uint_as_float(part[0] & 0xffff0000u);
  part[1] = bits_of(__floats2bfloat162_rn(a, b));
  a -= __uint_as_float(part[1] << 16);
  b -= __uint_as_float(part[1] & 0xffff0000u);
  part[2] = bits_of(__floats2bfloat162_rn(a, b));
}

// What is left of x once its first part is taken, and that part cut to 8 bits instead of rounded: for numbers so large
// that rounding would overflow. An infinite or NaN x is its first part alone.
__device__ __forceinline__ float take_large(float& x) {
  const uint32_t u = __float_as_uint(x);
  if ((u & 0x7fffffffu) < kRoundsToInfinity) return 0.f;
  if ((u & 0x7fffffffu) >= 0x7f800000u) {
    const float whole = (u & 0x7fffffffu) > 0x7f800000u ? __uint_as_float(0x7fff0000u) : x;
    x = 0.f;
    return whole;
  }
  const float cut = __uint_as_float(u & 0xffff0000u);
  x -= cut;
  return cut;
}

// The same for any eight numbers: words[p] holds part p of them. The test for large ones is one for all eight.
__device__ __forceinline__ void split_eight(const float* v, uint4 (&words)[3]) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
  uint32_t w[3][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t part[3];
    split_two(v[2 * j], v[2 * j + 1], part);
    w[0][j] = part[0];
    w[1][j] = part[1];
    w[2][j] = part[2];
  }
  if (top >= kRoundsToInfinity) {
#pragma unroll 1
    for (int j = 0; j < 8; ++j) {
      float x = v[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) x = i == j ? v[i] : x;
      const float first = take_large(x);
      if (first == 0.f) continue;  // an ordinary number
      uint32_t rest[3];
      split_two(x, 0.f, rest);
      const uint32_t halves[3] = {__float_as_uint(first) >> 16, rest[0] & 0xffffu, rest[1] & 0xffffu};
      const uint32_t shift = (j & 1) * 16;
#pragma unroll
      for (int p = 0; p < 3; ++p) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i == j / 2) w[p][i] = (w[p][i] & (0xffff0000u >> shift)) | (halves[p] << shift);
      }
    }
  }
#pragma unroll
  for (int p = 0; p < 3; ++p) words[p] = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
}

}  // namespace ragged
}  // namespace abacus
