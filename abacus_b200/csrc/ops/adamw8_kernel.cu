// AdamW over many tensors with both moments held in 8 bits.
//
//   m <- b1 m + (1 - b1) g                 u <- sqrt(b2 u^2 + (1 - b2) g^2)
//   w <- w (1 - lr wd) - lr / (1 - b1^t) * m / (u / sqrt(1 - b2^t) + eps)
//
// m and u (the root of the second moment) are e4m3 numbers times one power of
// two per 256 consecutive elements of a tensor, the one that brings the
// largest finite magnitude of those elements into [128, 256). The scale is a
// power of two, so a moment that a step leaves alone is stored back without a
// second rounding. u rather than u^2 is stored because e4m3 spans 2^17 and a
// second moment twice the octaves of its root.
//
// Rounding to 8 bits is stochastic: with b2 = 0.999 one step moves u by far
// less than half a step of a 3-bit mantissa, so rounding to nearest would
// freeze it. The 32 random bits of an element are an integer hash of (its
// number in its tensor, the step), 16 for each moment, so a step is a pure
// function of its inputs. A u that is not zero never rounds to zero: the next
// step divides by it. Everything before that rounding is fp32; the weight
// update uses m and u before they are rounded.
//
// Bound by memory: 16 bytes an element with fp32 gradients (weight read and
// written, gradient read, two one-byte moments read and written) and 8 bytes a
// block for each scale; 407 million parameters in 121 tensors take 1.16 to
// 1.27 ms by the GPU, 5.1 to 5.6 TB/s (a copy runs at 6.56), with three quarters
// of the issue slots taken. One warp takes a block of 256 elements, which makes
// the scale one warp-wide integer maximum (magnitudes of floats order as
// their bits), and each lane two groups of 4 elements, so all loads and stores
// of a warp are whole lines.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include "adamw8_kernel.h"

namespace abacus {
namespace ops {
namespace {

constexpr unsigned kInfinity = 0x7f800000u;

__device__ __forceinline__ unsigned mix(unsigned element, unsigned step_mix) {
  unsigned x = element * 0x9E3779B1u + step_mix;
  x = (x ^ (x >> 16)) * 0x6C62272Fu;
  x = (x ^ (x >> 15)) * 0x2F0B4C47u;
  return x ^ (x >> 16);
}

// The larger of `top` and |x|, NaN if either is.
__device__ __forceinline__ float largest(float top, float x) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(top), "f"(fabsf(x)));
  return y;
}
// Over the warp, as bits (of numbers that are not negative, which order as their bits do, NaN last).
__device__ __forceinline__ unsigned warp_top(float top) { return __reduce_max_sync(0xffffffffu, __float_as_uint(top)); }

// The special-function unit's root and 1 / (2 root); tiny enough not to matter, the sum keeps the latter finite at zero.
__device__ __forceinline__ float root(float x) {
  float y;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float half_over_root(float x) {
  float y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fmaf(x, 4.f, 0x1p-126f)));
  return y;
}

// The root of x rounded to nearest, from an approximation s of it: one step of Heron's method, s + (x - s^2) / (2 s) with
// the difference exact, is off by the square of s's error, so its rounding is the root's but for one number in a million.
// The moment that is kept needs that (which of two codes a number gets depends on its last bit where it meets its
// threshold, and one code is an eighth of it), the weight's update does not. The library's correctly rounded root took
// 586 to 1077 us for 200 million elements, by the blocks an SM that its registers leave; this one 580.
__device__ __forceinline__ float polished(float s, float x) { return fmaf(fmaf(-s, s, x), half_over_root(x), s); }

// The e4m3 code of x, rounded stochastically by 16 random bits; |x| < 256. Times 2^-120, e4m3's smallest normal number
// (2^-6) is fp32's (2^-126) and the two formats' exponent fields agree, subnormal numbers included: the code is the upper
// bits of the float, and adding the random bits below them before they are cut rounds up with the right probability and
// carries into the exponent where it should. (fp32 keeps 20 bits below the grid; what it drops in a subnormal product is
// rounded to nearest first.)
__device__ __forceinline__ uint32_t to_code(float x, unsigned noise16) {  // x times 2^-120
  const uint32_t t = __float_as_uint(x) + (noise16 << 4);
  return (t << 4) | (t & 0x80000000u);  // in the top byte
}
__device__ __forceinline__ uint32_t to_code_positive(float x, unsigned noise16) {
  return (__float_as_uint(x) + (noise16 << 4)) >> 20;  // in the lowest byte
}
__device__ __forceinline__ uint32_t top_bytes(const uint32_t (&x)[4]) {
  return __byte_perm(__byte_perm(x[0], x[1], 0x0073), __byte_perm(x[2], x[3], 0x0073), 0x5410);
}
__device__ __forceinline__ uint32_t low_bytes(const uint32_t (&x)[4]) {
  return __byte_perm(__byte_perm(x[0], x[1], 0x0040), __byte_perm(x[2], x[3], 0x0040), 0x5410);
}

__device__ __forceinline__ void unpack4(uint32_t codes, float (&x)[4]) {
  const __half2 lo(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes & 0xffffu), __NV_E4M3));
  const __half2 hi(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes >> 16), __NV_E4M3));
  const float2 a = __half22float2(lo), b = __half22float2(hi);
  x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
}

__global__ void __launch_bounds__(kAdam8Warps * 32, 6) adamw8_kernel(const __grid_constant__ Adam8Batch t, const Adam8Scalars s) {
  int lo = t.coarse[blockIdx.x >> t.shift];
  while (t.first[lo + 1] <= blockIdx.x) ++lo;
  const int lane = threadIdx.x % 32;
  const long long n = t.numel[lo];
  const long long block = static_cast<long long>(blockIdx.x - t.first[lo]) * kAdam8Warps + threadIdx.x / 32;
  const long long begin = block * kAdam8Block;
  if (begin >= n) return;
  const bool whole = t.wide[lo] && begin + kAdam8Block <= n;
  float* wp = t.w[lo] + begin;
  uint8_t* mp = t.m[lo] + begin;
  uint8_t* up = t.u[lo] + begin;

  // All loads first; the moments stay packed until they are used, and a weight leaves as soon as it is done.
  float w[2][4], g[2][4], m[2][4], u[2][4];
  uint32_t mc[2], uc[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = h * 128 + lane * 4;
    if (whole) {
      const float4 w4 = *reinterpret_cast<const float4*>(wp + i);
      w[h][0] = w4.x; w[h][1] = w4.y; w[h][2] = w4.z; w[h][3] = w4.w;
      if (t.g_bf16[lo]) {
        const uint2 raw = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(t.g[lo]) + begin + i);
        g[h][0] = __uint_as_float(raw.x << 16); g[h][1] = __uint_as_float(raw.x & 0xffff0000u);
        g[h][2] = __uint_as_float(raw.y << 16); g[h][3] = __uint_as_float(raw.y & 0xffff0000u);
      } else {
        const float4 g4 = *reinterpret_cast<const float4*>(static_cast<const float*>(t.g[lo]) + begin + i);
        g[h][0] = g4.x; g[h][1] = g4.y; g[h][2] = g4.z; g[h][3] = g4.w;
      }
      mc[h] = *reinterpret_cast<const uint32_t*>(mp + i);
      uc[h] = *reinterpret_cast<const uint32_t*>(up + i);
    } else {
      mc[h] = uc[h] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in = begin + i + e < n;
        w[h][e] = in ? wp[i + e] : 0.f;
        g[h][e] = !in ? 0.f
                  : t.g_bf16[lo] ? __bfloat162float(static_cast<const __nv_bfloat16*>(t.g[lo])[begin + i + e])
                                 : static_cast<const float*>(t.g[lo])[begin + i + e];
        mc[h] |= in ? static_cast<uint32_t>(mp[i + e]) << (8 * e) : 0u;
        uc[h] |= in ? static_cast<uint32_t>(up[i + e]) << (8 * e) : 0u;
      }
    }
  }

  const float ms = t.m_scale[lo][block], us = t.u_scale[lo][block];
  float m_max = 0.f, u_max = 0.f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = h * 128 + lane * 4;
    unpack4(mc[h], m[h]);
    unpack4(uc[h], u[h]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float gi = g[h][e];
      const float mi = __fadd_rn(__fmul_rn(m[h][e] * ms, s.b1), __fmul_rn(gi, s.c1));
      const float uo = u[h][e] * us;
      const float vi = __fadd_rn(__fmul_rn(__fmul_rn(uo, uo), s.b2), __fmul_rn(__fmul_rn(gi, gi), s.c2));
      const float near = root(vi), ui = polished(near, vi);
      w[h][e] = w[h][e] * s.decay - __fdividef(mi * s.step_size, near + s.eps);
      m[h][e] = mi;
      u[h][e] = ui;
      m_max = largest(m_max, mi);
      u_max = largest(u_max, ui);
    }
    if (whole) {
      *reinterpret_cast<float4*>(wp + i) = make_float4(w[h][0], w[h][1], w[h][2], w[h][3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (begin + i + e < n) wp[i + e] = w[h][e];
    }
  }
  unsigned m_top = warp_top(m_max), u_top = warp_top(u_max);
  const bool spoilt = max(m_top, u_top) >= kInfinity;  // somewhere in this block
  if (spoilt) {  // infinities and NaN set no scale
    m_max = u_max = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (isfinite(m[h][e])) m_max = largest(m_max, m[h][e]);
        if (isfinite(u[h][e])) u_max = largest(u_max, u[h][e]);
      }
    }
    m_top = warp_top(m_max);
    u_top = warp_top(u_max);
  }
  // Biased exponents of the scales; 1 (2^-126) is the smallest normal one.
  const int me = max(static_cast<int>(m_top >> 23) - 7, 1);
  const int ue = max(static_cast<int>(u_top >> 23) - 7, 1);
  // 1 / scale, times 2^-120 at once while that is a normal number (moments below 2^14).
  const bool usual = max(me, ue) <= 133;
  const float m_inv = __uint_as_float(static_cast<unsigned>(254 - me - (usual ? 120 : 0)) << 23);
  const float u_inv = __uint_as_float(static_cast<unsigned>(254 - ue - (usual ? 120 : 0)) << 23);
  if (lane == 0) {
    t.m_scale[lo][block] = __uint_as_float(static_cast<unsigned>(me) << 23);
    t.u_scale[lo][block] = __uint_as_float(static_cast<unsigned>(ue) << 23);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = h * 128 + lane * 4;
    uint32_t mq[4], uq[4];
    if (usual) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned noise = mix(static_cast<unsigned>(begin + i + e), s.step_mix);
        mq[e] = to_code(m[h][e] * m_inv, noise & 0xffffu);
        uq[e] = max(to_code_positive(u[h][e] * u_inv, noise >> 16), min(__float_as_uint(u[h][e]), 1u));
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned noise = mix(static_cast<unsigned>(begin + i + e), s.step_mix);
        mq[e] = to_code(m[h][e] * m_inv * 0x1p-120f, noise & 0xffffu);
        uq[e] = max(to_code_positive(u[h][e] * u_inv * 0x1p-120f, noise >> 16), min(__float_as_uint(u[h][e]), 1u));
      }
    }
    uint32_t m_codes = top_bytes(mq), u_codes = low_bytes(uq);
    if (spoilt) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t byte = 0xffu << (8 * e), nan = 0x7fu << (8 * e);
        if (!isfinite(m[h][e])) m_codes = (m_codes & ~byte) | nan;
        if (!isfinite(u[h][e])) u_codes = (u_codes & ~byte) | nan;
      }
    }
    if (whole) {
      *reinterpret_cast<uint32_t*>(mp + i) = m_codes;
      *reinterpret_cast<uint32_t*>(up + i) = u_codes;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (begin + i + e < n) {
          mp[i + e] = static_cast<uint8_t>(m_codes >> (8 * e));
          up[i + e] = static_cast<uint8_t>(u_codes >> (8 * e));
        }
      }
    }
  }
}

}  // namespace

cudaError_t launch_adamw8(const Adam8Batch& batch, const Adam8Scalars& scalars, unsigned ctas, cudaStream_t stream) {
  adamw8_kernel<<<ctas, kAdam8Warps * 32, 0, stream>>>(batch, scalars);
  return cudaGetLastError();
}

}  // namespace ops
}  // namespace abacus
