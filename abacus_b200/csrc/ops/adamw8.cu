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
// block for each scale. One warp takes a block of 256 elements, which makes
// the scale one warp-wide integer maximum (magnitudes of floats order as
// their bits), and each lane two groups of 4 elements, so all loads and stores
// of a warp are whole lines.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cmath>
#include <cstring>
#include "../common/host.h"
#include "adamw8.h"

namespace abacus {
namespace ops {
namespace {

constexpr int kBlock = 256;    // elements that share a scale (one warp)
constexpr int kWarps = 8;      // of a CTA
constexpr int kRounds = 4;     // blocks of a tensor taken by a warp of a large launch, to share finding the tensor
constexpr unsigned kInfinity = 0x7f800000u;
constexpr int kTensors = 128;  // tensors of one launch (their table is the kernel's argument)

struct Adam8Batch {
  float* w[kTensors];
  const void* g[kTensors];
  uint8_t* m[kTensors];
  float* m_scale[kTensors];
  uint8_t* u[kTensors];
  float* u_scale[kTensors];
  long long numel[kTensors];
  unsigned first[kTensors + 1];  // first CTA of each tensor
  uint8_t g_bf16[kTensors], wide[kTensors];
  int count;
  int rounds;  // blocks a warp
};
static_assert(sizeof(Adam8Batch) < 16 * 1024, "the table has to fit the kernel's arguments");

struct Adam8Scalars {
  float b1, c1, b2, c2, eps, decay, step_size;
  unsigned step_mix;
};

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

// The special-function unit's root (within 2^-22): a last-bit error of u is far below its rounding to 8 bits, and
// the correctly rounded root is a dozen instructions in a kernel that is short of issue slots.
__device__ __forceinline__ float root(float x) {
  float y;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The e4m3 code of x, rounded stochastically by 16 random bits; |x| < 256. Times 2^-120, e4m3's smallest normal number
// (2^-6) is fp32's (2^-126) and the two formats' exponent fields agree, subnormal numbers included: the code is the upper
// bits of the float, and adding the random bits below them before they are cut rounds up with the right probability and
// carries into the exponent where it should. (fp32 keeps 20 bits below the grid; what it drops in a subnormal product is
// rounded to nearest first.)
__device__ __forceinline__ uint32_t to_code(float x, unsigned noise16) {
  const uint32_t t = __float_as_uint(x * 0x1p-120f) + (noise16 << 4);
  return (t << 4) | (t & 0x80000000u);  // in the top byte
}
__device__ __forceinline__ uint32_t to_code_positive(float x, unsigned noise16) {
  return (__float_as_uint(x * 0x1p-120f) + (noise16 << 4)) >> 20;  // in the lowest byte
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

__global__ void __launch_bounds__(kWarps * 32, 5) adamw8_kernel(const __grid_constant__ Adam8Batch t, const Adam8Scalars s) {
  int lo = 0, hi = t.count - 1;  // the tensor of this CTA: the last whose first CTA is not after it
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (t.first[mid] <= blockIdx.x) lo = mid;
    else hi = mid - 1;
  }
  const int lane = threadIdx.x % 32;
  const long long n = t.numel[lo];
  long long block = static_cast<long long>(blockIdx.x - t.first[lo]) * (kWarps * t.rounds) + threadIdx.x / 32;
#pragma unroll 1
  for (int round = 0; round < t.rounds; ++round, block += kWarps) {
    const long long begin = block * kBlock;
    if (begin >= n) return;
    const bool whole = t.wide[lo] && begin + kBlock <= n;
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
        const float ui = root(__fadd_rn(__fmul_rn(__fmul_rn(uo, uo), s.b2), __fmul_rn(__fmul_rn(gi, gi), s.c2)));
        w[h][e] = w[h][e] * s.decay - __fdividef(mi * s.step_size, ui + s.eps);
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
    const float m_inv = __uint_as_float(static_cast<unsigned>(254 - me) << 23);
    const float u_inv = __uint_as_float(static_cast<unsigned>(254 - ue) << 23);
    if (lane == 0) {
      t.m_scale[lo][block] = __uint_as_float(static_cast<unsigned>(me) << 23);
      t.u_scale[lo][block] = __uint_as_float(static_cast<unsigned>(ue) << 23);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = h * 128 + lane * 4;
      uint32_t mq[4], uq[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned noise = mix(static_cast<unsigned>(begin + i + e), s.step_mix);
        mq[e] = to_code(m[h][e] * m_inv, noise & 0xffffu);
        uq[e] = max(to_code_positive(u[h][e] * u_inv, noise >> 16), min(__float_as_uint(u[h][e]), 1u));
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
}

bool aligned(const void* p, unsigned bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace

void adamw8_step(const std::vector<torch::Tensor>& weights, const std::vector<torch::Tensor>& grads,
                 const std::vector<torch::Tensor>& exp_avg, const std::vector<torch::Tensor>& exp_avg_scale,
                 const std::vector<torch::Tensor>& exp_rms, const std::vector<torch::Tensor>& exp_rms_scale, double lr,
                 double beta1, double beta2, double eps, double weight_decay, int64_t step) {
  const size_t count = weights.size();
  TORCH_CHECK(grads.size() == count && exp_avg.size() == count && exp_avg_scale.size() == count &&
                  exp_rms.size() == count && exp_rms_scale.size() == count,
              "adamw8: the lists differ in length");
  TORCH_CHECK(step >= 1, "adamw8: step must be at least 1, got ", step);
  if (count == 0) return;
  const c10::cuda::CUDAGuard guard(weights[0].device());
  Adam8Scalars s;
  s.b1 = static_cast<float>(beta1);
  s.c1 = static_cast<float>(1.0 - beta1);
  s.b2 = static_cast<float>(beta2);
  s.c2 = static_cast<float>(1.0 - beta2);
  // a m / (u / c + eps) = (a c) m / (u + eps c): one division an element.
  const double c = std::sqrt(1.0 - std::pow(beta2, static_cast<double>(step)));
  s.eps = static_cast<float>(eps * c);
  s.decay = static_cast<float>(1.0 - lr * weight_decay);
  s.step_size = static_cast<float>(lr * c / (1.0 - std::pow(beta1, static_cast<double>(step))));
  s.step_mix = static_cast<unsigned>(static_cast<uint64_t>(step) * 0x7F4A7C15ull);
  const auto stream = at::cuda::getCurrentCUDAStream();
  // Every tensor is looked at before the first is changed.
  for (size_t i = 0; i < count; ++i) {
    const auto &w = weights[i], &g = grads[i], &m = exp_avg[i], &u = exp_rms[i], &ms = exp_avg_scale[i],
               &us = exp_rms_scale[i];
    const int64_t n = w.numel(), blocks = (n + kBlock - 1) / kBlock;
    for (const auto* t : {&w, &g, &m, &u, &ms, &us}) {
      TORCH_CHECK(t->is_cuda() && t->device() == weights[0].device() && t->is_contiguous(),
                  "adamw8: tensors must be contiguous and on one CUDA device (tensor ", i, ")");
    }
    TORCH_CHECK(w.scalar_type() == torch::kFloat32 && ms.scalar_type() == torch::kFloat32 &&
                    us.scalar_type() == torch::kFloat32 && m.scalar_type() == torch::kFloat8_e4m3fn &&
                    u.scalar_type() == torch::kFloat8_e4m3fn &&
                    (g.scalar_type() == torch::kFloat32 || g.scalar_type() == torch::kBFloat16),
                "adamw8: fp32 weights and scales, float8_e4m3fn moments, fp32 or bf16 gradients (tensor ", i, ")");
    TORCH_CHECK(g.numel() == n && m.numel() == n && u.numel() == n && ms.numel() == blocks && us.numel() == blocks,
                "adamw8: sizes of tensor ", i, " (", n, " weights need ", blocks, " scales of each moment)");
    TORCH_CHECK(blocks < (1ll << 31), "adamw8: tensor ", i, " is too large");
  }
  // One block a warp while that leaves the launch within what the GPU holds at once, so that a small one is spread over
  // all of it (3.2 us against 6.9 for 100 thousand elements); else several (1152 us against 1193 for 407 million).
  unsigned long long all_blocks = 0;
  for (const auto& w : weights) all_blocks += (w.numel() + kBlock - 1) / kBlock;
  const int sms = at::cuda::getDeviceProperties(weights[0].get_device())->multiProcessorCount;
  Adam8Batch b;
  unsigned long long ctas = 0;
  b.count = 0;
  b.rounds = all_blocks > 5ull * sms * kWarps ? kRounds : 1;
  auto flush = [&] {
    if (b.count == 0) return;
    b.first[b.count] = static_cast<unsigned>(ctas);
    adamw8_kernel<<<static_cast<unsigned>(ctas), kWarps * 32, 0, stream>>>(b, s);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    host::note_launch();
    b.count = 0;
    ctas = 0;
  };
  for (size_t i = 0; i < count; ++i) {
    const int64_t n = weights[i].numel();
    if (n == 0) continue;
    const int64_t per_cta = static_cast<int64_t>(kBlock) * kWarps * b.rounds;
    const unsigned long long need = (n + per_cta - 1) / per_cta;
    if (b.count == kTensors || ctas + need >= (1ull << 31)) flush();
    const int c = b.count++;
    b.w[c] = weights[i].data_ptr<float>();
    b.g[c] = grads[i].data_ptr();
    b.m[c] = static_cast<uint8_t*>(exp_avg[i].data_ptr());
    b.m_scale[c] = exp_avg_scale[i].data_ptr<float>();
    b.u[c] = static_cast<uint8_t*>(exp_rms[i].data_ptr());
    b.u_scale[c] = exp_rms_scale[i].data_ptr<float>();
    b.numel[c] = n;
    b.first[c] = static_cast<unsigned>(ctas);
    b.g_bf16[c] = grads[i].scalar_type() == torch::kBFloat16;
    b.wide[c] = aligned(b.w[c], 16) && aligned(b.g[c], b.g_bf16[c] ? 8 : 16) && aligned(b.m[c], 4) && aligned(b.u[c], 4);
    ctas += need;
  }
  flush();
}

}  // namespace ops
}  // namespace abacus
