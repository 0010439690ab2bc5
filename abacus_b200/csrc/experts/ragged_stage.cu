// Operands of the ragged products that TMA cannot read as they are: fp32 ones
// (split into bf16 parts), and bf16 ones whose rows are not 16-byte aligned.
// Bound by memory: 4 bytes read and 2 per plane written an element. A thread
// makes 8 columns: two 16-byte loads where the layout allows, one 16-byte
// store per plane.
#include <cuda_bf16.h>
#include "../common/sm100.cuh"
#include "ragged.h"
#include "sigmoid.cuh"
#include "split.cuh"

namespace abacus {
namespace ragged {
namespace {

__global__ void __launch_bounds__(256) stage_kernel(const StageParams p, bool vec, long long groups) {
  const long long per_row = p.ld / 8;
  const long long plane = p.batch * p.rows * p.ld;
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < groups;
       i += static_cast<long long>(gridDim.x) * blockDim.x) {
    const long long row = i / per_row;  // of all batches
    const long long c0 = (i - row * per_row) * 8;
    const long long b = row / p.rows, r = row - b * p.rows;
    if (p.offsets != nullptr && p.offsets[b + 1] <= (b == 0 ? 0 : p.offsets[b])) continue;
    const long long at = b * p.stride_batch + r * p.stride_row + c0 * p.stride_col;
    uint4 words[3];
    if (p.src_bf16) {
      const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(p.src) + at;
      uint16_t x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = c0 + j < p.cols ? *reinterpret_cast<const uint16_t*>(src + j * p.stride_col) : 0;
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = x[2 * j] | (static_cast<uint32_t>(x[2 * j + 1]) << 16);
      words[0] = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      const float* src = static_cast<const float*>(p.src) + at;
      float x[8];
      if (vec) {  // whole groups of 8 columns, 16-byte aligned
        const float4 u = *reinterpret_cast<const float4*>(src), v = *reinterpret_cast<const float4*>(src + 4);
        x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
        x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = c0 + j < p.cols ? src[j * p.stride_col] : 0.f;
      }
      split_eight(x, words);
    }
    __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.dst) + row * p.ld + c0;
#pragma unroll
    for (int q = 0; q < 3; ++q)
      if (q < p.planes) *reinterpret_cast<uint4*>(dst + q * plane) = words[q];
  }
}

// A thread makes 8 columns: 12 bytes read (dh, g, u) and 4 per plane written (dg, du) an element.
__global__ void __launch_bounds__(256) swiglu_bwd_kernel(const SwiGLUBwdParams p, long long groups) {
  const long long per_row = p.ld_out / 8, plane = p.rows * p.ld_out;
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < groups;
       i += static_cast<long long>(gridDim.x) * blockDim.x) {
    const long long row = i / per_row, c0 = (i - row * per_row) * 8;
    float d[8], g[8], u[8];
#pragma unroll
    for (int q = 0; q < 8; q += 4) {
      const long long at = row * p.ld + c0 + q;
      const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
      const bool in = c0 + q < p.ld;  // rows are padded to 4 columns, the results' to 8
      const float4 a = in ? *reinterpret_cast<const float4*>(p.dh + at) : zero;
      const float4 b = in ? *reinterpret_cast<const float4*>(p.g + at) : zero;
      const float4 c = in ? *reinterpret_cast<const float4*>(p.u + at) : zero;
      d[q] = a.x; d[q + 1] = a.y; d[q + 2] = a.z; d[q + 3] = a.w;
      g[q] = b.x; g[q + 1] = b.y; g[q + 2] = b.z; g[q + 3] = b.w;
      u[q] = c.x; u[q + 1] = c.y; u[q + 2] = c.z; u[q + 3] = c.w;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float sig = sigmoid<24>(g[j]);
      const float through = d[j] * sig;
      d[j] = through * u[j] * (1.f + g[j] * (1.f - sig));
      g[j] *= through;
    }
    uint4 dg[3], du[3];
    split_eight(d, dg);
    split_eight(g, du);
    const long long to = row * p.ld_out + c0;
#pragma unroll
    for (int q = 0; q < 3; ++q) {
      if (q < p.planes) {
        *reinterpret_cast<uint4*>(p.dg + q * plane + to) = dg[q];
        *reinterpret_cast<uint4*>(p.du + q * plane + to) = du[q];
      }
    }
  }
}

}  // namespace

cudaError_t launch_swiglu_bwd(const SwiGLUBwdParams& p, int sms, cudaStream_t stream) {
  const long long groups = p.rows * (p.ld_out / 8);
  if (groups == 0) return cudaSuccess;
  const long long blocks = (groups + 255) / 256, most = static_cast<long long>(sms) * 32;
  swiglu_bwd_kernel<<<static_cast<unsigned>(blocks < most ? blocks : most), 256, 0, stream>>>(p, groups);
  return cudaGetLastError();
}

cudaError_t launch_stage(const StageParams& p, int sms, cudaStream_t stream) {
  const long long groups = p.batch * p.rows * (p.ld / 8);
  if (groups == 0) return cudaSuccess;
  const bool vec = !p.src_bf16 && p.stride_col == 1 && p.cols % 8 == 0 && p.stride_row % 4 == 0 &&
                   p.stride_batch % 4 == 0 && reinterpret_cast<uintptr_t>(p.src) % 16 == 0;
  const long long blocks = (groups + 255) / 256, most = static_cast<long long>(sms) * 32;
  stage_kernel<<<static_cast<unsigned>(blocks < most ? blocks : most), 256, 0, stream>>>(p, vec, groups);
  return cudaGetLastError();
}

cudaError_t launch(const Params& p, const Shape& s, long long units, int sms, cudaStream_t stream) {
  if (s.planes == 1)
    return s.pair ? launch_shape<1, true>(p, s, units, sms, stream) : launch_shape<1, false>(p, s, units, sms, stream);
  if (s.planes == 2)
    return s.pair ? launch_shape<2, true>(p, s, units, sms, stream) : launch_shape<2, false>(p, s, units, sms, stream);
  if (s.planes == 3)
    return s.pair ? launch_shape<3, true>(p, s, units, sms, stream) : launch_shape<3, false>(p, s, units, sms, stream);
  return cudaErrorInvalidValue;
}

}  // namespace ragged
}  // namespace abacus
