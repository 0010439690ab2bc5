// One launch of the AdamW step with 8-bit moments (see adamw8_kernel.cu).
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

namespace abacus {
namespace ops {

constexpr int kAdam8Block = 256;    // elements that share a scale (one warp)
constexpr int kAdam8Warps = 8;      // blocks of a tensor taken by one CTA
constexpr int kAdam8Tensors = 128;  // tensors of one launch (their table is the kernel's argument)

struct Adam8Batch {
  float* w[kAdam8Tensors];
  const void* g[kAdam8Tensors];
  uint8_t* m[kAdam8Tensors];
  float* m_scale[kAdam8Tensors];
  uint8_t* u[kAdam8Tensors];
  float* u_scale[kAdam8Tensors];
  long long numel[kAdam8Tensors];
  unsigned first[kAdam8Tensors + 1];  // first CTA of each tensor
  uint8_t g_bf16[kAdam8Tensors], wide[kAdam8Tensors];
  // The tensor of a CTA: coarse[CTA >> shift] is that of the first CTA of its run of 2^shift, and few tensors end inside a
  // run (a search through `first` cost every CTA seven dependent loads before its own).
  uint8_t coarse[256];
  int shift;
  int count;
};
static_assert(sizeof(Adam8Batch) < 16 * 1024, "the table has to fit the kernel's arguments");

struct Adam8Scalars {
  float b1, c1, b2, c2, eps, decay, step_size;
  unsigned step_mix;
};

cudaError_t launch_adamw8(const Adam8Batch& batch, const Adam8Scalars& scalars, unsigned ctas, cudaStream_t stream);

}  // namespace ops
}  // namespace abacus
